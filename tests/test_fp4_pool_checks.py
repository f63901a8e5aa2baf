"""The 4-bit pool's refusals and its block records' header, on the CPU."""

import pytest
import torch

from mini_infra_qwen3_amd.model import PagedAttentionMetadata, Qwen3Config, Qwen3ForCausalLM
from mini_infra_qwen3_amd.worker import KVBlockHeader, PagedKVCachePoolFp4


@pytest.mark.skipif(torch.cuda.device_count() > 0, reason="host-only: placeholder pointers")
def test_norm_rope_entry_refuses(native_lib):
    good = dict(q_out=16, k_out=None, v_out=None, q=16, q_stride=2048, k=16, k_stride=1024, v=16, v_stride=1024, q_weight=16,
                k_weight=16, cos=16, sin=16, tokens=3, heads=16, kv_heads=8, dim=128, eps=1e-6, slots=8, slot_stride=1,
                key_pool=16, value_pool=16, num_slots=32, stream=None)
    call = lambda **kw: native_lib.mi_qk_norm_rope_fp4(*{**good, **kw}.values())  # noqa: E731
    assert call(tokens=0) == 0
    for bad in (dict(tokens=-1), dict(heads=0), dict(kv_heads=0), dict(num_slots=-1), dict(dim=64), dict(q=None), dict(cos=None),
                dict(slots=None), dict(key_pool=None), dict(value_pool=None), dict(k_out=16), dict(slot_stride=0),
                dict(q_stride=2040), dict(k_stride=1016), dict(q=18), dict(v=8), dict(key_pool=8), dict(q_weight=4),
                dict(k_out=8, v_out=16), dict(v_stride=1028), dict(tokens=1 << 40)):
        assert call(**bad) != 0, bad
        assert b"mi_qk_norm_rope_fp4" in native_lib.mi_last_error()


def test_pool_needs_a_gpu():
    with pytest.raises(RuntimeError, match="GPU"):
        PagedKVCachePoolFp4(1, 4, 16, 8, 128, "cpu")


@pytest.mark.parametrize("geometry", [(0, 4, 16, 8, 128), (1, 0, 16, 8, 128), (1, 4, 24, 8, 128), (1, 4, 0, 8, 128),
                                      (1, 4, 16, 0, 128), (1, 4, 16, 8, 64)])
def test_pool_geometry(geometry):
    with pytest.raises(ValueError):
        PagedKVCachePoolFp4(*geometry, "cuda:0")


def test_record_header_of_4_bit_blocks():
    header = KVBlockHeader(28, 32, 8, 128, torch.uint8, 3, 7)
    raw = header.encode()
    assert int.from_bytes(raw[32:36], "little") == 4 and int.from_bytes(raw[36:40], "little") == 1
    assert header.record_shape == (28, 2, 2, 8, 1088)
    assert int.from_bytes(raw[48:56], "little") == header.record_bytes == 28 * 2 * 2 * 8 * 1088
    assert KVBlockHeader.decode(raw) == header
    for block_size, dim in ((24, 128), (32, 64)):
        bad = raw[:20] + block_size.to_bytes(4, "little") + raw[24:28] + dim.to_bytes(4, "little") + raw[32:]
        with pytest.raises(ValueError, match="4-bit"):
            KVBlockHeader.decode(bad)


def test_reference_numerics_refuse_a_4_bit_pool():
    config = Qwen3Config(vocab_size=10, hidden_size=256, intermediate_size=256, num_hidden_layers=1, num_attention_heads=2,
                         num_key_value_heads=1, head_dim=128)
    pools = ((torch.zeros(2, 1, 1, 1088, dtype=torch.uint8),) * 2,)
    ids = torch.zeros(1, 1, dtype=torch.long)
    meta = PagedAttentionMetadata(ids[:, 0], ids, ids[:, 0], pools)
    with pytest.raises(ValueError, match="exact=False"):
        Qwen3ForCausalLM(config)(ids, position_ids=ids, attn_metadata=meta)
