"""The 4-bit pool's refusals and its block records' header, on the CPU."""

import pytest
import torch

from mini_infra_qwen3_amd.model import PagedAttentionMetadata, Qwen3Config, Qwen3ForCausalLM
from mini_infra_qwen3_amd.worker import KVBlockHeader, PagedKVCachePoolFp4


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
