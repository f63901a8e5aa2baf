"""The 4-bit cache's entry points and block copies refuse bad calls on the host, before any launch; the oracle's own
format facts (all on the CPU)."""

import ctypes

import numpy as np
import pytest
import torch

from mini_infra_qwen3_amd import _native, data_plane
from oracle import fp4_ref

# The C calls hand placeholder pointers to calls that are refused: only without a visible device.
host_only = pytest.mark.skipif(torch.cuda.device_count() > 0, reason="host-only: placeholder pointers")
BAD, UNSUPPORTED, WORKSPACE, OK = (_native.MI_ERR_INVALID_ARGUMENT, _native.MI_ERR_UNSUPPORTED, _native.MI_ERR_WORKSPACE,
                                   _native.MI_OK)


def ptrs(*values):
    return (ctypes.c_void_p * len(values))(*values)


@host_only
@pytest.mark.parametrize("change,code", [
    ({"tokens": -1}, BAD), ({"slots": None}, BAD), ({"kv": 0}, BAD), ({"dim": 64}, UNSUPPORTED), ({"type": 9}, BAD),
    ({"stride": 0}, BAD), ({"pools": 24}, UNSUPPORTED), ({"keys": None}, BAD), ({"tokens": 1 << 40}, UNSUPPORTED),
    ({"tokens": 0}, OK), ({"rows": 0}, OK)])
def test_store_refusals(native_lib, change, code):
    a = {"tokens": 4, "slots": 16, "kv": 8, "dim": 128, "type": 1, "stride": 1, "pools": 16, "keys": 16, "rows": 1, **change}
    assert native_lib.mi_reshape_and_cache_fp4(
        ptrs(a["keys"]), ptrs(16), 0, 0, 0, 0, 0, 0, None, None, a["slots"], a["stride"], a["tokens"], a["rows"], 1,
        ptrs(a["pools"]), ptrs(16), 1, 64, a["kv"], a["dim"], a["type"], None) == code


@host_only
def test_store_checks_every_layer_before_the_first_launch(native_lib):
    """A null pointer in a layer of the second launch (more than 32 layers) refuses the whole call."""
    good = [16] * 40
    bad = good[:39] + [0]
    for keys, pools in ((bad, good), (good, bad)):
        assert native_lib.mi_reshape_and_cache_fp4(
            ptrs(*keys), ptrs(*good), 0, 0, 0, 0, 0, 0, None, None, 16, 1, 4, 1, 1, ptrs(*pools), ptrs(*good), 40, 64, 8, 128, 1,
            None) == BAD
    assert native_lib.mi_gather_blocks_fp4(ptrs(*good), ptrs(*bad), 8, 16, 4, 2, 4, ptrs(*good), ptrs(*good), 40, 8, 128,
                                           None) == BAD
    assert native_lib.mi_copy_blocks(ptrs(*good), ptrs(*bad), 8, 16, 16, 1, 40, 64, None) == BAD


@host_only
@pytest.mark.parametrize("change,code", [
    ({"batch": -1}, BAD), ({"blocks": 0}, BAD), ({"ids": None}, BAD), ({"stride": 3}, BAD), ({"dim": 64}, UNSUPPORTED),
    ({"kv": 0}, BAD), ({"out": 8}, UNSUPPORTED), ({"batch": 1 << 24}, UNSUPPORTED), ({"batch": 0}, OK)])
def test_gather_refusals(native_lib, change, code):
    a = {"batch": 2, "blocks": 8, "ids": 16, "stride": 4, "dim": 128, "kv": 8, "out": 16, **change}
    assert native_lib.mi_gather_blocks_fp4(ptrs(16), ptrs(16), a["blocks"], a["ids"], a["stride"], a["batch"], 4, ptrs(a["out"]),
                                           ptrs(16), 1, a["kv"], a["dim"], None) == code


@host_only
@pytest.mark.parametrize("change,code", [
    ({"batch": -1}, BAD), ({"batch": 0}, OK), ({"out": None}, BAD), ({"tables": None}, BAD), ({"blocks": 0}, BAD),
    ({"dim": 64}, UNSUPPORTED), ({"heads": 20}, UNSUPPORTED), ({"heads": 72}, UNSUPPORTED), ({"q": 8}, UNSUPPORTED),
    ({"q_row": 2052}, UNSUPPORTED), ({"bt_stride": 3}, BAD), ({"ctx_stride": 0}, BAD), ({"blocks": 1 << 32}, UNSUPPORTED),
    ({"scale": float("nan")}, BAD), ({"scale": float("inf")}, BAD), ({"ws": None}, WORKSPACE), ({"ws_bytes": 64}, WORKSPACE),
    ({"ws": 24}, UNSUPPORTED), ({"pool": 8}, UNSUPPORTED)])
def test_decode_refusals(native_lib, change, code):
    a = {"batch": 2, "out": 16, "tables": 16, "blocks": 4096, "dim": 128, "heads": 16, "q": 16, "q_row": 2048,
         "bt_stride": 4000, "ctx_stride": 1, "scale": 0.1, "ws": 16, "ws_bytes": 1 << 40, "pool": 16, **change}
    assert native_lib.mi_paged_decode_attention_fp4(
        a["out"], 2048, a["q"], a["q_row"], 128, a["pool"], 16, a["blocks"], a["tables"], a["bt_stride"], 4000, 16,
        a["ctx_stride"], a["batch"], a["heads"], 8, a["dim"], a["scale"], a["ws"], a["ws_bytes"], None) == code


@host_only
def test_decode_workspace_sizes(native_lib):
    size = native_lib.mi_paged_decode_fp4_workspace_bytes
    assert size(0, 100, 16, 8) == 0 and size(4, 0, 16, 8) == 0 and size(4, 100, 17, 8) == 0
    assert size(1, 4096, 16, 8) > 0
    assert data_plane.paged_decode_fp4_workspace_bytes(3, 512, 16, 8, 32) == size(3, 1024, 16, 8)
    for batch in (1, 3, 64, 256):  # longer tables never need less
        assert size(batch, 256, 16, 8) <= size(batch, 8192, 16, 8)


@host_only
@pytest.mark.parametrize("change,code", [
    ({"batch": -1}, BAD), ({"batch": 0}, OK), ({"L": 0}, OK), ({"q": None}, BAD), ({"hist": None}, BAD), ({"blocks": 0}, BAD),
    ({"dim": 64}, UNSUPPORTED), ({"heads": 20}, UNSUPPORTED), ({"q_tok": 2052}, UNSUPPORTED), ({"k": 8}, UNSUPPORTED),
    ({"stride": 3}, BAD), ({"lens_stride": 0}, BAD), ({"k_tok": 1 << 24}, UNSUPPORTED), ({"pool": 8}, UNSUPPORTED),
    ({"nb": 1 << 27, "stride": 1 << 27}, UNSUPPORTED), ({"scale": float("inf")}, BAD), ({"batch": 1 << 28}, UNSUPPORTED),
    ({"nb": 4000, "stride": 4000, "ws": None}, WORKSPACE), ({"nb": 4000, "stride": 4000, "ws_bytes": 64}, WORKSPACE),
    ({"nb": 4000, "stride": 4000, "ws": 24}, UNSUPPORTED)])
def test_prefill_refusals(native_lib, change, code):
    a = {"batch": 2, "L": 32, "q": 16, "hist": 16, "blocks": 64, "dim": 128, "heads": 16, "q_tok": 2048, "k": 16, "stride": 4,
         "lens_stride": 1, "k_tok": 1024, "pool": 16, "nb": 4, "scale": 0.1, "ws": 16, "ws_bytes": 1 << 40, **change}
    assert native_lib.mi_chunked_prefill_attention_fp4(
        16, 65536, 2048, a["q"], 65536, 128, a["q_tok"], a["k"], 32768, 128, a["k_tok"], 16, 32768, 128, 1024, a["pool"], 16,
        a["blocks"], a["hist"], a["stride"], a["nb"], 16, 16, a["lens_stride"], a["batch"], a["L"], a["heads"], 8, a["dim"],
        a["scale"], a["ws"], a["ws_bytes"], None) == code


@host_only
@pytest.mark.parametrize("change,code", [
    ({"pairs": -1}, BAD), ({"pairs": 0}, OK), ({"src": None}, BAD), ({"dst": None}, BAD), ({"pairs": 1 << 30}, UNSUPPORTED),
    ({"bytes": 1 << 36}, UNSUPPORTED), ({"blocks": 0}, OK)])
def test_copy_refusals(native_lib, change, code):
    a = {"pairs": 2, "src": 16, "dst": 16, "bytes": 64, "blocks": 8, **change}
    assert native_lib.mi_copy_blocks(ptrs(16), ptrs(16), a["blocks"], a["src"], a["dst"], a["pairs"], 1, a["bytes"], None) == code


def test_python_layer_takes_only_gpu_tensors():
    pool = torch.zeros(data_plane.fp4_pool_shape(4, 16, 2), dtype=torch.uint8)
    ids = torch.zeros(1, 1, dtype=torch.long)
    row = torch.zeros(1, 2, 1, 128, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="only on the GPU"):
        data_plane.reshape_and_cache_fp4([row], [row], ids[0], [pool], [pool])
    with pytest.raises(RuntimeError, match="only on the GPU"):
        data_plane.gather_blocks_fp4([pool], [pool], ids, [row], [row])
    with pytest.raises(RuntimeError, match="only on the GPU"):
        data_plane.paged_decode_attention_fp4(row[:, :, 0], pool, pool, ids, ids[0], 1.0)
    with pytest.raises(RuntimeError, match="only on the GPU"):
        data_plane.chunked_prefill_attention_fp4(row, row, row, pool, pool, ids, ids[0], ids[0], 1.0)
    with pytest.raises(RuntimeError, match="only on the GPU"):
        data_plane.copy_blocks([pool], [pool], ids[0], ids[0])


def test_pool_shape():
    assert data_plane.fp4_pool_shape(10, 16, 8) == (10, 1, 8, 1088)
    assert data_plane.fp4_pool_shape(10, 48, 3) == (10, 3, 3, 1088)
    for bad in ((10, 8, 8), (10, 24, 8), (10, 0, 8), (10, 16, 0), (-1, 16, 8)):
        with pytest.raises(ValueError):
            data_plane.fp4_pool_shape(*bad)
    with pytest.raises(ValueError):
        data_plane.fp4_pool_shape(10, 16, 8, head_dim=64)


# -------------------------------------------------------------------------------- the oracle
def test_oracle_quantiser():
    grid = fp4_ref.GRID
    x = np.zeros(128)
    x[:8] = grid
    x[32:40] = [0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0]  # the ties: to the even code
    x[64:67] = [7.0, 1.0, -0.25]                             # 7 takes the next scale
    x[96] = float("inf")
    codes, scales = fp4_ref.quantize_row(x)
    assert scales.tolist() == [127, 127, 128, 255]
    assert codes[:8].tolist() == list(range(8))
    assert codes[32:40].tolist() == [0, 2, 2, 4, 4, 6, 6, 7]
    assert codes[64:67].tolist() == [6, 1, 8]
    values = fp4_ref.values_of(codes, scales)
    assert values[:8].tolist() == grid.tolist() and values[64] == 8.0 and np.isnan(values[96:]).all()


def test_oracle_error_and_layout():
    """Every value within a quarter of its group's largest magnitude over 3.5 (half of the widest step, 2 s, at
    a >= 3.5 s), and what is stored is what is read, wherever it lies."""
    rng = np.random.default_rng(0)
    rows = rng.standard_normal((40, 2, 128)) * 2.0 ** rng.integers(-100, 100, (40, 2, 1))
    for value in (False, True):
        pool = np.zeros((3, 2, 1088), dtype=np.uint8)
        slots = rng.permutation(48)[:40]
        for s, row in zip(slots, rows):
            fp4_ref.store(pool, int(s), row, value)
        got = fp4_ref.load(pool, value).reshape(48, 2, 128)
        amax = np.repeat(np.abs(rows).reshape(40, 2, 4, 32).max(-1), 32, axis=-1)
        assert (np.abs(got[slots] - rows) <= amax / 3.5).all()
        rest = np.setdiff1d(np.arange(48), slots)
        assert not got[rest].any()
        at = {fp4_ref.code_at(value, t, d) for t in range(16) for d in range(128)}
        assert at == set(range(1024))
        assert {fp4_ref.scale_at(value, t, g) for t in range(16) for g in range(4)} == set(range(1024, 1088))
