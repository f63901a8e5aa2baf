"""Chunked prefill over 4-bit history with ragged rows, against the same rows left-padded (which the 64-bit oracle checks):
bit for bit, as only the rows' places in memory differ.  Tokens of no row hold NaN and must neither count nor be written."""

import numpy as np
import pytest
import torch

from mini_infra_qwen3_amd import _native, data_plane
from oracle import fp4_ref

SCALE = 128 ** -0.5
BAD, UNSUPPORTED, WORKSPACE = -1, -2, -3


def padded(rows, first, lens, width):
    """``[B, width, H, 128]`` left-padded copies of the rows' tokens of ``[C, H, 128]``."""
    out = torch.zeros(len(lens), width, *rows.shape[1:], dtype=rows.dtype, device=rows.device)
    for b, (at, n) in enumerate(zip(first, lens)):
        out[b, width - n:] = rows[at:at + n]
    return out


def case(device, seed, lens, starts, gaps, heads, kv_heads, table_width=None):
    gen = torch.Generator().manual_seed(seed)
    rng = np.random.default_rng(seed)
    first, at = [], 0
    for n, gap in zip(lens, gaps):
        first.append(at + gap)
        at += gap + n
    total = at + gaps[-1]
    q, k, v = (torch.full((total, h, 128), float("nan"), dtype=torch.bfloat16) for h in (heads, kv_heads, kv_heads))
    for t in (q, k, v):
        for f, n in zip(first, lens):
            t[f:f + n] = torch.randn(n, *t.shape[1:], generator=gen)
    counts = [-(-s // 16) for s in starts]
    table = np.zeros((len(lens), table_width or max(max(counts), 1)), dtype=np.int64)
    ids = rng.permutation(sum(counts) + 3) + 1
    for b, c in enumerate(counts):
        table[b, :c], ids = ids[:c], ids[c:]
    pools = [fp4_ref.to_torch(fp4_ref.random_pool(rng, sum(counts) + 4, kv_heads)).to(device) for _ in range(2)]
    move = lambda *x: [torch.as_tensor(t).to(device) for t in x]  # noqa: E731
    return move(q, k, v), pools, move(table, starts, lens, first), first


def run(tensors, pools, index, width, **kw):
    table, starts, lens, first = index
    return data_plane.chunked_prefill_attention_fp4(*(t.unsqueeze(0).transpose(1, 2) for t in tensors), *pools, table, starts, lens,
                                                    SCALE, chunk_first=first, max_len=width, **kw)


@pytest.mark.gpu
@pytest.mark.parametrize("lens,starts,gaps,heads,kv_heads,table_width", [
    ([1], [0], [0], 4, 2, None), ([1, 1, 1], [5, 0, 40], [0, 0, 0], 16, 8, None), ([70, 3, 0, 64], [33, 16, 7, 0], [2, 0, 5, 1], 16, 8, None),
    ([200, 333], [1500, 700], [0, 0], 16, 8, None),      # narrow
    ([40, 1, 60], [1000, 3, 2999], [1, 2, 3], 4, 2, 300),  # parts
    ([128] * 15, [0] * 15, [0] * 15, 16, 8, None), ([700, 650, 31], [40, 0, 9], [0, 64, 0], 16, 8, None), ([1500] * 6, [33] * 6, [1] * 6, 16, 8, None),
    ([90, 17], [100, 4], [0, 0], 5, 1, None), ([33, 95], [64, 31], [0, 0], 18, 2, None)])
def test_ragged_rows_are_the_padded_ones(native_lib, device, lens, starts, gaps, heads, kv_heads, table_width):
    tensors, pools, index, first = case(device, len(lens) + sum(lens), lens, starts, gaps, heads, kv_heads, table_width)
    width = max(lens)
    want = data_plane.chunked_prefill_attention_fp4(*(padded(t, first, lens, width).transpose(1, 2) for t in tensors), *pools,
                                                    *index[:3], SCALE)
    total = tensors[0].shape[0]
    out = torch.full((1, total, heads * 128), 7.0, dtype=torch.bfloat16, device=device)
    assert run(tensors, pools, index, width, out=out) is out
    expect = torch.full_like(out, 7.0)
    for b, (f, n) in enumerate(zip(first, lens)):
        expect[0, f:f + n] = want[b, width - n:]
    assert torch.equal(out, expect) and not bool(out.isnan().any())
    fresh = run(tensors, pools, index, width)
    covered = torch.zeros(total, dtype=torch.bool)
    for f, n in zip(first, lens):
        covered[f:f + n] = True
    assert torch.equal(fresh[0, covered], expect[0, covered]) and not fresh[0, ~covered].any()


@pytest.mark.gpu
@pytest.mark.parametrize("table_width", [None, 400])
def test_ragged_clamps(native_lib, device, table_width):
    """First tokens and lengths outside the tokens are moved inside; a length past max_len is cut to its first tokens."""
    lens, starts = [20, 30], [50, 20]
    tensors, pools, (table, start, _, _), first = case(device, 3, lens, starts, [0, 0], 4, 2, table_width)
    total = 50
    for given_first, given_lens, width, true_first, true_lens in (
            ([-3, 90], [20, 30], 30, [0, 20], [20, 30]), ([0, 20], [20, 30], 17, [0, 20], [17, 17]),
            ([0, 40], [-5, 999], 40, [0, 10], [0, 40]), ([0, 5], [0, 999], 60, [0, 0], [0, 50])):
        index = [table, start, torch.tensor(given_lens, device=device), torch.tensor(given_first, device=device)]
        out = torch.full((1, total, 512), 7.0, dtype=torch.bfloat16, device=device)
        run(tensors, pools, index, width, out=out)
        want = data_plane.chunked_prefill_attention_fp4(
            *(padded(t, true_first, true_lens, width).transpose(1, 2) for t in tensors), *pools, table, start,
            torch.tensor(true_lens, device=device), SCALE)
        expect = torch.full_like(out, 7.0)
        for b, (f, n) in enumerate(zip(true_first, true_lens)):
            expect[0, f:f + n] = want[b, width - n:]
        assert torch.equal(out, expect)


@pytest.mark.gpu
def test_ragged_graph_replays(native_lib, device):
    """Captured with empty rows, replayed with rows in other places, eager calls in between."""
    lens, starts = [40, 9, 25], [70, 0, 300]
    tensors, pools, index, first = case(device, 5, lens, starts, [3, 0, 2], 16, 8)
    total = tensors[0].shape[0]
    for t in tensors:
        t.nan_to_num_()
    static = [index[0], index[1], torch.zeros_like(index[2]), torch.zeros_like(index[3])]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run(tensors, pools, static, 50)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run(tensors, pools, static, 50)
    gen = torch.Generator().manual_seed(1)
    for step in range(4):
        for t in tensors:
            t.copy_(torch.randn(t.shape, generator=gen))
        static[2].copy_(torch.tensor([10 + step, 0 if step == 1 else 20, 30]))
        static[3].copy_(torch.tensor([0, 15, 40 + step]))
        eager = run(tensors, pools, static, 50)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, eager) and bool(out.any())
    assert total >= 73


@pytest.mark.gpu
def test_ragged_refusals_of_tensors(native_lib, device):
    tensors, pools, index, _ = case(device, 6, [5, 6], [0, 0], [0, 0], 4, 2)
    table, starts, lens, first = index
    views = [t.unsqueeze(0).transpose(1, 2) for t in tensors]
    call = lambda *a, **kw: data_plane.chunked_prefill_attention_fp4(*a, SCALE, **kw)  # noqa: E731
    with pytest.raises(ValueError, match="max_len"):
        call(*views, *pools, table, starts, lens, chunk_first=first)
    with pytest.raises(ValueError, match="one row"):
        call(*(torch.cat((t, t)) for t in views), *pools, table, starts, lens, chunk_first=first, max_len=6)
    with pytest.raises(ValueError, match="batch differs"):
        call(*views, *pools, table, starts, lens, chunk_first=first[:1], max_len=6)
    with pytest.raises(ValueError, match="int64"):
        call(*views, *pools, table, starts, lens, chunk_first=first.int(), max_len=6)
    with pytest.raises(ValueError, match="out must be"):
        call(*views, *pools, table, starts, lens, chunk_first=first, max_len=6, out=torch.zeros(2, 11, 512, dtype=torch.bfloat16, device=device))
    assert call(*views, *pools, table[:0], starts[:0], lens[:0], chunk_first=first[:0], max_len=6).shape == (1, 11, 512)
    assert not call(*views, *pools, table, starts, lens, chunk_first=first, max_len=0).any()


@pytest.mark.skipif(torch.cuda.device_count() > 0, reason="host-only: placeholder pointers")
@pytest.mark.parametrize("change,code", [
    ({"batch": 0}, 0), ({"tokens": 0}, 0), ({"max_len": 0}, 0), ({"batch": -1}, BAD), ({"tokens": -1}, BAD), ({"max_len": -1}, BAD),
    ({"first": None}, BAD), ({"first_stride": 0}, BAD), ({"lens_stride": 0}, BAD), ({"q": None}, BAD), ({"q": 24}, UNSUPPORTED),
    ({"k_tok": 1 << 24}, UNSUPPORTED), ({"q_tok": 2044}, UNSUPPORTED), ({"heads": 15}, UNSUPPORTED), ({"dim": 64}, UNSUPPORTED),
    ({"blocks": 0}, BAD), ({"stride": 3}, BAD), ({"scale": float("nan")}, BAD), ({"nb": 4000, "stride": 4000, "ws": None}, WORKSPACE)])
def test_ragged_entry_refuses(native_lib, change, code):
    a = {"batch": 2, "tokens": 40, "max_len": 32, "q": 16, "q_tok": 2048, "k_tok": 1024, "first": 16, "first_stride": 1, "lens_stride": 1,
         "heads": 16, "dim": 128, "blocks": 64, "nb": 4, "stride": 4, "scale": 0.1, "ws": 16, **change}
    assert native_lib.mi_ragged_prefill_attention_fp4(
        16, 2048, a["q"], 128, a["q_tok"], 16, 128, a["k_tok"], 16, 128, 1024, a["tokens"], 16, 16, a["blocks"], 16, a["stride"], a["nb"],
        16, 16, a["lens_stride"], a["first"], a["first_stride"], a["batch"], a["max_len"], a["heads"], 8, a["dim"], a["scale"], a["ws"],
        1 << 40, None) == code
    if code:
        assert b"mi_ragged_prefill_attention_fp4" in native_lib.mi_last_error()
    assert "mi_ragged_prefill_attention_fp4" in _native.SIGNATURES
