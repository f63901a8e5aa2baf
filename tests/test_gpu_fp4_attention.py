"""Attention over the 4-bit cache on the GPU, decode and chunked prefill, against the 64-bit oracle.

Tolerance of an output element o = sum_t p_t v_t (p the exact weights), from the kernels' roundings:
  * bf16 output: 2^-8 |o|;
  * each weight rounded to bf16 (and in the prefill kernel the weights' sum of the rounded ones): 2^-8 each, so
    2 * 2^-8 sum_t p_t |v_t|;
  * scores: sums of 128 products, taken as off by 2^-12 of the largest sum_d |q_d k_td| (the scaled matrix instruction
    drops terms 2^-13 below the largest of their eight, 7 x 2^-13 of it where all seven others are just below that, and
    adds the sixteen sums in fp32), so a weight is off by a factor within exp(+-2 e), e = 2^-12 max_t |scale| sum_d
    |q_d k_td|; the exponential's own error is far below;
  * fp32 sums: below all of these.
"""

import numpy as np
import pytest
import torch

from mini_infra_qwen3_amd import data_plane
from oracle import fp4_ref

pytestmark = pytest.mark.gpu

SCALE = 128 ** -0.5


def bound(out, weighed, size):
    e = 2.0 ** -12 * size[:, None]
    return 2.0 ** -8 * np.abs(out) + (2.0 ** -7 + np.expm1(2 * e)) * weighed + 1e-30


def tables_for(rng, counts, width=None):
    need = [-(-max(n, 0) // 16) for n in counts]
    num_blocks = 2 + sum(need)
    perm = rng.permutation(num_blocks - 1) + 1
    table = np.zeros((len(counts), width or max(max(need), 1)), dtype=np.int64)
    at = 0
    for i, n in enumerate(need):
        n = min(n, table.shape[1])
        table[i, :n] = perm[at:at + n]
        at += n
    return table, num_blocks


def decode_case(seed, contexts, heads, kv_heads, width=None, spread=(122, 130)):
    rng = np.random.default_rng(seed)
    table, num_blocks = tables_for(rng, contexts, width)
    kp, vp = (fp4_ref.random_pool(rng, num_blocks, kv_heads, *spread) for _ in range(2))
    q = torch.from_numpy(rng.standard_normal((len(contexts), heads, 128))).to(torch.bfloat16)
    return q, kp, vp, table


def check_decode(got, q, kp, vp, table, contexts, scale=SCALE):
    got = got.float().cpu().double().numpy().reshape(q.shape)
    keys, values = fp4_ref.load(kp, False), fp4_ref.load(vp, True)
    for b, n in enumerate(contexts):
        n = min(n, 16 * table.shape[1])
        if n <= 0:
            assert not got[b].any()
            continue
        ref, weighed, size = fp4_ref.attention(q[b].double().numpy(), fp4_ref.table_rows(keys, table[b], n),
                                               fp4_ref.table_rows(values, table[b], n), scale)
        assert (np.abs(got[b] - ref) <= bound(ref, weighed, size)).all(), (b, n, np.abs(got[b] - ref).max())


def run_decode(device, q, kp, vp, table, contexts, scale=SCALE, sub=1, **kw):
    return data_plane.paged_decode_attention_fp4(
        q.to(device), fp4_ref.to_torch(kp, sub).to(device), fp4_ref.to_torch(vp, sub).to(device),
        torch.from_numpy(table).to(device), torch.tensor(contexts).to(device), scale, **kw)


@pytest.mark.parametrize("heads,kv_heads", [(16, 8), (8, 8), (64, 8), (40, 8), (5, 1), (12, 4), (21, 3)])
def test_decode_heads(native_lib, device, heads, kv_heads):
    contexts = [1, 33, 0, 16, 300, 17]
    case = decode_case(heads, contexts, heads, kv_heads)
    check_decode(run_decode(device, *case, contexts), *case, contexts)


@pytest.mark.parametrize("contexts", [[1], [15, 16, 17], [31, 32, 33, -3], [127, 128, 129], [1023, 1024, 1025], [4099], [2, 9000, 0, 65]])
def test_decode_lengths(native_lib, device, contexts):
    case = decode_case(len(contexts) + contexts[0], contexts, 4, 2)
    check_decode(run_decode(device, *case, contexts), *case, contexts)


def test_decode_batch_of_many_lengths(native_lib, device):
    contexts = [int(x) for x in np.random.default_rng(7).integers(0, 700, 150)]
    case = decode_case(3, contexts, 4, 2)
    check_decode(run_decode(device, *case, contexts), *case, contexts)


@pytest.mark.parametrize("heads,kv_heads,batch,width", [
    (4, 2, 5, 60),       # whole sequences by 8 wavefronts (few pairs, short tables)
    (2, 2, 300, 100),    # whole by 4 (many pairs)
    (16, 8, 3, 900),     # parts
    (4, 2, 50, 1300),    # streams
    (64, 8, 40, 400),    # streams, 8 heads a group
    (5, 1, 130, 1000),
    (9, 3, 60, 700)])
def test_decode_forms(native_lib, device, heads, kv_heads, batch, width):
    """Tables wider than any context, so that each way of cutting the work sees short, empty and odd sequences."""
    rng = np.random.default_rng(batch)
    contexts = [int(x) for x in rng.integers(0, 330, batch)]
    contexts[0], contexts[-1], contexts[batch // 2] = 1, 0, 16 * min(width, 70)
    case = decode_case(batch, contexts, heads, kv_heads, width=width)
    check_decode(run_decode(device, *case, contexts), *case, contexts)
    if batch > 2:  # all but one empty; all empty
        few = [0] * batch
        check_decode(run_decode(device, *case, few), *case, few)
        few[batch // 2] = contexts[batch // 2]
        check_decode(run_decode(device, *case, few), *case, few)


def test_decode_long_ranges(native_lib, device):
    """Enough blocks for every range of the stream form to hold more than 64; against the values read back, in fp64."""
    contexts = [90000, 5, 70001, 0, 120000, 33333, 100000, 16]
    kv_heads, heads = 8, 16
    gen = torch.Generator(device=device).manual_seed(5)
    need = [-(-n // 16) for n in contexts]
    num_blocks = 1 + sum(need)
    kp, vp = (torch.randint(0, 256, data_plane.fp4_pool_shape(num_blocks, 16, kv_heads), generator=gen, device=device,
                            dtype=torch.uint8) for _ in range(2))
    for p in (kp, vp):
        p[..., 1024:] = p[..., 1024:] % 8 + 122
    perm = torch.randperm(num_blocks - 1, generator=gen, device=device) + 1
    table = torch.zeros(len(contexts), max(need), dtype=torch.long, device=device)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = perm[at:at + n]
        at += n
    q = torch.randn(len(contexts), heads, 128, generator=gen, device=device).to(torch.bfloat16)
    got = data_plane.paged_decode_attention_fp4(q, kp, vp, table, torch.tensor(contexts, device=device), SCALE)
    got = got.double().view(len(contexts), heads, 128)
    for b, n in enumerate(contexts):
        if n == 0:
            assert not got[b].any()
            continue
        k, v = (torch.empty(1, 16 * need[b], kv_heads, 128, dtype=torch.bfloat16, device=device) for _ in range(2))
        data_plane.gather_blocks_fp4([kp], [vp], table[b:b + 1, :need[b]], [k], [v])
        for h in range(heads):
            kh, vh, qh = k[0, :n, h // 2].double(), v[0, :n, h // 2].double(), q[b, h].double()
            p = torch.softmax(SCALE * (kh * qh).sum(1), 0)
            ref, weighed = (p[:, None] * vh).sum(0), (p[:, None] * vh.abs()).sum(0)
            size = SCALE * (kh * qh).abs().sum(1).max()
            e = torch.expm1(2.0 ** -11 * size)
            assert ((got[b, h] - ref).abs() <= 2.0 ** -8 * ref.abs() + (2.0 ** -7 + e) * weighed).all(), (b, h)


def test_decode_context_beyond_its_table(native_lib, device):
    contexts = [500, 49]
    case = decode_case(4, contexts, 4, 2, width=3)
    check_decode(run_decode(device, *case, contexts), *case, contexts)


@pytest.mark.parametrize("scale", [-0.11, 0.0, 1.7])
def test_decode_scales(native_lib, device, scale):
    contexts = [40, 1100]
    case = decode_case(5, contexts, 4, 2, spread=(120, 126))
    check_decode(run_decode(device, *case, contexts, scale), *case, contexts, scale)


def test_decode_larger_blocks(native_lib, device):
    contexts = [70, 0, 161]
    rng = np.random.default_rng(6)
    blocks = np.array([[3, 1, 0, 0], [0, 0, 0, 0], [2, 5, 4, 6]])  # of 48 tokens
    kp, vp = (fp4_ref.random_pool(rng, 7 * 3, 2) for _ in range(2))
    q = torch.from_numpy(rng.standard_normal((3, 4, 128))).to(torch.bfloat16)
    table = (blocks[:, :, None] * 3 + np.arange(3)).reshape(3, -1)
    check_decode(run_decode(device, q, kp, vp, blocks, contexts, sub=3), q, kp, vp, table, contexts)


@pytest.mark.parametrize("width", [None, 900, 4000])  # whole sequences, parts, streams
def test_decode_hidden_tokens_never_count(native_lib, device, width):
    """NaN scales after each context, in the null block and in unused blocks change no bit."""
    contexts = [1, 47, 0, 1030, 128]
    q, kp, vp, table = decode_case(8, contexts, 16, 8, width=width)
    clean = run_decode(device, q, kp, vp, table, contexts)
    for pool, value in ((kp, False), (vp, True)):
        used = np.zeros((pool.shape[0], 16), dtype=bool)
        for b, n in enumerate(contexts):
            for t in range(n):
                used[table[b, t // 16], t % 16] = True
        for block, token in zip(*np.where(~used)):
            for g in range(4):
                pool[block, :, fp4_ref.scale_at(value, token, g)] = 255
    dirty = run_decode(device, q, kp, vp, table, contexts)
    assert torch.equal(clean.view(torch.int16), dirty.view(torch.int16))


@pytest.mark.parametrize("width", [None, 21000])  # parts, streams
def test_decode_visible_nan_reaches_its_output_alone(native_lib, device, width):
    contexts = [40, 41, 1500]
    q, kp, vp, table = decode_case(9, contexts, 4, 2, width=width)
    kp[table[0, 1], 0, fp4_ref.scale_at(False, 3, 2)] = 255  # sequence 0, KV head 0: every dim
    vp[table[2, 70], 1, fp4_ref.scale_at(True, 5, 1)] = 255  # sequence 2, KV head 1: dims 32 .. 63
    out = run_decode(device, q, kp, vp, table, contexts).view(3, 4, 128).isnan().cpu()
    expect = torch.zeros(3, 4, 128, dtype=torch.bool)
    expect[0, :2] = True
    expect[2, 2:, 32:64] = True
    assert torch.equal(out, expect)


def test_decode_query_extremes(native_lib, device):
    """Queries whose elements span many binades, zero queries, an infinity (a NaN row, as inf - inf in the softmax)."""
    contexts = [50, 50, 50]
    q, kp, vp, table = decode_case(10, contexts, 4, 2, spread=(121, 125))
    q[0] = q[0] * torch.exp2(torch.arange(128) % 40 - 38.0)
    q[1, 1] = 0
    got = run_decode(device, q, kp, vp, table, contexts)
    check_decode(got, q, kp, vp, table, contexts)
    q[2, 3, 5] = float("inf")
    dirty = run_decode(device, q, kp, vp, table, contexts).view(3, 4, 128)
    assert dirty[2, 3].isnan().all() and torch.equal(dirty[2, :3], got.view(3, 4, 128)[2, :3])


def test_decode_strides_out_and_workspace(native_lib, device):
    """A query view of a projection, strided tables and contexts, a strided out, a workspace kept by the caller."""
    contexts = [2000, 3, 1029]
    q, kp, vp, table = decode_case(11, contexts, 16, 8)
    plain = run_decode(device, q, kp, vp, table, contexts)
    wide_q = torch.randn(3, 40, 128).to(torch.bfloat16).to(device)
    wide_q[:, 8:24] = q.to(device)
    packed = torch.zeros(3, table.shape[1] + 5, dtype=torch.long, device=device)
    packed[:, 3], packed[:, 4:-1] = torch.tensor(contexts), torch.from_numpy(table)
    need = data_plane.paged_decode_fp4_workspace_bytes(3, table.shape[1], 16, 8)
    assert need > 0
    workspace = torch.full((need + 100,), 255, dtype=torch.uint8, device=device)
    buffer = torch.full((4, 16 * 128 + 64), 3.0, dtype=torch.bfloat16, device=device)
    kp_t, vp_t = fp4_ref.to_torch(kp).to(device), fp4_ref.to_torch(vp).to(device)
    for _ in range(2):
        out = data_plane.paged_decode_attention_fp4(wide_q[:, 8:24], kp_t, vp_t, packed[:, 4:-1], packed[:, 3], SCALE,
                                                    out=buffer[:3, :2048], workspace=workspace)
        assert torch.equal(out, plain) and out.data_ptr() == buffer.data_ptr()
    assert (buffer[3] == 3.0).all() and (buffer[:, 2048:] == 3.0).all()
    assert (workspace[need:] == 255).all()


def test_decode_out_of_range_ids_read_the_null_block(native_lib, device):
    contexts = [60]
    q, kp, vp, table = decode_case(12, contexts, 4, 2)
    table[0, 1], table[0, 2] = -7, 1 << 40
    check_decode(run_decode(device, q, kp, vp, table, contexts), q, kp, vp, table, contexts)


def test_decode_graph_replays(native_lib, device):
    """Captured once, replayed with other contents, eager calls between the replays."""
    contexts = [700, 0, 1300, 20]
    q, kp, vp, table = decode_case(13, contexts, 16, 8)
    kp_t, vp_t, bt = fp4_ref.to_torch(kp).to(device), fp4_ref.to_torch(vp).to(device), torch.from_numpy(table).to(device)
    q_t, ctx = q.to(device), torch.tensor(contexts).to(device)
    call = lambda: data_plane.paged_decode_attention_fp4(q_t, kp_t, vp_t, bt, ctx, SCALE)  # noqa: E731
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for step in range(4):
        q_t.copy_(torch.randn(q.shape).to(torch.bfloat16))
        ctx.copy_(torch.tensor([700 - step, step, 1300 - 300 * step, 20]))
        eager = call().clone()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, eager)


# ------------------------------------------------------------------------------ chunked prefill
def prefill_case(seed, starts, lens, width, heads, kv_heads, spread=(122, 130)):
    rng = np.random.default_rng(seed)
    table, num_blocks = tables_for(rng, starts)
    kp, vp = (fp4_ref.random_pool(rng, num_blocks, kv_heads, *spread) for _ in range(2))
    gen = torch.Generator().manual_seed(seed)
    q, k, v = (torch.randn(len(starts), width, h, 128, generator=gen).to(torch.bfloat16) for h in (heads, kv_heads, kv_heads))
    return q, k, v, kp, vp, table


def run_prefill(device, case, starts, lens, scale=SCALE, sub=1, **kw):
    q, k, v, kp, vp, table = case
    seen = [t.to(device).transpose(1, 2) for t in (q, k, v)]
    return data_plane.chunked_prefill_attention_fp4(
        *seen, fp4_ref.to_torch(kp, sub).to(device), fp4_ref.to_torch(vp, sub).to(device), torch.from_numpy(table).to(device),
        torch.tensor(starts).to(device), torch.tensor(lens).to(device), scale, **kw)


def check_prefill(got, case, starts, lens, scale=SCALE, queries=None):
    q, k, v, kp, vp, table = case
    width, heads = q.shape[1:3]
    got = got.float().cpu().double().numpy().reshape(q.shape)
    keys, values = fp4_ref.load(kp, False), fp4_ref.load(vp, True)
    for b, (past, n) in enumerate(zip(starts, lens)):
        past, n = max(min(past, 16 * table.shape[1]), 0), max(min(n, width), 0)
        first = width - n
        assert not got[b, :first].any()
        hist = [fp4_ref.table_rows(x, table[b], past) for x in (keys, values)]
        k_all = np.concatenate((hist[0], k[b, first:].double().numpy()))
        v_all = np.concatenate((hist[1], v[b, first:].double().numpy()))
        for i in range(first, width) if queries is None else [i for i in queries if i >= first]:
            seen = past + i - first + 1
            ref, weighed, size = fp4_ref.attention(q[b, i].double().numpy(), k_all[:seen], v_all[:seen], scale)
            assert (np.abs(got[b, i] - ref) <= bound(ref, weighed, size)).all(), (b, i, np.abs(got[b, i] - ref).max())


@pytest.mark.parametrize("heads,kv_heads", [(16, 8), (8, 8), (40, 8), (5, 1), (12, 4), (18, 2)])
def test_prefill_heads(native_lib, device, heads, kv_heads):
    starts, lens = [50, 0, 7], [9, 20, 20]
    case = prefill_case(heads, starts, lens, 20, heads, kv_heads)
    check_prefill(run_prefill(device, case, starts, lens), case, starts, lens)


@pytest.mark.parametrize("starts,lens,width", [
    ([0], [1], 1), ([1], [1], 1), ([0, 0], [0, 3], 3), ([64, 63, 65], [16, 17, 15], 17), ([15, 16, 17], [33, 32, 31], 33),
    ([500], [64], 64), ([127, 129], [65, 1], 65), ([0, 0], [129, 128], 129), ([1000, 3], [40, 0], 70)])
def test_prefill_lengths(native_lib, device, starts, lens, width):
    case = prefill_case(width + starts[0], starts, lens, width, 4, 2)
    check_prefill(run_prefill(device, case, starts, lens), case, starts, lens)


@pytest.mark.parametrize("rows,width,past,heads,kv_heads", [
    (2, 330, 200, 4, 2),      # few workgroups: narrow tiles, the keys in two halves
    (3, 450, 70, 16, 8),
    (8, 700, 90, 16, 8),
    (20, 130, 0, 16, 8),
    (20, 130, 60, 16, 8),
    (6, 1500, 33, 16, 8)])    # many: wide tiles
def test_prefill_workgroup_shapes(native_lib, device, rows, width, past, heads, kv_heads):
    starts = [max(past - 5 * b, 0) for b in range(rows)]
    lens = [width - 7 * b for b in range(rows)]
    case = prefill_case(rows, starts, lens, width, heads, kv_heads)
    queries = sorted({0, 31, 32, 63, 64, 127, 128, width // 2, width - 65, width - 64, width - 2, width - 1})
    check_prefill(run_prefill(device, case, starts, lens), case, starts, lens, queries=queries)


@pytest.mark.parametrize("starts,lens,width,table,heads,kv_heads", [
    ([0], [1], 1, 300, 4, 2),                      # many parts, next to nothing in them
    ([4700], [1], 1, 300, 4, 2),
    ([3000, 0, 17, 2999], [40, 33, 0, 1], 40, 200, 16, 8),
    ([1100, 1023], [70, 12], 70, 80, 5, 1),
    ([64 * 18], [64], 64, 72, 4, 4),               # parts that end on the chunk's first tile
    ([900], [200], 200, 60, 2, 1)])
def test_prefill_parts(native_lib, device, starts, lens, width, table, heads, kv_heads):
    """Short chunks with wide history tables: the keys of a row cut over workgroups."""
    assert data_plane.chunked_prefill_fp4_workspace_bytes(len(starts), width, heads, kv_heads, table) > 0
    case = prefill_case(width + table, starts, lens, width, heads, kv_heads)
    wide = np.zeros((len(starts), table), dtype=np.int64)
    wide[:, :case[5].shape[1]] = case[5]
    case = (*case[:5], wide)
    out = run_prefill(device, case, starts, lens)
    check_prefill(out, case, starts, lens)
    need = data_plane.chunked_prefill_fp4_workspace_bytes(len(starts), width, heads, kv_heads, table)
    workspace = torch.full((need + 64,), 255, dtype=torch.uint8, device=device)  # NaN: what is read was written
    again = run_prefill(device, case, starts, lens, workspace=workspace)
    assert torch.equal(out, again) and (workspace[need:] == 255).all()


@pytest.mark.parametrize("scale", [-0.11, 0.0, 1.3])
def test_prefill_scales(native_lib, device, scale):
    starts, lens = [90], [37]
    case = prefill_case(21, starts, lens, 40, 4, 2, spread=(120, 126))
    check_prefill(run_prefill(device, case, starts, lens, scale), case, starts, lens, scale)


def test_prefill_without_history_or_with_a_short_table(native_lib, device):
    starts, lens = [0, 0], [12, 5]
    case = prefill_case(22, starts, lens, 12, 4, 2)
    case = (*case[:5], case[5][:, :0])
    check_prefill(run_prefill(device, case, starts, lens), case, starts, lens)
    starts = [200, 40]
    case = prefill_case(23, [48, 40], lens, 12, 4, 2)  # tables of 3 blocks
    check_prefill(run_prefill(device, case, starts, lens), case, starts, lens)


def test_prefill_larger_blocks(native_lib, device):
    rng = np.random.default_rng(24)
    starts, lens = [70, 40], [20, 9]
    blocks = np.array([[3, 1, 0], [2, 4, 0]])  # of 32 tokens
    q, k, v, _, _, _ = prefill_case(24, [0, 0], lens, 20, 4, 2)
    kp, vp = (fp4_ref.random_pool(rng, 5 * 2, 2) for _ in range(2))
    blocks[0, 2] = 0
    table = (blocks[:, :, None] * 2 + np.arange(2)).reshape(2, -1)
    got = run_prefill(device, (q, k, v, kp, vp, blocks), starts, lens, sub=2)
    check_prefill(got, (q, k, v, kp, vp, table), starts, lens)


@pytest.mark.parametrize("rows,width,wide", [(2, 100, 0), (16, 300, 0), (2, 100, 200)])  # the last in parts
def test_prefill_hidden_tokens_never_count(native_lib, device, rows, width, wide):
    """NaN in history slots past start_lens, unused blocks and the chunk's padding rows changes no bit."""
    starts = [70 - 3 * b for b in range(rows)]
    lens = [width - 11 * b for b in range(rows)]
    q, k, v, kp, vp, table = prefill_case(25, starts, lens, width, 4, 2)
    table = np.pad(table, ((0, 0), (0, wide)))
    clean = run_prefill(device, (q, k, v, kp, vp, table), starts, lens)
    for pool, value in ((kp, False), (vp, True)):
        used = np.zeros((pool.shape[0], 16), dtype=bool)
        for b, n in enumerate(starts):
            for t in range(n):
                used[table[b, t // 16], t % 16] = True
        for block, token in zip(*np.where(~used)):
            for g in range(4):
                pool[block, :, fp4_ref.scale_at(value, token, g)] = 255
    for b, n in enumerate(lens):
        q[b, :width - n], k[b, :width - n], v[b, :width - n] = float("nan"), float("inf"), float("nan")
    dirty = run_prefill(device, (q, k, v, kp, vp, table), starts, lens)
    assert torch.equal(clean.view(torch.int16), dirty.view(torch.int16))


def test_prefill_visible_nan_reaches_its_rows_alone(native_lib, device):
    starts, lens = [80, 80], [10, 30]
    q, k, v, kp, vp, table = prefill_case(26, starts, lens, 30, 4, 2)
    kp[table[0, 4], 0, fp4_ref.scale_at(False, 15, 0)] = 255
    vp[table[1, 0], 1, fp4_ref.scale_at(True, 5, 3)] = 255
    out = run_prefill(device, (q, k, v, kp, vp, table), starts, lens).view(2, 30, 4, 128).isnan().cpu()
    expect = torch.zeros(2, 30, 4, 128, dtype=torch.bool)
    expect[0, 20:, :2] = True
    expect[1, :, 2:, 96:] = True
    assert torch.equal(out, expect)


def test_prefill_strided_out_and_lens(native_lib, device):
    starts, lens = [33, 5], [7, 18]
    case = prefill_case(27, starts, lens, 18, 4, 2)
    plain = run_prefill(device, case, starts, lens)
    buffer = torch.full((3, 20, 600), 2.0, dtype=torch.bfloat16, device=device)
    q, k, v, kp, vp, table = case
    packed = torch.zeros(2, 2 + table.shape[1] + 3, dtype=torch.long, device=device)
    packed[:, 0], packed[:, 1], packed[:, 2:-3] = torch.tensor(starts), torch.tensor(lens), torch.from_numpy(table)
    out = data_plane.chunked_prefill_attention_fp4(
        *[t.to(device).transpose(1, 2).contiguous() for t in (q, k, v)], fp4_ref.to_torch(kp).to(device),
        fp4_ref.to_torch(vp).to(device), packed[:, 2:-3], packed[:, 0], packed[:, 1], SCALE, out=buffer[:2, :18, 8:520])
    assert torch.equal(out, plain)
    assert (buffer[2] == 2.0).all() and (buffer[:, 18:] == 2.0).all() and (buffer[..., :8] == 2.0).all()


def test_prefill_graph_replays(native_lib, device):
    starts, lens = [200, 64], [40, 33]
    q, k, v, kp, vp, table = prefill_case(28, starts, lens, 40, 16, 8)
    seen = [t.to(device).transpose(1, 2) for t in (q, k, v)]
    rest = (fp4_ref.to_torch(kp).to(device), fp4_ref.to_torch(vp).to(device), torch.from_numpy(table).to(device))
    st, ln = torch.tensor(starts).to(device), torch.tensor(lens).to(device)
    call = lambda: data_plane.chunked_prefill_attention_fp4(*seen, *rest, st, ln, SCALE)  # noqa: E731
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for step in range(4):
        seen[0].copy_(torch.randn(seen[0].shape).to(torch.bfloat16))
        st.copy_(torch.tensor([200 - 50 * step, 64 + step]))
        ln.copy_(torch.tensor([40 - step, 5 * step]))
        eager = call().clone()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, eager)


def test_prefill_then_decode_of_stored_tokens(native_lib, device):
    """The pieces as a server uses them: chunk by chunk prefill with stores between, then decode with appends; each
    step against the oracle on what the cache then holds."""
    gen = torch.Generator().manual_seed(31)
    heads, kv_heads, blocks = 4, 2, 12
    shape = data_plane.fp4_pool_shape(blocks, 16, kv_heads)
    kp, vp = (torch.zeros(shape, dtype=torch.uint8, device=device) for _ in range(2))
    tables = torch.tensor([[3, 7, 1, 9, 2], [8, 4, 10, 5, 6]])
    past = [0, 0]
    rand = lambda *s: torch.randn(*s, generator=gen).to(torch.bfloat16)  # noqa: E731
    pools = lambda: [p.cpu().numpy().reshape(blocks, kv_heads, 1088) for p in (kp, vp)]  # noqa: E731
    for lens in ([20, 33], [17, 1]):
        width = max(lens)
        q, k, v = rand(2, width, heads, 128), rand(2, width, kv_heads, 128), rand(2, width, kv_heads, 128)
        seen = [t.to(device).transpose(1, 2) for t in (q, k, v)]
        out = data_plane.chunked_prefill_attention_fp4(*seen, kp, vp, tables.to(device), torch.tensor(past).to(device),
                                                       torch.tensor(lens).to(device), SCALE)
        check_prefill(out, (q, k, v, *pools(), tables.numpy()), past, lens)
        index = torch.tensor([(b, width - n + t, int(tables[b, (past[b] + t) // 16]) * 16 + (past[b] + t) % 16)
                              for b, n in enumerate(lens) for t in range(n)]).t().contiguous().to(device)
        data_plane.reshape_and_cache_fp4([seen[1]], [seen[2]], index[2], [kp], [vp], token_rows=index[0], token_positions=index[1])
        past = [p + n for p, n in zip(past, lens)]
    for _ in range(12):
        q, k, v = rand(2, heads, 128), rand(2, kv_heads, 1, 128).to(device), rand(2, kv_heads, 1, 128).to(device)
        slots = torch.tensor([int(tables[b, p // 16]) * 16 + p % 16 for b, p in enumerate(past)]).to(device)
        data_plane.reshape_and_cache_fp4([k], [v], slots, [kp], [vp])
        past = [p + 1 for p in past]
        out = data_plane.paged_decode_attention_fp4(q.to(device), kp, vp, tables.to(device), torch.tensor(past).to(device), SCALE)
        check_decode(out, q, *pools(), tables.numpy(), past)
