"""The 4-bit operators and block copies where a caller may take them: pools past 4 GiB, streams of their own side by side,
captured stores, gathers and copies, subnormal rows.

Each is compared bit for bit with the same call in plain circumstances, or with the oracle."""

import numpy as np
import pytest
import torch

from mini_infra_qwen3_amd import data_plane
from oracle import fp4_ref

pytestmark = pytest.mark.gpu

SCALE = 128 ** -0.5


def test_pools_past_4_gib(native_lib, device):
    """500,000 blocks of 8704 bytes: the same contents at the pool's far end and in a small pool."""
    far, n = 500_000, 12
    small = [torch.zeros(n + 1, 1, 8, 1088, dtype=torch.uint8, device=device) for _ in range(2)]
    large = [torch.zeros(far, 1, 8, 1088, dtype=torch.uint8, device=device) for _ in range(2)]
    gen = torch.Generator().manual_seed(0)
    rows = [torch.randn(1, 8, n * 16, 128, generator=gen).to(torch.bfloat16).to(device) for _ in range(2)]
    positions = torch.arange(n * 16, device=device)
    zero = torch.zeros_like(positions)
    near_ids, far_ids = torch.arange(1, n + 1, device=device), far - 1 - torch.arange(n, device=device)
    for pools, ids in ((small, near_ids), (large, far_ids)):
        slots = (ids[:, None] * 16 + torch.arange(16, device=device)).reshape(-1)
        data_plane.reshape_and_cache_fp4([rows[0]], [rows[1]], slots, [pools[0]], [pools[1]], token_rows=zero, token_positions=positions)
    assert torch.equal(large[0][far_ids], small[0][1:]) and torch.equal(large[1][far_ids], small[1][1:])
    q = torch.randn(1, 16, 128, generator=gen).to(torch.bfloat16).to(device)
    chunk = [torch.randn(1, h, 40, 128, generator=gen).to(torch.bfloat16).to(device) for h in (16, 8, 8)]
    outs = []
    for pools, ids in ((small, near_ids), (large, far_ids)):
        gathered = [torch.empty(1, n * 16, 8, 128, dtype=torch.bfloat16, device=device) for _ in range(2)]
        data_plane.gather_blocks_fp4([pools[0]], [pools[1]], ids[None], [gathered[0]], [gathered[1]])
        wide = torch.zeros(1, 3000, dtype=torch.long, device=device)  # enough blocks for parts
        wide[0, :n] = ids
        tensors = [*gathered]
        for table in (ids[None], wide):
            tensors.append(data_plane.paged_decode_attention_fp4(q, *pools, table, torch.tensor([n * 16 - 3], device=device), SCALE))
            tensors.append(data_plane.chunked_prefill_attention_fp4(
                *chunk, *pools, table, torch.tensor([n * 16 - 5], device=device), torch.tensor([37], device=device), SCALE))
        outs.append(tensors)
    for a, b in zip(*outs):
        assert torch.equal(a, b) and bool(a.any())
    many = torch.zeros(256, 600, dtype=torch.long, device=device)  # streams
    many[:, :n] = far_ids
    contexts = torch.arange(256, device=device) % (n * 16 + 1)
    at_far = data_plane.paged_decode_attention_fp4(q.expand(256, -1, -1), *large, many, contexts, SCALE)
    many[:, :n] = near_ids
    assert torch.equal(at_far, data_plane.paged_decode_attention_fp4(q.expand(256, -1, -1), *small, many, contexts, SCALE))
    data_plane.copy_blocks([large[0]], [large[1]], far_ids[:3], torch.tensor([5, far - 100, 7], device=device))
    for at, source in ((5, 0), (far - 100, 1), (7, 2)):
        assert torch.equal(large[0][at], small[0][1 + source]) and torch.equal(large[1][at], small[1][1 + source])


def attention_calls(device, seed):
    """A decode of streams, one of parts, and a prefill of parts, with their own tensors."""
    rng = np.random.default_rng(seed)
    kp, vp = (fp4_ref.to_torch(fp4_ref.random_pool(rng, 200, 8)).to(device) for _ in range(2))
    gen = torch.Generator().manual_seed(seed)
    randn = lambda *s: torch.randn(*s, generator=gen).to(torch.bfloat16).to(device)  # noqa: E731
    table = lambda b, n: torch.from_numpy(rng.integers(1, 200, (b, n))).to(device)  # noqa: E731
    lens = lambda b, top: torch.from_numpy(rng.integers(0, top, b)).to(device)  # noqa: E731
    q1, t1, l1 = randn(200, 16, 128), table(200, 300), lens(200, 2000)
    q2, t2, l2 = randn(3, 16, 128), table(3, 300), lens(3, 4800)
    q3, k3, v3, t3 = randn(1, 16, 60, 128), randn(1, 8, 60, 128), randn(1, 8, 60, 128), table(1, 250)
    starts, chunk = torch.tensor([3901], device=device), torch.tensor([53], device=device)
    return [lambda **kw: data_plane.paged_decode_attention_fp4(q1, kp, vp, t1, l1, SCALE, **kw),
            lambda **kw: data_plane.paged_decode_attention_fp4(q2, kp, vp, t2, l2, SCALE, **kw),
            lambda **kw: data_plane.chunked_prefill_attention_fp4(q3, k3, v3, kp, vp, t3, starts, chunk, SCALE, **kw)]


@pytest.mark.parametrize("given", [False, True])
def test_calls_on_two_streams_at_once(native_lib, device, given):
    """Overlapping calls, each with a workspace of its own (allocated by the call, or given and reused within its stream)."""
    calls = [attention_calls(device, seed) for seed in (1, 2)]
    want = [[call() for call in side] for side in calls]
    streams = [torch.cuda.Stream() for _ in calls]
    space = [torch.empty(64 << 20, dtype=torch.uint8, device=device) if given else None for _ in calls]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(6):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                got[i].append([call(workspace=space[i]) for call in calls[i]])
    torch.cuda.synchronize()
    for i in range(2):
        for outs in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(outs, want[i]))


def test_captured_store_gather_and_copy(native_lib, device):
    """One graph of the three, replayed on new rows and other slots and blocks, with eager calls in between."""
    layers, blocks = 3, 20
    pools = torch.zeros(2, layers, blocks, 1, 4, 1088, dtype=torch.uint8, device=device)
    again = torch.zeros_like(pools)
    src = torch.zeros(2, layers, 5, 4, 7, 128, dtype=torch.bfloat16, device=device)
    slots, src_ids, dst_ids = (torch.zeros(n, dtype=torch.long, device=device) for n in (5, 3, 3))
    table = torch.zeros(2, 4, dtype=torch.long, device=device)
    out = torch.empty(2, layers, 2, 64, 4, 128, dtype=torch.bfloat16, device=device)
    position = torch.zeros(5, dtype=torch.long, device=device)

    def run(to, gathered):
        data_plane.reshape_and_cache_fp4(list(src[0]), list(src[1]), slots, list(to[0]), list(to[1]), token_positions=position)
        data_plane.copy_blocks(list(to[0]), list(to[1]), src_ids, dst_ids)
        data_plane.gather_blocks_fp4(list(to[0]), list(to[1]), table, list(gathered[0]), list(gathered[1]))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    slots.copy_(torch.arange(16, 21))
    dst_ids.copy_(torch.tensor([7, 8, 9]))
    with torch.cuda.stream(side):
        run(again, torch.empty_like(out))
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run(pools, out)
    pools.zero_(), again.zero_()
    gen = torch.Generator().manual_seed(4)
    for step in range(5):
        src.copy_(torch.randn(src.shape, generator=gen))
        position.copy_(torch.randint(0, 7, (5,), generator=gen))
        slots.copy_(torch.randperm(blocks * 16, generator=gen)[:5])
        ids = torch.randperm(blocks, generator=gen)
        src_ids.copy_(ids[:3]), dst_ids.copy_(ids[3:6])
        table.copy_(torch.randint(0, blocks, (2, 4), generator=gen))
        eager = torch.empty_like(out)
        run(again, eager)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(pools, again) and torch.equal(out, eager)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_subnormal_rows(native_lib, device, dtype):
    """Multiples of 2^-129 up to 2^-123, around the smallest scale (2^-126): codes are rounded like any other, and read back."""
    row = (torch.arange(-64, 64).view(1, 1, 1, 128).double() * 2.0 ** -129).to(dtype)
    pools = [torch.zeros(2, 1, 1, 1088, dtype=torch.uint8, device=device) for _ in range(2)]
    data_plane.reshape_and_cache_fp4([row.to(device)], [row.to(device)], torch.tensor([16 + 5], device=device), [pools[0]], [pools[1]])
    want = [np.zeros((2, 1, 1088), dtype=np.uint8) for _ in range(2)]
    for value in (False, True):
        fp4_ref.store(want[value], 16 + 5, row[0, :, 0].double().numpy(), value)
        assert np.array_equal(pools[value].cpu().numpy().reshape(2, 1, 1088), want[value])
    out = [torch.empty(1, 16, 1, 128, dtype=torch.bfloat16, device=device) for _ in range(2)]
    data_plane.gather_blocks_fp4([pools[0]], [pools[1]], torch.tensor([[1]], device=device), [out[0]], [out[1]])
    read = fp4_ref.values_of(*fp4_ref.quantize_row(row[0, 0, 0].double().numpy()))
    assert np.abs(read).max() >= 2.0 ** -125
    for o in out:
        assert np.array_equal(o[0, 5, 0].cpu().view(torch.int16).numpy(),
                              torch.from_numpy(read).to(torch.bfloat16).view(torch.int16).numpy())


def test_calls_run_with_their_tensors_device_current(monkeypatch):
    """Workspace sizes and launches of tensors on another device than the current one (forced from the host)."""
    seen = []

    class Entry:
        @staticmethod
        def mi_probe(*args):
            seen.append((torch.cuda.current_device(), args))
            return 7

    monkeypatch.setattr(data_plane._native, "load", lambda: Entry)
    assert data_plane._on_device(torch.device("cuda", 0), "mi_probe", 1, 2) == 7
    entered = []
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: 1)

    class Guard:
        def __init__(self, device):
            entered.append(device)

        def __enter__(self):
            entered.append("in")

        def __exit__(self, *exc):
            entered.append("out")

    monkeypatch.setattr(torch.cuda, "device", Guard)
    assert data_plane._on_device(torch.device("cuda", 0), "mi_probe", 3) == 7
    assert entered == [torch.device("cuda", 0), "in", "out"] and len(seen) == 2
