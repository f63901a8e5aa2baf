"""The 4-bit cache on the GPU: quantising store, dequantising gather and block copies, against the 64-bit oracle.

Codes, scales and read-back values are exact (scaling by powers of two and one rounding to nearest even),
so everything here is compared bit for bit.
"""

import numpy as np
import pytest
import torch

from mini_infra_qwen3_amd import data_plane
from oracle import fp4_ref

pytestmark = pytest.mark.gpu


def sources(gen, dtype, layers, rows, heads, width):
    """Token-major buffers seen as [rows, heads, width, 128] per layer; values over many binades, ties among them."""
    x = torch.randn(layers, rows, width, heads, 128, generator=gen)
    x = x * torch.exp2(torch.randint(-12, 9, x.shape[:-1] + (4,), generator=gen).float()).repeat_interleave(32, -1)
    ties = torch.randint(-32, 33, x.shape, generator=gen).float() * 0.25
    x = torch.where(torch.rand(x.shape, generator=gen) < 0.3, ties, x).to(dtype)
    return [t.transpose(1, 2) for t in x]


def check_store(device, dtype=torch.bfloat16, layers=1, rows=2, heads=2, width=21, sub=1, tokens=None, views=lambda t: t,
                edit=None):
    gen = torch.Generator().manual_seed(rows * 100 + heads * 10 + width + sub)
    keys, values = sources(gen, dtype, layers, rows, heads, width), sources(gen, dtype, layers, rows, heads, width)
    if edit:
        edit(keys, values)
    num_blocks = 4 + rows * (-(-width // (16 * sub)))
    n = rows * width if tokens is None else tokens
    slots = torch.randperm(num_blocks * 16 * sub, generator=gen)[:n]
    flat = torch.randperm(rows * width, generator=gen)[:n]
    token_rows, positions = flat // width, flat % width
    rng = np.random.default_rng(0)
    before = [fp4_ref.random_pool(rng, num_blocks * sub, heads) for _ in range(2 * layers)]
    pools = [fp4_ref.to_torch(p, sub).to(device) for p in before]
    index = torch.stack((slots, token_rows, positions), 1).to(device)  # columns: a common stride of 3
    data_plane.reshape_and_cache_fp4([views(k.to(device)) for k in keys], [views(v.to(device)) for v in values], index[:, 0],
                                     pools[:layers], pools[layers:], token_rows=index[:, 1], token_positions=index[:, 2])
    for i, pool in enumerate(pools):
        expect, src = before[i].copy(), (keys + values)[i].double().numpy()
        for s, r, p in zip(slots.tolist(), token_rows.tolist(), positions.tolist()):
            fp4_ref.store(expect, s, src[r, :, p], i >= layers)
        assert np.array_equal(pool.cpu().numpy().reshape(expect.shape), expect)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("rows,heads,width", [(1, 1, 1), (2, 8, 17), (3, 5, 33)])
def test_store_is_exact(native_lib, device, dtype, rows, heads, width):
    check_store(device, dtype, rows=rows, heads=heads, width=width)


def test_store_of_many_layers_and_large_blocks(native_lib, device):
    check_store(device, layers=35, rows=1, heads=1, width=3)  # more layers than a launch takes
    check_store(device, sub=3, rows=2, heads=2, width=50)     # blocks of 48 tokens


def test_store_takes_unaligned_rows(native_lib, device):
    def odd(t):
        buf = torch.empty(t.numel() + 1, dtype=t.dtype, device=t.device)
        out = buf[1:].view(t.transpose(1, 2).shape).transpose(1, 2)
        out.copy_(t)
        return out

    for dtype in (torch.bfloat16, torch.float32):
        check_store(device, dtype, views=odd)


def test_store_of_non_finite_and_extreme_rows(native_lib, device):
    def edit(keys, values):
        keys[0][0, 0, 0, 40] = float("inf")
        keys[0][0, 1, 1, 7] = float("nan")
        keys[0][1, 0, 2] = 0.0
        keys[0][1, 0, 3] = -0.0
        keys[0][1, 0, 4] = 3.3e38
        keys[0][1, 0, 5] = 2.0 ** -126
        values[0][1, 1, 6, ::2] = float("-inf")
        values[0][1, 1, 7] = 1e-39
        values[0][1, 1, 8, 5] = -3.38e38

    check_store(device, edit=edit)


def test_store_skips_what_is_out_of_range(native_lib, device):
    rng = np.random.default_rng(1)
    before = fp4_ref.random_pool(rng, 4, 2)
    kp, vp = fp4_ref.to_torch(before).to(device), fp4_ref.to_torch(before).to(device)
    src = torch.randn(3, 2, 5, 128).to(torch.bfloat16).to(device)
    slots = torch.tensor([-1, 64, 1 << 40, 5, 6, 7, 8], device=device)
    rows = torch.tensor([0, 0, 0, 3, -1, 0, 0], device=device)
    positions = torch.tensor([0, 0, 0, 0, 0, 5, -1], device=device)
    data_plane.reshape_and_cache_fp4([src], [src], slots, [kp], [vp], token_rows=rows, token_positions=positions)
    assert np.array_equal(kp.cpu().numpy().reshape(before.shape), before) and torch.equal(kp, vp)
    # the decode form: row i, position 0; no tokens at all
    data_plane.reshape_and_cache_fp4([src], [src], slots[:0], [kp], [vp])
    data_plane.reshape_and_cache_fp4([src[:, :, :1]], [src[:, :, :1]], slots[3:6], [kp], [vp])
    expect_k, expect_v = before.copy(), before.copy()
    for i, s in enumerate((5, 6, 7)):
        fp4_ref.store(expect_k, s, src[i, :, 0].cpu().double().numpy(), False)
        fp4_ref.store(expect_v, s, src[i, :, 0].cpu().double().numpy(), True)
    assert np.array_equal(kp.cpu().numpy().reshape(before.shape), expect_k)
    assert np.array_equal(vp.cpu().numpy().reshape(before.shape), expect_v)


@pytest.mark.parametrize("heads,sub,layers,nb", [(1, 1, 1, 1), (2, 1, 3, 5), (8, 1, 1, 7), (3, 2, 1, 3), (11, 1, 34, 1)])
def test_gather_is_exact(native_lib, device, heads, sub, layers, nb):
    rng = np.random.default_rng(heads)
    num_blocks = 9
    raw = [fp4_ref.random_pool(rng, num_blocks * sub, heads, 1, 253) for _ in range(2 * layers)]
    raw[0][3, 0, fp4_ref.CODES + 5] = 255
    raw[0][4, 0, fp4_ref.CODES:] = 0
    pools = [fp4_ref.to_torch(p, sub).to(device) for p in raw]
    wide = torch.from_numpy(rng.integers(0, num_blocks, (2, nb + 3)))
    wide[0, 0], wide[1, nb - 1] = num_blocks, -5  # read the null block
    ids = wide.to(device)[:, :nb]
    outs = [torch.full((2, nb * 16 * sub, heads, 128), 7.0, dtype=torch.bfloat16, device=device) for _ in range(2 * layers)]
    data_plane.gather_blocks_fp4(pools[:layers], pools[layers:], ids, outs[:layers], outs[layers:])
    at = np.where((wide[:, :nb].numpy() < 0) | (wide[:, :nb].numpy() >= num_blocks), 0, wide[:, :nb].numpy())
    for i, out in enumerate(outs):
        values = fp4_ref.load(raw[i], i >= layers).reshape(num_blocks, 16 * sub, heads, 128)
        expect = torch.from_numpy(values[at].reshape(2, nb * 16 * sub, heads, 128)).to(torch.bfloat16)
        assert torch.equal(out.cpu().view(torch.int16)[~expect.isnan()], expect.view(torch.int16)[~expect.isnan()])
        assert torch.equal(out.cpu().isnan(), expect.isnan())


@pytest.mark.parametrize("dtype,shape", [(torch.bfloat16, (16, 8, 128)), (torch.uint8, (1, 8, 1088)), (torch.float32, (3, 1, 5)),
                                         (torch.uint8, (1, 1, 7)), (torch.float16, (1, 3, 7))])
@pytest.mark.parametrize("layers", [1, 33])
def test_copy_blocks(native_lib, device, dtype, shape, layers):
    gen = torch.Generator().manual_seed(layers)
    x = torch.randint(0, 200, (layers, 2, 12, *shape), generator=gen).to(dtype)
    got = x.to(device)
    src = torch.tensor([3, 3, 3, 5, 12, 4, 6, 2, -1])
    dst = torch.tensor([1, 7, 8, 9, 10, 4, 12, -1, 11])  # 4 to itself, 6 nowhere, 2 nowhere; 12 and -1 read block 0
    data_plane.copy_blocks([p[0] for p in got], [p[1] for p in got], src.to(device), dst.to(device))
    for s, d in ((3, 1), (3, 7), (3, 8), (5, 9), (0, 10), (0, 11)):
        x[:, :, d] = x[:, :, s]
    assert torch.equal(got.cpu(), x)


def test_copy_blocks_checks_with_index_checks(native_lib, device):
    pool = torch.zeros(8, 1, 1, 1088, dtype=torch.uint8, device=device)
    ids = lambda *x: torch.tensor(x, device=device)  # noqa: E731
    previous = data_plane.set_index_checks(True)
    try:
        with pytest.raises(IndexError):
            data_plane.copy_blocks([pool], [pool.clone()], ids(8), ids(1))
        with pytest.raises(IndexError):
            data_plane.copy_blocks([pool], [pool.clone()], ids(1), ids(-1))
        with pytest.raises(ValueError, match="twice"):
            data_plane.copy_blocks([pool], [pool.clone()], ids(1, 2), ids(3, 3))
        with pytest.raises(ValueError, match="source"):
            data_plane.copy_blocks([pool], [pool.clone()], ids(1, 2), ids(2, 3))
        data_plane.copy_blocks([pool], [pool.clone()], ids(1, 2), ids(1, 3))  # a block onto itself is no move
    finally:
        data_plane.set_index_checks(previous)
