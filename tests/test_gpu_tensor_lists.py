"""Per-layer lists of the store, the gather and the block copies: whatever is not uniform is refused, wherever it stands in a
list, and tuples and other sequences are taken like lists."""

import pytest
import torch

from mini_infra_qwen3_amd import _native, data_plane

LAYERS = 5


def test_cpu_tensors_and_other_things_have_no_addresses(native_lib):
    t = torch.zeros(2, 3)
    assert _native.addresses([t, t], t) is None
    assert _native.addresses([t, 3], t) is None
    assert _native.addresses("no", t) is None
    assert _native.addresses([t], 3) is None
    with pytest.raises(TypeError):
        _native._tensor_lists.addresses([t], t)


@pytest.mark.gpu
def test_addresses(native_lib, device):
    ts = [torch.zeros(4, 6, device=device)[:, :4] for _ in range(3)]
    assert _native.addresses(ts, ts[0]) is None  # not contiguous
    assert list(_native.addresses(tuple(ts), ts[0], True)) == [t.data_ptr() for t in ts]
    whole = [t.contiguous() for t in ts]
    assert list(_native.addresses(whole, whole[0])) == [t.data_ptr() for t in whole]
    assert _native.addresses(whole + ts[:1], whole[0], True) is None  # other strides
    assert list(_native.addresses([], ts[0])) == []
    empty = torch.zeros(0, 4, device=device)
    assert list(_native.addresses([empty], empty)) == [None]  # address 0
    assert _native.addresses([torch.zeros(4, 4, device=device).to_sparse()], whole[0]) is None


def odd_ones(t):
    """Tensors that do not go with t."""
    return [t.cpu(), t.to(torch.int16), torch.cat((t, t[:1])), t.transpose(0, -1).contiguous().transpose(0, -1),
            t.reshape(1, *t.shape)]


class Other(list):
    pass


def calls(device):
    pools = [[torch.zeros(6, 1, 2, 1088, dtype=torch.uint8, device=device) for _ in range(LAYERS)] for _ in range(2)]
    rows = [[torch.randn(3, 2, 4, 128, device=device).to(torch.bfloat16) for _ in range(LAYERS)] for _ in range(2)]
    outs = [[torch.zeros(2, 48, 2, 128, dtype=torch.bfloat16, device=device) for _ in range(LAYERS)] for _ in range(2)]
    slots = torch.tensor([5, 17, 40], device=device)
    ids = torch.tensor([[1, 2, 3], [0, 1, 5]], device=device)
    pair = torch.tensor([1], device=device), torch.tensor([4], device=device)
    return {"store": (lambda k, v, a, b: data_plane.reshape_and_cache_fp4(k, v, slots, a, b), [*rows, *pools]),
            "gather": (lambda a, b, k, v: data_plane.gather_blocks_fp4(a, b, ids, k, v), [*pools, *outs]),
            "copy": (lambda a, b: data_plane.copy_blocks(a, b, *pair), pools)}


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["store", "gather", "copy"])
def test_odd_tensors_are_refused(native_lib, device, name):
    call, lists = calls(device)[name]
    call(*lists)
    for which in range(len(lists)):
        for at in (0, 2, LAYERS - 1):
            for odd in odd_ones(lists[which][at]):
                if at == 0 and name == "store" and which < 2 and odd.dtype is torch.bfloat16 and odd.is_cuda and odd.dim() == 4:
                    continue  # the first decides the sources' rows and strides; the others are then the odd ones
                changed = [list(x) for x in lists]
                changed[which][at] = odd
                with pytest.raises((ValueError, RuntimeError)):
                    call(*changed)
    for short in range(len(lists)):
        with pytest.raises(ValueError):
            call(*[x[:-1] if i == short else x for i, x in enumerate(lists)])


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["store", "gather", "copy"])
def test_sequences(native_lib, device, name):
    """Lists, tuples, subclasses and other sequences write the same."""
    call, lists = calls(device)[name]
    if name != "store":
        for p in lists[0] + lists[1]:
            p.copy_(torch.randint(0, 120, p.shape, device=device, dtype=torch.uint8))
    written = lists[2:] if len(lists) == 4 else lists
    before = [[t.clone() for t in x] for x in lists]
    results = []
    for kind in (list, tuple, Other, lambda x: __import__("collections").UserList(x)):
        for x, y in zip(lists, before):
            for t, s in zip(x, y):
                t.copy_(s)
        call(*[kind(x) for x in lists])
        results.append([t.clone() for x in written for t in x])
    for other in results[1:]:
        assert all(torch.equal(a, b) for a, b in zip(results[0], other))
    assert any(not torch.equal(a, b) for a, b in zip(results[0], [t for x in (before[2:] if len(lists) == 4 else before) for t in x]))
