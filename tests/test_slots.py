"""Slot moves of StateSlots against the same moves one by one; everything is bit for bit."""

import pytest
import torch

import causal_conv1d_cute as C
from causal_conv1d_cute import _lib

BF, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def caches(slots, device="cuda", seed=0):
    """Caches of several dtypes and slot sizes: vectors, odd bytes, a view of a wider tensor, nothing."""
    r = torch.Generator().manual_seed(seed)
    new = lambda *s: torch.randn(slots, *s, generator=r)  # noqa: E731
    wide = new(2, 3, 40).to(F16).to(device)
    return [new(48, 3).to(BF).to(device), new(2, 16, 128).to(device), new(5).to(torch.bfloat16).to(device),
            (new(7) * 50).to(torch.int8).to(device), new(1025).to(device), wide[:, 1], new(0, 4).to(device),
            new().to(device), new(3).to(torch.float64).to(device)]


def apply(group, src, dst, pad=-1, source=None):
    """The definition: one pair after another."""
    slots = group[0].shape[0]
    for s, d in zip(src, dst):
        if d == pad or not 0 <= d < slots or (s != pad and not 0 <= s < (source or group)[0].shape[0]):
            continue
        for i, c in enumerate(group):
            c[d] = 0 if s == pad else (source or group)[i][s].clone()


def same(a, b):
    for x, y in zip(a, b):
        assert torch.equal(x.cpu().reshape(-1).contiguous().view(torch.uint8), y.cpu().reshape(-1).contiguous().view(torch.uint8))


def int32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda").reshape(-1)


def test_group_errors():
    with pytest.raises(ValueError):
        C.StateSlots([])
    with pytest.raises(ValueError):
        C.StateSlots([torch.zeros(3, 2), torch.zeros(4, 2)])
    with pytest.raises(ValueError):
        C.StateSlots([torch.tensor(1.0)])
    with pytest.raises(C.Unsupported):
        C.StateSlots([torch.zeros(3, 2)])


def test_c_abi_refuses_before_launch():
    lib = _lib.load()
    import ctypes

    def table(dst=1 << 20, src=1 << 20, ds=64, ss=64, row=64):
        return (ctypes.c_int64 * 5)(dst, src, ds, ss, row)

    copy, compact = lib.cc1d_slots_copy, lib.cc1d_slots_compact
    call = lambda t, n=1, pairs=1, a=4, b=4, s=1, d=1: copy(t, n, s, d, pairs, a, b, -1, None, None)  # noqa: E731
    assert call(table(), n=65) == 1 and call(table(), n=-1) == 1 and call(None) == 1
    assert call(table(dst=0)) == 1 and call(table(ds=32)) == 1 and call(table(row=-1)) == 1
    assert call(table(), pairs=-1) == 1 and call(table(), a=2**31) == 1 and call(table(), s=None) == 1
    assert call(table(), pairs=0) == 0 and call(table(), n=0) == 0
    assert call(table(src=(1 << 20) + 128)) == 1 and b"overlap" in lib.cc1d_last_error()
    assert call(table(), a=3) == 1
    assert compact(table(), 1, 1, 4, 1, None, 1, None) == 1 and compact(table(), 1, None, 4, 1, 1, 1, None) == 1
    assert compact(table(src=4096), 1, 1, 4, 1, 1, 1, None) == 1
    assert compact(table(), 1, 1, 2**30, 1, 1, 1, None) == 1


@pytest.mark.gpu
def test_group_errors_on_gpu():
    a = torch.zeros(4, 8, device="cuda")
    with pytest.raises(ValueError, match="share"):
        C.StateSlots([a, a])
    with pytest.raises(ValueError, match="share"):
        C.StateSlots([a, a[:, 4:]])
    with pytest.raises(ValueError, match="share"):
        C.StateSlots([a[:1].expand(4, 8)])
    with pytest.raises(C.Unsupported):
        C.StateSlots([torch.zeros(4, 8, 3, device="cuda").transpose(1, 2)])
    C.StateSlots([a[:, :4], a[:, 4:]])
    g = C.StateSlots([a])
    with pytest.raises(ValueError):
        g.copy(int32([0, 1]), int32([2]))
    with pytest.raises(ValueError):
        g.copy(int32([0]), int32([1]), source=C.StateSlots([torch.zeros(4, 9, device="cuda")]))
    with pytest.raises(ValueError, match="share"):
        g.copy(int32([0]), int32([1]), source=C.StateSlots([a]))
    with pytest.raises(ValueError):
        g.compact(torch.ones(5, dtype=torch.bool, device="cuda"))


LISTS = {
    "none": ([], []),
    "one": ([2], [5]),
    "fork": ([1, 1, 1, 4], [0, 7, 9, 10]),
    "free": ([-1, 3, -1], [2, 8, 0]),
    "skip": ([1, 2, 3], [-1, 6, -1]),
    "self": ([3, 4], [3, 9]),
    "chain": ([0, 1, 2, 3], [1, 2, 3, 4]),
    "swap": ([0, 1], [1, 0]),
    "twice": ([0, 1, 2], [5, 5, 5]),
    "free-then-copy": ([-1, 2, 2], [2, 3, 4]),
    "many": (list(range(0, 11)) * 2, list(range(11, 22)) + list(range(22, 33))),
}


@pytest.mark.gpu
@pytest.mark.parametrize("name", sorted(LISTS))
def test_copy(name):
    src, dst = LISTS[name]
    group, want = caches(33), caches(33)
    apply(want, src, dst)
    C.StateSlots(group).copy(int32(src), int32(dst))
    same(group, want)


@pytest.mark.gpu
@pytest.mark.parametrize("seed", range(6))
def test_copy_of_random_lists(seed):
    """Long lists, with and without repeated destinations and chains, wide index types."""
    r = torch.Generator().manual_seed(seed)
    n = [3, 9, 40, 64, 65, 200][seed]
    slots = 150
    group, want = caches(slots, seed=seed), caches(slots, seed=seed)
    src, dst = torch.randint(-1, slots, (n,), generator=r), torch.randint(-1, slots, (n,), generator=r)
    if seed % 2:
        p = torch.randperm(slots, generator=r)
        m = min(n, slots // 2)
        dst, src = p[:m], p[m:][torch.randint(0, slots - m, (m,), generator=r)]
    apply(want, src.tolist(), dst.tolist())
    C.StateSlots(group).copy(src.cuda(), dst.cuda())
    same(group, want)


@pytest.mark.gpu
def test_copy_pad_value_and_bad_indices(request):
    request.node._expect_status = True
    group, want = caches(6), caches(6)
    apply(want, [0, 99, 2], [1, 3, 99], pad=99)
    C.StateSlots(group).copy(int32([0, 99, 2]), int32([1, 3, 99]), pad_slot_id=99)
    assert C.device_status() == 0
    same(group, want)
    C.StateSlots(group).copy(int32([0, 6, -3, 1]), int32([6, 2, 3, 4]))
    assert C.device_status() == _lib.DEV_BAD_SLOT
    apply(want, [1], [4])
    same(group, want)


@pytest.mark.gpu
def test_commit_from_another_group():
    """The recorded states of a verified draft, rows x steps, committed to the slots."""
    group, want, rec = caches(9), caches(9), caches(12, seed=5)
    apply(want, [3, 0, 11, -1], [8, 2, 2, 4], source=rec)
    C.StateSlots(group).copy(int32([3, 0, 11, -1]), int32([8, 2, 2, 4]), source=C.StateSlots(rec))
    same(group, want)


@pytest.mark.gpu
def test_more_caches_than_one_launch_takes():
    group = [torch.randn(5, 3 + i % 7, device="cuda") for i in range(150)]
    want = [c.clone() for c in group]
    apply(want, [1, 0], [4, 2])
    g = C.StateSlots(group)
    g.copy(int32([1, 0]), int32([4, 2]))
    same(group, want)
    live = torch.tensor([0, 1, 0, 1, 1], dtype=torch.bool, device="cuda")
    remap, count = g.compact(live)
    assert remap.tolist() == [-1, 1, -1, 0, 2] and int(count) == 3
    apply(want, [3, 4], [0, 2])
    same(group, want)


@pytest.mark.gpu
def test_more_slots_than_the_bitmap_holds():
    slots = (1 << 18) + 5
    a = torch.arange(slots, dtype=torch.int32, device="cuda").reshape(-1, 1).repeat(1, 4)
    want = [a.clone()]
    src, dst = [slots - 1, slots - 2, 0, -1], [0, slots - 1, 7, 3]
    apply(want, src, dst)
    C.StateSlots([a]).copy(int32(src), int32(dst))
    same([a], want)


@pytest.mark.gpu
@pytest.mark.parametrize("slots", [1, 2, 31, 33, 1024, 1025, 2500])
@pytest.mark.parametrize("share", [0.0, 0.1, 0.5, 0.9, 1.0])
def test_compact(slots, share):
    r = torch.Generator().manual_seed(slots)
    live = torch.rand(slots, generator=r) < share
    group = [torch.randn(slots, 24, device="cuda"), torch.randn(slots, 5, device="cuda").to(BF)]
    want = [c.clone() for c in group]
    m = int(live.sum())
    holes = [i for i in range(m) if not live[i]]
    movers = [i for i in range(m, slots) if live[i]]
    apply(want, movers, holes)
    place = dict(zip(movers, holes))
    remap, count = C.StateSlots(group).compact(live.cuda())
    assert remap.dtype == count.dtype == torch.int32 and int(count) == m
    assert remap.tolist() == [place.get(i, i) if live[i] else -1 for i in range(slots)]
    same(group, want)


@pytest.mark.gpu
def test_moves_in_a_graph():
    group, want = caches(12), caches(12)
    g = C.StateSlots(group)
    src, dst = int32([1, 2]), int32([5, 6])
    live = torch.tensor([0, 1] * 6, dtype=torch.bool, device="cuda")
    C.device_status()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        g.copy(src, dst)
        remap, count = g.compact(live)
    src.copy_(int32([3, -1]))
    graph.replay()
    torch.cuda.synchronize()
    apply(want, [3, -1], [5, 6])
    apply(want, [7, 9, 11], [0, 2, 4])
    same(group, want)
    assert int(count) == 6 and remap.tolist() == [-1, 1, -1, 3, -1, 5, -1, 0, -1, 2, -1, 4]
