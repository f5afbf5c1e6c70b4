"""Groups of state caches beside one another in memory, and groups without slots."""

import ctypes
import itertools

import pytest
import torch

import causal_conv1d_cute as C
from causal_conv1d_cute import _lib
from causal_conv1d_cute.slots import _apart
from test_slots import apply, int32, same


@pytest.mark.parametrize("slots,stride", [(1, 10), (2, 10), (4, 10), (3, 7)])
def test_apart_is_exact_for_equal_strides(slots, stride):
    """Every placement of up to three caches against the sets of their bytes."""

    def bytes_of(p, row):
        return {p + s * stride + b for s in range(slots) for b in range(row)}

    rows = (3, 4, 5)[: stride // 3]
    for q, r in itertools.product(range(0, slots * stride + 6, 1), repeat=2):
        spans = [(20, stride, rows[0]), (20 + q, stride, rows[1]), (14 + r, stride, rows[-1])]
        if slots == 1:  # one slot: the stride is the row
            spans = [(p, row, row) for p, _, row in spans]
        sets = [bytes_of(p, row) for p, _, row in spans]
        want = not any(a & b for a, b in itertools.combinations(sets, 2))
        assert _apart(slots, spans) == want, spans


def test_third_cache_in_the_next_slot_of_the_first():
    assert not _apart(4, [(0, 100, 40), (50, 100, 40), (95, 100, 40)])
    assert not _apart(4, [(0, 10, 4), (4, 10, 4), (8, 10, 4)])
    assert _apart(4, [(0, 12, 4), (4, 12, 4), (8, 12, 4)])
    assert not _apart(4, [(0, 100, 40), (50, 60, 10)])


@pytest.mark.gpu
def test_group_with_such_a_cache_is_refused():
    memory = torch.zeros(64, device="cuda")
    views = [memory[at:].as_strided((4, 4), (10, 1)) for at in (0, 4, 8)]
    with pytest.raises(ValueError, match="share"):
        C.StateSlots(views)
    C.StateSlots(views[:2])


@pytest.mark.gpu
@pytest.mark.parametrize("first", ["source", "destination"])
def test_source_right_behind_a_view(first):
    """The last slot of an interleaved cache ends where the other group begins."""
    # Five lines of 1024 bytes; the view has the second halves of four of them, the other group (128
    # floats a slot) lies before the first of these or behind the last.
    memory = torch.arange(2 * 5 * 128, dtype=torch.float32, device="cuda")
    if first == "source":
        other, view = memory[:128].view(1, 128), memory[: 4 * 256].view(4, 256)[:, 128:]
    else:
        view, other = memory[: 4 * 256].view(4, 256)[:, 128:], memory[4 * 256 :].view(2, 128)
    want, rec = [view.clone()], [other.clone()]
    apply(want, [0, -1], [3, 1], source=rec)
    C.StateSlots([view]).copy(int32([0, -1]), int32([3, 1]), source=C.StateSlots([other]))
    same([view], want)
    # The other way round: from the view.
    apply(rec, [2], [0], source=want)
    C.StateSlots([other]).copy(int32([2]), int32([0]), source=C.StateSlots([view]))
    same([other, view], rec + want)


@pytest.mark.gpu
def test_source_without_slots():
    """Nothing to read: lists that are empty or clear slots only."""
    group = C.StateSlots([torch.ones(3, 8, device="cuda")])
    none = C.StateSlots([torch.ones(0, 8, device="cuda")])
    group.copy(int32([]), int32([]), source=none)
    group.copy(int32([-1]), int32([1]), source=none)
    assert group.caches[0].sum(1).tolist() == [8, 0, 8]
    none.copy(int32([]), int32([]), source=group)


def swap_data(cache, other):
    cache.data = other


@pytest.mark.gpu
@pytest.mark.parametrize("change", [swap_data, lambda cache, other: cache.set_(other)])
@pytest.mark.parametrize("step", ["copy", "compact", "source"])
def test_cache_with_other_memory(change, step):
    """A cache is followed to the memory that it was given; the memory before is left alone."""
    caches = [torch.randn(4, 8, device="cuda"), torch.randn(4, 3, device="cuda")]
    rec = [torch.randn(2, 8, device="cuda"), torch.randn(2, 3, device="cuda")]
    group, source = C.StateSlots(caches), C.StateSlots(rec)
    live = torch.tensor([0, 1, 0, 1], dtype=torch.bool, device="cuda")
    group.copy(int32([0]), int32([1]))
    group.copy(int32([0]), int32([1]), source=source)
    moved = rec if step == "source" else caches
    old = moved[0].detach()
    before = old.clone()
    change(moved[0], torch.randn(len(old), 8, device="cuda"))
    want = [c.clone() for c in caches]
    if step == "copy":
        group.copy(int32([0, -1]), int32([1, 3]))
        apply(want, [0, -1], [1, 3])
    elif step == "compact":
        group.compact(live)
        apply(want, [3], [0])
    else:
        group.copy(int32([1]), int32([2]), source=source)
        apply(want, [1], [2], source=rec)
    same(caches, want)
    assert torch.equal(old, before)


@pytest.mark.gpu
def test_cache_with_memory_that_does_not_fit():
    caches = [torch.zeros(4, 8, device="cuda"), torch.zeros(4, 3, device="cuda")]
    group = C.StateSlots(caches)
    caches[0].data = torch.zeros(5, 8, device="cuda")
    for _ in range(2):
        with pytest.raises(ValueError, match="slots"):
            group.copy(int32([0]), int32([1]))
    caches[0].data = torch.zeros(4, 3, 8, device="cuda").transpose(1, 2)
    with pytest.raises(C.Unsupported):
        group.compact(torch.ones(4, dtype=torch.bool, device="cuda"))
    caches[0].data = caches[1].data
    with pytest.raises(ValueError, match="share"):
        group.copy(int32([0]), int32([1]))
    caches[0].data, caches[1].data = torch.ones(6, 8, device="cuda"), torch.ones(6, 3, device="cuda")
    group.copy(int32([-1]), int32([5]))
    assert len(group) == 6 and [c.sum().item() for c in caches] == [40, 15]


@pytest.mark.gpu
def test_compaction_of_no_slots_through_c():
    """Caches whose slots have bytes, but of which there are none: the count is 0 and nothing moves."""
    memory = torch.arange(64, dtype=torch.uint8, device="cuda")
    work = torch.full((2,), 7, dtype=torch.int32, device="cuda")
    table = (ctypes.c_int64 * 5)(memory.data_ptr(), memory.data_ptr(), 16, 16, 16)
    lib = _lib.load()
    stream = torch.cuda.current_stream().cuda_stream
    assert lib.cc1d_slots_compact(table, 1, None, 0, None, work[:1].data_ptr(), work[1:].data_ptr(), stream) == 0
    assert work.tolist() == [0, 0] and memory.tolist() == list(range(64))


@pytest.mark.gpu
def test_wide_indices_outside_int32(request):
    """Their low 32 bits name slots; they are skipped and reported all the same."""
    request.node._expect_status = True
    cache = torch.arange(6.0, device="cuda").reshape(6, 1).repeat(1, 4)
    want = cache.clone()
    wide = lambda *x: torch.tensor(x, device="cuda")  # noqa: E731
    group = C.StateSlots([cache])
    group.copy(wide(2**32, 1, 2**32 + 3), wide(2, 2**32 + 3, 4))
    assert C.device_status() == _lib.DEV_BAD_SLOT and torch.equal(cache, want)
    group.copy(wide(-(2**32) - 1, 5, -1), wide(1, -(2**32) - 1, 2**32 - 1))
    assert C.device_status() == _lib.DEV_BAD_SLOT and torch.equal(cache, want)
    group.copy(wide(1, -1), wide(0, 5))
    assert C.device_status() == 0 and cache[:, 0].tolist() == [1, 1, 2, 3, 4, 0]


@pytest.mark.gpu
@pytest.mark.parametrize("pad", [2**32, 2**31, -(2**31) - 1, -(2**63)])
def test_pad_outside_int32(pad):
    """Its low 32 bits name a slot, which would then be cleared or skipped."""
    cache = torch.ones(3, 4, device="cuda")
    with pytest.raises(ValueError, match="pad_slot_id"):
        C.StateSlots([cache]).copy(int32([0]), int32([1]), pad_slot_id=pad)
    assert (cache == 1).all()
    C.StateSlots([cache]).copy(int32([2**31 - 1]), int32([1]), pad_slot_id=2**31 - 1)
    assert cache.sum(1).tolist() == [4, 0, 4]
