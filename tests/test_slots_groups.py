"""Groups of state caches beside one another in memory, and groups without slots."""

import pytest
import torch

import causal_conv1d_cute as C
from test_slots import apply, int32, same


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
