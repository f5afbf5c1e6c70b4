"""Slot moves between the state caches of a model: copy, fork, clear, commit and compaction.

A serving engine keeps, for every layer, a conv-state cache (slots, dim, width - 1) and a
delta-rule state cache (slots, heads, dk, dv); a request owns one slot in all of them. StateSlots
holds such a group and moves whole slots of every cache in one launch (cc1d_slots_copy,
cc1d_slots_compact).
"""

import ctypes

import torch

from . import _ops
from .functional import PAD_SLOT_ID, _flags, _int32, _unsupported

_MAX_CACHES = 64  # caches one launch takes
_data_ptr, _numel, _stride = torch.Tensor.data_ptr, torch.Tensor.numel, torch.Tensor.stride


def _apart(slots, spans):
    """Whether no byte belongs to two of the caches (address, bytes from slot to slot, bytes of a slot).

    Caches whose address ranges meet are apart if they are interleaved layers of one allocation: equal
    strides, and the rows of one between those of the other.
    """
    spans = sorted(spans)
    for i, (p, ps, pr) in enumerate(spans):
        end = p + (slots - 1) * ps + pr
        for q, qs, qr in spans[i + 1 :]:
            if q >= end:
                break
            at = (q - p) % ps
            if ps != qs or at < pr or at + qr > ps:
                return False
    return True


def _slot_list(index, device):
    """Slots as contiguous int32 on device; wider ones outside it stay outside every cache."""
    if index.dtype == torch.int64:
        index = index.clamp(-(2**31), 2**31 - 1)
    return _int32(index, device).contiguous()


class StateSlots:
    """A group of caches whose first axis is the slot.

    The caches keep their own storage and dtypes; the object holds references to them. Addresses are
    taken once, and again when a cache has been given other memory, size or strides (cache.data = ...,
    set_, resize_), which then has to satisfy the constructor's rules.
    """

    def __init__(self, caches):
        """Args:
            caches: CUDA tensors of shape (slots, ...) with the same number of slots, each slot
                contiguous in memory, and no two of them sharing memory.

        Raises:
            ValueError: shapes that do not form a group, or caches that share memory.
            Unsupported: CPU tensors, or slots that are not contiguous.
        """
        self.caches = list(caches)
        self._layout()

    def _place(self):
        """What the addresses of the slots depend on (0.3 us a cache)."""
        c = self.caches
        return [*map(_data_ptr, c), *map(_numel, c), *map(_stride, c)]

    def _fresh(self):
        if self._place() != self._placed:
            self._layout()
        return self

    def _layout(self):
        """Check the caches and take their addresses."""
        caches = self.caches
        self._placed = self._own = None  # nothing is kept of caches that are refused
        if not caches or any(c.dim() < 1 for c in caches):
            raise ValueError("StateSlots needs one cache at least, each with a slot axis")
        if any(c.shape[0] != caches[0].shape[0] for c in caches):
            raise ValueError(f"caches have {[c.shape[0] for c in caches]} slots")
        if not all(c.is_cuda for c in caches):
            _unsupported("a cache is not a CUDA tensor")
        if any(c.device != caches[0].device for c in caches):
            _unsupported("caches are on different devices")
        for c in caches:
            if c.shape[0] and not c[0].is_contiguous():
                _unsupported(f"slots of a cache with strides {c.stride()} are not contiguous")
        self.slots = caches[0].shape[0]
        self.device = caches[0].device
        # (pointer, bytes from slot to slot, bytes of a slot) of each cache that holds anything
        self._rows = []
        spans = []
        for c in caches:
            size = c.element_size()
            row = (c[0].numel() if c.shape[0] else 0) * size
            stride = c.stride(0) * size if c.shape[0] > 1 else row
            if c.shape[0] > 1 and stride < row:
                raise ValueError(f"slots of a cache with strides {c.stride()} share memory")
            self._rows.append((c.data_ptr(), stride, row))
            if row:
                spans.append((c.data_ptr(), stride, row))
        # A byte of two caches would make a later move depend on the launch order.
        if not _apart(self.slots, spans):
            raise ValueError("two caches of a group share memory")
        self._placed = self._place()

    def _table(self, source):
        """cc1d_slot_cache arrays of at most 64 caches each, for moves out of source, as (address,
        caches, the memory itself); those of moves within the group are made once."""
        if source is self and self._own is not None:
            return self._own
        rows = [(d, s, ds, ss, n) for (d, ds, n), (s, ss, _) in zip(self._rows, source._rows) if n]
        tables = []
        for i in range(0, len(rows), _MAX_CACHES):
            part = rows[i : i + _MAX_CACHES]
            flat = (ctypes.c_int64 * (5 * len(part)))(*(x for r in part for x in r))
            tables.append((ctypes.addressof(flat), len(part), flat))
        if source is self:
            self._own = tables
        return tables

    def copy(self, src_indices, dst_indices, source=None, pad_slot_id=PAD_SLOT_ID):
        """For each pair i, in order: slot dst_indices[i] becomes a copy of slot src_indices[i].

        A prompt is forked by repeating its slot among the sources; a slot is freed (cleared) by a
        source of pad_slot_id; a pair with a destination of pad_slot_id is skipped. The result is
        that of the pairs applied one after another, so a later pair sees what an earlier one wrote.

        Args:
            src_indices, dst_indices: (pairs,) integer slots; pairs with other indices outside the
                caches are skipped (and reported through device_status()).
            source: StateSlots to copy from (default: this one), with caches of the same slot sizes
                and dtypes in the same order and apart from these: for instance the recorded states
                of a verified draft, viewed as (rows * steps, ...).
            pad_slot_id: the index value described above.
        """
        self._fresh()
        source = self if source is None else source._fresh()
        if src_indices.dim() != 1 or src_indices.shape != dst_indices.shape:
            raise ValueError(
                f"index lists of shapes {tuple(src_indices.shape)} and {tuple(dst_indices.shape)}"
            )
        if not -(2**31) <= pad_slot_id < 2**31:
            raise ValueError(f"pad_slot_id {pad_slot_id} is not a 32-bit index")
        if source is not self:
            if source.device != self.device:
                _unsupported("source caches are on another device")
            if [(c.dtype, tuple(c.shape[1:])) for c in source.caches] != [
                (c.dtype, tuple(c.shape[1:])) for c in self.caches
            ]:
                raise ValueError("source caches differ in slot shape or dtype")
            self._check_other(source)
        src, dst = _slot_list(src_indices, self.device), _slot_list(dst_indices, self.device)
        for at, n, _ in self._table(source):
            _ops.slots_copy(self.caches, source.caches if source is not self else [], at, n, src, dst,
                            source.slots, self.slots, pad_slot_id)

    def _check_other(self, source):
        """Every source cache lies apart from every cache of this group."""
        mine = [(p, p + (self.slots - 1) * s + r) for p, s, r in self._rows if r]
        for p, s, r in source._rows:
            end = p + (source.slots - 1) * s + r
            if r and any(p < e and b < end for b, e in mine):
                raise ValueError("source caches share memory with these")

    def compact(self, live):
        """Move the live slots to the front with the fewest moves.

        With m live slots, the i-th free slot below m receives the i-th live slot from m on, both
        in ascending order; live slots below m stay. Slots from m on keep their old contents.

        Args:
            live: (slots,) bool/uint8, nonzero for slots in use.

        Returns:
            (remap, count): int32 (slots,) new slot of each old one (-1: not live), and int32 ()
            the number of live slots, both on the device (nothing is synchronised).
        """
        self._fresh()
        if tuple(live.shape) != (self.slots,):
            raise ValueError(f"live must have shape ({self.slots},), got {tuple(live.shape)}")
        live = _flags(live, self.device)
        live = live if live.is_contiguous() else live.contiguous()
        # One allocation: remap, the count, and the list of moves.
        n = self.slots
        work = torch.empty(3 * n + 2, dtype=torch.int32, device=self.device)
        remap, count, moves = work[:n], work[n], work[n + 1 :]
        tables = self._table(self) or [(0, 0, None)]
        for at, k, _ in tables:
            _ops.slots_compact(self.caches, at, k, live, remap, count, moves)
        return remap, count

    def __len__(self):
        return self.slots


__all__ = ["StateSlots"]
