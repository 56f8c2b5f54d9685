"""Paged storage of keys and values.

A `KVGroup` serves all entries of the run order whose mixers have the same need
(kv heads, head size, all keys or a window).  It owns a pool of pages of 64
positions, one page table (a row per slot), and for each of its entries a key and
a value array [n_pages, n_kv_heads, 64, head_dim].  A sequence's pages are the
same for every entry of the group: table entry e of a slot names the page that
holds positions 64e..64e+63 (all-keys group) or, in a window group, the positions
p with (p // 64) % ring_pages == e: a ring of ring_pages = ceil(window / 64) pages
that is written round and round.

With `need.bits` 4 the arrays are uint8 [n_pages, n_kv_heads, ops.tile4_bytes(head_dim)]:
codes of 4 bits with a scale and a middle per 64 numbers (parts/attention4.py).

Slots may share pages (a forked sequence begins with the pages of the one it comes
from): a page counts its holders, and `grow` gives a slot that is about to write
into a page with other holders a page of its own with the same contents first.

The host keeps the table and the lengths; `flush()` copies changed rows to the
device before a step runs.
"""
from __future__ import annotations

from typing import Dict, List, Optional, Sequence

import numpy as np
import torch

from .. import ops
from ..errors import CacheError
from ..parts.base import KVNeed
from .pool import IdPool

PAGE = ops.PAGE_TOKENS


def _best_runs(table: np.ndarray, members: List[int]) -> tuple:
    """(pages saved, [(members, pages)]): rows of page numbers as a tree of common beginnings; a branch is one run as far as all of
    it agrees, or what its branches save by themselves if that is more."""
    m, n = table.shape
    agree = (table == table[0]).all(axis=0)
    common = n if agree.all() else int(np.argmin(agree))
    whole = ((m - 1) * common, [(members, common)] if common else [])
    if m <= 2 or common == n:
        return whole
    saved, runs = 0, []
    pages, which = np.unique(table[:, common], return_inverse=True)
    for b in range(len(pages)):
        rows = np.flatnonzero(which == b)
        if len(rows) > 1:
            s, r = _best_runs(table[rows], [members[i] for i in rows])
            saved, runs = saved + s, runs + r
    return whole if whole[0] >= saved else (saved, runs)


class KVGroup:
    def __init__(self, need: KVNeed, n_entries: int, n_pages: int, n_slots: int,
                 max_seq_len: int, dtype: torch.dtype, device: torch.device, chunk_tokens: int = 1):
        self.need = need
        self.n_entries = n_entries
        # A step that continues a sequence by n tokens stores all n before any of them attends, so
        # the ring must still hold the window of the first while it holds the last: window + n - 1
        # positions.  `chunk_tokens` is the n the ring is made for (a sequence holds at most
        # ceil(length / 64) pages in any case, so a longer ring costs nothing until it is filled).
        self.ring_pages = 0 if need.window is None else (need.window + max(1, chunk_tokens) - 1 + PAGE - 1) // PAGE
        full_entries = (max_seq_len + PAGE - 1) // PAGE
        self.table_stride = max(1, min(full_entries, self.ring_pages) if self.ring_pages else full_entries)
        self.pages = IdPool(n_pages, "page")
        if need.bits is not None:
            from ..parts import attention4
            if need.bits != 4 or need.keys_only or (need.v_head_dim or need.head_dim) != need.head_dim or not attention4.supports(need.head_dim):
                raise CacheError(f"no cache in {need.bits} bits for heads of {need.head_dim} numbers: 4 bits are offered for keys and "
                                 f"values of {attention4.GROUP} to {attention4.MAX_HEAD_DIM} numbers, a multiple of {attention4.GROUP}")
            dtype = torch.uint8
            shape = v_shape = (n_pages, need.n_kv_heads, ops.tile4_bytes(need.head_dim))
        else:
            shape = (n_pages, need.n_kv_heads, PAGE, need.head_dim)
            v_shape = (n_pages, need.n_kv_heads, PAGE, need.v_head_dim or need.head_dim)
        # zero-filled once: a page's unwritten rows are never selected by a mask, but they
        # are multiplied by zero weights, and 0 * NaN would not be 0
        self.k = [torch.zeros(shape, dtype=dtype, device=device) for _ in range(n_entries)]
        self.v = [None if need.keys_only else torch.zeros(v_shape, dtype=dtype, device=device) for _ in range(n_entries)]
        self.table_host = torch.zeros((n_slots, self.table_stride), dtype=torch.int32)
        self._table_np = self.table_host.numpy()       # the same memory: an entry is written without a tensor operation
        self.table_dev = torch.zeros((n_slots, self.table_stride), dtype=torch.int32, device=device)
        self._slot_pages: Dict[int, List[int]] = {}
        self._holders: Dict[int, int] = {}             # pages that several slots hold -> how many
        self.version = 0                               # moves on whenever a slot's pages change
        self.joins = 0                                 # and this whenever they change otherwise than by one more of its own
        self._dirty: set = set()
        self._views: Dict[int, ops.PagedKVArgs] = {}
        # what ops.copy_pages wants of the arrays (the keys', then the values'): address and bytes of a page
        arrays = self.k + [v for v in self.v if v is not None]
        page = [a[0].numel() * a.element_size() for a in arrays]
        self._most_bytes = max(page)
        self._arrays = torch.tensor([[a.data_ptr(), b] for a, b in zip(arrays, page)], dtype=torch.int64).to(device)

    def chunk_room(self):
        """The most tokens a sequence may bring in one step that attends over this group's
        storage (None: any number)."""
        if self.ring_pages == 0:
            return None
        return self.ring_pages * PAGE - self.need.window + 1

    def pages_for(self, length: int) -> int:
        n = (length + PAGE - 1) // PAGE
        return min(n, self.table_stride)

    def open_slot(self, slot: int) -> None:
        if slot in self._slot_pages:
            raise CacheError(f"slot {slot} is opened twice")
        self._slot_pages[slot] = []
        self.version += 1
        self.joins += 1

    def shared_before(self, slot: int, old_len: int, new_len: int) -> List[int]:
        """Table entries of the slot that positions old_len..new_len-1 are written to and whose pages others hold too."""
        if not self._holders or new_len <= old_len:
            return []
        held, first, last = self._slot_pages[slot], old_len // PAGE, (new_len - 1) // PAGE
        if self.ring_pages:
            entries = {p % self.ring_pages for p in range(max(first, last - self.ring_pages + 1), last + 1)}
        else:
            entries = range(first, last + 1)
        return [e for e in sorted(entries) if e < len(held) and held[e] in self._holders]

    def more_pages(self, slots: Sequence[int], old_lens: Sequence[int], new_lens: Sequence[int]) -> int:
        """Pages that `grow` takes for these slots, one after another: of a shared page the last holder needs no copy."""
        more, copied = 0, {}
        for slot, old, new in zip(slots, old_lens, new_lens):
            more += max(0, self.pages_for(new) - len(self._slot_pages[slot]))
            for e in self.shared_before(slot, old, new):
                page = self._slot_pages[slot][e]
                copied[page] = min(copied.get(page, 0) + 1, self._holders[page] - 1)
        return more + sum(copied.values())

    def grow(self, slot: int, new_len: int, old_len: Optional[int] = None) -> None:
        """Make sure the slot has pages for positions < new_len, and that no other slot holds those that positions from old_len on
        are written to."""
        held = self._slot_pages[slot]
        want = self.pages_for(new_len)
        if self.ring_pages == 0 and (new_len + PAGE - 1) // PAGE > self.table_stride:
            raise CacheError(f"a sequence of {new_len} tokens is longer than the cache's tables "
                             f"hold ({self.table_stride * PAGE})")
        row = self._table_np[slot]
        shared = self.shared_before(slot, new_len if old_len is None else old_len, new_len)
        if shared:
            olds = [held[e] for e in shared]
            news = [self.pages.take() for _ in shared]
            try:
                self._copy_listed(olds, news)
            except Exception:
                for page in news:
                    self.pages.give_back(page)
                raise
            for e, old, new in zip(shared, olds, news):
                row[e] = held[e] = new
                self._let_go(old)
            self._dirty.add(slot)
            self.version += 1
            self.joins += 1
        while len(held) < want:
            page = self.pages.take()
            self.version += 1
            row[len(held)] = page
            held.append(page)
            self._dirty.add(slot)

    def close_slot(self, slot: int) -> None:
        self.version += 1
        self.joins += 1
        for page in self._slot_pages.pop(slot):
            self._let_go(page)

    def _let_go(self, page: int) -> None:
        """One holder less; the last one gives the page back."""
        n = self._holders.pop(page, 1)
        if n == 1:
            self.pages.give_back(page)
        elif n > 2:
            self._holders[page] = n - 1

    def share(self, slot: int, new_slot: int, length: int) -> None:
        """The (open, empty) new slot holds the pages of the slot's first `length` positions too."""
        pages = self._slot_pages[slot][:self.pages_for(length)]
        for page in pages:
            self._holders[page] = self._holders.get(page, 1) + 1
        self._slot_pages[new_slot] = list(pages)
        self._table_np[new_slot, :len(pages)] = pages
        self._dirty.add(new_slot)
        self.version += 1
        self.joins += 1

    def shared_runs(self, slots: Sequence[int], lengths: Sequence[int]) -> List[tuple]:
        """Where sequences of these lengths share pages: [(places in `slots`, first logical page, the page behind the last)], each
        place in one run at most, the runs chosen so that the fewest pages are read when a run's are read once.  In a ring only what
        all of a run's sequences still hold counts.  A run stays true until one of the slots' pages changes (`version`)."""
        if not self._holders or len(slots) < 2:
            return []
        last = (np.asarray(lengths, dtype=np.int64) - 1) // PAGE
        out: List[tuple] = []
        for members in self._families(slots, last):
            lo, hi = 0, int(last[members].min()) + 1
            if self.ring_pages:
                lo = max(0, int(last[members].max()) - self.ring_pages + 1)             # what the longest has not written over
            if hi <= lo:
                continue
            entries = np.arange(lo, hi)
            if self.ring_pages:
                entries %= self.ring_pages
            table = self._table_np[np.asarray([slots[i] for i in members])][:, entries]
            out += [(m, lo, lo + n) for m, n in _best_runs(table, members)[1]]
        return out

    def _families(self, slots: Sequence[int], last: np.ndarray) -> List[List[int]]:
        """Places of sequences that may share pages.  Sequences that share one share all before it: its first page, or, in a ring, the
        first that all of them still hold.  Where there is none (lengths too unlike), those that hold a page in common, directly or by way
        of others, are a family."""
        at = max(0, int(last.max()) - self.ring_pages + 1) if self.ring_pages else 0
        if at <= int(last.min()):
            first = self._table_np[np.asarray(slots), at % self.ring_pages if self.ring_pages else 0].tolist()
            by_page: Dict[int, List[int]] = {}
            for i, page in enumerate(first):
                if page in self._holders:
                    by_page.setdefault(page, []).append(i)
            return [m for m in by_page.values() if len(m) > 1]
        kin = list(range(len(slots)))

        def root(i: int) -> int:
            while kin[i] != i:
                kin[i] = kin[kin[i]]
                i = kin[i]
            return i

        seen: Dict[int, int] = {}
        for i, s in enumerate(slots):
            for page in self._slot_pages[s]:
                if page in self._holders:
                    kin[root(i)] = root(seen.setdefault(page, i))
        families: Dict[int, List[int]] = {}
        for i in range(len(slots)):
            families.setdefault(root(i), []).append(i)
        return [m for m in families.values() if len(m) > 1]

    def compact(self) -> int:
        """Move the held pages to the front of the arrays; the number of them."""
        n = self.pages.n_held
        olds = sorted(p for p in self.pages.held() if p >= n)
        if olds:
            news = self.pages.lowest_free(len(olds))
            self._copy_listed(olds, news)
            self.pages.exchange(olds, news)
            self.version += 1
            self.joins += 1
            to = dict(zip(olds, news))
            self._holders = {to.get(p, p): k for p, k in self._holders.items()}
            for slot, held in self._slot_pages.items():
                if any(p in to for p in held):
                    held[:] = [to.get(p, p) for p in held]
                    self._table_np[slot, :len(held)] = held
                    self._dirty.add(slot)
        return n

    def new_arrays(self, n_pages: int) -> None:
        """Arrays of n_pages pages in the place of the old ones, one after another, with what the pages of both sizes hold; the held pages
        must be among those, and no other may be taken while this runs.  Each old array's memory goes back before the next is made.  If there is
        no room for one of them, the arrays made so far stay: each of them holds the pages that both sizes have."""
        for arrays, name, first in ((self.k, "k_pages", 0), (self.v, "v_pages", self.n_entries)):
            for i in range(self.n_entries):
                if arrays[i] is None:
                    continue
                new = torch.zeros((n_pages,) + tuple(arrays[i].shape[1:]), dtype=arrays[i].dtype, device=arrays[i].device)
                keep = min(n_pages, arrays[i].shape[0])
                new[:keep].copy_(arrays[i][:keep])
                arrays[i] = new
                self._arrays[first + i, 0].fill_(new.data_ptr())
                if i in self._views:
                    setattr(self._views[i], name, new)
                    self._views[i].four = None

    def copy_pages(self, src: torch.Tensor, dst: torch.Tensor) -> None:
        """Page src[i] to page dst[i] (int32, on the cache's device) in the arrays of all entries, in one launch; pairs with a page
        outside the arrays copy nothing.  No page may be written twice, or read and written, in one call."""
        ops.copy_pages(self._arrays, self._most_bytes, src, dst, self.pages.n)

    def _copy_listed(self, src: Sequence[int], dst: Sequence[int]) -> None:
        if self.table_dev.device.type != "cuda":            # the bookkeeping without a GPU
            for a in self.k + [v for v in self.v if v is not None]:
                a[list(dst)] = a[list(src)]
            return
        pairs = torch.tensor([list(src), list(dst)], dtype=torch.int32).pin_memory().to(self.table_dev.device, non_blocking=True)
        self.copy_pages(pairs[0], pairs[1])

    def flush(self) -> None:
        """Changed rows of the table go to the device: staged in pinned memory (the host may change the
        table again before the copy runs), one asynchronous copy per run of neighbouring rows, no kernel."""
        if not self._dirty:
            return
        rows = sorted(self._dirty)
        self._dirty.clear()
        on_gpu = self.table_dev.device.type == "cuda"
        staged = torch.empty((len(rows), self.table_stride), dtype=torch.int32, pin_memory=on_gpu)
        torch.index_select(self.table_host, 0, torch.tensor(rows, dtype=torch.long), out=staged)
        at = 0
        while at < len(rows):
            end = at + 1
            while end < len(rows) and rows[end] == rows[end - 1] + 1:
                end += 1
            self.table_dev[rows[at]:rows[at] + end - at].copy_(staged[at:end], non_blocking=on_gpu)
            at = end

    def view(self, entry: int) -> ops.PagedKVArgs:
        """What the kernels take of an entry: one object an entry, which always names the arrays that there are."""
        if entry not in self._views:
            self._views[entry] = ops.PagedKVArgs(self.k[entry], self.v[entry], self.table_dev, self.ring_pages,
                                                 self.need.n_kv_heads, self.need.head_dim, self.need.v_head_dim or 0, self.need.bits)
        return self._views[entry]

    def bytes_per_token(self) -> int:
        if self.need.bits is not None:
            return self.n_entries * 2 * self.need.n_kv_heads * ops.tile4_bytes(self.need.head_dim) // PAGE
        e = self.k[0].element_size()
        per_head = self.need.head_dim + (0 if self.need.keys_only else (self.need.v_head_dim or self.need.head_dim))
        return self.n_entries * self.need.n_kv_heads * per_head * e
