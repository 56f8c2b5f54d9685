"""Attention of sequences that share pages (a conversation and its forks): the pages that several of a step's sequences hold in
common are read once for all of their rows, the others sequence by sequence, and a row's parts are joined (csrc/attention_shared.cu).

`plan` finds what is shared, once a step and group of the cache; `attend` is attention over the group's pages in any of its layers.
bfloat16 keys and values; heads of a multiple of 16 numbers up to 256; any number of rows a sequence."""
from __future__ import annotations

import ctypes
from typing import Dict, Optional, Sequence

import numpy as np
import torch

from .. import ops
from ..errors import KernelError

MAX_HEAD_DIM = 256
OPEN = 1 << 30                 # a page behind every sequence's last
ITEM_INTS = 12
PAIRS, BLOCK = 16, 128         # (row, head) pairs of an item, of a big one
MOST_PARTS = 64 << 20          # bytes of the parts that wait for the merge

_libs: Dict[int, ops.Library] = {}


def supports(head_dim: int) -> bool:
    return head_dim % 16 == 0 and 16 <= head_dim <= MAX_HEAD_DIM


def lib_for(head_dim: int) -> ops.Library:
    lib = _libs.get(head_dim)
    if lib is None:
        lib = _libs[head_dim] = ops.Library(f"shared_hd{head_dim}")
    return lib


class SharedPlan:
    """What is shared by the sequences of a step in one group of the cache: `runs` (see KVGroup.shared_runs) and the rows of each
    sequence; made into lists of work for the kernels once per number of query heads."""

    def __init__(self, group, runs, rows: Sequence[range], slots: Sequence[int], lengths: Sequence[int], n_rows: int):
        self.group, self.version = group, group.version
        self.runs, self.rows, self.slots, self.lengths, self.n_rows = runs, rows, slots, lengths, n_rows
        self._work: Dict[int, "Work"] = {}

    def work(self, n_heads: int) -> "Work":
        w = self._work.get(n_heads)
        if w is None:
            need = self.group.need
            made = lists(self.runs, self.rows, self.slots, self.lengths, self.n_rows, n_heads // need.n_kv_heads, need.n_kv_heads,
                         need.head_dim, need.window, has_big(need.head_dim))
            w = self._work[n_heads] = Work(made, self.group, n_heads)
        return w


class Lists:
    """Items (of up to 16 pairs, then of up to 128), their rows, and each row's number of parts, on the host."""

    def __init__(self, items: np.ndarray, big: np.ndarray, rows: np.ndarray, n_parts: np.ndarray):
        self.items, self.big, self.rows, self.n_parts = items, big, rows, n_parts
        self.parts = int(n_parts.max()) if n_parts.size else 0


class SharedWork(ctypes.Structure):
    """A list of work as csrc/attention_shared.cu takes it."""
    _fields_ = [(name, ctypes.c_void_p) for name in ("counts", "n_parts", "items", "big_items", "rows", "page_table")] + \
               [(name, ctypes.c_int) for name in ("most", "big_most", "parts", "table_stride", "ring_pages", "n_heads", "n_kv_heads", "window")]


class Work:
    """The lists on the device, in one array: the numbers of items, the rows' parts, the items, their rows."""

    def __init__(self, made: Lists, group, n_heads: int):
        table, need = group.table_dev, group.need
        n = len(made.n_parts)
        at = -(-(4 + n) // 4) * 4
        flat = np.concatenate([np.asarray([len(made.items), len(made.big), 0, 0], dtype=np.int32), made.n_parts, np.zeros(at - 4 - n, dtype=np.int32),
                               made.items.reshape(-1), made.big.reshape(-1), made.rows])
        host = torch.from_numpy(flat)
        if table.device.type == "cuda":
            host = host.pin_memory()
        self.array = host.to(table.device, non_blocking=True)
        self._host = host                                   # the copy reads it
        base = self.array.data_ptr()
        items, big = base + 4 * at, base + 4 * (at + made.items.size)
        self.parts = made.parts
        self.fields = SharedWork(base, base + 16, items, big, big + 4 * made.big.size, table.data_ptr(), len(made.items), len(made.big), made.parts,
                                 table.shape[1], group.ring_pages, n_heads, need.n_kv_heads, need.window or 0)
        self.address = ctypes.addressof(self.fields)
        self.floats = n * n_heads * made.parts * (need.head_dim + 2)


def has_big(head_dim: int) -> bool:
    """Whether blocks of up to 128 pairs have a kernel (tcgen05)."""
    return head_dim in (64, 128, 256)


def _pages(length: int, new: int, window: Optional[int]) -> tuple:
    """(first, behind the last) logical page that the last `new` rows of a sequence see."""
    lowest = max(0, length - new + 1 - window) if window else 0
    return lowest // ops.PAGE_TOKENS, (length - 1) // ops.PAGE_TOKENS + 1


def share_pages(pages: Sequence[int], per_item: int) -> int:
    """Pages of a share at most, for items of so many pages that each run `per_item` times: as many shares as fill the SMs once."""
    total = sum(pages) * per_item
    return max(2, -(-total // ops.sm_count()))


def lists(runs, rows: Sequence[range], slots: Sequence[int], lengths: Sequence[int], n_rows: int, per: int, kv: int, head_dim: int,
          window: Optional[int], big: bool) -> Lists:
    """The work: a run's rows in blocks of up to 16 pairs, or of up to 128 where they are more and a kernel has such blocks (`big`), over
    the run's pages, each sequence's over the rest of its own."""
    big = big and per <= BLOCK
    chunks = -(-per // PAIRS)
    skip = [(0, 0)] * len(slots)
    blocks = []                                              # (big, rows, slot, lp0, lp1, skip0, skip1, pages)

    def cut(of: Sequence[int], *rest) -> None:
        large = big and len(of) * per > PAIRS
        size = max(1, (BLOCK if large else PAIRS) // per)
        n = -(-len(of) // size)                              # blocks of like sizes
        for i in range(n):
            blocks.append((large, of[len(of) * i // n:len(of) * (i + 1) // n], *rest))

    for members, lo, hi in runs:
        seen = [_pages(lengths[i], len(rows[i]), window) for i in members]
        n = min(hi, max(b for _, b in seen)) - max(lo, min(a for a, _ in seen))
        if n <= 0:
            continue
        for i in members:
            skip[i] = (lo, hi)
        cut([r for i in members for r in rows[i]], slots[members[0]], lo, hi, OPEN, OPEN, n)
    for i, slot in enumerate(slots):
        a, b = _pages(lengths[i], len(rows[i]), window)
        lo, hi = skip[i]
        cut(rows[i], slot, 0, OPEN, lo, hi, max(1, b - a - max(0, min(b, hi) - max(a, lo))))
    share = share_pages([b[7] for b in blocks], kv * chunks)
    most = max(2, MOST_PARTS // max(1, 4 * n_rows * per * kv * (head_dim + 2)))
    n_parts = np.zeros(n_rows, dtype=np.int32)
    made, listed = ([], []), []
    for large, of_block, slot, lp0, lp1, skip0, skip1, n in blocks:
        splits = max(1, min(-(-n // share), most // 2))
        part = int(n_parts[of_block[0]])
        for s in range(splits):
            made[large].append((len(listed), len(of_block), slot, lp0, lp1, skip0, skip1, s, splits, part + s, -(-n // splits), 0))
        listed.extend(of_block)
        for r in of_block:
            n_parts[r] += splits
    items = [np.asarray(sorted(m, key=lambda it: -it[10]), dtype=np.int32).reshape(-1, ITEM_INTS) for m in made]      # the longest first
    return Lists(items[0], items[1], np.asarray(listed, dtype=np.int32), n_parts)


def plan(group, step) -> SharedPlan:
    """What the sequences of the step share in this group of the cache (which must have the pages of the step's tokens already: after
    CacheManager.extend_all and flush).  It holds for every layer of the group in this step, and for later ones while no page of
    the sequences changes and their rows lie alike."""
    if group.need.bits is not None or group.need.keys_only or (group.need.v_head_dim or group.need.head_dim) != group.need.head_dim:
        raise KernelError("attention over shared pages takes keys and values of one size, in the model's type")
    if not supports(group.need.head_dim):
        raise KernelError(f"attention over shared pages takes heads of a multiple of 16 numbers up to {MAX_HEAD_DIM}, found {group.need.head_dim}")
    if len(step.cu_host) != step.n_seqs + 1 or len(step.slots_host) != step.n_seqs or len(step.starts_host) != step.n_seqs:
        raise KernelError("attention over shared pages is planned from the step's lists on the host")
    cu, slots = step.cu_host, list(step.slots_host)
    rows = [range(cu[i], cu[i + 1]) for i in range(step.n_seqs)]
    lengths = [s + len(r) for s, r in zip(step.starts_host, rows)]
    for s, n in zip(slots, lengths):
        if s not in group._slot_pages or group.pages_for(n) > len(group._slot_pages[s]):
            raise KernelError(f"slot {s} has no pages for {n} tokens")
    return SharedPlan(group, group.shared_runs(slots, lengths), rows, slots, lengths, step.n_tokens)


def attend(q: torch.Tensor, out: torch.Tensor, step, cache: ops.PagedKVArgs, plan: SharedPlan, n_heads: int, scale: float,
           softcap: float = 0.0, window: Optional[int] = None) -> None:
    """out[N, n_heads * head_dim] = softmax attention of the step's rows, each at its own position, over what the cache's pages hold up
    to and with that position (the last `window` of it).  Padding rows become zeros."""
    ops._check_here(q, "queries")
    ops._check_rows(q, "queries", torch.bfloat16)
    ops._check_rows(out, "attention output", torch.bfloat16)
    n, kv, dim = q.shape[0], cache.n_kv_heads, cache.head_dim
    if cache.k_pages.dtype != torch.bfloat16:
        raise KernelError("attention over shared pages takes a cache in bfloat16")
    if n_heads <= 0 or n_heads % kv:
        raise KernelError(f"attend: {n_heads} query heads over {kv} kv heads")
    if not scale > 0.0:
        raise KernelError(f"attend: a scale of {scale}")
    if q.shape[1] != n_heads * dim or out.shape != q.shape:
        raise KernelError(f"queries {tuple(q.shape)} and output {tuple(out.shape)} for {n_heads} heads of {dim}")
    if step.n_tokens != n or plan.n_rows != n:
        raise KernelError(f"attend: {n} rows for a step of {step.n_tokens} tokens and a plan of {plan.n_rows}")
    group = plan.group
    if cache.page_table is not group.table_dev or window != group.need.window:
        raise KernelError("attend: the plan is of another group of the cache")
    if plan.version != group.version:
        raise KernelError("attend: pages have changed since the plan was made")
    if n == 0:
        return
    work = plan.work(n_heads)
    ws = torch.empty(work.floats, dtype=torch.float32, device=q.device)
    lib_for(dim).call("hos_attn_shared", q.data_ptr(), q.stride(0), out.data_ptr(), out.stride(0), n, step.token_pos.data_ptr(), cache.k_pages.data_ptr(),
                      cache.v_pages.data_ptr(), cache.k_pages.shape[0], work.address, scale, softcap, ws.data_ptr(), ops._stream())
