"""Keys and values held in 4 bits (a cache group whose need says `bits=4`): rows put into the pages, attention over them.

Per 64 neighbouring numbers of a head a scale s and a middle m in bfloat16 and codes -8..7; what is held is code * s + m
(csrc/attention4.cu has the rounding).  Head sizes 64, 128, 192 and 256; rows in bfloat16 or in 32 bits."""
from __future__ import annotations

from typing import Optional

import torch

from .. import ops
from ..errors import KernelError

GROUP = 64                     # numbers of a head that share a scale
MAX_HEAD_DIM = 256


def supports(head_dim: int) -> bool:
    return head_dim % GROUP == 0 and 0 < head_dim <= MAX_HEAD_DIM


def _check_cache(cache: ops.PagedKVArgs) -> None:
    if cache.bits != 4:
        raise KernelError("a cache in 4 bits is wanted (KVNeed(bits=4))")


def _check_step(n: int, step, what: str) -> None:
    if step.n_tokens != n:
        raise KernelError(f"{what}: {n} rows for a step of {step.n_tokens} tokens")


def store(rows: torch.Tensor, step, cache: ops.PagedKVArgs, held: Optional[torch.Tensor] = None) -> None:
    """Put the rows [N, 2 * n_kv_heads * head_dim] (keys, then values, rotated) into the pages at the step's places.  `held` (like
    rows, or rows itself) receives what the pages then hold, rounded to its type: prompts attend over that, so that they see
    the keys and values that later steps see.  Padding rows store nothing."""
    _check_cache(cache)
    ops._check_rows(rows, "rows of keys and values")
    n, width = rows.shape
    if width != 2 * cache.n_kv_heads * cache.head_dim:
        raise KernelError(f"rows of {width} numbers for {cache.n_kv_heads} kv heads of {cache.head_dim}")
    _check_step(n, step, "store")
    if held is not None:
        ops._check_rows(held, "what is held", rows.dtype)
        if held.shape != rows.shape:
            raise KernelError("what is held and the rows differ in size")
    ops.fourbit().call("hos_store4", rows.data_ptr(), ops.dtype_code(rows.dtype), rows.stride(0), held.data_ptr() if held is not None else None,
                       held.stride(0) if held is not None else 0, step.token_pos.data_ptr(), step.token_seq.data_ptr(), step.seq_slot.data_ptr(),
                       step.seq_len_after.data_ptr(), step.cu_seqlens.data_ptr(), step.row_offset, step.n_seqs, step.seq_offset, int(step.single_token),
                       ops.paged4(cache), n, ops._stream())


MAX_SHARES, CLUSTER_SHARES, MANY_SHARES = 1024, 8, 32


def shares(rows: int, kv_items: int, longest: int, window: Optional[int], fill: float = 1.0):
    """(pages of a share, shares of a row, whether the shares are a cluster): `rows` rows times `kv_items` (kv heads, times the eights of
    query heads that share one) over up to `longest` keys.  Two CTAs fit an SM: rows that leave CTAs free are cut into as many shares
    as fill them; many rows of unequal lengths (`fill`: the sum of the keys over rows * the longest) into shares of up to 32 pages,
    which CTAs take as they come free.  Up to 8 shares of few rows of like lengths merge as a cluster (of unlike lengths the CTAs
    without keys would wait for the others: 32 rows of up to 4,000 keys 19 us, through the workspace 15); more cost a second kernel,
    about the time of 4 pages, and have to save that.  Beyond 32 shares one CTA an SM is enough, as the sums that are merged cost more
    than the second brings (8 heads of 256 over 4, 8,192 keys: 64 shares 16.5 us, 32 shares 14.0; 32,000 keys: 63 shares 26.2, 32
    shares 24.8)."""
    span = min(longest, window) if window else longest
    pages = max(1, -(-span // ops.PAGE_TOKENS) + (1 if window and longest > window else 0))
    places, items = 2 * ops.sm_count(), max(1, rows * kv_items)
    few = items * fill < places
    if few:
        share = -(-pages // max(1, int(places // max(1.0, items * fill))))
        if -(-pages // share) > MANY_SHARES:
            share = -(-pages // max(MANY_SHARES, int(places // 2 // max(1.0, items * fill))))
    else:
        share = pages if fill > 0.9 and items % places == 0 else 32
    share = max(1, min(share, pages), -(-pages // MAX_SHARES))
    least = -(-pages // CLUSTER_SHARES)
    if few and share < least <= share + 4:
        share = least
    splits = -(-pages // share)
    return share, splits, few and fill > 0.8 and 1 < splits <= CLUSTER_SHARES


def attend(q: torch.Tensor, out: torch.Tensor, step, cache: ops.PagedKVArgs, n_heads: int, scale: float, softcap: float = 0.0,
           window: Optional[int] = None) -> None:
    """out[N, n_heads * head_dim] = softmax attention of the step's rows, each at its own position, over what the pages hold up to
    and with that position (the last `window` of it).  Padding rows become zeros."""
    _check_cache(cache)
    ops._check_rows(q, "queries")
    ops._check_rows(out, "attention output", q.dtype)
    n = q.shape[0]
    if q.shape[1] != n_heads * cache.head_dim or out.shape != q.shape:
        raise KernelError(f"queries {tuple(q.shape)} and output {tuple(out.shape)} for {n_heads} heads of {cache.head_dim}")
    _check_step(n, step, "attend")
    kv = cache.n_kv_heads
    items = kv * -(-(n_heads // kv) // 8)
    if _tiles_take(q, out, step, n_heads // kv):
        return _attend_tiles(q, out, step, cache, n_heads, scale, softcap, window)
    together = 1 if step.single_token else max(1, 8 // (n_heads // kv))      # rows of a sequence that share a walk
    key = ("shares of 4-bit pages", n, items, together, window, step.row_offset)
    plan = step.shared.get(key)                      # once per step and kind of layer
    if plan is None:
        walks = n if together == 1 else -(-n // together)
        plan = step.shared[key] = shares(walks, items, step.max_len_after, window, step.fill_for(window))
    share, splits, cluster = plan
    parts = None
    if splits > 1 and not cluster:
        parts = torch.empty(n * n_heads * splits * (cache.head_dim + 2), dtype=torch.float32, device=q.device)
    ops.fourbit().call("hos_attend4", q.data_ptr(), ops.dtype_code(q.dtype), q.stride(0), out.data_ptr(), out.stride(0), step.token_pos.data_ptr(),
                       step.token_seq.data_ptr(), step.seq_slot.data_ptr(), step.token_slot.data_ptr() if step.token_slot is not None else None,
                       step.cu_seqlens.data_ptr() if together > 1 else None, step.row_offset, step.n_seqs, ops.paged4(cache), n, n_heads,
                       scale, softcap, window or 0, share, splits, parts.data_ptr() if parts is not None else None, ops._stream())


TILE_ROWS = 128                # (row, head) pairs of a kv head that a block of the kernel for pieces takes
TILE_MIN_PAIRS = 48


def _tiles_take(q, out, step, per: int) -> bool:
    """Whether the rows go to the kernel for pieces: bfloat16 rows on 16 bytes, and sequences that bring enough (row, head) pairs."""
    return (not step.single_token and q.dtype == torch.bfloat16 and step.max_new * per >= TILE_MIN_PAIRS and per <= TILE_ROWS and q.stride(0) % 8 == 0
            and out.stride(0) % 8 == 0 and q.data_ptr() % 16 == 0 and out.data_ptr() % 16 == 0)


def _attend_tiles(q, out, step, cache: ops.PagedKVArgs, n_heads: int, scale: float, softcap: float, window: Optional[int]) -> None:
    n, kv = q.shape[0], cache.n_kv_heads
    size = TILE_ROWS // (n_heads // kv)
    key = ("tiles over 4-bit pages", n, size, kv, window, step.row_offset)
    plan = step.shared.get(key)                      # once per step and kind of layer
    if plan is None:
        plan = step.shared[key] = tile_shares(-(-n // size) if not step.cu_host else
                                              sum(-(-(b - a) // size) for a, b in zip(step.cu_host, step.cu_host[1:])), kv,
                                              step.max_len_after, step.max_new, window)
    share, splits = plan
    parts = None
    if splits > 1:
        parts = torch.empty(n * n_heads * splits * (cache.head_dim + 2), dtype=torch.float32, device=q.device)
    lib = ops.fourbit()
    lib.call("hos_attend4_tiles", q.data_ptr(), q.stride(0), out.data_ptr(), out.stride(0), step.token_pos.data_ptr(), step.seq_slot.data_ptr(),
             step.seq_offset, step.cu_seqlens.data_ptr(), step.row_offset, step.n_seqs, ops.paged4(cache), n, n_heads, scale, softcap, window or 0, share,
             splits, parts.data_ptr() if parts is not None else None, ops._stream())
    if splits > 1:
        lib.call("hos_attend4_merge", out.data_ptr(), ops.dtype_code(out.dtype), out.stride(0), cache.head_dim, n, n_heads, splits, parts.data_ptr(),
                 ops._stream())


def tile_shares(blocks: int, kv: int, longest: int, new: int, window: Optional[int]):
    """(pages of a share, shares) for `blocks` blocks of rows and kv heads of which an SM takes one at a time: as many shares as fill
    the SMs, each of at least 8 pages (a share costs about 2 besides, and its sums are written, read and merged)."""
    span = min(longest, window + new) if window else longest
    pages = max(1, -(-span // ops.PAGE_TOKENS) + (1 if window else 0))
    splits = max(1, min(pages // 8, ops.sm_count() // max(1, blocks * kv)))
    share = -(-pages // splits)
    return share, -(-pages // share)
