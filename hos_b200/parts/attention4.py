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
    if not step.token_pos.is_cuda:               # a step's arrays are made together
        raise KernelError(f"{what}: the step must be on the GPU")


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


def _pages(longest: int, window: Optional[int], new: int = 0) -> int:
    """Pages that a walk for `new` more rows than one sees at most."""
    span = min(longest, window + new) if window else longest
    return max(1, -(-span // ops.PAGE_TOKENS) + (1 if window and longest > window else 0))


def shares(rows: int, kv_items: int, longest: int, window: Optional[int], fill: float = 1.0):
    """(pages of a share, shares of a row, whether the shares are a cluster): `rows` rows times `kv_items` (kv heads, times the eights of
    query heads that share one) over up to `longest` keys.  Two CTAs fit an SM: rows that leave CTAs free are cut into as many shares
    as fill them, of 2 pages at least (8 rows, 8 heads of 256 over 4, 500 keys: 8 shares of a page 10.6 us, 4 of two 9.0); many rows of
    unequal lengths (`fill`: the sum of the keys over rows * the longest) into shares of up to 32 pages, which CTAs take as they come free.  2, 4 or 8 shares of few rows of like lengths merge as a cluster (16 rows, 8 heads of 256 over 4,
    2,000 keys, 4 shares: 20.0 us, through the workspace 22.5), not 3 or 6, whose clusters leave places of their neighbourhood of SMs
    empty and run in two rounds (12 rows, 6 shares 28.9 us, through the workspace 20.4), nor, for the same reason, 4 or 8 in more than
    256 CTAs (36 rows, 16 heads of 64 over 2, 4 shares 35.4 and 25.0), nor of unlike lengths, where CTAs without keys would wait for the
    others (32 rows of up to 4,000 keys 19 us, 15).  More cost a second kernel, about the time of 4 pages, and have to save that.
    Beyond 32 shares one CTA an SM is enough, as the sums that are merged cost more than the second brings (8 heads of 256 over 4,
    8,192 keys: 64 shares 16.5 us, 32 shares 14.0; 32,000 keys: 63 shares 26.2, 32 shares 24.8)."""
    pages = _pages(longest, window)
    places, items = 2 * ops.sm_count(), max(1, rows * kv_items)
    few = items * fill < places
    if few:
        share = max(2, -(-pages // max(1, int(places // max(1.0, items * fill)))))
        if -(-pages // share) > MANY_SHARES:
            share = -(-pages // max(MANY_SHARES, int(places // 2 // max(1.0, items * fill))))
    else:
        share = pages if fill > 0.9 and items % places == 0 else 32
    share = max(1, min(share, pages), -(-pages // MAX_SHARES))
    least = -(-pages // CLUSTER_SHARES)
    if few and share < least <= share + 4:
        share = least
    splits = -(-pages // share)
    return share, splits, few and fill > 0.8 and (splits == 2 or splits in (4, 8) and items * splits <= 256)


MOST_PARTS = 64 << 20          # bytes of the shares' sums that wait for the merge


def bounded_shares(n: int, rows: int, kv_items: int, n_heads: int, head_dim: int, longest: int, window: Optional[int], fill: float = 1.0):
    """As `shares`, for n rows in `rows` walks, but shares that merge through the workspace are no more than MOST_PARTS holds (one, if not two):
    rows in such numbers fill the GPU without (2,048 rows of 32 heads of 128 on 131,072 keys would be 64 shares and 2 GB)."""
    share, splits, cluster = shares(rows, kv_items, longest, window, fill)
    most = max(1, MOST_PARTS // (4 * n * n_heads * (head_dim + 2)))
    if splits > most and not cluster:
        pages = _pages(longest, window)
        share = -(-pages // most)
        splits = -(-pages // share)
    return share, splits, cluster


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
    if n_heads <= 0 or n_heads % kv:
        raise KernelError(f"attend: {n_heads} query heads over {kv} kv heads")
    items = kv * -(-(n_heads // kv) // 8)
    if _tiles_take(q, out, step, n_heads // kv):
        plan = _tile_plan(n, step, cache, n_heads // kv, items, window)
        if plan is not None:
            return _attend_tiles(q, out, step, cache, n_heads, scale, softcap, window, plan)
    together = 1 if step.single_token else max(1, 8 // (n_heads // kv))      # rows of a sequence that share a walk
    key = ("shares of 4-bit pages", n, items, together, n_heads, cache.head_dim, window, step.row_offset)
    plan = step.shared.get(key)                      # once per step and kind of layer
    if plan is None:
        walks = n if together == 1 else -(-n // together)
        plan = step.shared[key] = bounded_shares(n, walks, items, n_heads, cache.head_dim, step.max_len_after, window, step.fill_for(window))
    share, splits, cluster = plan
    parts = None
    if splits > 1 and not cluster:
        parts = torch.empty(n * n_heads * splits * (cache.head_dim + 2), dtype=torch.float32, device=q.device)
    ops.fourbit().call("hos_attend4", q.data_ptr(), ops.dtype_code(q.dtype), q.stride(0), out.data_ptr(), out.stride(0), step.token_pos.data_ptr(),
                       step.token_seq.data_ptr(), step.seq_slot.data_ptr(), step.token_slot.data_ptr() if step.token_slot is not None else None,
                       step.cu_seqlens.data_ptr() if together > 1 else None, step.row_offset, step.n_seqs, ops.paged4(cache), n, n_heads,
                       scale, softcap, window or 0, share, splits, parts.data_ptr() if parts is not None else None, ops._stream())


TILE_ROWS = 128                # (row, head) pairs of a kv head that a block of the kernel for pieces takes
TILE_LEAST = 2                 # pages of a share at least


def _tiles_take(q, out, step, per: int) -> bool:
    """Whether the kernel for pieces could take the rows: bfloat16 rows on 16 bytes of sequences that go on by several tokens."""
    return (not step.single_token and q.dtype == torch.bfloat16 and per <= TILE_ROWS and q.stride(0) % 8 == 0 and out.stride(0) % 8 == 0
            and q.data_ptr() % 16 == 0 and out.data_ptr() % 16 == 0)


def _tile_plan(n: int, step, cache: ops.PagedKVArgs, per: int, items: int, window: Optional[int]):
    """(pages of a share, shares) of the kernel for pieces, or None where the kernel of few rows is the faster by both's estimates."""
    size, kv = TILE_ROWS // per, cache.n_kv_heads
    key = ("tiles over 4-bit pages", n, size, kv, cache.head_dim, window, step.row_offset)
    if key not in step.shared:                       # once per step and kind of layer
        blocks = -(-n // size) if not step.cu_host else sum(-(-(b - a) // size) for a, b in zip(step.cu_host, step.cu_host[1:]))
        blocks = max(1, blocks)
        plan = tile_shares(blocks, kv, step.max_len_after, step.max_new, window, cache.head_dim)
        walks = -(-n // max(1, 8 // per))
        take = tiles_are_faster(blocks * kv, plan, n / (blocks * size), walks * items * _pages(step.max_len_after, window),
                                step.fill_for(window), cache.head_dim)
        step.shared[key] = plan if take else None
    return step.shared[key]


def tiles_are_faster(blocks: int, plan, filled: float, row_pages: float, fill: float, dim: int) -> bool:
    """Microseconds of both kernels, fitted to batches of pieces (B200; heads of 64, 128 and 256, 16 to 1,000 rows on up to 16,000 keys):
    an SM's page with 128 pairs, or with some of a block's eight warps at work (`filled`), no less than 0.6 of it; and a page for eight
    pairs in one of two CTAs an SM.  Of 114 batches 107 run within 4% of the faster kernel's time, the worst 1.23 times it.  8 heads of 256
    over 4, tiles / few rows: 739 on 7,453 312 us / 412, 400 on 2,600 93 / 125, 128 on 872 38 / 27, 16 on 7,984 36 / 26."""
    share, splits = plan
    two = dim == 64 and blocks * splits > ops.sm_count()      # on an SM, which slows each
    tiles = (1.6 if two else 1.0) * max(1.0, blocks * splits * fill / ((2 if two else 1) * ops.sm_count())) * share * max(0.6, min(1.0, filled)) * (0.65 + 0.03 * dim) + 10 + dim / 25
    rows = row_pages * fill / (2 * ops.sm_count()) * (0.2 + 0.0055 * dim) + 7 + dim / 50
    return tiles < rows


def _attend_tiles(q, out, step, cache: ops.PagedKVArgs, n_heads: int, scale: float, softcap: float, window: Optional[int], plan) -> None:
    n = q.shape[0]
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


def tile_shares(blocks: int, kv: int, longest: int, new: int, window: Optional[int], head_dim: int = 128):
    """(pages of a share, shares) for `blocks` blocks of rows and kv heads of which an SM takes one at a time (of heads of 64 two: 400 rows
    on 7,600 keys, 16 heads over 2, shares for one 180 us, for two 110; of 128 two gain 3% at most and few rows lose): as many shares as fill
    the SMs, each of at least 2 pages (48 rows on 952 keys, 8 heads of 256 over 4: 30 us, of 4 pages 40, of 8 62)."""
    pages = _pages(longest, window, new)
    splits = max(1, min(pages // TILE_LEAST, (2 if head_dim == 64 else 1) * ops.sm_count() // max(1, blocks * kv)))
    share = -(-pages // splits)
    return share, -(-pages // share)
