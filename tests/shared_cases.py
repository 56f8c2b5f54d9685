"""Sequences that were forked from one another, with the keys and values that each of them holds, for tests of attention over
shared pages."""
import math

import torch

from hos_b200 import ops
from hos_b200.cache import CacheManager
from hos_b200.engine.batch import build_step
from hos_b200.parts.base import KVNeed


class Tree:
    """A cache of one layer.  `new(n)` starts a sequence of n tokens, `fork(i)` another that goes on from sequence i, `go_on({i: n})`
    brings n more tokens to some.  `k[i]`, `v[i]`: what sequence i holds, float64 [length, kv, dim], rounded as the cache holds it."""

    def __init__(self, kv, dim, window=None, device="cuda", max_seq_len=2048, slots=64, chunk=64, seed=0, pages=None):
        self.kv, self.dim, self.window, self.dev = kv, dim, window, torch.device(device)
        self.cache = CacheManager([KVNeed(kv, dim, window)], [None], [[]], (pages or 16 * slots) * 64, max_seq_len,
                                  torch.bfloat16, self.dev, max_slots=slots, chunk_tokens=chunk)
        self.group, self.view = self.cache.groups[0], self.cache.stores[0].kv
        self.gen = torch.Generator().manual_seed(seed)
        self.slots, self.k, self.v = [], [], []

    def _rows(self, n):
        x = torch.randn(n, self.kv, self.dim, generator=self.gen)
        return (x * (1 + 3 * (torch.rand(self.dim, generator=self.gen) < 0.05))).to(torch.bfloat16)

    def bring(self, which, counts):
        starts = [len(self.k[i]) for i in which]
        slots = [self.slots[i] for i in which]
        self.cache.extend_all(slots, [s + n for s, n in zip(starts, counts)])
        self.cache.flush()
        k, v = [self._rows(n) for n in counts], [self._rows(n) for n in counts]
        for i, a, b in zip(which, k, v):
            self.k[i], self.v[i] = torch.cat([self.k[i], a.double()]), torch.cat([self.v[i], b.double()])
        if self.dev.type == "cuda":
            step = build_step([[0] * n for n in counts], starts, slots, self.dev, 1)
            rows = torch.cat([torch.cat(k).flatten(1), torch.cat(v).flatten(1)], dim=1).to(self.dev)
            ops.rope_kv_write(rows, 0, step.token_pos, step.token_seq, step.seq_slot, step.seq_len_after, None, 0, 0, self.view, self.kv, self.dim)

    def new(self, n):
        self.slots += self.cache.admit([0])
        self.k.append(torch.zeros(0, self.kv, self.dim, dtype=torch.float64))
        self.v.append(self.k[-1])
        self.bring([len(self.slots) - 1], [n])
        return len(self.slots) - 1

    def fork(self, i, n=1):
        new = self.cache.fork(self.slots[i], n)
        for s in new:
            self.slots.append(s)
            self.k.append(self.k[i])
            self.v.append(self.v[i])
        return list(range(len(self.slots) - n, len(self.slots)))

    def step(self, which, news):
        """The step of the last news[j] tokens of sequences which[j] (which hold them already)."""
        return build_step([[0] * n for n in news], [len(self.k[i]) - n for i, n in zip(which, news)], [self.slots[i] for i in which], self.dev, 1)

    def exact(self, q, which, news, heads, scale, cap, window):
        out, at = [], 0
        q = q.double().cpu().view(-1, heads, self.dim)
        for i, n in zip(which, news):
            k, v, length = self.k[i], self.v[i], len(self.k[i])
            per = heads // self.kv
            s = torch.einsum("nhd,khd->nhk", q[at:at + n], k.repeat_interleave(per, 1)) * scale
            if cap:
                s = cap * torch.tanh(s / cap)
            d = torch.arange(length - n, length)[:, None] - torch.arange(length)
            s.masked_fill_(((d < 0) | (d >= window) if window else d < 0)[:, None], -math.inf)
            out.append(torch.einsum("nhk,khd->nhd", s.softmax(-1), v.repeat_interleave(per, 1)).flatten(1))
            at += n
        return torch.cat(out)


def share_bound(v_abs, exact):
    """Bound on the difference of attention whose weights are rounded to bfloat16 and whose sums are 32-bit, rounded to bfloat16 at
    the end.  bfloat16 keeps 8 bits: a rounding is off by half a step, torch.finfo(torch.bfloat16).eps / 2 = 2^-8 of the number (1 + 2^-8 lies
    in the middle between 1 and its neighbour 1 + 2^-7).  A weight is off by 2^-8 of itself from its rounding and by e from its score's: a
    score of 256 products rounded at 32 bits, its soft-cap through an exponential, together under 2^-13 of what a score may be (8 here):
    e < 2^-10.  The rounding acts on the numerator alone (the sum of weights is of the unrounded), e on both, each on the weighted mean of
    |v| over the keys, which `v_abs` gives: (2^-8 + 2 * 2^-10) v_abs; the result's own rounding: 2^-8 of it, and sums of 32 bits 2^-15 of
    v_abs."""
    half_step = torch.finfo(torch.bfloat16).eps / 2
    return (half_step + 2 * 2.0 ** -10 + 2.0 ** -15) * v_abs + half_step * exact.abs()
