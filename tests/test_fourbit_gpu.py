"""Products with 4-bit weights, keys and values in 4-bit pages, attention over them, copied pages: each against the formula in
64 bits, at the sizes, masks and strides where it can go wrong, and its refusals.

Tolerances, from the roundings there are.  A result in bfloat16 is within 2^-8 of itself; sums in 32 bits of products that are
exact or rounded to 32 bits are within 2^-18 (2^-20 for rows in 32 bits, whose result is not rounded further) of the sum of the
products' magnitudes; weights that are formed in bfloat16 first (many rows) are within 2^-9 of themselves.  In attention a weight
times a value's scale is rounded to bfloat16 before the product (2^-9 of itself), and a score's error, 2^-21 of the sum of the
magnitudes of its products and as much of the score, multiplies its weight."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, F32 = torch.bfloat16, torch.float32


def gen(seed):
    return torch.Generator().manual_seed(seed)


# ---- products --------------------------------------------------------------------------------------------------------
def made_weights(rows, k, group, zeros, seed):
    g = gen(seed)
    codes = torch.randint(0, 16, (rows, k), generator=g, dtype=torch.uint8)
    groups = -(-k // group)
    scales = (torch.rand(rows, groups, generator=g) + 0.1).mul(0.02).to(BF)
    z = torch.randint(0, 16, (rows, groups), generator=g, dtype=torch.uint8) if zeros else None
    at = torch.arange(k) // group
    w = (codes.double() - (z.double()[:, at] if zeros else 8.0)) * scales.double()[:, at]
    return codes.to(DEV), scales.to(DEV), z.to(DEV) if zeros else None, w.to(DEV)


def gelu(x):
    return torch.nn.functional.gelu(x, approximate="tanh")


def check_product(m, n, k, group, zeros, gated, dtype, out_dtype=None, act=0, limit=0.0, pad=0, seed=1):
    from hos_b200 import ops
    from hos_b200.parts import linear
    from hos_b200.parts.weights4 import Weight4
    blocks = 2 if gated else 1
    codes, scales, z, w = made_weights(blocks * n, k, group, zeros, seed)
    w4 = Weight4.from_codes(codes, scales, z, group, blocks=blocks)
    x = torch.randn(m, k + pad, generator=gen(seed + 1)).to(dtype).to(DEV)[:, :k]
    kw = dict(epilogue=ops.EPI_GATED, act=act, cap=limit) if gated else {}
    got = linear.matmul(x, w4, out_dtype, **kw)
    assert got.shape == (m, n) and got.dtype == (out_dtype or dtype)
    xd = x.double()
    y, size = xd @ w.T, xd.abs() @ w.abs().T
    eps = 2.0 ** -20 if dtype == F32 else 2.0 ** -18 + (2.0 ** -9 if m > 32 else 0.0)
    err = size * eps
    if gated:
        g, u, eg, eu = y[:, :n], y[:, n:], err[:, :n], err[:, n:]
        if act == 2:
            lim = limit or math.inf
            g, u = g.clamp(max=lim), u.clamp(-lim, lim)
            a, u = g * torch.sigmoid(1.702 * g), u + 1
        else:
            a = gelu(g) if act == 0 else torch.nn.functional.silu(g)
        y, err = a * u, 1.2 * eg * u.abs() + a.abs() * eu + 1.2 * eg * eu + 2.0 ** -19 * (a * u).abs()
    if got.dtype == BF:
        err = err + 2.0 ** -8 * y.abs()
    worst = ((got.double() - y).abs() - err).max()
    assert float(worst) <= 1e-30, f"off by {float((got.double() - y).abs().max()):.3g} where {float(err.max()):.3g} is allowed"


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("group", [32, 64, 128, 192])
@pytest.mark.parametrize("m,n,k", [(1, 1, 1), (1, 16, 64), (3, 17, 65), (8, 48, 448), (9, 33, 1000), (17, 130, 777), (32, 16, 2304), (33, 40, 320)])
def test_products(m, n, k, group, zeros, dtype):
    check_product(m, n, k, group, zeros, False, dtype)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("m,n,k,group,zeros,act,limit", [(1, 1, 3, 32, True, 0, 0.0), (5, 24, 130, 64, False, 1, 0.0), (8, 100, 512, 128, True, 0, 0.0),
                                                          (12, 33, 257, 32, False, 2, 1.5), (20, 16, 64, 64, True, 2, 0.0), (70, 50, 96, 32, True, 1, 0.0)])
def test_gated_products(m, n, k, group, zeros, act, limit, dtype):
    check_product(m, n, k, group, zeros, True, dtype, act=act, limit=limit)


@pytest.mark.parametrize("m,n,k,dtype,out_dtype", [(1, 2304, 9216, BF, F32), (4, 2304, 9216, F32, F32), (16, 4096, 2304, BF, BF), (31, 515, 4608, BF, BF),
                                                   (200, 515, 1984, BF, BF), (513, 640, 1160, BF, BF), (300, 128, 640, BF, F32), (150, 257, 333, F32, F32)])
def test_products_of_real_widths_and_many_rows(m, n, k, dtype, out_dtype):
    check_product(m, n, k, 64, False, False, dtype, out_dtype)


@pytest.mark.parametrize("m", [1, 7, 40])
@pytest.mark.parametrize("pad", [1, 3, 8])
def test_rows_further_apart_than_they_are_long(m, pad):
    check_product(m, 20, 136, 64, True, False, BF, pad=pad)
    check_product(m, 20, 136, 64, True, False, F32, pad=pad)


def test_a_product_into_rows_of_a_wider_matrix_leaves_the_rest_alone():
    from hos_b200.parts.weights4 import Weight4
    codes, scales, z, w = made_weights(20, 96, 32, True, 3)
    w4 = Weight4.from_codes(codes, scales, z, 32)
    for m in (2, 50):
        x = torch.randn(m, 96, device=DEV).to(BF)
        wide = torch.full((m, 31), 7.0, device=DEV, dtype=BF)
        w4.product(x, out=wide[:, 5:25])
        assert float((wide[:, :5] - 7).abs().max()) == 0 and float((wide[:, 25:] - 7).abs().max()) == 0
        assert torch.equal(wide[:, 5:25], w4.product(x))


def test_a_row_of_a_product_hangs_on_no_other_row_and_repeats():
    from hos_b200.parts.weights4 import Weight4
    codes, scales, z, _ = made_weights(300, 1000, 64, False, 4)
    w4 = Weight4.from_codes(codes, scales, None, 64)
    x = torch.randn(30, 1000, device=DEV).to(BF)
    a = w4.product(x)
    assert torch.equal(a, w4.product(x))
    x2 = x.clone()
    x2[1:] = math.nan
    assert torch.equal(w4.product(x2)[0], a[0])


def test_rounding_a_matrix_to_four_bits():
    from hos_b200.parts.weights4 import Weight4
    w = torch.randn(40, 200, device=DEV)
    w[3, :64] = 0.0                                              # a group of zeros
    eye = torch.eye(200, device=DEV)
    for zeros in (False, True):
        back = Weight4.from_matrix(w, 64, zeros).product(eye).T           # the matrix that the codes stand for
        g = torch.nn.functional.pad(w, (0, 56)).view(40, 4, 64)
        step = (g.amax(-1).clamp(min=0) - g.amin(-1).clamp(max=0)) / 15 if zeros else g.abs().amax(-1) / 7
        bound = (step * (1.0 + 15 * 2.0 ** -8)).repeat_interleave(64, 1)[:, :200]        # half a step, the zero code's half, the scale's rounding
        assert bool(((back - w).abs() <= bound + 1e-12).all())
        assert float(back[3, :64].abs().max()) == 0


def test_first_rows_of_a_matrix():
    from hos_b200.parts.weights4 import Weight4
    codes, scales, z, w = made_weights(48, 130, 32, True, 6)
    w4 = Weight4.from_codes(codes, scales, z, 32)
    x = torch.randn(3, 130, device=DEV)
    assert torch.equal(w4.first_rows(32).product(x), w4.product(x)[:, :32])
    assert w4.first_rows(20) is None


def test_products_refuse_what_does_not_fit():
    from hos_b200 import ops
    from hos_b200.errors import KernelError, SpecError
    from hos_b200.parts import linear
    from hos_b200.parts.weights4 import Weight4
    codes, scales, z, _ = made_weights(32, 128, 64, True, 7)
    for bad in (dict(group=48), dict(group=0), dict(group=-64), dict(group=128), dict(blocks=3), dict(codes=codes.float()), dict(codes=codes + 16),
                dict(zeros=z + 16), dict(zeros=z.float()), dict(scales=scales[:, :1]), dict(codes=codes[:0], scales=scales[:0], zeros=None)):
        with pytest.raises(SpecError):
            Weight4.from_codes(**{**dict(codes=codes, scales=scales, zeros=z, group=64), **bad})
    with pytest.raises(SpecError, match="NaN"):
        Weight4.from_matrix(torch.full((4, 64), math.nan, device=DEV))
    w4 = Weight4.from_codes(codes, scales, z, 64)
    x = torch.randn(2, 128, device=DEV)
    for call in (lambda: linear.matmul(x[:, :64], w4), lambda: linear.matmul(x.half(), w4), lambda: linear.matmul(x, w4, epilogue=ops.EPI_GATED),
                 lambda: linear.matmul(x, w4, epilogue=ops.EPI_SOFTCAP, cap=3.0), lambda: linear.matmul(x.cpu(), w4), lambda: linear.matmul(x.t(), w4),
                 lambda: linear.matmul(x, w4, out_dtype=BF), lambda: linear.matmul(x, w4, out=torch.empty(2, 31, device=DEV)),
                 lambda: linear.matmul(x, w4, bias=torch.zeros(32, device=DEV)), lambda: linear.matmul(torch.randn(4, 64, device=DEV)[:, ::2], w4)):
        with pytest.raises(KernelError):
            call()
    assert linear.matmul(x[:0], w4).shape == (0, 32)


# ---- rows into pages -------------------------------------------------------------------------------------------------
def quantised(x):
    """(codes, scales, middles) of [..., 64 j] in 32 bits: the definition, on the CPU."""
    g = x.detach().cpu().float().unflatten(-1, (-1, 64))
    lo, hi = g.amin(-1), g.amax(-1)
    s = ((hi - lo) / torch.tensor(15.0)).to(BF).float()
    s = torch.where(s < 2.0 ** -126, 0.0, s)
    m = (lo + 8 * s).to(BF).float()
    odd = ~(torch.isfinite(g).all(-1) & torch.isfinite(s) & torch.isfinite(m))
    c = torch.round((g - m[..., None]) / torch.where(s > 0, s, 1.0)[..., None]).nan_to_num(0.0, 0.0, 0.0).clamp(-8, 7)
    c = torch.where((odd | (s == 0))[..., None], 0.0, c)
    s, m = torch.where(odd, math.nan, s), torch.where(odd, math.nan, m)
    return c, s, m


def held_of(x):
    c, s, m = quantised(x)
    return (c * s[..., None] + m[..., None]).flatten(-2)


def unpacked(tile, dim, values):
    """What a page's tile [36 * dim] uint8 stands for: float32 [64, dim], from the layout's description."""
    t = tile.cpu()
    groups = dim // 64
    out = torch.empty(64, dim)
    codes, sm = t[:32 * dim].view(4, groups, 32, 16), t[32 * dim:].view(64, groups, 4).contiguous().view(BF).view(64, groups, 2).float()
    for row in range(64):
        for d in range(dim):
            r, e = row % 16, d % 64
            if values:
                byte = int(codes[row // 16, d // 64, (e % 8) * 4 + (r % 8) // 2, (e // 16) * 4 + (r % 2) * 2 + r // 8])
                code = byte >> (4 if (e // 8) % 2 else 0) & 15
            else:
                word = codes[row // 16, d // 64, (r % 8) * 4 + e // 16, ((r // 8) * 2 + (e // 8) % 2) * 4:][:4]
                j = e % 8
                nibble = j // 2 + 4 * (j % 2)
                code = int(word[nibble // 2]) >> (4 * (nibble % 2)) & 15
            out[row, d] = (code - 8) * sm[row, d // 64, 0] + sm[row, d // 64, 1]
    return out


class Paged:
    """Sequences in a 4-bit cache whose pages lie in no order; what is not written is NaN's bytes."""

    def __init__(self, lens, kv, dim, window=None, dtype=BF, seed=1, chunk=1, room=0):
        from hos_b200.cache import CacheManager
        from hos_b200.parts.base import KVNeed
        total = sum(-(-n // 64) * 64 for n in lens) + room + 64
        self.c = CacheManager([KVNeed(kv, dim, window, bits=4)], [None], [[]], total, max(total, 64), dtype, torch.device(DEV), max_slots=len(lens) + 3,
                              chunk_tokens=chunk)
        g = self.c.groups[0]
        g.k[0].fill_(255)
        g.v[0].fill_(255)
        self.slots = self.c.admit([0] * len(lens))[::-1]
        order = torch.randperm(len(lens), generator=gen(seed)).tolist()
        step = 64
        while step < max(lens) + 64:                              # pages are handed out in turn, not sequence by sequence
            for i in order:
                if min(lens[i], step) > self.c.lengths[self.slots[i]]:
                    self.c.extend(self.slots[i], min(lens[i], step))
            step += 64
        self.c.flush()
        self.lens, self.kv, self.dim, self.dtype = lens, kv, dim, dtype
        self.view = self.c.stores[0].kv

    def step(self, news, starts=None, pad=0):
        from hos_b200.engine.batch import build_step
        starts = [n - k for n, k in zip(self.lens, news)] if starts is None else starts
        return build_step([[0] * n for n in news], starts, self.slots, torch.device(DEV), 1, pad_to=pad)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("dim,kv", [(64, 1), (64, 3), (128, 2), (192, 1), (256, 2)])
def test_stored_rows_are_the_definitions_bit_for_bit(dim, kv, dtype):
    from hos_b200.parts import attention4
    p = Paged([70, 1, 130], kv, dim, dtype=dtype)
    n = 201
    rows = (torch.randn(n + 5, 2 * kv * dim, generator=gen(2)) * torch.rand(n + 5, 1, generator=gen(3)) * 10).to(dtype).to(DEV)
    held = torch.empty_like(rows)
    step = p.step([70, 1, 130], pad=n + 5)
    attention4.store(rows, step, p.view, held=held)
    want = held_of(rows)
    assert torch.equal(held.cpu().float(), want.to(dtype).float())
    g, base = p.c.groups[0], 0
    for slot, length in zip(p.slots, p.lens):
        for page in range(-(-length // 64)):
            at = int(g.table_host[slot, page])
            there = min(64, length - 64 * page)
            for head in range(kv):
                for arr, off, val in ((g.k[0], 0, False), (g.v[0], kv * dim, True)):
                    got = unpacked(arr[at, head], dim, val)[:there]
                    lo = base + 64 * page
                    assert torch.equal(got, want[lo:lo + there, off + head * dim:off + (head + 1) * dim])
        base += length
    # in place, and out of a wider row: the same
    wide = torch.randn(n + 5, 2 * kv * dim + 24, device=DEV).to(dtype)
    wide[:, 24:] = rows
    part = wide[:, 24:]
    before = g.k[0].clone(), g.v[0].clone()
    attention4.store(part, step, p.view, held=part)
    assert torch.equal(part, held) and torch.equal(g.k[0], before[0]) and torch.equal(g.v[0], before[1])


def test_odd_numbers_in_rows():
    from hos_b200.parts import attention4
    for dtype in (BF, F32):
        p = Paged([12], 1, 64, dtype=dtype)
        rows = torch.randn(12, 128, generator=gen(5))
        rows[0, :] = 0.0
        rows[1, :] = 3.25
        rows[2, 5] = math.inf
        rows[3, 70] = -math.inf
        rows[4, 100] = math.nan
        rows[5, 0], rows[5, 1] = 3.0e38, -3.0e38                  # the range overflows
        rows[6, :] = 1000.0 + 1e-3 * rows[6, :]
        rows[7, :64] = 1e-39 * torch.arange(64)                   # a subnormal scale
        rows[8, :] = torch.arange(128) % 16 * 0.5                  # ties of codes and steps that are exact
        rows[9, :] = -0.0
        rows[10, 3] = 1e30
        rows[11, :] = rows[11, :] * 1e-30
        rows = rows.to(dtype).to(DEV)
        held = torch.empty_like(rows)
        attention4.store(rows, p.step([12]), p.view, held=held)
        want = held_of(rows).to(dtype).float()
        got = held.cpu().float()
        assert torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(got.nan_to_num(1.5), want.nan_to_num(1.5))


def test_a_ring_keeps_the_last_positions_of_a_long_prompt_and_padding_stores_nothing():
    from hos_b200.parts import attention4
    p = Paged([200], 1, 64, window=100)
    g = p.c.groups[0]
    assert g.ring_pages == 2
    rows = torch.randn(203, 128, generator=gen(6)).to(BF).to(DEV)
    attention4.store(rows, p.step([200], pad=203), p.view)
    want = held_of(rows)
    for e, lo, hi in ((0, 128, 192), (1, 72, 128)):               # entry 1 holds 64..127, then 192..199 over it
        got = unpacked(g.k[0][int(g.table_host[p.slots[0], e]), 0], 64, False)
        for q in range(lo, hi):
            assert torch.equal(got[q % 64], want[q, :64])
    got = unpacked(g.v[0][int(g.table_host[p.slots[0], 1]), 0], 64, True)
    for q in range(192, 200):
        assert torch.equal(got[q % 64], want[q, 64:])
    assert int((g.k[0].view(g.k[0].shape[0], -1) != 255).any(1).sum()) == 2                # no other page was touched


def test_many_rows_are_stored_as_few_are():
    from hos_b200.parts import attention4
    lens = [1, 63, 64, 65, 500, 16, 129]
    for kv, dim, dtype in ((2, 128, BF), (1, 256, F32)):
        rows = torch.randn(sum(lens), 2 * kv * dim, generator=gen(8)).to(dtype).to(DEV)
        a, b = Paged(lens, kv, dim, dtype=dtype), Paged(lens, kv, dim, dtype=dtype)
        attention4.store(rows, a.step(lens), a.view)
        base = [sum(lens[:i]) for i in range(len(lens))]
        for at in range(0, 500, 23):                              # a few tokens at a time, from odd positions on
            live = [i for i, n in enumerate(lens) if n > at]
            news = [min(23, lens[i] - at) for i in live]
            from hos_b200.engine.batch import build_step
            step = build_step([[0] * n for n in news], [at] * len(live), [b.slots[i] for i in live], torch.device(DEV), 1)
            attention4.store(torch.cat([rows[base[i] + at:base[i] + at + n] for i, n in zip(live, news)]), step, b.view)
        assert torch.equal(a.c.groups[0].k[0], b.c.groups[0].k[0]) and torch.equal(a.c.groups[0].v[0], b.c.groups[0].v[0])


# ---- attention -------------------------------------------------------------------------------------------------------
def check_attention(lens, news, heads, kv, dim, window=None, cap=0.0, dtype=BF, seed=1, pad=0, size=1.0, chunk=1, scale=None):
    from hos_b200.parts import attention4
    scale = dim ** -0.5 if scale is None else scale
    p = Paged(lens, kv, dim, window, dtype, seed, chunk)
    rows = (torch.randn(sum(lens), 2 * kv * dim, generator=gen(seed)) * size).to(dtype).to(DEV)
    # fill the pages in steps that a ring has room for
    base, filled = [sum(lens[:i]) for i in range(len(lens))], 0
    piece = max(lens) if window is None else 64 * p.c.groups[0].ring_pages - window + 1
    from hos_b200.engine.batch import build_step
    while filled < max(lens):
        live = [i for i, n in enumerate(lens) if n > filled]
        take = [min(piece, lens[i] - filled) for i in live]
        step = build_step([[0] * n for n in take], [filled] * len(live), [p.slots[i] for i in live], torch.device(DEV), 1)
        attention4.store(torch.cat([rows[base[i] + filled:base[i] + filled + n] for i, n in zip(live, take)]), step, p.view)
        filled += piece
    n = sum(news)
    q = torch.randn(n + pad, heads * dim, generator=gen(seed + 9)).to(dtype).to(DEV)
    wide = torch.full((n + pad, heads * dim + 40), 3.0, dtype=dtype, device=DEV)
    wide[:, 16:16 + heads * dim] = q
    out = torch.full((n + pad, heads * dim + 8), 5.0, dtype=dtype, device=DEV)
    attention4.attend(wide[:, 16:16 + heads * dim], out[:, :heads * dim], p.step(news, pad=n + pad), p.view, heads, scale, cap, window)
    assert float((out[:, heads * dim:] - 5).abs().max()) == 0
    got = out[:, :heads * dim]
    if pad:
        assert float(got[n:].abs().max()) == 0
    held = held_of(rows).double().to(DEV)
    c, s, _ = quantised(rows)
    moved = (c.abs() * s[..., None]).flatten(-2).double().to(DEV)          # what of a value its code makes: the part that is rounded
    at = 0
    for i, length in enumerate(lens):
        k, v, vm = (t[base[i]:base[i] + length, lo:lo + kv * dim].view(length, kv, dim)
                    for t, lo in ((held, 0), (held, kv * dim), (moved, kv * dim)))
        new = news[i]
        qs = q[at:at + new].double().view(new, kv, heads // kv, dim)
        y = torch.einsum("nkgd,lkd->nkgl", qs, k) * scale
        mag = torch.einsum("nkgd,lkd->nkgl", qs.abs(), k.abs()) * scale
        if cap:
            y = cap * torch.tanh(y / cap)
        dist = torch.arange(length - new, length, device=DEV)[:, None] - torch.arange(length, device=DEV)
        hidden = (dist < 0) | ((dist >= window) if window else (dist < 0))
        hid = hidden[:, None, None].expand_as(y)
        prob = y.masked_fill(hid, -math.inf).softmax(-1)
        want = torch.einsum("nkgl,lkd->nkgd", prob, v)
        err_score = 2.0 ** -21 * (mag + y.abs() + 4)
        err = 2 * torch.einsum("nkgl,lkd->nkgd", prob * err_score, v.abs()) + 2 * (prob * err_score).sum(-1, keepdim=True) * want.abs()
        if dtype == BF:
            err = err + torch.einsum("nkgl,lkd->nkgd", prob, vm) * 2.0 ** -8 + 2.0 ** -8 * want.abs()
        else:
            err = err + torch.einsum("nkgl,lkd->nkgd", prob, v.abs()) * 2.0 ** -18
        diff = (got[at:at + new].double().view_as(want) - want).abs()
        assert bool((diff <= err + 1e-30).all()), f"sequence {i}: off by {float(diff.max()):.3g}, allowed {float(err.max()):.3g}"
        at += new


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("dim", [64, 128, 192, 256])
@pytest.mark.parametrize("heads,kv", [(1, 1), (2, 1), (8, 4), (10, 2), (16, 1), (17, 1), (40, 2)])
def test_single_tokens(heads, kv, dim, dtype):
    check_attention([1, 2, 15, 16, 17, 63, 64, 65, 200], [1] * 9, heads, kv, dim, cap=20.0 if heads == 8 else 0.0, dtype=dtype)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("window", [1, 2, 16, 63, 64, 100, 1000])
def test_single_tokens_in_a_window(window, dtype):
    check_attention([1, 17, 64, 129, 300, 777], [1] * 6, 4, 2, 64, window=window, cap=5.0, dtype=dtype)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("lens", [[5000], [1, 3000, 10, 2999], [700] * 20, [1] * 70 + [4100]])
def test_long_and_unequal_lengths(lens, dtype):
    check_attention(lens, [1] * len(lens), 4, 2, 128, cap=30.0, dtype=dtype)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("lens,news,window", [([40], [40], None), ([5, 300], [5, 7], None), ([100, 90, 300, 301], [100, 30, 64, 129], None),
                                             ([500, 260], [200, 100], 130), ([1000], [2], None), ([129, 130, 5], [20, 3, 1], 64)])
def test_several_tokens_a_sequence(lens, news, window, dtype):
    check_attention(lens, news, 4, 2, 128, window=window, cap=0.0, dtype=dtype, chunk=256)
    check_attention(lens, news, 6, 1, 64, window=window, cap=9.0, dtype=dtype, chunk=256)


def test_a_long_piece():
    check_attention([1500, 640], [739, 600], 8, 4, 256, cap=50.0, chunk=1024)
    check_attention([1500], [333], 4, 2, 128, window=400, chunk=512)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_padding_rows_become_zeros(dtype):
    check_attention([1, 30, 70], [1, 1, 1], 4, 2, 128, dtype=dtype, pad=5)
    check_attention([90, 70], [50, 20], 4, 2, 128, dtype=dtype, pad=3)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_large_scores_and_tiny_ones(dtype):
    check_attention([300], [1], 4, 2, 64, dtype=dtype, size=60.0, scale=1.0)               # one key takes all
    check_attention([300], [1], 4, 2, 64, dtype=dtype, size=1e-4)                          # all keys alike
    check_attention([300], [1], 4, 2, 64, dtype=dtype, size=60.0, scale=1.0, cap=50.0)


def test_what_the_mask_hides_may_be_anything():
    """NaN and infinities before the window, behind the position and in rows of a page that nobody wrote."""
    from hos_b200.parts import attention4
    for dtype in (BF, F32):
        p = Paged([200], 2, 64, dtype=dtype)
        rows = torch.randn(200, 256, generator=gen(4)).to(dtype).to(DEV)
        bad = rows.clone()
        bad[:110] = math.nan
        bad[170:] = math.inf
        outs = []
        for r in (rows, bad):
            attention4.store(r, p.step([200]), p.view)
            q = torch.randn(30, 256, generator=gen(7)).to(dtype).to(DEV)
            for new in (1, 30):
                step = p.step([new], starts=[170 - new])
                out = torch.empty(new, 256, dtype=dtype, device=DEV)
                attention4.attend(q[:new], out, step, p.view, 4, 0.125, 0.0, 20)
                outs.append(out)
        assert bool(torch.isfinite(outs[2]).all()) and torch.equal(outs[0], outs[2])
        assert torch.equal(outs[1], outs[3])


def test_attention_repeats_bit_for_bit_and_runs_on_another_stream():
    from hos_b200.parts import attention4
    p = Paged([3000, 2000], 2, 128)
    rows = torch.randn(5000, 512, generator=gen(4)).to(BF).to(DEV)
    attention4.store(rows, p.step([3000, 2000]), p.view)
    q = torch.randn(2, 512, generator=gen(7)).to(BF).to(DEV)
    step = p.step([1, 1])
    outs = []
    for i in range(4):
        out = torch.empty_like(q)
        attention4.attend(q, out, step, p.view, 4, 0.1)
        outs.append(out)
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        out = torch.empty_like(q)
        attention4.attend(q, out, step, p.view, 4, 0.1)
        outs.append(out)
    torch.cuda.synchronize()
    assert all(torch.equal(outs[0], o) for o in outs)


def test_the_cache_refuses_what_does_not_fit():
    from hos_b200 import ops
    from hos_b200.errors import KernelError
    from hos_b200.parts import attention4
    p = Paged([10, 20], 2, 64)
    step, rows, q = p.step([1, 1]), torch.zeros(2, 256, device=DEV, dtype=BF), torch.zeros(2, 256, device=DEV, dtype=BF)
    plain = ops.PagedKVArgs(torch.zeros(4, 2, 64, 64, device=DEV, dtype=BF), torch.zeros(4, 2, 64, 64, device=DEV, dtype=BF), p.view.page_table, 0, 2, 64)
    for call in (lambda: attention4.store(rows, step, plain), lambda: attention4.store(rows[:, :192], step, p.view), lambda: attention4.store(rows[:1], step, p.view),
                 lambda: attention4.store(rows.half(), step, p.view), lambda: attention4.store(rows.cpu(), step, p.view),
                 lambda: attention4.store(rows, step, p.view, held=rows.float()), lambda: attention4.store(rows, step, p.view, held=rows[:1]),
                 lambda: attention4.attend(q, torch.empty_like(q), step, plain, 4, 1.0), lambda: attention4.attend(q, torch.empty_like(q), step, p.view, 5, 1.0),
                 lambda: attention4.attend(q, torch.empty_like(q).float(), step, p.view, 4, 1.0), lambda: attention4.attend(q[:1], q[:1].clone(), step, p.view, 4, 1.0),
                 lambda: attention4.attend(q[:, :192], q[:, :192].clone(), step, p.view, 3, 1.0),
                 lambda: attention4.attend(q, q.t(), step, p.view, 4, 1.0),
                 lambda: ops.attn_plain(q, 256, torch.empty_like(q), step.token_pos, step.token_seq, 2, 4, 2, 64, 1.0, 0.0, None, seq_slot=step.seq_slot, cache=p.view)):
        with pytest.raises(KernelError):
            call()


# ---- pages -----------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype,kv,dim,bits", [(BF, 4, 256, None), (F32, 1, 16, None), (BF, 3, 48, None), (BF, 2, 64, 4), (F32, 5, 128, 4)])
def test_copied_pages(dtype, kv, dim, bits):
    from hos_b200.cache.kv import KVGroup
    from hos_b200.parts.base import KVNeed
    g = KVGroup(KVNeed(kv, dim, None, bits=bits), 3, 40, 4, 4096, dtype, torch.device(DEV))
    arrays = g.k + g.v
    for a in arrays:
        a.copy_(torch.randint(0, 255, a.shape, dtype=torch.uint8) if bits else torch.randn(a.shape))
    before = [a.clone() for a in arrays]
    src = [3, 39, 0, 5, 5, -1, 7, 40, 8, 9]
    dst = [4, 1, 38, 6, 2, 10, -1, 11, 8, 40]                     # the last five copy nothing
    g.copy_pages(torch.tensor(src, dtype=torch.int32, device=DEV), torch.tensor(dst, dtype=torch.int32, device=DEV))
    for a, b in zip(arrays, before):
        for s, d in zip(src[:5], dst[:5]):
            b[d] = b[s]
        assert torch.equal(a, b)
    g.copy_pages(torch.empty(0, dtype=torch.int32, device=DEV), torch.empty(0, dtype=torch.int32, device=DEV))
    for a, b in zip(arrays, before):
        assert torch.equal(a, b)


def test_copied_pages_of_arrays_with_pages_of_unequal_size():
    from hos_b200.cache.kv import KVGroup
    from hos_b200.parts.base import KVNeed
    g = KVGroup(KVNeed(2, 192, None, v_head_dim=16), 2, 300, 4, 4096, BF, torch.device(DEV))
    for a in g.k + g.v:
        a.copy_(torch.randn(a.shape))
    before = [a.clone() for a in g.k + g.v]
    order = torch.randperm(300, generator=gen(1)).to(torch.int32).to(DEV)
    g.copy_pages(order[:150].contiguous(), order[150:].contiguous())
    for a, b in zip(g.k + g.v, before):
        b[order[150:].long()] = b[order[:150].long()]
        assert torch.equal(a, b)


def test_copies_refuse_what_does_not_fit():
    from hos_b200.cache.kv import KVGroup
    from hos_b200.errors import KernelError
    from hos_b200.parts.base import KVNeed
    g = KVGroup(KVNeed(2, 64, None), 1, 8, 4, 512, BF, torch.device(DEV))
    a = torch.zeros(3, dtype=torch.int32, device=DEV)
    for src, dst in ((a, a[:2]), (a.long(), a.long()), (a.cpu(), a.cpu()), (a[None], a[None])):
        with pytest.raises(KernelError):
            g.copy_pages(src, dst)
