"""The 4-bit operators where numbers are far apart in size, where kernels cut their work otherwise than usual, and a wait that runs
out.

Tolerances: many rows' weights are formed in half precision (2^-12 of a weight down to 2^-14 of the feature's largest scale, below that
2^-25 of that scale) and rows to 2^-11 of a number or 2^-34 of the row's largest; attention's weights are within 2^-11 of themselves down to
2^-20 of the largest (below 2^-30 of it lost), scores as in test_fourbit_gpu.py; results are rounded to bfloat16."""
import math

import pytest
import torch

from test_fourbit_gpu import Paged, check_product, gen, held_of, made_weights

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, F32 = torch.bfloat16, torch.float32


@pytest.mark.parametrize("tile_rows,shares", [(16, 1), (16, 8), (48, 2), (96, 4), (128, 1), (128, 8), (176, 1), (240, 1), (256, 1)])
@pytest.mark.parametrize("group,zeros,gated", [(64, False, False), (32, True, False), (128, True, True), (32, False, True)])
def test_tiles_and_shares_of_many_rows(tile_rows, shares, group, zeros, gated):
    from hos_b200 import ops
    from hos_b200.parts.weights4 import Weight4
    m, n, k = 301, 200, 584
    blocks = 2 if gated else 1
    codes, scales, z, w = made_weights(blocks * n, k, group, zeros, 5)
    w4 = Weight4.from_codes(codes, scales, z, group, blocks=blocks)
    x = torch.randn(m, k, generator=gen(6)).to(BF).to(DEV)
    out = torch.empty(m, n, dtype=F32, device=DEV)
    ops.product4_tc(x, w4._address, k, out, 0, 0.0, tile_rows, shares)
    y, size = x.double() @ w.T, x.double().abs() @ w.abs().T
    err = size * 2.0 ** -11
    if gated:
        g, u, eg, eu = y[:, :n], y[:, n:], err[:, :n], err[:, n:]
        a = torch.nn.functional.gelu(g, approximate="tanh")
        y, err = a * u, 1.2 * eg * u.abs() + a.abs() * eu + 1.2 * eg * eu + 2.0 ** -19 * (a * u).abs()
    assert bool(((out.double() - y).abs() <= err).all())
    again = torch.empty_like(out)
    ops.product4_tc(x, w4._address, k, again, 0, 0.0, tile_rows, shares)
    assert torch.equal(out, again)


@pytest.mark.parametrize("k", [64, 65, 71, 200, 333])
def test_many_rows_of_any_width(k):
    for m, pad in ((33, 0), (64, 5), (130, 8)):
        check_product(m, 150, k, 32, True, False, BF, pad=pad)
        check_product(m, 50, k, 64, False, True, BF, act=1, pad=pad)


def test_rows_and_scales_far_apart_in_size():
    from hos_b200.parts.weights4 import Weight4
    m, n, k, group = 80, 140, 512, 64
    codes, scales, z, _ = made_weights(n, k, group, True, 7)
    scales = (scales.float() * torch.exp2(torch.randint(-12, 1, scales.shape, generator=gen(8)).to(DEV).float())
              * torch.exp2(torch.linspace(-90, 90, n, device=DEV).round())[:, None]).to(BF)
    scales[3] = 0.0
    at = torch.arange(k, device=DEV) // group
    w = (codes.double() - z.double()[:, at]) * scales.double()[:, at]
    x = torch.randn(m, k, generator=gen(9)).to(DEV) * torch.exp2(torch.linspace(-30, 30, m, device=DEV).round())[:, None]
    x[5] = 0.0
    x[6, 1:] = 0.0
    x = x.to(BF)
    got = Weight4.from_codes(codes, scales, z, group).product(x, torch.float32)
    xd = x.double()
    y, size = xd @ w.T, xd.abs() @ w.abs().T
    largest = scales.double().amax(1)
    err = size * 2.0 ** -11 + xd.abs().sum(1, keepdim=True) * largest[None] * 2.0 ** -24 + xd.abs().amax(1, keepdim=True) * 2.0 ** -33 * w.abs().sum(1)[None]
    assert bool(torch.isfinite(got).all()) and bool(((got.double() - y).abs() <= err + 1e-40).all())
    assert float(got[5].abs().max()) == 0 and float(got[:, 3].abs().max()) == 0


def test_a_row_that_is_not_a_number_spoils_itself_alone():
    from hos_b200.parts.weights4 import Weight4
    codes, scales, z, _ = made_weights(130, 256, 64, False, 4)
    w4 = Weight4.from_codes(codes, scales, None, 64)
    x = torch.randn(70, 256, device=DEV).to(BF)
    want = w4.product(x)
    x[10, 3], x[20, 4], x[69, 255] = math.nan, math.inf, -math.inf
    got = w4.product(x)
    bad = torch.zeros(70, dtype=torch.bool, device=DEV)
    bad[[10, 20, 69]] = True
    assert torch.equal(got[~bad], want[~bad]) and not bool(torch.isfinite(got[bad]).any())


def test_a_wait_that_runs_out_is_told_and_the_next_product_is_right():
    from hos_b200 import ops
    from hos_b200.errors import KernelError
    from hos_b200.parts.weights4 import Weight4
    codes, scales, z, _ = made_weights(300, 1024, 64, False, 4)
    w4 = Weight4.from_codes(codes, scales, None, 64)
    x = torch.randn(100, 1024, device=DEV).to(BF)
    want = w4.product(x)
    torch.cuda.synchronize()
    ops.check_errors()
    for tile_rows, shares in ((112, 1), (112, 4)):
        ops.product4_tc(x, w4._address, 1024, torch.empty_like(want), 0, 0.0, tile_rows, shares, wait_cycles=2_000_000, stop_stage=1)
        torch.cuda.synchronize()
        with pytest.raises(KernelError, match="4-bit weights"):
            ops.check_errors()
    assert torch.equal(w4.product(x), want)
    torch.cuda.synchronize()
    ops.check_errors()


def attention(p, rows, lens, news, heads, kv, dim, window=None, cap=0.0, scale=None):
    """(what the kernels give, the same in 64 bits of what is held) of the last `news` tokens."""
    from hos_b200.parts import attention4
    scale = dim ** -0.5 if scale is None else scale
    attention4.store(rows, p.step(lens, starts=[0] * len(lens)), p.view)
    q = torch.randn(sum(news), heads * dim, generator=gen(9)).to(rows.dtype).to(DEV)
    out = torch.empty_like(q)
    attention4.attend(q, out, p.step(news), p.view, heads, scale, cap, window)
    held, want, at, base = held_of(rows).double().to(DEV), [], 0, 0
    for length, new in zip(lens, news):
        k, v = (held[base:base + length, lo:lo + kv * dim].view(length, kv, dim) for lo in (0, kv * dim))
        y = torch.einsum("nkgd,lkd->nkgl", q[at:at + new].double().view(new, kv, heads // kv, dim), k) * scale
        y = cap * torch.tanh(y / cap) if cap else y
        dist = torch.arange(length - new, length, device=DEV)[:, None] - torch.arange(length, device=DEV)
        hidden = (dist < 0) | ((dist >= window) if window else (dist < 0))
        want.append(torch.einsum("nkgl,lkd->nkgd", y.masked_fill(hidden[:, None, None].expand_as(y), -math.inf).softmax(-1), v).reshape(new, -1))
        at, base = at + new, base + length
    return out, torch.cat(want)


@pytest.mark.parametrize("new,heads,kv,dim", [(1, 8, 4, 256), (1, 4, 4, 64), (60, 8, 4, 256), (70, 4, 2, 128), (5, 4, 2, 64)])
def test_long_rows_lose_no_more_than_the_results_rounding(new, heads, kv, dim):
    """The output of many keys is a small mean of them: its error, relative to its norm, is the rounding's of the result alone."""
    lens = [6000]
    p = Paged(lens, kv, dim)
    got, want = attention(p, torch.randn(6000, 2 * kv * dim, generator=gen(3)).to(BF).to(DEV), lens, [new], heads, kv, dim)
    assert float((got.double() - want).norm() / want.norm()) < 2.0 ** -9 + 2.0 ** -12


@pytest.mark.parametrize("new", [1, 3, 60])
@pytest.mark.parametrize("order", ["rising", "falling", "jumps", "tiny"])
def test_values_far_apart_in_size(new, order):
    """Scales of values from 2^-40 to 2^40 along a sequence (or all of them below any normal weight), unwritten places full of what would
    be the largest of all."""
    lens, heads, kv, dim = [700, 330], 4, 2, 128
    at = torch.cat([torch.linspace(0, 1, n) for n in lens])
    e = {"rising": 80 * at - 40, "falling": 40 - 80 * at, "jumps": torch.where((torch.arange(len(at)) * 7) % 11 < 2, 40.0, -5.0),
         "tiny": torch.full_like(at, -110.0)}[order]
    rows = torch.randn(sum(lens), 2 * kv * dim, generator=gen(5))
    rows[:, kv * dim:] *= torch.exp2(e.round())[:, None]
    p = Paged(lens, kv, dim)
    for a in p.c.groups[0].k + p.c.groups[0].v:
        a.fill_(0x7e)                                             # as a scale and a middle in bfloat16: 8.4e37
    rows = rows.to(BF).to(DEV)
    got, want = attention(p, rows, lens, [new, new], heads, kv, dim)
    largest = torch.cat([held_of(rows)[lo:hi, kv * dim:].double().abs().view(hi - lo, kv, -1).amax((0, 2)).to(DEV).repeat_interleave(heads // kv)
                         .repeat_interleave(dim).expand(new, -1) for lo, hi in ((0, lens[0]), (lens[0], sum(lens)))])
    assert bool(torch.isfinite(got).all()) and bool(((got.double() - want).abs() <= 2.0 ** -7 * want.abs() + 2.0 ** -8 * largest).all())
    close = (got.double() - want).norm(dim=1) / want.norm(dim=1)
    assert float(close.max()) < 2.0 ** -8


def test_many_heads_and_odd_groups_in_pieces():
    for heads, kv, dim, new in ((6, 2, 64, 40), (5, 1, 128, 30), (48, 2, 64, 9), (24, 1, 256, 7), (130, 1, 64, 3)):
        lens = [300, 100 + new]
        got, want = attention(Paged(lens, kv, dim), torch.randn(sum(lens), 2 * kv * dim, generator=gen(3)).to(BF).to(DEV), lens, [new, new], heads, kv, dim,
                              window=90, cap=20.0)
        assert float((got.double() - want).norm() / want.norm()) < 2.0 ** -9 + 2.0 ** -11
