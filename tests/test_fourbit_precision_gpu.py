"""How near the 4-bit operators' bfloat16 forms come: operands in half precision, not in bfloat16, whose error would pass these bounds.

Tolerances.  Products of more than 32 rows: weights are rounded once to half precision, 2^-11 of themselves; sums in 32 bits of exact products
are within 2^-18 of the sum of the magnitudes; a bfloat16 result is within 2^-8 of itself.  Attention: what of a value its code makes (code
times scale) has a weight that is rounded to half precision, 2^-11 of itself down to 2^-22 of the largest (weights may be 2^8 times the
running maximum's, half precision has 2^14 to 2^-14 at full length), an error in that part of 2^-30 of the largest value a key below; scores as in
test_fourbit_gpu.py."""
import math

import pytest
import torch

from test_fourbit_gpu import Paged, gen, held_of, made_weights, quantised

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, F32 = torch.bfloat16, torch.float32


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("m,n,k,group,zeros", [(33, 40, 320, 64, False), (64, 130, 777, 32, True), (200, 515, 1984, 64, False), (513, 640, 1160, 128, True),
                                               (1000, 300, 2304, 64, True)])
def test_products_of_many_rows(m, n, k, group, zeros, dtype):
    from hos_b200.parts.weights4 import Weight4
    codes, scales, z, w = made_weights(n, k, group, zeros, 31)
    x = torch.randn(m, k, generator=gen(32)).to(BF).to(DEV)
    got = Weight4.from_codes(codes, scales, z, group).product(x, dtype).double()
    y, size = x.double() @ w.T, x.double().abs() @ w.abs().T
    err = size * (2.0 ** -11 + 2.0 ** -18) + (2.0 ** -8 * y.abs() if dtype == BF else 0.0)
    assert bool(((got - y).abs() <= err).all())
    if dtype == F32:                                             # roundings that fall either way: far below their bound, and below bfloat16's
        assert float((got - y).norm() / (size.norm() / math.sqrt(k))) < 2.0 ** -11


@pytest.mark.parametrize("new", [1, 3, 60])
@pytest.mark.parametrize("heads,kv,dim,window,cap", [(8, 4, 256, None, 50.0), (4, 2, 128, 700, 0.0), (6, 1, 64, None, 0.0), (3, 3, 192, 100, 9.0)])
def test_attention(heads, kv, dim, window, cap, new):
    from hos_b200.parts import attention4
    length, scale = 1500, dim ** -0.5
    p = Paged([length], kv, dim)                                 # no ring: the window is the call's alone
    rows = torch.randn(length, 2 * kv * dim, generator=gen(33)).to(BF).to(DEV)
    attention4.store(rows, p.step([length], starts=[0]), p.view)
    q = torch.randn(new, heads * dim, generator=gen(34)).to(BF).to(DEV)
    out = torch.empty_like(q)
    attention4.attend(q, out, p.step([new]), p.view, heads, scale, cap, window)
    held = held_of(rows).double().to(DEV)
    c, s, _ = quantised(rows)
    moved = (c.abs() * s[..., None]).flatten(-2).double().to(DEV)
    k, v, vm = (t[:, lo:lo + kv * dim].view(length, kv, dim) for t, lo in ((held, 0), (held, kv * dim), (moved, kv * dim)))
    qs = q.double().view(new, kv, heads // kv, dim)
    y, mag = torch.einsum("nkgd,lkd->nkgl", qs, k) * scale, torch.einsum("nkgd,lkd->nkgl", qs.abs(), k.abs()) * scale
    y = cap * torch.tanh(y / cap) if cap else y
    dist = torch.arange(length - new, length, device=DEV)[:, None] - torch.arange(length, device=DEV)
    hidden = ((dist < 0) | ((dist >= window) if window else (dist < 0)))[:, None, None].expand_as(y)
    prob = y.masked_fill(hidden, -math.inf).softmax(-1)
    want = torch.einsum("nkgl,lkd->nkgd", prob, v)
    score = 2.0 ** -21 * (mag + y.abs() + 4)
    err = 2 * torch.einsum("nkgl,lkd->nkgd", prob * score, v.abs()) + 2 * (prob * score).sum(-1, keepdim=True) * want.abs()
    err = err + torch.einsum("nkgl,lkd->nkgd", prob, vm) * 2.0 ** -11 + 2.0 ** -8 * want.abs() + length * 2.0 ** -30 * float(vm.max())
    assert bool(((out.double().view_as(want) - want).abs() <= err).all())
