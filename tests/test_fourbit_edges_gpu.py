"""The 4-bit operators at the edges of what numbers can be: scales of one feature far apart, infinities, numbers near the largest, and
what the host refuses.

Tolerances: weights formed in half precision are rounded once, to 2^-11 of themselves; 32-bit sums and what is held as exact as in
test_fourbit_gpu.py."""
import math

import pytest
import torch

from test_fourbit_gpu import Paged, check_attention, gen, made_weights

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, F32 = torch.bfloat16, torch.float32


@pytest.mark.parametrize("group,zeros", [(32, False), (32, True), (64, True), (128, False)])
def test_weights_of_many_rows_are_rounded_once_however_small_their_scale_is(group, zeros):
    """A row of x that is one number alone gives back one weight: no other group hides what a small scale loses.  Scales down to 2^-24 of
    their feature's largest."""
    from hos_b200.parts.weights4 import Weight4
    n, k = 80, 512
    groups = k // group
    codes, _, z, _ = made_weights(n, k, group, zeros, 11)
    exponent = -torch.round(torch.arange(groups) * 24 / (groups - 1))
    scales = ((1 + torch.rand(n, groups, generator=gen(12))) * torch.exp2(exponent)).to(BF).to(DEV)
    at = torch.arange(k, device=DEV) // group
    w = (codes.double() - (z.double()[:, at] if zeros else 8.0)) * scales.double()[:, at]
    got = Weight4.from_codes(codes, scales, z, group).product(torch.eye(k, device=DEV, dtype=BF), F32)
    assert bool(((got.double() - w.T).abs() <= 2.0 ** -11 * w.T.abs()).all())


def check_odd_rows(x, w4, w, eps):
    """A product's row is infinite, or not a number, where the definition's is; elsewhere as near as ever."""
    got = w4.product(x, F32).double()
    xd = x.double()
    y, size = xd @ w.T, xd.abs() @ w.abs().T
    assert torch.equal(torch.isnan(got), torch.isnan(y))
    inf = torch.isinf(y)
    assert torch.equal(torch.isinf(got), inf) and torch.equal(got[inf], y[inf])
    fine = torch.isfinite(y)
    assert bool(((got - y).abs() <= size * eps)[fine].all())


@pytest.mark.parametrize("dtype,eps", [(BF, 2.0 ** -18), (F32, 2.0 ** -20)])
@pytest.mark.parametrize("group,zeros", [(32, True), (64, False), (128, True)])
@pytest.mark.parametrize("m", [1, 7, 12, 32])
def test_infinities_in_rows_give_infinities(m, group, zeros, dtype, eps):
    from hos_b200.parts.weights4 import Weight4
    codes, scales, z, w = made_weights(100, 333, group, zeros, 13)
    w4 = Weight4.from_codes(codes, scales, z, group)
    x = torch.randn(m, 333, generator=gen(14)).to(dtype).to(DEV)
    x[m // 2, 5] = math.inf
    check_odd_rows(x, w4, w, eps)
    x[m - 1, 332] = -math.inf
    check_odd_rows(x, w4, w, eps)
    x[0, 100] = math.nan
    check_odd_rows(x, w4, w, eps)


@pytest.mark.parametrize("dtype,eps", [(BF, 2.0 ** -18), (F32, 2.0 ** -20)])
@pytest.mark.parametrize("m", [1, 7, 12, 32])
def test_rows_of_numbers_near_the_largest(m, dtype, eps):
    """Sums of codes times numbers pass the largest that 32 bits hold, sums of weights times numbers do not."""
    from hos_b200.parts.weights4 import Weight4
    for zeros in (False, True):
        codes, scales, z, w = made_weights(100, 512, 64, zeros, 15)
        w4 = Weight4.from_codes(codes, scales, z, 64)
        x = torch.randn(m, 512, generator=gen(16)).to(DEV)
        x[m // 2] = 2.0 ** 121 * (1 + torch.rand(512, generator=gen(17)).to(DEV))
        check_odd_rows(x.to(dtype), w4, w, eps)


@pytest.mark.parametrize("m", [1, 20])
def test_gated_products_of_infinities(m):
    from hos_b200 import ops
    from hos_b200.parts import linear
    from hos_b200.parts.weights4 import Weight4
    codes, scales, z, w = made_weights(2 * 50, 256, 64, False, 18)
    scales = scales.abs() + 0.001
    codes = torch.where(codes == 8, 9, codes).to(torch.uint8)      # no weight is 0: an infinity times it is one
    w4 = Weight4.from_codes(codes, scales, None, 64, blocks=2)
    w = (codes.double() - 8) * scales.double().repeat_interleave(64, 1)
    x = torch.randn(m, 256, generator=gen(19)).to(BF).to(DEV)
    x[m - 1, 77] = -math.inf
    got = linear.matmul(x, w4, F32, epilogue=ops.EPI_GATED, act=ops.ACT_GELU_TANH).double()
    gate, up = (x.double() @ w.T).split(50, dim=1)
    row = torch.where(gate[m - 1] > 0, gate[m - 1] * up[m - 1], math.nan)      # gelu of -infinity is 0, or, as formed, not a number
    pos = gate[m - 1] > 0
    assert bool(pos.any()) and torch.equal(got[m - 1][pos], row[pos])
    assert bool(torch.isfinite(got[:m - 1]).all())


@pytest.mark.parametrize("shares", [1, 4])
@pytest.mark.parametrize("scale,row", [(112, -112), (-112, 112), (120, -100), (-120, 100)])
def test_a_features_scale_and_a_rows_size_far_from_one_undo_each_other(scale, row, shares):
    from hos_b200 import ops
    from hos_b200.parts.weights4 import Weight4
    codes, scales, z, w = made_weights(150, 512, 64, True, 20)
    scales = (scales.float() * 2.0 ** scale).to(BF)                # some of the smallest are subnormal: rounded here
    w4 = Weight4.from_codes(codes, scales, z, 64)
    at = torch.arange(512, device=DEV) // 64
    w = (codes.double() - z.double()[:, at]) * scales.double()[:, at]
    x = (torch.randn(48, 512, generator=gen(21)) * 2.0 ** row).to(BF).to(DEV)
    got = torch.empty(48, 150, device=DEV)
    ops.product4_tc(x, w4._address, 512, got, 0, 0.0, 48, shares)
    y, size = x.double() @ w.T, x.double().abs() @ w.abs().T
    assert bool(((got.double() - y).abs() <= size * 2.0 ** -10.9).all())


@pytest.mark.parametrize("shares", [1, 4])
def test_nothing_times_the_largest_powers_is_nothing(shares):
    from hos_b200 import ops
    from hos_b200.parts.weights4 import Weight4
    codes = torch.full((128, 256), 8, dtype=torch.uint8, device=DEV)
    codes[1] = 9                                                   # one feature whose products pass the largest number
    w4 = Weight4.from_codes(codes, torch.full((128, 4), 2.0 ** 120, device=DEV, dtype=BF), None, 64)
    x = torch.full((48, 256), 2.0 ** 100, device=DEV, dtype=BF)
    got = torch.empty(48, 128, device=DEV)
    ops.product4_tc(x, w4._address, 256, got, 0, 0.0, 48, shares)
    assert bool(torch.isinf(got[:, 1]).all())
    got[:, 1] = 0
    assert float(got.abs().max()) == 0


def test_scales_and_zero_codes_that_lie_elsewhere_than_the_codes_are_refused():
    from hos_b200.errors import SpecError
    from hos_b200.parts.weights4 import Weight4
    codes, scales, z, _ = made_weights(32, 128, 64, True, 22)
    for bad in (dict(codes=codes.cpu()), dict(scales=scales.cpu()), dict(scales=scales.cpu(), zeros=None), dict(zeros=z.cpu()),
                dict(codes=codes.cpu(), scales=scales.cpu(), zeros=None)):
        with pytest.raises(SpecError, match="GPU"):
            Weight4.from_codes(**{**dict(codes=codes, scales=scales, zeros=z, group=64), **bad})


def test_matrices_and_codes_whose_numbers_do_not_lie_side_by_side():
    from hos_b200.parts.weights4 import Weight4
    codes, scales, z, _ = made_weights(48, 128, 64, True, 23)
    x = torch.randn(3, 128, device=DEV)
    want = Weight4.from_codes(codes, scales, z, 64, blocks=1).product(x)
    apart = Weight4.from_codes(codes.t().contiguous().t(), scales.t().contiguous().t(), z.repeat_interleave(2, 1)[:, ::2], 64)
    assert torch.equal(apart.product(x), want)
    w = torch.randn(128, 48, device=DEV).t()
    for zeros in (False, True):
        assert torch.equal(Weight4.from_matrix(w, 64, zeros).product(x), Weight4.from_matrix(w.contiguous(), 64, zeros).product(x))


def test_views_and_steps_of_another_kind_are_refused():
    import dataclasses
    from hos_b200.engine.batch import build_step
    from hos_b200.errors import KernelError
    from hos_b200.parts import attention4
    p = Paged([10, 20], 2, 64)
    rows, q, step = torch.zeros(2, 256, device=DEV, dtype=BF), torch.zeros(2, 256, device=DEV, dtype=BF), p.step([1, 1])
    attention4.store(rows, step, p.view)
    on_host = build_step([[0], [0]], [9, 19], p.slots, torch.device("cpu"), 1)
    for call in (lambda s, v: attention4.store(rows, s, v), lambda s, v: attention4.attend(q, torch.empty_like(q), s, v, 4, 1.0)):
        with pytest.raises(KernelError, match="GPU"):
            call(on_host, p.view)
        for other in (dict(k_pages=p.view.k_pages.cpu()), dict(v_pages=p.view.v_pages.cpu()), dict(page_table=p.view.page_table.cpu()),
                      dict(k_pages=p.view.k_pages.float()), dict(v_pages=p.view.v_pages[:, :1].contiguous()), dict(head_dim=128),
                      dict(page_table=p.view.page_table.long()), dict(k_pages=p.view.k_pages[:, :, ::2]), dict(v_pages=p.view.v_pages[:1])):
            with pytest.raises(KernelError):
                call(step, dataclasses.replace(p.view, four=None, **other))


@pytest.mark.parametrize("keys_only", [False, True])
def test_the_first_copy_of_a_cache_and_the_first_after_a_resize_upload_nothing(monkeypatch, keys_only):
    from hos_b200.cache import CacheManager, kv
    from hos_b200.parts.base import KVNeed
    c = CacheManager([KVNeed(2, 64, None, keys_only)] * 3, [None] * 3, [[]] * 3, 20 * 64, 640, BF, torch.device(DEV))
    g, pairs = c.groups[0], torch.tensor([[0, 3], [1, 7]], dtype=torch.int32, device=DEV)

    def none(*a, **kw):
        raise AssertionError("an upload")
    for pages in (20, 10, 30):
        if pages != 20:
            c.resize(pages * 64)
        arrays = [a for a in g.k + g.v if a is not None]
        assert len(arrays) == (3 if keys_only else 6)
        for a in arrays:
            a.copy_(torch.randn(a.shape))
        want = [a.clone() for a in arrays]
        for a in want:
            a[[1, 7]] = a[[0, 3]]
        with monkeypatch.context() as m:
            m.setattr(kv.torch, "tensor", none)
            g.copy_pages(pairs[0], pairs[1])
        assert all(torch.equal(a, b) for a, b in zip(arrays, want))


@pytest.mark.parametrize("most", [1, 40000, 1 << 30])
def test_shares_within_the_workspace_give_the_same(monkeypatch, most):
    from hos_b200.parts import attention4
    monkeypatch.setattr(attention4, "MOST_PARTS", most)
    check_attention([3000, 2500, 100], [9, 1, 1], 8, 4, 64, dtype=F32)
    check_attention([5000] * 3, [1] * 3, 4, 4, 128, window=3000)


@pytest.mark.parametrize("new", [1, 3])
@pytest.mark.parametrize("heads", [1, 3, 0])
def test_heads_that_are_no_multiple_of_the_kv_heads_are_refused(heads, new):
    from hos_b200.errors import KernelError
    from hos_b200.parts import attention4
    p = Paged([10, 20], 2, 64)
    q = torch.zeros(2 * new, heads * 64, device=DEV, dtype=BF)
    with pytest.raises(KernelError, match="heads"):
        attention4.attend(q, torch.empty_like(q), p.step([new, new]), p.view, heads, 1.0)
