"""Every kernel and cut that the 4-bit operators choose among by sizes, at sizes where another would be chosen: results have to be right
whichever runs.  Tolerances are those of test_fourbit_gpu.py and test_fourbit_ranges_gpu.py, which know nothing of the choice."""
import math

import pytest
import torch

import test_fourbit_ranges_gpu as ranges
from test_fourbit_gpu import Paged, check_attention, check_product, gen

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, F32 = torch.bfloat16, torch.float32


@pytest.fixture(params=["tiles", "few rows"])
def kernel(request, monkeypatch):
    from hos_b200.parts import attention4
    asked = []

    def choose(*args):
        asked.append(args)
        return request.param == "tiles"
    monkeypatch.setattr(attention4, "tiles_are_faster", choose)
    yield request.param
    assert asked                                   # the choice was the two kernels'


@pytest.mark.parametrize("lens,news,window", [([40], [40], None), ([5, 300], [5, 7], None), ([100, 90, 300, 301], [100, 30, 64, 129], None),
                                              ([500, 260], [200, 100], 130), ([1000], [2], None), ([129, 130, 5], [20, 3, 1], 64)])
def test_pieces(kernel, lens, news, window):
    check_attention(lens, news, 4, 2, 128, window=window, dtype=BF, chunk=256)
    check_attention(lens, news, 6, 1, 64, window=window, cap=9.0, dtype=BF, chunk=256)
    check_attention(lens, news, 8, 4, 256, window=window, cap=50.0, dtype=BF, chunk=256)


def test_long_pieces(kernel):
    check_attention([1500, 640], [739, 600], 8, 4, 256, cap=50.0, chunk=1024)
    check_attention([1500], [333], 4, 2, 128, window=400, chunk=512)
    check_attention([4000], [60], 2, 2, 192)


def test_padding_behind_pieces(kernel):
    check_attention([90, 70], [50, 20], 4, 2, 128, pad=3)
    check_attention([9, 90, 70], [9, 3, 2], 8, 1, 256, pad=1)


@pytest.mark.parametrize("order", ["rising", "falling", "jumps", "tiny"])
def test_values_far_apart(kernel, order):
    ranges.test_values_far_apart_in_size(60, order)


def test_odd_heads(kernel):
    for heads, kv, dim, new in ((6, 2, 64, 40), (5, 1, 128, 30), (48, 2, 64, 9), (24, 1, 256, 7), (40, 1, 128, 3)):
        check_attention([300, 100 + new], [new, new], heads, kv, dim, cap=20.0)


def test_two_shares_as_a_cluster_and_through_the_workspace_agree_in_size():
    """Both merges of the same shares differ by the rounding of the result alone."""
    from hos_b200.parts import attention4
    p, lens = Paged([700, 650], 2, 128), [700, 650]
    rows = torch.randn(sum(lens), 512, generator=gen(2)).to(BF).to(DEV)
    attention4.store(rows, p.step(lens, starts=[0, 0]), p.view)
    q, got = torch.randn(2, 1024, generator=gen(3)).to(BF).to(DEV), []
    before = attention4.shares
    try:
        for cluster in (True, False):
            attention4.shares = lambda *a: (6, 2, cluster)
            out = torch.empty_like(q)
            attention4.attend(q, out, p.step([1, 1]), p.view, 8, 128 ** -0.5)
            got.append(out.double())
    finally:
        attention4.shares = before
    assert float((got[0] - got[1]).abs().max()) <= 2.0 ** -7 * float(got[0].abs().max())


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("share,cluster", [(9, True), (4, True), (2, False), (3, False), (5, False), (1, False), (8, False)])
def test_shares_of_single_tokens(monkeypatch, share, cluster, dtype):
    """17 pages in up to 17 shares: a cluster, one thread a number, four, of which some have a share fewer or none."""
    from hos_b200.parts import attention4
    monkeypatch.setattr(attention4, "shares", lambda *a: (share, -(-17 // share), cluster))
    for heads, kv, dim in ((8, 4, 256), (9, 3, 64)):
        check_attention([1, 1088, 900, 64, 65], [1] * 5, heads, kv, dim, cap=30.0, dtype=dtype)


@pytest.mark.parametrize("share", [1, 2, 3, 8])
def test_shares_of_pieces(monkeypatch, share):
    from hos_b200.parts import attention4
    monkeypatch.setattr(attention4, "tile_shares", lambda *a: (share, -(-17 // share)))
    monkeypatch.setattr(attention4, "tiles_are_faster", lambda *a: True)
    check_attention([300, 1088, 70], [300, 70, 3], 4, 2, 128, cap=30.0)


@pytest.mark.parametrize("kv,dim,dtype", [(16, 128, BF), (12, 256, F32)])
def test_rows_of_many_heads_are_stored_as_few_rows_are(kv, dim, dtype):
    from hos_b200.engine.batch import build_step
    from hos_b200.parts import attention4
    lens = [1, 63, 64, 65, 500, 16, 129]
    rows = torch.randn(sum(lens), 2 * kv * dim, generator=gen(8)).to(dtype).to(DEV)
    a, b = Paged(lens, kv, dim, dtype=dtype), Paged(lens, kv, dim, dtype=dtype)
    held = torch.empty_like(rows)
    attention4.store(rows, a.step(lens), a.view, held)
    base = [sum(lens[:i]) for i in range(len(lens))]
    for at in range(0, 500, 37):
        live = [i for i, n in enumerate(lens) if n > at]
        news = [min(37, lens[i] - at) for i in live]
        step = build_step([[0] * n for n in news], [at] * len(live), [b.slots[i] for i in live], torch.device(DEV), 1)
        part = torch.cat([rows[base[i] + at:base[i] + at + n] for i, n in zip(live, news)])
        some = torch.empty_like(part)
        attention4.store(part, step, b.view, some)
        assert torch.equal(some, torch.cat([held[base[i] + at:base[i] + at + n] for i, n in zip(live, news)]))
    assert torch.equal(a.c.groups[0].k[0], b.c.groups[0].k[0]) and torch.equal(a.c.groups[0].v[0], b.c.groups[0].v[0])


@pytest.mark.parametrize("m", [16, 17, 24, 32, 33])
@pytest.mark.parametrize("n,k,gated", [(8200, 4100, False), (4104, 4160, True)])
def test_products_of_many_weights(m, n, k, gated):
    check_product(m, n, k, 64, True, gated, BF)
