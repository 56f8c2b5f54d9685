"""Attention over pages that sequences share, against the formula in 64 bits on what each sequence holds (bound: shared_cases.share_bound)."""
import random

import pytest
import torch
from shared_cases import Tree, share_bound

from hos_b200.errors import KernelError
from hos_b200.parts import shared_attention as sa

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True, params=["as estimated", "never alone"])
def merged(request, monkeypatch):
    """Short sequences are an item each, without a merge, where the estimate says so; all of these tests run with that ruled out too."""
    if request.param == "never alone":
        monkeypatch.setattr(sa, "MERGE_US", -1e9)
    return request.param


def compare(t, which, news, heads, cap=0.0, scale=None, plan=None, q=None, out=None):
    step = t.step(which, news)
    plan = plan or sa.plan(t.group, step)
    scale = scale if scale is not None else t.dim ** -0.5
    if q is None:
        q = torch.randn(sum(news), heads * t.dim, generator=t.gen).to(torch.bfloat16).to(t.dev)
    out = out if out is not None else torch.full(q.shape, 7.0, dtype=q.dtype, device=t.dev)
    sa.attend(q, out, step, t.view, plan, heads, scale, cap, t.window)
    got = out.double().cpu()
    want = t.exact(q, which, news, heads, scale, cap, t.window)
    keep = t.v
    t.v = [v.abs() for v in keep]                            # the weighted means of |v|
    bound = share_bound(t.exact(q, which, news, heads, scale, cap, t.window), want)
    t.v = keep
    worst = ((got - want).abs() / bound).max()
    assert worst <= 1, float(worst)
    return plan


@pytest.mark.parametrize("dim,kv,per", [(64, 2, 2), (128, 2, 4), (256, 2, 2), (256, 1, 1), (16, 2, 3), (80, 1, 5), (48, 3, 1), (32, 2, 8), (128, 1, 16), (64, 1, 20),
                                        (192, 1, 2)])
@pytest.mark.parametrize("prefix,forks", [(1, 1), (64, 2), (130, 7), (700, 20)])
def test_forks_of_a_prompt(dim, kv, per, prefix, forks):
    t = Tree(kv, dim, seed=dim + prefix)
    a = t.new(prefix)
    all_ = [a] + t.fork(a, forks)
    for j, i in enumerate(all_):
        t.bring([i], [1 + (17 * j) % 90])
    compare(t, all_, [1] * len(all_), per * kv, cap=50.0 if kv > 1 else 0.0)


@pytest.mark.parametrize("window,chunk", [(70, 1), (200, 1), (200, 64), (1000, 64)])
@pytest.mark.parametrize("dim", [64, 256])
def test_windows_and_rings(window, chunk, dim):
    t = Tree(2, dim, window=window, chunk=chunk, seed=window + chunk)
    a, b = t.new(500), t.new(90)
    fa, fb = t.fork(a, 4), t.fork(b, 2)
    order = fb + [a] + fa + [b]
    for j, i in enumerate(order):
        for _ in range(1 + j % 3):
            t.bring([i], [min(chunk, 1 + 31 * j)])
    compare(t, order, [1] * len(order), 4, cap=30.0)


@pytest.mark.parametrize("dim,per", [(64, 2), (128, 4), (256, 2), (80, 3)])
@pytest.mark.parametrize("window", [None, 150])
@pytest.mark.parametrize("news", [(2, 2, 2, 2), (37, 37, 37, 37), (1, 64, 3, 20)])
def test_pieces_of_several_rows(dim, per, window, news):
    t = Tree(2, dim, window=window, chunk=64, seed=dim)
    a = t.new(333)
    all_ = [a] + t.fork(a, 3)
    t.bring(all_, list(news))
    compare(t, all_, list(news), 2 * per, cap=50.0)


@pytest.mark.parametrize("dim,kv,per,forks", [(64, 2, 1, 63), (64, 1, 8, 40), (128, 2, 2, 63), (128, 1, 5, 30), (256, 2, 2, 63), (256, 1, 16, 20), (64, 1, 100, 3), (128, 1, 128, 2)])
@pytest.mark.parametrize("prefix,cap", [(1, 0.0), (700, 50.0), (1500, 0.0)])
def test_many_forks(dim, kv, per, forks, prefix, cap, merged):
    t = Tree(kv, dim, seed=forks + prefix)
    a = t.new(prefix)
    all_ = [a] + t.fork(a, forks)
    for j, i in enumerate(all_):
        t.bring([i], [1 + (37 * j) % 130])
    plan = compare(t, all_, [1] * len(all_), per * kv, cap=cap)
    assert prefix < 64 or merged == "as estimated" or plan.work(per * kv).fields.big_most > 0


@pytest.mark.parametrize("dim", [64, 128, 256])
def test_windows_of_many_rows_cut_pages_at_both_ends(dim):
    t = Tree(2, dim, window=150, chunk=64, seed=dim)
    a = t.new(310)
    all_ = [a] + t.fork(a, 39)
    for j, i in enumerate(all_):
        for _ in range(1 + j % 4):
            t.bring([i], [1 + (13 * j) % 50])
    compare(t, all_, [1] * 40, 8, cap=50.0)


def test_a_tree_of_forks_in_no_order_with_strangers():
    t = Tree(2, 128, seed=9)
    a, x = t.new(300), t.new(77)
    b, = t.fork(a)
    t.bring([a], [200]), t.bring([b], [130])
    fa, fb = t.fork(a, 3), t.fork(b, 5)
    order = [x, a, b] + fa + fb
    random.Random(3).shuffle(order)
    for i in order:
        t.bring([i], [5])
    compare(t, order, [1] * len(order), 8)


def test_sequences_that_share_nothing():
    t = Tree(2, 64, seed=4)
    order = [t.new(n) for n in (1, 64, 200, 1000)]
    plan = compare(t, order, [1] * 4, 4)
    assert plan.runs == []


def test_long_sequences_are_cut():
    t = Tree(1, 64, seed=5, max_seq_len=20000, pages=800)
    a = t.new(16000)
    all_ = [a] + t.fork(a, 2)
    t.bring(all_, [900, 1, 64])
    plan = compare(t, all_, [1, 1, 1], 2)
    assert plan.work(2).parts > 40


def test_scores_far_apart_and_a_steep_scale():
    t = Tree(2, 128, seed=6)
    a = t.new(400)
    all_ = [a] + t.fork(a, 5)
    t.bring(all_, [3] * 6)
    compare(t, all_, [1] * 6, 4, cap=8.0, scale=1.0)
    # one key far above the others
    q = torch.zeros(6, 4 * 128)
    q[:, ::128] = 8.0
    compare(t, all_, [1] * 6, 4, scale=0.125, q=q.to(torch.bfloat16).cuda())


def test_rows_apart_another_stream_and_a_replayed_graph():
    t = Tree(2, 64, seed=7)
    a = t.new(500)
    all_ = [a] + t.fork(a, 9)
    t.bring(all_, [20 + 7 * i for i in range(10)])
    big = torch.randn(10, 3 * 256, generator=t.gen).to(torch.bfloat16).cuda()
    q, out = big[:, 256:512], torch.zeros(10, 600, dtype=torch.bfloat16, device="cuda")
    plan = compare(t, all_, [1] * 10, 4, q=q, out=out[:, 8:264])
    assert not out[:, :8].any() and not out[:, 264:].any()
    step = t.step(all_, [1] * 10)
    first = out[:, 8:264].clone()
    side = torch.cuda.Stream()
    other = torch.zeros_like(first)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        sa.attend(q, other, step, t.view, plan, 4, 0.125)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(other, first)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        sa.attend(q, other, step, t.view, plan, 4, 0.125)
    q.copy_(torch.randn(10, 256, generator=t.gen))
    graph.replay()
    second = other.clone()
    compare(t, all_, [1] * 10, 4, q=q.contiguous(), out=other)
    assert torch.equal(second, other) and not torch.equal(second, first)


def test_refusals():
    t = Tree(2, 64)
    a = t.new(70)
    f, = t.fork(a)
    t.bring([a, f], [1, 1])
    step, q = t.step([a, f], [1, 1]), torch.zeros(2, 256, dtype=torch.bfloat16, device="cuda")
    plan = sa.plan(t.group, step)
    for bad in (dict(q=q.float()), dict(q=q[:1]), dict(n_heads=3), dict(n_heads=2), dict(out=q[:, :128]), dict(window=64), dict(out=q.float()), dict(n_heads=0), dict(scale=0.0), dict(scale=-1.0)):
        k = dict(dict(q=q, out=q.clone(), n_heads=4, window=None, scale=1.0), **bad)
        with pytest.raises(KernelError):
            sa.attend(k["q"], k["out"], step, t.view, plan, k["n_heads"], k["scale"], 0.0, k["window"])
    with pytest.raises(KernelError, match="16 bytes"):
        sa.attend(torch.zeros(2, 257, dtype=torch.bfloat16, device="cuda")[:, 1:], q.clone(), step, t.view, plan, 4, 1.0)
    t.bring([f], [64])
    with pytest.raises(KernelError, match="changed"):
        sa.attend(q, q.clone(), step, t.view, plan, 4, 1.0)


@pytest.mark.parametrize("dim,per,forks,news,window", [(64, 2, 3, 1, None), (64, 2, 3, 1, 100), (128, 2, 40, 1, None), (256, 2, 40, 1, 70), (128, 4, 2, 37, 90), (80, 3, 6, 5, 100),
                                                       (64, 2, 70, 1, 130), (64, 2, 3, 1, 5), (128, 2, 40, 1, 3)])
def test_what_no_row_sees_may_be_anything(dim, per, forks, news, window):
    """NaN and infinities in the pages behind every sequence's last token, before its window, and in the pages that nothing holds: the
    outputs are the same to the bit."""
    t = Tree(2, dim, window=window, seed=dim, chunk=64, slots=80)
    a = t.new(300)
    all_ = [a] + t.fork(a, forks)
    for j, i in enumerate(all_):
        t.bring([i], [news + j % 5])
    step = t.step(all_, [news] * len(all_))
    q = torch.randn(news * len(all_), 2 * per * dim, generator=t.gen).to(torch.bfloat16).cuda()
    outs = []                                                # (a window of 3 or 5: less than the 16 keys of a warp)
    for poison in (None, float("nan"), float("inf"), float("-inf")):
        if poison is not None:
            seen = torch.zeros(t.group.k[0].shape[0], 64, dtype=torch.bool)         # (page, place)
            for i in all_:
                n = len(t.k[i])
                for pos in range(max(0, n - news + 1 - window) if window else 0, n):
                    entry = pos // 64 % t.group.ring_pages if t.group.ring_pages else pos // 64
                    seen[int(t.group.table_host[t.slots[i], entry]), pos % 64] = True
            for pages in (t.group.k[0], t.group.v[0]):
                rows = pages.view(pages.shape[0], 2, 64, dim)                       # (a token's numbers stay in its row)
                rows.masked_fill_(~seen.cuda()[:, None, :, None], poison)
        out = torch.empty_like(q)
        sa.attend(q, out, step, t.view, sa.plan(t.group, step), 2 * per, dim ** -0.5, 20.0, window)
        outs.append(out)
    assert outs[0].isfinite().all()
    for out in outs[1:]:
        assert torch.equal(out, outs[0])


@pytest.mark.parametrize("dim,forks,cap", [(64, 3, 0.0), (64, 70, 30.0), (128, 70, 0.0), (256, 70, 30.0), (80, 5, 0.0)])
def test_a_nan_that_a_row_sees_is_its_own(dim, forks, cap):
    t = Tree(2, dim, seed=3, slots=80)
    a = t.new(1500)
    all_ = [a] + t.fork(a, forks)
    t.bring(all_, [3] * len(all_))
    step = t.step(all_, [1] * len(all_))
    plan = sa.plan(t.group, step)
    q = torch.randn(len(all_), 4 * dim, generator=t.gen).to(torch.bfloat16).cuda()
    out, bad = torch.empty_like(q), torch.empty_like(q)
    sa.attend(q, out, step, t.view, plan, 4, dim ** -0.5, cap, None)
    q[1, dim + 3] = float("nan")
    q[2] = float("nan")
    sa.attend(q, bad, step, t.view, plan, 4, dim ** -0.5, cap, None)
    hit = torch.zeros_like(q, dtype=torch.bool)
    hit[1, dim:2 * dim] = True
    hit[2] = True
    assert bad[hit].isnan().all() and torch.equal(bad[~hit], out[~hit])
    place = int(t.group.table_host[t.slots[all_[3]], 1502 // 64])                   # the last sequence's own page but one
    t.group.v[0].view(-1, 2, 64, dim)[place, 1, 1502 % 64] = float("nan")           # a value of kv head 1 of one sequence alone
    sa.attend(q, bad, step, t.view, plan, 4, dim ** -0.5, cap, None)
    hit[3, 2 * dim:] = True
    assert bad[hit].isnan().all() and torch.equal(bad[~hit], out[~hit])


def test_steps_that_are_not_the_plans_are_refused():
    from hos_b200.engine.batch import build_step
    t = Tree(2, 64, seed=4)
    a = t.new(200)
    f, = t.fork(a)
    t.bring([a, f], [5, 5])
    plan = sa.plan(t.group, t.step([a, f], [2, 2]))
    q = torch.randn(4, 256, generator=t.gen).to(torch.bfloat16).cuda()
    for which, news in (([f, a], [2, 2]), ([a, f], [1, 3])):
        with pytest.raises(KernelError, match="those of the plan"):
            sa.attend(q, q.clone(), t.step(which, news), t.view, plan, 4, 1.0)
    slots = [t.slots[a], t.slots[f]]
    with pytest.raises(KernelError, match="before the end"):
        sa.attend(q, q.clone(), build_step([[0] * 2] * 2, [203, 100], slots, t.dev, 1), t.view, plan, 4, 1.0)
    earlier = build_step([[0] * 2] * 2, [201, 202], slots, t.dev, 1)                # before the plan's, behind what is shared: 192 tokens
    out = torch.empty_like(q)
    sa.attend(q, out, earlier, t.view, plan, 4, 64 ** -0.5)
    t.k, t.v = ([x[i][:n] for i, n in ((a, 203), (f, 204))] for x in (t.k, t.v))
    want = t.exact(q, [0, 1], [2, 2], 4, 64 ** -0.5, 0.0, None)
    t.v = [v.abs() for v in t.v]
    assert ((out.double().cpu() - want).abs() <= share_bound(t.exact(q, [0, 1], [2, 2], 4, 64 ** -0.5, 0.0, None), want)).all()


def test_short_sequences_need_no_merge(merged):
    t = Tree(4, 256, seed=2)
    a = t.new(130)
    all_ = [a] + t.fork(a)
    t.bring(all_, [9, 5])
    plan = compare(t, all_, [1, 1], 8, cap=50.0)
    assert plan.work(8).fields.direct == (merged == "as estimated") and bool(plan.work(8).floats) == (merged != "as estimated")
    many = t.fork(t.new(1200), 3)                            # forked, nothing brought yet: rows in a page that all share
    with pytest.raises(KernelError, match="flush"):
        sa.plan(t.group, t.step(many, [1, 1, 1]))
    t.cache.flush()
    assert compare(t, many + all_, [1] * 5, 8).work(8).fields.direct == 0
