"""What sequences share, the lists of work that are made of it, and what is refused: without a GPU."""
import random

import numpy as np
import pytest
import torch
from shared_cases import Tree

from hos_b200.errors import KernelError
from hos_b200.parts import shared_attention as sa

PAGE = 64


def tree(**kw):
    return Tree(2, 64, device="cpu", **kw)


def runs(t, which=None, more=1):
    which = list(range(len(t.slots))) if which is None else which
    return t.group.shared_runs([t.slots[i] for i in which], [len(t.k[i]) for i in which])


def test_forks_share_their_whole_pages():
    t = tree()
    a = t.new(200)
    f = t.fork(a, 3)
    t.bring([a] + f, [1, 1, 1, 1])
    assert runs(t) == [([0, 1, 2, 3], 0, 3)]                 # the fourth page was copied when it was written into
    t.bring([a], [100])
    assert runs(t) == [([0, 1, 2, 3], 0, 3)]
    assert runs(t, [2, 0]) == [([0, 1], 0, 3)]
    assert runs(t, [1]) == []


def test_sequences_of_their_own_share_nothing():
    t = tree()
    t.new(100), t.new(100)
    assert runs(t) == []
    a = t.new(500)
    t.fork(a, 1)
    t.bring([2, 3], [1, 1])
    assert runs(t) == [([2, 3], 0, 7)]


def test_of_a_tree_of_forks_the_runs_save_the_most():
    t = tree()
    a = t.new(128)
    b, = t.fork(a)
    t.bring([a], [640]), t.bring([b], [640])
    fa, fb = t.fork(a, 3), t.fork(b, 3)
    order = [a, b] + fa + fb
    t.bring(order, [1] * 8)
    got = runs(t, order)                                     # four and four over 12 pages each, not eight over two
    assert sorted((sorted(order[i] for i in m), lo, hi) for m, lo, hi in got) == sorted([(sorted([a] + fa), 0, 12), (sorted([b] + fb), 0, 12)])
    assert runs(t, [a, b]) == [([0, 1], 0, 2)]


def test_in_a_ring_counts_what_all_still_hold():
    t = tree(window=200, chunk=1)                            # a ring of four pages
    assert t.group.ring_pages == 4
    a = t.new(500)                                           # pages 4 to 7
    f = t.fork(a, 2)
    t.bring([a] + f, [1, 1, 1])
    assert runs(t) == [([0, 1, 2], 4, 7)]
    t.bring([a], [80])                                       # page 9 lies where page 5 did
    assert runs(t) == [([0, 1, 2], 6, 7)]
    assert runs(t, f) == [([0, 1], 4, 7)]
    for _ in range(4):
        t.bring([a], [64])
    assert runs(t) == [([1, 2], 4, 7)] and runs(t, f) == [([0, 1], 4, 7)]       # the first holds nothing of theirs any more


def test_a_plan_ends_when_pages_change():
    t = tree()
    a = t.new(200)
    f, = t.fork(a)
    t.bring([a, f], [1, 1])
    before = t.group.version
    assert t.group.shared_runs(t.slots, [201, 201]) and t.group.version == before
    t.cache.extend(t.slots[a], 257)
    assert t.group.version != before
    before = t.group.version
    t.cache.release(t.slots[f])
    assert t.group.version != before
    before = t.group.version
    t.cache.compact()
    t.cache.fork(t.slots[a])
    assert t.group.version != before


@pytest.mark.parametrize("seed", range(60))
def test_every_key_that_a_row_sees_is_in_one_of_its_items(seed):
    rng = random.Random(seed)
    window = rng.choice([None, None, 70, 200, 300])
    t = tree(window=window, chunk=rng.choice([1, 64]), max_seq_len=1024, slots=24, seed=seed)
    for _ in range(rng.randint(1, 3)):
        t.new(rng.choice([1, 63, 64, 65, rng.randint(1, 400)]))
    for _ in range(rng.randint(1, 4)):
        t.fork(rng.randrange(len(t.slots)), rng.randint(1, 4))
        for i in rng.sample(range(len(t.slots)), rng.randint(1, len(t.slots))):
            t.bring([i], [rng.choice([1, 2, rng.randint(1, 60)])])
    which = rng.sample(range(len(t.slots)), rng.randint(1, len(t.slots)))
    for i in which:
        t.bring([i], [1])
    news = [1 if window and t.group.ring_pages * 64 < window + 64 else min(len(t.k[i]), rng.choice([1, 1, 3, 40, 64])) for i in which]
    order = sorted(range(len(which)), key=lambda i: len(t.k[which[i]]) > news[i])
    which, news = [which[i] for i in order], [news[i] for i in order]
    step = t.step(which, news)
    plan = sa.plan(t.group, step)
    per = rng.choice([1, 2, 3, 5, 16, 20])
    made = sa.lists(plan.runs, plan.rows, plan.slots, plan.lengths, plan.n_rows, per, 2, 64, window, rng.random() < 0.5)
    pos, seq = step.token_pos.tolist(), step.token_seq.tolist()
    seen = [dict() for _ in pos]
    parts = [set() for _ in pos]
    for j, (row0, n_rows, slot, lp0, lp1, skip0, skip1, share, n_shares, part, _, _, *inline) in enumerate(made.items.tolist() + made.big.tolist()):
        rows = made.rows[row0:row0 + n_rows].tolist()
        assert n_rows * per <= 128 if j >= len(made.items) else n_rows * per <= 8 or n_rows == 1
        assert j >= len(made.items) or inline[:n_rows] == rows
        lo = min(max(0, pos[r] + 1 - window) // PAGE if window else 0 for r in rows)
        hi = max(pos[r] // PAGE for r in rows)
        pages = [p for p in range(max(lp0, lo), min(lp1, hi + 1)) if not skip0 <= p < skip1]
        each = -(-len(pages) // n_shares)
        for r in rows:
            assert part not in parts[r]
            parts[r].add(part)
            table = t.group._table_np[slot]
            mine = t.group._table_np[t.slots[which[seq[r]]]]
            for p in pages[share * each:(share + 1) * each]:
                e = p % t.group.ring_pages if t.group.ring_pages else p
                if p * PAGE <= pos[r] and (not window or p * PAGE + PAGE - 1 > pos[r] - window):
                    assert table[e] == mine[e], "another sequence's page"
                    assert p not in seen[r], "a page twice"
                    seen[r][p] = True
    for r, p in enumerate(pos):
        lo = max(0, p + 1 - window) // PAGE if window else 0
        assert sorted(seen[r]) == list(range(lo, p // PAGE + 1))
        assert parts[r] == set(range(int(made.n_parts[r])))


def test_refusals():
    t = tree()
    a = t.new(70)
    f, = t.fork(a)
    t.bring([a, f], [1, 1])
    step = t.step([a, f], [1, 1])
    plan = sa.plan(t.group, step)
    assert plan.runs == [([0, 1], 0, 1)]
    q = torch.zeros(2, 256, dtype=torch.bfloat16)
    with pytest.raises(KernelError, match="on the GPU"):
        sa.attend(q, q.clone(), step, t.view, plan, 4, 1.0)
    step.cu_host = ()
    with pytest.raises(KernelError, match="lists on the host"):
        sa.plan(t.group, step)
    with pytest.raises(KernelError, match="no pages"):
        sa.plan(t.group, t.step([a], [1]).__class__(**{**t.step([a], [1]).__dict__, "starts_host": (500,)}))
    odd = Tree(2, 40, device="cpu")
    odd.new(5)
    with pytest.raises(KernelError, match="multiple of 16"):
        sa.plan(odd.group, odd.step([0], [1]))
    assert not sa.supports(24) and not sa.supports(272) and sa.supports(80)


@pytest.mark.parametrize("small,big,kv", [([1], [], 1), ([125] * 2 + [2] * 8, [], 4), ([6] * 64, [61] * 8, 16), ([], [2000] * 4, 8), ([3] * 200, [], 8),
                                          ([], [46] * 3 + [2] * 5, 4)])
@pytest.mark.parametrize("dim", [16, 64, 128, 256])
def test_shares_leave_no_round_of_big_items_nearly_empty(small, big, kv, dim):
    (n_small, n_big, sms), _ = sa.estimate(np.asarray(small, dtype=np.int64), np.asarray(big, dtype=np.int64), np.asarray([128] * len(big), dtype=np.int64), kv, kv, dim, sum(small) + sum(big))
    assert n_small >= 1 and n_big >= 1 and 1 <= sms <= 148
    items = sum(-(-p // n_big) for p in big) * kv
    assert items <= 148 or len(big) * kv > 148 or items > 2 * 148 - 8 * kv


def test_blocks_of_few_pairs_and_of_many():
    rows = [range(i, i + 1) for i in range(40)]
    made = sa.lists([(list(range(4)), 0, 50), (list(range(8, 40)), 0, 60)], rows, list(range(40)), [4000] * 40, 40, 2, 4, 128, None, True)
    assert sorted({it[1] for it in made.items.tolist()}) == [1, 4] and {it[1] for it in made.big.tolist()} == {32}
    plain = sa.lists([(list(range(40)), 0, 60)], rows, list(range(40)), [4000] * 40, 40, 2, 4, 128, None, False)
    assert len(plain.big) == 0 and max(it[1] for it in plain.items.tolist()) == 4


def test_a_cut_is_kept_while_it_costs_little():
    small, big = np.asarray([3, 1, 4, 1, 5], dtype=np.int64), np.asarray([125], dtype=np.int64)
    pairs = np.asarray([16], dtype=np.int64)
    first, us = sa.estimate(small, big, pairs, 4, 4, 256, 139)
    for more in range(1, 12):
        best, least = sa.estimate(small + more, big, pairs, 4, 4, 256, 139 + 5 * more)
        kept, costs = sa.estimate(small + more, big, pairs, 4, 4, 256, 139 + 5 * more, first)
        assert least <= costs <= 1.1 * least and (kept == best or kept[1] == first[1])
    far, _ = sa.estimate(np.asarray([900], dtype=np.int64), big, pairs, 4, 4, 256, 1025, (sa.OPEN, 2, 20))
    assert far[0] < 900                                      # what costs more is not kept
