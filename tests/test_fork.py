"""Sequences that share pages, on the host (no GPU): forks, copies before writes, compaction, other sizes, freeing."""
import random

import pytest
import torch

from hos_b200.cache import CacheManager
from hos_b200.errors import CacheError
from hos_b200.parts.base import KVNeed, StateNeed

CPU = torch.device("cpu")


def make(max_tokens=1024, window=100, max_seq_len=512, entries=2, bits=None, **kw):
    needs = [KVNeed(2, 64, window if i % 2 == 0 else None, bits=bits) for i in range(entries)]
    states = [[StateNeed("s", (3,))] for _ in needs]
    return CacheManager(needs, [None] * entries, states, max_tokens, max_seq_len, torch.float32, CPU, **kw)


def write(c, slot, lo, hi, value):
    """What a step does: pages first, then numbers at the positions (here one number a position and group)."""
    c.extend(slot, hi)
    c.flush()
    for g in c.groups:
        for p in range(lo, hi):
            e = p // 64 % g.ring_pages if g.ring_pages else p // 64
            g.k[0][int(g.table_dev[slot, e]), :, p % 64] = value + p


def read(c, slot, g, p):
    e = p // 64 % g.ring_pages if g.ring_pages else p // 64
    return float(g.k[0][int(g.table_dev[slot, e]), 0, p % 64, 0])


def test_a_fork_shares_pages_until_one_of_them_writes():
    c = make()
    a = c.admit([0])[0]
    write(c, a, 0, 150, 1000)
    held = [g.pages.n_held for g in c.groups]
    c.stores[0].state["s"][a] = torch.tensor([1.0, 2.0, 3.0])
    c.record[a, 0] = 150
    b, d = c.fork(a, 2)
    c.check()
    assert c.lengths[b] == c.lengths[d] == 150 and int(c.record[b, 0]) == 150
    assert c.stores[0].state["s"][d].tolist() == [1.0, 2.0, 3.0]
    assert [g.pages.n_held for g in c.groups] == held
    write(c, b, 150, 151, 2000)                          # the last page, in both groups, and nothing else
    c.check()
    assert [g.pages.n_held for g in c.groups] == [h + 1 for h in held]
    full = [g for g in c.groups if not g.ring_pages][0]
    for s in (a, b, d):
        assert read(c, s, full, 149) == 1149 and read(c, s, full, 10) == 1010
    assert read(c, b, full, 150) == 2150 and read(c, a, full, 150) == 0
    write(c, a, 150, 151, 3000)
    write(c, d, 150, 151, 4000)                          # the last holder keeps the page
    c.check()
    assert [g.pages.n_held for g in c.groups] == [h + 2 for h in held]
    assert [read(c, s, full, 150) for s in (a, b, d)] == [3150, 2150, 4150]
    for s in (a, b, d):
        c.release(s)
    c.check()
    assert all(g.pages.n_held == 0 for g in c.groups)


def test_a_ring_that_is_written_round_keeps_the_others_keys():
    c = make(window=100, chunk_tokens=1)
    ring = [g for g in c.groups if g.ring_pages][0]
    assert ring.ring_pages == 2
    a = c.admit([0])[0]
    write(c, a, 0, 130, 0)                               # positions 128, 129 lie in the first page of the ring again
    b = c.fork(a)[0]
    write(c, b, 130, 260, 5000)
    c.check()
    for p in list(range(66, 128)) + [128, 129]:
        assert read(c, a, ring, p) == p
    assert read(c, b, ring, 259) == 5259 and read(c, b, ring, 192) == 5192


def test_a_step_of_forks_takes_what_it_needs_and_no_more():
    c = make(max_tokens=256, window=None, max_seq_len=256)
    g = c.groups[0]
    a = c.admit([0])[0]
    write(c, a, 0, 100, 0)
    b, d = c.fork(a, 2)
    assert g.pages.n_free == 2                           # 2 held, 2 copies for three writers: exactly enough
    c.extend_all([a, b, d], [101, 101, 101])
    c.check()
    assert g.pages.n_free == 0
    e = c.fork(a)[0]
    with pytest.raises(CacheError, match="no free"):
        c.extend_all([a, e], [102, 102])
    assert c.lengths[a] == c.lengths[e] == 101
    c.check()


def test_a_length_that_was_set_back_is_written_again_in_a_page_of_its_own():
    c = make(window=None)
    a = c.admit([0])[0]
    write(c, a, 0, 70, 0)
    c.lengths[a] = 66
    b = c.fork(a)[0]
    write(c, a, 66, 67, 900)
    write(c, b, 66, 67, 800)
    g = c.groups[0]
    assert read(c, a, g, 66) == 966 and read(c, b, g, 66) == 866 and read(c, b, g, 65) == 65


def test_compaction_moves_pages_and_a_smaller_cache_keeps_them():
    c = make(max_tokens=1024, window=None, max_seq_len=512)
    g = c.groups[0]
    s = c.admit([0, 0, 0])
    for i, slot in enumerate(s):
        write(c, slot, 0, 200, 1000 * i)
    f = c.fork(s[2])[0]
    c.release(s[0])
    c.compact()
    c.check()
    c.flush()
    assert g.pages.held() == set(range(8))
    for p in range(200):
        assert read(c, s[1], g, p) == 1000 + p and read(c, s[2], g, p) == 2000 + p and read(c, f, g, p) == 2000 + p
    with pytest.raises(CacheError, match="do not fit"):
        c.resize(7 * 64)
    c.resize(8 * 64)
    c.check()
    assert g.k[0].shape[0] == 8 and c.stores[0].kv.k_pages is g.k[0] and c.tokens_capacity() == 512 and g.pages.n_free == 0
    c.resize(1024)
    c.check()
    assert g.pages.n_free == 8 and read(c, f, g, 199) == 2199
    for p in range(200):
        assert read(c, s[1], g, p) == 1000 + p


def test_refusals():
    c = make()
    with pytest.raises(CacheError, match="holds no sequence"):
        c.fork(3)
    a = c.admit([0])[0]
    with pytest.raises(CacheError, match="free slots"):
        c.fork(a, c.n_slots)
    with pytest.raises(CacheError, match="at least one"):
        c.resize(0)
    for need in (KVNeed(2, 48, None, bits=4), KVNeed(2, 64, None, bits=8), KVNeed(2, 64, None, True, bits=4), KVNeed(2, 320, None, bits=4),
                 KVNeed(2, 64, None, False, 128, bits=4)):
        with pytest.raises(CacheError, match="bits"):
            CacheManager([need], [None], [[]], 256, 256, torch.float32, CPU)


def test_four_bit_pages_are_small_and_fork_too():
    c = make(bits=4)
    assert c.groups[0].k[0].dtype == torch.uint8 and c.groups[0].k[0].shape[1:] == (2, 36 * 64)
    assert c.bytes_per_token() == 2 * 2 * 2 * 36                   # groups x (keys, values) x heads x bytes a head
    a = c.admit([0])[0]
    c.extend(a, 10)
    c.groups[0].k[0][int(c.groups[0].table_host[a, 0])] = 7
    b = c.fork(a)[0]
    c.extend(b, 11)
    c.check()
    assert int(c.groups[0].k[0][int(c.groups[0].table_host[b, 0])].min()) == 7


def test_random_life():
    rng = random.Random(5)
    c = make(max_tokens=2048, window=130, max_seq_len=512, max_slots=12)
    want = {}
    for _ in range(400):
        act = rng.random()
        live = list(want)
        try:
            if act < 0.25 or not live:
                s = c.admit([0])[0]
                want[s] = {}
            elif act < 0.5:
                s = rng.choice(live)
                lo = c.lengths[s]
                hi = min(512, lo + rng.choice([1, 1, 3, 40, 100]))
                if hi > lo:
                    base = rng.randrange(1 << 16)
                    write(c, s, lo, hi, base)
                    want[s].update({p: float(base + p) for p in range(lo, hi)})
            elif act < 0.7:
                s = rng.choice(live)
                want[c.fork(s)[0]] = dict(want[s])
            elif act < 0.85:
                s = rng.choice(live)
                c.release(s)
                del want[s]
            elif act < 0.95:
                c.compact()
            else:
                held = max(g.pages.n_held for g in c.groups)
                c.resize(64 * rng.randint(max(1, held), 40))
        except CacheError as e:
            assert "free" in str(e)
        c.flush()
        c.check()
        for s, at in want.items():
            n = c.lengths[s]
            for g in c.groups:
                seen = [p for p in at if p >= n - (g.need.window or n)]
                for p in rng.sample(seen, min(6, len(seen))):
                    assert read(c, s, g, p) == at[p]
