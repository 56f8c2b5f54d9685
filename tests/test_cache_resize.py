"""A cache that is made smaller or larger while sequences live in it, and what is left when that fails (no GPU)."""
import pytest
import torch

from test_fork import make


def full_of(monkeypatch, allowed):
    """torch.zeros that makes `allowed` more page arrays and then has no memory left."""
    from hos_b200.cache import kv
    left, real = [allowed], torch.zeros

    def zeros(shape, *a, **kw):
        if len(shape) > 2:
            left[0] -= 1
            if left[0] < 0:
                raise torch.OutOfMemoryError("no memory left")
        return real(shape, *a, **kw)
    monkeypatch.setattr(kv.torch, "zeros", zeros)


@pytest.mark.parametrize("bits", [None, 4])
@pytest.mark.parametrize("allowed", range(8))
@pytest.mark.parametrize("pages", [4, 40])
def test_a_resize_that_runs_out_of_memory_leaves_a_cache_that_goes_on(monkeypatch, pages, allowed, bits):
    c = make(max_tokens=1024, window=100, max_seq_len=512, entries=4, bits=bits)
    arrays = 8                                           # of keys and of values, of two groups with two entries
    a, gone = c.admit([0, 0])
    c.extend(gone, 70)
    c.extend(a, 70)
    c.release(gone)
    c.flush()
    for g in c.groups:
        for t in g.k + g.v:
            t[torch.tensor(g._slot_pages[a])] = 7
    with monkeypatch.context() as m:
        full_of(m, allowed)
        with pytest.raises(torch.OutOfMemoryError):
            c.resize(pages * 64)
    c.check()
    assert allowed < arrays and c.tokens_capacity() == min(pages, 16) * 64
    owners = [next((g for g in c.groups if any(store.kv.k_pages is k for k in g.k)), None) for store in c.stores]
    for g, store in zip(owners, c.stores):               # the kernels read the arrays that the groups write and copy in
        assert g is not None and any(store.kv.v_pages is v for v in g.v)
        assert all(t.shape[0] >= g.pages.n for t in g.k + g.v)
    b = c.fork(a)[0]
    c.extend(b, 71)                                      # copies the page that it writes into
    c.flush()
    c.check()
    for g, store in zip(owners, c.stores):
        for slot in (a, b):
            for t in (store.kv.k_pages, store.kv.v_pages):
                assert float(t[g.table_dev[slot, :2].long()].float().min()) == 7
    c.resize(pages * 64)                                 # with memory again
    c.check()
    assert c.tokens_capacity() == pages * 64 and all(t.shape[0] == pages for g in c.groups for t in g.k + g.v)


def test_a_resize_takes_one_array_more_at_a_time():
    """The views let go of an old array as soon as the new one stands in its place."""
    import weakref
    c = make(max_tokens=1024, window=None, entries=3)
    g = c.groups[0]
    old, alive, real = [weakref.ref(t) for t in g.k + g.v], [], torch.zeros

    class Watch:
        def __getattr__(self, name):
            return getattr(torch, name)

        def zeros(self, *a, **kw):
            alive.append(sum(r() is not None for r in old))
            return real(*a, **kw)
    from hos_b200.cache import kv
    kv.torch, before = Watch(), kv.torch
    try:
        c.resize(512)
    finally:
        kv.torch = before
    assert alive == [6, 5, 4, 3, 2, 1] and all(r() is None for r in old)


@pytest.mark.parametrize("act", ["write", "compact"])
def test_a_copy_that_fails_takes_no_page(monkeypatch, act):
    c = make(max_tokens=512, window=None, max_seq_len=256)
    g = c.groups[0]
    gone, a = c.admit([0, 0])
    c.extend(gone, 64)
    c.extend(a, 100)
    c.flush()
    for page in g._slot_pages[a]:
        g.k[0][page] = page + 1
    b = c.fork(a)[0]
    c.release(gone)
    want = [float(g.k[0][p].max()) for p in g._slot_pages[a]]

    def fails(src, dst):
        raise RuntimeError("no pinned memory left")
    run = (lambda: c.extend(b, 101)) if act == "write" else c.compact
    with monkeypatch.context() as m:
        m.setattr(g, "_copy_listed", fails)
        with pytest.raises(RuntimeError, match="pinned"):
            run()
    c.check()
    assert c.lengths[b] == 100 and g.pages.n_held == 2
    for slot in (a, b):
        assert [float(g.k[0][p].max()) for p in g._slot_pages[slot]] == want
    run()
    c.check()
    for slot in (a, b):
        assert [float(g.k[0][p].max()) for p in g._slot_pages[slot]] == want
