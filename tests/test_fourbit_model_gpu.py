"""The engine with a 4-bit cache against the engine whose cache holds 32-bit numbers, which are what the 4-bit cache would hold: the
rotation, the scale, the window, the soft-cap and the pages are then the other attention's, and the rounding the definition's."""
import pytest
import torch

from test_fourbit_engine_gpu import engine, ids
from test_fourbit_gpu import held_of

pytestmark = pytest.mark.gpu


def holds_rounded(eng, monkeypatch):
    """Keys and values of this (32-bit) engine become what 4 bits hold of them before they are stored and attended over."""
    from hos_b200 import ops
    eng.runner.use_sessions = False
    real = ops.rope_kv_write

    def rope_kv_write(qkv, n_heads, pos, seq, slot, after, inv_freq, rotary_dim, style, cache, n_kv, head_dim, partials=None):
        if cache is None or cache.bits is not None:
            return real(qkv, n_heads, pos, seq, slot, after, inv_freq, rotary_dim, style, cache, n_kv, head_dim, partials=partials)
        real(qkv, n_heads, pos, seq, slot, after, inv_freq, rotary_dim, style, None, n_kv, head_dim, partials=partials)
        qkv[:, n_heads * head_dim:] = held_of(qkv[:, n_heads * head_dim:]).to(qkv.device)
        real(qkv, n_heads, pos, seq, slot, after, None, 0, style, cache, n_kv, head_dim)          # as they are, into the pages
    monkeypatch.setattr(ops, "rope_kv_write", rope_kv_write)


def logits_of(eng):
    """Prompts whole, a piece on top, single tokens, and two sequences that go on by unlike numbers of tokens."""
    r, p, out = eng.runner, ids(170, 11), []
    a, b = r.admit(2)
    out.append(r.step([a, b], [p[:130], p[100:109]], [[0, 60, 129], [8]]))
    out.append(r.step([a], [p[130:160]], [[0, 29]]))
    for t in p[160:164]:
        out.append(r.step([a, b], [[t], [t]]))
    out.append(r.step([b, a], [p[20:90], p[164:167]], [[0, 69], [2]]))
    return torch.cat(out)


def test_a_cache_in_four_bits_is_a_cache_of_what_four_bits_hold(monkeypatch):
    got = logits_of(engine("float32", cache_bits=4))
    full = engine("float32")
    unrounded = logits_of(full)
    full = engine("float32")
    holds_rounded(full, monkeypatch)
    want = logits_of(full)
    size = float(want.abs().max())
    assert float((unrounded - want).abs().max()) > 0.05 * size          # the rounding is there to be seen
    assert float((got - want).abs().max()) < 0.002 * size               # a code that falls to the other side here or there
