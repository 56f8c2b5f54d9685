"""The engine with weights, keys and values in 4 bits, and sequences that are forked: consistent with itself however tokens are
cut into steps, and with a model whose matrices are what the codes stand for."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda"
RAW = dict(architectures=["Gemma2ForCausalLM"], num_hidden_layers=4, hidden_size=128, num_attention_heads=4, num_key_value_heads=2, head_dim=64,
           intermediate_size=320, vocab_size=640, rope_theta=10000.0, sliding_window=48, max_position_embeddings=512, query_pre_attn_scalar=64,
           attn_logit_softcapping=20.0, final_logit_softcapping=15.0, rms_norm_eps=1e-6)


def engine(dtype="bfloat16", seed=3, raw=RAW, **kw):
    from hos_b200 import Engine
    from hos_b200.registry import config_from_dict
    return Engine.from_config(config_from_dict(raw), seed=seed, dtype=dtype, max_batch=6, max_seq_len=512, **kw)


def ids(n, seed):
    return torch.randint(0, 640, (n,), generator=torch.Generator().manual_seed(seed)).tolist()


@pytest.mark.parametrize("dtype,tol", [("float32", 0.01), ("bfloat16", 0.1)])
def test_the_cut_into_steps_does_not_matter(dtype, tol):
    """A prompt whole, in pieces, and token by token: roundings differ, and with them here and there a code by one (a third of a
    key's spread, in one number of some thousand): in bfloat16, whose roundings are 1/50 of a code, in one number of a hundred."""
    eng = engine(dtype, weight_bits=4, cache_bits=4)
    r, p = eng.runner, ids(150, 1)
    a, b, c = r.admit(3)
    whole = r.step([a], [p], [[149]])
    for lo in range(0, 150, 37):
        pieces = r.step([b], [p[lo:lo + 37]])
    r.step([c], [p[:100]])
    for t in p[100:]:
        single = r.step([c], [[t]])
    size = float(whole.abs().max())
    assert float((whole - pieces).abs().max()) < tol * size and float((whole - single).abs().max()) < tol * size


def test_weights_in_four_bits_are_the_matrix_that_the_codes_stand_for():
    eng, full = engine("float32", weight_bits=4), engine("float32")
    from hos_b200.parts.weights4 import Weight4
    for mine, other in zip(eng.runner.model.layers, full.runner.model.layers):
        for part, names in (("mixer", ("w_qkv", "w_o")), ("feed_forward", ("w_gate_up", "w_down"))):
            for name in names:
                w4, w = getattr(getattr(mine, part), name), getattr(getattr(other, part), name)
                assert isinstance(w4, Weight4) and w4.shape == w.shape and w4.nbytes() < 0.2 * w.numel() * 4
                again = Weight4(w4.codes, w4.records, w4.n, w4.k, w4.group, 1, w4.zeros)           # gate and up one after the other
                if w4.blocks == 2:
                    half = w4.codes.shape[0] // 2
                    again = [Weight4(w4.codes[i * half:(i + 1) * half], w4.records[i * half:(i + 1) * half], w4.n, w4.k, w4.group, 1, w4.zeros) for i in (0, 1)]
                    back = torch.cat([g.product(torch.eye(w4.k, device=DEV)).T for g in again])
                else:
                    back = again.product(torch.eye(w4.k, device=DEV)).T
                w.copy_(back)
                if name == "w_qkv":
                    getattr(other, part).w_q = w[: getattr(other, part).q_dim]
    p = [ids(70, 2), ids(9, 3)]
    assert eng.generate_ids(p, 12, stop_ids=[]) == full.generate_ids(p, 12, stop_ids=[])
    x, y = (e.runner.step(e.runner.admit(2), p) for e in (eng, full))
    assert float((x - y).abs().max()) < 1e-4


@pytest.mark.parametrize("how", [dict(), dict(cache_bits=4), dict(weight_bits=4, cache_bits=4)])
@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
def test_forks_go_on_as_sequences_of_their_own_would(how, dtype):
    eng = engine(dtype, **how)
    p = ids(130, 4)
    first, = eng.open(1)
    eng.generate_from_ids([first], [p], max_tokens=5, stop_ids=[])
    alone = eng.open(3)
    for c in alone:                                       # each as the first was run, so that the same numbers are in its pages
        eng.generate_from_ids([c], [p], max_tokens=5, stop_ids=[])
    forks = [first] + first.fork(2)
    eng.runner.cache.check()
    turns = [ids(3, 5), ids(20, 6), [9]]
    got = eng.generate_from_ids(forks, turns, max_tokens=70, temp=0.7, seed=7, stop_ids=[])
    want = eng.generate_from_ids(alone, turns, max_tokens=70, temp=0.7, seed=7, stop_ids=[])
    eng.runner.cache.check()
    assert got == want
    for c in forks[1:] + alone:
        c.close()
    eng.runner.resize_cache(first.position + 64)
    eng.runner.cache.check()
    assert len(eng.generate_from_ids([first], [[5]], max_tokens=8, stop_ids=[])[0]) == 8


def test_a_resized_cache_goes_on_where_it_was():
    for how in (dict(), dict(cache_bits=4)):
        eng = engine("float32", **how)
        a, b = eng.open(2)
        p = [ids(100, 8), ids(40, 9)]
        eng.generate_from_ids([a, b], p, max_tokens=4, stop_ids=[])
        c, d = eng.open(2)
        eng.generate_from_ids([c, d], p, max_tokens=4, stop_ids=[])
        want = eng.generate_from_ids([c, d], [[1], [2]], max_tokens=20, stop_ids=[])
        c.close(), d.close()
        eng.runner.resize_cache(320)
        assert eng.generate_from_ids([a, b], [[1], [2]], max_tokens=20, stop_ids=[]) == want


def test_models_that_cannot_are_refused():
    from hos_b200 import HosError
    with pytest.raises(HosError, match="weight_bits"):
        engine(weight_bits=8)
    with pytest.raises(HosError, match="cache_bits"):
        engine(cache_bits=2)
    with pytest.raises(HosError, match="bits"):
        engine(cache_bits=4, raw=dict(RAW, head_dim=32))


def test_the_example_runs(tmp_path, capsys):
    import importlib.util
    import json
    import os
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "several_answers.py")
    spec = importlib.util.spec_from_file_location("several_answers", path)
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    cfg = tmp_path / "config.json"
    cfg.write_text(json.dumps(RAW))
    assert mod.main(["--random", str(cfg), "-p", "2,5,9,11", "--answers", "3", "-n", "6", "--max-seq-len", "256"]) == 0
    lines = capsys.readouterr().out.strip().splitlines()
    assert len(lines) == 3 and len(set(lines)) > 1


def test_prompts_over_their_own_rows_take_the_kernel_for_them(monkeypatch):
    """A prompt attends over its own rows, which are bfloat16 whatever the pages hold: not the plain kernel's business."""
    from hos_b200 import ops

    def plain(*a, **kw):
        raise AssertionError("the plain attention kernel ran")
    monkeypatch.setattr(ops, "attn_plain", plain)
    eng = engine("bfloat16", cache_bits=4)
    eng.runner.step(eng.runner.admit(2), [ids(40, 1), ids(300, 2)])
    eng.runner.step(eng.runner.admit(1), [ids(400, 3)], [[0, 399]])
    torch.cuda.synchronize()
