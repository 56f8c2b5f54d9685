"""Several answers to a prompt through the engine: forked conversations that read their common pages once, the log probabilities of what is
generated, and the scores of given answers; against the plain implementation and against the engine's own steps."""
import json
import os
import random

import pytest
import torch
from helpers import TINY, assert_close, make_folder, plain_model, random_tokens
from plain import gemma2_plain as P

from hos_b200.errors import HosError
from hos_b200.parts import shared_attention as sa

pytestmark = pytest.mark.gpu


@pytest.fixture
def shared(monkeypatch):
    """Steps share however little that spares; how often attention over shared pages ran."""
    monkeypatch.setattr(sa, "SHARE_BYTES", 0)
    monkeypatch.setattr(sa, "MERGE_US", -1e9)               # (short sequences share too)
    calls = []
    run = sa._run

    def counted(*a):
        calls.append(a[0].shape[0])
        return run(*a)
    monkeypatch.setattr(sa, "_run", counted)
    return calls


def runner_for(folder, **kw):
    from hos_b200.engine import Runner
    return Runner.from_folder(folder, **dict(dict(dtype="bfloat16", max_tokens=8192, share_prefix=True), **kw))


@pytest.mark.parametrize("name", ["C", "D", "F", "G"])
@pytest.mark.parametrize("prompt,answers", [(1, 3), (64, 2), (200, 5), (330, 20)])
def test_forks_decode_together(tmp_path, name, prompt, answers, shared):
    """Single-token steps of forks (replayed), of which some leave and another is forked on the way, and a stranger among them."""
    folder = make_folder(tmp_path, name)
    w, cfg = plain_model(folder)
    vocab = TINY[name][0]["vocab_size"]
    rng = random.Random(prompt + answers)
    r = runner_for(folder, chunk_tokens=1)
    first = random_tokens(rng, prompt, vocab)
    a, = r.admit(1)
    r.step([a], [first])
    other, = r.admit(1)
    strange = random_tokens(rng, 77, vocab)
    r.step([other], [strange])
    slots = [a] + r.fork(a, answers - 1) + [other]
    held = [list(first) for _ in range(answers)] + [strange]
    logits = []
    for t in range(6):
        if t == 2 and answers > 3:
            gone = slots.pop(1)
            held.pop(1)
            r.release(gone)
        if t == 4:
            slots.insert(0, r.fork(slots[0])[0])
            held.insert(0, list(held[0]))
        new = random_tokens(rng, len(slots), vocab)
        logits.append((r.step(slots, [[x] for x in new]), [h + [x] for h, x in zip(held, new)]))
        held = list(logits[-1][1])
        r.cache.check()
    assert shared or prompt < 64
    for got, seqs in logits:
        for row, seq in list(zip(got, seqs))[:4] + [(got[-1], seqs[-1])]:
            assert_close(row, P.forward_logits(w, cfg, seq)[-1], "bfloat16", f"{name} {len(seq)}")


@pytest.mark.parametrize("name", ["D", "F", "G"])
def test_forks_bring_pieces(tmp_path, name, shared):
    """Steps of several tokens a sequence, all places wanted, longer than what a pass takes, beside a sequence that starts."""
    folder = make_folder(tmp_path, name)
    w, cfg = plain_model(folder)
    vocab = TINY[name][0]["vocab_size"]
    rng = random.Random(5)
    r = runner_for(folder, chunk_tokens=24)
    first = random_tokens(rng, 260, vocab)
    a, = r.admit(1)
    r.step([a], [first])
    slots, fresh = [a] + r.fork(a, 3), r.admit(1)
    pieces = [random_tokens(rng, n, vocab) for n in (1, 9, 40, 17)]
    start = random_tokens(rng, 30, vocab)
    got = r.step(slots + fresh, pieces + [start], [range(len(p)) for p in pieces] + [range(30)])
    assert shared
    at = 0
    for p in pieces:
        assert_close(got[at:at + len(p)], P.forward_logits(w, cfg, first + p)[260:], "bfloat16", f"piece of {len(p)}")
        at += len(p)
    assert_close(got[at:], P.forward_logits(w, cfg, start), "bfloat16", "the one that starts")
    shared.clear()
    last = r.step(slots, [p[:3] + p[:2] for p in (pieces * 2)[1:5]])        # a second turn, last places only
    assert shared
    for i, p in enumerate((pieces * 2)[1:5]):
        assert_close(last[i], P.forward_logits(w, cfg, first + pieces[i] + p[:3] + p[:2])[-1], "bfloat16", "second turn")


def test_many_steps_with_rings_that_wrap(tmp_path, shared):
    folder = make_folder(tmp_path, "C")                      # a window of 40 in a ring of one page
    w, cfg = plain_model(folder)
    rng = random.Random(8)
    r = runner_for(folder, chunk_tokens=1)
    first = random_tokens(rng, 150, 331)
    a, = r.admit(1)
    r.step([a], [first])
    slots = [a] + r.fork(a, 2)
    seqs = [first + random_tokens(rng, 140, 331) for _ in slots]
    rows = [r.step(slots, [[s[150 + t]] for s in seqs]) for t in range(140)]
    assert len(shared) > 2
    for i, s in enumerate(seqs):
        want = P.forward_logits(w, cfg, s)[150:]
        assert_close(torch.stack([row[i] for row in rows]), want, "bfloat16", f"sequence {i}")


def test_too_little_to_share_runs_as_before(tmp_path):
    folder = make_folder(tmp_path, "D")
    got = []
    for share in (False, True):
        r = runner_for(folder, share_prefix=share)
        a, = r.admit(1)
        r.step([a], [[5] * 200])
        slots = [a] + r.fork(a, 3)
        got.append(torch.cat([r.step(slots, [[t], [t + 1], [7], [9]]) for t in range(4)]))
    assert torch.equal(got[0], got[1])


def test_steps_of_sequences_that_will_be_longer(tmp_path, shared):
    """The lists of work may be made for the length that sequences will have some steps on (pages are taken ahead), rings that wrap meanwhile
    among them."""
    for name in ("C", "D"):
        folder = make_folder(tmp_path / name, name)
        w, cfg = plain_model(folder)
        vocab = TINY[name][0]["vocab_size"]
        rng = random.Random(4)
        r = runner_for(folder, chunk_tokens=1)
        first = random_tokens(rng, 240, vocab)
        a, = r.admit(1)
        r.step([a], [first])
        slots = [a] + r.fork(a, 2)
        seqs = [first + random_tokens(rng, 70, vocab) for _ in slots]
        r.cache.extend_all(slots, [310] * 3)
        sess = r.decode_session(3)
        rows = []
        for t in range(70):
            sess.upload(slots, [s[240 + t] for s in seqs], lengths=[310] * 3)
            rows.append(sess.run_step().clone())
        assert shared or name == "C"
        for i, s in enumerate(seqs):
            assert_close(torch.stack([row[i] for row in rows]), P.forward_logits(w, cfg, s)[240:], "bfloat16", f"{name}, sequence {i}")


def test_timed_steps_share(tmp_path, shared):
    r = runner_for(make_folder(tmp_path, "D"), chunk_tokens=1)
    a, = r.admit(1)
    r.step([a], [[3, 8, 1] * 80])
    slots = [a] + r.fork(a, 4)
    ms, launches = r.decode_steps_timed(slots, [[i] for i in range(5)], 3, 80)
    r.wait()
    assert shared and ms > 0 and launches > 0 and [r.length(s) for s in slots] == [323] * 5
    assert r.step(slots, [[2]] * 5).isfinite().all()


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("temp", [0.0, 0.9])
def test_generated_tokens_with_their_log_probabilities(tmp_path, dtype, temp):
    from hos_b200 import Engine
    folder = make_folder(tmp_path, "D")
    eng = Engine(folder, dtype=dtype, max_batch=4)
    prompts = [[5, 6, 7], [9] * 20, [1, 2], [3]]
    kw = dict(max_tokens=12, temp=temp, seed=3, stop_ids=())
    plain = eng.generate(prompts, **kw)
    scored = eng.generate(prompts, logprobs=4, **kw)
    assert plain == scored and not hasattr(plain[0][0], "logprob")
    for p, out in zip(prompts, scored):
        slot, = eng.runner.admit(1)
        logits = eng.step([slot], [p + [int(t) for t in out[:-1]]], [range(len(p) - 1, len(p) + len(out) - 1)])
        eng.runner.release(slot)
        lp = torch.log_softmax(logits.double(), 1).cpu()
        tol = 1e-4 if dtype == "float32" else 5e-2           # (a step in pieces rounds otherwise than steps of a token)
        for row, t in zip(lp, out):
            assert abs(t.logprob - float(row[t])) < tol
            assert abs(t.entropy - float(-(row.exp() * row).sum())) < 2 * tol
            best = torch.sort(row, descending=True).values[:4]
            assert [abs(a - float(b)) < tol for (_, a), b in zip(t.top, best)] == [True] * 4
            assert all(abs(float(row[i]) - p) < tol for i, p in t.top)
    none = eng.generate(prompts[0], logprobs=0, **kw)
    assert none == scored[0] and none[0].top == [] and none[0].logprob == pytest.approx(scored[0][0].logprob, abs=1e-5)
    got = []
    eng.generate(prompts[1], logprobs=1, on_token=lambda i, t: got.append(t.logprob), **kw)
    assert len(got) == 12
    chat, = eng.open(1)
    a = eng.generate_from_ids([chat], [[5, 6, 7]], max_tokens=6, temp=temp, seed=3, stop_ids=(), logprobs=2)
    b = eng.generate_from_ids([chat], [[8]], max_tokens=2, temp=temp, seed=3, stop_ids=(), logprobs=2)
    assert a[0] == plain[0][:6] and len(b[0]) == 2 and len(b[0][0].top) == 2
    chat.close()


@pytest.mark.parametrize("dtype,tol", [("float32", 1e-4), ("bfloat16", 6e-2)])
@pytest.mark.parametrize("share", [False, True])
@pytest.mark.parametrize("prompt", [1, 2, 150])
def test_scores_of_answers(tmp_path, dtype, tol, share, prompt, monkeypatch):
    from hos_b200 import Engine
    if share and dtype == "float32":
        pytest.skip("shared pages are read once in bfloat16")
    if share:
        monkeypatch.setattr(sa, "SHARE_BYTES", 0)
    folder = make_folder(tmp_path, "D")
    w, cfg = plain_model(folder)
    eng = Engine(folder, dtype=dtype, max_batch=3, share_prefix=share)
    rng = random.Random(2)
    first = random_tokens(rng, prompt, 1000)
    answers = [random_tokens(rng, n, 1000) for n in (1, 7, 30, 2, 90, 90)]
    free = [g.pages.n_free for g in eng.runner.cache.groups]
    for top in (0, 3):
        got = eng.score(first, answers, top)
        assert got == answers and [g.pages.n_free for g in eng.runner.cache.groups] == free
        for a, out in zip(answers, got):
            lp = torch.log_softmax(P.forward_logits(w, cfg, first + a).double()[prompt - 1:-1], 1)
            for row, t in zip(lp, out):
                assert abs(t.logprob - float(row[t])) < tol and abs(t.entropy - float(-(row.exp() * row).sum())) < 3 * tol
                assert len(t.top) == top and all(abs(p - float(row[i])) < tol for i, p in t.top)
    if dtype == "float32" and prompt > 1:
        n, mean, _ = eng.perplexity(first + answers[2])
        more = eng.score(first[:1], [first[1:] + answers[2]])[0]
        assert len(more) == n and -sum(t.logprob for t in more) / n == pytest.approx(mean, abs=1e-5)
    assert eng.score(first, []) == []


def test_scores_with_little_room(tmp_path):
    """A cache that holds the prompt and one answer at a time."""
    from hos_b200 import Engine
    folder = make_folder(tmp_path, "D")
    small, large = Engine(folder, dtype="float32", max_batch=4, max_tokens=256), Engine(folder, dtype="float32", max_batch=4)
    first, answers = [4] * 100, [[7] * 60, [8] * 3, [9] * 64]
    a, b = small.score(first, answers), large.score(first, answers)
    assert a == b and [[round(t.logprob, 3) for t in x] for x in a] == [[round(t.logprob, 3) for t in x] for x in b]
    with pytest.raises(HosError):
        small.score([4] * 200, [[7] * 60])
    small.runner.cache.check()
    assert not small.runner.cache.lengths


def test_refusals(tmp_path):
    from hos_b200 import Engine
    folder = make_folder(tmp_path, "D")
    for kw in (dict(dtype="float32"), dict(cache_bits=4)):
        with pytest.raises(HosError, match="share_prefix"):
            Engine(folder, share_prefix=True, **kw)
    eng = Engine(folder, max_batch=2)
    for bad in (-1, 33):
        with pytest.raises(HosError, match="alternatives"):
            eng.generate([1, 2], max_tokens=2, logprobs=bad)
        with pytest.raises(HosError, match="alternatives"):
            eng.score([1, 2], [[3]], bad)
    for prompt, answers in (([], [[1]]), ([1], [[]]), ([1], [[2], []]), ([1], [[1000]]), ([1000], [[1]]), ([1] * 1000, [[1] * 60])):
        with pytest.raises(HosError):
            eng.score(prompt, answers)
    r = eng.runner
    a, = r.admit(1)
    for slots, tokens, targets, top in (([a], [[1]], [[2, 3]], 0), ([a], [[]], [[]], 0), ([a, a], [[1], [1]], [[1], [1]], 0), ([a], [[1]], [[2]], 33), ([99], [[1]], [[2]], 0)):
        with pytest.raises(HosError):
            r.scores(slots, tokens, targets, top)
    assert r.cache.lengths[a] == 0


@pytest.mark.parametrize("shared_pages", [True, False])
def test_the_example_ranks_answers(tmp_path, shared_pages, shared, capsys):
    import importlib.util
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "several_answers.py")
    spec = importlib.util.spec_from_file_location("several_answers", path)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    from test_fourbit_engine_gpu import RAW                  # (heads that keys in 4 bits take)
    config = tmp_path / "config.json"
    config.write_text(json.dumps(RAW))
    prompt = ",".join(str(3 + i % 90) for i in range(140))
    args = ["--random", str(config), "-p", prompt, "--answers", "3", "-n", "5", "--max-seq-len", "256", "--rank"] + (["--shared"] if shared_pages else [])
    assert example.main(args) == 0
    got = capsys.readouterr()
    means = [float(x) for x in [l for l in got.err.splitlines() if "mean log" in l][0].split()[4:]]
    assert len(got.out.strip().splitlines()) == 3 and means == sorted(means, reverse=True) and bool(shared) == shared_pages


def test_the_command_line(tmp_path):
    import subprocess
    hos = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "bin", "hos")
    folder = make_folder(tmp_path, "D")
    p = subprocess.run([hos, "-m", folder, "-p", "5,6", "-n", "3", "--logprobs", "2", "--no-echo"], capture_output=True, text=True)
    assert p.returncode == 0 and p.stderr.count("logprob") == len(p.stdout.strip().split(","))
    p = subprocess.run([hos, "-m", folder, "-p", "5,6", "--score", "7,8", "--score", "9", "--share-prefix"], capture_output=True, text=True)
    lines = p.stdout.strip().splitlines()
    assert p.returncode == 0 and [l.split(" : ")[0] for l in lines] == ["7,8", "9"] and all(float(l.split(" : ")[1]) < 0 for l in lines)
    p = subprocess.run([hos, "-m", folder, "--score", "7,8"], capture_output=True, text=True)
    assert p.returncode == 1 and "one prompt" in p.stderr


def test_a_cache_of_another_size_and_a_released_fork(tmp_path, shared):
    """Lists of work are made anew after the cache was resized, after forks left and others came into their slots."""
    folder = make_folder(tmp_path, "D")
    w, cfg = plain_model(folder)
    rng = random.Random(6)
    r = runner_for(folder, chunk_tokens=1, max_slots=8)
    first = random_tokens(rng, 200, 1000)
    a, = r.admit(1)
    r.step([a], [first])
    slots = [a] + r.fork(a, 3)
    seqs = [list(first) for _ in slots]
    for t in range(6):
        if t == 2:
            r.resize_cache(2048)
        if t == 4:                                           # a stranger in a fork's slot
            r.release(slots[2])
            slots[2], = r.admit(1)
            seqs[2] = random_tokens(rng, 150, 1000)
            r.step([slots[2]], [seqs[2]])
        new = random_tokens(rng, 4, 1000)
        seqs = [s + [x] for s, x in zip(seqs, new)]
        got = r.step(slots, [[x] for x in new])
        for row, s in zip(got, seqs):
            assert_close(row, P.forward_logits(w, cfg, s)[-1], "bfloat16", f"step {t}, {len(s)} tokens")
    assert len(shared) > 1


def test_sequences_that_grow_by_many_pages(tmp_path, shared):
    """The lists of a replayed step stay while sequences take pages of their own."""
    folder = make_folder(tmp_path, "G")
    w, cfg = plain_model(folder)
    vocab = TINY["G"][0]["vocab_size"]
    rng = random.Random(7)
    r = runner_for(folder, chunk_tokens=1)
    first = random_tokens(rng, 70, vocab)
    a, = r.admit(1)
    r.step([a], [first])
    slots = [a] + r.fork(a, 1)
    seqs = [first + random_tokens(rng, 300, vocab) for _ in slots]
    rows = [r.step(slots, [[s[70 + t]] for s in seqs]) for t in range(300)]
    assert shared
    for i, s in enumerate(seqs):
        assert_close(torch.stack([row[i] for row in rows]), P.forward_logits(w, cfg, s)[70:], "bfloat16", f"sequence {i}")


@pytest.mark.parametrize("share", [True, False])
def test_sequences_that_are_set_back(tmp_path, shared, share, monkeypatch):
    """Forks set back into the pages that they share (their records and lengths), then stepped on: what lies behind is not seen.  (A window
    as wide as the sequences: a ring of pages no longer has what lies before a narrow one.)"""
    monkeypatch.setitem(TINY, "wide", (dict(TINY["D"][0], sliding_window=1000), 3))
    folder = make_folder(tmp_path, "wide")
    w, cfg = plain_model(folder)
    rng = random.Random(9)
    r = runner_for(folder, chunk_tokens=1, share_prefix=share)
    first = random_tokens(rng, 250, 1000)
    a, = r.admit(1)
    r.step([a], [first])
    slots = [a] + r.fork(a, 3)
    seqs = [first + random_tokens(rng, 1, 1000) for _ in slots]
    got = r.step(slots, [s[250:] for s in seqs])
    assert bool(shared) == share
    r.write_records(slots, pos=[100, 250, 140, 70])
    seqs = [first[:n] + random_tokens(rng, 1, 1000) for n in (100, 250, 140, 70)]
    got = r.step(slots, [s[-1:] for s in seqs])
    for row, s in zip(got, seqs):
        assert_close(row, P.forward_logits(w, cfg, s)[-1], "bfloat16", f"{len(s)} tokens")
    r.cache.check()


def test_few_programs_are_kept(tmp_path, shared, monkeypatch):
    """Steps whose lists want another program every time: the oldest go, and the steps stay right."""
    from hos_b200.engine import decode
    monkeypatch.setattr(decode, "SHARED_PROGRAMS", 2)
    refill, number = sa.ReplayedWork.refill, iter(range(100))

    def another(self, made):
        ok = refill(self, made)
        self.key = self.key + (next(number),)
        return ok
    monkeypatch.setattr(sa.ReplayedWork, "refill", another)
    runners = [runner_for(make_folder(tmp_path / str(share), "D"), chunk_tokens=1, share_prefix=share) for share in (True, False)]
    slots = []
    for r in runners:
        a, = r.admit(1)
        r.step([a], [[3, 8, 1] * 80])
        slots.append([a] + r.fork(a, 3))
    for t in range(8):
        runners[0].decode_session(4)._paged_for = None       # new lists, and by the above another program
        got, want = (r.step(s, [[t]] * 4) for r, s in zip(runners, slots))
        assert_close(got, want.cpu(), "bfloat16", f"step {t}")
        assert sum(bool(k[-1]) for k in runners[0].decode_session(4)._programs) <= 3
