"""Log probabilities of tokens, the entropy and the likeliest tokens against the same in 64 bits.

Tolerances.  A term e^d of a sum is exp2 of a rounded product: with |d| <= 32 (what lies lower adds nothing) its relative error is at
most 3 half steps of 32 bits times 32 ln 2 plus the exponential's own 2 steps: 3 * 32 * 0.7 * 2^-24 + 2^-22 < 5e-6; sums of V terms of one
sign keep that, plus V / 256 half steps a thread and a tree: for V <= 2^18 at most 1,024 2^-24 = 6e-5 if every rounding went one way, and
sqrt(1,024) 2^-24 = 2e-6 as they fall.  log S has the sum's relative error as an absolute one: 1e-5 is twice what adds up.  The entropy's
second term U / S is at most 13 with the same relative errors: 13 * 7e-6 + 1e-5 < 1e-4.  A logarithm's own rounding: 2^-24 of up to 120."""
import math

import pytest
import torch

from hos_b200 import ops
from hos_b200.errors import KernelError
from hos_b200.sampling import TokenScores, log_probs

pytestmark = pytest.mark.gpu
DEV = "cuda"


def plain(logits, tokens, top):
    x = logits.double().cpu()
    t = tokens.long().cpu()
    lp = torch.log_softmax(x, 1)
    p = lp.exp()
    ent = -torch.where(p > 0, p * lp, 0.0).sum(1)
    out = [lp.gather(1, t[:, None])[:, 0], ent]
    if top:
        order = torch.sort(x, dim=1, descending=True, stable=True).indices[:, :top]
        out += [order.int(), lp.gather(1, order)]
    return out


def check(got, want):
    for a, b, atol in zip(got, want, (1e-5, 1e-4, 0, 1e-5)):
        if a is None:
            continue
        a = a.cpu()
        if a.dtype == torch.int32:
            assert torch.equal(a, b)
            continue
        a = a.double()
        assert torch.equal(a.isnan(), b.isnan()) and torch.equal(a.isinf(), b.isinf())
        ok = b.isfinite()
        assert ((a - b).abs()[ok] <= atol + 2.0 ** -23 * b.abs()[ok]).all(), float((a - b).abs()[ok].max())


@pytest.mark.parametrize("rows,vocab,top", [
    (1, 1, 1), (1, 2, 2), (3, 5, 5), (2, 31, 7), (1, 100, 32), (5, 1023, 1), (7, 8191, 20), (2, 8192, 20), (3, 8193, 32), (1, 32769, 5),
    (9, 32003, 20), (1, 256000, 20), (18, 256000, 5), (19, 100003, 0), (200, 50021, 3), (601, 9001, 2), (1500, 300, 32), (40, 256000, 32)])
@pytest.mark.parametrize("kind", ["normal", "sure"])
def test_scores(rows, vocab, top, kind):
    g = torch.Generator().manual_seed(rows * 1000 + vocab)
    x = torch.randn(rows, vocab, generator=g)
    if kind == "sure":
        x[:, vocab // 2] += 25
    t = torch.randint(0, vocab, (rows,), generator=g, dtype=torch.int32)
    t[0] = vocab // 2
    x, t = x.to(DEV), t.to(DEV)
    check(log_probs(x, t, top), plain(x, t, top))


@pytest.mark.parametrize("blocks,threads", [(1, 128), (8, 128), (1, 256), (2, 256), (8, 256), (1, 1024), (4, 1024)])
def test_every_cut_of_a_row_gives_the_same_tokens(blocks, threads, monkeypatch):
    monkeypatch.setattr(ops, "log_probs_blocks", lambda r, v: (threads, blocks))
    g = torch.Generator().manual_seed(5)
    x = torch.randn(4, 70001, generator=g).to(DEV)
    t = torch.tensor([0, 70000, 35000, 17], dtype=torch.int32, device=DEV)
    check(log_probs(x, t, 32), plain(x, t, 32))
    small = x[:, :9].contiguous()                    # blocks without a number
    check(log_probs(small, t % 9, 9), plain(small, t % 9, 9))


@pytest.mark.parametrize("vocab", [50, 9000, 70001])
@pytest.mark.parametrize("kind", ["equal", "few", "rising", "falling", "one left", "steps", "zeros", "plateau at the end"])
def test_orders_and_ties_of_the_likeliest(kind, vocab):
    top = 20
    i = torch.arange(vocab, dtype=torch.float32)
    x = {"equal": torch.zeros(vocab) + 3, "rising": i * 1e-3, "falling": -i * 1e-3, "steps": (i * 7 % 5), "zeros": torch.where(i % 2 == 0, 0.0, -0.0),
         "few": torch.where(i % (vocab // 7) == 3, i * 1e-4, -math.inf), "one left": torch.where(i == vocab - 2, 1.0, -math.inf),
         "plateau at the end": torch.where(i > vocab - 40, 5.0, (i * 0.37) % 4)}[kind]
    x = torch.stack([x, x.flip(0)]).to(DEV)
    t = torch.tensor([vocab - 2, 1], dtype=torch.int32, device=DEV)
    check(log_probs(x, t, top), plain(x, t, top))


def test_rows_without_a_distribution_and_padding_rows():
    x = torch.randn(6, 9000, generator=torch.Generator().manual_seed(1))
    x[0] = -math.inf
    x[1, 5000] = math.inf
    x[2, 7] = math.nan
    t = torch.tensor([3, 5000, 9, -1, 9000, 8999], dtype=torch.int32, device=DEV)
    got = log_probs(x.to(DEV), t, 4)
    lp, ent = got.logprob.cpu(), got.entropy.cpu()
    assert lp[:3].isnan().all() and ent[:3].isnan().all()
    assert lp[3:5].tolist() == [0, 0] and ent[3:5].tolist() == [0, 0]
    ids = got.top_ids.cpu()
    assert ids[0].tolist() == [0, 1, 2, 3] and ids[1, 0] == 5000 and ids[3].tolist() == ids[4].tolist() == [-1] * 4
    rest = x[2].clone()
    rest[7] = -math.inf
    assert ids[2].tolist() == torch.sort(rest, descending=True, stable=True).indices[:4].tolist()
    check([v[5:] for v in got], plain(x[5:], t[5:], 4))


def test_rows_apart_that_begin_anywhere():
    big = torch.randn(5, 10007, generator=torch.Generator().manual_seed(2)).to(DEV)
    t = torch.tensor([0, 1, 8999, 4000, 77], dtype=torch.int32, device=DEV)
    for lo in (0, 1, 2, 3):
        x = big[:, lo:lo + 9000]
        check(log_probs(x, t, 3), plain(x, t, 3))
    check(log_probs(big[::2, 5:], t[::2].contiguous(), 3), plain(big[::2, 5:], t[::2], 3))


def test_into_given_scores_on_another_stream_captured_and_replayed():
    x = torch.randn(3, 60000, generator=torch.Generator().manual_seed(3)).to(DEV)
    t = torch.tensor([5, 6, 7], dtype=torch.int32, device=DEV)
    out = TokenScores.empty(3, 5, DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        log_probs(x, t, 5, out=out)
    torch.cuda.current_stream().wait_stream(side)
    check(out, plain(x, t, 5))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        log_probs(x, t, 5, out=out)
    x.copy_(torch.randn(3, 60000, generator=torch.Generator().manual_seed(4)))
    g.replay()
    check(out, plain(x, t, 5))
    again = [v.clone() for v in out]
    g.replay()
    assert all(torch.equal(a, b) for a, b in zip(again, out))


def test_refusals():
    x, t = torch.zeros(2, 8, device=DEV), torch.zeros(2, dtype=torch.int32, device=DEV)
    for bad in (dict(logits=x.bfloat16()), dict(logits=x.T), dict(logits=x[0]), dict(tokens=t.long()), dict(tokens=t[:1]), dict(top=9),
                dict(logits=torch.zeros(2, 64, device=DEV), top=33), dict(tokens=t.cpu()), dict(out=TokenScores.empty(3, 1, DEV))):
        a = dict(dict(logits=x, tokens=t, top=1), **bad)
        with pytest.raises(KernelError):
            log_probs(a["logits"], a["tokens"], a["top"], a.get("out"))
    assert log_probs(x[:0], t[:0], 2).top_ids.shape == (0, 2)


@pytest.mark.parametrize("rows,vocab", [(1, 2), (3, 40), (1, 100), (5, 3000), (2, 9000), (1, 256000), (20, 70001), (70, 130000), (300, 5003)])
def test_nearly_sure_rows_keep_their_digits(rows, vocab):
    """A row that is sure of a token to 1e-3 or 1e-12: the log probability and the entropy, which are as small, to 2e-5 of themselves.  With d = l - max
    down to -40 a weight e^d is off by 2^-24 |d| from d's own rounding, as much from d log2 e's, 1.3e-8 |d| from the constant and 2^-22 from the
    exponential: 6e-6; sums of positive numbers in trees and of up to some hundred a thread add 1e-6 each; the entropy is the sum of two positive
    terms of such numbers, one with a factor d."""
    g = torch.Generator().manual_seed(vocab)
    for lead in (7.0, 20.0, 28.0):
        logits = torch.rand(rows, vocab, generator=g) * 3
        best = torch.randint(0, vocab, (rows,), generator=g)
        logits[torch.arange(rows), best] = 3 + math.log(vocab) + lead * (0.5 + 0.5 * torch.rand(rows, generator=g))
        got = log_probs(logits.to(DEV), best.to(torch.int32).to(DEV), 1)
        x = logits.double()
        d = x - x.amax(1, keepdim=True)
        rest = d.exp()
        rest[torch.arange(rows), best] = 0
        small = rest.sum(1)
        lp = -torch.log1p(small)
        entropy = torch.log1p(small) - (rest * d).sum(1) / (1 + small)
        assert got.top_ids[:, 0].tolist() == best.tolist()
        for a, b in ((got.logprob, lp), (got.entropy, entropy), (got.top_logprobs[:, 0], lp)):
            assert ((a.double().cpu() - b).abs() <= 2e-5 * b.abs()).all(), (lead, float(((a.double().cpu() - b) / b).abs().max()))


@pytest.mark.parametrize("vocab", [7, 500, 20000, 256000])
@pytest.mark.parametrize("equal", [2, 5])
def test_several_equal_maxima_count_each(vocab, equal):
    """`equal` tokens 40 above all others: log probabilities -log(equal), entropy log(equal), wherever in the row they lie."""
    g = torch.Generator().manual_seed(vocab + equal)
    logits = torch.rand(12, vocab, generator=g) - 40
    where = torch.stack([torch.randperm(vocab, generator=g)[:equal] if i % 3 else torch.arange(equal) for i in range(12)])
    logits.scatter_(1, where, 5.0)
    got = log_probs(logits.to(DEV), where[:, 1].to(torch.int32).to(DEV), equal)
    assert got.top_ids.tolist() == where.sort(1).values.tolist()
    assert (got.logprob.cpu() + math.log(equal)).abs().max() < 1e-6 and (got.entropy.cpu() - math.log(equal)).abs().max() < 1e-6


def test_softcap_in_place():
    """30 tanh(l / 30): tanhf is off by 2 units in the last place at most (2 * 2^-24 below 1), 30 times that is 3.6e-6; the product of up to 30 is rounded
    by 2^-20, 1.0e-6; the quotient by 2^-24 of itself, which x / cosh^2 x < 0.45 makes 30 * 0.45 * 2^-24 = 0.8e-6: 5.4e-6."""
    from hos_b200 import ops
    x = (torch.randn(3, 70001, generator=torch.Generator().manual_seed(1)) * 40).to(DEV)
    want = 30 * torch.tanh(x.double() / 30)
    ops.softcap(x, 30.0)
    assert (x.double() - want).abs().max() < 5.5e-6
    ops.softcap(x[:0], 30.0)
    for bad in ((x, 0.0), (x, -1.0), (x.T, 3.0), (x.bfloat16(), 3.0), (x.cpu(), 3.0)):
        with pytest.raises(KernelError):
            ops.softcap(*bad)
