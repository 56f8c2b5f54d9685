"""Log probabilities of tokens straight from hidden rows in front of a head, against the same in 64 bits.

Tolerances.  A logit is a sum of K products of bfloat16 numbers, exact in 32 bits, added in 32 bits: off by at most K 2^-24 of sum |x w|
if every addition rounded one way; the products of the cases here add up to at most 25 (|x| 1.2, |w| 0.02, K 1,024: sum |x w| is about
0.8 * 0.8 * 1.2 * 0.02 K), so by 1e-3 at the very most and by sqrt(K) 2^-24 * 25 < 5e-5 as roundings fall; a cap c tanh(l / c) with an
absolute error of 4 2^-24 of c = 30: 1e-5.  The scores' own error is 1e-5 and 1e-4 (test_log_probs_gpu.py).  Together 1e-4 for
log probabilities and 3e-4 for entropies (a mean of logits, and a logarithm of their sum)."""
import pytest
import torch

from hos_b200.errors import KernelError
from hos_b200.parts import linear

pytestmark = pytest.mark.gpu
DEV = "cuda"


def make(rows, width, vocab, seed, dtype=torch.bfloat16):
    g = torch.Generator().manual_seed(seed)
    w = (torch.randn(vocab, width, generator=g) * 0.02).to(dtype)
    t = torch.randint(0, vocab, (rows,), generator=g, dtype=torch.int32)
    x = torch.randn(rows, width, generator=g) + (torch.rand(rows, 1, generator=g) * 12 / 0.02 ** 2 / width) * w[t.long()].float()
    return x.to(dtype).to(DEV), w.to(DEV), t.to(DEV)


def plain(x, w, t, cap):
    logits = x.double() @ w.double().T
    if cap:
        logits = cap * torch.tanh(logits / cap)
    lp = torch.log_softmax(logits, 1)
    return lp.gather(1, t.long()[:, None])[:, 0], -(lp.exp() * lp).sum(1), lp


def check(got, want):
    for a, b, atol in ((got.logprob, want[0], 1e-4), (got.entropy, want[1], 3e-4)):
        assert ((a.double() - b).abs() <= atol + 2.0 ** -23 * b.abs()).all(), float((a.double() - b).abs().max())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,width,vocab", [(1, 64, 50), (3, 256, 1000), (17, 264, 777), (33, 128, 5003), (128, 256, 2048), (129, 64, 256), (130, 72, 257),
                                              (255, 520, 1021), (256, 512, 4096), (257, 1024, 30011), (700, 136, 513), (1500, 64, 100)])
@pytest.mark.parametrize("cap", [0.0, 30.0])
def test_scores_of_hidden_rows(rows, width, vocab, cap, dtype):
    x, w, t = make(rows, width, vocab, rows + vocab, dtype)
    check(linear.log_probs(x, w, t, cap), plain(x, w, t, cap))


@pytest.mark.parametrize("rows,top", [(5, 3), (200, 20)])
def test_with_alternatives(rows, top):
    x, w, t = make(rows, 256, 3001, 4)
    got, want = linear.log_probs(x, w, t, 30.0, top), plain(x, w, t, 30.0)
    check(got, want)
    best = torch.sort(want[2], dim=1, descending=True).values[:, :top]
    assert ((got.top_logprobs.double() - best).abs() <= 1e-4).all()
    assert ((want[2].gather(1, got.top_ids.long()) - best).abs() <= 1e-4).all()          # whose order near ties is the logits'


@pytest.mark.parametrize("rows", [4, 300])
def test_padding_rows_and_sure_rows(rows):
    x, w, t = make(rows, 128, 999, 6)
    x[1] *= 40                                                # a row of which one token has it all
    t[0], t[3] = -1, 999
    got, want = linear.log_probs(x, w, t), plain(x, w, t.clamp(0, 998), 0.0)
    assert got.logprob[[0, 3]].tolist() == [0, 0] and got.entropy[[0, 3]].tolist() == [0, 0]
    keep = torch.tensor([i for i in range(rows) if i not in (0, 1, 3)])
    check(type(got)(got.logprob[keep], got.entropy[keep]), [v[keep] for v in want])
    # logits of row 1 are 40 times as large, and so is what their sums are off by
    assert (got.logprob[1].double() - want[0][1]).abs() < 4e-3 and (got.entropy[1].double() - want[1][1]).abs() < 1e-2


@pytest.mark.parametrize("rows", [2, 200])
def test_rows_without_a_distribution(rows):
    x, w, t = make(rows, 64, 600, 7)
    x[0, 5] = float("nan")
    w[3] = 0
    got = linear.log_probs(x, w, t)
    assert got.logprob[0].isnan() and got.entropy[0].isnan() and got.logprob[1:].isfinite().all()


@pytest.mark.parametrize("rows", [3, 400])
def test_rows_apart_another_stream_and_a_replayed_graph(rows):
    x, w, t = make(rows, 256, 2003, 8)
    wide = torch.zeros(rows, 512, dtype=x.dtype, device=DEV)
    wide[:, 128:384] = x
    want = linear.log_probs(x, w, t, 30.0)
    again = linear.log_probs(wide[:, 128:384], w, t, 30.0)
    check(again, plain(x, w, t, 30.0))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = linear.log_probs(x, w, t, 30.0)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(other.logprob, want.logprob) and torch.equal(other.entropy, want.entropy)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        other = linear.log_probs(x, w, t, 30.0)
    x2, _, t2 = make(rows, 256, 2003, 9)
    x.copy_(x2), t.copy_(t2)
    g.replay()
    check(other, plain(x, w, t, 30.0))


@pytest.mark.parametrize("rows", [8, 9, 24, 32, 64, 65, 90, 96, 97, 128])
@pytest.mark.parametrize("cap,top", [(0.0, 0), (0.0, 2), (30.0, 0)])
def test_few_rows_and_a_large_vocabulary(rows, cap, top):
    x, w, t = make(rows, 136, 20011, rows)
    got, want = linear.log_probs(x, w, t, cap, top), plain(x, w, t, cap)
    check(got, want)
    if top:
        assert ((want[2].gather(1, got.top_ids.long()) - got.top_logprobs.double()).abs() <= 1e-4).all()


def test_many_rows_go_some_at_a_time(monkeypatch):
    from hos_b200.parts import gemm_tc
    x, w, t = make(1300, 128, 3000, 7)
    whole = linear.log_probs(x, w, t, 30.0)
    monkeypatch.setattr(gemm_tc, "SCORE_BYTES", 600 * 32 * 12)
    check(linear.log_probs(x, w, t, 30.0), plain(x, w, t, 30.0))
    monkeypatch.setattr(linear, "LOGITS_BYTES", 4 * 3000 * 300)
    some = linear.log_probs(x, w, t, 30.0, 2)
    assert (some.logprob - whole.logprob).abs().max() < 1e-4 and some.top_ids.shape == (1300, 2)


@pytest.mark.parametrize("rows", [3, 12, 30, 60, 96, 110, 300])
@pytest.mark.parametrize("cap", [0.0, 30.0])
def test_long_sums_lose_little(rows, cap):
    """Tensor cores cut their sums at every 16 products: by half of the last bit in the middle, 0.36 * 2^-23 of a sum that has grown to half of its
    chunk's on average.  3,584 products in chunks of up to 48 steps: 48 * 0.36 * 2^-23 / 2 = 1.0e-6 of a logit (all
    of them in one sum would be 4.8e-6); the scores' own roundings are below 4e-7 of it.  A log probability is the difference of two logits (one
    of them a mean), each low by such a part of itself, an entropy the difference of a logarithm of sums and a mean: errors are a part of the
    row's largest logit, not of the score, which may be smaller (a row of logits of 9 and a log probability of -0.3)."""
    x, w, t = make(rows, 3584, 6000, 5)
    got, want = linear.log_probs(x, w, t, cap), plain(x, w, t, cap)
    largest = (x.double() @ w.double().T).abs().amax(1).norm()
    for a, b, part in zip((got.logprob, got.entropy), want, (2e-6, 4e-6)):
        assert (a.double() - b).norm() < part * largest, float((a.double() - b).norm() / largest)


@pytest.mark.parametrize("rows", [1, 8, 9, 24, 64, 97, 200])
@pytest.mark.parametrize("cap", [0.0, 30.0])
def test_a_row_that_is_nearly_sure(rows, cap):
    """The product's scores keep the digits of small log probabilities, where the logits do: an error e of logits of 25 (2^-20 of them, and of the cap)
    moves what the others have, and so the log probability, by 5e-5 of itself."""
    x, w, t = make(rows, 512, 3000, 9)
    w = torch.cat([w, torch.zeros(8, 512, dtype=w.dtype, device=DEV)])
    w[t.long()] = (w[t.long()].float() * 4).to(w.dtype)
    x = (w[t.long()].float() * (25 / (w[t.long()].float() ** 2).sum(1, keepdim=True))).to(w.dtype)
    got, want = linear.log_probs(x, w, t, cap), plain(x, w, t, cap)
    assert (want[0] > -1e-2).all() and (want[0] < -1e-8).all()
    for a, b in zip((got.logprob, got.entropy), want):
        assert ((a.double() - b).abs() <= 1e-4 * b.abs()).all(), float(((a.double() - b) / b).abs().max())


def test_heads_that_do_not_fit_are_refused():
    for rows in (4, 20, 200):
        x, w, t = make(rows, 64, 20000, 1)
        for head in (w[:, :56], w[:0], w[0], w.cpu()):
            with pytest.raises(KernelError):
                linear.log_probs(x, head, t)


def test_refusals():
    x, w, t = make(4, 64, 100, 1)
    for bad in ((x, w, t[:2]), (x.half(), w, t), (x[0], w, t[:1]), (x.cpu(), w, t), (x, w, t.long())):
        with pytest.raises(KernelError):
            linear.log_probs(*bad)
    assert linear.log_probs(x[:0], w, t[:0]).logprob.shape == (0,)
