"""What is measured of the operators for several answers to a prompt: attention of sequences that begin alike, the log
probabilities of tokens from logits, and straight from the hidden rows in front of the head.

A case names its operator:

  attend    softmax attention of the last `new` tokens of sequences over paged keys and values, causal, with an optional window
            and soft-cap.  There are `prompts` prompts of `prefix` tokens, each with up to `answers` sequences that were forked
            from it and go on with up to `own` tokens of their own
  logprobs  of rows of logits l: log p(t) = l_t - log sum exp l of a given token t, the entropy -sum p log p, and the `top`
            likeliest tokens (the lower id first where two are alike) with their log probabilities
  score     the first two of hidden rows h in front of a head W [vocab, width]: l = h . W^T, soft-capped c tanh(l / c) if `cap`

Sizes are those of Gemma-2 at 2B, 9B and 27B (heads, widths, vocabulary), and odd ones.
"""
from __future__ import annotations

import math

import torch

own = False

PAGE = 64                   # positions of a page
DEV = "cuda"


# ---- cases ------------------------------------------------------------------------------------------------------
def _attend(prompts, answers, prefix, tail, new, heads, kv, dim, window, cap, mixed):
    return dict(op="attend", prompts=prompts, answers=answers, prefix=prefix, own=tail, new=new, heads=heads, kv=kv, dim=dim, window=window, cap=cap,
                mixed=mixed)


def _logprobs(rows, vocab, top, masked):
    return dict(op="logprobs", rows=rows, vocab=vocab, top=top, masked=masked)


def _score(rows, width, vocab, cap):
    return dict(op="score", rows=rows, width=width, vocab=vocab, cap=cap)


def listed():
    return [
        # two answers to a short question, one more token each: latency counts
        dict(_attend(1, 2, 130, 9, 1, 8, 4, 256, 0, 50.0, False), name="attend-2-short"),
        # eight answers on top of a long chat, one more token each
        dict(_attend(1, 8, 8000, 120, 1, 8, 4, 256, 0, 50.0, False), name="attend-8-answers"),
        # many samples of one problem, unequally far along, 27B heads
        dict(_attend(1, 64, 3900, 700, 1, 32, 16, 128, 0, 50.0, False), name="attend-64-samples"),
        # several prompts, each with some answers, in no order, 9B heads in a layer with a window
        dict(_attend(6, 8, 5003, 300, 1, 16, 8, 256, 4096, 50.0, True), name="attend-6-prompts"),
        # five candidate answers of 37 tokens are scored against a text
        dict(_attend(1, 5, 3001, 37, 37, 8, 4, 256, 0, 50.0, False), name="attend-5-candidates"),
        # 32 samples on a long document, heads of 128 without a soft-cap
        dict(_attend(1, 32, 65536, 500, 1, 32, 8, 128, 0, 0.0, False), name="attend-32-document"),
        # one sequence's next token, the five likeliest beside it
        dict(_logprobs(1, 256000, 5, False), name="logprobs-1-top-5"),
        # 64 sequences' next tokens with twenty alternatives, some of the vocabulary ruled out
        dict(_logprobs(64, 256000, 20, True), name="logprobs-64-top-20"),
        # every token of a text, a small vocabulary that fills no tile
        dict(_logprobs(1999, 32003, 1, False), name="logprobs-1999-odd"),
        # candidate answers: 185 tokens at 2B widths
        dict(_score(185, 2304, 256000, 30.0), name="score-185"),
        # a text of 2,048 tokens at 9B widths
        dict(_score(2048, 3584, 256000, 30.0), name="score-2048"),
        # the next tokens of 24 sequences, no soft-cap, a vocabulary that fills no tile
        dict(_score(24, 2048, 50021, 0.0), name="score-24-odd"),
    ]


def _between(rng, lo, hi):
    """A whole number between lo and hi, spread over the logarithm."""
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    most = [work(c) for c in listed()]
    while True:
        op = rng.choice(["attend", "attend", "logprobs", "score"])
        if op == "attend":
            kv, per = rng.choice([1, 2, 4, 8, 16]), rng.choice([1, 2, 2, 4, 4, 8])
            new = 1 if rng.random() < 0.7 else _between(rng, 2, 128)
            case = _attend(_between(rng, 1, 8), _between(rng, 2, 64), _between(rng, 1, 65536), max(new, _between(rng, 1, 1024)), new, kv * per, kv,
                           rng.choice([64, 128, 256]), rng.choice([0, 0, 1024, 4096]), rng.choice([0.0, 50.0]), rng.random() < 0.5)
            # the plain form holds every pair's score, padded, and all keys and values in 32 bits
            seqs = case["prompts"] * case["answers"]
            if seqs * new * case["heads"] * (case["prefix"] + case["own"]) > 2e8 or seqs > 256:
                continue
            if (case["prompts"] * case["prefix"] + seqs * case["own"]) * kv * case["dim"] > 3e8:
                continue
        elif op == "logprobs":
            case = _logprobs(_between(rng, 1, 2048), _between(rng, 100, 256000), rng.choice([0, 1, 5, 20]), rng.random() < 0.3)
        else:
            case = _score(_between(rng, 1, 2048), 8 * _between(rng, 16, 576), _between(rng, 500, 256000), rng.choice([0.0, 30.0]))
        w, like = work(case), [m for c, m in zip(listed(), most) if c["op"] == op]
        if w["bytes"] <= max(m["bytes"] for m in like) and w["flops"] <= max(m["flops"] for m in like):
            return case


def _spread(n, least, most):
    """n numbers between least and most, the first of them the most, the others spread in no order."""
    return [max(least, round(most - (most - least) * (0.6180339887 * i % 1.0))) for i in range(n)]


def _sequences(case):
    """[(prompt, length of its own)] of each sequence, in the order of the batch."""
    if case["prompts"] == 1:
        many = [case["answers"]]
    else:
        many = _spread(case["prompts"], 1, case["answers"])
    which = [p for p, n in enumerate(many) for _ in range(n)]
    seqs = list(zip(which, _spread(len(which), case["new"], case["own"])))
    if case["mixed"]:                                        # a stride that visits each once
        n = len(seqs)
        step = next(s for s in range(max(2, round(0.381966 * n)), n + 3) if math.gcd(s, n) == 1)
        seqs = [seqs[i * step % n] for i in range(n)]
    return seqs


def work(case):
    if case["op"] == "attend":
        seqs, new, window, prefix = _sequences(case), case["new"], case["window"], case["prefix"]
        numbers, read, pairs, first = case["kv"] * case["dim"], 0, 0, {}
        for p, tail in seqs:
            n = prefix + tail
            lowest = max(0, n - new + 1 - window) if window else 0          # the lowest key that the sequence's rows see
            first[p] = min(first.get(p, prefix), lowest)
            read += n - max(prefix, lowest)
            for j in range(new):
                pairs += min(n - new + j + 1, window or n)
        read += sum(prefix - lowest for lowest in first.values())           # a prompt's keys count once
        return {"bytes": 4 * read * numbers + 4 * len(seqs) * new * case["heads"] * case["dim"], "flops": 4 * pairs * case["heads"] * case["dim"]}
    if case["op"] == "logprobs":
        return {"bytes": 4 * case["rows"] * case["vocab"] + case["rows"] * (12 + 8 * case["top"]), "flops": 8 * case["rows"] * case["vocab"]}
    return {"bytes": 2 * (case["rows"] + case["vocab"]) * case["width"] + 12 * case["rows"], "flops": 2 * case["rows"] * case["vocab"] * case["width"]}


# ---- inputs -----------------------------------------------------------------------------------------------------
def _rows(gen, *shape):
    """Activations: most numbers near 1, some channels several times as large."""
    channel = 1 + 4 * (torch.rand(shape[-1], generator=gen, device=DEV) < 0.02)
    return (torch.randn(*shape, generator=gen, device=DEV) * channel).to(torch.bfloat16)


def _made(case, seed):
    """The inputs that both forms and the exact one start from."""
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    if case["op"] == "attend":
        seqs = _sequences(case)
        width, total = case["kv"] * case["dim"], sum(n for _, n in seqs)
        made = {"q": _rows(gen, len(seqs) * case["new"], case["heads"] * case["dim"])}
        for name in ("k", "v"):
            made[name] = _rows(gen, case["prompts"], case["prefix"], width)
            made["own_" + name] = _rows(gen, total, width)
        return made
    rows, vocab = case["rows"], case["vocab"]
    tokens = torch.randint(0, vocab, (rows,), generator=gen, device=DEV)
    if case["op"] == "logprobs":
        # most rows are sure of a few tokens, some of none; half of the given tokens are among those
        logits = torch.randn(rows, vocab, generator=gen, device=DEV).mul_(2.0)
        peaks = torch.randint(0, vocab, (rows, 8), generator=gen, device=DEV)
        logits.scatter_add_(1, peaks, 15 * torch.rand(rows, 8, generator=gen, device=DEV) * (torch.rand(rows, 1, generator=gen, device=DEV) < 0.8))
        if case["masked"]:
            logits[:, torch.rand(vocab, generator=gen, device=DEV) < 0.3] = -math.inf
        tokens = torch.where(torch.rand(rows, generator=gen, device=DEV) < 0.5, peaks[:, 0], tokens)
        return {"logits": logits, "tokens": tokens.to(torch.int32)}
    width = case["width"]
    head = torch.empty(vocab, width, dtype=torch.bfloat16, device=DEV).normal_(0.0, 0.02, generator=gen)
    sure = 12 * torch.rand(rows, 1, generator=gen, device=DEV) / (0.02 * width)        # logits of up to about 12
    likely = torch.randint(0, vocab, (rows,), generator=gen, device=DEV)
    h = torch.randn(rows, width, generator=gen, device=DEV) + sure * head[likely].float() / 0.02
    tokens = torch.where(torch.rand(rows, generator=gen, device=DEV) < 0.7, likely, tokens)
    return {"h": h.to(torch.bfloat16), "head": head, "tokens": tokens.to(torch.int32)}


def prepare(case, seed):
    made = _made(case, seed)
    state = {"case": case, **made}
    if case["op"] != "attend":
        return state
    seqs, new, prefix = _sequences(case), case["new"], case["prefix"]
    if own:
        state["cache"], state["step"], state["plan"] = _forked(case, seqs, made)
        state["out"] = torch.empty_like(made["q"])
        del state["k"], state["v"], state["own_k"], state["own_v"]
        return state
    # each prompt's sequences, and each sequence's own rows, padded to the most
    by_prompt = [[i for i, (p, _) in enumerate(seqs) if p == q] for q in range(case["prompts"])]
    most, longest = max(len(b) for b in by_prompt), max(n for _, n in seqs)
    at, base = torch.zeros(len(seqs), longest, dtype=torch.long), 0
    for i, (_, n) in enumerate(seqs):
        at[i, :n] = torch.arange(base, base + n)
        base += n
    state["at"] = at.to(DEV)
    state["members"] = torch.tensor([b + [b[0]] * (most - len(b)) for b in by_prompt], device=DEV)
    place = {i: (q, j) for q, b in enumerate(by_prompt) for j, i in enumerate(b)}
    state["place"] = torch.tensor([place[i][0] * most + place[i][1] for i in range(len(seqs))], device=DEV)
    state["first"] = torch.tensor([prefix + n - new for _, n in seqs], device=DEV)      # position of each sequence's first row
    return state


def _forked(case, seqs, made):
    """A cache of one layer whose sequences were forked from their prompts, and the step that brings their last rows: what a program
    has after it ran the prompts, forked them and went on."""
    from hos_b200 import ops
    from hos_b200.cache import CacheManager
    from hos_b200.engine.batch import build_step
    from hos_b200.parts import shared_attention
    from hos_b200.parts.base import KVNeed
    dev, prefix = torch.device(DEV), case["prefix"]
    pages = case["prompts"] * (-(-prefix // PAGE)) + sum(-(-n // PAGE) + 1 for _, n in seqs)
    cache = CacheManager([KVNeed(case["kv"], case["dim"], case["window"] or None)], [None], [[]], pages * PAGE, prefix + max(n for _, n in seqs),
                         torch.bfloat16, dev, max_slots=len(seqs), chunk_tokens=max(case["own"], case["new"]))
    view = cache.stores[0].kv

    def bring(slots, starts, counts, k, v):
        cache.extend_all(slots, [s + n for s, n in zip(starts, counts)])
        cache.flush()
        step = build_step([[0] * n for n in counts], starts, slots, dev, 1)
        ops.rope_kv_write(torch.cat([k, v], dim=1), 0, step.token_pos, step.token_seq, step.seq_slot, step.seq_len_after, None, 0, 0, view, case["kv"],
                          case["dim"])

    roots = cache.admit([0] * case["prompts"])
    bring(roots, [0] * len(roots), [prefix] * len(roots), made["k"].flatten(0, 1), made["v"].flatten(0, 1))
    waiting = [[r] + cache.fork(r, sum(p == q for p, _ in seqs) - 1) for q, r in enumerate(roots)]
    slots = [waiting[p].pop() for p, _ in seqs]
    tails = [n for _, n in seqs]
    bring(slots, [prefix] * len(slots), tails, made["own_k"], made["own_v"])
    new = case["new"]
    step = build_step([[0] * new] * len(slots), [prefix + n - new for n in tails], slots, dev, 1)
    return view, step, shared_attention.plan(cache.groups[0], step)


# ---- one pass ---------------------------------------------------------------------------------------------------
def run(state):
    return _own(state) if own else _plain(state)


def _own(state):
    case = state["case"]
    if case["op"] == "attend":
        from hos_b200.parts import shared_attention
        shared_attention.attend(state["q"], state["out"], state["step"], state["cache"], state["plan"], case["heads"], case["dim"] ** -0.5, case["cap"],
                                case["window"] or None)
        return state["out"]
    if case["op"] == "logprobs":
        from hos_b200.sampling import log_probs
        got = log_probs(state["logits"], state["tokens"], case["top"])
        return [got.logprob, got.entropy] + ([got.top_ids, got.top_logprobs] if case["top"] else [])
    from hos_b200.parts import linear
    got = linear.log_probs(state["h"], state["head"], state["tokens"], cap=case["cap"])
    return [got.logprob, got.entropy]


def _token_scores(logits, tokens):
    """(log probability of the given token, entropy, log of the sum of exponentials) of each row, the long sums in 64 bits."""
    top = logits.amax(dim=1, keepdim=True)
    shifted = logits - top
    e = torch.exp(shifted)
    total = e.sum(dim=1, dtype=torch.float64)
    weighted = torch.where(e > 0, e * shifted, 0.0).sum(dim=1, dtype=torch.float64)
    log_total = torch.log(total)
    logprob = shifted.gather(1, tokens.long()[:, None])[:, 0].double() - log_total
    return logprob.float(), (log_total - weighted / total).float(), top[:, 0].double() + log_total


def _plain(state):
    case = state["case"]
    if case["op"] == "logprobs":
        logprob, entropy, norm = _token_scores(state["logits"], state["tokens"])
        if not case["top"]:
            return [logprob, entropy]
        values, ids = torch.sort(state["logits"], dim=1, descending=True, stable=True)
        best = values[:, :case["top"]].double() - norm[:, None]
        return [logprob, entropy, ids[:, :case["top"]].to(torch.int32), best.float()]
    if case["op"] == "score":
        logits = state["h"].float() @ state["head"].float().T
        if case["cap"]:
            logits = case["cap"] * torch.tanh(logits / case["cap"])
        return list(_token_scores(logits, state["tokens"])[:2])
    new, kv, dim, prefix, window = case["new"], case["kv"], case["dim"], case["prefix"], case["window"]
    per, seqs = case["heads"] // kv, state["first"].shape[0]
    q = state["q"].float().view(seqs, new, kv, per, dim).permute(0, 2, 3, 1, 4).reshape(seqs, kv, per * new, dim)
    at = state["first"][:, None] + torch.arange(new, device=DEV)                               # [seqs, new]: each row's position

    def score(rows, keys):
        s = rows @ keys.transpose(-1, -2) * dim ** -0.5
        return case["cap"] * torch.tanh(s / case["cap"]) if case["cap"] else s

    def hidden(position):                                                                      # of [keys], for [seqs, new] rows
        d = at[..., None] - position
        return (d < 0) | (d >= window) if window else d < 0

    # the prompts' keys, all sequences of a prompt together
    members = state["members"]
    k, v = (state[name].float().unflatten(-1, (kv, dim)).transpose(1, 2) for name in ("k", "v"))      # [prompts, kv, prefix, dim]
    rows = q[members].permute(0, 2, 1, 3, 4).flatten(2, 3)                                      # [prompts, kv, members * per * new, dim]
    over = score(rows, k).view(*rows.shape[:2], members.shape[1], per, new, prefix)
    over = over.masked_fill(hidden(torch.arange(prefix, device=DEV))[members][:, None, :, None], -math.inf)
    # each sequence's own keys
    k_own, v_own = (state["own_" + name].float()[state["at"]].unflatten(-1, (kv, dim)).transpose(1, 2) for name in ("k", "v"))
    mine = score(q, k_own).view(seqs, kv, per, new, -1)
    mine = mine.masked_fill(hidden(prefix + torch.arange(k_own.shape[2], device=DEV))[:, None, None], -math.inf)
    # one softmax over both
    back = lambda t: t.transpose(1, 2).flatten(0, 1)[state["place"]]                            # noqa: E731  to [seqs, kv, per, new, ..]
    top = torch.maximum(back(over.amax(-1)), mine.amax(-1))
    p_own = torch.exp(mine - top[..., None])
    p_over = torch.exp(over - top[members].transpose(1, 2)[..., None])
    total = back(p_over.sum(-1)) + p_own.sum(-1)
    out = back((p_over.flatten(2, 4) @ v).view(*over.shape[:-1], dim)) + (p_own.flatten(2, 3) @ v_own).view(seqs, kv, per, new, dim)
    out = (out / total[..., None]).permute(0, 3, 1, 2, 4)
    return out.reshape(seqs * new, -1).to(state["q"].dtype)


# ---- the same in 64 bits ----------------------------------------------------------------------------------------
def exact(case, seed):
    made = _made(case, seed)
    if case["op"] == "attend":
        kv, dim, new, prefix, out, base = case["kv"], case["dim"], case["new"], case["prefix"], [], 0
        for i, (p, tail) in enumerate(_sequences(case)):                    # sequence by sequence, all of its keys in a row
            k, v = (torch.cat([made[name][p], made["own_" + name][base:base + tail]]).double().view(-1, kv, dim) for name in ("k", "v"))
            base += tail
            n = prefix + tail
            q = made["q"][i * new:(i + 1) * new].double().view(new, kv, -1, dim)
            s = torch.einsum("ngpd,kgd->ngpk", q, k) / math.sqrt(dim)
            if case["cap"]:
                s = torch.tanh(s / case["cap"]) * case["cap"]
            back = torch.arange(n - new, n, device=DEV)[:, None] - torch.arange(n, device=DEV)
            unseen = (back < 0) if not case["window"] else (back < 0) | (back >= case["window"])
            s[unseen[:, None, None].expand_as(s)] = -math.inf
            out.append(torch.einsum("ngpk,kgd->ngpd", s.softmax(-1), v).reshape(new, -1))
        return torch.cat(out)
    tokens, found = made["tokens"].long(), []
    for lo in range(0, case["rows"], 128):                                  # some rows at a time
        if case["op"] == "logprobs":
            logits = made["logits"][lo:lo + 128].double()
        else:
            h = made["h"][lo:lo + 128].double()
            logits = torch.cat([h @ w.double().T for w in made["head"].split(16384)], dim=1)
            if case["cap"]:
                logits = torch.tanh(logits / case["cap"]) * case["cap"]
        logp = torch.log_softmax(logits, dim=1)
        rows = [logp.gather(1, tokens[lo:lo + 128, None])[:, 0], torch.special.entr(logp.exp()).sum(1)]
        if case.get("top"):
            # the likeliest, one after another; of equal ones the first
            ids, left = [], logits.clone()
            for _ in range(case["top"]):
                best = left.amax(1, keepdim=True)
                at = torch.where(left == best, torch.arange(left.shape[1], device=DEV), left.shape[1]).amin(1)
                ids.append(at)
                left.scatter_(1, at[:, None], -math.inf)
            ids = torch.stack(ids, dim=1)
            rows += [ids.to(torch.int32), logp.gather(1, ids)]
        found.append(rows)
    return [torch.cat(parts) for parts in zip(*found)]
