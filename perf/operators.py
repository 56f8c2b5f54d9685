"""What is measured of the low-bit operators: products with 4-bit weights, keys and values put into 4-bit pages, attention over
them, and pages copied inside a cache.

A case names its operator:

  product   x . W^T with W in 4-bit codes, a scale (and, with `zeros`, a zero code) per `group` weights of a row; `gated`: gelu(gate) * up of
            two such matrices.  w = (c - z) s, z = 8 without zeros
  store     rows of keys and values into 4-bit pages: per 64 numbers of a head s = bf16((max - min) / 15), m = bf16(min + 8 s),
            c = clamp(rint((x - m) / s), -8, 7); what is held is c s + m
  attend    softmax attention of the last `new` tokens of each sequence over its held keys and values, causal, with an optional window
            and soft-cap
  pages     pages copied to other pages, in every array of a group of layers

Sizes are those of Gemma-2 at 2B, 9B and 27B (layer widths, heads, pages), and odd ones.
"""
from __future__ import annotations

import math

import torch

own = False

GROUP = 64                  # numbers of a head that share a scale in the cache
PAGE = 64                   # positions of a page
DEV = "cuda"
TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
BYTES = {"bf16": 2, "f32": 4}


# ---- cases ------------------------------------------------------------------------------------------------------
def _product(rows, n, k, group, zeros, gated, dtype):
    return dict(op="product", rows=rows, n=n, k=k, group=group, zeros=zeros, gated=gated, dtype=dtype)


def _store(rows, kv, dim, dtype):
    return dict(op="store", rows=rows, kv=kv, dim=dim, dtype=dtype)


def _attend(seqs, longest, new, heads, kv, dim, window, cap, ragged, dtype):
    return dict(op="attend", seqs=seqs, longest=longest, new=new, heads=heads, kv=kv, dim=dim, window=window, cap=cap, ragged=ragged, dtype=dtype)


def _pages(arrays, pages, copies, kv, dim, dtype):
    return dict(op="pages", arrays=arrays, pages=pages, copies=copies, kv=kv, dim=dim, dtype=dtype)


def listed():
    return [
        # one sequence's next token: the down projection of a 2B layer
        dict(_product(1, 2304, 9216, 64, False, False, "bf16"), name="product-1-down"),
        # eight sequences' next tokens: gate and up of a 27B layer
        dict(_product(8, 36864, 4608, 128, False, True, "bf16"), name="product-8-gate-up"),
        # five rows in 32-bit arithmetic, sizes that fill no tile, groups of 32 with zero codes
        dict(_product(5, 2051, 1999, 32, True, False, "f32"), name="product-5-odd-f32"),
        # a prompt of 512 tokens: gate and up of a 9B layer
        dict(_product(512, 14336, 3584, 128, True, True, "bf16"), name="product-512-gate-up"),
        # a decode step of eight sequences stores a token each
        dict(_store(8, 4, 256, "bf16"), name="store-8"),
        # prompts of 8,192 tokens in all, 27B heads
        dict(_store(8192, 16, 128, "bf16"), name="store-8192"),
        # one sequence's next token early in a chat
        dict(_attend(1, 1000, 1, 8, 4, 256, 0, 50.0, False, "bf16"), name="attend-1-short"),
        # eight long sequences side by side
        dict(_attend(8, 8192, 1, 8, 4, 256, 0, 50.0, False, "bf16"), name="attend-8-long"),
        # many sequences of unequal lengths, 27B heads, a layer with a window
        dict(_attend(48, 8000, 1, 32, 16, 128, 4096, 50.0, True, "bf16"), name="attend-48-ragged"),
        # a second turn of 739 tokens on top of a long first one
        dict(_attend(1, 8192, 739, 8, 4, 256, 0, 50.0, False, "bf16"), name="attend-turn-739"),
        # a conversation is forked: its last page is copied in the 13 layers of a 2B group
        dict(_pages(26, 64, 1, 4, 256, "bf16"), name="pages-fork"),
        # a cache is compacted: 100 pages move, 23 layers of 27B heads
        dict(_pages(46, 220, 100, 16, 128, "bf16"), name="pages-compact"),
    ]


def _between(rng, lo, hi):
    """A whole number between lo and hi, spread over the logarithm."""
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    most = [work(c) for c in listed()]
    while True:
        op = rng.choice(["product", "store", "attend", "pages"])
        dtype = rng.choice(["bf16", "bf16", "f32"])
        if op == "product":
            case = _product(_between(rng, 1, 512), _between(rng, 16, 36864), _between(rng, 64, 16384), rng.choice([32, 64, 128]),
                            rng.random() < 0.5, rng.random() < 0.4, dtype)
        elif op == "store":
            case = _store(_between(rng, 1, 8192), rng.choice([1, 2, 4, 8, 16]), rng.choice([64, 128, 256]), dtype)
        elif op == "attend":
            kv, longest = rng.choice([1, 2, 4, 8, 16]), _between(rng, 1, 32768)
            new = 1 if rng.random() < 0.7 else min(longest, _between(rng, 2, 1024))
            case = _attend(_between(rng, 1, 64), longest, new, kv * rng.choice([1, 2, 2, 4, 5, 8, 16]), kv, rng.choice([64, 128, 256]),
                           rng.choice([0, 0, 1024, 4096]), rng.choice([0.0, 50.0]), rng.random() < 0.5, dtype)
            # the plain form holds every pair's score and all keys and values in 32 bits
            if case["seqs"] * case["heads"] * longest * new > 1.5e8 or case["seqs"] * longest * kv * case["dim"] > 8.5e8:
                continue
        else:
            pages = _between(rng, 2, 512)
            case = _pages(2 * rng.randint(1, 23), pages, _between(rng, 1, pages // 2), rng.choice([1, 2, 4, 8, 16]), rng.choice([64, 128, 256]), dtype)
            if case["arrays"] * pages * case["kv"] * PAGE * case["dim"] * BYTES[dtype] > 2.7e9:
                continue
        w, like = work(case), [m for c, m in zip(listed(), most) if c["op"] == op]
        if w["bytes"] <= max(m["bytes"] for m in like) and w["flops"] <= max(m["flops"] for m in like):
            return case


def _lengths(case):
    """Each sequence's length after the step: all the longest, or spread over 1..longest in no order (but sequences that held nothing
    before the step come first, as in every step)."""
    if not case["ragged"]:
        return [case["longest"]] * case["seqs"]
    spread = [max(case["new"], round(case["longest"] * (1.0 - (0.6180339887 * i) % 1.0))) for i in range(case["seqs"])]
    return sorted(spread, key=lambda n: n > case["new"])


def work(case):
    e = BYTES[case["dtype"]]
    if case["op"] == "product":
        n = case["n"] * (2 if case["gated"] else 1)
        groups = -(-case["k"] // case["group"])
        return {"bytes": n * case["k"] / 2 + n * groups * (2.5 if case["zeros"] else 2) + case["rows"] * (case["k"] + case["n"]) * e,
                "flops": 2 * case["rows"] * n * case["k"]}
    numbers = case["kv"] * case["dim"]
    held = 0.5 + 4 / GROUP                      # bytes a number: half a byte of code, scale and middle per 64
    if case["op"] == "store":                   # rows read, pages written, what is held handed back
        return {"bytes": 2 * case["rows"] * numbers * (2 * e + held), "flops": 2 * case["rows"] * numbers * 8}
    if case["op"] == "attend":
        new, window = case["new"], case["window"]
        read = pairs = 0
        for n in _lengths(case):
            read += min(n, window + new - 1) if window else n
            for j in range(new):
                pairs += min(n - new + j + 1, window or n)
        return {"bytes": 2 * read * numbers * held + 2 * case["seqs"] * new * case["heads"] * case["dim"] * e,
                "flops": 4 * pairs * case["heads"] * case["dim"]}
    return {"bytes": 2 * case["arrays"] * case["copies"] * PAGE * numbers * e, "flops": 0}


# ---- inputs -----------------------------------------------------------------------------------------------------
def _quantise_weights(w, group, zeros):
    """Codes 0..15 [n, k] (uint8), scales [n, groups] (bfloat16), zero codes [n, groups] (uint8) or None."""
    n, k = w.shape
    pad = -k % group
    g = torch.nn.functional.pad(w, (0, pad)).view(n, -1, group)
    if zeros:
        lo, hi = g.amin(-1).clamp(max=0), g.amax(-1).clamp(min=0)
        s = ((hi - lo) / 15).clamp(min=1e-8).to(torch.bfloat16)
        z = torch.round(-lo / s.float()).clamp(0, 15)
    else:
        s = (g.abs().amax(-1) / 7).clamp(min=1e-8).to(torch.bfloat16)
        z = torch.full_like(s, 8, dtype=torch.float32)
    c = torch.round(g / s.float()[..., None] + z[..., None]).clamp_(0, 15).to(torch.uint8)
    return c.view(n, -1)[:, :k].contiguous(), s, (z.to(torch.uint8) if zeros else None)


def _quantise_rows(x):
    """(codes -8..7, scales, middles) of rows [..., dim] in groups of 64, in 32 bits: the format's definition."""
    g = x.float().unflatten(-1, (-1, GROUP))
    lo, hi = g.amin(-1), g.amax(-1)
    s = ((hi - lo) / torch.full((), 15.0, device=x.device)).to(torch.bfloat16).float()
    m = (lo + 8 * s).to(torch.bfloat16).float()
    c = torch.round((g - m[..., None]) / torch.where(s > 0, s, 1.0)[..., None]).clamp_(-8, 7)
    return c.to(torch.int8), s, m


def _held(c, s, m):
    return (c.float() * s[..., None] + m[..., None]).flatten(-2)


def _rows(case, gen, n, out_dim):
    """Activations: most numbers near 1, some channels several times as large."""
    channel = 1 + 4 * (torch.rand(out_dim, generator=gen, device=DEV) < 0.02)
    return (torch.randn(n, out_dim, generator=gen, device=DEV) * channel).to(TYPES[case["dtype"]])


def _made(case, seed):
    """The inputs that both forms and the exact one start from."""
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    op = case["op"]
    if op == "product":
        parts = 2 if case["gated"] else 1
        made = [_quantise_weights(torch.randn(case["n"], case["k"], generator=gen, device=DEV) * case["k"] ** -0.5, case["group"], case["zeros"])
                for _ in range(parts)]
        codes, scales = torch.cat([m[0] for m in made]), torch.cat([m[1] for m in made])
        zeros = torch.cat([m[2] for m in made]) if case["zeros"] else None
        return {"x": _rows(case, gen, case["rows"], case["k"]), "codes": codes, "scales": scales, "zeros": zeros}
    if op == "store":
        return {"rows": _rows(case, gen, case["rows"], 2 * case["kv"] * case["dim"])}
    if op == "attend":
        lens, width = _lengths(case), case["kv"] * case["dim"]
        total = sum(lens)
        q = _rows(case, gen, case["seqs"] * case["new"], case["heads"] * case["dim"])
        return {"lens": lens, "q": q, "k": _rows(case, gen, total, width), "v": _rows(case, gen, total, width)}
    order = torch.randperm(case["pages"], generator=gen, device=DEV).to(torch.int32)
    shape = (case["arrays"], case["pages"], case["kv"], PAGE, case["dim"])
    data = torch.empty(shape, dtype=TYPES[case["dtype"]], device=DEV)
    for a in data:
        a.normal_(generator=gen)
    return {"data": data, "src": order[:case["copies"]].contiguous(), "dst": order[case["copies"]:2 * case["copies"]].contiguous()}


def prepare(case, seed):
    made = _made(case, seed)
    state = {"case": case, **made}
    op = case["op"]
    if op == "product":
        if own:
            from hos_b200.parts.weights4 import Weight4
            state["w"] = Weight4.from_codes(made["codes"], made["scales"], made["zeros"], case["group"], blocks=2 if case["gated"] else 1)
            del state["codes"], state["scales"], state["zeros"]
    elif op == "store":
        state["held"] = torch.empty_like(made["rows"])
        if own:
            state["step"], state["cache"] = _cache(case, [case["rows"]], [case["rows"]])
    elif op == "attend":
        del state["k"], state["v"]
        new, lens = case["new"], made["lens"]
        if own:
            from hos_b200.parts import attention4
            fill, cache = _cache(case, lens, lens)
            attention4.store(torch.cat([made["k"], made["v"]], dim=1), fill, cache)
            state["step"], state["cache"] = _step(lens, [new] * len(lens)), cache
            state["out"] = torch.empty_like(made["q"])
        else:
            # every sequence's rows from its first position on, padded to the longest
            at = torch.zeros(len(lens), max(lens), dtype=torch.long, device=DEV)
            base = 0
            for i, n in enumerate(lens):
                at[i, :n] = torch.arange(base, base + n, device=DEV)
                base += n
            for name in ("k", "v"):
                c, s, m = _quantise_rows(made[name].unflatten(-1, (case["kv"], case["dim"])))
                state[name] = (c[at], s[at], m[at])
            state["len"] = torch.tensor(lens, device=DEV)
    elif own:
        from hos_b200.cache import CacheManager
        from hos_b200.parts.base import KVNeed
        cache = CacheManager([KVNeed(case["kv"], case["dim"], None)] * (case["arrays"] // 2), [None] * (case["arrays"] // 2),
                             [[]] * (case["arrays"] // 2), case["pages"] * PAGE, case["pages"] * PAGE, TYPES[case["dtype"]], torch.device(DEV))
        state["group"] = cache.groups[0]
        for mine, a in zip(state["group"].k + state["group"].v, made["data"]):
            mine.copy_(a)
        del state["data"]
    return state


def _step(lens, news):
    """The step that brings the last `news` tokens of sequences 0, 1, ...: what the framework's step function hands to its parts."""
    from hos_b200.engine.batch import build_step
    return build_step([[0] * n for n in news], [n - k for n, k in zip(lens, news)], list(range(len(lens))), torch.device(DEV), 1)


def _cache(case, lens, news):
    """A cache of one layer in 4 bits with room for the sequences, and the step that fills it."""
    from hos_b200.cache import CacheManager
    from hos_b200.parts.base import KVNeed
    room = sum(-(-n // PAGE) * PAGE for n in lens)
    cache = CacheManager([KVNeed(case["kv"], case["dim"], None, bits=4)], [None], [[]], room, room, TYPES[case["dtype"]], torch.device(DEV),
                         max_slots=len(lens))
    cache.extend_all(cache.admit([0] * len(lens)), lens)
    cache.flush()
    return _step(lens, news), cache.stores[0].kv


# ---- one pass ---------------------------------------------------------------------------------------------------
def run(state):
    return _own(state) if own else _plain(state)


def _own(state):
    case = state["case"]
    op = case["op"]
    if op == "product":
        from hos_b200 import ops
        from hos_b200.parts import linear
        if case["gated"]:
            return linear.matmul(state["x"], state["w"], epilogue=ops.EPI_GATED, act=ops.ACT_GELU_TANH)
        return linear.matmul(state["x"], state["w"])
    if op == "store":
        from hos_b200.parts import attention4
        attention4.store(state["rows"], state["step"], state["cache"], held=state["held"])
        return state["held"]
    if op == "attend":
        from hos_b200.parts import attention4
        attention4.attend(state["q"], state["out"], state["step"], state["cache"], case["heads"], case["dim"] ** -0.5, case["cap"], case["window"] or None)
        return state["out"]
    state["group"].copy_pages(state["src"], state["dst"])
    return state["group"].k + state["group"].v


def _plain(state):
    case = state["case"]
    op = case["op"]
    if op == "product":
        zeros = state["zeros"].float() if case["zeros"] else torch.full_like(state["scales"], 8, dtype=torch.float32)
        w = state["codes"].float()
        z, s = (t.repeat_interleave(case["group"], dim=1)[:, :case["k"]] for t in (zeros, state["scales"].float()))
        y = state["x"].float() @ ((w - z) * s).T
        if case["gated"]:
            gate, up = y[:, :case["n"]], y[:, case["n"]:]
            y = 0.5 * gate * (1 + torch.tanh(math.sqrt(2 / math.pi) * (gate + 0.044715 * gate ** 3))) * up
        return y.to(state["x"].dtype)
    if op == "store":
        state["held"].copy_(_held(*_quantise_rows(state["rows"])))
        return state["held"]
    if op == "attend":
        b, new, kv, dim = case["seqs"], case["new"], case["kv"], case["dim"]
        per = case["heads"] // kv
        k, v = (_held(*state[name]).permute(0, 2, 1, 3) for name in ("k", "v"))              # [b, kv, keys, dim]
        q = state["q"].float().view(b, new, kv, per, dim).permute(0, 2, 3, 1, 4).reshape(b, kv, per * new, dim)
        score = q @ k.transpose(2, 3) * dim ** -0.5
        if case["cap"]:
            score = case["cap"] * torch.tanh(score / case["cap"])
        key = torch.arange(k.shape[2], device=DEV)
        at = state["len"][:, None] - new + torch.arange(new, device=DEV)                       # [b, new]: each query's position
        seen = key <= at[..., None]
        if case["window"]:
            seen = seen & (key > at[..., None] - case["window"])
        score = score.view(b, kv, per, new, -1).masked_fill(~seen[:, None, None], -math.inf)
        p = torch.exp(score - score.amax(-1, keepdim=True))
        p = (p / p.sum(-1, keepdim=True)).view(b, kv, per * new, -1)
        out = (p @ v).view(b, kv, per, new, dim).permute(0, 3, 1, 2, 4)
        return out.reshape(b * new, -1).to(state["q"].dtype)
    state["data"][:, state["dst"].long()] = state["data"][:, state["src"].long()]
    return list(state["data"].unbind(0))


# ---- the same in 64 bits ----------------------------------------------------------------------------------------
def exact(case, seed):
    made = _made(case, seed)
    op = case["op"]
    if op == "product":
        x, rows = made["x"].double(), made["codes"].shape[0]
        if case["rows"] * rows * case["k"] > 2e11:
            return None
        y = torch.zeros(case["rows"], rows, dtype=torch.float64, device=DEV)
        for g in range(made["scales"].shape[1]):                    # group by group: the codes' product, then the scale
            lo, hi = g * case["group"], min(case["k"], (g + 1) * case["group"])
            part = x[:, lo:hi] @ made["codes"][:, lo:hi].double().T
            zero = made["zeros"][:, g].double() if case["zeros"] else 8.0
            y += (part - x[:, lo:hi].sum(1, keepdim=True) * zero) * made["scales"][:, g].double()
        if case["gated"]:
            gate, up = y.split(case["n"], dim=1)
            return torch.nn.functional.gelu(gate, approximate="tanh") * up
        return y
    if op == "store":
        x = made["rows"].double()
        g = x.reshape(x.shape[0], -1, GROUP)
        lo, hi = g.min(-1).values, g.max(-1).values
        s = ((hi - lo) / 15).to(torch.bfloat16).double()
        m = (lo + 8 * s).to(torch.bfloat16).double()
        c = ((g - m.unsqueeze(-1)) / s.clamp(min=1e-300).unsqueeze(-1)).round().clamp(-8, 7)
        return (c * s.unsqueeze(-1) + m.unsqueeze(-1)).reshape(x.shape)
    if op == "attend":
        new, kv, dim, per = case["new"], case["kv"], case["dim"], case["heads"] // case["kv"]
        out, base = [], 0
        for i, n in enumerate(made["lens"]):                        # sequence by sequence, query by query block
            k, v = (_held(*_quantise_rows(made[name][base:base + n].unflatten(-1, (kv, dim)))).double() for name in ("k", "v"))
            base += n
            q = made["q"][i * new:(i + 1) * new].double().view(new, kv, per, dim)
            score = torch.einsum("nkpd,lkd->nkpl", q, k) / math.sqrt(dim)
            if case["cap"]:
                score = torch.tanh(score / case["cap"]) * case["cap"]
            dist = torch.arange(n - new, n, device=DEV)[:, None] - torch.arange(n, device=DEV)
            hidden = (dist < 0) | (dist >= case["window"] if case["window"] else dist < 0)
            score[hidden[:, None, None].expand_as(score)] = -math.inf
            out.append(torch.einsum("nkpl,lkd->nkpd", score.softmax(-1), v).reshape(new, -1))
        return torch.cat(out)
    return [a.clone() for a in _moved(made)]


def _moved(made):
    for a in made["data"]:
        for s, d in zip(made["src"].tolist(), made["dst"].tolist()):
            a[d] = a[s]
        yield a
