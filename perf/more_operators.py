"""Cases of 8-bit projections and of token scores: rows normalised into 8 bits, weights in 8-bit blocks, their product, and
what a vocabulary's logits say about given tokens.

A projection of a prompt or a batch in 8 bits, and the end of a scoring pass:

  rows     h = x + add, y = h / sqrt(mean h^2 + eps) * weight (each of the two may be left out), and y as e4m3 codes with a
           scale for each 128 adjacent values of a row
  blocks   a weight matrix as e4m3 codes with a scale for each 128 x 128 block
  product  out = rows weight^T (+ add), each 128-deep part of a sum taking its row's and its block's scale
  tokens   of every row of logits: the log probability and rank of a given token, the entropy, and the best alternatives

A group's scale is a / 448 with a = max(|y|, 2^-116) over the group, a code is y * (448 / a) rounded to e4m3 (to nearest, ties to
even) and stands for code * scale. The row's sum h is rounded to its type before it is normalised, as the next layer reads it.

Tokens: entries at -inf have no probability and are no alternatives; alternatives go by their logits, equal ones by the lower
index (-0 equals +0), and places that stay empty hold -1 and -inf. rank counts the entries before the token in that order. A token
below zero is none: 0 and rank -1. A row of nothing but -inf: log probabilities -inf, entropy 0.

`run` with `own` false is the plain form in elementary torch operations; with `own` true, the calls of a user.
"""

import math
import os
import sys

import torch

own = False

GROUP = 128
TINY = 2.0 ** -116
_kept = {}  # what a program keeps for its life: the library


def listed():
    return [
        # one token's decode step: the mixer's output joins the residual, normalised for the MoE layer's projections
        dict(name="rows_1", kind="rows", rows=1, cols=2048, dtype="f32", add=True, norm=True, normed=True, pad=0),
        # the output of a mixer without a norm, cut from a wider buffer; columns that end inside a group
        dict(name="rows_ragged", kind="rows", rows=777, cols=1744, dtype="bf16", add=False, norm=False, normed=False, pad=48),
        # a prompt's rows before a projection
        dict(name="rows_prompt", kind="rows", rows=8192, cols=4096, dtype="bf16", add=True, norm=True, normed=False, pad=0),
        # a router's weight, laid out once: rows that end inside a block
        dict(name="blocks_513", kind="blocks", rows=513, cols=2048, dtype="f32"),
        # an input projection's weight
        dict(name="blocks_12352", kind="blocks", rows=12352, cols=2048, dtype="bf16"),
        # the input projection of one token
        dict(name="product_1", kind="product", m=1, n=12352, k=2048, dtype="f32", add=False),
        # the head of a batch's decode step
        dict(name="product_head_32", kind="product", m=32, n=151936, k=2048, dtype="f32", add=False),
        # the output projection of a short prompt, added into the residual
        dict(name="product_add_333", kind="product", m=333, n=2048, k=4096, dtype="f32", add=True),
        # the input projection of a long prompt
        dict(name="product_prompt", kind="product", m=8192, n=12352, k=2048, dtype="bf16", add=False),
        # the chosen token of one decode step with its alternatives
        dict(name="tokens_1", kind="tokens", rows=1, vocab=151936, dtype="f32", top=20, pad=0, masked=False),
        # a batch's step under a grammar: most of the vocabulary masked, one row's mask leaves nothing
        dict(name="tokens_32", kind="tokens", rows=32, vocab=151936, dtype="f32", top=5, pad=0, masked=True),
        # scoring a long prompt
        dict(name="tokens_2048", kind="tokens", rows=2048, vocab=151936, dtype="bf16", top=20, pad=0, masked=False),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    kind = rng.choice(["rows", "blocks", "product", "product", "tokens", "tokens"])
    dtype = rng.choice(["f32", "bf16"])
    if kind == "rows":
        norm = rng.random() < 0.7
        return dict(kind=kind, rows=_log(rng, 1, 8192), cols=16 * _log(rng, 1, 256), dtype=dtype, add=rng.random() < 0.6, norm=norm,
                    normed=norm and rng.random() < 0.4, pad=16 * rng.choice([0, 0, 1, 5]))
    if kind == "blocks":
        return dict(kind=kind, rows=_log(rng, 1, 12352), cols=16 * _log(rng, 1, 256), dtype=dtype)
    if kind == "product":
        while True:
            m, n, k = _log(rng, 1, 8192), _log(rng, 1, 151936), 16 * _log(rng, 1, 512)
            if m * n * k <= 8192 * 12352 * 2048 and n * k <= 151936 * 2048 and m * n <= 1 << 28:
                return dict(kind=kind, m=m, n=n, k=k, dtype=dtype, add=rng.random() < 0.4)
    return dict(kind=kind, rows=_log(rng, 1, 2048), vocab=_log(rng, 1, 151936), dtype=dtype, top=rng.choice([0, 1, 5, 20, 32]),
                pad=rng.choice([0, 0, 1, 64]), masked=rng.random() < 0.4)


def _dtype(c):
    return torch.float32 if c["dtype"] == "f32" else torch.bfloat16


def _codes(y, dims):
    """e4m3 codes of y and what a step of each group is worth; `dims`: the axes of a group in y."""
    a = y.abs().amax(dims, keepdim=True).clamp(min=TINY)
    return (y * (448.0 / a)).to(torch.float8_e4m3fn), a / 448.0


def _row_codes(y):
    rows, cols = y.shape
    groups = -(-cols // GROUP)
    wide = torch.zeros(rows, groups * GROUP, device="cuda")
    wide[:, :cols] = y
    q, scale = _codes(wide.view(rows, groups, GROUP), (2,))
    return q.view(rows, -1)[:, :cols].contiguous(), scale.view(rows, groups)


def _block_codes(w):
    rows, cols = w.shape
    down, along = -(-rows // GROUP), -(-cols // GROUP)
    wide = torch.zeros(down * GROUP, along * GROUP, device="cuda")
    wide[:rows, :cols] = w
    q, scale = _codes(wide.view(down, GROUP, along, GROUP), (1, 3))
    return q.view(down * GROUP, -1)[:rows, :cols].contiguous(), scale.view(down, along)


def prepare(case, seed):
    c = dict(case)
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    rand = lambda *shape: torch.randn(*shape, device="cuda", generator=g)  # noqa: E731
    s = {"case": c}
    if c["kind"] == "rows":
        rows, cols = c["rows"], c["cols"]
        # a residual stream: values that grow with the layers, a few columns far above the others
        both = rand(rows, cols + c["pad"]) * (1 + 20 * (torch.rand(cols + c["pad"], device="cuda", generator=g) < 0.01))
        s["x"] = both.to(_dtype(c))[:, c["pad"]:]
        s["add"] = rand(rows, cols).to(_dtype(c)) if c["add"] else None
        s["weight"] = 1 + 0.1 * rand(cols) if c["norm"] else None
        s["total"] = torch.empty(rows, cols, dtype=_dtype(c), device="cuda") if c["add"] else None
        s["normed"] = torch.empty(rows, cols, dtype=_dtype(c), device="cuda") if c["normed"] else None
        s["q"] = torch.empty(rows, cols, dtype=torch.float8_e4m3fn, device="cuda")
        s["scale"] = torch.empty(rows, -(-cols // GROUP), device="cuda")
        return s
    if c["kind"] == "blocks":
        s["w"] = (rand(c["rows"], c["cols"]) * 0.02).to(_dtype(c))
        return s
    if c["kind"] == "product":
        s["xq"], s["xs"] = _row_codes(rand(c["m"], c["k"]))
        s["wq"], s["ws"] = _block_codes(rand(c["n"], c["k"]) * 0.02)
        s["add"] = rand(c["m"], c["n"]).to(_dtype(c)) if c["add"] else None
        s["out"] = torch.empty(c["m"], c["n"], dtype=_dtype(c), device="cuda")
        return s
    rows, vocab = c["rows"], c["vocab"]
    # from flat rows to ones that are nearly sure
    x = torch.randn(rows, vocab + c["pad"], device="cuda", generator=g, dtype=_dtype(c))
    x *= 1 + 2.5 * torch.rand(rows, 1, device="cuda", generator=g).to(x.dtype)
    at = torch.randint(vocab, (rows,), device="cuda", generator=g)
    x.scatter_add_(1, at[:, None], 12 * torch.rand(rows, 1, device="cuda", generator=g).to(x.dtype))
    s["logits"] = x[:, :vocab]
    token = torch.where(torch.rand(rows, device="cuda", generator=g) < 0.5, at, torch.randint(vocab, (rows,), device="cuda", generator=g))
    if c["masked"]:
        # what a grammar leaves: a twentieth of the vocabulary; the rest at -inf, or at the type's lowest value
        hide = torch.rand(rows, vocab, device="cuda", generator=g) < 0.95
        low = torch.where(torch.arange(rows, device="cuda") % 3 == 1, torch.finfo(x.dtype).min, -math.inf).to(x.dtype)
        s["logits"].copy_(torch.where(hide, low[:, None], s["logits"]))
        if rows > 4:
            s["logits"][3] = -math.inf
        token[5::7] = -1
    s["tokens"] = token.to(torch.int32)
    return s


# ---- the plain form


def _plain_rows(s):
    h, out = s["x"].float(), {}
    if s["add"] is not None:
        out["total"] = (h + s["add"].float()).to(s["x"].dtype)
        h = out["total"].float()
    if s["weight"] is not None:
        # the sum over a row in 64 bits: its rounding decides codes next to a border
        r = torch.rsqrt(h.double().square().mean(1, keepdim=True) + 1e-6).float()
        h = h * r * s["weight"]
    if s["normed"] is not None:
        out["normed"] = h.to(s["x"].dtype)
    out["q"], out["scale"] = _row_codes(h)
    return out


def _plain_blocks(s):
    q, scale = _block_codes(s["w"].float())
    return {"q": q, "scale": scale}


def _plain_product(s):
    k = s["case"]["k"]
    x = s["xq"].float() * s["xs"].repeat_interleave(GROUP, 1)[:, :k]
    w = s["wq"].float() * s["ws"].repeat_interleave(GROUP, 0)[:s["case"]["n"]].repeat_interleave(GROUP, 1)[:, :k]
    y = x @ w.T
    if s["add"] is not None:
        y = y + s["add"].float()
    return y.to(_dtype(s["case"]))


def _plain_tokens(s):
    x, token, top = s["logits"].float() + 0.0, s["tokens"].long()[:, None], s["case"]["top"]
    rows, vocab = x.shape
    index = torch.arange(vocab, device="cuda")
    best = x.amax(1, keepdim=True)
    none = best == -math.inf
    best = torch.where(none, 0.0, best)
    d = x - best
    e = torch.exp(d)
    total = e.sum(1, keepdim=True)
    norm = torch.log(total)
    entropy = torch.where(none, 0.0, norm - torch.where(e > 0, e * d, 0.0).sum(1, keepdim=True) / total)
    given = x.gather(1, token.clamp(min=0))
    logprob = torch.where(none, -math.inf, given - best - norm)
    rank = ((x > given) | ((x == given) & (index < token))).sum(1, keepdim=True)
    out = {"logprob": torch.where(token < 0, 0.0, logprob)[:, 0], "rank": torch.where(token < 0, -1, rank)[:, 0].to(torch.int32),
           "entropy": entropy[:, 0]}
    if top:
        # value and index as one whole number, the largest first: equal values by the lower index
        bits = x.view(torch.int32)
        key = (bits ^ ((bits >> 31) & 0x7fffffff)).long() * (1 << 32) + (0xffffffff - index)
        want = min(top, vocab)
        at = 0xffffffff - (key.topk(want, 1).values & 0xffffffff)
        value = x.gather(1, at)
        empty = value == -math.inf
        ids = torch.full((rows, top), -1, dtype=torch.int32, device="cuda")
        ids[:, :want] = torch.where(empty, -1, at).to(torch.int32)
        logs = torch.full((rows, top), -math.inf, device="cuda")
        logs[:, :want] = torch.where(empty, -math.inf, value - best - norm)
        out["top_ids"], out["top_logprobs"] = ids, logs
    return out


# ---- the calls of a user


def _library():
    """The library and the layers over it, once a process."""
    if not _kept:
        at = os.path.join(os.getcwd(), "faie2-flashnext_b200", "flashnext")
        if at not in sys.path:
            sys.path.insert(0, at)
        from fn import FN
        import fp8
        import logprobs
        _kept.update(fn=FN(), fp8=fp8, logprobs=logprobs)
    return _kept["fn"], _kept["fp8"], _kept["logprobs"]


def run(state):
    s, kind = state, state["case"]["kind"]
    if not own:
        return {"rows": _plain_rows, "blocks": _plain_blocks, "product": _plain_product, "tokens": _plain_tokens}[kind](s)
    fn, fp8, logprobs = _library()
    if kind == "rows":
        got = fp8.quantise_rows(fn, s["x"], add=s["add"], total=s["total"], weight=s["weight"], eps=1e-6, normed=s["normed"],
                                out=fp8.Fp8Rows(s["q"], s["scale"]))
        return {k: v for k, v in (("total", s["total"]), ("normed", s["normed"]), ("q", got.q), ("scale", got.scale)) if v is not None}
    if kind == "blocks":
        w = fp8.Fp8Weight.quantise(fn, s["w"])
        return {"q": w.q, "scale": w.scale}
    if kind == "product":
        if "weight" not in s:
            s["weight"] = fp8.Fp8Weight(fn, s["wq"], s["ws"])
        return s["weight"].product(fp8.Fp8Rows(s["xq"], s["xs"]), add=s["add"], out=s["out"])
    got = logprobs.token_logprobs(fn, s["logits"], s["tokens"], top=s["case"]["top"])
    out = {"logprob": got.logprob, "rank": got.rank, "entropy": got.entropy}
    return out | ({"top_ids": got.top_ids, "top_logprobs": got.top_logprobs} if s["case"]["top"] else {})


# ---- what a pass cannot do without


def work(case):
    c = case
    size = 4 if c["dtype"] == "f32" else 2
    if c["kind"] == "rows":
        n, groups = c["rows"] * c["cols"], c["rows"] * -(-c["cols"] // GROUP)
        streams = 1 + 2 * c["add"] + c["normed"]
        return {"bytes": n * (streams * size + 1) + 4 * groups + 4 * c["cols"] * c["norm"], "flops": n * (2 + c["add"] + 4 * c["norm"])}
    if c["kind"] == "blocks":
        n = c["rows"] * c["cols"]
        return {"bytes": n * (size + 1) + 4 * -(-c["rows"] // GROUP) * -(-c["cols"] // GROUP), "flops": 2 * n}
    if c["kind"] == "product":
        m, n, k = c["m"], c["n"], c["k"]
        groups = -(-k // GROUP)
        return {"bytes": (m + n) * k + 4 * groups * (m + -(-n // GROUP)) + m * n * size * (1 + c["add"]), "flops": 2 * m * n * k}
    n = c["rows"] * c["vocab"]
    return {"bytes": n * size + c["rows"] * (4 + 12 + 8 * c["top"]), "flops": 7 * n}


# ---- the definition in 64 bits


def _e4m3(v):
    """v rounded to the nearest e4m3 number, ties to even."""
    step = torch.exp2(torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6))) - 3)
    return (torch.round(v / step) * step).clamp(-448, 448)


def _grouped(y, down):
    """Codes and scales of groups of `down` rows by 128 columns, block by block of the columns."""
    q, scales = torch.empty_like(y), []
    rows = y.shape[0]
    group = torch.arange(rows, device="cuda") // down
    for at in range(0, y.shape[1], GROUP):
        part = y[:, at:at + GROUP]
        a = torch.zeros(-(-rows // down), dtype=y.dtype, device="cuda").scatter_reduce(0, group, part.abs().amax(1), "amax")
        a = a.clamp(min=TINY)
        q[:, at:at + GROUP] = _e4m3(part * 448 / a[group][:, None])
        scales.append(a / 448)
    return q, torch.stack(scales, 1)


def exact(case, seed):
    c = dict(case)
    s = prepare(case, seed)
    if c["kind"] == "rows":
        out, y = {}, s["x"].double()
        if c["add"]:
            y = (y + s["add"].double())
            out["total"] = y
            y = y.to(s["x"].dtype).double()
        if c["norm"]:
            y = y / torch.sqrt((y * y).sum(1, keepdim=True) / c["cols"] + 1e-6) * s["weight"].double()
        if c["normed"]:
            out["normed"] = y
        out["q"], out["scale"] = _grouped(y, 1)
        return out
    if c["kind"] == "blocks":
        q, scale = _grouped(s["w"].double(), GROUP)
        return {"q": q, "scale": scale}
    if c["kind"] == "product":
        y = torch.zeros(c["m"], c["n"], dtype=torch.float64, device="cuda")
        row = torch.arange(c["n"], device="cuda") // GROUP
        for j, at in enumerate(range(0, c["k"], GROUP)):
            part = s["xq"][:, at:at + GROUP].double() @ s["wq"][:, at:at + GROUP].double().T
            y += part * s["xs"][:, j:j + 1].double() * s["ws"][row, j].double()
        return y + s["add"].double() if c["add"] else y
    out = {"logprob": [], "entropy": [], "top_logprobs": []}
    for at in range(0, c["rows"], 256):
        x, token = s["logits"][at:at + 256].double(), s["tokens"][at:at + 256].long()
        dead = torch.isinf(x).all(1)
        x = torch.where(dead[:, None], 0.0, x)
        logs = x - torch.logsumexp(x, 1, keepdim=True)
        p = torch.exp(logs)
        given = logs.gather(1, token.clamp(min=0)[:, None])[:, 0]
        out["logprob"].append(torch.where(token < 0, 0.0, torch.where(dead, -math.inf, given)))
        out["entropy"].append(torch.where(dead, 0.0, -(p * torch.where(p > 0, logs, 0.0)).sum(1)))
        best = torch.full((x.shape[0], c["top"]), -math.inf, dtype=torch.float64, device="cuda")
        want = min(c["top"], c["vocab"])
        best[:, :want] = torch.sort(logs, 1, descending=True).values[:, :want]
        best[dead] = -math.inf
        out["top_logprobs"].append(best)
    got = {k: torch.cat(v) for k, v in out.items()} | {"rank": None, "top_ids": None}
    return got if c["top"] else {k: v for k, v in got.items() if not k.startswith("top")}
