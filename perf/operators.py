"""Cases of the paged 4-bit KV cache: planning a step on the GPU, storing and reading rows, attention over the pages.

The operators serve a batch of requests of different lengths whose keys and values live in pages of 4-bit codes:

  plan   from every request's cached length and new tokens: the page table with newly taken pages, the free-page stack,
         and for each new token its slot, position and request (a request with new < 0 is finished: its pages go back)
  store  rows of keys and values, quantised into their slots; load: the values that slots stand for
  attn   softmax(q k^T scale) v of every new token over its request's pages (causal, grouped heads, optional sigmoid
         gate), for one new token per request as for prompts

The cache: `pages` is uint8 [pages][kv heads][record]; a record holds page_size tokens of one head as K codes
[hd / 64][page_size][32 bytes], V codes likewise, K scales fp16 [hd / 64][page_size], V scales likewise. 64 dims share a
scale d; dim i of the 64 is nibble i (low nibble first) c and stands for d (c - 8). Slot = page * page_size + place.

`run` with `own` false is the plain form in elementary torch operations; with `own` true, the calls of a user.
"""

import math
import os
import sys

import torch

own = False

GROUP = 64  # dims that share a scale
PHI = 0.6180339887498949  # fractional parts of its multiples spread lengths evenly over their range
_kept = {}  # what a program keeps for its life: the library and the attention's workspace


def record_bytes(hd, bs):
    return 2 * bs * (hd // 2 + hd // GROUP * 2)


def listed():
    return [
        # one decode step of a full batch: every request one more token, a few of them a new page
        dict(name="plan_decode_32", kind="plan", n=32, bs=64, lo=1, hi=8191, prompts=0, prompt=0, done=0, max_tokens=32),
        # a step of a busy server: decoding requests, admitted prompts, finished requests whose pages go back
        dict(name="plan_mixed_256", kind="plan", n=256, bs=16, lo=1, hi=4000, prompts=24, prompt=700, done=20,
             max_tokens=16384),
        # a decode step's keys and values of 32 requests, the columns of a fused projection
        dict(name="store_step_f32", kind="store", tokens=32, nkv=2, hd=256, bs=64, dtype="f32", pad=8192),
        # a prompt slice of odd length, fp32 columns of a fused projection
        dict(name="store_prompt_f32", kind="store", tokens=1027, nkv=2, hd=256, bs=32, dtype="f32", pad=8192),
        # prompts of many requests in bf16, small pages
        dict(name="store_prompts_bf16", kind="store", tokens=8192, nkv=8, hd=128, bs=16, dtype="bf16", pad=0),
        # the first tokens of one conversation: latency
        dict(name="attn_one_short", kind="attn", n=1, nh=16, nkv=2, hd=256, bs=64, dtype="f32", qlo=1, qhi=1, lo=77, hi=77,
             gate=True, holes=False),
        # the gated attention layer at batch 32, requests of all ages
        dict(name="attn_decode_32_f32", kind="attn", n=32, nh=16, nkv=2, hd=256, bs=64, dtype="f32", qlo=1, qhi=1, lo=65,
             hi=4096, gate=True, holes=False),
        # one request with a long document behind it
        dict(name="attn_decode_long", kind="attn", n=1, nh=16, nkv=2, hd=256, bs=64, dtype="bf16", qlo=1, qhi=1,
             lo=131071, hi=131071, gate=False, holes=False),
        # a large decode batch, eight key heads, small pages
        dict(name="attn_decode_64_bf16", kind="attn", n=64, nh=32, nkv=8, hd=128, bs=16, dtype="bf16", qlo=1, qhi=1, lo=100,
             hi=8192, gate=False, holes=False),
        # checking five drafted tokens per request, seven query heads to a key head, idle and refused requests among them
        dict(name="attn_verify_f32", kind="attn", n=16, nh=28, nkv=4, hd=128, bs=32, dtype="f32", qlo=5, qhi=5, lo=9,
             hi=2000, gate=False, holes=True),
        # a slice of a long prompt through the gated attention layer
        dict(name="attn_prompt_f32", kind="attn", n=1, nh=16, nkv=2, hd=256, bs=64, dtype="f32", qlo=2048, qhi=2048,
             lo=4096, hi=4096, gate=True, holes=False),
        # prompts of several requests in one call, some behind a cached prefix
        dict(name="attn_prompts_bf16", kind="attn", n=8, nh=32, nkv=8, hd=128, bs=16, dtype="bf16", qlo=70, qhi=1500,
             lo=70, hi=4500, gate=False, holes=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["plan", "store", "attn", "attn", "attn"])
    bs = rng.choice([16, 32, 64])
    if kind == "plan":
        n, prompt = _log(rng, 1, 1000), _log(rng, 1, 2000)
        prompts = rng.randrange(0, n // 4 + 1)
        return dict(kind=kind, n=n, bs=bs, lo=1, hi=_log(rng, 50, 16000), prompts=prompts, prompt=prompt,
                    done=rng.randrange(0, n // 4 + 1), max_tokens=min(n + prompts * prompt, 16384))
    hd, nkv, dtype = rng.choice([64, 128, 256]), rng.choice([1, 2, 4, 8]), rng.choice(["f32", "bf16"])
    if kind == "store":
        tokens = min(_log(rng, 1, 8192), (1 << 23) // (nkv * hd))
        return dict(kind=kind, tokens=tokens, nkv=nkv, hd=hd, bs=bs, dtype=dtype, pad=rng.choice([0, 64, 1000]))
    group = rng.choice([1, 2, 3, 4, 5, 7, 8, 8, 16])
    form = rng.choice(["decode", "decode", "verify", "prompt"])
    if form == "prompt":
        n, qhi = _log(rng, 1, 8), _log(rng, 17, 1500)
        hi = max(1, min(qhi + _log(rng, 1, 3000), 100_000_000 // (n * qhi * nkv * group)))
        qlo = rng.randrange(1, qhi + 1)
    else:
        n = _log(rng, 1, 64)
        qlo = qhi = 1 if form == "decode" else rng.randrange(2, 9)
        hi = max(1, min(_log(rng, 1, 100_000), 270_000_000 // (n * nkv * hd), 100_000_000 // (n * qhi * nkv * group)))
    return dict(kind=kind, n=n, nh=nkv * group, nkv=nkv, hd=hd, bs=bs, dtype=dtype, qlo=qlo, qhi=qhi,
                lo=rng.randrange(1, hi + 1), hi=hi, gate=rng.random() < 0.3, holes=n > 3 and rng.random() < 0.4)


def spread(n, lo, hi, turn=0.0):
    """n lengths over lo..hi, the last one hi."""
    got = [lo + int((hi - lo + 1) * math.modf((r + 1) * PHI + turn)[0]) for r in range(n)]
    return got[:-1] + [hi]


def plan_lengths(c):
    """Cached lengths and new tokens of every request: every tenth or so is finished (-1) or a prompt with no past."""
    ctx, add = spread(c["n"], c["lo"], c["hi"]), [1] * c["n"]
    for j in range(c["prompts"]):
        r = int(c["n"] * (j + 0.5) / c["prompts"])
        ctx[r], add[r] = 0, spread(c["prompts"], 1, c["prompt"], 0.3)[j]
    for j in range(c["done"]):
        r = int(c["n"] * (j + 0.25) / c["done"])
        add[r] = -1
    return ctx, add


def attn_lengths(c):
    """New tokens and total length of every request. With holes: a refused request (length 0), one with fewer cached
    tokens than rows (its first rows see nothing), an idle one (no rows)."""
    new = spread(c["n"], c["qlo"], c["qhi"], 0.4)
    total = [max(t, q) for t, q in zip(spread(c["n"], c["lo"], c["hi"]), new)]
    if c["holes"]:
        total[0] = 0
        if c["n"] > 1:
            total[1] = new[1] // 2
        if c["n"] > 2:
            new[2] = 0
    return new, total


def _dtype(c):
    return torch.float32 if c["dtype"] == "f32" else torch.bfloat16


def _codes(x):
    """Blocks of 64 dims (last axis) as codes and scales: d = (the value of largest magnitude; of two opposite ones the
    positive) / -8."""
    big, small = x.amax(-1, keepdim=True), x.amin(-1, keepdim=True)
    d = torch.where(big >= -small, big, small) / -8.0
    inv = torch.where(d == 0, torch.zeros_like(d), 1.0 / d)
    c = torch.clamp((x * inv + 8.5).to(torch.int32), 0, 15).to(torch.uint8)
    return c[..., 0::2] | (c[..., 1::2] << 4), d.squeeze(-1).to(torch.float16)


def _random_pages(count, c, g):
    """Pages of quantised normal values."""
    nkv, hd, bs, out = c["nkv"], c["hd"], c["bs"], []
    pages = torch.empty(count, nkv, record_bytes(hd, bs), dtype=torch.uint8, device="cuda")
    kb, sb = bs * hd // 2, bs * (hd // GROUP) * 2
    for at in range(0, count, 4096):
        m = min(4096, count - at)
        for part in range(2):
            x = torch.randn(m, nkv, hd // GROUP, bs, GROUP, device="cuda", generator=g)
            q, d = _codes(x)
            pages[at:at + m, :, part * kb:(part + 1) * kb] = q.reshape(m, nkv, kb)
            pages[at:at + m, :, 2 * kb + part * sb:2 * kb + (part + 1) * sb] = d.reshape(m, nkv, -1).view(torch.uint8)
    return pages


def prepare(case, seed):
    c = dict(case)
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    s = {"case": c}
    if c["kind"] == "plan":
        ctx, add = plan_lengths(c)
        have = [-(-v // c["bs"]) for v in ctx]
        width = max(-(-(v + max(a, 0)) // c["bs"]) for v, a in zip(ctx, add)) + 1
        # the pool: what the requests hold and need, and a few more
        pages = sum(-(-(v + max(a, 0)) // c["bs"]) for v, a in zip(ctx, add)) + 5
        ids = torch.randperm(pages, device="cuda", generator=g).to(torch.int32)
        table = torch.full((c["n"], width), -1, dtype=torch.int32, device="cuda")
        held = torch.arange(width, device="cuda")[None, :] < i32(have)[:, None]
        table[held] = ids[:sum(have)]
        free = torch.full((pages,), -1, dtype=torch.int32, device="cuda")
        free[:pages - sum(have)] = ids[sum(have):]
        s.update(ctx=i32(ctx), add=i32(add), table=table, free=free, free_count=i32([pages - sum(have)]), pages=pages)
        return s
    if c["kind"] == "store":
        t, row = c["tokens"], c["nkv"] * c["hd"]
        count = -(-t // c["bs"]) + 3
        both = torch.randn(t, c["pad"] + 2 * row, device="cuda", generator=g).to(_dtype(c))
        s["k"] = both[:, c["pad"]:c["pad"] + row].unflatten(1, (c["nkv"], c["hd"]))
        s["v"] = both[:, c["pad"] + row:].unflatten(1, (c["nkv"], c["hd"]))
        # tokens in whole pages of a shuffled pool, one in 64 of them padding
        order = torch.randperm(count, device="cuda", generator=g)
        slots = (order[:, None] * c["bs"] + torch.arange(c["bs"], device="cuda")[None, :]).reshape(-1)[:t].contiguous()
        slots[63::64] = -1
        s.update(slots=slots, spare=order[-1], pages=torch.zeros(count, c["nkv"], record_bytes(c["hd"], c["bs"]), dtype=torch.uint8,
                                                               device="cuda"))
        return s
    new, total = attn_lengths(c)
    used = [-(-v // c["bs"]) for v in total]
    count, width = sum(used) + 2, max(max(used), 1)
    s["pages"] = _random_pages(count, c, g)
    table = torch.full((c["n"], width), -1, dtype=torch.int32, device="cuda")
    held = torch.arange(width, device="cuda")[None, :] < i32(used)[:, None]
    table[held] = torch.randperm(count, device="cuda", generator=g)[:sum(used)].to(torch.int32)
    # the places of a last page that no token has written yet hold what was there before: here, NaN scales
    sb = c["bs"] * (c["hd"] // GROUP)
    scales = s["pages"].view(torch.float16)[:, :, -2 * sb:].unflatten(2, (2, c["hd"] // GROUP, c["bs"]))
    for r in range(c["n"]):
        if total[r] % c["bs"]:
            scales[table[r, used[r] - 1].long(), :, :, :, total[r] % c["bs"]:] = float("nan")
    rows = sum(new)
    qg = torch.randn(max(rows, 1), c["nh"], 2 * c["hd"] if c["gate"] else c["hd"], device="cuda", generator=g)
    qg = qg[:rows].to(_dtype(c))
    cu = [0]
    for q in new:
        cu.append(cu[-1] + q)
    s.update(q=qg[..., :c["hd"]], gate=qg[..., c["hd"]:] if c["gate"] else None, cu=i32(cu), kv_len=i32(total),
             table=table, longest=max(total), most=max(new))
    return s


# ---- the plain form


def _plain_plan(s):
    c, bs = s["case"], s["case"]["bs"]
    ctx, add, table, free = s["ctx"].long(), s["add"].long(), s["table"].long(), s["free"].long()
    n, width = table.shape
    cap, top = c["max_tokens"], s["free_count"].long()
    new = add.clamp(min=0)
    end = torch.cumsum(new, 0)
    have, want = (ctx + bs - 1) // bs, (ctx + new + bs - 1) // bs
    fits = (new == 0) | ((want <= width) & (end <= cap))
    need = torch.where((new > 0) & fits, want - have, 0)
    back = torch.where(add < 0, have.clamp(max=width), 0)
    back_end, need_end = torch.cumsum(back, 0), torch.cumsum(need, 0)
    col = torch.arange(width, device="cuda")[None, :]
    # the pages of finished requests go on top of the stack, then the new pages come from its top
    given = col < back[:, None]
    to = torch.where(given, top + (back_end - back)[:, None] + col, s["pages"])
    free = torch.cat([free, free.new_zeros(1)])
    free[to] = torch.where(given, table, 0)
    free = free[:-1]
    top = top + back_end[-1:]
    served = fits & ((need == 0) | (need_end <= top))
    taken = served[:, None] & (col >= have[:, None]) & (col < (have + need)[:, None])
    take = top - 1 - ((need_end - need)[:, None] + col - have[:, None])
    table = torch.where(taken, free[take.clamp(0, s["pages"] - 1)], table)
    kv_len = torch.where((add < 0) | ~served, 0, ctx + new)
    left = top - torch.where(served & (need > 0), need_end, 0).amax().clamp(min=0)
    cu = torch.cat([end.new_zeros(1), end]).clamp(max=cap)
    row = torch.arange(cap, device="cuda")
    req = torch.searchsorted(cu[1:].contiguous(), row, right=True)
    live = req < n
    req = req.clamp(max=n - 1)
    pos = ctx[req] + row - cu[req]
    put = live & served[req]
    slot = table[req, (pos // bs).clamp(max=width - 1)] * bs + pos % bs
    i32 = lambda t: t.to(torch.int32)  # noqa: E731
    return {"table": i32(table), "free": i32(free), "free_count": i32(left), "cu": i32(cu), "kv_len": i32(kv_len),
            "slots": torch.where(put, slot, -1), "positions": i32(torch.where(put, pos, -1)),
            "requests": i32(torch.where(live, req, -1)), "status": i32((~served).sum()[None])}


def _split(pages, hd, bs):
    """K codes, V codes [.., hd / 64, bs, 32] and their scales [.., hd / 64, bs] of page records."""
    kb, sb, ng = bs * hd // 2, bs * (hd // GROUP) * 2, hd // GROUP
    at = lambda lo, n: pages[..., lo:lo + n].contiguous()  # noqa: E731
    return (at(0, kb).unflatten(-1, (ng, bs, 32)), at(kb, kb).unflatten(-1, (ng, bs, 32)),
            at(2 * kb, sb).view(torch.float16).unflatten(-1, (ng, bs)),
            at(2 * kb + sb, sb).view(torch.float16).unflatten(-1, (ng, bs)))


def _values(codes, scales):
    """What codes [.., 32 bytes] stand for, fp32 [.., 64]."""
    c = torch.stack([codes & 15, codes >> 4], -1).flatten(-2)
    return (c.float() - 8.0) * scales.float()[..., None]


def _plain_store(s):
    c, flat, hd, bs = s["case"], s["pages"].view(-1), s["case"]["hd"], s["case"]["bs"]
    kb, sb, ng = bs * hd // 2, bs * (hd // GROUP) * 2, hd // GROUP
    live = s["slots"] >= 0
    # padding rows go to a page that nobody reads
    slot = torch.where(live, s["slots"], s["spare"] * bs)
    rec = (slot // bs)[:, None] * c["nkv"] + torch.arange(c["nkv"], device="cuda")[None, :]
    line = torch.arange(ng, device="cuda")[None, None, :] * bs + (slot % bs)[:, None, None]  # [tokens][1][groups]
    rec = rec[:, :, None] * record_bytes(hd, bs)
    out = {}
    for name, code, scale in (("k", 0, 2 * kb), ("v", kb, 2 * kb + sb)):
        q, d = _codes(s[name].float().unflatten(2, (ng, GROUP)))
        at = (rec + code + line * 32)[..., None] + torch.arange(32, device="cuda")
        sat = (rec + scale + line * 2)[..., None] + torch.arange(2, device="cuda")
        flat[at] = q
        flat[sat] = d[..., None].view(torch.uint8)
        x = _values(flat[at], flat[sat].view(torch.float16).squeeze(-1)).flatten(2)
        out[name] = torch.where(live[:, None, None], x, torch.zeros((), device="cuda")).to(_dtype(c))
    return out


def _plain_attn(s):
    c, hd, bs, n, nkv = s["case"], s["case"]["hd"], s["case"]["bs"], s["case"]["n"], s["case"]["nkv"]
    group, rows = c["nh"] // nkv, s["q"].shape[0]
    wide, most = max(-(-s["longest"] // bs), 1), max(s["most"], 1)
    kc, vc, ks, vs = _split(s["pages"][s["table"][:, :wide].clamp(min=0).long()], hd, bs)
    # [n][page][head][group][place][64] -> [n][head][token][hd]
    lay = lambda x: x.permute(0, 2, 1, 4, 3, 5).reshape(n, nkv, wide * bs, hd)  # noqa: E731
    there = (torch.arange(wide * bs, device="cuda")[None, :] < s["kv_len"][:, None])[:, None, :, None]
    zero = torch.zeros((), device="cuda")
    k = torch.where(there, lay(_values(kc, ks)), zero)
    v = torch.where(there, lay(_values(vc, vs)), zero)
    cu, new = s["cu"].long(), (s["cu"][1:] - s["cu"][:-1]).long()
    at = (cu[:-1, None] + torch.arange(most, device="cuda")[None, :]).clamp(max=max(rows - 1, 0))
    q = s["q"][at].float().unflatten(2, (nkv, group)).permute(0, 2, 1, 3, 4).reshape(n, nkv, most * group, hd)
    w = (q @ k.transpose(2, 3)) * (1.0 / math.sqrt(hd))
    # row i of a request is at position length - rows + i and sees the keys up to itself
    last = s["kv_len"].long()[:, None] - new[:, None] + torch.arange(most, device="cuda")[None, :]
    see = torch.arange(wide * bs, device="cuda")[None, None, :] <= last[:, :, None]
    see = (see & there[:, 0, None, :, 0]).repeat_interleave(group, 1)[:, None]
    w = torch.where(see, w, torch.full((), float("-inf"), device="cuda"))
    top = w.amax(-1, keepdim=True)
    w = torch.exp(w - torch.where(torch.isinf(top), zero, top))
    total = w.sum(-1, keepdim=True)
    o = (w @ v) / torch.where(total > 0, total, torch.ones((), device="cuda"))
    o = o.reshape(n, nkv, most, group, hd).permute(0, 2, 1, 3, 4).reshape(n, most, c["nh"], hd)
    row = torch.arange(rows, device="cuda")
    req = torch.searchsorted(cu[1:].contiguous(), row, right=True)
    o = o[req, row - cu[req]]
    if s["gate"] is not None:
        o = o / (1.0 + torch.exp(-s["gate"].float()))
    return o.to(_dtype(c))


# ---- the calls of a user


def _cache(s):
    """The planner, or the cache object over the state's pages: made at the first pass and kept."""
    if "cache" not in s:
        if "fn" not in _kept:
            at = os.path.join(os.getcwd(), "faie2-flashnext_b200", "flashnext")
            if at not in sys.path:
                sys.path.insert(0, at)
            from fn import FN
            import kv4
            _kept["fn"], _kept["kv4"] = FN(), kv4
            _kept["ws"] = kv4.KV4Workspace(_kept["fn"])
        c, kv4 = s["case"], _kept["kv4"]
        s["cache"] = (kv4.KV4Planner(_kept["fn"], c["bs"]) if c["kind"] == "plan" else
                      kv4.KV4Cache(_kept["fn"], c["nkv"], c["hd"], c["bs"], pages=s["pages"], workspace=_kept["ws"]))
    return s["cache"]


def run(state):
    kind = state["case"]["kind"]
    if not own:
        return {"plan": _plain_plan, "store": _plain_store, "attn": _plain_attn}[kind](state)
    cache = _cache(state)
    if kind == "plan":
        step = cache.plan(state["ctx"], state["add"], state["table"], state["free"], state["free_count"],
                          state["case"]["max_tokens"])
        return {"table": state["table"], "free": state["free"], "free_count": step.free_count, "cu": step.cu,
                "kv_len": step.kv_len, "slots": step.slots, "positions": step.positions, "requests": step.requests,
                "status": step.status}
    if kind == "store":
        cache.store(state["k"], state["v"], state["slots"])
        k, v = cache.load(state["slots"], state["k"].dtype)
        return {"k": k, "v": v}
    return cache.attn(state["q"], state["cu"], state["kv_len"], state["table"], max_new=state["most"], gate=state["gate"])


# ---- what a pass cannot do without


def work(case):
    c = case
    if c["kind"] == "plan":
        ctx, add = plan_lengths(c)
        pages = sum(-(-(v + a) // c["bs"]) - -(-v // c["bs"]) for v, a in zip(ctx, add) if a > 0)
        back = sum(-(-v // c["bs"]) for v, a in zip(ctx, add) if a < 0)
        # lengths in; offsets and lengths out; taken and returned ids read and written; slot, position, request of a row
        return {"bytes": 8 * c["n"] + 8 * c["n"] + 8 * (pages + back) + 16 * c["max_tokens"], "flops": 0}
    size = 4 if c["dtype"] == "f32" else 2
    token = c["nkv"] * c["hd"] * 2 * (0.5 + 2 / GROUP)  # bytes of a token's keys and values in the cache
    if c["kind"] == "store":
        live = c["tokens"] - c["tokens"] // 64
        row = c["nkv"] * c["hd"] * 2 * size
        return {"bytes": live * (row + token) + live * token + c["tokens"] * (row + 16),
                "flops": live * c["nkv"] * c["hd"] * 2 * 4}
    new, total = attn_lengths(c)
    pairs = sum(sum(max(0, t - q + i + 1) for i in range(q)) for q, t in zip(new, total))
    rows = sum(new) * c["nh"] * c["hd"] * size
    return {"bytes": rows * (3 if c["gate"] else 2) + sum(t for q, t in zip(new, total) if q) * token,
            "flops": 4 * c["hd"] * c["nh"] * pairs}


# ---- the definition in 64 bits


def exact(case, seed):
    c = dict(case)
    if c["kind"] == "plan":
        return None
    s = prepare(case, seed)
    ng, hd = c["hd"] // GROUP, c["hd"]
    if c["kind"] == "store":
        out = {}
        for name in ("k", "v"):
            x = s[name].double().reshape(c["tokens"], c["nkv"], ng, GROUP)
            big, small = x.amax(-1, keepdim=True), x.amin(-1, keepdim=True)
            d = -torch.where(big >= -small, big, small) / 8
            code = torch.floor(x / torch.where(d == 0, 1, d) + 8.5).clamp(0, 15)
            y = (code - 8) * d.to(torch.float16).double()
            y[s["slots"] < 0] = 0
            out[name] = y.reshape(c["tokens"], c["nkv"], hd)
        return out
    new, total = attn_lengths(c)
    group, bs, at = c["nh"] // c["nkv"], c["bs"], 0
    kb, sb = bs * hd // 2, bs * ng * 2
    out = torch.zeros(sum(new), c["nh"], hd, dtype=torch.float64, device="cuda")
    for r in range(c["n"]):
        q, t = new[r], total[r]
        if q and t:
            rec = s["pages"][s["table"][r, :-(-t // bs)].long()]
            kv = []
            for part in range(2):
                byte = rec[:, :, part * kb:(part + 1) * kb].reshape(-1, c["nkv"], ng, bs, 32).int()
                val = torch.empty(*byte.shape[:-1], GROUP, dtype=torch.float64, device="cuda")
                val[..., 0::2], val[..., 1::2] = (byte % 16 - 8).double(), (byte // 16 - 8).double()
                d = rec[:, :, 2 * kb + part * sb:2 * kb + (part + 1) * sb].contiguous().view(torch.float16)
                val *= d.reshape(-1, c["nkv"], ng, bs, 1).double()
                kv.append(val.permute(1, 0, 3, 2, 4).reshape(c["nkv"], -1, hd)[:, :t])
            first = max(0, q - t)  # the rows before it see nothing
            pos = torch.arange(t - q + first, t, device="cuda")
            hide = torch.arange(t, device="cuda")[None, :] > pos[:, None]
            for h in range(c["nh"]):
                w = s["q"][at + first:at + q, h].double() @ kv[0][h // group].T / math.sqrt(hd)
                w = torch.softmax(w.masked_fill(hide, float("-inf")), -1)
                out[at + first:at + q, h] = w @ kv[1][h // group]
        at += q
    if s["gate"] is not None:
        out *= torch.sigmoid(s["gate"].double())
    return out
