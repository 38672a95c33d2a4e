"""GPU parity of the paged 4-bit KV cache (flashnext/kv4.py over fn_kv4_*) against the float64 oracle (oracle/kv4.py).

Tolerances, from the formats: planning and page bytes are equal. Loaded values are code times scale, exact in fp32, and
rounded once for bf16: equal. Attention, relative to the largest |v| that a row sees (the output is a convex
combination of the v): fp32 rows keep scores to a few 2^-22 of their size (|s| < 16 here, so 2^-17 at most in the exponent)
and products in fp32: 2e-5. bf16 rows: the output's half ulp, at most 2^-8 of itself, and the probabilities' and values'
rounding to 11 bits (2^-12 each, less on average over the keys): 2^-8 |out| + 2^-10.
"""

import numpy as np
import pytest
import torch

from oracle import kv4 as O

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "bf16": torch.bfloat16}


@pytest.fixture(scope="module")
def kv4(fn):
    import kv4 as m
    return m


@pytest.fixture(scope="module")
def ws(fn, kv4):
    return kv4.KV4Workspace(fn)


def dev(a, dtype=None):
    t = torch.from_numpy(np.ascontiguousarray(a)).cuda()
    return t if dtype is None else t.to(dtype)


# ---- planning


def make_plan(rng, n, bs, hi, prompt, spare, width_cut=0):
    ctx = rng.integers(0, hi + 1, n).astype(np.int32)
    add = np.ones(n, np.int32)
    kind = rng.random(n)
    add[kind < 0.2] = 0
    add[kind < 0.1] = -1
    fresh = kind > 0.85
    ctx[fresh], add[fresh] = 0, rng.integers(1, prompt + 1, int(fresh.sum()))
    have = -(-ctx.astype(np.int64) // bs)
    want = -(-(ctx.astype(np.int64) + np.maximum(add, 0)) // bs)
    width = max(int(want.max()) - width_cut, int(have.max()), 1)
    n_pages = int(have.sum()) + max(int((want - have).sum()) + spare, 1)
    ids = rng.permutation(n_pages).astype(np.int32)
    table = np.full((n, width), -1, np.int32)
    table[np.arange(width)[None] < have[:, None]] = ids[:have.sum()]
    free = np.full(n_pages, -7, np.int32)
    free[:n_pages - have.sum()] = ids[have.sum():]
    return ctx, add, table, free, int(n_pages - have.sum()), n_pages


def run_plan(kv4, fn, bs, ctx, add, table, free, count, max_tokens):
    t, f = dev(table), dev(free)
    p = kv4.KV4Planner(fn, bs).plan(dev(ctx), dev(add), t, f, dev(np.array([count], np.int32)), max_tokens)
    fn.sync(torch.cuda.current_stream().cuda_stream)
    got = {k: getattr(p, k).cpu().numpy() for k in ("cu", "kv_len", "slots", "positions", "requests")}
    return {**got, "table": t.cpu().numpy(), "free": f.cpu().numpy(), "free_count": int(p.free_count),
            "status": int(p.status)}


def same_plan(got, want):
    for k, v in want.items():
        assert np.array_equal(got[k], v), k


@pytest.mark.parametrize("n, bs, hi, prompt, spare, cut, room", [
    (1, 16, 0, 1, 0, 0, 1), (1, 64, 64, 1, 0, 0, 3), (7, 16, 40, 33, 2, 0, 200), (32, 64, 8191, 1, 0, 0, 32),
    (33, 32, 300, 100, -5, 0, 900), (100, 16, 100, 50, -40, 0, 2000), (64, 16, 200, 90, 3, 4, 4000),
    (64, 32, 200, 90, 3, 0, 150), (1023, 16, 60, 3, 0, 0, 1300), (1025, 64, 500, 40, 9, 0, 9000),
    (4096, 16, 90, 2, -100, 0, 5000), (250, 16, 3000, 700, 11, 0, 20000)])
def test_plan(fn, kv4, n, bs, hi, prompt, spare, cut, room):
    rng = np.random.default_rng(n + bs + room)
    ctx, add, table, free, count, n_pages = make_plan(rng, n, bs, hi, prompt, spare, cut)
    want = O.plan(ctx, add, table, bs, free, count, n_pages, room)
    same_plan(run_plan(kv4, fn, bs, ctx, add, table, free, count, room), want)


def test_plan_of_nothing_left_refuses_and_takes_nothing(fn, kv4):
    table, free = np.full((3, 3), -1, np.int32), np.array([4, 5], np.int32)
    ctx, add = np.array([0, 16, 3], np.int32), np.array([40, 1, 1], np.int32)  # 3 pages wanted, then 1, then none
    table[1, 0], table[2, 0] = 8, 9
    got = run_plan(kv4, fn, 16, ctx, add, table, free, 2, 64)
    assert got["status"] == 2 and got["free_count"] == 2 and list(got["kv_len"]) == [0, 0, 4]
    assert (got["slots"][:41] == -1).all() and got["slots"][41] == 9 * 16 + 3
    same_plan(got, O.plan(ctx, add, table, 16, free, 2, 2, 64))


def test_plan_clamps_negative_lengths_and_counts(fn, kv4):
    table, free = np.full((2, 1), -1, np.int32), np.array([0, 1], np.int32)
    got = run_plan(kv4, fn, 16, np.array([-5, 0], np.int32), np.array([1, 1], np.int32), table, free, -3, 4)
    assert got["status"] == 2 and got["free_count"] == 0 and not got["kv_len"].any()


def test_plan_in_place_count_and_steps_of_a_server(fn, kv4):
    """Requests admitted, decoded over page ends, finished and replaced: the count updated in place, every step as the oracle's."""
    rng = np.random.default_rng(5)
    n, bs, width, n_pages = 6, 16, 8, 30
    table, free = np.full((n, width), -1, np.int32), rng.permutation(n_pages).astype(np.int32)
    ctx, count = np.zeros(n, np.int32), n_pages
    pl, t, f, c = kv4.KV4Planner(fn, bs), dev(table), dev(free), dev(np.array([count], np.int32))
    for step in range(60):
        add = np.where(ctx == 0, rng.integers(0, 40, n), 1).astype(np.int32)
        add[ctx > rng.integers(40, 120)] = -1
        want = O.plan(ctx, add, table, bs, free, count, n_pages, 128)
        p = pl.plan(dev(ctx), dev(add), t, f, c, 128)
        c.copy_(p.free_count)
        fn.sync(torch.cuda.current_stream().cuda_stream)
        for k in ("cu", "kv_len", "slots", "positions", "requests"):
            assert np.array_equal(getattr(p, k).cpu().numpy(), want[k]), (step, k)
        table, free, count = want["table"], want["free"], want["free_count"]
        assert np.array_equal(t.cpu().numpy(), table) and int(c) == count
        live = np.where(add < 0, 0, np.where(want["kv_len"] > 0, want["kv_len"], ctx))
        held = [table[r, :-(-int(live[r]) // bs)] for r in range(n)]
        ids = np.concatenate([free[:count]] + held)
        assert len(ids) == n_pages and len(set(ids.tolist())) == n_pages  # no page lost, none twice
        ctx = live.astype(np.int32)


# ---- store and load


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("hd, nkv, bs, rows, pad", [(64, 1, 16, 1, 0), (128, 3, 32, 37, 0), (256, 2, 64, 65, 8), (256, 2, 16, 5, 3),
                                                    (64, 8, 64, 200, 1)])
def test_store_and_load(fn, kv4, ws, dtype, hd, nkv, bs, rows, pad):
    """Columns of a fused projection: token stride with padding (odd padding: rows aligned to their type only)."""
    rng = np.random.default_rng(rows + hd)
    g = torch.Generator("cuda").manual_seed(rows)
    x = torch.randn(rows, pad + 2 * nkv * hd, device="cuda", generator=g).to(DT[dtype])
    x[:, pad:pad + 64] *= 1e-3  # a block of small values, one of large ones
    x[:, -64:] *= 1e4
    k, v = x[:, pad:pad + nkv * hd].unflatten(1, (nkv, hd)), x[:, pad + nkv * hd:].unflatten(1, (nkv, hd))
    n_pages = -(-rows // bs) + 2
    slots = rng.permutation(n_pages * bs)[:rows].astype(np.int64)
    slots[1::5] = -1
    pages = rng.integers(0, 256, (n_pages, nkv, O.record_bytes(hd, bs)), dtype=np.uint8)
    want = pages.copy()
    O.store(want, hd, bs, k.float().cpu().numpy(), v.float().cpu().numpy(), slots)
    c = kv4.KV4Cache(fn, nkv, hd, bs, dev(pages), ws)
    c.store(k, v, dev(slots))
    assert np.array_equal(c.pages.cpu().numpy(), want)
    gk, gv = c.load(dev(slots), DT[dtype])
    wk, wv = O.load(want, hd, bs, slots)
    for got, ref in ((gk, wk), (gv, wv)):
        if dtype == "f32":
            assert np.array_equal(got.cpu().numpy(), ref.astype(np.float32))
        else:
            assert torch.equal(got.cpu(), torch.from_numpy(ref).to(torch.bfloat16))


def test_store_marks_what_has_no_scale(fn, kv4, ws):
    c = kv4.KV4Cache(fn, 1, 64, 16, 1, ws)
    k = torch.ones(5, 1, 64, device="cuda")
    k[0, 0, 3], k[1, 0, 4], k[2, 0, 5], k[3] = float("nan"), float("-inf"), 65504 * 8.5, 0
    v = torch.randn(5, 1, 64, device="cuda")
    slots = torch.arange(5, device="cuda")
    c.store(k, v, slots)
    lk, lv = c.load(slots)
    assert lk[:3].isnan().all() and (lk[3] == 0).all() and not lv.isnan().any()
    assert ((lk[4] - 1).abs() <= 2.0 ** -11).all()


def test_slots_past_the_pages_are_skipped_and_reported(fn, kv4, ws):
    c = kv4.KV4Cache(fn, 2, 64, 16, 2, ws)
    x = torch.randn(3, 2, 64, device="cuda")
    slots = torch.tensor([31, 32, 1 << 40], device="cuda")
    c.store(x, x, slots)
    with pytest.raises(RuntimeError, match="argument check"):
        fn.sync(torch.cuda.current_stream().cuda_stream)
    k, _ = c.load(slots)
    assert k[0].any() and not k[1:].any()
    with pytest.raises(RuntimeError, match="argument check"):
        fn.sync(torch.cuda.current_stream().cuda_stream)


# ---- attention


def build(kv4, fn, ws, rng, hd, nkv, bs, lens, stale=True, n_pages=None, base=0):
    """A cache with requests of the given lengths on shuffled pages; unwritten places hold NaN scales and random codes."""
    used = [-(-t // bs) for t in lens]
    total = n_pages or base + sum(used) + 1
    pages = rng.integers(0, 256, (sum(used) + 1, nkv, O.record_bytes(hd, bs)), dtype=np.uint8)
    if stale:
        sb = bs * (hd // 64) * 4
        pages[..., -sb:] = 0xff  # fp16 NaN
    table = np.full((len(lens), max(max(used), 1) + 1), -1, np.int32)
    ids, at = rng.permutation(sum(used)).astype(np.int32), 0
    slots = []
    for r, t in enumerate(lens):
        table[r, :used[r]] = ids[at:at + used[r]]
        at += used[r]
        slots += [int(table[r, i // bs]) * bs + i % bs for i in range(t)]
    k = rng.standard_normal((len(slots), nkv, hd)).astype(np.float32)
    v = rng.standard_normal((len(slots), nkv, hd)).astype(np.float32) + 0.3
    O_pages = pages
    slots = np.array(slots, np.int64)
    small = kv4.KV4Cache(fn, nkv, hd, bs, dev(pages), ws)
    if len(slots):
        small.store(dev(k), dev(v), dev(slots))
    O_pages = small.pages.cpu().numpy()
    if total == len(pages) and not base:
        return small, O_pages, table, table
    big = torch.empty(total, nkv, O.record_bytes(hd, bs), dtype=torch.uint8, device="cuda")
    big[base:base + len(pages)] = small.pages
    return kv4.KV4Cache(fn, nkv, hd, bs, big, ws), O_pages, table, np.where(table >= 0, table + base, table).astype(np.int32)


def check(got, want, dtype, vmax=4.0):
    got = got.float().cpu().numpy().astype(np.float64)
    assert np.isfinite(got).all()
    if dtype == "f32":
        tol = 2e-5 * vmax
        assert np.abs(got - want).max() <= tol, np.abs(got - want).max()
    else:
        assert (np.abs(got - want) <= np.abs(want) * 2.0 ** -8 + vmax * 2.0 ** -10).all(), np.abs(got - want).max()


def offsets(news):
    return np.concatenate([[0], np.cumsum(news)]).astype(np.int32)


def attn_case(fn, kv4, ws, seed, hd, nkv, group, bs, dtype, lens, news, gate=False, extra_rows=0, max_new=None, qscale=1.0):
    rng = np.random.default_rng(seed)
    c, pages, table, dtable = build(kv4, fn, ws, rng, hd, nkv, bs, lens)
    cu, nh = offsets(news), nkv * group
    rows = int(cu[-1]) + extra_rows
    q = dev(rng.standard_normal((rows, nh, 2 * hd)).astype(np.float32) * qscale, DT[dtype])
    g = q[..., hd:] if gate else None
    out = c.attn(q[..., :hd], dev(cu), dev(np.array(lens, np.int32)), dev(dtable), max(news) if max_new is None else max_new, gate=g)
    fn.sync(torch.cuda.current_stream().cuda_stream)
    want = O.attn(pages, hd, bs, q[..., :hd].float().cpu().numpy(), cu, lens, table,
                  gate=g.float().cpu().numpy() if gate else None)
    check(out, want, dtype)
    return c, q, cu, dtable, out


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("hd, nkv, group, bs", [(64, 1, 1, 16), (64, 2, 8, 64), (128, 1, 7, 32), (128, 4, 2, 16), (256, 2, 8, 64),
                                                (256, 1, 3, 16), (128, 1, 16, 64), (64, 1, 20, 32)])
def test_decode(fn, kv4, ws, dtype, hd, nkv, group, bs):
    """One new token per request: lengths from one, at page and tile ends and past them, an empty request among them."""
    lens = [1, bs - 1, bs, bs + 1, 0, 63, 64, 65, 127, 128, 129, 200]
    attn_case(fn, kv4, ws, hd + group, hd, nkv, group, bs, dtype, lens, [1] * len(lens), gate=hd == 256, extra_rows=2)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("hd, nkv, group, bs", [(64, 2, 4, 16), (128, 1, 7, 32), (256, 2, 8, 64), (128, 2, 1, 64)])
def test_few_new_tokens(fn, kv4, ws, dtype, hd, nkv, group, bs):
    """Drafted tokens, idle requests, a refused one (length 0), rows before the first key."""
    lens, news = [70, 5, 0, 33, 130, 2], [5, 5, 3, 0, 1, 4]
    attn_case(fn, kv4, ws, hd * 3 + group, hd, nkv, group, bs, dtype, lens, news, gate=True, extra_rows=1)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("hd, nkv, group, bs", [(64, 1, 8, 16), (128, 2, 5, 32), (256, 1, 8, 64), (256, 2, 1, 16)])
def test_prompts(fn, kv4, ws, dtype, hd, nkv, group, bs):
    lens, news = [150, 64, 300, 40, 97], [150, 64, 41, 100, 1]
    attn_case(fn, kv4, ws, hd * 5 + group, hd, nkv, group, bs, dtype, lens, news, gate=hd == 128)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("hd, n, length", [(256, 1, 9001), (128, 3, 5000), (64, 2, 12345)])
def test_long_requests_are_split(fn, kv4, ws, dtype, hd, n, length):
    lens = [length - 777 * i for i in range(n)]
    c, q, cu, table, out = attn_case(fn, kv4, ws, hd, hd, 1, 8, 64, dtype, lens, [1] * n)
    for _ in range(3):  # the same bits again, from the same workspace
        assert torch.equal(c.attn(q[..., :hd], dev(cu), dev(np.array(lens, np.int32)), dev(table), 1), out)


@pytest.mark.parametrize("max_new", [1, 64])
def test_more_requests_than_threads(fn, kv4, ws, max_new):
    """Several requests a thread in the scan of the lengths (both kernels), idle and empty ones among them."""
    rng = np.random.default_rng(23)
    lens = rng.integers(0, 40, 1100).tolist()
    news = rng.integers(0, 3, 1100).tolist()
    lens[600], news[600] = 500, 2
    attn_case(fn, kv4, ws, 24, 64, 1, 2, 16, "f32", lens, news, max_new=max_new, extra_rows=1)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_one_long_request_among_short_ones(fn, kv4, ws, dtype):
    """Many row tiles, one of them in dozens of parts; the same for a prompt slice behind a long context."""
    attn_case(fn, kv4, ws, 21, 64, 1, 8, 64, dtype, [20000] + [5 + i for i in range(39)], [1] * 40)
    attn_case(fn, kv4, ws, 22, 64, 1, 1, 64, dtype, [20000], [100])


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_long_prompt_slices(fn, kv4, ws, dtype):
    attn_case(fn, kv4, ws, 9, 128, 1, 2, 16, dtype, [2500, 900], [130, 333])


@pytest.mark.parametrize("max_new", [1, 3, 64, 4096])
def test_the_bound_on_new_tokens_only_chooses_the_kernel(fn, kv4, ws, max_new):
    for dtype in ("f32", "bf16"):
        attn_case(fn, kv4, ws, 11, 128, 2, 4, 32, dtype, [100, 37, 260], [1, 37, 9], max_new=max_new)


@pytest.mark.parametrize("qscale", [1e-6, 30.0])
def test_flat_and_peaked_rows(fn, kv4, ws, qscale):
    """Scores near zero, and scores of some hundreds. Their error grows with their size: compared where one key holds all."""
    rng = np.random.default_rng(3)
    c, pages, table, dtable = build(kv4, fn, ws, rng, 128, 1, 32, [200, 90])
    q = rng.standard_normal((2, 4, 128)).astype(np.float32) * qscale
    out = c.attn(dev(q), dev(offsets([1, 1])), dev(np.array([200, 90], np.int32)), dev(dtable), 1)
    want = O.attn(pages, 128, 32, q, [0, 1, 2], [200, 90], table)
    # a score of size S = 12 qscale is off by up to 2^-20 S, a weight by that share
    tol = (2e-5 + 2.0 ** -20 * 12 * qscale) * 4
    assert np.abs(out.cpu().numpy() - want).max() <= tol


def test_values_of_any_scale(fn, kv4, ws):
    """V of 1e-6 and of 3e4 beside each other: the sums keep their precision relative to each block's size."""
    rng = np.random.default_rng(4)
    for s in (1e-4, 1.0, 3e4):
        hd, bs = 128, 16
        c = kv4.KV4Cache(fn, 1, hd, bs, 8, ws)
        k = rng.standard_normal((100, 1, hd)).astype(np.float32)
        v = (rng.standard_normal((100, 1, hd)) * s).astype(np.float32)
        slots = np.arange(100)
        c.store(dev(k), dev(v), dev(slots))
        table = np.arange(7, dtype=np.int32)[None]
        q = rng.standard_normal((1, 8, hd)).astype(np.float32)
        out = c.attn(dev(q), dev(offsets([1])), dev(np.array([100], np.int32)), dev(table), 1)
        want = O.attn(c.pages.cpu().numpy(), hd, bs, q, [0, 1], [100], table)
        assert np.abs(out.cpu().numpy() - want).max() <= 2e-5 * 4 * s


def test_nan_reaches_only_the_rows_that_see_it(fn, kv4, ws):
    rng = np.random.default_rng(6)
    for hd, news in ((128, 8), (256, 60)):
        c, pages, table, dtable = build(kv4, fn, ws, rng, hd, 1, 16, [70, 70])
        bad = 66  # position whose value is NaN, in request 0
        x = torch.randn(1, 1, hd, device="cuda")
        nan = x.clone()
        nan[0, 0, 0] = float("nan")
        c.store(x, nan, torch.tensor([int(dtable[0, bad // 16]) * 16 + bad % 16], device="cuda"))
        q = torch.randn(2 * news, 4, hd, device="cuda")
        out = c.attn(q, dev(offsets([news, news])), dev(np.array([70, 70], np.int32)), dev(dtable), news)
        sees = torch.arange(70 - news, 70) >= bad
        assert out[:news][sees].isnan()[..., :64].all() and not out[:news][sees].isnan()[..., 64:].any()
        assert not out[:news][~sees].isnan().any() and not out[news:].isnan().any()


def test_nan_query_rows_stay_alone(fn, kv4, ws):
    rng = np.random.default_rng(7)
    for hd, news in ((128, 1), (128, 40)):
        c, _, _, dtable = build(kv4, fn, ws, rng, hd, 1, 16, [70])
        q = torch.randn(news, 4, hd, device="cuda")
        clean = c.attn(q, dev(offsets([news])), dev(np.array([70], np.int32)), dev(dtable), news)
        q2 = q.clone()
        q2[0, 1, 5] = float("nan")
        out = c.attn(q2, dev(offsets([news])), dev(np.array([70], np.int32)), dev(dtable), news)
        assert out[0, 1].isnan().all()
        out[0, 1] = clean[0, 1]
        assert torch.equal(out, clean)


def test_pages_past_four_gigabytes(fn, kv4, ws):
    rng = np.random.default_rng(8)
    hd, nkv, bs = 256, 2, 64
    base = (5 << 30) // (nkv * O.record_bytes(hd, bs))
    lens, news = [130, 64], [1, 20]
    c, pages, table, dtable = build(kv4, fn, ws, rng, hd, nkv, bs, lens, n_pages=base + 10, base=base)
    q = rng.standard_normal((21, 16, hd)).astype(np.float32)
    want = O.attn(pages, hd, bs, q, offsets(news), lens, table)
    for max_new in (1, 20):
        check(c.attn(dev(q), dev(offsets(news)), dev(np.array(lens, np.int32)), dev(dtable), max_new), want, "f32")
    slot = torch.tensor([int(dtable[0, 0]) * bs + 5], device="cuda")
    k, v = c.load(slot)
    wk, wv = O.load(pages, hd, bs, [int(table[0, 0]) * bs + 5])
    assert np.array_equal(k.cpu().numpy(), wk.astype(np.float32)) and np.array_equal(v.cpu().numpy(), wv.astype(np.float32))


@pytest.mark.parametrize("news", [1, 30])
def test_bad_page_ids_are_reported(fn, kv4, ws, news):
    """A table entry that is no page: its keys count as unseen, the call is reported, other requests are untouched."""
    rng = np.random.default_rng(10)
    c, pages, table, dtable = build(kv4, fn, ws, rng, 128, 2, 32, [100, 100])
    cu, lens = offsets([news, news]), [100, 100]
    q = rng.standard_normal((2 * news, 4, 128)).astype(np.float32)
    want = O.attn(pages, 128, 32, q, cu, lens, table)
    for bad in (-1, 1 << 20):
        t = dtable.copy()
        t[0, 1] = bad
        out = c.attn(dev(q), dev(cu), dev(np.array(lens, np.int32)), dev(t), news)
        with pytest.raises(RuntimeError, match="argument check"):
            fn.sync(torch.cuda.current_stream().cuda_stream)
        check(out[news:], want[news:], "f32")


@pytest.mark.parametrize("news", [1, 30])
def test_lengths_past_the_table_are_clamped(fn, kv4, ws, news):
    rng = np.random.default_rng(12)
    c, pages, table, dtable = build(kv4, fn, ws, rng, 64, 1, 16, [96])
    t = dtable[:, :6].copy()  # 96 tokens and no more
    q = rng.standard_normal((news, 2, 64)).astype(np.float32)
    a = c.attn(dev(q), dev(offsets([news])), dev(np.array([96], np.int32)), dev(t), news)
    b = c.attn(dev(q), dev(offsets([news])), dev(np.array([1000], np.int32)), dev(t), news)
    fn.sync(torch.cuda.current_stream().cuda_stream)
    assert torch.equal(a, b)


@pytest.mark.parametrize("news", [1, 40])
def test_other_streams_strides_and_given_outputs(fn, kv4, ws, news):
    rng = np.random.default_rng(13)
    own = kv4.KV4Workspace(fn)
    hd, nh = 128, 8
    c, pages, table, dtable = build(kv4, fn, own, rng, hd, 2, 16, [200, 77])
    cu, lens = dev(offsets([news, news])), dev(np.array([200, 77], np.int32))
    wide = torch.randn(2 * news, 3, nh, hd + 8, device="cuda")
    q, g = wide[:, 0, :, :hd], wide[:, 2, :, 8:]  # token stride 3 nh (hd + 8), head stride hd + 8
    want = O.attn(pages, hd, 16, q.cpu().numpy(), offsets([news, news]), [200, 77], table, gate=g.cpu().numpy())
    buf = torch.full((2 * news, nh * hd + 24), 7.0, device="cuda")
    out = buf[:, :nh * hd].unflatten(1, (nh, hd))
    t = dev(dtable)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        assert c.attn(q, cu, lens, t, news, gate=g, out=out) is out
    s.synchronize()
    check(out, want, "f32")
    assert (buf[:, nh * hd:] == 7).all()


@pytest.mark.parametrize("news", [1, 40])
def test_unaligned_rows(fn, kv4, ws, news):
    """q, gate and out whose rows start at any multiple of their type."""
    rng = np.random.default_rng(14)
    for dtype in ("f32", "bf16"):
        hd, nh = 64, 3
        c, pages, table, dtable = build(kv4, fn, ws, rng, hd, 1, 16, [90])
        x = torch.randn(news, nh * hd + 1, device="cuda").to(DT[dtype])
        q = x[:, 1:].unflatten(1, (nh, hd))
        out = torch.empty(news, nh * hd + 3, device="cuda", dtype=DT[dtype])[:, 1:1 + nh * hd].unflatten(1, (nh, hd))
        c.attn(q, dev(offsets([news])), dev(np.array([90], np.int32)), dev(dtable), news, gate=q, out=out)
        f = q.float().cpu().numpy()
        check(out, O.attn(pages, hd, 16, f, [0, news], [90], table, gate=f), dtype)


def test_a_step_in_a_cuda_graph(fn, kv4, ws):
    """plan, store and attend captured once, replayed with other lengths: the device-side lengths decide everything."""
    rng = np.random.default_rng(15)
    n, hd, nkv, bs, nh, width = 4, 128, 2, 16, 8, 8
    c = kv4.KV4Cache(fn, nkv, hd, bs, n * width, ws)
    pl = kv4.KV4Planner(fn, bs)
    free = dev(rng.permutation(n * width).astype(np.int32))
    table = torch.full((n, width), -1, dtype=torch.int32, device="cuda")
    count = torch.tensor([n * width], dtype=torch.int32, device="cuda")
    ctx = torch.zeros(n, dtype=torch.int32, device="cuda")
    add = torch.ones(n, dtype=torch.int32, device="cuda")
    k, v = torch.randn(2, n, nkv, hd, device="cuda")
    q = torch.randn(n, nh, hd, device="cuda")
    out = torch.empty_like(q)

    def step():
        p = pl.plan(ctx, add, table, free, count, n)
        c.store(k, v, p.slots)
        c.attn(q, p.cu, p.kv_len, table, 1, out=out)
        ctx.copy_(p.kv_len)
        count.copy_(p.free_count)

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    s.synchronize()
    keep = [(k.clone(), v.clone())]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s, capture_error_mode="thread_local"):
        step()
    for i in range(40):
        with torch.cuda.stream(s):
            k.normal_()
            v.normal_()
            q.normal_()
            keep.append((k.clone(), v.clone()))
            graph.replay()
        s.synchronize()
        if i in (0, 14, 15, 39):
            assert ctx.tolist() == [i + 2] * n
            pages = c.pages.cpu().numpy()
            want = O.attn(pages, hd, bs, q.cpu().numpy(), np.arange(n + 1), ctx.tolist(), table.cpu().numpy())
            check(out, want, "f32")
            first = O.load(pages, hd, bs, [int(table[0, t // bs]) * bs + t % bs for t in range(i + 2)])[0]
            ref = torch.stack([x[0][0] for x in keep]).cpu().numpy()
            cc, ss = O.quantise(ref.reshape(i + 2, nkv, -1, 64))
            assert np.array_equal(first, O.values(cc, ss).reshape(i + 2, nkv, hd))


def test_tensors_of_the_wrong_kind_are_refused(fn, kv4, ws):
    c = kv4.KV4Cache(fn, 2, 64, 16, 4, ws)
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    q, cu, kv_len, table = torch.zeros(1, 4, 64, device="cuda"), i32(0, 1), i32(3), i32([0, 1])
    for bad in (dict(q=q.half()), dict(q=q[..., :32]), dict(q=q.cpu()), dict(cu=cu.long()), dict(kv_len=kv_len.cpu()),
                dict(table=table.long()), dict(cu=i32(0, 1, 1)), dict(q=torch.zeros(1, 4, 128, device="cuda")[..., ::2]),
                dict(gate=q[:, :2]), dict(out=torch.zeros(2, 4, 64, device="cuda")), dict(gate=q.bfloat16())):
        a = dict(q=q, cu=cu, kv_len=kv_len, table=table, max_new=1)
        a.update(bad)
        with pytest.raises(ValueError):
            c.attn(**a)
    with pytest.raises(RuntimeError, match="head counts"):
        c.attn(torch.zeros(1, 5, 64, device="cuda"), cu, kv_len, table, 1)
    k = torch.zeros(2, 2, 64, device="cuda")
    for a in ((k, k, i32(0, 1)), (k, k[:1], torch.zeros(2, dtype=torch.int64, device="cuda")), (k, k.bfloat16(), torch.zeros(
            2, dtype=torch.int64, device="cuda")), (k[:, :1], k, torch.zeros(2, dtype=torch.int64, device="cuda"))):
        with pytest.raises(ValueError):
            c.store(*a)
    with pytest.raises(ValueError):
        c.load(torch.zeros(2, dtype=torch.int64, device="cuda"), torch.float16)
    with pytest.raises(ValueError):
        kv4.KV4Cache(fn, 2, 64, 16, torch.zeros(4, 2, 100, dtype=torch.uint8, device="cuda"), ws)
