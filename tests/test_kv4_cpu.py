"""CPU: the paged 4-bit KV cache's oracle on hand-made cases, and the C entries' refusals (before any device work)."""

import ctypes as C

import numpy as np
import pytest

from fn import FN, FnKv4
from oracle import kv4 as O


def test_oracle_quantises_to_half_a_step():
    rng = np.random.default_rng(0)
    x = rng.standard_normal((50, 64)).astype(np.float32)
    c, s = O.quantise(x)
    # the signed maximum takes code 0 exactly; on its side the codes reach it, on the other they end at 7 d
    err = np.abs(O.values(c, s) - x)
    step = np.abs(s.astype(np.float64))[:, None]
    # half a step, a whole one at the clipped end (x / d in 7.5 .. 8), and the scale's fp16 rounding over 8 steps
    assert (err <= np.where(x / s[:, None] > 7.5 - 1e-2, 1.0, 0.5) * step * (1 + 1e-4) + 8 * step * 2.0 ** -11).all()
    i = np.abs(x).argmax(-1)
    assert (c[np.arange(50), i] == 0).all()


def test_oracle_blocks_of_zeros_and_nans():
    x = np.zeros((4, 64), np.float32)
    x[1, 3] = np.nan
    x[2, 5] = np.inf
    x[3, 7] = 8.1 * 65504
    c, s = O.quantise(x)
    assert (O.values(c[:1], s[:1]) == 0).all()
    assert np.isnan(O.values(c[1:], s[1:])).all()


def test_oracle_opposite_extremes_take_the_positive():
    x = np.zeros((1, 64), np.float32)
    x[0, 10], x[0, 20] = -3.0, 3.0
    c, s = O.quantise(x)
    assert s[0] == -0.375 and c[0, 20] == 0 and c[0, 10] == 15


def test_oracle_store_load_round_trip():
    rng = np.random.default_rng(1)
    hd, bs, nkv = 128, 16, 3
    pages = np.zeros((4, nkv, O.record_bytes(hd, bs)), np.uint8)
    k, v = rng.standard_normal((2, 5, nkv, hd)).astype(np.float32)
    slots = [17, 63, -1, 0, 64]  # the third is padding, the last past the pages
    O.store(pages, hd, bs, k, v, slots)
    lk, lv = O.load(pages, hd, bs, slots)
    for t in (0, 1, 3):
        assert np.abs(lk[t] - k[t]).max() < 0.6 and np.abs(lv[t] - v[t]).max() < 0.6
        c, s = O.quantise(k[t].reshape(nkv, -1, 64))
        assert np.array_equal(lk[t], O.values(c, s).reshape(nkv, hd))
    assert not lk[[2, 4]].any() and not lv[[2, 4]].any()


def test_oracle_attention_is_softmax_over_the_visible_keys():
    rng = np.random.default_rng(2)
    hd, bs = 64, 16
    pages = np.zeros((3, 1, O.record_bytes(hd, bs)), np.uint8)
    k, v = rng.standard_normal((2, 20, 1, hd)).astype(np.float32)
    table = np.array([[2, 0]], np.int32)
    slots = [int(table[0, t // bs]) * bs + t % bs for t in range(20)]
    O.store(pages, hd, bs, k, v, slots)
    lk, lv = O.load(pages, hd, bs, slots)
    q = rng.standard_normal((22, 2, hd))
    out = O.attn(pages, hd, bs, q, [0, 22], [20], table)
    assert not out[:2].any()  # two rows more than keys: the first two see nothing
    assert np.allclose(out[2, 1], lv[0, 0])  # the next sees one key
    s = lk[:, 0] @ q[21, 0] / 8
    p = np.exp(s) / np.exp(s).sum()
    assert np.allclose(out[21, 0], p @ lv[:, 0])


def test_oracle_plan_takes_and_returns_pages():
    table = np.full((3, 4), -1, np.int32)
    table[0, :2] = [5, 3]
    table[1, :1] = [7]
    free = np.array([9, 8, 1, 0, 0], np.int32)
    o = O.plan([30, 16, 0], [-1, 1, 20], table, 16, free, 3, 10, 24)
    # request 0 returns 5 and 3; request 1 takes 3; request 2 takes 5 and 1
    assert list(o["table"][1, :2]) == [7, 3] and list(o["table"][2, :2]) == [5, 1]
    assert o["free_count"] == 2 and list(o["free"][:2]) == [9, 8] and o["status"] == 0
    assert list(o["cu"]) == [0, 0, 1, 21] and list(o["kv_len"]) == [0, 17, 20]
    assert list(o["slots"][:2]) == [48, 80] and list(o["slots"][17:]) == [16, 17, 18, 19, -1, -1, -1]
    assert list(o["requests"][20:]) == [2, -1, -1, -1]


@pytest.fixture(scope="module")
def f(libpath):
    return FN(libpath)


def cache(pages=0x10000, n_pages=4, page_size=16, nkv=2, hd=128):
    return FnKv4(pages, n_pages, page_size, nkv, hd)


ONE = 0x20000  # a pointer that must never be read


def refused(rc, f, word):
    assert rc == -1
    assert word in f.d.fn_error().decode()


@pytest.mark.parametrize("bad, word", [
    (dict(pages=0), "no cache"), (dict(pages=0x10008), "aligned"), (dict(hd=96), "head dim"), (dict(page_size=48), "page size"),
    (dict(page_size=128), "page size"), (dict(nkv=0), "counts"), (dict(n_pages=0), "counts")])
def test_bad_caches_are_refused(f, bad, word):
    c = C.byref(cache(**bad))
    refused(f.d.fn_kv4_store(c, 0, ONE, 256, 128, ONE, 256, 128, ONE, 1, None), f, word)
    refused(f.d.fn_kv4_load(c, 0, ONE, 1, ONE, ONE, None), f, word)
    refused(f.d.fn_kv4_attn(c, 0, 1, 1, 4, ONE, 512, 128, None, 0, 0, ONE, 512, ONE, ONE, ONE, 4, 1, 1.0, ONE, 1 << 40, None),
            f, word)


def test_bad_rows_are_refused(f):
    c = C.byref(cache())
    refused(f.d.fn_kv4_store(c, 1, ONE, 256, 128, ONE, 256, 128, ONE, 1, None), f, "F32 or BF16")
    refused(f.d.fn_kv4_store(c, 0, None, 256, 128, ONE, 256, 128, ONE, 1, None), f, "null")
    refused(f.d.fn_kv4_store(c, 0, ONE + 2, 256, 128, ONE, 256, 128, ONE, 1, None), f, "aligned")
    refused(f.d.fn_kv4_store(c, 0, ONE, 256, 128, ONE, 256, 128, ONE, -1, None), f, "row count")
    refused(f.d.fn_kv4_load(c, 8, ONE, 1, ONE, ONE, None), f, "F32 or BF16")
    refused(f.d.fn_kv4_load(c, 0, ONE, 1, None, None, None), f, "null")
    refused(f.d.fn_kv4_load(c, 0, ONE, 1, ONE + 4, ONE, None), f, "aligned")
    assert f.d.fn_kv4_store(c, 0, None, 0, 0, None, 0, 0, None, 0, None) == 0  # no rows, nothing to do
    assert f.d.fn_kv4_load(c, 0, None, 0, None, None, None) == 0


def attn_args(**k):
    a = dict(type=0, n=1, rows=1, nh=4, q=ONE, qt=512, qh=128, gate=None, gt=0, gh=0, out=ONE, ot=512, cu=ONE, kv=ONE,
             table=ONE, max_pages=4, max_new=1, scale=1.0, ws=ONE, wsb=1 << 40, stream=None)
    a.update(k)
    return list(a.values())


@pytest.mark.parametrize("bad, word", [
    (dict(type=8), "F32 or BF16"), (dict(n=0), "requests"), (dict(n=4097), "requests"), (dict(nh=5), "head counts"),
    (dict(nh=0), "head counts"), (dict(nh=130), "head counts"), (dict(rows=-1), "counts"), (dict(max_pages=0), "counts"),
    (dict(max_new=-1), "counts"), (dict(q=None), "null"), (dict(out=None), "null"), (dict(ws=None), "null"),
    (dict(table=None), "null"), (dict(rows=1 << 30), "too many rows"), (dict(max_pages=1 << 28), "too wide"),
    (dict(q=ONE + 2), "aligned"), (dict(gate=ONE + 1), "aligned"), (dict(wsb=8), "workspace"), (dict(ws=ONE + 16), "workspace")])
def test_bad_attention_calls_are_refused(f, bad, word):
    refused(f.d.fn_kv4_attn(C.byref(cache()), *attn_args(**bad)), f, word)


def test_attention_of_no_rows_does_nothing(f):
    assert f.d.fn_kv4_attn(C.byref(cache()), *attn_args(rows=0, q=None, out=None)) == 0


@pytest.mark.parametrize("at, value, word", [
    (0, 0, "requests"), (0, 4097, "requests"), (5, 20, "page size"), (4, 0, "counts"), (7, 0, "counts"), (10, -1, "counts"),
    (1, None, "null"), (9, None, "null"), (13, None, "null"), (12, ONE, "array of its own")])
def test_bad_plans_are_refused(f, at, value, word):
    a = [1, ONE, ONE + 64, ONE, 4, 16, ONE, 4, ONE, ONE, 8, ONE, ONE + 128, ONE, ONE, ONE, ONE, None]
    a[at] = value
    refused(f.d.fn_kv4_plan(*a), f, word)
