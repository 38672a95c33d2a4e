"""GPU parity of the token scores (flashnext/logprobs.py over fn_logprobs) against the float64 oracle (oracle/logprobs.py).

Tolerances. Ids and ranks are equal. A logarithm of a sum: its terms carry ex2.approx's 2^-22 and the rounding of their exponents
(2^-24 of y, weighted with 2^y y: below 2^-24), a sum over n threads' partials in a tree of depth below 400 additions 2^-24 each of
which hits the partial sum only: 2^-21 in all for the rows here, absolutely in ln Z. Subtracting m and ln Z rounds at 2^-24 of
the result's parts. So logprob: 2^-20 + 2^-22 |x|; entropy, a mean of |y| times the same relative errors plus ln Z's: 2^-19 + 2^-20 H.
"""

import numpy as np
import pytest
import torch

from oracle import logprobs as O

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "bf16": torch.bfloat16}


@pytest.fixture(scope="module")
def lp(fn):
    import logprobs as m
    return m


def check(fn, lp, x, tokens, top, want_x=None, out=None):
    """x: a CUDA tensor; want_x: its values on the host (default: read back)."""
    tok = None if tokens is None else torch.tensor(tokens, dtype=torch.int32, device="cuda")
    got = lp.token_logprobs(fn, x, tok, top, out=out)
    fn.sync(torch.cuda.current_stream().cuda_stream)
    h = x.double().cpu().numpy()
    want = O.rows(h, [-1] * len(h) if tokens is None else tokens, top)
    assert np.array_equal(got.top_ids.cpu().numpy(), want["top_ids"])
    if tokens is not None:
        assert np.array_equal(got.rank.cpu().numpy(), want["rank"])
    big = np.abs(np.where(np.isfinite(h), h, 0)).max(1)
    for name, tol in (("logprob", 2.0 ** -20 + 2.0 ** -22 * big), ("top_logprobs", (2.0 ** -20 + 2.0 ** -22 * big)[:, None]),
                      ("entropy", 2.0 ** -19 + 2.0 ** -20 * np.nan_to_num(want["entropy"]))):
        if name == "logprob" and tokens is None:
            assert got.logprob is None and got.rank is None
            continue
        g, w = getattr(got, name).double().cpu().numpy(), want[name].astype(np.float64)
        # results are fp32: -max beside +max is -2 max, which that type rounds to -inf
        w = np.where(w < -3.4028235e38, -np.inf, w)
        assert np.array_equal(np.isnan(g), np.isnan(w)), name
        fine = np.isfinite(w)
        assert np.array_equal(g[~fine & ~np.isnan(w)], w[~fine & ~np.isnan(w)]), name
        off = np.where(fine, np.abs(np.where(fine, g, 0) - np.where(fine, w, 0)), 0)
        assert (off <= tol).all(), (name, float(off.max()))
    return got


def logits(rows, vocab, dtype, pad=0, seed=0, scale=3.0):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    x = torch.randn(rows, vocab + pad, device="cuda", generator=g) * scale
    return x.to(DT[dtype])[:, :vocab]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows, vocab, top, pad", [
    (1, 1, 0, 0), (1, 1, 32, 0), (3, 2, 5, 0), (2, 7, 7, 1), (5, 8, 3, 0), (4, 31, 32, 3), (1, 255, 20, 0), (3, 1023, 1, 5),
    (2, 4097, 20, 0), (1, 8191, 32, 0), (1, 16384, 20, 0), (1, 65537, 5, 1), (2, 151936, 20, 0), (40, 33000, 8, 7),
    (150, 9001, 32, 0), (700, 1500, 20, 3), (1, 262147, 20, 0)])
def test_rows(fn, lp, rows, vocab, top, pad, dtype):
    x = logits(rows, vocab, dtype, pad, seed=rows + vocab)
    tokens = np.random.default_rng(vocab).integers(0, vocab, rows)
    tokens[::2] = x[::2].float().argmax(1).cpu().numpy()
    check(fn, lp, x, tokens, top)


@pytest.mark.parametrize("vocab", [3, 900, 40000])
def test_no_tokens(fn, lp, vocab):
    check(fn, lp, logits(3, vocab, "f32"), None, 4)
    check(fn, lp, logits(3, vocab, "f32"), [-1, 2, -7], 4)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("vocab", [6, 513, 20001, 151936])
def test_orders_and_ties(fn, lp, vocab, dtype):
    """Rising, falling and equal entries, few values, the best entries all in one thread's words, and -0 beside +0."""
    i = torch.arange(vocab, device="cuda", dtype=torch.float32)
    few = logits(1, vocab, "f32", seed=3)[0].round().clamp(-1, 1)
    lump = logits(1, vocab, "f32", seed=4)[0]
    lump[(i.long() // 8) % 256 == 5] += 40
    zeros = torch.where(i % 2 == 0, -0.0, 0.0)
    start = torch.where(i < 40, 10.0, 0.0)
    end = torch.where(i >= vocab - 40, 10.0, 0.0)
    x = torch.stack([i / vocab * 8, -i / vocab * 8, i * 0, few, lump, zeros, start, end]).to(DT[dtype])
    for t in (0, vocab // 2, vocab - 1):
        check(fn, lp, x, [t] * len(x), 32)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("vocab", [5, 777, 30001])
def test_masks_and_extremes(fn, lp, vocab, dtype):
    low, inf = torch.finfo(DT[dtype]).min, float("inf")
    x = logits(12, vocab, dtype, seed=5).clone()
    x[0] = -inf
    x[1] = low
    x[2, 1:] = -inf
    x[3, :-1] = low
    x[4, ::2] = -inf
    x[5, 1::2] = low
    x[6, vocab // 2] = float("nan")
    x[7, vocab // 3] = inf
    x[8] = -inf
    x[8, 2] = -torch.finfo(DT[dtype]).max
    x[9] = torch.finfo(DT[dtype]).max
    x[10] = low
    x[10, 3] = torch.finfo(DT[dtype]).max
    x[11] *= 0
    for t in (0, 3, vocab // 2, vocab - 1):
        check(fn, lp, x, [t] * 12, min(20, 32))


def test_sure_rows(fn, lp):
    """One entry far above the others: the rest of the sum is small, and so is the entropy."""
    x = logits(6, 50000, "f32", seed=6)
    for r, far in enumerate((20.0, 30.0, 60.0, 100.0, 1e4, 1e30)):
        x[r, 7] = far
    check(fn, lp, x, [7] * 6, 3)


def test_tokens_past_the_vocabulary(fn, lp):
    x = logits(3, 100, "f32")
    tok = torch.tensor([5, 100, 2**31 - 1], dtype=torch.int32, device="cuda")
    got = lp.token_logprobs(fn, x, tok, 2)
    with pytest.raises(RuntimeError):
        fn.sync(torch.cuda.current_stream().cuda_stream)
    assert got.rank.tolist()[1:] == [-1, -1] and torch.isnan(got.logprob[1:]).all() and torch.isfinite(got.logprob[0])
    fn.sync(torch.cuda.current_stream().cuda_stream)


def test_far_rows(fn, lp):
    """Rows whose offset passes 2^31 elements."""
    buf = torch.zeros(2, (1 << 31) + 64, dtype=torch.bfloat16, device="cuda")
    x = buf[:, :5000]
    x.copy_(logits(2, 5000, "bf16", seed=8))
    check(fn, lp, x, [4, 4999], 9)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_counts_of_long_rows(fn, lp, dtype):
    """One long row, taken once and by as many rows as have small CTAs: ranks of millions are whole numbers. Two levels, e apart: n / 2
    entries of each, so Z e^-1 = n / 2 (1 + 1 / e); the sums are of equal terms, off by 2^-24 a step of a thread's 2^18 at most."""
    n, rows = 1 << 26, 200
    x = torch.zeros(n, device="cuda", dtype=torch.float32 if dtype == "f32" else torch.bfloat16)
    x[:n // 2] = 1
    tokens = torch.arange(rows, device="cuda", dtype=torch.int32) * 331337 + 5
    tokens[-1], tokens[-2], tokens[-3] = n - 1, n // 2, n // 2 - 1
    z = np.log(n / 2) + np.log1p(np.exp(-1.0))
    p = 1 / (1 + np.exp(-1.0))
    for r in (rows, 1):
        got = lp.token_logprobs(fn, x.expand(r, n), tokens[-r:].contiguous())
        torch.cuda.synchronize()
        assert torch.equal(got.rank, tokens[-r:])  # by value, then by index
        want = np.where(tokens[-r:].cpu().numpy() < n // 2, 0.0, -1.0) - z
        assert np.abs(got.logprob.double().cpu().numpy() - want).max() <= 2.0 ** -6
        assert abs(float(got.entropy[0]) - (z + 1 - p)) <= 2.0 ** -5


def test_streams_graphs_and_buffers(fn, lp):
    x, y = logits(8, 151936, "f32", seed=1), logits(700, 20000, "bf16", seed=2)
    tok = torch.arange(8, dtype=torch.int32, device="cuda")
    toky = torch.arange(700, dtype=torch.int32, device="cuda")
    a, b = lp.token_logprobs(fn, x, tok, 20), lp.token_logprobs(fn, y, toky, 7)
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(5):
        with torch.cuda.stream(s1):
            a1 = lp.token_logprobs(fn, x, tok, 20)
        with torch.cuda.stream(s2):
            b1 = lp.token_logprobs(fn, y, toky, 7)
    torch.cuda.synchronize()
    for p, q in zip(a + b, a1 + b1):
        assert torch.equal(p, q)
    xs, out = x.clone(), lp.token_logprobs(fn, x, tok, 20)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s1, capture_error_mode="thread_local"):
        lp.token_logprobs(fn, xs, tok, 20, out=out)
    xs.copy_(x.roll(1, 0))
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(out.entropy, a.entropy.roll(1, 0)) and torch.equal(out.top_ids, a.top_ids.roll(1, 0))
    with pytest.raises(ValueError, match="out"):
        lp.token_logprobs(fn, x, tok, 19, out=out)
    with pytest.raises(ValueError, match="out"):
        lp.token_logprobs(fn, x, None, 20, out=out)
    with pytest.raises(ValueError, match="tokens"):
        lp.token_logprobs(fn, x, tok.long(), 20)
    with pytest.raises(ValueError, match="logits"):
        lp.token_logprobs(fn, x.T, None, 20)


def test_same_bits_in_any_batch(fn, lp):
    """A row's results do not depend on the rows beside it, as long as it is shared between as many CTAs."""
    x = logits(700, 5000, "bf16", seed=11)
    tok = torch.zeros(700, dtype=torch.int32, device="cuda")
    a, b = lp.token_logprobs(fn, x, tok, 5), lp.token_logprobs(fn, x[100:400], tok[100:400], 5)
    for p, q in zip(a, b):
        assert torch.equal(p[100:400], q)
