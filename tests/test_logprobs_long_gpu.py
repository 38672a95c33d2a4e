"""GPU: sums of long rows of logits (flashnext/logprobs.py), against the definition in 64 bits.

Tolerance of ln Z and the entropy's quotient: a thread adds up to 512 terms before they join a sum in 64 bits. A sum of n terms, none
below zero, whose partial sums grow evenly is off by at most 2^-24 n / 2 of itself (a half step of each partial sum): 2^-16. The exponentials
carry 2^-22, their exponents' rounding 2^-24 of y weighted with 2^y y, the joins of 1024 threads and 8 CTAs 13 additions, 2^-20 in all. So
log probabilities are right within 2^-16 + 2^-20 + 2^-22 |x|; the entropy is ln Z - t / Z, two such errors, the second of them times t / Z.
"""

import pytest
import torch

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "bf16": torch.bfloat16}


def exact(x):
    """(ln Z, entropy) of one row in 64 bits, in pieces."""
    m = x.max().double()
    z = t = torch.zeros((), dtype=torch.float64, device="cuda")
    for part in x.split(1 << 24):
        d = part.double() - m
        e = torch.exp(d)
        z, t = z + e.sum(), t + (e * d).sum()
    return float(m + torch.log(z)), float(torch.log(z) - t / z), float((t / z).abs())


def row(kind, n, dtype):
    g = torch.Generator(device="cuda")
    g.manual_seed(n % 1000)
    if kind == "equal":
        x = torch.zeros(n, device="cuda", dtype=DT[dtype])
    elif kind == "two levels":
        x = torch.zeros(n, device="cuda", dtype=DT[dtype])
        x[:n // 2] = 1
    elif kind == "rising":  # the maximum moves all along
        x = torch.linspace(-30, 30, n, device="cuda").to(DT[dtype])
    else:
        x = torch.empty(n, device="cuda", dtype=DT[dtype]).normal_(generator=g).mul_(2)
    return x


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("kind", ["equal", "two levels", "rising", "random"])
@pytest.mark.parametrize("n, rows", [((1 << 26) + 3, 150), ((1 << 26) + 3, 1), ((1 << 26) + 3, 100), (151936, 200), (600011, 200), (1 << 28, 150), (1 << 28, 1)])
def test_sums_of_long_rows(fn, kind, n, rows, dtype):
    """rows 150, 200: CTAs of 256 threads; 1: eight CTAs a row; 100: one of 1024 threads."""
    import logprobs as lp
    x = row(kind, n, dtype)
    tokens = (torch.arange(rows, device="cuda") * (n // rows)).int()
    got = lp.token_logprobs(fn, x.expand(rows, n), tokens)
    fn.sync(torch.cuda.current_stream().cuda_stream)
    lnz, entropy, mean = exact(x)
    given = x[tokens.long()].double()
    tol = 2.0 ** -16 + 2.0 ** -20
    assert bool(((got.logprob.double() - (given - lnz)).abs() <= tol + 2.0 ** -22 * (given.abs() + abs(lnz))).all())
    assert float((got.entropy.double() - entropy).abs().max()) <= tol * (1 + mean) + 2.0 ** -22 * abs(entropy)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_sick_long_rows(fn, dtype):
    """NaN and +inf early and late in a long row, and -inf all along, reach the sums as in short ones."""
    import logprobs as lp
    n = (1 << 22) + 5
    x = torch.zeros(4, n, device="cuda", dtype=DT[dtype])
    x[0, 7], x[1, n - 9], x[2, 11] = float("nan"), float("inf"), float("inf")
    x[3] = -float("inf")
    for many in (1, 50):
        y = x.repeat(many, 1)
        got = lp.token_logprobs(fn, y, torch.full((4 * many,), 3, dtype=torch.int32, device="cuda"))
        fn.sync(torch.cuda.current_stream().cuda_stream)
        logprob, entropy = got.logprob.view(many, 4), got.entropy.view(many, 4)
        assert bool(torch.isnan(logprob[:, :3]).all()) and bool(torch.isnan(entropy[:, :3]).all())
        assert bool((logprob[:, 3] == -float("inf")).all()) and bool((entropy[:, 3] == 0).all())
