"""GPU parity of 8-bit rows, weights and their product (flashnext/fp8.py over fn_fp8_*) against the float64 oracle (oracle/fp8.py).

Tolerances. Codes, scales, sums and normed rows are equal: the oracle takes the kernels' reciprocals and products in fp32 (a row's factor
from a sum in 64 bits, rounded once). Products: of small whole numbers and powers of two every sum is exact, so they are equal. Of any
numbers: a group's 128 products are exact, and an MMA adds 32 of them and the sum so far, aligned to the largest and cut no higher
than 2^-23 of it; four MMAs a group, 33 terms each: below 4 * 33 * 2^-23 < 2^-15 of the sum of the terms' magnitudes. The scales' product
and the sum over groups round at 2^-24 a step, for up to 64 groups 2^-18. bf16 outputs: 2^-8 of the value on top, fp32 2^-24.
"""

import numpy as np
import pytest
import torch

from oracle import fp8 as O

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "bf16": torch.bfloat16}


@pytest.fixture(scope="module")
def fp8(fn):
    import fp8 as m
    return m


def sync(fn):
    fn.sync(torch.cuda.current_stream().cuda_stream)


def rand(rows, cols, dtype, seed, scale=1.0, stride=None, shift=0):
    """[rows][cols] with a row stride of its own, `shift` elements from an aligned address."""
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    x = torch.empty(rows * (stride or cols) + shift, dtype=DT[dtype], device="cuda")[shift:].view(rows, -1)[:, :cols]
    x.copy_(torch.randn(rows, cols, device="cuda", generator=g) * scale)
    return x


def np64(t):
    return t.double().cpu().numpy()


def check_rows(fn, fp8, x, add, weight, eps=1e-6, in_place=False, normed=True):
    h = np64(x)
    if add is not None:
        h = np64((x.float() + add.float()).to(x.dtype))
    total = None if add is None else (x if in_place else torch.empty_like(x))
    y = torch.full_like(x, 7.0) if normed else None
    got = fp8.quantise_rows(fn, x, add=add, total=total, weight=weight, eps=eps, normed=y)
    sync(fn)
    want = O.rms(h, np64(weight), eps) if weight is not None else h.astype(np.float32)
    if total is not None:
        assert np.array_equal(np64(total), h, equal_nan=True)
    if normed:
        assert np.array_equal(np64(y), np64(torch.from_numpy(want.astype(np.float32)).to(x.dtype)), equal_nan=True)
    q, s = O.groups(want, 1)
    assert np.array_equal(np64(got.scale), s, equal_nan=True)
    assert np.array_equal(np64(got.q), q, equal_nan=True)
    return got


SHAPES = [(1, 16), (3, 128), (1, 144), (9, 256), (5, 272), (2, 512), (7, 1040), (1, 2048), (33, 2048), (4, 2064), (3, 4096), (2, 6000),
          (3, 8192), (2, 8208), (1, 16384), (300, 48)]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows, cols", SHAPES)
def test_rows(fn, fp8, rows, cols, dtype):
    x, add = rand(rows, cols, dtype, 1, 3.0), rand(rows, cols, dtype, 2)
    w = 1 + 0.1 * rand(1, cols, "f32", 3)[0]
    check_rows(fn, fp8, x, None, None)
    check_rows(fn, fp8, x, None, w, normed=False)
    check_rows(fn, fp8, x, add, w)
    check_rows(fn, fp8, x, add, None)
    check_rows(fn, fp8, x.clone(), add, w, in_place=True)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("cols, stride, shift", [(96, 97, 0), (2048, 2051, 1), (8208, 8209, 1), (2048, 4096, 0), (272, 272, 1)])
def test_rows_strided(fn, fp8, cols, stride, shift, dtype):
    x, add = rand(3, cols, dtype, 4, 1.0, stride, shift), rand(3, cols, dtype, 5, 1.0, stride + 3)
    w = rand(1, cols, "f32", 6)[0]
    check_rows(fn, fp8, x, add, w, in_place=True)
    check_rows(fn, fp8, x, None, None)


def test_rows_of_any_size(fn, fp8):
    """Values whose squares leave fp32, rows of zeros, tiny rows, infinities and NaN."""
    x = rand(9, 640, "f32", 7)
    for r, s in enumerate((1e30, 1e-30, 1e-38, 0.0, 1e38)):
        x[r] *= s
    x[5, 300], x[6, 1], x[7, 129] = float("nan"), float("inf"), 3e38
    x[8, 128:256] = 0
    w = rand(1, 640, "f32", 8)[0]
    check_rows(fn, fp8, x, None, None, normed=False)
    got = fp8.quantise_rows(fn, x, weight=w)
    sync(fn)
    bad = torch.isnan(got.values())
    assert bad[5].all() and bad[6].any() and not bad[[0, 1, 2, 3, 4, 7, 8]].any()
    want = O.rms(np64(x), np64(w), 1e-6, fp32=False)
    for r in (0, 1, 2, 3, 4, 7, 8):
        q, s = O.groups(want[r:r + 1], 1, fp32=False)
        # half a step of e4m3, or half the smallest one, and a last bit of the factors
        off = np.abs(np64(got.values())[r] - want[r])
        assert (off <= np.abs(want[r]) * (2.0 ** -4 + 2.0 ** -20) + O.spread(s, 1, 640, 1)[0] * 2.0 ** -9.9).all(), r


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows, cols", [(1000, 512), (3, 4096), (400, 8192), (150, 8208)])
def test_rows_in_place(fn, fp8, rows, cols, dtype):
    """total over add and normed over x, columns of one buffer side by side, one row added to all."""
    both = rand(rows, 2 * cols, dtype, 12)
    add, w = rand(1, cols, dtype, 13)[0].expand(rows, cols), 1 + 0.1 * rand(1, cols, "f32", 14)[0]
    h = (both[:, :cols].float() + add.float()).to(both.dtype)
    want = fp8.quantise_rows(fn, h, weight=w, normed=(y := torch.empty_like(h)))
    for norm, rows_ in ((w, want), (None, fp8.quantise_rows(fn, h))):
        b, t = both.clone(), torch.empty_like(h)
        got = fp8.quantise_rows(fn, b[:, :cols], add=add, total=b[:, cols:], weight=norm, normed=t)
        assert torch.equal(b[:, cols:], h) and torch.equal(b[:, :cols], both[:, :cols]) and torch.equal(t, y if norm is not None else h)
        x, a = both[:, :cols].clone(), add.clone()
        again = fp8.quantise_rows(fn, x, add=a, total=a, weight=norm, normed=x)
        assert torch.equal(a, h) and torch.equal(x, t)
        x, a = both[:, :cols].clone(), add.clone()
        third = fp8.quantise_rows(fn, a, add=x, weight=norm, normed=x)
        assert torch.equal(x, t)
        for r in (got, again, third):
            assert torch.equal(r.scale, rows_.scale) and torch.equal(r.q.view(torch.uint8), rows_.q.view(torch.uint8))
    with pytest.raises(RuntimeError, match="lie over"):
        fp8.quantise_rows(fn, both[:, :cols], add=add, total=both[:, 16:16 + cols])
    with pytest.raises(RuntimeError, match="overlap"):
        fp8.quantise_rows(fn, both[:, :cols], add=add, total=add)


@pytest.mark.parametrize("m, n", [(1, 16), (20, 5000), (40, 333), (600, 12352)])
def test_product_into_part_of_a_buffer(fn, fp8, m, n):
    """out among other columns, which stay as they were; one row added to all; add beside out."""
    x, w = fp8.quantise_rows(fn, rand(m, 272, "f32", 15)), fp8.Fp8Weight.quantise(fn, rand(n, 272, "f32", 16))
    bias, b = rand(1, n, "f32", 17)[0], rand(m, 2 * n + 8, "f32", 18)
    old, want = b.clone(), w.product(x)
    w.product(x, add=bias.expand(m, n), out=b[:, 4:4 + n])
    assert torch.equal(b[:, 4:4 + n], w.product(x, add=bias.expand(m, n).contiguous()))
    assert torch.equal(b[:, :4], old[:, :4]) and torch.equal(b[:, 4 + n:], old[:, 4 + n:])
    assert ((b[:, 4:4 + n] - want - bias).abs() <= 2.0 ** -22 * (want.abs() + bias.abs())).all()
    w.product(x, add=b[:, 4 + n:4 + 2 * n], out=b[:, 4:4 + n])
    assert torch.equal(b[:, 4:4 + n], w.product(x, add=old[:, 4 + n:4 + 2 * n].contiguous())) and torch.equal(b[:, 4 + n:], old[:, 4 + n:])
    if m > 1:
        with pytest.raises(RuntimeError, match="other rows of add"):
            w.product(x, add=b[:, :n], out=b[:, 4:4 + n])
        with pytest.raises(RuntimeError, match="overlap"):
            w.product(x, out=torch.empty(m, n, device="cuda")[:1].expand(m, n))


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows, cols", [(5, 2048), (1, 48), (700, 512)])
def test_rows_without_codes(fn, fp8, rows, cols, dtype):
    """The residual's addition and the norm alone."""
    x, add, w = rand(rows, cols, dtype, 9), rand(rows, cols, dtype, 10), rand(1, cols, "f32", 11)[0]
    y, want = torch.empty_like(x), (x.float() + add.float()).to(x.dtype)
    fp8.add_norm(fn, x, add, w, 1e-6, x, y)
    sync(fn)
    assert torch.equal(x, want)
    assert np.array_equal(np64(y), np64(torch.from_numpy(O.rms(np64(want), np64(w), 1e-6)).to(x.dtype)))
    with pytest.raises(ValueError, match="normed"):
        fp8.add_norm(fn, x, add, w, 1e-6, x, y[:, :16])
    with pytest.raises(ValueError, match="weight"):
        fp8.add_norm(fn, x, add, w[:16], 1e-6, x, y)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("rows, cols, stride, shift", [(1, 16, 16, 0), (128, 128, 128, 0), (513, 2048, 2048, 0), (130, 272, 275, 1), (7, 400, 400, 0),
                                                       (129, 128, 129, 0)])
def test_blocks(fn, fp8, rows, cols, stride, shift, dtype):
    w = rand(rows, cols, dtype, 12, 0.02, stride, shift)
    got = fp8.Fp8Weight.quantise(fn, w)
    sync(fn)
    q, s = O.groups(np64(w), 128)
    assert np.array_equal(np64(got.scale), s) and np.array_equal(np64(got.q), q)
    want = q * O.spread(s, rows, cols, 128)
    assert (np.abs(np64(got.values()) - want) <= 2.0 ** -24 * np.abs(want)).all()


# ---- products


def whole(rows, cols, down, seed):
    """Codes that are small whole numbers, scales that are powers of two."""
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    q = torch.randint(-4, 5, (rows, cols), device="cuda", generator=g).float().to(torch.float8_e4m3fn)
    s = torch.exp2(torch.randint(-1, 2, (-(-rows // down), -(-cols // 128)), device="cuda", generator=g).float())
    return q, s


def exact_product(xq, xs, wq, ws):
    x = xq.double() * xs.double().repeat_interleave(128, 1)[:, :xq.shape[1]]
    w = wq.double() * ws.double().repeat_interleave(128, 0)[:wq.shape[0]].repeat_interleave(128, 1)[:, :wq.shape[1]]
    return x @ w.T


PRODUCTS = [(1, 1, 16), (1, 8, 128), (2, 129, 144), (1, 12352, 256), (5, 513, 2048), (16, 128, 4096), (17, 2048, 2048), (32, 1000, 1040),
            (33, 257, 384), (50, 3000, 512), (64, 640, 272), (65, 130, 128), (80, 19000, 128), (97, 255, 656), (128, 128, 8192), (129, 384, 256),
            (200, 2048, 512), (333, 2048, 4096), (257, 100, 2064), (512, 512, 512), (1000, 1111, 1024), (2000, 4100, 384), (4096, 24, 128),
            (8192, 513, 256), (300, 20000, 144), (1500, 12352, 256), (2305, 5001, 1040), (3000, 8200, 144), (40, 12352, 128), (20, 30011, 384),
            (31, 9000, 1168)]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("m, n, k", PRODUCTS)
def test_products_of_whole_numbers(fn, fp8, m, n, k, dtype):
    (xq, xs), (wq, ws) = whole(m, k, 1, m + k), whole(n, k, 128, n + k)
    want = exact_product(xq, xs, wq, ws)
    w = fp8.Fp8Weight(fn, wq, ws)
    got = w.product(fp8.Fp8Rows(xq, xs), dtype=DT[dtype])
    sync(fn)
    assert torch.equal(got.double(), want.to(DT[dtype]).double())
    # added in, in place, in rows of a wider buffer whose other columns and rows stay
    buf = torch.randint(-50, 50, (m + 2, n + 5), device="cuda").to(DT[dtype])
    old = buf.clone()
    out = buf[1:m + 1, 2:n + 2]
    w.product(fp8.Fp8Rows(xq, xs), add=out, out=out)
    sync(fn)
    want = (want + old[1:m + 1, 2:n + 2].double()).to(DT[dtype])
    assert torch.equal(out, want)
    old[1:m + 1, 2:n + 2] = want
    assert torch.equal(buf, old)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("m, n, k", [(1, 2048, 2048), (32, 515, 4096), (100, 700, 8192), (333, 2048, 2048), (700, 1300, 1040), (2048, 1024, 2048)])
def test_products(fn, fp8, m, n, k, dtype):
    x = fp8.quantise_rows(fn, rand(m, k, "f32", m, 2.0) * torch.exp(rand(1, k, "f32", 1)))
    w = fp8.Fp8Weight.quantise(fn, rand(n, k, "f32", n, 0.02))
    add = rand(m, n, dtype, 5)
    got = np64(w.product(x, add=add, dtype=DT[dtype]))
    sync(fn)
    want, size = O.product(np64(x.q), np64(x.scale), np64(w.q), np64(w.scale))
    want = want + np64(add)
    off = np.abs(got - want)
    half = 2.0 ** -8 if dtype == "bf16" else 2.0 ** -24
    assert (off <= (2.0 ** -15 + 2.0 ** -18) * size + half * np.abs(want) * 1.01).all()
    # the cuts of a group's 132 additions, if all fell one way by half their bound of the largest product (some 2^3 of its rms, which
    # an output is sqrt(k) of): 66 * 2^-23 * 8 * k / 128 / sqrt(k) = 2^-21 sqrt(k) of an output, 2^-15 at most here
    assert np.sqrt((off ** 2).mean()) <= (2.0 ** -15 + half) * np.sqrt((want ** 2).mean())


def test_product_passes_nan_and_infinity(fn, fp8):
    (xq, xs), (wq, ws) = whole(40, 256, 1, 3), whole(300, 256, 128, 4)
    xs[3, 1], xs[5, 0] = float("nan"), float("inf")
    ws[2, 0] = float("nan")
    xq.view(torch.uint8)[7, 9] = 0x7f
    wq.view(torch.uint8)[11, 200] = 0xff
    got = fp8.Fp8Weight(fn, wq, ws).product(fp8.Fp8Rows(xq, xs))
    sync(fn)
    want = exact_product(xq, xs, wq, ws)
    bad = torch.isnan(got)
    assert bad[3].all() and bad[7].all() and bad[:, 256:].all() and bad[:, 11].all()
    fine = torch.isfinite(want)
    fine[5] = False
    assert torch.equal(got[fine].double(), want[fine])
    assert (~torch.isfinite(got[5])).all()


def test_a_row_is_the_same_in_any_batch(fn, fp8):
    x, w = fp8.quantise_rows(fn, rand(600, 1024, "f32", 1)), fp8.Fp8Weight.quantise(fn, rand(900, 1024, "f32", 2))
    whole_ = w.product(x)
    for lo, hi in ((0, 1), (7, 40), (100, 229), (0, 300), (300, 600)):
        part = w.product(fp8.Fp8Rows(x.q[lo:hi], x.scale[lo:hi]))
        assert torch.equal(part, whole_[lo:hi])
    sync(fn)


def test_far_rows(fn, fp8):
    """Codes and outputs whose offsets pass 32 bits."""
    row = rand(1, 4096, "bf16", 19)
    n = (1 << 20) + 3
    got = fp8.quantise_rows(fn, row.expand(n, 4096))
    want = fp8.quantise_rows(fn, row)
    sync(fn)
    for r in (0, 1, n // 2, n - 2, n - 1):
        assert torch.equal(got.q[r].view(torch.uint8), want.q[0].view(torch.uint8)) and torch.equal(got.scale[r], want.scale[0])
    del got
    x, w = fp8.quantise_rows(fn, rand(17001, 128, "bf16", 20)), fp8.Fp8Weight.quantise(fn, rand(262152, 128, "bf16", 21))
    out = w.product(x, dtype=torch.bfloat16)
    sync(fn)
    for lo in (0, 8000, 16900):
        assert torch.equal(out[lo:lo + 101], w.product(fp8.Fp8Rows(x.q[lo:lo + 101], x.scale[lo:lo + 101]), dtype=torch.bfloat16))
    h = fp8.Fp8Weight.quantise(fn, rand(3, 4096, "bf16", 22))
    far = torch.empty(1 << 28, 20, device="cuda", dtype=torch.bfloat16)[::1 << 20, :3]  # rows 40 MB apart
    assert torch.equal(h.product(fp8.Fp8Rows(want.q.expand(256, 4096).contiguous(), want.scale.expand(256, 32).contiguous()), out=far),
                       h.product(want, dtype=torch.bfloat16).expand(256, 3))


def test_streams_and_graphs(fn, fp8):
    """Weights quantised, rows normed and multiplied in one stream without waits, two streams at once, and a captured chain."""
    h, d = rand(40, 2048, "bf16", 1), rand(40, 2048, "bf16", 2)
    norm, wt = rand(1, 2048, "f32", 3)[0], rand(700, 2048, "f32", 4, 0.02)

    def chain(h, w, total, x, out):
        fp8.quantise_rows(fn, h, add=d, total=total, weight=norm, out=x)
        return w.product(x, out=out)

    def buffers():
        return torch.empty_like(h), fp8.empty_rows(40, 2048), torch.empty(40, 700, device="cuda")

    w = fp8.Fp8Weight.quantise(fn, wt)
    torch.cuda.synchronize()
    want = chain(h, w, *buffers()).clone()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    outs = []
    for _ in range(4):
        for s in (s1, s2):
            with torch.cuda.stream(s):
                outs.append(chain(h, fp8.Fp8Weight.quantise(fn, wt), *buffers()))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)
    b, hs = buffers(), h.clone()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s1, capture_error_mode="thread_local"):
        chain(hs, w, *b)
    hs.copy_(h.roll(1, 0))
    d.copy_(d.roll(1, 0))
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(b[2], want.roll(1, 0))


def test_layer_refuses(fn, fp8):
    x, w = fp8.quantise_rows(fn, rand(4, 256, "f32", 1)), fp8.Fp8Weight.quantise(fn, rand(20, 256, "f32", 2))
    z = lambda *s, **k: torch.zeros(*s, device="cuda", **k)  # noqa: E731
    for bad, words in ((dict(x=fp8.Fp8Rows(x.q[:, :128], x.scale)), "x"), (dict(x=fp8.Fp8Rows(x.q, x.scale[:2])), "scales"),
                       (dict(x=fp8.quantise_rows(fn, z(4, 128))), "columns"), (dict(x=x, out=z(4, 21)), "out"),
                       (dict(x=x, out=z(4, 20, dtype=torch.float16)), "out"), (dict(x=x, add=z(4, 20, dtype=torch.bfloat16)), "add"),
                       (dict(x=x, dtype=torch.float16), "dtype"), (dict(x=x, out=z(20, 4).T), "out"),
                       (dict(x=fp8.Fp8Rows(x.q.cpu(), x.scale.cpu())), "x")):
        with pytest.raises(ValueError, match=words):
            w.product(**bad)
    for bad, words in ((dict(x=z(2, 24)), "16"), (dict(x=z(2, 32), add=z(2, 48)), "add"), (dict(x=z(2, 32), total=z(2, 32, dtype=torch.bfloat16)), "total"),
                       (dict(x=z(2, 32), weight=z(16)), "weight"), (dict(x=z(2, 32), normed=z(3, 32)), "normed"), (dict(x=z(2, 32), out=x), "out")):
        with pytest.raises(ValueError, match=words):
            fp8.quantise_rows(fn, **bad)
    assert w.product(fp8.empty_rows(0, 256)).shape == (0, 20)
