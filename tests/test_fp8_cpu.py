"""CPU: the oracle of 8-bit rows and weights against torch's e4m3 and hand-made cases, and the refusals (before any device work)."""

import ctypes as C

import numpy as np
import pytest
import torch

from fn import FN, FnFp8
from oracle import fp8 as O


def test_oracle_values_are_e4m3():
    codes = np.arange(256, dtype=np.uint8)
    want = torch.from_numpy(codes).view(torch.float8_e4m3fn).double().numpy()
    assert np.array_equal(O.value(codes), want, equal_nan=True)


def test_oracle_rounds_as_e4m3():
    rng = np.random.default_rng(0)
    v = np.unique(O.value(np.arange(127)))
    mid = (v[1:] + v[:-1]) / 2
    x = np.concatenate([v, mid, mid * (1 + 2e-7), mid * (1 - 2e-7), rng.uniform(0, 448, 2000), rng.uniform(0, 0.02, 500)]).astype(np.float32)
    x = np.concatenate([x, -x])
    want = torch.from_numpy(x).to(torch.float8_e4m3fn).double().numpy()
    assert np.array_equal(O.e4m3(x), want)
    assert set(np.abs(O.e4m3(x))) <= set(v)


def test_oracle_groups():
    rng = np.random.default_rng(1)
    y = rng.standard_normal((5, 272)).astype(np.float32)
    y[2, 128:256] = 0
    y[3, 256:] = 1e-37
    q, s = O.groups(y, 1)
    assert s.shape == (5, 3) and s[2, 1] == np.float32(O.TINY) * (np.float32(1) / np.float32(448)) and not q[2, 128:256].any()
    assert np.abs(q).max(1).min() <= 448
    # half a step of e4m3 (2^-4 of the value) where codes are normal numbers, half the smallest step below; scales' and quotients' roundings
    off = np.abs(q * O.spread(s, 5, 272, 1) - y)
    assert (off <= np.abs(y) * (2.0 ** -4 + 2.0 ** -20) + O.spread(s, 5, 272, 1) * 2.0 ** -10).all()
    q, s = O.groups(rng.standard_normal((130, 144)), 128)
    assert s.shape == (2, 2) and (np.abs(q[:128, :128]).max(), np.abs(q[128:, 128:]).max()) == (448, 448)


def test_oracle_product_is_the_matrix_product():
    rng = np.random.default_rng(2)
    x, w = rng.standard_normal((3, 160)), rng.standard_normal((131, 160))
    xq, xs = O.groups(x, 1, fp32=False)
    wq, ws = O.groups(w, 128, fp32=False)
    y, size = O.product(xq, xs, wq, ws)
    want = sum(np.outer(xs[:, g], ws[np.arange(131) // 128, g]) * (xq[:, g * 128:(g + 1) * 128] @ wq[:, g * 128:(g + 1) * 128].T) for g in range(2))
    assert np.abs(y - want).max() <= 1e-12 * size.max()
    assert np.abs(y - x @ w.T).max() <= 2 ** -3 * size.max()


ROWS = dict(dtype=0, x=4096, x_stride=64, add=4096, add_stride=64, weight=4096, eps=1e-6, rows=2, cols=64, total=4096, total_stride=64,
            normed=4096, normed_stride=64, codes=4096, scales=4096)
BLOCKS = dict(dtype=0, w=4096, stride=64, rows=2, cols=64, codes=4096, scales=4096)
PRODUCT = dict(codes=4096, scales=4096, rows=2, dtype=0, add=4096, add_stride=64, out=4096, out_stride=64)


@pytest.mark.parametrize("change, words", [
    (dict(dtype=1), "F32 or BF16"), (dict(rows=-1), "bad row count"), (dict(cols=0), "multiple of 16"), (dict(cols=24), "multiple of 16"),
    (dict(x=None), "null pointer"), (dict(codes=None), "null pointer"), (dict(scales=None), "null pointer"),
    (dict(codes=None, scales=None, total=None, normed=None), "nothing to write"), (dict(x=4098), "aligned to their type"),
    (dict(add=4097, dtype=30), "aligned to their type"), (dict(weight=4100), "16-byte"), (dict(codes=4104), "16-byte")])
def test_rows_refuse(libpath, change, words):
    with pytest.raises(RuntimeError, match=words):
        FN(libpath).fp8_rows(**{**ROWS, **change})


@pytest.mark.parametrize("change, words", [
    (dict(dtype=8), "F32 or BF16"), (dict(rows=-1), "bad row count"), (dict(cols=8), "multiple of 16"), (dict(w=None), "null pointer"),
    (dict(codes=None), "null pointer"), (dict(scales=None), "null pointer"), (dict(w=4097), "aligned"), (dict(codes=4104), "aligned")])
def test_blocks_refuse(libpath, change, words):
    with pytest.raises(RuntimeError, match=words):
        FN(libpath).fp8_blocks(**{**BLOCKS, **change})


@pytest.mark.parametrize("weight, change, words", [
    ((None, 4096, 5, 64), {}, "no weight"), ((4096, None, 5, 64), {}, "no weight"), ((4096, 4096, 0, 64), {}, "bad weight"),
    ((4096, 4096, 5, 40), {}, "bad weight"), ((4104, 4096, 5, 64), {}, "16-byte"), ((4096, 4096, 5, 64), dict(dtype=1), "F32 or BF16"),
    ((4096, 4096, 5, 64), dict(rows=-1), "bad row"), ((4096, 4096, 5, 64), dict(codes=None), "null pointer"),
    ((4096, 4096, 5, 64), dict(scales=None), "null pointer"), ((4096, 4096, 5, 64), dict(out=None), "null pointer"),
    ((4096, 4096, 5, 64), dict(codes=4100), "16-byte"), ((4096, 4096, 5, 64), dict(out=4098), "aligned to their types"),
    ((4096, 4096, 5, 64), dict(add=4097, dtype=30), "aligned to their types"), ((4096, 4098, 5, 64), {}, "aligned to their types")])
def test_product_refuses(libpath, weight, change, words):
    with pytest.raises(RuntimeError, match=words):
        FN(libpath).fp8_product(C.byref(FnFp8(*weight)), **{**PRODUCT, **change})


@pytest.mark.parametrize("change, words", [
    (dict(total_stride=60), "rows that are written overlap"), (dict(normed_stride=0), "rows that are written overlap"), (dict(normed=4096), "total and normed"),
    (dict(total=4112), "lie over"), (dict(total=4096 + 256), "lie over"), (dict(normed=1 << 20, add=(1 << 20) - 16), "lie over"),
    (dict(total=1 << 20, add=1 << 20, add_stride=0), "lie over"), (dict(normed=(1 << 20) + 128, total=1 << 20, total_stride=128, normed_stride=128), "total and normed"),
    (dict(normed=(1 << 20) - 128, total=1 << 20, total_stride=128, normed_stride=128), "total and normed"), (dict(cols=(1 << 24) + 16), "bad row count")])
def test_rows_refuse_to_overlap(libpath, change, words):
    with pytest.raises(RuntimeError, match=words):
        FN(libpath).fp8_rows(**{**ROWS, "normed": 1 << 16, **change})


def test_more_refusals(libpath):
    f = FN(libpath)
    with pytest.raises(RuntimeError, match="bad row count"):
        f.fp8_blocks(**{**BLOCKS, "cols": (1 << 24) + 16})
    for change, words in ((dict(out_stride=63), "rows of out overlap"), (dict(add=4096 + 256), "other rows of add"), (dict(add=4080), "other rows of add"),
                          (dict(add_stride=0), "other rows of add")):
        with pytest.raises(RuntimeError, match=words):
            f.fp8_product(C.byref(FnFp8(1 << 16, 1 << 16, 64, 64)), **{**PRODUCT, **change})


def test_no_rows_is_no_work(libpath):
    f = FN(libpath)
    f.fp8_rows(**{**ROWS, "rows": 0})
    f.fp8_blocks(**{**BLOCKS, "rows": 0})
    f.fp8_product(C.byref(FnFp8(4096, 4096, 5, 64)), **{**PRODUCT, "rows": 0})


def test_layer_refuses(libpath):
    import fp8
    f = FN(libpath)
    with pytest.raises(ValueError, match="x"):
        fp8.quantise_rows(f, torch.zeros(2, 64))
    with pytest.raises(ValueError, match="w"):
        fp8.Fp8Weight.quantise(f, torch.zeros(2, 64))
    with pytest.raises(ValueError, match="weight"):
        fp8.Fp8Weight(f, torch.zeros(2, 64), torch.zeros(1, 1))
