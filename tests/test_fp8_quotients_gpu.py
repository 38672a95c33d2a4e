"""GPU: 8-bit rows and weights against true quotients, a / 448 and y 448 / a in 64 bits.

Tolerances. A scale is a times the rounded 1 / 448, rounded: 2 roundings, 2^-23 of itself. A code is the rounding of y times 448 times the
rounded 1 / a, three roundings before the one to e4m3: it is what some number within 3 * 2^-24 < 2^-22 of the true quotient rounds to. From
a = 2^126 on 1 / a is below fp32's normal numbers and rounded at 2^-150, so up to 2^-22 of itself more: 2^-21. A group that holds an infinity
(the largest scale makes some) has no quotients: its scale is infinite, its codes are NaN there and 0 elsewhere.
"""

import numpy as np
import pytest
import torch
from test_fp8_gpu import fp8, np64, rand  # noqa: F401

from oracle import fp8 as O

pytestmark = pytest.mark.gpu


def near(got, scale, y, down):
    rows, cols = y.shape
    a = np.zeros(scale.shape)
    for i in range(a.shape[0]):
        for j in range(a.shape[1]):
            a[i, j] = max(np.abs(y[i * down:(i + 1) * down, j * 128:(j + 1) * 128]).max(), O.TINY)
    sick, sick_y = np.isinf(a), np.isinf(O.spread(a, rows, cols, down))
    assert (scale[sick] == np.inf).all() and (np.isnan(got[sick_y]) == np.isinf(y[sick_y])).all() and (np.nan_to_num(got[sick_y]) == 0).all()
    got, y, a, scale = np.where(sick_y, 0, got), np.where(sick_y, 0, y), np.where(sick, 1, a), np.where(sick, 1 / 448, scale)
    assert (np.abs(scale - a / 448) <= 2.0 ** -23 * a / 448).all()
    v, tol = y * 448 / O.spread(a, rows, cols, down), np.where(O.spread(a, rows, cols, down) < 2.0 ** 126, 2.0 ** -22, 2.0 ** -21)
    lo, hi = np.sort(np.stack([O.e4m3(v * (1 - tol)), O.e4m3(v * (1 + tol))]), 0)
    assert ((got >= lo) & (got <= hi)).all()


@pytest.mark.parametrize("scale", [1.0, 1e-30, 2.0 ** 100, 6e37])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_true_quotients(fn, fp8, dtype, scale):  # noqa: F811
    x, w = rand(300, 1040, dtype, 1, scale), rand(400, 528, dtype, 2, scale)
    got, blocks = fp8.quantise_rows(fn, x), fp8.Fp8Weight.quantise(fn, w)
    near(np64(got.q), np64(got.scale), np64(x), 1)
    near(np64(blocks.q), np64(blocks.scale), np64(w), 128)
