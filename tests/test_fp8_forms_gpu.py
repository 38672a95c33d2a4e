"""GPU: the product of 8-bit rows and weights in each of its forms, on numbers of any kind: the weight on the lanes (up to 32 rows of a
large weight), x on the lanes, pairs of SMs. With 148 SMs the rule of fn_fp8_product gives the forms that the cases are named by.

Tolerances: those of tests/test_fp8_gpu.py (up to 32 groups here). A row's bits are the same in every form: each adds a group's products
by MMAs 32 deep, four a group, scales a group's sum by the same rounded product of two scales and adds the groups in order.
"""

import pytest
import torch
from test_fp8_gpu import DT, exact_product, fp8, rand, sync  # noqa: F401

pytestmark = pytest.mark.gpu

FORMS = [("lanes16", 1, 12352, 2048), ("lanes16", 16, 5003, 4096), ("lanes32", 17, 12352, 1040), ("lanes32", 32, 12352, 4096),
         ("lanes32", 31, 151936, 2048), ("rows", 300, 12352, 2048), ("pairs", 1500, 12352, 2048), ("pairs", 513, 12351, 4096),
         ("pairs", 256, 12352, 2064)]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("form, m, n, k", FORMS)
def test_products_of_any_numbers(fn, fp8, form, m, n, k, dtype):  # noqa: F811
    x = fp8.quantise_rows(fn, rand(m, k, "f32", m, 2.0) * torch.exp(rand(1, k, "f32", 1)))
    w = fp8.Fp8Weight.quantise(fn, rand(n, k, "f32", n, 0.02) * torch.exp(rand(n, 1, "f32", 2)))
    add = rand(m, n, dtype, 5)
    got = w.product(x, add=add, dtype=DT[dtype]).double()
    want = exact_product(x.q, x.scale, w.q, w.scale) + add.double()
    size = exact_product(x.q.float().abs(), x.scale, w.q.float().abs(), w.scale)
    off = (got - want).abs()
    half = 2.0 ** -8 if dtype == "bf16" else 2.0 ** -24
    assert bool((off <= (2.0 ** -15 + 2.0 ** -18) * size + half * want.abs() * 1.01).all())
    assert float(off.square().mean().sqrt()) <= (2.0 ** -15 + half) * float(want.square().mean().sqrt())


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_a_row_is_the_same_in_any_form(fn, fp8, dtype):  # noqa: F811
    x, w = fp8.quantise_rows(fn, rand(1500, 2048, "f32", 1)), fp8.Fp8Weight.quantise(fn, rand(12352, 2048, "f32", 2))
    pairs = w.product(x, dtype=DT[dtype])
    for lo, hi in ((0, 1), (7, 20), (7, 27), (100, 140), (300, 600), (1244, 1500)):
        assert torch.equal(w.product(fp8.Fp8Rows(x.q[lo:hi], x.scale[lo:hi]), dtype=DT[dtype]), pairs[lo:hi]), (lo, hi)
    sync(fn)
