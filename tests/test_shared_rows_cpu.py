"""CPU: calls whose outputs share memory with what they read are refused before any device work, whatever the strides' signs are, and the
host code that tells agrees with sets of addresses."""

import ctypes as C
import os
import subprocess

import pytest

from fn import FN, FnFp8

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "faie2-flashnext_b200", "csrc")
AT = 1 << 20  # an address that must never be read

ROWS = dict(dtype=0, x=AT, x_stride=64, add=None, add_stride=0, weight=None, eps=1e-6, rows=2, cols=64, total=AT << 1, total_stride=64, normed=None,
            normed_stride=0, codes=AT << 2, scales=AT << 3)


@pytest.mark.parametrize("change", [
    dict(x_stride=-64, total=AT - 512), dict(x_stride=-64, total=AT - 256), dict(x_stride=-80, total=AT - 300),
    dict(add=AT << 1, add_stride=-64, total=(AT << 1) - 256), dict(x_stride=-64, normed=AT - 512, normed_stride=64)])
def test_rows_that_go_backwards(libpath, change):
    with pytest.raises(RuntimeError, match="lie over"):
        FN(libpath).fp8_rows(**{**ROWS, **change})


def test_products_into_rows_that_go_backwards(libpath):
    for out in (AT - 512, AT - 256, AT - 511 * 4):
        with pytest.raises(RuntimeError, match="other rows of add"):
            FN(libpath).fp8_product(C.byref(FnFp8(AT << 3, AT << 4, 64, 64)), AT << 1, AT << 2, 8, 0, AT, -64, out, 64)


@pytest.mark.parametrize("change", [
    dict(codes=AT), dict(codes=AT + 240), dict(codes=AT - 112), dict(scales=AT + 508), dict(scales=AT - 4), dict(add=AT << 4, add_stride=64, codes=(AT << 4) + 256),
    dict(codes=(AT << 1) + 496), dict(scales=AT << 1), dict(normed=AT << 4, normed_stride=64, scales=(AT << 4) + 4), dict(scales=(AT << 2) + 124),
    dict(weight=AT << 2), dict(weight=(AT << 3) - 240), dict(weight=(AT << 1) + 496), dict(weight=AT << 4, normed=(AT << 4) - 500, normed_stride=64),
    dict(x_stride=-64, codes=AT - 256), dict(x_stride=1 << 20, total=AT << 5, codes=AT + (4 << 20)), dict(x_stride=0, codes=AT + 240)])
def test_rows_whose_codes_lie_over_what_is_read(libpath, change):
    with pytest.raises(RuntimeError, match="share memory"):
        FN(libpath).fp8_rows(**{**ROWS, **change})


@pytest.mark.parametrize("change", [dict(codes=AT), dict(codes=AT + 256 * 4 + 240), dict(scales=AT + 4), dict(stride=1 << 20, scales=AT + (16 << 20)),
                                    dict(scales=(AT << 1) + 319)])
def test_blocks_whose_codes_lie_over_what_is_read(libpath, change):
    change = {k: v & ~3 if k == "scales" else v for k, v in change.items()}
    with pytest.raises(RuntimeError, match="share memory"):
        FN(libpath).fp8_blocks(**{**dict(dtype=0, w=AT, stride=64, rows=5, cols=64, codes=AT << 1, scales=AT << 2), **change})


@pytest.mark.parametrize("change", [dict(codes=AT), dict(codes=AT - 112), dict(scales=AT + 3 * 64 * 4 - 4), dict(scales=AT - 8), dict(weight=AT + 16),
                                    dict(weight=AT - 64 * 64 + 16), dict(w_scales=AT), dict(out_stride=1 << 20, codes=AT + (8 << 20))])
def test_products_over_what_they_read(libpath, change):
    c = {**dict(codes=AT << 1, scales=AT << 2, weight=AT << 3, w_scales=AT << 4, out_stride=64), **change}
    with pytest.raises(RuntimeError, match="out lies over codes or scales"):
        FN(libpath).fp8_product(C.byref(FnFp8(c["weight"], c["w_scales"], 64, 64)), c["codes"], c["scales"], 3, 0, None, 0, AT, c["out_stride"])


SCORES = dict(dtype=0, logits=AT, stride=128, rows=4, vocab=100, tokens=AT << 1, logprob=AT << 2, rank=AT << 3, entropy=AT << 4, top=3, top_ids=AT << 5,
              top_logprobs=AT << 6)


@pytest.mark.parametrize("change", [
    dict(logprob=AT), dict(rank=AT - 12), dict(entropy=AT + 3 * 512 + 396), dict(top_ids=AT + 512), dict(top_logprobs=AT - 44), dict(dtype=30, rank=AT + 256),
    dict(stride=-128, rank=AT - 3 * 512), dict(stride=0, top_ids=AT + 396), dict(logprob=(AT << 1) + 4), dict(rank=(AT << 1) - 4),
    dict(top_ids=AT << 1), dict(top_logprobs=(AT << 1) - 44)])
def test_scores_over_what_they_read(libpath, change):
    with pytest.raises(RuntimeError, match="lie over logits or tokens"):
        FN(libpath).logprobs(**{**SCORES, **change})


def run(tmp_path, body):
    src = tmp_path / "t.cpp"
    src.write_text('#include <cstdio>\n#include <random>\n#include <set>\n#include "fn_rows.h"\nint main() {\n std::mt19937 r(1);\n'
                   ' auto in = [&](int lo, int hi) { return (int64_t)(r() % (hi - lo + 1)) + lo; };\n' + body + "}\n")
    subprocess.run(["g++", "-std=c++20", "-O1", "-I", CSRC, str(src), "-o", str(tmp_path / "t")], check=True)
    return subprocess.run([str(tmp_path / "t")], check=True, capture_output=True, text=True).stdout


def test_mixed_rows_are_told(tmp_path):
    """Never apart when an address is both a written row's and another row's; apart for columns side by side and rows far off."""
    out = run(tmp_path, """
 int apart = 0, wrong = 0;
 for (int i = 0; i < 200000; ++i) {
     const int64_t rows = in(1, 5), cols = in(1, 6), a = 1000 + in(0, 40), as = cols + in(0, 8), b = 1000 + in(-10, 50);
     const int64_t bs = in(0, 3) ? (in(0, 1) ? as : -as) : in(-12, 12);
     bool meet = false;
     for (int64_t p = 0; p < rows; ++p)
         for (int64_t q = 0; q < rows; ++q)
             for (int64_t j = 0; j < cols; ++j) {
                 const int64_t k = a + p * as + j - b - q * bs;  // b's column at a's address
                 if (k >= 0 && k < cols && !(a == b && (as == bs || rows == 1))) meet = true;
             }
     const bool said = fn::rows_mixed((void *)(a * 4), as, (void *)(b * 4), bs, rows, cols, 4);
     wrong += meet && !said;
     apart += !said;
     if (!meet && as == bs && said) ++wrong;  // one step: told exactly
 }
 std::printf("%d %d\\n", wrong, apart > 20000);
""")
    assert out.split() == ["0", "1"]


def test_rows_and_bytes_are_told_exactly(tmp_path):
    out = run(tmp_path, """
 int wrong = 0, apart = 0;
 for (int i = 0; i < 300000; ++i) {
     const int64_t rows = in(1, 5), bytes = in(1, 9), p = 1000 + in(0, 30), stride = in(-20, 20), q = 1000 + in(-100, 130), n = in(1, 25);
     bool meet = false;
     for (int64_t k = 0; k < rows; ++k)
         for (int64_t j = 0; j < bytes; ++j) {
             const int64_t at = p + k * stride + j;
             if (at >= q && at < q + n) meet = true;
         }
     const bool said = fn::rows_meet_bytes((void *)p, stride, rows, bytes, (void *)q, n);
     wrong += meet != said;
     apart += !said;
 }
 std::printf("%d %d\\n", wrong, apart > 50000);
""")
    assert out.split() == ["0", "1"]
