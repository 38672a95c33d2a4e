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
