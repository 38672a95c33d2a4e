"""CPU: refusals of the paged 4-bit cache's later entries and layers, before any device work; what is done once per device."""

import os
import subprocess
from types import SimpleNamespace

import pytest

from fn import FN

ONE = 0x20000  # a pointer that must never be read


@pytest.fixture(scope="module")
def f(libpath):
    return FN(libpath)


@pytest.mark.parametrize("at, value, word", [(0, 0, "requests"), (5, 20, "page size"), (1, None, "null"), (17, ONE, "next must be"),
                                             (17, ONE + 64, "next must be"), (17, ONE + 128, "next must be")])
def test_bad_plans_with_carried_lengths_are_refused(f, at, value, word):
    a = [1, ONE, ONE + 64, ONE, 4, 16, ONE, 4, ONE, ONE, 8, ONE, ONE + 128, ONE, ONE, ONE, ONE, None, None]
    a[at] = value
    assert f.d.fn_kv4_plan_next(*a) == -1 and word in f.d.fn_error().decode()


def test_a_kernel_is_prepared_on_every_device(tmp_path):
    """The shared-memory limit of a kernel is raised where it was not: on each device, and from several threads."""
    csrc = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "faie2-flashnext_b200", "csrc")
    (tmp_path / "once.cpp").write_text("""
#include <thread>
#include <vector>
#include "fn_once.h"
int main() {
    fn::OncePerDevice once;
    int k[2];
    if (once.has(&k[0], 0)) return 1;
    once.add(&k[0], 0);
    if (!once.has(&k[0], 0) || once.has(&k[0], 1) || once.has(&k[1], 0)) return 2;
    std::vector<std::thread> t;
    for (int d = 0; d < 8; ++d) t.emplace_back([&, d] { for (int i = 0; i < 1000; ++i) once.add((char *)k + i, d); });
    for (auto &x : t) x.join();
    for (int d = 0; d < 8; ++d)
        for (int i = 0; i < 1000; ++i)
            if (!once.has((char *)k + i, d)) return 3;
    return 0;
}
""")
    subprocess.run(["g++", "-std=c++20", "-O1", "-pthread", "-I", csrc, str(tmp_path / "once.cpp"), "-o", str(tmp_path / "once")], check=True)
    assert subprocess.run([str(tmp_path / "once")]).returncode == 0


def test_tensors_of_another_device_are_refused():
    import kv4
    import torch

    def tensor(device, dtype=torch.int32):
        return SimpleNamespace(dtype=dtype, shape=(3,), is_contiguous=lambda: True, get_device=lambda: device, device=f"cuda:{device}")

    kv4._ints("cu", tensor(1), (3,), 1)
    for t, dev in ((tensor(0), 1), (tensor(1), 0), (tensor(-1), 0), (tensor(-1), -1), (tensor(0, torch.int64), 0)):
        with pytest.raises(ValueError, match="cu: a contiguous int32"):
            kv4._ints("cu", t, (3,), dev)
    # a planner's tensors have to be where its lengths are
    z = [torch.zeros(s, dtype=torch.int32) for s in ((2,), (2,), (2, 3), (4,), (1,))]
    with pytest.raises(ValueError, match="cuda"):
        kv4.KV4Planner(None, 16).plan(*z, 4)


def test_rows_that_may_meet_are_found(tmp_path):
    """Whether outputs may lie over q or gate, against every element of small layouts: nothing that does is missed, and columns of one
    buffer that do not are told apart."""
    csrc = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "faie2-flashnext_b200", "csrc")
    (tmp_path / "meet.cpp").write_text("""
#include <random>
#include <set>
#include "fn_rows.h"
int main() {
    std::mt19937 g(1);
    auto in = [&](int lo, int hi) { return (int64_t)(lo + (int)(g() % (unsigned)(hi - lo + 1))); };
    int told = 0;
    for (int i = 0; i < 200000; ++i) {
        const int64_t rows = in(1, 4), nh = in(1, 3), hd = in(1, 4), ah = hd, bh = in(0, 3) ? hd + in(0, 3) : 2 * hd;
        const int64_t wide = (nh - 1) * bh + hd, at = in(0, 2) ? wide + in(0, 12) : in(0, 20), bt = in(0, 1) ? at : in(0, 20);
        const int64_t a = 1000 + in(-60, 60), b = 1000;
        std::set<int64_t> s;
        bool meet = false;
        for (int r = 0; r < rows; ++r)
            for (int h = 0; h < nh; ++h)
                for (int d = 0; d < hd; ++d) s.insert(b + r * bt + h * bh + d);
        for (int r = 0; r < rows; ++r)
            for (int h = 0; h < nh; ++h)
                for (int d = 0; d < hd; ++d) meet |= s.count(a + r * at + h * ah + d) != 0;
        const bool said = fn::kv4_rows_meet((void *)(a * 4), at, ah, (void *)(b * 4), bt, bh, rows, nh, hd, 4);
        if (meet && !said) return 1;
        told += !said && a - b < (rows - 1) * bt && b - a < (rows - 1) * at;  // within one another's rows
    }
    return told > 1000 ? 0 : 2;
}
""")
    subprocess.run(["g++", "-std=c++20", "-O1", "-I", csrc, str(tmp_path / "meet.cpp"), "-o", str(tmp_path / "meet")], check=True)
    assert subprocess.run([str(tmp_path / "meet")]).returncode == 0
