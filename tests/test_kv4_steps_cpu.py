"""CPU: refusals of the paged 4-bit cache's later entries and layers, before any device work."""

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
