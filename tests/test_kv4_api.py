"""CPU: settings of the 4-bit cache's entry points that need no device."""
import pytest

from test_kv4 import call

ZERO_REST = 256


def test_wait_polls(xtg):
    f = xtg.lib().xtg_cuda_kv4_wait_polls
    default = f(-1)
    assert default * 4e-6 < 2   # seconds: a look takes 4 us
    try:
        assert f(100) == default and f(-5) == 100 and f(0) == 100
        assert f(2 ** 31 - 1) == 0 and f(-1) == 1 << 24   # the most
    finally:
        f(default)


@pytest.mark.parametrize("entry,dtype", [("load", ZERO_REST + 3), ("attention", ZERO_REST + 7), ("load", 2 * ZERO_REST),
                                         ("store", ZERO_REST + 1), ("attention", -ZERO_REST)])
def test_the_flag_for_zeros_hides_no_bad_type(xtg, entry, dtype):
    rc, why = call(xtg, entry, dtype=dtype)
    assert rc == -1 and "f32" in why, why


@pytest.mark.parametrize("entry", ["load", "attention"])
def test_the_flag_for_zeros_with_no_rows(xtg, entry):
    assert call(xtg, entry, dict(rows=0), dtype=ZERO_REST + 1) == (0, "")
