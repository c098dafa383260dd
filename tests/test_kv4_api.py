"""CPU: settings of the 4-bit cache's entry points that need no device."""


def test_wait_polls(xtg):
    f = xtg.lib().xtg_cuda_kv4_wait_polls
    default = f(-1)
    assert default * 4e-6 < 2   # seconds: a look takes 4 us
    try:
        assert f(100) == default and f(-5) == 100 and f(0) == 100
        assert f(2 ** 31 - 1) == 0 and f(-1) == 1 << 24   # the most
    finally:
        f(default)
