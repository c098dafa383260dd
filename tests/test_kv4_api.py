"""CPU: settings of the 4-bit cache's entry points that need no device."""


def test_wait_polls(xtg):
    f = xtg.lib().xtg_cuda_kv4_wait_polls
    assert f(-1) == 1 << 24
    try:
        assert f(100) == 1 << 24 and f(-5) == 100 and f(0) == 100
        assert f(2 ** 31 - 1) == 0 and f(-1) == 1 << 24   # the default is the most
    finally:
        f(1 << 24)
