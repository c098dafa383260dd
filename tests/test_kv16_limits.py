"""CPU: the largest calls of the 16-bit caches' append that are taken."""
import pytest

from test_kv16 import LATENT, call


@pytest.mark.parametrize("cache,rows", [
    ({}, dict(heads=1 << 27)),   # 16 units of 8 dims a head: past 2^31 of them
    ({}, dict(heads=(1 << 23) - 3)), (dict(kv_heads=65535), dict(heads=(1 << 23) - 2 * 65535 + 1)),
    (LATENT, dict(heads=(1 << 24) - 8, rotary=64, v_head=0)),
])
def test_a_row_of_too_many_values(xtg, cache, rows):
    rc, why = call(xtg, "append", cache, rows)
    assert rc == -1 and "2^30" in why, why


@pytest.mark.parametrize("cache,rows", [
    ({}, dict(heads=(1 << 23) - 4)), (dict(kv_heads=65535), dict(heads=(1 << 23) - 2 * 65535)),
    (LATENT, dict(heads=(1 << 24) - 9, rotary=64, v_head=0)),
])
def test_the_largest_row(xtg, cache, rows):
    # refused for what is checked next: pointers
    rc, why = call(xtg, "append", dict(cache, k_head=64 * 128), dict(rows, k=None))
    assert rc == -1 and "null" in why, why
