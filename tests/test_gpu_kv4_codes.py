"""GPU: stored bytes where the quantiser's offset lies far outside the codes' range: groups of one value, whose scale is the
least there is, and groups whose spread is small beside their values."""
import numpy as np
import pytest

from test_gpu_kv4 import Setup, dtype_of, torch  # noqa: F401 (a fixture)

pytestmark = pytest.mark.gpu


def stored(torch, xtg, k, dtype):  # noqa: F811
    """Whether rows k [rows][64] give the definition's bytes as keys, and their negatives as values."""
    s = Setup(torch, xtg, 40, [len(k)], [0], 1, 64)
    k = torch.from_numpy(k.astype(np.float32)[:, None]).cuda().to(dtype_of(torch, dtype))
    v = (-k.flip(0)).contiguous()
    s.ref.store(k.float().cpu().numpy(), v.float().cpu().numpy(), s.table, s.pos, s.cu)
    xtg.kv4_store(s.pool, k, v, *s.where)
    torch.cuda.synchronize()
    return s.same_pool()


def test_groups_of_one_small_value(cuda, xtg, torch):  # noqa: F811
    """x - z, up to 2^-8 |x|, is 2^13 to 2^40 times the least scale, 2^-100: past every integer that f32 holds exactly."""
    x = [2.0 ** -67 * (1 + 0.75 * 2.0 ** -7), -(2.0 ** -67) * (1 + 0.25 * 2.0 ** -7)]
    rng = np.random.default_rng(41)
    x += [sign * 2.0 ** e * (1 + rng.random()) for e in range(-82, -50) for sign in (1, -1) for _ in range(16)]
    assert stored(torch, xtg, np.repeat(np.array(x)[:, None], 64, 1), "f32")


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_groups_far_from_zero(cuda, xtg, torch, dtype):  # noqa: F811
    """Values within 2^0 .. 2^-23 of a common one: the offset's rounding cuts codes off at either end."""
    rng = np.random.default_rng(42)
    base = np.exp2(rng.uniform(-6, 6, (600, 1))) * rng.choice([-1, 1], (600, 1))
    x = base * (1 + np.exp2(rng.uniform(-23, 0, (600, 1))) * rng.uniform(-1, 1, (600, 64)))
    assert stored(torch, xtg, x, dtype)
