"""GPU: values of the 16-bit caches that are not finite, where scores lie so far apart that weights round to zero: each makes its
dim of the rows that see it not finite and nothing else, whatever the tiling; and what carries no gradient."""
import math

import pytest
import torch

import kv16_ref as R
from kv16_cases import BF16, F16, check, ints, normal, pools, tables

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("heads,kvh,d,dv", [(24, 6, 128, 128), (16, 4, 256, 256), (8, 8, 64, 64), (4, 4, 192, 128)])
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("hint", [1, 5, 14, 1000])
def test_values_that_are_not_finite_under_small_weights(xtg, cuda, heads, kvh, d, dv, dtype, hint):
    gen = torch.Generator(device="cuda").manual_seed(d + hint)
    rows, pos = [40, 6, 1], [2500, 126, 3000]
    table, p, cu, pages = tables(gen, rows, pos, 64)
    k_pool, v_pool = pools(gen, pages, kvh, 64, d, dv, dtype)
    # positions that all rows of a sequence see, and that some see
    for i, x, value, dim in ((0, 100, math.inf, 3), (0, 1700, math.nan, 5), (0, 2499, -math.inf, dv - 1), (0, 2520, math.inf, 17),
                             (0, 2539, math.nan, 18), (1, 64, -math.inf, 1), (1, 129, math.inf, 2), (2, 2900, math.inf, 9),
                             (2, 40, math.nan, 10)):
        at = R.places(table, i, x, 1, 64, pages)[0]
        v_pool[at[1], :, at[2], dim] = value
    q = normal(gen, sum(rows), heads, d, dtype=dtype)
    scale = 25 / math.sqrt(d)   # a row's scores are spread over 100 and more
    ref = R.attention(q, k_pool, v_pool, table, p, cu, scale)
    got = xtg.kv16_attention(q, k_pool, v_pool, table, p, cu, scale=scale, rows_per_seq=hint)
    assert torch.equal(got.isfinite(), ref[0].isfinite())
    fine = ref[0].isfinite()
    check(got[fine], ref[0][fine], R.tolerance(ref, dtype, d, 3001)[fine])


@pytest.mark.parametrize("hint", [1, 1000])
def test_latent_values_that_are_not_finite(xtg, cuda, hint):
    # a latent vector's value is its key too: the rows that see it are not finite, and no other
    gen = torch.Generator(device="cuda").manual_seed(hint)
    table, p, cu, pages = tables(gen, [6, 1], [700, 77], 64)
    pool = normal(gen, pages, 64, 576, dtype=F16)
    at = R.places(table, 0, 703, 1, 64, pages)[0]
    pool[at[1], at[2], 7] = math.inf
    q, q_rot = normal(gen, 7, 16, 512, dtype=F16), normal(gen, 7, 16, 64, dtype=F16)
    got = xtg.latent_attention(q, q_rot, pool, table, p, cu, scale=1.0, rows_per_seq=hint)
    assert got[:3].isfinite().all() and not got[3:6, :, 7].isfinite().any() and got[6:].isfinite().all()


def test_results_carry_no_gradient(xtg, cuda):
    gen = torch.Generator(device="cuda").manual_seed(1)
    k_pool, v_pool = xtg.kv16_pool(2, 1, 64), xtg.kv16_pool(2, 1, 64)
    where = (ints([[0]]), ints([0]), ints([0, 3]))
    q, k, v = (normal(gen, 3, n, 64, dtype=BF16).requires_grad_() for n in (2, 1, 1))
    turned = xtg.kv16_append(k_pool, v_pool, k, v, *where, q=q)
    out = xtg.kv16_attention(q, k_pool, v_pool, *where, scale=0.1)
    assert not (turned.requires_grad or k_pool.requires_grad or v_pool.requires_grad or out.requires_grad)
    assert torch.equal(out, xtg.kv16_attention(q.detach(), k_pool, v_pool, *where, scale=0.1))
