"""GPU: attention over a cache of latent vectors (the absorbed form) against the definition in 64 bits, and against the expanded
form of the same model."""
import math

import pytest
import torch

import kv16_ref as R
from kv16_cases import BF16, F16, check, ints, normal, tables

pytestmark = pytest.mark.gpu


def reference(q, q_rot, pool, where, scale, window=0):
    k_pool = pool[:, None]
    return R.attention(torch.cat([q, q_rot], -1), k_pool, k_pool[..., :q.shape[2]], *where, scale, window)


def compare(xtg, q, q_rot, pool, where, scale, window=0, **kw):
    got = xtg.latent_attention(q, q_rot, pool, *where, scale=scale, window=window, **kw)
    ref = reference(q, q_rot, pool, where, scale, window)
    n = int(where[2][-1])
    longest = int((where[1] + where[2].diff()).max())
    tol = R.tolerance(ref, q.dtype, pool.shape[2], longest)
    check(got[:n], ref[0][:n], tol[:n])
    return got, ref[0]


@pytest.mark.parametrize("latent,heads", [(512, 1), (512, 16), (512, 128), (256, 40), (256, 64), (512, 300)])
@pytest.mark.parametrize("dtype,page", [(BF16, 64), (F16, 16), (BF16, 32), (F16, 128)])
@pytest.mark.parametrize("rows,pos,window", [
    ([1], [0], 0), ([1, 1, 1], [4000, 62, 64], 0), ([4, 0, 2], [900, 7, 0], 0), ([20, 3], [100, 1000], 50)])
def test_attention(xtg, cuda, latent, heads, dtype, page, rows, pos, window):
    gen = torch.Generator(device="cuda").manual_seed(heads + len(rows))
    table, p, cu, pages = tables(gen, rows, pos, page)
    pool = normal(gen, pages, page, latent + 64, dtype=dtype)
    n = sum(rows)
    q, q_rot = normal(gen, n, heads, latent, dtype=dtype), normal(gen, n, heads, 64, dtype=dtype)
    compare(xtg, q, q_rot, pool, (table, p, cu), 2 / math.sqrt(latent + 64), window)


def test_views(xtg, cuda):
    # q as a batched product leaves it (heads first), the rotated dims behind others, a pool within a wider one
    gen = torch.Generator(device="cuda").manual_seed(1)
    table, p, cu, pages = tables(gen, [1, 3], [300, 40], 64)
    q = normal(gen, 32, 4, 512, dtype=BF16).transpose(0, 1)
    q_rot = normal(gen, 4, 32, 192, dtype=BF16)[..., 128:]
    pool = normal(gen, pages, 64, 640, dtype=BF16)[..., :576]
    compare(xtg, q, q_rot, pool, (table, p, cu), 0.05)


def test_what_a_row_does_not_see_and_what_is_not_finite(xtg, cuda):
    gen = torch.Generator(device="cuda").manual_seed(2)
    for latent, heads in ((512, 16), (256, 24)):
        rows, pos = [6, 1], [250, 77]
        table, p, cu, pages = tables(gen, rows, pos, 64, spare=2, slack=1)
        pool = normal(gen, pages, 64, latent + 64, dtype=F16)
        seen = torch.zeros(pages, 64, dtype=torch.bool)
        for i, a, n, p0 in R.sequences(table, p, cu):
            for x, pg, sl in R.places(table, i, 0, p0 + n, 64, pages):
                seen[pg, sl] = True
        pool.masked_fill_(~seen.cuda()[..., None], math.nan)
        q, q_rot = normal(gen, 7, heads, latent, dtype=F16), normal(gen, 7, heads, 64, dtype=F16)
        got, _ = compare(xtg, q, q_rot, pool, (table, p, cu), 0.05)
        assert got.isfinite().all()
        at = R.places(table, 0, 253, 1, 64, pages)[0]
        pool[at[1], at[2]] = math.nan   # position 253: the rows from there on
        got = xtg.latent_attention(q, q_rot, pool, table, p, cu, scale=0.05)
        assert got[:3].isfinite().all() and got[3:6].isnan().all() and got[6:].isfinite().all()


def test_rows_that_see_nothing(xtg, cuda):
    gen = torch.Generator(device="cuda").manual_seed(3)
    pool = normal(gen, 3, 16, 576, dtype=BF16)
    where = (ints([[0, 1], [-1, -1]]), ints([-2, 20]), ints([0, 5, 6]))
    q, q_rot = normal(gen, 8, 100, 512, dtype=BF16), normal(gen, 8, 100, 64, dtype=BF16)
    got, _ = compare(xtg, q, q_rot, pool, where, 0.05)
    assert not got[:2].any() and got[2:5].any() and not got[5:].any()


def test_waits_that_give_up(xtg, cuda):
    gen = torch.Generator(device="cuda").manual_seed(4)
    table, p, cu, pages = tables(gen, [1, 2], [900, 30], 64)
    pool = normal(gen, pages, 64, 576, dtype=BF16)
    q, q_rot = normal(gen, 3, 128, 512, dtype=BF16), normal(gen, 3, 128, 64, dtype=BF16)
    err = ints([0])
    before = xtg.lib().xtg_cuda_kv16_wait_polls(0)
    try:
        got = xtg.latent_attention(q, q_rot, pool, table, p, cu, scale=0.05, err=err)
        torch.cuda.synchronize()
    finally:
        xtg.lib().xtg_cuda_kv16_wait_polls(before)
    with pytest.raises(xtg.XtgError, match="timed out"):
        xtg.kv4_check(err)
    assert got.isnan().all()
    compare(xtg, q, q_rot, pool, (table, p, cu), 0.05)


@pytest.mark.parametrize("interleaved", [False, True])
def test_expanded_and_absorbed_forms_agree(xtg, cuda, interleaved):
    """A conversation of a latent model's layer: a prompt in the expanded form (keys and values of every head made from the
    latent vectors), then tokens one by one in the absorbed form over the latent cache; every output against plain
    arithmetic in 64 bits from the layer's inputs."""
    gen = torch.Generator(device="cuda").manual_seed(5)
    heads, latent, nope, rot, dv, page = 4, 512, 128, 64, 128, 64
    prompt, steps = 150, 5
    n = prompt + steps
    w_k = normal(gen, heads, nope, latent, dtype=BF16) / math.sqrt(latent)
    w_v = normal(gen, heads, dv, latent, dtype=BF16) / math.sqrt(latent)
    c, k_rot = normal(gen, n, latent, dtype=BF16), normal(gen, n, rot, dtype=BF16)
    q = normal(gen, n, heads, nope + rot, dtype=BF16)
    freq = (10000.0 ** (-torch.arange(rot // 2, dtype=torch.float64) / (rot // 2))).float().cuda()
    scale = 1 / math.sqrt(nope + rot)
    at = torch.arange(n, device="cuda")
    # 64 bits
    k = torch.cat([torch.einsum("pl,hdl->phd", c.double(), w_k.double()),
                   R.rotate(k_rot[:, None], at, freq, interleaved).expand(n, heads, rot)], -1)
    v = torch.einsum("pl,hdl->phd", c.double(), w_v.double())
    x = torch.cat([q[..., :nope].double(), R.rotate(q[..., nope:], at, freq, interleaved)], -1)
    s = (torch.einsum("nhd,phd->hnp", x, k) * scale).masked_fill(at[None] > at[:, None], -math.inf)
    prob = torch.softmax(s, -1)
    want = torch.einsum("hnp,phd->nhd", prob, v)
    mass = torch.einsum("hnp,phd->nhd", prob, v.abs())
    # Half a step (2^-8) of each bf16 operand: keys and queries move the scores by 2 x 2^-8 of scale |q| |k|, the absorbed
    # query by as much again, at most 3 x 2^-8 of sqrt(nope + rot) x 4 for normal values: 0.65 of the mass's spread
    # would be the worst; the roundings are independent, so their sum grows with the root of the dims, which divides it by
    # about 8. Weights and values 3 x 2^-8, the projection's input and output 2 x 2^-8.
    tol = mass * (0.65 / 8 + 5 * 2.0 ** -8) + 2.0 ** -8 * want.abs()
    one = ints([0, 1])
    # the prompt, expanded
    table, p, cu, pages = tables(gen, [prompt], [0], page)
    pools = [xtg.kv16_pool(pages, heads, d, page=page) for d in (nope + rot, dv)]
    keys = torch.cat([torch.einsum("pl,hdl->phd", c[:prompt], w_k), k_rot[:prompt, None].expand(prompt, heads, rot)], -1)
    values = torch.einsum("pl,hdl->phd", c[:prompt], w_v)
    turned = xtg.kv16_append(*pools, keys, values, table, p, cu, freq=freq, q=q[:prompt], first=nope, interleaved=interleaved)
    check(xtg.kv16_attention(turned, *pools, table, p, cu, scale=scale), want[:prompt], tol[:prompt], "expanded")
    # the same prompt into the latent cache, then the steps
    table, p, cu, pages = tables(gen, [n], [0], page)
    pool = xtg.latent_pool(pages, latent, page=page)
    xtg.latent_append(pool, c[:prompt], k_rot[:prompt], table, p, ints([0, prompt]), freq=freq, interleaved=interleaved)
    for i in range(prompt, n):
        pos = ints([i])
        row = slice(i, i + 1)
        q_rot = xtg.latent_append(pool, c[row], k_rot[row], table, pos, one, freq=freq, q=q[row, :, nope:],
                                  interleaved=interleaved)
        absorbed = torch.einsum("nhd,hdl->nhl", q[row, :, :nope], w_k)
        o = xtg.latent_attention(absorbed, q_rot, pool, table, pos, one, scale=scale)
        check(torch.einsum("nhl,hdl->nhd", o, w_v), want[row], tol[row], f"absorbed, position {i}")


def test_refusals(xtg, cuda):
    pool = torch.zeros(2, 16, 576, dtype=BF16, device="cuda")
    where = (ints([[0]]), ints([0]), ints([0, 1]))
    q, r = (torch.zeros(1, 4, d, dtype=BF16, device="cuda") for d in (512, 64))

    def refused(match, q=q, r=r, pool=pool, **kw):
        with pytest.raises(xtg.XtgError, match=match):
            xtg.latent_attention(q, r, pool, *where, scale=1.0, **kw)
    refused("type", q=q.float())
    refused("type", r=r.to(F16))
    refused(r"\[rows\]\[heads\]", r=r[:, :3])
    refused(r"\[rows\]\[heads\]", q=torch.zeros(1, 4, 576, dtype=BF16, device="cuda"))
    refused("tensor", r=None)
    refused("pool", pool=pool[:, None])
    refused("head_dim", pool=torch.zeros(2, 16, 448, dtype=BF16, device="cuda"), q=torch.zeros(1, 4, 384, dtype=BF16, device="cuda"))
    c, k = torch.zeros(1, 512, device="cuda"), torch.zeros(1, 64, device="cuda")
    for bad in (dict(c=c[:, :256]), dict(k=c), dict(c=c.to(BF16)), dict(freq=torch.zeros(64, device="cuda"))):
        with pytest.raises(xtg.XtgError):
            xtg.latent_append(pool, **{**dict(c=c, k=k), **bad}, table=where[0], pos=where[1], cu_rows=where[2])
