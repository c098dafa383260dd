"""GPU: attention over the 16-bit caches against the definition in 64 bits (tolerances: kv16_ref.tolerance)."""
import math

import pytest
import torch

import kv16_ref as R
from kv16_cases import BF16, F16, check, ints, normal, pools, tables

pytestmark = pytest.mark.gpu


def compare(xtg, q, k_pool, v_pool, where, scale, window=0, what="", **kw):
    got = xtg.kv16_attention(q, k_pool, v_pool, *where, scale=scale, window=window, **kw)
    ref = R.attention(q, k_pool, v_pool, *where, scale, window)
    longest = int((where[1] + where[2].diff()).max())
    n = int(where[2][-1])
    tol = R.tolerance(ref, q.dtype, q.shape[2], longest)
    check(got[:n], ref[0][:n], tol[:n], what)
    return got, ref[0]


SHAPES = [(24, 6, 128, 128), (16, 4, 256, 256), (8, 8, 64, 64), (12, 1, 128, 128), (4, 4, 192, 128), (3, 1, 64, 64)]


@pytest.mark.parametrize("heads,kvh,d,dv", SHAPES)
@pytest.mark.parametrize("dtype,page", [(BF16, 64), (F16, 16), (BF16, 128), (F16, 1024)])
@pytest.mark.parametrize("rows,pos,window", [
    ([1], [0], 0), ([1], [4095], 0), ([1, 1, 1], [63, 64, 700], 0), ([8, 8], [1000, 3], 100), ([3, 0, 5, 1], [0, 9, 126, 640], 0),
    ([130, 70], [0, 333], 0), ([200], [50], 17), ([40, 1], [500, 40], 1)])
def test_attention(xtg, cuda, heads, kvh, d, dv, dtype, page, rows, pos, window):
    gen = torch.Generator(device="cuda").manual_seed(sum(rows) + d)
    table, p, cu, pages = tables(gen, rows, pos, page)
    k_pool, v_pool = pools(gen, pages, kvh, page, d, dv, dtype, "nhd" if heads == 24 else "hnd")
    q = normal(gen, sum(rows), heads, d, dtype=dtype)
    compare(xtg, q, k_pool, v_pool, (table, p, cu), 1.5 / math.sqrt(d), window)


@pytest.mark.parametrize("hint", [1, 2, 9, 40, 1000])
def test_any_hint_gives_the_result(xtg, cuda, hint):
    gen = torch.Generator(device="cuda").manual_seed(5)
    table, p, cu, pages = tables(gen, [1, 30, 7, 0, 90], [2000, 0, 500, 3, 1111], 64)
    k_pool, v_pool = pools(gen, pages, 2, 64, 128, 128, BF16)
    q = normal(gen, 128, 8, 128, dtype=BF16)
    compare(xtg, q, k_pool, v_pool, (table, p, cu), 0.1, 0, rows_per_seq=hint)
    compare(xtg, q, k_pool, v_pool, (table, p, cu), 0.1, 333, rows_per_seq=hint)


@pytest.mark.parametrize("seqs", [100, 700])
def test_many_sequences(xtg, cuda, seqs):
    # more than the copies' warp plans alone, of every length, some without rows, some of pages that are not there
    gen = torch.Generator(device="cuda").manual_seed(seqs)
    rows = [(7 * i) % 4 for i in range(seqs)]
    pos = [(97 * i) % 900 for i in range(seqs)]
    table, p, cu, pages = tables(gen, rows, pos, 64)
    table[::5, 0] = -1
    k_pool, v_pool = pools(gen, pages, 2, 64, 64, 64, F16)
    q = normal(gen, sum(rows), 4, 64, dtype=F16)
    compare(xtg, q, k_pool, v_pool, (table, p, cu), 0.2)


def test_long_sequences_of_one_sign(xtg, cuda):
    # every value and weight adds to the sums with the same sign: a loss of the last bit a step would show
    gen = torch.Generator(device="cuda").manual_seed(7)
    for dtype in (F16, BF16):
        table, p, cu, pages = tables(gen, [1, 1], [131071, 20000], 64)
        k_pool, v_pool = pools(gen, pages, 1, 64, 64, 64, dtype)
        k_pool.mul_(0.05)
        v_pool.abs_().add_(1)
        q = normal(gen, 2, 4, 64, dtype=dtype)
        compare(xtg, q, k_pool, v_pool, (table, p, cu), 0.05)


def test_scores_that_rise_and_fall(xtg, cuda):
    # the reference has to move late, by a little and by a lot, and must not where scores fall
    gen = torch.Generator(device="cuda").manual_seed(8)
    for dtype in (F16, BF16):
        for slope in (30.0, -30.0, 2000.0):
            table, p, cu, pages = tables(gen, [1, 9], [3000, 1500], 64)
            k_pool, v_pool = pools(gen, pages, 1, 64, 128, 128, dtype)
            for i in range(2):
                n = int(p[i]) + 9
                for x, pg, sl in R.places(table, i, 0, -(-n // 64) * 64, 64, pages):
                    k_pool[pg, 0, sl, 0] = slope * x / 3000
            q = normal(gen, 10, 3, 128, dtype=dtype)
            q[..., 0] = 1
            compare(xtg, q, k_pool, v_pool, (table, p, cu), 1.0, what=str(slope))


def test_what_a_row_does_not_see(xtg, cuda):
    # everything past the lengths, below the window and on pages in no table is NaN or infinite
    gen = torch.Generator(device="cuda").manual_seed(9)
    for heads, kvh, d, dv in SHAPES:
        for window in (0, 100):
            for page in (16, 64, 256):
                rows, pos = [1, 8, 33], [300, 700, 0]
                table, p, cu, pages = tables(gen, rows, pos, page, spare=3, slack=2)
                k_pool, v_pool = pools(gen, pages, kvh, page, d, dv, BF16)
                seen = torch.zeros(pages, page, dtype=torch.bool)
                for i, a, n, p0 in R.sequences(table, p, cu):
                    for x, pg, sl in R.places(table, i, 0, p0 + n, page, pages):
                        if window == 0 or x > p0 - window:
                            seen[pg, sl] = True
                hidden = ~seen.cuda()[:, None, :, None]
                k_pool.masked_fill_(hidden, math.nan)
                v_pool.masked_fill_(hidden, math.inf)
                q = normal(gen, sum(rows), heads, d, dtype=BF16)
                got, want = compare(xtg, q, k_pool, v_pool, (table, p, cu), 0.1, window)
                assert got.isfinite().all()


@pytest.mark.parametrize("heads,kvh,d,dv", SHAPES)
@pytest.mark.parametrize("window", [0, 5, 200])
def test_values_that_are_not_finite(xtg, cuda, heads, kvh, d, dv, window):
    # at positions that some rows of a block see: those alone get them; others keep their numbers
    gen = torch.Generator(device="cuda").manual_seed(10)
    rows, pos = [40, 6], [250, 126]
    table, p, cu, pages = tables(gen, rows, pos, 64)
    k_pool, v_pool = pools(gen, pages, kvh, 64, d, dv, F16)
    for x, value, dim in ((260, math.nan, 3), (277, math.inf, 5), (289, -math.inf, dv - 1), (255, math.inf, 17), (252, -math.inf, 17),
                          (100, math.inf, 40)):
        at = R.places(table, 0, x, 1, 64, pages)[0]
        v_pool[at[1], :, at[2], dim] = value
    at = R.places(table, 1, 129, 1, 64, pages)[0]
    v_pool[at[1], :, at[2]] = math.nan
    q = normal(gen, sum(rows), heads, d, dtype=F16)
    got, want = compare(xtg, q, k_pool, v_pool, (table, p, cu), 0.1, window)
    assert torch.equal(got[:len(want)].isfinite(), want.isfinite())
    # a key that is not finite makes its rows NaN and no other
    at = R.places(table, 0, 280, 1, 64, pages)[0]
    v_pool = torch.nan_to_num(v_pool, nan=0, posinf=0, neginf=0)
    k_pool[at[1], :, at[2], 1] = math.nan
    got = xtg.kv16_attention(q, k_pool, v_pool, table, p, cu, scale=0.1, window=window)
    t = torch.arange(250, 290, device="cuda")
    hit = (t >= 280) & ((t - 280 < window) if window else True)
    assert got[:40][hit].isnan().all() and got[:40][~hit].isfinite().all() and got[40:].isfinite().all()


def test_rows_that_see_nothing(xtg, cuda):
    gen = torch.Generator(device="cuda").manual_seed(11)
    # before position 0; on a page that is not there; a window whose pages were given back; an empty table beside a full one
    rows, pos, page = [5, 2, 3, 20], [-3, 10, 200, -7], 16
    table = ints([[0] + [-1] * 13, [-1] * 14, [1, 2, 3] + [-1] * 11, [4] + [-1] * 13])
    p, cu = ints(pos), ints([0, 5, 7, 10, 30])
    for heads, kvh, d, dv in SHAPES:
        k_pool, v_pool = pools(gen, 6, kvh, page, d, dv, F16)
        q = normal(gen, 30, heads, d, dtype=F16)
        got, _ = compare(xtg, q, k_pool, v_pool, (table, p, cu), 0.1, 100)
        assert not got[:3].any() and not got[5:10].any() and not got[10:17].any()
        assert got[3:5].any() and got[17:].any()


def test_a_page_that_is_not_there_in_between(xtg, cuda):
    gen = torch.Generator(device="cuda").manual_seed(12)
    for page in (16, 64, 256):
        table, p, cu, pages = tables(gen, [2, 50], [1500, 900], page)
        table[0, 1], table[0, 3], table[1, 2] = -1, -1, -1
        k_pool, v_pool = pools(gen, pages, 2, page, 256, 256, BF16)
        q = normal(gen, 52, 4, 256, dtype=BF16)
        compare(xtg, q, k_pool, v_pool, (table, p, cu), 0.1)


def test_positions_past_the_table_and_pages_past_the_pool(xtg, cuda):
    gen = torch.Generator(device="cuda").manual_seed(13)
    table, p, cu, pages = tables(gen, [4, 1], [126, 300], 64)
    k_pool, v_pool = pools(gen, pages, 2, 64, 128, 128, BF16)
    q = normal(gen, 5, 4, 128, dtype=BF16)
    err = ints([0])
    bad = table.clone()
    bad[1, 2] = pages
    got = xtg.kv16_attention(q, k_pool, v_pool, bad, p, cu, scale=0.1, err=err)
    with pytest.raises(xtg.XtgError, match="past the pool"):
        xtg.kv4_check(err)
    ref = R.attention(q, k_pool, v_pool, bad, p, cu, 0.1)
    check(got, ref[0], R.tolerance(ref, BF16, 128, 301))
    short = table[:, :2].contiguous()   # positions from 128 on lie past it
    got = xtg.kv16_attention(q, k_pool, v_pool, short, p, cu, scale=0.1, err=err)
    with pytest.raises(xtg.XtgError, match="page table"):
        xtg.kv4_check(err)
    ref = R.attention(q, k_pool, v_pool, short, p, cu, 0.1)
    check(got, ref[0], R.tolerance(ref, BF16, 128, 301))
    xtg.kv16_attention(q, k_pool, v_pool, table, p, cu, scale=0.1, err=err)
    xtg.kv4_check(err)


def test_rows_of_no_sequence(xtg, cuda):
    gen = torch.Generator(device="cuda").manual_seed(14)
    table, p, cu, pages = tables(gen, [3, 2], [70, 10], 64)
    k_pool, v_pool = pools(gen, pages, 2, 64, 64, 64, BF16)
    q = normal(gen, 9, 4, 64, dtype=BF16)
    got, _ = compare(xtg, q, k_pool, v_pool, (table, p, cu), 0.1)
    assert not got[5:].any()
    out = torch.full_like(q, 3.0)
    assert xtg.kv16_attention(q, k_pool, v_pool, table, p, cu, scale=0.1, out=out).data_ptr() == out.data_ptr()
    assert torch.equal(out[:5], got[:5]) and (out[5:] == 3).all()
    none = xtg.kv16_attention(q, k_pool, v_pool, table[:0], p[:0], cu[:1], scale=0.1)
    assert not none.any()
    assert xtg.kv16_attention(q[:0], k_pool, v_pool, table, p, ints([0, 0, 0]), scale=0.1).shape == (0, 4, 64)


def test_views_of_queries_and_pools(xtg, cuda):
    gen = torch.Generator(device="cuda").manual_seed(15)
    table, p, cu, pages = tables(gen, [3, 20], [700, 0], 32)
    wide = normal(gen, pages, 32, 3, 2, 128, dtype=F16)   # keys, values and something else of a page side by side
    k_pool, v_pool = wide[:, :, 0].transpose(1, 2), wide[:, :, 2].transpose(1, 2)
    fused = normal(gen, 23, 10 * 128, dtype=F16)
    q = fused[:, 128:128 + 8 * 128].view(23, 8, 128)
    compare(xtg, q, k_pool, v_pool, (table, p, cu), 0.1)
    q = normal(gen, 8, 23, 128, dtype=F16).transpose(0, 1)
    compare(xtg, q, k_pool, v_pool, (table, p, cu), 0.1)
    one = normal(gen, 1, 1, 16, 64, dtype=BF16)   # strides of what there is one of are any
    q = normal(gen, 1, 1, 64, dtype=BF16)
    compare(xtg, q.as_strided((1, 1, 64), (3, 5, 1)), one.as_strided((1, 1, 16, 64), (7, 3, 64, 1)), one,
            (ints([[0]]), ints([9]), ints([0, 1])), 0.1)


def test_offsets_past_32_bits(xtg, cuda):
    # a pool of more than 2^32 values: its last pages, which are written and read alone
    pages = (1 << 32) // (4 * 64 * 256) + 40
    k_pool = torch.empty(pages, 4, 64, 256, dtype=F16, device="cuda")
    gen = torch.Generator(device="cuda").manual_seed(16)
    table = ints([list(range(pages - 1, pages - 21, -1))])
    k_pool[-20:] = normal(gen, 20, 4, 64, 256, dtype=F16)
    q = normal(gen, 1, 16, 256, dtype=F16)
    where = (table, ints([1200]), ints([0, 1]))
    small = (torch.arange(19, -1, -1, dtype=torch.int32, device="cuda")[None], *where[1:])
    row = normal(gen, 1, 4, 256, dtype=F16)
    xtg.kv16_append(k_pool, k_pool, row, row, *where)
    got = xtg.kv16_attention(q, k_pool, k_pool, *where, scale=0.1)
    tail = k_pool[-20:].clone()
    del k_pool
    assert torch.equal(tail[19 - 1200 // 64, :, 1200 % 64], row[0])
    ref = R.attention(q, tail, tail, *small, 0.1)
    check(got, ref[0], R.tolerance(ref, F16, 256, 1201))


def test_streams_and_captured_calls(xtg, cuda):
    gen = torch.Generator(device="cuda").manual_seed(17)
    table, p, cu, pages = tables(gen, [1, 1, 1], [900, 30, 2000], 64, slack=1)
    k_pool, v_pool = pools(gen, pages, 2, 64, 128, 128, BF16)
    q = normal(gen, 3, 8, 128, dtype=BF16)
    args = (q, k_pool, v_pool, table, p, cu)
    want = xtg.kv16_attention(*args, scale=0.1)
    torch.cuda.synchronize()
    outs, streams = [], [torch.cuda.Stream() for _ in range(3)]
    for s in streams * 5:   # at once, each with a workspace of its own
        with torch.cuda.stream(s):
            outs.append(xtg.kv16_attention(*args, scale=0.1))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)   # and the same bits every time
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = xtg.kv16_attention(*args, scale=0.1)
    for n in ([900, 30, 2000], [5, 1700, 0], [64, 63, 65]):
        p.copy_(ints(n))
        g.replay()
        ref = R.attention(q, k_pool, v_pool, table, p, cu, 0.1)   # some pages are not there
        check(out, ref[0], R.tolerance(ref, BF16, 128, 2001))


def test_waits_that_give_up(xtg, cuda):
    gen = torch.Generator(device="cuda").manual_seed(18)
    table, p, cu, pages = tables(gen, [1, 20, 3], [900, 30, -9], 64)
    L = xtg.lib()
    for heads, kvh, d, dv in SHAPES[:4]:
        k_pool, v_pool = pools(gen, pages, kvh, 64, d, dv, BF16)
        q = normal(gen, 24, heads, d, dtype=BF16)
        err = ints([0])
        before = L.xtg_cuda_kv16_wait_polls(0)
        try:
            got = xtg.kv16_attention(q, k_pool, v_pool, table, p, cu, scale=0.1, err=err)
            torch.cuda.synchronize()
        finally:
            L.xtg_cuda_kv16_wait_polls(before)
        with pytest.raises(xtg.XtgError, match="timed out"):
            xtg.kv4_check(err)
        assert got[:21].isnan().all()
        compare(xtg, q, k_pool, v_pool, (table, p, cu), 0.1)


def test_refusals(xtg, cuda):
    k_pool = torch.zeros(2, 2, 16, 64, dtype=BF16, device="cuda")
    where = (ints([[0]]), ints([0]), ints([0, 1]))
    q = torch.zeros(1, 4, 64, dtype=BF16, device="cuda")

    def refused(match, q=q, k=k_pool, v=k_pool, where=where, scale=1.0, **kw):
        with pytest.raises(xtg.XtgError, match=match):
            xtg.kv16_attention(q, k, v, *where, scale=scale, **kw)
    refused("type", q=q.float())
    refused("type", q=q.to(F16))
    refused(r"\[rows\]\[heads\]", q=torch.zeros(1, 4, 128, dtype=BF16, device="cuda"))
    refused("multiple", q=q[:, :3])
    refused("scale", scale=float("nan"))
    refused("scale", scale="x")
    refused("window", window=-1)
    refused("rows_per_seq", rows_per_seq=0)
    refused("out", out=torch.zeros(1, 4, 64, device="cuda"))
    refused("table", where=(where[0].long(), *where[1:]))
    refused("seqs", where=(where[0], ints([0, 1]), where[2]))
    refused("v_pool", v=k_pool[:1])
    refused("head_dim", k=torch.zeros(2, 2, 16, 96, dtype=BF16, device="cuda"), v=torch.zeros(2, 2, 16, 96, dtype=BF16, device="cuda"),
            q=torch.zeros(1, 4, 96, dtype=BF16, device="cuda"))
    refused("tensor", v=3)
