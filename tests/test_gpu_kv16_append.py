"""GPU: keys, values and queries appended to the 16-bit caches with their rotation, against the definition in 64 bits."""
import pytest
import torch

import kv16_ref as R
from kv16_cases import BF16, F16, F32, check, ints, normal, tables

pytestmark = pytest.mark.gpu


def freqs(m):
    return (10000.0 ** (-torch.arange(m, dtype=torch.float64) / m)).float().cuda()


def turned(x, pos, freq, first, interleaved):
    """x [rows][heads][d] with dims first .. turned, 64 bits, and how far f32 arithmetic may be off"""
    y = x.double().clone()
    r = 0 if freq is None else 2 * freq.numel()
    room = torch.zeros_like(y)
    if r:
        part = x[..., first:first + r]
        y[..., first:first + r] = R.rotate(part, pos, freq, interleaved)
        a = part.double().abs()
        m = r // 2
        both = (a[..., ::2] + a[..., 1::2]).repeat_interleave(2, -1) if interleaved else (a[..., :m] + a[..., m:]).repeat(1, 1, 2)
        # the half turns' last bit (pi 2^-25), sine and cosine's (2^-23), two products' and a sum's (3 x 2^-24)
        room[..., first:first + r] = both * 2.0 ** -21
    return y, room


def close(got, y, room, what):
    h = torch.finfo(got.dtype).eps / 2
    tiny = torch.finfo(got.dtype).tiny * torch.finfo(got.dtype).eps
    check(got, y, room + h * (y.abs() + room) + tiny, what)


@pytest.mark.parametrize("d,dv,heads,kvh,first,pairs", [
    (128, 128, 24, 6, 0, 64), (64, 64, 8, 8, 0, 32), (256, 256, 16, 4, 0, 128), (192, 128, 4, 4, 128, 32),
    (128, 128, 12, 1, 8, 24), (128, 128, 4, 2, 0, 0)])
@pytest.mark.parametrize("rows_dtype,dtype", [(F32, BF16), (BF16, BF16), (F16, F16), (F16, BF16), (F32, F16)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_append(xtg, cuda, d, dv, heads, kvh, first, pairs, rows_dtype, dtype, interleaved):
    gen = torch.Generator(device="cuda").manual_seed(d + heads)
    rows, pos, page = [3, 0, 70, 1], [1021, 5, 100000, 0], 16 if heads == 8 else 64
    table, p, cu, pages = tables(gen, rows, pos, page)
    n = sum(rows)
    freq = freqs(pairs) if pairs else None
    k_pool, v_pool = normal(gen, pages, kvh, page, d, dtype=dtype), normal(gen, pages, kvh, page, dv, dtype=dtype)
    k, v = normal(gen, n, kvh, d, dtype=rows_dtype), normal(gen, n, kvh, dv, dtype=rows_dtype)
    q = normal(gen, n, heads, d, dtype=rows_dtype)
    at = torch.cat([torch.arange(a, a + m) for m, a in zip(rows, pos)]).cuda()
    want_k, want_v = k_pool.double(), v_pool.double()
    room = torch.zeros_like(want_k)
    y, ry = turned(k, at, freq, first, interleaved)
    for i, a, m, p0 in R.sequences(table, p, cu):
        for j, (x, pg, sl) in enumerate(R.places(table, i, p0, m, page, pages)):
            want_k[pg, :, sl], room[pg, :, sl], want_v[pg, :, sl] = y[a + j], ry[a + j], v[a + j].double()
    got = xtg.kv16_append(k_pool, v_pool, k, v, table, p, cu, freq=freq, q=q, first=first, interleaved=interleaved)
    assert got.dtype == dtype and got.shape == q.shape
    close(got, *turned(q, at, freq, first, interleaved), "q")
    close(k_pool, want_k, room, "keys")
    close(v_pool, want_v, torch.zeros_like(want_v), "values")
    assert xtg.kv16_append(k_pool, v_pool, k, v, table, p, cu, freq=freq, first=first, interleaved=interleaved) is None


@pytest.mark.parametrize("latent,heads,rows_dtype,dtype", [(512, 32, F32, BF16), (256, 5, F16, F16), (512, 1, BF16, BF16)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_latent_append(xtg, cuda, latent, heads, rows_dtype, dtype, interleaved):
    gen = torch.Generator(device="cuda").manual_seed(latent + heads)
    rows, pos, page = [2, 33, 1], [0, 4093, 70], 32
    table, p, cu, pages = tables(gen, rows, pos, page)
    n, freq = sum(rows), freqs(32)
    pool = normal(gen, pages, page, latent + 64, dtype=dtype)
    both = normal(gen, n, latent + 64, dtype=rows_dtype)   # one projection's output, taken apart by views
    c, k = both[:, :latent], both[:, latent:]
    q = normal(gen, n, heads, 192, dtype=rows_dtype)[..., 128:]
    at = torch.cat([torch.arange(a, a + m) for m, a in zip(rows, pos)]).cuda()
    want, room = pool.double(), torch.zeros(pool.shape, dtype=torch.float64, device="cuda")
    y, ry = turned(k[:, None], at, freq, 0, interleaved)
    for i, a, m, p0 in R.sequences(table, p, cu):
        for j, (x, pg, sl) in enumerate(R.places(table, i, p0, m, page, pages)):
            want[pg, sl] = torch.cat([c[a + j].double(), y[a + j, 0]])
            room[pg, sl, latent:] = ry[a + j, 0]
    got = xtg.latent_append(pool, c, k, table, p, cu, freq=freq, q=q, interleaved=interleaved)
    close(got, *turned(q, at, freq, 0, interleaved), "q")
    close(pool, want, room, "pool")


def test_far_positions_keep_their_angles(xtg, cuda):
    # one radian a position: in 32 bits position 2^24 + 1 has no angle of its own
    pos = [(1 << 24) + 1, 2000003, 123456789]
    k = torch.zeros(3, 1, 64, device="cuda")
    k[..., :32] = 1
    pools = [torch.zeros(3, 1, 16, 64, dtype=F16, device="cuda") for _ in range(2)]
    table = torch.full((3, pos[2] // 16 + 1), -1, dtype=torch.int32, device="cuda")
    for i, p in enumerate(pos):
        table[i, p // 16] = i
    freq = torch.full((32,), 1.0, device="cuda")
    xtg.kv16_append(*pools, k, k, table, ints(pos), ints([0, 1, 2, 3]), freq=freq)
    for i, p in enumerate(pos):
        a = torch.tensor(float(p), dtype=torch.float64)
        got = pools[0][i, 0, p % 16].double().cpu()
        # 2^-11 of f16, and the turns' 2^-52 of the position
        assert abs(got[0] - a.cos()) <= 2.0 ** -11 + 1e-6 and abs(got[32] - a.sin()) <= 2.0 ** -11 + 1e-6


@pytest.mark.parametrize("order", ["hnd", "nhd"])
def test_what_holds_nothing_is_left(xtg, cuda, order):
    gen = torch.Generator(device="cuda").manual_seed(1)
    page, kvh, d = 16, 2, 64
    shape = (6, kvh, page, d) if order == "hnd" else (6, page, kvh, d)
    pools = [torch.full(shape, 7.0, dtype=BF16, device="cuda") for _ in range(2)]
    k_pool, v_pool = [x if order == "hnd" else x.transpose(1, 2) for x in pools]
    # rows before position 0, on a page that is not there, past the table, past the pool, of no sequence
    table = ints([[0, -1, 2], [3, 4, 5], [1, 9, 1]])
    pos, cu = ints([-2, 40, 14]), ints([0, 20, 30, 34])
    k = normal(gen, 36, kvh, d, dtype=BF16)
    q = normal(gen, 36, 4, d, dtype=BF16)
    err = ints([0])
    got = xtg.kv16_append(k_pool, v_pool, k, k, table, pos, cu, q=q, err=err)
    assert int(err) in (6, 7)
    with pytest.raises(xtg.XtgError):
        xtg.kv4_check(err)
    assert int(err) == 0
    want = torch.full((6, kvh, page, d), 7.0, dtype=BF16, device="cuda")
    want[0, :, 0:16] = k[2:18].transpose(0, 1)     # positions 0 .. 15 of sequence 0; 16, 17 have no page
    want[5, :, 8:16] = k[20:28].transpose(0, 1)    # positions 40 .. 47 of sequence 1; 48, 49 lie past the table
    want[1, :, 14:16] = k[30:32].transpose(0, 1)   # positions 14, 15 of sequence 2; 16, 17 on a page past the pool
    assert torch.equal(k_pool, want) and torch.equal(v_pool, want)
    assert torch.equal(got[:34], q[:34]) and not got[34:].any()


def test_thousands_of_rows(xtg, cuda):
    # enough that a CTA takes several rows, of sequences of every length
    gen = torch.Generator(device="cuda").manual_seed(2)
    rows = [(37 * i) % 90 for i in range(150)]
    pos = [(53 * i) % 300 for i in range(150)]
    table, p, cu, pages = tables(gen, rows, pos, 64)
    n, freq = sum(rows), freqs(32)
    assert n > 148 * 8 * 4
    pools = [torch.zeros(pages, 2, 64, 64, dtype=F16, device="cuda") for _ in range(2)]
    k, v = normal(gen, n, 2, 64), normal(gen, n, 2, 64)
    q = normal(gen, n, 3, 64)
    at = torch.cat([torch.arange(a, a + m) for m, a in zip(rows, pos)]).cuda()
    got = xtg.kv16_append(*pools, k, v, table, p, cu, freq=freq, q=q)
    close(got, *turned(q, at, freq, 0, False), "q")
    seq = torch.repeat_interleave(torch.arange(150, device="cuda"), torch.tensor(rows, device="cuda"))
    pg, sl = table[seq, at // 64].long(), at % 64
    y, room = turned(k, at, freq, 0, False)
    close(pools[0][pg, :, sl], y, room, "keys")
    assert torch.equal(pools[1][pg, :, sl], v.to(F16))
    for x in pools:
        x[pg, :, sl] = 0
        assert not x.any()


def test_a_captured_append_follows_the_tables(xtg, cuda):
    gen = torch.Generator(device="cuda").manual_seed(3)
    pools = [torch.zeros(4, 1, 16, 64, dtype=BF16, device="cuda") for _ in range(2)]
    table, pos, cu = ints([[0, 1]]), ints([3]), ints([0, 1])
    k, v, q = (normal(gen, 1, h, 64) for h in (1, 1, 2))
    freq = freqs(32)
    args = (*pools, k, v, table, pos, cu)
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        xtg.kv16_append(*args, freq=freq, q=q)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = xtg.kv16_append(*args, freq=freq, q=q)
    for p, page in ((17, 2), (31, 3)):
        pos.fill_(p)
        table[0, 1] = page
        k.copy_(normal(gen, 1, 1, 64))
        q.copy_(normal(gen, 1, 2, 64))
        g.replay()
        at = torch.tensor([p], device="cuda")
        close(out, *turned(q, at, freq, 0, False), "q")
        close(pools[0][page, :, p % 16][None], *turned(k, at, freq, 0, False), "keys")


def test_refusals(xtg, cuda):
    k_pool = torch.zeros(2, 2, 16, 64, dtype=BF16, device="cuda")
    table, pos, cu = ints([[0]]), ints([0]), ints([0, 1])
    x = torch.zeros(1, 2, 64, device="cuda")

    def refused(match, k=x, v=x, pools=(k_pool, k_pool), **kw):
        with pytest.raises(xtg.XtgError, match=match):
            xtg.kv16_append(*pools, k, v, table, pos, cu, **kw)
    refused("type", v=x.to(BF16))
    refused("float32", k=x.double(), v=x.double())
    refused(r"\[rows\]\[heads\]", k=x[:, :1])
    refused("contiguous dims", k=x.transpose(1, 2).contiguous().transpose(1, 2))
    refused("strides", k=torch.zeros(1, 2, 66, device="cuda")[..., :64])
    refused("freq", freq=torch.zeros(32, dtype=torch.float64, device="cuda"))
    refused("freq", freq=torch.zeros(32))
    refused("rotary", freq=torch.zeros(30, device="cuda"))
    refused("head", freq=torch.zeros(32, device="cuda"), first=8)
    refused("v_pool", pools=(k_pool, k_pool.to(F16)))
    refused("page", pools=(k_pool[:, :, :15], k_pool[:, :, :15]))
    refused("strides", pools=(k_pool[:1, :1].expand(2, 2, 16, 64), k_pool))
