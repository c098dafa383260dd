"""GPU: the 4-bit paged cache's store, load and attention against its definition in numpy (tests/kv4_ref.py). Stored
bytes and values read back are exact; attention is within kv4_ref.attention_bound. Every pool starts as garbage: what a
call does not write, and what no row sees, may hold anything."""
import numpy as np
import pytest

import kv4_ref as R

pytestmark = pytest.mark.gpu

MANTISSA = {"f32": 23, "bf16": 8, "f16": 11}   # an output's rounding is within 2^-mantissa of it


@pytest.fixture(scope="module")
def torch():
    import torch
    assert torch.cuda.is_available()
    return torch


def dtype_of(torch, name):
    return {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}[name]


class Setup:
    """Sequences of `rows` rows at positions `pos`, their pages scattered over a garbage pool on both sides."""

    def __init__(self, torch, xtg, seed, rows, pos, kvh, d, max_pages=None, garbage=True):
        self.torch, self.xtg = torch, xtg
        self.rng = np.random.default_rng(seed)
        self.pos = np.array(pos, np.int32)
        self.cu = np.concatenate([[0], np.cumsum(rows)]).astype(np.int32)
        most = max(max(int(p) + n for p, n in zip(pos, rows)), 1)
        self.max_pages = max_pages or -(-most // 64)
        pages = len(rows) * self.max_pages + 3
        self.table = self.rng.permutation(pages)[:len(rows) * self.max_pages].astype(np.int32).reshape(len(rows), -1)
        self.ref = R.Cache(pages, kvh, d)
        if garbage:   # any bits, NaN and infinite scales among them
            self.ref.words[:] = self.rng.integers(0, 1 << 32, self.ref.words.shape, dtype=np.uint32)
        self.kvh, self.d = kvh, d
        self.upload()

    def upload(self):
        t = lambda a: self.torch.from_numpy(np.ascontiguousarray(a)).cuda()
        self.pool = t(self.ref.bytes).view(len(self.ref.words), self.kvh, 72 * self.d)
        self.where = (t(self.table), t(self.pos), t(self.cu))
        self.err = self.torch.zeros(1, dtype=self.torch.int32, device="cuda")

    def same_pool(self):
        return np.array_equal(self.pool.cpu().numpy().reshape(-1), self.ref.bytes.reshape(-1))

    def rows_of(self, heads, scale=1.0, rows=None):
        return (self.rng.standard_normal((rows or self.cu[-1], heads, self.d)) * scale).astype(np.float32)

    def fill(self, upto):
        """Valid keys and values at positions 0 .. upto[s] - 1 of every sequence, on both sides."""
        zero = np.zeros(len(upto), np.int32)
        cu = np.concatenate([[0], np.cumsum(upto)]).astype(np.int32)
        k = self.rng.standard_normal((cu[-1], self.kvh, self.d)).astype(np.float32) + 0.3
        v = self.rng.standard_normal((cu[-1], self.kvh, self.d)).astype(np.float32)
        self.ref.store(k, v, self.table, zero, cu)
        self.upload()

    def check_attention(self, heads, dtype="bf16", window=0, scale=None, strided=False, **kw):
        torch = self.torch
        scale = scale or 1.5 / np.sqrt(self.d)
        q = torch.from_numpy(self.rows_of(heads, 2.0)).cuda().to(dtype_of(torch, dtype))
        if strided:   # the q part of a fused q | k | v row
            wide = torch.full((q.shape[0], heads + 2 * self.kvh, self.d), float("nan"), dtype=q.dtype, device="cuda")
            wide[:, :heads] = q
            q = wide[:, :heads]
        got = self.xtg.kv4_attention(q, self.pool, *self.where, scale=scale, window=window, err=self.err, **kw)
        torch.cuda.synchronize()
        assert got.dtype == q.dtype and got.shape == q.shape
        want, reach, top = self.ref.attention(q.double().cpu().numpy(), self.table, self.pos, self.cu, scale, window)
        g = got.double().cpu().numpy()
        assert np.array_equal(np.isnan(g), np.isnan(want))
        off = np.nan_to_num(np.abs(g - want)) / np.nan_to_num(R.attention_bound(want, reach, top, MANTISSA[dtype]),
                                                              nan=1.0)
        assert off.max() <= 1, (off.max(), np.unravel_index(off.argmax(), off.shape))
        return got


CASES = [  # rows, pos of each sequence
    ([1], [0]), ([1], [63]), ([1], [64]), ([64], [0]), ([65], [63]), ([200], [17]),
    ([3, 1, 0, 130, 2], [5, 127, 9, 60, 0]), ([1] * 40, list(range(0, 400, 10))),
]


@pytest.mark.parametrize("rows,pos", CASES)
@pytest.mark.parametrize("kvh,d,dtype", [(2, 128, "f32"), (1, 64, "bf16"), (3, 256, "f16"), (2, 128, "bf16")])
def test_store_is_bit_exact_and_leaves_the_rest(cuda, xtg, torch, rows, pos, kvh, d, dtype):
    s = Setup(torch, xtg, 1, rows, pos, kvh, d)
    k, v = (torch.from_numpy(s.rows_of(kvh)).cuda().to(dtype_of(torch, dtype)) for _ in range(2))
    s.ref.store(k.float().cpu().numpy(), v.float().cpu().numpy(), s.table, s.pos, s.cu)
    xtg.kv4_store(s.pool, k, v, *s.where, err=s.err)
    torch.cuda.synchronize()
    assert s.same_pool()
    xtg.kv4_check(s.err)


def test_store_takes_strided_rows(cuda, xtg, torch):
    s = Setup(torch, xtg, 2, [70, 3], [30, 0], 2, 128)
    fused = torch.from_numpy(s.rows_of(8 + 2 + 2)).cuda()   # q | k | v
    k, v = fused[:, 8:10], fused[:, 10:]
    s.ref.store(k.cpu().numpy(), v.cpu().numpy(), s.table, s.pos, s.cu)
    xtg.kv4_store(s.pool, k, v, *s.where)
    torch.cuda.synchronize()
    assert s.same_pool()


def test_store_of_extremes(cuda, xtg, torch):
    """Constants, zeros, subnormals, the type's largest values (their spread leaves f32), infinities and NaN."""
    s = Setup(torch, xtg, 3, [12], [60], 1, 128)
    k = s.rows_of(1)
    k[0], k[1], k[2] = 0, 10.01, np.float32(1e-42)
    k[3, 0, 5], k[4, 0, 70], k[5, 0, 127] = np.nan, np.inf, -np.inf
    k[6, 0, :2] = [3.4e38, -3.4e38]
    k[7] *= np.float32(1e-38)
    k[8] *= np.float32(1e37)
    k[9] += 1e6
    v = -k[::-1].copy()
    with np.errstate(all="ignore"):
        s.ref.store(k, v, s.table, s.pos, s.cu)
    xtg.kv4_store(s.pool, torch.from_numpy(k).cuda(), torch.from_numpy(v).cuda(), *s.where)
    torch.cuda.synchronize()
    assert s.same_pool()
    kk, _ = xtg.kv4_load(s.pool, *s.where, rows=12, dtype=torch.float32)
    nan = torch.isnan(kk[:, 0]).cpu().numpy()
    assert nan[3, :64].all() and not nan[3, 64:].any() and nan[4, 64:].all() and nan[5, 64:].all()
    assert nan[6, :64].all() and not nan[[0, 1, 2, 7, 8, 9]].any()


@pytest.mark.parametrize("rows,pos", CASES)
@pytest.mark.parametrize("kvh,d,dtype", [(2, 128, "f32"), (1, 64, "f16"), (3, 256, "bf16"), (2, 128, "bf16")])
def test_load_is_exact(cuda, xtg, torch, rows, pos, kvh, d, dtype):
    s = Setup(torch, xtg, 4, rows, pos, kvh, d, garbage=False)
    s.fill([p + n for p, n in zip(pos, rows)])
    got = xtg.kv4_load(s.pool, *s.where, rows=int(s.cu[-1]), dtype=dtype_of(torch, dtype), err=s.err)
    want = s.ref.load(s.table, s.pos, s.cu)
    for g, w in zip(got, want):
        assert torch.equal(g.cpu(), torch.from_numpy(w.astype(np.float32)).to(g.dtype))
    xtg.kv4_check(s.err)


def test_nothing_there(cuda, xtg, torch):
    """Absent pages and negative positions: a store skips them, a load gives zeros, attention does not see them; a
    sequence without rows touches nothing."""
    rows, pos = [70, 5, 0, 6, 130], [20, -2, 3, -9, 0]
    s = Setup(torch, xtg, 5, rows, pos, 2, 128, garbage=False)
    s.fill([90, 3, 3, 0, 130])
    s.table[0, 0] = -1
    s.table[4, 1] = -7
    s.upload()
    k, v = s.rows_of(2), s.rows_of(2)
    s.ref.store(k, v, s.table, s.pos, s.cu)
    xtg.kv4_store(s.pool, torch.from_numpy(k).cuda(), torch.from_numpy(v).cuda(), *s.where, err=s.err)
    torch.cuda.synchronize()
    assert s.same_pool()
    got = xtg.kv4_load(s.pool, *s.where, rows=int(s.cu[-1]), dtype=torch.float32, err=s.err)
    for g, w in zip(got, s.ref.load(s.table, s.pos, s.cu)):
        assert np.array_equal(g.cpu().numpy(), w.astype(np.float32))
    out = s.check_attention(8, "f32")
    assert not out[:44].any()   # sequence 0's rows at 20 .. 63: their page is absent
    assert not out[75:81].any() and not out[70:72].any()   # negative positions
    xtg.kv4_check(s.err)


ATTENTION = [  # rows, pos
    ([1], [0]), ([1], [62]), ([1], [63]), ([1], [64]), ([1], [700]), ([8], [0]), ([8], [60]), ([8], [1016]),
    ([5], [333]), ([64], [100]), ([70], [0]), ([1, 1, 1, 1, 1], [0, 3, 64, 511, 1000]),
    ([3, 1, 0, 17, 2], [5, 127, 9, 60, 0]),
]


@pytest.mark.parametrize("rows,pos", ATTENTION)
@pytest.mark.parametrize("heads,kvh,d,dtype,window", [
    (24, 6, 128, "bf16", 0), (8, 2, 128, "f32", 0), (16, 4, 256, "f16", 0), (8, 8, 64, "f32", 0),
    (12, 1, 128, "bf16", 100), (4, 2, 256, "f32", 64), (5, 1, 64, "f16", 1), (8, 2, 128, "f16", 37),
])
def test_attention(cuda, xtg, torch, rows, pos, heads, kvh, d, dtype, window):
    s = Setup(torch, xtg, 6, rows, pos, kvh, d)
    s.fill([p + n for p, n in zip(pos, rows)])
    s.check_attention(heads, dtype, window)
    xtg.kv4_check(s.err)


@pytest.mark.parametrize("window", [0, 1, 3, 70, 2 ** 31 - 1])
def test_rows_before_the_first_position(cuda, xtg, torch, window):
    """Rows at negative positions, some beside rows that see something in the same block, with windows of every size."""
    rows, pos = [9, 3, 70, 2], [-4, -3, -6, -2 ** 31]
    s = Setup(torch, xtg, 16, rows, pos, 2, 128, max_pages=2)
    s.fill([5, 0, 64, 0])
    out = s.check_attention(8, "f32", window)
    assert not out[:4].any() and not out[9:12].any() and not out[12:18].any() and out[4:9].any()
    xtg.kv4_check(s.err)


def test_attention_over_more_sequences_than_threads(cuda, xtg, torch):
    rows = [1 + i % 3 if i % 7 else 0 for i in range(700)]
    pos = [(37 * i) % 150 for i in range(700)]
    s = Setup(torch, xtg, 7, rows, pos, 1, 64)
    s.fill([p + n for p, n in zip(pos, rows)])
    s.check_attention(2, "f32")
    k, v = s.rows_of(1), s.rows_of(1)
    s.ref.store(k, v, s.table, s.pos, s.cu)
    xtg.kv4_store(s.pool, torch.from_numpy(k).cuda(), torch.from_numpy(v).cuda(), *s.where)
    torch.cuda.synchronize()
    assert s.same_pool()


@pytest.mark.parametrize("hint", [1, 2, 3, 8, 1000])
def test_attention_holds_for_any_tiling(cuda, xtg, torch, hint):
    s = Setup(torch, xtg, 8, [9, 1, 30], [100, 450, 3], 2, 128)
    s.fill([109, 451, 33])
    s.check_attention(6, "f32", rows_per_seq=hint)


def test_attention_of_strided_queries_twice_the_same(cuda, xtg, torch):
    s = Setup(torch, xtg, 9, [8, 8], [900, 40], 2, 128)
    s.fill([908, 48])
    s.check_attention(8, "bf16", strided=True)
    q = torch.from_numpy(s.rows_of(8)).cuda()
    a, b = (xtg.kv4_attention(q, s.pool, *s.where, scale=0.2) for _ in range(2))
    assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_attention_of_loud_values(cuda, xtg, torch, dtype):
    """Scores whose softmax is one position, V scales that differ by powers of ten between positions and groups."""
    s = Setup(torch, xtg, 10, [4], [300], 2, 128)
    k = s.rows_of(2, rows=304)
    v = s.rows_of(2, rows=304) * (10.0 ** s.rng.integers(-6, 7, (304, 2, 1)))
    v[:, :, 64:] *= 1e-3
    s.ref.store(k, v.astype(np.float32), s.table, np.zeros(1, np.int32), np.array([0, 304], np.int32))
    s.upload()
    s.check_attention(8, dtype, scale=3.0)
    s.check_attention(8, dtype, scale=1e-3)


@pytest.mark.parametrize("dtype,factor,scale", [
    ("f32", 1.0, -0.2), ("bf16", 1.0, -0.2), ("f32", 1.0, 0.0), ("f16", 1.0, 0.0), ("f32", 1e-30, 2e29),
    ("f32", 1e30, 2e-31), ("bf16", 1e-30, 2e29), ("f16", 1e-4, 2e3), ("f32", 0.0, 1.0),
])
def test_attention_of_queries_of_any_size(cuda, xtg, torch, dtype, factor, scale):
    """Negative and zero scales, queries near the ends of their type beside a scale that undoes it, rows of zeros, and
    rows whose values differ by a factor of 2^20 within the row."""
    s = Setup(torch, xtg, 17, [3], [150], 2, 128)
    s.fill([153])
    rows = s.rows_of(8)
    rows[1, :, ::3] *= 2.0 ** -20
    rows[2, 3] = 0
    q = torch.from_numpy(rows * np.float32(factor)).cuda().to(dtype_of(torch, dtype))
    got = xtg.kv4_attention(q, s.pool, *s.where, scale=scale).double().cpu().numpy()
    want, reach, top = s.ref.attention(q.double().cpu().numpy(), s.table, s.pos, s.cu, scale)
    assert (np.abs(got - want) <= R.attention_bound(want, reach, top, MANTISSA[dtype])).all()


def test_nan_stays_with_the_rows_that_see_it(cuda, xtg, torch):
    """A NaN key at position 102 and a NaN value group at 104: rows up to 101 are clean, rows to 103 all NaN from the
    key; a query with a NaN spoils its own row."""
    s = Setup(torch, xtg, 11, [8], [98], 1, 128)
    k, v = s.rows_of(1, rows=106), s.rows_of(1, rows=106)
    v[104, 0, 70] = np.nan
    zero, cu = np.zeros(1, np.int32), np.array([0, 106], np.int32)
    s.ref.store(k, v, s.table, zero, cu)
    s.upload()
    q = torch.from_numpy(s.rows_of(4)).cuda()
    q[1, 2, 5] = float("nan")
    out = xtg.kv4_attention(q, s.pool, *s.where, scale=0.1)
    nan = torch.isnan(out).cpu().numpy()
    assert nan[1, 2].all() and not nan[1, [0, 1, 3]].any() and not nan[[0, 2, 3, 4, 5]].any()
    assert nan[6:, :, 64:].all() and not nan[6:, :, :64].any()
    k[102, 0, 3] = np.inf
    s.ref.store(k, v, s.table, zero, cu)
    s.upload()
    nan = torch.isnan(xtg.kv4_attention(q[:, :, :].nan_to_num(0), s.pool, *s.where, scale=0.1)).cpu().numpy()
    assert not nan[:4].any() and nan[4:].all()


def test_errors_are_recorded(cuda, xtg, torch):
    s = Setup(torch, xtg, 12, [3, 2], [126, 0], 1, 128, max_pages=2)   # position 128 lies past the table
    s.fill([128, 2])
    k = torch.from_numpy(s.rows_of(1)).cuda()
    xtg.kv4_store(s.pool, k, k, *s.where, err=s.err)
    with pytest.raises(xtg.XtgError, match="past its sequence's page table"):
        xtg.kv4_check(s.err)
    xtg.kv4_check(s.err)   # cleared
    _, v = xtg.kv4_load(s.pool, *s.where, rows=5, dtype=torch.float32, err=s.err)
    assert not v[2].any() and v[1].any()
    with pytest.raises(xtg.XtgError, match="page table"):
        xtg.kv4_check(s.err)
    xtg.kv4_attention(k, s.pool, *s.where, scale=0.1, err=s.err)
    with pytest.raises(xtg.XtgError, match="page table"):
        xtg.kv4_check(s.err)
    for seqs in (2, 20, 50):   # the last sequence's row past its table, whichever way the work is shared out
        t = Setup(torch, xtg, 18, [1] * seqs, [5] * (seqs - 1) + [64], 1, 64, max_pages=1)
        t.fill([6] * (seqs - 1) + [64])
        t.check_attention(2, "f32")
        with pytest.raises(xtg.XtgError, match="page table"):
            xtg.kv4_check(t.err)
    s.table[1, 0] = len(s.ref.words)
    s.upload()
    for call in (lambda: xtg.kv4_store(s.pool, k, k, *s.where, err=s.err),
                 lambda: xtg.kv4_load(s.pool, *s.where, rows=5, err=s.err),
                 lambda: xtg.kv4_attention(k[3:], s.pool, s.where[0][1:], s.where[1][1:], s.where[2][1:] - 3,
                                           scale=0.1, err=s.err)):
        call()
        with pytest.raises(xtg.XtgError):
            xtg.kv4_check(s.err)
    kk = k.cpu().numpy()
    s.ref.store(kk, kk, s.table, s.pos, s.cu)
    s.check_attention(1, "f32")   # nothing there: not seen


def test_another_stream_and_a_captured_graph(cuda, xtg, torch):
    """Calls run on the current stream; a captured call follows the later contents of pos and q."""
    s = Setup(torch, xtg, 13, [1, 1], [199, 70], 2, 128)
    s.fill([200, 200])
    q = torch.from_numpy(s.rows_of(8)).cuda()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        first = xtg.kv4_attention(q, s.pool, *s.where, scale=0.2)
    stream.synchronize()
    assert torch.equal(first, xtg.kv4_attention(q, s.pool, *s.where, scale=0.2))
    out = torch.empty_like(q)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        xtg.kv4_attention(q, s.pool, *s.where, scale=0.2, out=out)
    q.neg_()
    s.pos[:] = [50, 180]
    s.where[1].copy_(torch.from_numpy(s.pos))
    graph.replay()
    want, reach, top = s.ref.attention(q.double().cpu().numpy(), s.table, s.pos, s.cu, 0.2)
    off = np.abs(out.double().cpu().numpy() - want) / R.attention_bound(want, reach, top, 23)
    assert off.max() <= 1


def test_a_pool_past_32_bit_offsets(cuda, xtg, torch):
    """Pages whose byte offsets pass 2^32."""
    d, kvh = 256, 8
    pages = (1 << 32) // (72 * d * kvh) + 40
    pool = xtg.kv4_pool(pages, kvh, d)
    t = lambda a: torch.tensor(a, dtype=torch.int32, device="cuda")
    table = t([[pages - 1, 3, pages - 2]])
    rng = np.random.default_rng(14)
    k, v = (torch.from_numpy(rng.standard_normal((150, kvh, d)).astype(np.float32)).cuda() for _ in range(2))
    xtg.kv4_store(pool, k, v, table, t([0]), t([0, 150]))
    small = R.Cache(3, kvh, d)
    small.store(k.cpu().numpy(), v.cpu().numpy(), np.array([[0, 1, 2]]), np.array([0]), [0, 150])
    got = pool[table[0].long()].cpu().numpy().reshape(-1)
    assert np.array_equal(got, small.bytes.reshape(-1))
    kk, _ = xtg.kv4_load(pool, table, t([0]), t([0, 150]), rows=150, dtype=torch.float32)
    assert np.array_equal(kk.cpu().numpy(), small.load(np.array([[0, 1, 2]]), [0], [0, 150])[0].astype(np.float32))
    q = torch.from_numpy(rng.standard_normal((1, kvh, d)).astype(np.float32)).cuda()
    out = xtg.kv4_attention(q, pool, table, t([149]), t([0, 1]), scale=0.1)
    want, reach, top = small.attention(q.double().cpu().numpy(), np.array([[0, 1, 2]]), np.array([149]), [0, 1], 0.1)
    assert (np.abs(out.double().cpu().numpy() - want) <= R.attention_bound(want, reach, top, 23)).all()


def test_python_refusals(cuda, xtg, torch):
    s = Setup(torch, xtg, 15, [2], [0], 2, 128)
    k = torch.zeros((2, 2, 128), device="cuda")
    table, pos, cu = s.where
    bad = [
        lambda: xtg.kv4_store(s.pool, k, k.half(), table, pos, cu),
        lambda: xtg.kv4_store(s.pool, k[:, :1], k[:, :1], table, pos, cu),
        lambda: xtg.kv4_store(s.pool, k[..., :64], k[..., :64], table, pos, cu),
        lambda: xtg.kv4_store(s.pool, k.transpose(1, 2), k, table, pos, cu),
        lambda: xtg.kv4_store(s.pool, k.double(), k.double(), table, pos, cu),
        lambda: xtg.kv4_store(s.pool, torch.zeros((2, 2, 129), device="cuda")[..., 1:], k, table, pos, cu),
        lambda: xtg.kv4_store(s.pool, k, k, table.long(), pos, cu),
        lambda: xtg.kv4_store(s.pool, k, k, table, pos, cu[:1]),
        lambda: xtg.kv4_store(s.pool[:, :1], k, k, table, pos, cu),
        lambda: xtg.kv4_load(s.pool, table, pos, cu, rows=2, dtype=torch.float64),
        lambda: xtg.kv4_attention(torch.zeros((2, 3, 128), device="cuda"), s.pool, table, pos, cu, scale=1.0),
        lambda: xtg.kv4_attention(k, s.pool, table, pos, cu, scale=1.0, window=-1),
        lambda: xtg.kv4_attention(k, s.pool, table, pos, cu, scale=1.0, out=k.half()),
        lambda: xtg.kv4_attention(k, s.pool, table, pos, cu.cpu(), scale=1.0),
    ]
    for call in bad:
        with pytest.raises(xtg.XtgError):
            call()


def test_the_serving_example(cuda, xtg, torch):
    """examples/kv4_serving.py: prompts in chunks, one token steps, pages given back and taken again. 4-bit values are
    off by a uniform error of at most half a step: a step is a 15th of the range of 64 normal values, about 4.8 sigma, so
    0.32 sigma and 0.093 sigma rms; values' errors average as the values themselves do (9 %), and keys' errors move a
    score of sigma 1 by 0.09, whose effect on the weights adds about as much. 0.25 leaves room for the single rows."""
    import importlib.util
    import os
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "kv4_serving.py")
    spec = importlib.util.spec_from_file_location("kv4_serving", path)
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    worst, pages = mod.serve(prompts=(200, 65, 1, 130), steps=10)
    assert worst < 0.25 and pages == 4 + 2 + 1 + 3
    worst, pages = mod.serve(prompts=(400, 1), steps=12, window=100, heads=8, kv_heads=2)
    assert worst < 0.25 and pages <= 3 + 1
