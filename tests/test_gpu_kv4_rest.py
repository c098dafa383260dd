"""GPU: rows of a call that are no sequence's: zeros in outputs that the package makes, left alone in the caller's."""
import numpy as np
import pytest

from test_gpu_kv4 import Setup, dtype_of, torch  # noqa: F401 (a fixture)

pytestmark = pytest.mark.gpu


def litter(torch):  # noqa: F811
    """Leaves memory that is not zero where the next outputs are likely to be allocated."""
    for n in (1 << 12, 1 << 16, 1 << 20, 1 << 22):
        for _ in range(4):
            torch.full((n,), float("nan"), device="cuda")


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows,pos,more", [([3], [0], 1), ([1], [100], 700), ([70, 0, 2], [5, 3, 60], 9),
                                           ([1] * 40, list(range(40)), 24), ([0, 0], [0, 7], 5)])
def test_rows_past_the_last_sequence(cuda, xtg, torch, rows, pos, more, dtype):  # noqa: F811
    s = Setup(torch, xtg, 50, rows, pos, 2, 128, garbage=False)
    s.fill([p + n for p, n in zip(pos, rows)])
    n = sum(rows)
    t = dtype_of(torch, dtype)
    litter(torch)
    k, v = xtg.kv4_load(s.pool, *s.where, rows=n + more, dtype=t, err=s.err)
    want = s.ref.load(s.table, s.pos, s.cu)
    for got, w in ((k, want[0]), (v, want[1])):
        assert torch.equal(got[:n].cpu(), torch.from_numpy(w.astype(np.float32)).to(t)) and not got[n:].any()
    q = torch.from_numpy(s.rows_of(8, rows=n + more)).cuda().to(t)
    litter(torch)
    out = xtg.kv4_attention(q, s.pool, *s.where, scale=0.1, err=s.err)
    assert not out[n:].any()
    if n:
        assert torch.equal(out[:n], xtg.kv4_attention(q[:n], s.pool, *s.where, scale=0.1,
                                                      rows_per_seq=-(-(n + more) // len(rows))))
    given = torch.full_like(q, 7)
    xtg.kv4_attention(q, s.pool, *s.where, scale=0.1, out=given)
    assert torch.equal(given[:n], out[:n]) and (given[n:] == 7).all()
    xtg.kv4_check(s.err)


def test_rows_before_the_first_sequence(cuda, xtg, torch):  # noqa: F811
    s = Setup(torch, xtg, 51, [4, 2], [0, 0], 2, 128)
    s.fill([4, 2])
    first = s.where[2] + 3
    q = torch.from_numpy(s.rows_of(4, rows=12)).cuda()
    litter(torch)
    out = xtg.kv4_attention(q, s.pool, *s.where[:2], first, scale=0.1)
    k, v = xtg.kv4_load(s.pool, *s.where[:2], first, rows=12)
    for x in (out, k, v):
        assert not x[:3].any() and not x[9:].any() and x[3:9].any((1, 2)).all()


@pytest.mark.parametrize("d", [64, 128, 256])
def test_no_sequences(cuda, xtg, torch, d):  # noqa: F811
    i32 = dict(dtype=torch.int32, device="cuda")
    pool = xtg.kv4_pool(2, 2, d)
    where = torch.zeros((0, 3), **i32), torch.zeros(0, **i32), torch.zeros(1, **i32)
    q = torch.ones((5, 4, d), device="cuda", dtype=torch.bfloat16)
    litter(torch)
    out = xtg.kv4_attention(q, pool, *where, scale=0.1)
    k, v = xtg.kv4_load(pool, *where, rows=5, dtype=torch.float32)
    assert out.shape == q.shape and k.shape == (5, 2, d) and not (out.any() or k.any() or v.any())
    xtg.kv4_store(pool, k, v, *where)
    assert not pool.any()
