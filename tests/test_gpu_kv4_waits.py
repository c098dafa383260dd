"""GPU: attention over the 4-bit cache when its waits give up. With a limit of no polls every wait does so at once, while
the copies of the ring's first stages are under way: the call has to end, with the error recorded and no row that looks
like a result, and the next call has to be right."""
import numpy as np
import pytest

from test_gpu_kv4 import Setup, torch  # noqa: F401 (a fixture)

pytestmark = pytest.mark.gpu


@pytest.fixture
def polls(xtg):
    L = xtg.lib()
    before = L.xtg_cuda_kv4_wait_polls(-1)
    yield L.xtg_cuda_kv4_wait_polls
    L.xtg_cuda_kv4_wait_polls(before)


@pytest.mark.parametrize("rows,pos", [([1], [0]), ([1], [1000]), ([9, 1, 70, 2, 1], [700, 1100, 0, 64, 1])])
@pytest.mark.parametrize("heads,kvh,d,dtype", [(8, 2, 128, "bf16"), (4, 4, 64, "f32"), (8, 2, 256, "f16")])
def test_waits_that_give_up(cuda, xtg, torch, polls, rows, pos, heads, kvh, d, dtype):  # noqa: F811
    s = Setup(torch, xtg, 21, rows, pos, kvh, d)
    s.fill([p + n for p, n in zip(pos, rows)])
    right = s.check_attention(heads, dtype)
    s.rng = np.random.default_rng(22)
    q = torch.from_numpy(s.rows_of(heads)).cuda().to(right.dtype)
    attend = lambda **kw: xtg.kv4_attention(q, s.pool, *s.where, scale=0.2, **kw)
    right = attend()
    polls(0)
    out = attend(err=s.err)
    torch.cuda.synchronize()
    assert torch.isnan(out).all()
    with pytest.raises(xtg.XtgError, match="timed out"):
        xtg.kv4_check(s.err)
    assert torch.isnan(attend()).all()   # nobody to tell: the rows still do
    for n in (1, 2, 5, 40):   # some waits give up, some do not: a row is right or NaN
        polls(n)
        for _ in range(5):
            out = attend(err=s.err)
            same = ((out == right) | torch.isnan(out)).all()
            recorded = int(s.err.item())
            assert same and (recorded == 1 or not torch.isnan(out).any())
            s.err.zero_()
    polls(1 << 18)
    assert torch.equal(attend(err=s.err), right)
    xtg.kv4_check(s.err)
