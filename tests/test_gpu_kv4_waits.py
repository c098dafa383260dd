"""GPU: attention over the 4-bit cache when its waits give up. With a limit of no polls every wait does so at once, while
the copies of the ring's first stages are under way: the call has to end, with the error recorded and no row that looks
like a result, and the next call has to be right."""
import numpy as np
import pytest

from test_gpu_kv4 import Setup, torch  # noqa: F401 (a fixture)
from test_gpu_kv4_ring import Shared

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


@pytest.mark.parametrize("d,rows,dtype", [(128, 1, "bf16"), (128, 2, "f16"), (64, 5, "f32"), (256, 2, "bf16")])
def test_waits_that_give_up_over_many_parts(cuda, xtg, torch, polls, d, rows, dtype):  # noqa: F811
    """A warp that gave up goes through the CTA's other parts, several turns of the ring, without its waits."""
    table = np.arange(22)[None].repeat(4, 0)
    s = Shared(torch, xtg, 23, rows, [1290, 70, 0, 639], table, 8, 2, d, dtype)
    right = s.run(600, 0.1)
    for n in (0, 1, 2, 5):
        polls(n)
        for _ in range(3):
            out, err = s.attend(600, 0.1)
            nan = torch.isnan(out)
            assert ((out == right) | nan).all() and (int(err.item()) == 1 or not nan.any())
            assert n > 0 or nan.all()
    polls(1 << 18)
    assert torch.equal(s.run(600, 0.1), right)
