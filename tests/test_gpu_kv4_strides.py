"""GPU: rows whose stride has no meaning, because there is one of them: any number will do."""
import pytest

from test_gpu_kv4 import Setup, torch  # noqa: F401 (a fixture)

pytestmark = pytest.mark.gpu


def test_one_row_of_an_odd_projection(cuda, xtg, torch):  # noqa: F811
    """One row of q | k | v | 3 more values: its parts start and stand as they should, only the stride to a next row is odd,
    which contiguous() leaves as it is."""
    s = Setup(torch, xtg, 60, [1], [70], 2, 128)
    s.fill([70])
    fused = torch.randn((1, 12 * 128 + 3), device="cuda").bfloat16()
    q, k, v = (fused.as_strided((1, b - a, 128), (fused.shape[1], 128, 1), 128 * a) for a, b in ((0, 8), (8, 10), (10, 12)))
    assert q.stride(0) % 8 and q.contiguous().stride(0) % 8
    s.ref.store(k.float().cpu().numpy(), v.float().cpu().numpy(), s.table, s.pos, s.cu)
    xtg.kv4_store(s.pool, k, v, *s.where)
    torch.cuda.synchronize()
    assert s.same_pool()
    want = xtg.kv4_attention(q.clone(memory_format=torch.contiguous_format), s.pool, *s.where, scale=0.1)
    assert torch.equal(xtg.kv4_attention(q, s.pool, *s.where, scale=0.1), want)
    two = torch.cat([fused, fused]).as_strided((2, 8, 128), q.stride())   # here the stride counts
    with pytest.raises(xtg.XtgError, match="strides"):
        xtg.kv4_attention(two, s.pool, *s.where, scale=0.1)


def test_one_head(cuda, xtg, torch):  # noqa: F811
    s = Setup(torch, xtg, 61, [5], [0], 1, 64)
    wide = torch.randn((5, 72), device="cuda")
    k = torch.as_strided(wide, (5, 1, 64), (72, 3, 1))   # the stride to a second head, which is not there
    s.ref.store(k.cpu().numpy(), k.cpu().numpy(), s.table, s.pos, s.cu)
    xtg.kv4_store(s.pool, k, k, *s.where)
    torch.cuda.synchronize()
    assert s.same_pool()
    assert torch.equal(xtg.kv4_attention(k, s.pool, *s.where, scale=0.1),
                       xtg.kv4_attention(k.clone(memory_format=torch.contiguous_format), s.pool, *s.where, scale=0.1))
