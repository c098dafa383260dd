"""Inputs of the 16-bit caches' GPU tests."""
import torch

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def normal(gen, *shape, dtype=F32):
    return torch.randn(shape, generator=gen, device="cuda").to(dtype)


def tables(gen, rows, pos, page, spare=1, slack=0):
    """(table, pos, cu_rows, pages) of sequences with these rows at these positions; their pages in any order, -1 past them."""
    need = [-(-max(p + n, 0) // page) for n, p in zip(rows, pos)]
    width, pages = max(need + [1]) + slack, sum(need) + spare
    order = torch.randperm(pages, generator=gen, device="cuda").tolist()
    table, at = [], 0
    for n in need:
        table.append(order[at:at + n] + [-1] * (width - n))
        at += n
    cu = [0]
    for n in rows:
        cu.append(cu[-1] + n)
    return ints(table), ints(pos), ints(cu), pages


def pools(gen, pages, kv_heads, page, d, dv, dtype, order="hnd"):
    """Keys and values; "nhd": as [pages][page][kv_heads][d] in memory."""
    out = []
    for dim in (d, dv):
        shape = (pages, kv_heads, page, dim) if order == "hnd" else (pages, page, kv_heads, dim)
        x = normal(gen, *shape, dtype=dtype)
        out.append(x if order == "hnd" else x.transpose(1, 2))
    return out


def check(got, want, tol, what=""):
    got = got.double()
    off = (got - want).abs()
    bad = ~((off <= tol) | (got == want) | (got.isnan() & want.isnan()))
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float((off - tol)[bad].max())} over the bound"
