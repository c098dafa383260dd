"""The 16-bit paged caches' definition in 64 bits, on torch tensors of any device."""
import math

import torch


def rotate(x, pos, freq, interleaved):
    """Rows x [n][heads][2 m] turned by their positions pos [n]: 64 bits."""
    angle = pos.double()[:, None] * freq.double()
    c, s = torch.cos(angle)[:, None], torch.sin(angle)[:, None]
    x = x.double()
    m = freq.numel()
    a, b = (x[..., ::2], x[..., 1::2]) if interleaved else (x[..., :m], x[..., m:])
    y = torch.stack([a * c - b * s, b * c + a * s], -1 if interleaved else -2)
    return y.flatten(-2)


def sequences(table, pos, cu_rows):
    """(sequence, its first row, its rows, the position of its first row)"""
    cu, p = cu_rows.tolist(), pos.tolist()
    return [(i, cu[i], cu[i + 1] - cu[i], p[i]) for i in range(table.shape[0])]


def places(table, i, first, n, page, pages):
    """(position, page or -1, slot) of n positions of sequence i from `first` on."""
    row = table[i].tolist()
    out = []
    for p in range(first, first + n):
        at = row[p // page] if 0 <= p // page < len(row) and p >= 0 else -1
        out.append((p, at if at < pages else -1, p % page))
    return out


def held(pool, table, i, n, page):
    """Positions 0 .. n - 1 of sequence i in pool [pages][kv_heads][page][d]: ([n][kv_heads][d] in 64 bits, which are there)."""
    pages = pool.shape[0]
    at = places(table, i, 0, n, page, pages)
    ok = torch.tensor([x[1] >= 0 for x in at], device=pool.device)
    pg = torch.tensor([max(x[1], 0) for x in at], device=pool.device, dtype=torch.long)
    sl = torch.tensor([x[2] for x in at], device=pool.device, dtype=torch.long)
    return pool[pg, :, sl].double(), ok


def attention(q, k_pool, v_pool, table, pos, cu_rows, scale, window=0):
    """(out, mass, score): out [rows][heads][v_dim] in 64 bits (NaN in rows that are no sequence's), mass = sum_p P |v| / sum P
    of each output and score = max_p scale sum |q k| of each row and head, from which tolerances are made."""
    rows, heads, d = q.shape
    kvh, dv, page = k_pool.shape[1], v_pool.shape[3], k_pool.shape[2]
    g = heads // kvh
    out = torch.full((rows, heads, dv), math.nan, dtype=torch.float64, device=q.device)
    mass, score = torch.zeros_like(out), torch.zeros((rows, heads), dtype=torch.float64, device=q.device)
    for i, a, n, p0 in sequences(table, pos, cu_rows):
        last = min(p0 + n, table.shape[1] * page)
        if n == 0:
            continue
        if last <= 0:
            out[a:a + n] = 0
            continue
        k, ok = held(k_pool, table, i, last, page)
        v, _ = held(v_pool, table, i, last, page)
        key = torch.arange(last, device=q.device)
        t = torch.arange(p0, p0 + n, device=q.device)[:, None]
        see = (key <= t) & ok
        if window:
            see &= key > t - window
        for h in range(kvh):
            x = q[a:a + n, h * g:(h + 1) * g].double()
            s = torch.einsum("ngd,pd->ngp", x, k[:, h]) * scale
            s = s.masked_fill(~see[:, None], -math.inf)
            m = s.amax(-1, keepdim=True)
            w = torch.where(see[:, None], torch.exp(s - torch.where(m == -math.inf, 0, m)), 0)
            total = w.sum(-1, keepdim=True)
            w = torch.where(total > 0, w / total, w)
            # a position that a row does not see must not enter, whatever is there
            clean = torch.nan_to_num(v[:, h], nan=0, posinf=0, neginf=0)
            o = torch.einsum("ngp,pd->ngd", w, clean)
            for p in torch.nonzero(~torch.isfinite(v[:, h]).all(-1))[:, 0].tolist():
                bad = torch.where(torch.isfinite(v[p, h]), torch.zeros_like(v[p, h]), v[p, h])
                o += torch.where(see[:, None, p, None], bad, 0)
            out[a:a + n, h * g:(h + 1) * g] = o
            mass[a:a + n, h * g:(h + 1) * g] = torch.einsum("ngp,pd->ngd", w, clean.abs())
            kk = torch.nan_to_num(k[:, h], nan=0, posinf=0, neginf=0)
            z = torch.einsum("ngd,pd->ngp", x.abs(), kk.abs()) * abs(scale)
            score[a:a + n, h * g:(h + 1) * g] = torch.where(see[:, None], z, 0).amax(-1)
    return out, mass, score


def tolerance(ref, dtype, dims, positions):
    """How far out may be off. h: half a step of the type. The weights are rounded to it (numerator and sum: 2 h mass) and the
    output once (h |out|); the scores' sums in f32 lose up to 2^-23 a step (2 x dims steps x score x mass, since the weights
    move with the scores and so does their sum), the sums over positions as much a step of 16 of them; ex2 and the factors
    2^-20; weights below the type's least normal number up to 2^-25 each, of sums that are at least 2^3."""
    out, mass, score = ref
    h = torch.finfo(dtype).eps / 2
    most = mass.amax(-1, keepdim=True)
    return (mass * (2 * h + 2 * dims * 2.0 ** -23 * score[..., None] + positions / 16 * 2.0 ** -23 + 2.0 ** -20)
            + h * out.abs() + positions * 2.0 ** -28 * most + 2.0 ** -24)
