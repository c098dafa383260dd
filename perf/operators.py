"""What is measured of the 4-bit key/value cache: rows quantised into its pages, rows read back, attention over it.

`listed()` names the cases, `draw()` gives more of the same ranges, `prepare()` makes what a server holds before the
call, `run()` is one pass (`own`: through the framework's entry points, else in plain torch operations in 32 bits),
`exact()` the same results from the operators' definition in 64 bits, `work()` the bytes and operations that a pass
cannot do without.

The cache: `pool` [pages][kv_heads][72 head_dim] bytes. A page holds 64 positions of a head as
  K codes   [head_dim / H][64 slots][4][H / 32] words, H = min(head_dim, 128): nibble n of word [h][slot][a][b] is the
            code of head dim H h + 32 b + 8 a + n
  K params  [head_dim / 64][64 slots] words: of a slot's group of 64 head dims the scale s (bf16, high half) and the
            offset z (bf16, low half)
  V codes   [2][head_dim / 32][8][4][4] words: nibble n of word [h][c][g][a][t] is the code of head dim
            32 c + 8 t + g at slot 32 h + 8 (n % 4) + 2 a + n / 4
  V params  as K's
and a code c stands for s (c - 8) + z. Position p of sequence i is slot p % 64 of page table[i][p / 64]; the rows
cu_rows[i] .. cu_rows[i + 1] - 1 of a call stand at positions pos[i], pos[i] + 1, ...
"""
import importlib
import math
import random

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
PAGE = 64


# ---------------------------------------------------------------------------------------------------------------
# The cases
# ---------------------------------------------------------------------------------------------------------------

def _case(name, op, seqs, rows, length, heads, kv_heads, head_dim, dtype, window=0, ragged=False):
    c = dict(op=op, seqs=seqs, rows=rows, length=length, heads=heads, kv_heads=kv_heads, head_dim=head_dim,
             dtype=dtype, window=window, ragged=ragged)
    return dict(c, name=name) if name else c


def listed():
    """Two model shapes: 24 q / 6 KV heads of 128 (a context of 32768, verify steps of 8 rows, prompt chunks of 64, a
    sliding window of 1024, 64 sequences) and 16 q / 4 KV heads of 256. `length` counts a sequence's positions after
    the call, `rows` those of the call (the last ones)."""
    return [
        # the smallest call: one session appends one token's keys and values in its activations' type
        _case("store_read_1x1", "store", 1, 1, 4096, 24, 6, 128, "f32"),
        # a verify round's rows of 64 sequences at their own positions
        _case("store_read_64x8", "store", 64, 8, 8192, 24, 6, 128, "bf16", ragged=True),
        # whole prompts of several sequences written at once, the wider heads
        _case("store_read_8x4096", "store", 8, 4096, 4096, 16, 4, 256, "f16"),
        # a short prefix read back, starting and ending inside a page
        _case("read_1x1000", "load", 1, 1000, 1301, 24, 6, 128, "f32"),
        # the caches of 64 conversations read back (moved to another cache, or attended by another kernel)
        _case("read_64x4096", "load", 64, 4096, 4096, 24, 6, 128, "bf16", ragged=True),
        # one token of one conversation: latency
        _case("decode_1x4096", "attention", 1, 1, 4096, 24, 6, 128, "bf16"),
        # one token over a long document
        _case("decode_1x131072", "attention", 1, 1, 131072, 24, 6, 128, "bf16"),
        # a server's batch, every sequence at its own length: bandwidth
        _case("decode_64x32768", "attention", 64, 1, 32768, 24, 6, 128, "bf16", ragged=True),
        # a verify step's 8 rows, in the activations' own type
        _case("verify_1x8_at_32768", "attention", 1, 8, 32768, 24, 6, 128, "f32"),
        # the sliding layers of a batched verify round
        _case("verify_64x8_window", "attention", 64, 8, 16384, 24, 6, 128, "bf16", window=1024, ragged=True),
        # a prompt chunk over what is already cached
        _case("chunk_1x64_at_8192", "attention", 1, 64, 8192, 24, 6, 128, "bf16"),
        # the wider heads, lengths that end inside a page
        _case("decode_16x8191_d256", "attention", 16, 1, 8191, 16, 4, 256, "f16"),
    ]


_HEADS = [(24, 6, 128), (16, 4, 256), (8, 2, 128), (8, 8, 64), (12, 1, 128)]   # grouped, one each, one for all


def draw(rng):
    most = max(_cost(c) for c in listed())

    def log(a, b):
        return int(round(math.exp(rng.uniform(math.log(a), math.log(b)))))

    while True:
        op = rng.choice(["store", "load", "attention", "attention", "attention"])
        heads, kv_heads, head_dim = rng.choice(_HEADS)
        dtype = rng.choice(["f32", "bf16", "f16"])
        seqs = log(1, 64)
        length = log(40, 131072)
        if op == "attention":
            rows = min(log(1, 64), length)
            window = rng.choice([0, 0, log(16, 2048)])
        else:
            rows = min(log(1, 8192), length)
            window = 0
        c = _case(None, op, seqs, rows, length, heads, kv_heads, head_dim, dtype, window, rng.random() < 0.7)
        if _cost(c) <= most and seqs * length <= 64 * 32768:
            return c


def _plan(case):
    """Each sequence's rows in the call and its position before it, by the case alone."""
    rng = random.Random(repr([case[k] for k in ("op", "seqs", "rows", "length", "window")]))
    rows, pos = [], []
    for _ in range(case["seqs"]):
        n, length = case["rows"], case["length"]
        if case["ragged"]:
            length = rng.randint((length + 1) // 2, length)
            if case["op"] != "attention" or n > 8:   # a verify step's rows are the same for all
                n = rng.randint((n + 1) // 2, n)
            n = min(n, length)
        rows.append(n)
        pos.append(length - n)
    return rows, pos


def _seen(case):
    """(positions that some row of its sequence sees, (row, position) pairs), over all sequences."""
    held = pairs = 0
    w = case["window"]
    for n, p in zip(*_plan(case)):
        held += p + n - (max(0, p - w + 1) if w else 0)
        pairs += sum(min(w, p + i + 1) if w else p + i + 1 for i in range(n))
    return held, pairs


def work(case):
    d, kvh, heads = case["head_dim"], case["kv_heads"], case["heads"]
    size = DTYPES[case["dtype"]].itemsize
    rows = sum(_plan(case)[0])
    slot = 72 * d // PAGE * kvh   # a position's bytes in the cache
    if case["op"] == "attention":
        held, pairs = _seen(case)
        return {"bytes": held * slot + 2 * rows * heads * d * size, "flops": 4 * pairs * heads * d}
    wide = 2 * rows * kvh * d
    if case["op"] == "load":
        return {"bytes": rows * slot + wide * size, "flops": 2 * wide}
    return {"bytes": 2 * rows * slot + 2 * wide * size, "flops": 8 * wide}   # written, then read back


def _cost(case):
    w = work(case)
    return max(w["bytes"], w["flops"] / 50)


# ---------------------------------------------------------------------------------------------------------------
# The plain form
# ---------------------------------------------------------------------------------------------------------------

def _quantise(x):
    """f32 [..., head_dim] -> codes 0..15 (uint8) and each group's scale and offset [..., head_dim / 64] (f32)."""
    g = x.unflatten(-1, (-1, 64))
    lo, hi = g.amin(-1), g.amax(-1)
    s = (hi - lo) * (1.0 / 15.0)
    s = ((s.view(torch.int32) + 0xFFFF) & -0x10000).view(torch.float32).clamp_min(2.0 ** -100)
    z = (lo + 8.0 * s).to(torch.bfloat16).float()
    c = torch.round((g - z[..., None]) * (1.0 / s)[..., None]).clamp(-8, 7) + 8
    return c.to(torch.uint8).flatten(-2), s, z


def _to_params(s, z):
    """[n][64][kv_heads][groups] -> the pages' words [n][kv_heads][groups][64]."""
    w = (s.view(torch.int32) & -0x10000) | ((z.view(torch.int32) >> 16) & 0xFFFF)
    return w.permute(0, 2, 3, 1).contiguous()


def _of_params(w):
    """The pages' words [n][kv_heads][groups][64] -> s, z [n][64][kv_heads][groups]."""
    w = w.permute(0, 3, 1, 2).contiguous()
    return (w & -0x10000).view(torch.float32), (w << 16).view(torch.float32)


def _pack(k, v):
    """(codes [n][64][kv_heads][head_dim], s, z) of K and of V -> pages [n][kv_heads][72 head_dim]."""
    n, _, kvh, d = k[0].shape
    half = min(d, 128)
    kc = k[0].view(n, 64, kvh, d // half, half // 32, 4, 4, 2).permute(0, 2, 3, 1, 5, 4, 6, 7)
    vc = v[0].view(n, 2, 2, 2, 4, 2, kvh, d // 32, 4, 8).permute(0, 6, 1, 7, 9, 4, 8, 5, 2, 3)
    parts = [kc[..., 0] | (kc[..., 1] << 4), _to_params(k[1], k[2]).view(torch.uint8),
             vc[..., 0] | (vc[..., 1] << 4), _to_params(v[1], v[2]).view(torch.uint8)]
    return torch.cat([p.reshape(n, kvh, -1) for p in parts], -1)


def _unpack_k(pages, d):
    n, kvh = pages.shape[:2]
    half = min(d, 128)
    b = pages[..., :32 * d].reshape(n, kvh, d // half, 64, 4, half // 32, 4)
    c = torch.stack([b & 15, b >> 4], -1).permute(0, 3, 1, 2, 5, 4, 6, 7).reshape(n, 64, kvh, d)
    return (c, *_of_params(pages[..., 32 * d:36 * d].contiguous().view(torch.int32).view(n, kvh, d // 64, 64)))


def _unpack_v(pages, d):
    n, kvh = pages.shape[:2]
    b = pages[..., 36 * d:68 * d].reshape(n, kvh, 2, d // 32, 8, 4, 4, 2, 2)
    c = torch.stack([b & 15, b >> 4], -1).permute(0, 2, 8, 9, 5, 7, 1, 3, 6, 4).reshape(n, 64, kvh, d)
    return (c, *_of_params(pages[..., 68 * d:].contiguous().view(torch.int32).view(n, kvh, d // 64, 64)))


def _values(c, s, z):
    """codes and parameters -> f32 [n][64][kv_heads][head_dim]."""
    x = c.float().unflatten(-1, (-1, 64))
    return x.sub_(8.0).mul_(s[..., None]).add_(z[..., None]).flatten(-2)


def _row_places(st):
    """Each row's page and slot."""
    r = torch.arange(st["rows"], device=st["pos"].device)
    seq = torch.searchsorted(st["cu_rows"][1:].long(), r, right=True)
    p = st["pos"].long()[seq] + r - st["cu_rows"].long()[seq]
    return st["table"].long()[seq, p // PAGE], p % PAGE


def _plain_store(st):
    d = st["head_dim"]
    page, slot = _row_places(st)
    pages, at = torch.unique_consecutive(page, return_inverse=True)
    held = st["pool"][pages]
    new = []
    for old, x in ((_unpack_k(held, d), st["k"]), (_unpack_v(held, d), st["v"])):
        new.append(tuple(o.index_put((at, slot), q) for o, q in zip(old, _quantise(x.float()))))
    st["pool"][pages] = _pack(*new)


def _plain_load(st):
    d, dtype = st["head_dim"], st["dtype"]
    page, slot = _row_places(st)
    pages, at = torch.unique_consecutive(page, return_inverse=True)
    held = st["pool"][pages]
    return tuple(_values(*f(held, d))[at, slot].to(dtype) for f in (_unpack_k, _unpack_v))


def _plain_attention(st):
    d, q, w = st["head_dim"], st["q"], st["window"]
    rows, heads, _ = q.shape
    seqs, kvh = st["table"].shape[0], st["pool"].shape[1]
    pos, cu = st["pos"].long(), st["cu_rows"].long()
    n = cu[1:] - cu[:-1]
    # the pages that a row of the sequence sees, from its first one
    first = ((pos - w + 1).clamp_min(0) if w else torch.zeros_like(pos)) // PAGE
    page = (first[:, None] + torch.arange(st["span"], device=q.device)).clamp_max(st["table"].shape[1] - 1)
    held = st["pool"][st["table"].long().gather(1, page).flatten()]
    # rows padded to the longest sequence's: [seqs][kv_heads][rows x group][d]
    at = torch.arange(st["most_rows"], device=q.device)
    src = (cu[:-1, None] + at).clamp_max(rows - 1)
    x = q[src].float().view(seqs, -1, kvh, heads // kvh, d).permute(0, 2, 1, 3, 4).flatten(2, 3)
    k = _values(*_unpack_k(held, d)).view(seqs, -1, kvh, d).permute(0, 2, 3, 1)
    scores = torch.matmul(x, k).mul_(st["scale"]).unflatten(2, (-1, heads // kvh))
    del k
    t = (pos[:, None] + at)[:, :, None]
    p = (first * PAGE)[:, None, None] + torch.arange(scores.shape[-1], device=q.device)
    see = p <= t if not w else (p <= t) & (p > t - w)
    scores.masked_fill_(~see[:, None, :, None, :], -math.inf)
    prob = scores.sub_(scores.amax(-1, keepdim=True)).exp_()
    total = prob.sum(-1, keepdim=True)
    v = _values(*_unpack_v(held, d)).view(seqs, -1, kvh, d).permute(0, 2, 1, 3)
    o = torch.matmul(prob.flatten(2, 3), v).unflatten(2, (-1, heads // kvh)).div_(total)
    o = o.permute(0, 2, 1, 3, 4).reshape(seqs, -1, heads, d)
    return o[at < n[:, None]].to(q.dtype)


# ---------------------------------------------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------------------------------------------

def _keys_values(case, rows, gen):
    """Keys as a per-head norm leaves them, with a few channels louder than the rest and an offset; plain values."""
    shape = (rows, case["kv_heads"], case["head_dim"])
    k = torch.randn(shape, generator=gen, device="cuda")
    k[..., ::37] *= 3.0
    k = k + 0.5 * torch.randn(shape[1:], generator=gen, device="cuda")
    k = k / k.norm(dim=-1, keepdim=True)
    return k, torch.randn(shape, generator=gen, device="cuda")


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rows, pos = _plan(case)
    seqs, kvh, d, heads = case["seqs"], case["kv_heads"], case["head_dim"], case["heads"]
    dtype = DTYPES[case["dtype"]]
    total, most = sum(rows), -(-case["length"] // PAGE)
    pages = seqs * most
    st = dict(op=case["op"], head_dim=d, dtype=dtype, window=case["window"], rows=total, most_rows=max(rows))
    # the sequences' pages lie anywhere in the pool
    st["table"] = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32).view(seqs, most)
    st["pos"] = torch.tensor(pos, dtype=torch.int32, device="cuda")
    st["cu_rows"] = torch.tensor([0] + rows, device="cuda").cumsum(0).to(torch.int32)
    st["pool"] = torch.zeros((pages, kvh, 72 * d), dtype=torch.uint8, device="cuda")
    if case["op"] == "store":
        k, v = _keys_values(case, total, gen)
        st["k"], st["v"] = k.to(dtype), v.to(dtype)
        return st
    step = max(1, (1 << 27) // (PAGE * kvh * d))
    for a in range(0, pages, step):
        n = min(step, pages - a)
        kv = [x.view(n, PAGE, kvh, d) for x in _keys_values(case, n * PAGE, gen)]
        st["pool"][a:a + n] = _pack(*[_quantise(x) for x in kv])
    if case["op"] == "attention":
        # queries whose scores spread by about 4 over the unit keys, as a trained q scale gives
        q = torch.randn((total, heads, d), generator=gen, device="cuda")
        st["q"] = (q / q.norm(dim=-1, keepdim=True) * 6.0).to(dtype)
        st["scale"] = 0.75 * math.sqrt(d)
        w = case["window"]
        first = [max(0, p - w + 1) // PAGE if w else 0 for p in pos]
        st["span"] = max(-(-(p + n) // PAGE) - f for p, n, f in zip(pos, rows, first))
    return st


def run(st):
    if own:
        x = importlib.import_module("xtier-go_b200")
        where = (st["table"], st["pos"], st["cu_rows"])
        if st["op"] == "attention":
            return x.kv4_attention(st["q"], st["pool"], *where, scale=st["scale"], window=st["window"])
        if st["op"] == "store":
            x.kv4_store(st["pool"], st["k"], st["v"], *where)
        return x.kv4_load(st["pool"], *where, rows=st["rows"], dtype=st["dtype"])
    if st["op"] == "attention":
        return _plain_attention(st)
    if st["op"] == "store":
        _plain_store(st)
    return _plain_load(st)


# ---------------------------------------------------------------------------------------------------------------
# From the definition, in 64 bits
# ---------------------------------------------------------------------------------------------------------------

def _exact_places(d):
    """For every (slot, head dim) of a page: the word and the shift of K's and of V's code, and the parameter word."""
    slot, dim = np.meshgrid(np.arange(64), np.arange(d), indexing="ij")
    h = min(d, 128)
    kw = ((dim // h * 64 + slot) * 4 + dim % 32 // 8) * (h // 32) + dim % h // 32
    ks = 4 * (dim % 8)
    s32 = slot % 32
    vw = (((slot // 32 * (d // 32) + dim // 32) * 8 + dim % 8) * 4 + s32 % 8 // 2) * 4 + dim % 32 // 8
    vs = 4 * (s32 // 8 + 4 * (s32 % 2))
    par = dim // 64 * 64 + slot
    return [(kw, ks, 8 * d + par), (9 * d + vw, vs, 17 * d + par)]


def _exact_page_values(pages, d):
    """K and V of pages [n][kv_heads][72 d] as 64-bit values [n][64][kv_heads][d]."""
    words = pages.contiguous().view(torch.int32).long() & 0xFFFFFFFF
    out = []
    for where in _exact_places(d):
        word, shift, par = (torch.from_numpy(x).to(pages.device) for x in where)
        code = (words[..., word] >> shift) & 15
        w = words[..., par]
        s = (w >> 16 << 16).int().view(torch.float32).double()
        z = ((w & 0xFFFF) << 16).int().view(torch.float32).double()
        out.append(((code - 8) * s + z).permute(0, 2, 1, 3))
    return out


def _exact_rounded(x, way):
    m, e = np.frexp(x.astype(np.float64))
    return np.ldexp(way(m * 256) / 256, e)


def _exact_row_values(x):
    """What rows [rows][kv_heads][d] stand for once quantised. The codes, scales and offsets are whole numbers and bf16
    numbers that the definition's f32 steps fix bit by bit; the values they stand for are taken in 64 bits."""
    g = x.reshape(*x.shape[:-1], -1, 64).astype(np.float32)
    lo, hi = g.min(-1), g.max(-1)
    s = _exact_rounded((hi - lo) * np.float32(1 / 15), np.ceil)
    s = np.maximum(s, 2.0 ** -100).astype(np.float32)
    z = _exact_rounded(lo + np.float32(8) * s, np.rint).astype(np.float32)
    c = np.rint((g - z[..., None]) * (np.float32(1) / s)[..., None]).clip(-8, 7)
    return (c.astype(np.float64) * s[..., None] + z[..., None].astype(np.float64)).reshape(x.shape)


def exact(case, seed):
    st = prepare(case, seed)
    rows, pos = _plan(case)
    d, kvh, heads, w = case["head_dim"], case["kv_heads"], case["heads"], case["window"]
    if case["op"] == "store":
        return tuple(_exact_row_values(st[n].float().cpu().numpy()) for n in ("k", "v"))
    outs, at = [], 0
    for i, (n, p) in enumerate(zip(rows, pos)):
        first = p // PAGE if case["op"] == "load" else max(0, p - w + 1) // PAGE if w else 0
        last = -(-(p + n) // PAGE)
        k, v = (x.reshape(-1, kvh, d)[:p + n - first * PAGE]
                for x in _exact_page_values(st["pool"][st["table"][i, first:last].long()], d))
        if case["op"] == "load":
            outs.append((k[p - first * PAGE:], v[p - first * PAGE:]))
            continue
        q = st["q"][at:at + n].double().view(n, kvh, heads // kvh, d)
        at += n
        key = torch.arange(first * PAGE, p + n, device="cuda")
        row = torch.arange(p, p + n, device="cuda")[:, None]
        hide = (key > row) | (key <= row - w) if w else key > row
        a = torch.einsum("nkgd,pkd->kgnp", q, k) * st["scale"]
        a = torch.softmax(a.masked_fill(hide, -math.inf), -1)
        outs.append(torch.einsum("kgnp,pkd->nkgd", a, v).reshape(n, heads, d))
    if case["op"] == "load":
        return tuple(torch.cat([o[j] for o in outs]) for j in (0, 1))
    return torch.cat(outs)
