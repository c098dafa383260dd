"""What is measured of the 16-bit paged caches: keys and values appended with their rotation, attention over them, and the
same for a cache of latent vectors.

`listed()` names the cases, `draw()` gives more of the same ranges, `prepare()` makes what a server holds before the
call, `run()` is one pass (`own`: through the framework's entry points, else in plain torch operations in 32 bits),
`exact()` the same results from the operators' definition in 64 bits, `work()` the bytes and operations that a pass
cannot do without.

The caches: `k_pool` [pages][kv_heads][page][head_dim] and `v_pool` [pages][kv_heads][page][v_dim], or one `pool`
[pages][page][latent + rotary] of latent vectors with a shared rotated key behind each. Position p of sequence i is slot
p % page of page table[i][p // page], a negative entry holds nothing; the rows cu_rows[i] .. cu_rows[i + 1] - 1 of a call
stand at positions pos[i], pos[i] + 1, ...
"""
import importlib
import math
import random

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
ROTARY = 64   # rotated dims of a latent cache's key, and of keys of 192 (the last ones)


# ---------------------------------------------------------------------------------------------------------------
# The cases
# ---------------------------------------------------------------------------------------------------------------

def _case(name, op, seqs, rows, length, heads, kv_heads, head_dim, v_dim, dtype, rows_dtype=None, page=64, window=0,
          ragged=False, interleaved=False):
    c = dict(op=op, seqs=seqs, rows=rows, length=length, heads=heads, kv_heads=kv_heads, head_dim=head_dim,
             v_dim=v_dim, dtype=dtype, rows_dtype=rows_dtype or dtype, page=page, window=window, ragged=ragged,
             interleaved=interleaved)
    return dict(c, name=name) if name else c


def listed():
    """`length` counts a sequence's positions after the call, `rows` those of the call (the last ones). For a latent cache
    head_dim is latent + 64 rotated dims, v_dim the latent's."""
    return [
        # the smallest call: one conversation's next token, in the activations' own type
        _case("append_1x1", "append", 1, 1, 4096, 24, 6, 128, 128, "bf16", "f32"),
        # whole prompts of several conversations, the wider heads
        _case("append_8x4096", "append", 8, 4096, 8192, 16, 4, 256, 256, "f16", ragged=True),
        # a verify round of a latent model's conversations
        _case("latent_append_64x4", "latent_append", 64, 4, 16384, 32, 1, 576, 512, "bf16", ragged=True),
        # a latent model's prompts, far positions
        _case("latent_append_4x4096", "latent_append", 4, 4096, 131072, 128, 1, 576, 512, "bf16", interleaved=True),
        # one token of one conversation: latency
        _case("decode_1x4096", "attention", 1, 1, 4096, 24, 6, 128, 128, "bf16"),
        # a server's batch, every sequence at its own length: bandwidth
        _case("decode_64x32768", "attention", 64, 1, 32768, 24, 6, 128, 128, "bf16", ragged=True),
        # the sliding layers of a batched verify round, small pages
        _case("verify_64x8_window", "attention", 64, 8, 16384, 24, 6, 128, 128, "f16", page=16, window=1024, ragged=True),
        # a prompt chunk over what is already cached, the wider heads, lengths that end inside a page
        _case("chunk_1x501_at_16383", "attention", 1, 501, 16383, 16, 4, 256, 256, "f16"),
        # a latent model's prompts in the expanded form: keys of 128 + 64, values of 128, each head its own
        _case("expanded_4x2048", "attention", 4, 2048, 2048, 16, 16, 192, 128, "bf16", ragged=True),
        # one token of one conversation of a latent model
        _case("latent_1x1_at_8192", "latent_attention", 1, 1, 8192, 32, 1, 576, 512, "bf16"),
        # verify steps of a smaller latent model
        _case("latent_16x4_at_4095", "latent_attention", 16, 4, 4095, 16, 1, 320, 256, "f16", ragged=True),
        # a server's batch of a latent model with many heads: tensor cores and bandwidth alike
        _case("latent_64x1_at_16384", "latent_attention", 64, 1, 16384, 128, 1, 576, 512, "bf16", ragged=True),
    ]


# q heads, KV heads, dims of keys and of values: grouped, one each, one for all, the expanded form
_HEADS = [(24, 6, 128, 128), (16, 4, 256, 256), (8, 2, 128, 128), (8, 8, 64, 64), (12, 1, 128, 128), (16, 16, 192, 128)]


def draw(rng):
    most = max(_cost(c) for c in listed())

    def log(a, b):
        return int(round(math.exp(rng.uniform(math.log(a), math.log(b)))))

    while True:
        op = rng.choice(["append", "latent_append", "attention", "attention", "latent_attention"])
        if op.startswith("latent"):
            latent = rng.choice([256, 512])
            shape = (rng.choice([8, 16, 32, 64, 128]), 1, latent + ROTARY, latent)
        else:
            shape = rng.choice(_HEADS)
        dtype = rng.choice(["bf16", "f16"])
        seqs, length, window = log(1, 64), log(40, 131072), 0
        if op.endswith("append"):
            rows = min(log(1, 8192), length)
            rows_dtype = rng.choice([dtype, dtype, "f32"])
        else:
            rows = min(log(1, 1024 if op == "attention" else 16), length)
            rows_dtype = dtype
            window = rng.choice([0, 0, log(16, 2048)]) if op == "attention" else 0
        c = _case(None, op, seqs, rows, length, *shape, dtype, rows_dtype, rng.choice([16, 64, 64, 128]), window,
                  rng.random() < 0.7, rng.random() < 0.3)
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
            if n > 8:   # a verify step's rows are the same for all
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
    d, dv, kvh, heads = case["head_dim"], case["v_dim"], case["kv_heads"], case["heads"]
    size = DTYPES[case["rows_dtype"]].itemsize
    rows = sum(_plan(case)[0])
    if case["op"] == "append":   # k, v and q read, k, v and the rotated q written
        return {"bytes": rows * (kvh * (d + dv) + heads * d) * (size + 2), "flops": 3 * rows * (kvh + heads) * d}
    if case["op"] == "latent_append":   # the latent vector, its key and the q heads' rotated dims
        return {"bytes": rows * (d + heads * ROTARY) * (size + 2), "flops": 3 * rows * (1 + heads) * ROTARY}
    held, pairs = _seen(case)
    slot = kvh * (d if case["op"] == "latent_attention" else d + dv) * 2
    return {"bytes": held * slot + rows * heads * (d + dv) * 2, "flops": 2 * pairs * heads * (d + dv)}


def _cost(case):
    w = work(case)
    return max(w["bytes"], w["flops"] / 100)


# ---------------------------------------------------------------------------------------------------------------
# The plain form
# ---------------------------------------------------------------------------------------------------------------

def _row_places(st):
    """Each row's position, page and slot."""
    r = torch.arange(st["rows"], device=st["pos"].device)
    seq = torch.searchsorted(st["cu_rows"][1:].long(), r, right=True)
    p = st["pos"].long()[seq] + r - st["cu_rows"].long()[seq]
    return p, st["table"].long()[seq, p // st["page"]], p % st["page"]


def _rotated(x, p, freq, interleaved):
    """x [rows][heads][2 len(freq)] turned by its positions, f32; the angles in 64 bits."""
    angle = p.double()[:, None] * freq.double()
    c, s = angle.cos().float()[:, None], angle.sin().float()[:, None]
    half = freq.numel()
    x = x.float()
    a, b = (x[..., 0::2], x[..., 1::2]) if interleaved else (x[..., :half], x[..., half:])
    y = (a * c - b * s, b * c + a * s)
    return torch.stack(y, -1).flatten(-2) if interleaved else torch.cat(y, -1)


def _plain_append(st):
    p, page, slot = _row_places(st)
    first, dtype, turn = st["first"], st["dtype"], (p, st["freq"], st["interleaved"])
    q = torch.cat([st["q"][..., :first].float(), _rotated(st["q"][..., first:], *turn)], -1).to(dtype)
    k = torch.cat([st["k"][..., :first].float(), _rotated(st["k"][..., first:], *turn)], -1).to(dtype)
    st["k_pool"][page, :, slot] = k
    st["v_pool"][page, :, slot] = st["v"].to(dtype)
    return q, st["k_pool"], st["v_pool"]


def _plain_latent_append(st):
    p, page, slot = _row_places(st)
    dtype, turn = st["dtype"], (p, st["freq"], st["interleaved"])
    q = _rotated(st["q"], *turn).to(dtype)
    k = _rotated(st["k"][:, None], *turn)[:, 0]
    st["pool"][page, slot] = torch.cat([st["c"].float(), k], -1).to(dtype)
    return q, st["pool"]


def _plain_attention(st):
    """Some sequences at a time, as many as leave the scores and the gathered keys small."""
    w, page, latent = st["window"], st["page"], "pool" in st
    q = torch.cat([st["q"], st["q_rot"]], -1) if latent else st["q"]
    rows, heads, d = q.shape
    k_pool = st["pool"][:, None] if latent else st["k_pool"]
    v_pool = k_pool[..., :d - ROTARY] if latent else st["v_pool"]
    kvh, dv = k_pool.shape[1], v_pool.shape[3]
    pos, cu = st["pos"].long(), st["cu_rows"].long()
    n = cu[1:] - cu[:-1]
    # the pages that a row of a sequence sees, from its first one
    first = ((pos - w + 1).clamp_min(0) if w else torch.zeros_like(pos)) // page
    at = torch.arange(st["most_rows"], device=q.device)
    key = torch.arange(st["span"] * page, device=q.device)
    index = (first[:, None] + key[::page] // page).clamp_max(st["table"].shape[1] - 1)
    src = (cu[:-1, None] + at).clamp_max(rows - 1)
    t = pos[:, None] + at
    p = (first * page)[:, None] + key
    out = torch.empty((rows, heads, dv), dtype=q.dtype, device=q.device)
    each = 4 * key.numel() * (kvh * (d + dv) + 2 * heads * at.numel())
    step = max(1, (8 << 30) // each)
    for a in range(0, len(n), step):
        s = slice(a, a + step)
        held = st["table"].long()[s].gather(1, index[s])
        # rows padded to the longest sequence's: [seqs][kv_heads][rows x group][d]
        x = q[src[s]].float().unflatten(2, (kvh, -1)).permute(0, 2, 1, 3, 4).flatten(2, 3)
        k = k_pool[held].float().permute(0, 2, 4, 1, 3).flatten(3)
        scores = torch.matmul(x, k).mul_(st["scale"]).unflatten(2, (-1, heads // kvh))
        see = p[s, None, :] <= t[s, :, None]
        if w:
            see &= p[s, None, :] > t[s, :, None] - w
        scores.masked_fill_(~see[:, None, :, None, :], -math.inf)
        prob = scores.sub_(scores.amax(-1, keepdim=True)).exp_()
        total = prob.sum(-1, keepdim=True)
        v = v_pool[held].float().permute(0, 2, 1, 3, 4).flatten(2, 3)
        o = torch.matmul(prob.flatten(2, 3), v).unflatten(2, (-1, heads // kvh)).div_(total)
        o = o.permute(0, 2, 1, 3, 4).flatten(2, 3)[at < n[s, None]]
        first_row = int(st["starts"][a])
        out[first_row:first_row + len(o)] = o.to(q.dtype)
    return out


# ---------------------------------------------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------------------------------------------

def _keys(shape, gen):
    """Keys as a per-head norm leaves them, a few channels louder than the rest."""
    k = torch.randn(shape, generator=gen, device="cuda")
    k[..., ::37] *= 3.0
    return k / k.norm(dim=-1, keepdim=True)


def _fill(pool, gen, make):
    step = max(1, (1 << 27) // pool[0].numel())
    for a in range(0, len(pool), step):
        b = pool[a:a + step]
        b.copy_(make(b.shape, gen))


def _values(shape, gen):
    return torch.randn(shape, generator=gen, device="cuda")


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rows, pos = _plan(case)
    op, seqs, page, w = case["op"], case["seqs"], case["page"], case["window"]
    d, dv, kvh, heads = case["head_dim"], case["v_dim"], case["kv_heads"], case["heads"]
    dtype, rows_dtype = DTYPES[case["dtype"]], DTYPES[case["rows_dtype"]]
    total, latent, append = sum(rows), op.startswith("latent"), op.endswith("append")
    st = dict(op=op, dtype=dtype, window=w, rows=total, most_rows=max(rows), page=page,
              interleaved=case["interleaved"], starts=[sum(rows[:i]) for i in range(seqs)])
    # the pages that the call meets lie anywhere in the pool; what lies before them has been given back, or is not looked at
    first = [(p if append else max(0, p - w + 1) if w else 0) // page for p in pos]
    last = [-(-(p + n) // page) for p, n in zip(pos, rows)]
    st["span"] = max(b - a for a, b in zip(first, last))
    pages = sum(b - a for a, b in zip(first, last))
    order = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32)
    st["table"] = torch.full((seqs, max(last)), -1, dtype=torch.int32, device="cuda")
    at = 0
    for i, (a, b) in enumerate(zip(first, last)):
        st["table"][i, a:b] = order[at:at + b - a]
        if not append:   # the plain form gathers a full span for every sequence; what it masks may be any page
            st["table"][i, b:] = order[at]
        at += b - a
    st["pos"] = torch.tensor(pos, dtype=torch.int32, device="cuda")
    st["cu_rows"] = torch.tensor([0] + rows, device="cuda").cumsum(0).to(torch.int32)
    rotary = ROTARY if latent or d == 192 else d
    st["first"] = 0 if latent else d - rotary
    if append:
        st["freq"] = (10000.0 ** (-torch.arange(0, rotary, 2, dtype=torch.float64) / rotary)).float().cuda()
    if latent:
        st["pool"] = torch.empty((pages, page, d), dtype=dtype, device="cuda")
        _fill(st["pool"], gen, _values)
        if append:
            st["c"] = _values((total, dv), gen).to(rows_dtype)
            st["k"] = _values((total, ROTARY), gen).to(rows_dtype)
            st["q"] = _values((total, heads, ROTARY), gen).to(rows_dtype)
            return st
        # scores that spread by about 2.5
        q = _values((total, heads, d), gen).to(dtype)
        st["q"], st["q_rot"] = q[..., :dv].contiguous(), q[..., dv:].contiguous()
        st["scale"] = 2.5 / math.sqrt(d)
        return st
    st["k_pool"] = torch.empty((pages, kvh, page, d), dtype=dtype, device="cuda")
    st["v_pool"] = torch.empty((pages, kvh, page, dv), dtype=dtype, device="cuda")
    _fill(st["k_pool"], gen, _keys)
    _fill(st["v_pool"], gen, _values)
    # queries whose scores spread by about 4 over the unit keys, as a trained q scale gives
    q = _values((total, heads, d), gen)
    st["q"] = (q / q.norm(dim=-1, keepdim=True) * 6.0).to(rows_dtype)
    st["scale"] = 0.75 * math.sqrt(d)
    if append:
        st["k"] = _keys((total, kvh, d), gen).to(rows_dtype)
        st["v"] = _values((total, kvh, dv), gen).to(rows_dtype)
    return st


def run(st):
    op = st["op"]
    if own:
        x = importlib.import_module("xtier-go_b200")
        where = (st["table"], st["pos"], st["cu_rows"])
        if op == "attention":
            return x.kv16_attention(st["q"], st["k_pool"], st["v_pool"], *where, scale=st["scale"], window=st["window"])
        if op == "latent_attention":
            return x.latent_attention(st["q"], st["q_rot"], st["pool"], *where, scale=st["scale"])
        if op == "append":
            q = x.kv16_append(st["k_pool"], st["v_pool"], st["k"], st["v"], *where, freq=st["freq"], q=st["q"],
                              first=st["first"], interleaved=st["interleaved"])
            return q, st["k_pool"], st["v_pool"]
        q = x.latent_append(st["pool"], st["c"], st["k"], *where, freq=st["freq"], q=st["q"],
                            interleaved=st["interleaved"])
        return q, st["pool"]
    if op == "append":
        return _plain_append(st)
    if op == "latent_append":
        return _plain_latent_append(st)
    return _plain_attention(st)


# ---------------------------------------------------------------------------------------------------------------
# From the definition, in 64 bits
# ---------------------------------------------------------------------------------------------------------------

def _exact_turn(x, pos, freq, interleaved):
    """Pairs (a, b) as complex numbers a + i b times e^(i pos freq), per sequence's rows x [n][heads][2 m]."""
    n, heads, r = x.shape
    x = x.double()
    pair = x.view(n, heads, r // 2, 2) if interleaved else x.view(n, heads, 2, r // 2).transpose(2, 3)
    z = torch.view_as_complex(pair.contiguous())
    angle = torch.outer(torch.arange(pos, pos + n, device=x.device, dtype=torch.float64), freq.double())
    y = torch.view_as_real(z * torch.polar(torch.ones_like(angle), angle)[:, None])
    return (y if interleaved else y.transpose(2, 3)).reshape(n, heads, r)


def _exact_append(case, st, rows, pos):
    page, dv, latent = case["page"], case["v_dim"], case["op"] == "latent_append"
    if latent:
        pools = [st["pool"].double()[:, None]]
        parts = [torch.cat([st["c"], st["k"]], -1)[:, None]]
    else:
        pools = [st["k_pool"].double(), st["v_pool"].double()]
        parts = [st["k"], st["v"]]
    first = dv if latent else st["first"]
    q_first = 0 if latent else first
    qs, at = [], 0
    for i, (n, p) in enumerate(zip(rows, pos)):
        q = st["q"][at:at + n].double()
        q[..., q_first:] = _exact_turn(q[..., q_first:], p, st["freq"], case["interleaved"])
        qs.append(q)
        for j, (pool, part) in enumerate(zip(pools, parts)):
            x = part[at:at + n].double()
            if j == 0:
                x[..., first:] = _exact_turn(x[..., first:], p, st["freq"], case["interleaved"])
            done = 0
            while done < n:   # a page at a time
                slot = (p + done) % page
                m = min(page - slot, n - done)
                pool[int(st["table"][i, (p + done) // page]), :, slot:slot + m] = x[done:done + m].transpose(0, 1)
                done += m
        at += n
    if latent:
        return torch.cat(qs), pools[0][:, 0]
    return torch.cat(qs), pools[0], pools[1]


def exact(case, seed):
    st = prepare(case, seed)
    rows, pos = _plan(case)
    if case["op"].endswith("append"):
        st["table"] = st["table"].cpu()
        return _exact_append(case, st, rows, pos)
    page, dv, heads, w = case["page"], case["v_dim"], case["heads"], case["window"]
    kvh = case["kv_heads"]
    outs, at = [], 0
    for i, (n, p) in enumerate(zip(rows, pos)):
        low = max(0, p - w + 1) // page if w else 0
        held = st["table"][i, low:-(-(p + n) // page)].long()
        if case["op"] == "latent_attention":
            x = st["pool"][held].reshape(-1, 1, case["head_dim"])[:p + n - low * page]
            k, v = x, x[..., :dv]
            q = torch.cat([st["q"][at:at + n], st["q_rot"][at:at + n]], -1)
        else:
            k, v = (st[s][held].transpose(1, 2).flatten(0, 1)[:p + n - low * page] for s in ("k_pool", "v_pool"))
            q = st["q"][at:at + n]
        at += n
        key = torch.arange(low * page, p + n, device="cuda")
        row = torch.arange(p, p + n, device="cuda")[:, None]
        hide = (key > row) | (key <= row - w) if w else key > row
        out = torch.empty((n, heads, dv), dtype=torch.float64, device="cuda")
        for h in range(kvh):
            g = slice(h * (heads // kvh), (h + 1) * (heads // kvh))
            step = max(1, (1 << 28) // (len(key) * (heads // kvh)))
            for r in range(0, n, step):
                s = torch.einsum("ngd,pd->ngp", q[r:r + step, g].double(), k[:, h].double()) * st["scale"]
                s = torch.softmax(s.masked_fill(hide[r:r + step, None], -math.inf), -1)
                out[r:r + step, g] = torch.einsum("ngp,pd->ngd", s, v[:, h].double())
        outs.append(out)
    return torch.cat(outs)
