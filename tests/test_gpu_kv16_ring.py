"""GPU: attention over the 16-bit caches where a CTA brings many more chunks than its ring holds, in parts of one chunk and of
many, for every kernel (head dims, row block, type). Sequences share pages that are only read, so that a small pool gives every
CTA several turns; a reference is worked out once for each kind of sequence."""
import math

import pytest
import torch

import kv16_ref as R
from kv16_cases import BF16, F16, ints, normal
from test_gpu_kv16_long import SHAPES

pytestmark = pytest.mark.gpu

SLOTS = 12   # of the longest ring, two a chunk


@pytest.mark.parametrize("window", [0, 300])
@pytest.mark.parametrize("dtype,page", [(BF16, 64), (F16, 16)])
@pytest.mark.parametrize("d,dv,latent,heads,rows", SHAPES)
def test_many_parts(xtg, cuda, d, dv, latent, heads, rows, dtype, page, window):
    gen = torch.Generator(device="cuda").manual_seed(d + heads + window)
    kvh, pos = 1 if latent else 2, [1290, 70, 0, 639]
    kinds, width = len(pos), 1408 // page
    heads *= kvh   # the row blocks of SHAPES
    table = torch.stack([torch.randperm(width, generator=gen, device="cuda") for _ in pos]).int()
    table[0, 512 // page:640 // page] = -1   # a chunk that is not there, and half of one
    table[3, 576 // page:640 // page] = -1
    k = normal(gen, width, kvh, page, d, dtype=dtype)
    v = k[..., :dv] if latent else normal(gen, width, kvh, page, dv, dtype=dtype)
    q = normal(gen, kinds * rows, heads, d, dtype=dtype)
    scale = 1.5 / math.sqrt(d)
    cu = torch.arange(kinds + 1, dtype=torch.int32, device="cuda") * rows
    ref = R.attention(q, k, v, table, ints(pos), cu, scale, window)
    tol = R.tolerance(ref, dtype, d, max(pos) + rows)
    shape = (kinds, rows, heads, dv)
    want, tol = ref[0].view(shape), tol.view(shape)
    # chunks of a sequence of each kind; a part's start counts up to 4 more where the work is shared out
    size = 128 if d <= 192 else 64
    first = [max(0, p - window + 1) // size if window else 0 for p in pos]
    chunks = sum(-(-(p + rows) // size) - f for p, f in zip(pos, first))
    ctas = 2 * torch.cuda.get_device_properties(0).multi_processor_count
    seqs = kinds * -(-3 * SLOTS // 2 * ctas // (kvh * (chunks - kinds * 4 if chunks > kinds * 8 else chunks // 2)))
    kind = torch.arange(seqs, device="cuda") % kinds
    x = q.view(kinds, rows, heads, d)[kind].flatten(0, 1)
    err = ints([0])
    where = (table[kind].contiguous(), ints(pos)[kind].contiguous(), ints(range(0, seqs * rows + 1, rows)))
    if latent:
        got = xtg.latent_attention(x[..., :dv], x[..., dv:], k[:, 0], *where, scale=scale, window=window, err=err)
    else:
        got = xtg.kv16_attention(x, k, v, *where, scale=scale, window=window, err=err)
    xtg.kv4_check(err)
    off = (got.view(-1, *shape) - want).abs() / tol
    assert off.max() <= 1, float(off.max())   # NaN fails too
