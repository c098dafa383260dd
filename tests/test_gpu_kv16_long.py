"""GPU: attention over the 16-bit caches in parts of 131072 positions, for every kernel (head dims, row block, type): what a sum
over positions loses must not grow with their number. The tables repeat a few pages, so that a reference is the softmax over
these with their positions counted."""
import math

import pytest
import torch

from kv16_cases import BF16, F16, ints, normal

pytestmark = pytest.mark.gpu

PAGE, PAGES, LENGTH, KINDS = 64, 8, 131072, 4
# (head_dim, v_dim, latent, q heads x rows of a sequence): blocks of 16, 32, 64 and 128 rows
SHAPES = ([(d, dv, False, *x) for d, dv in ((64, 64), (128, 128), (192, 128), (256, 256)) for x in ((4, 1), (5, 5), (12, 5), (25, 5))]
          + [(d + 64, d, True, *x) for d in (256, 512) for x in ((4, 1), (5, 5), (16, 4))])
SCALE = 0.05


def reference(q, k, v, table):
    """Rows q [kinds][rows][heads][d] at LENGTH - rows, ... over pages k, v [pages][page][d]: (out, sum_p w |v - out|), 64 bits."""
    kinds, rows = q.shape[:2]
    a = torch.einsum("crhd,psd->crhps", q.double(), k.double()) * SCALE
    out, spread = [], []
    for c in range(kinds):
        for r in range(rows):
            seen = LENGTH - rows + r + 1
            times = torch.bincount(table[c, :seen // PAGE].long(), minlength=PAGES).double()[:, None].repeat(1, PAGE)
            if seen % PAGE:
                times[int(table[c, seen // PAGE]), :seen % PAGE] += 1
            w = (a[c, r] - a[c, r].amax((-2, -1), keepdim=True)).exp() * times
            w /= w.sum((-2, -1), keepdim=True)
            out.append(torch.einsum("hps,psd->hd", w, v.double()))
            spread.append(torch.einsum("hps,hpsd->hd", w, (v.double() - out[-1][:, None, None]).abs()))
    shape = (kinds, rows, *out[0].shape)
    return torch.stack(out).view(shape), torch.stack(spread).view(shape)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("rise", [None, 3.0, -3.0])   # of the scores from a page's positions, all together, to the next's
@pytest.mark.parametrize("d,dv,latent,heads,rows", SHAPES)
def test_long_parts(xtg, cuda, d, dv, latent, heads, rows, rise, dtype):
    gen = torch.Generator(device="cuda").manual_seed(d + heads)
    # a dim's values are of one sign and of its own size: sums that only grow, outputs spread over the roundings
    size = torch.rand(dv, generator=gen, device="cuda") + 1
    size[1::2] *= -1
    v = (size * (0.5 + torch.rand(PAGES, PAGE, dv, generator=gen, device="cuda"))).to(dtype)
    k = torch.cat([v, normal(gen, PAGES, PAGE, 64, dtype=dtype)], -1) if latent else normal(gen, PAGES, PAGE, d, dtype=dtype)
    q = normal(gen, KINDS, rows, heads, d, dtype=dtype)
    if latent:
        q[..., :dv] *= 0.05   # scores of about +-1
    table = torch.stack([torch.randperm(LENGTH // PAGE, generator=gen, device="cuda") % PAGES for _ in range(KINDS)]).int()
    if rise:
        table = table.sort(-1).values
        q[..., -64] = 1
        k[..., -64] = (torch.arange(PAGES, device="cuda") * rise / SCALE)[:, None]
    # twice as many sequences as there can be CTAs: every CTA has whole sequences
    seqs = KINDS * -(-4 * torch.cuda.get_device_properties(0).multi_processor_count // KINDS)
    kind = torch.arange(seqs, device="cuda") % KINDS
    x = q[kind].flatten(0, 1)
    where = (table[kind].contiguous(), ints([LENGTH - rows] * seqs), ints(range(0, seqs * rows + 1, rows)))
    if latent:
        got = xtg.latent_attention(x[..., :dv], x[..., dv:], k, *where, scale=SCALE)
    else:
        got = xtg.kv16_attention(x, k[:, None], v[:, None], *where, scale=SCALE)
    got = got.view(-1, KINDS, rows, heads, dv).double()
    assert (got == got[:1]).all()
    want, spread = reference(q, k, v, table)
    off = got[0] - want
    # h: half a step. The output's rounding; the weights' (numerator and sum alike, so of the values' spread); the scores' sums
    # as kv16_ref.tolerance has them, of the spread; ex2 and factors. Sums over positions: the matrix unit adds 256 steps of 16
    # for f16, 1024 for bf16, each cut off up to four times (by 2^-23); these and the weights are then added in f32 (at most 32
    # and 1024 of them, 2^-24).
    h = torch.finfo(dtype).eps / 2
    steps = 256 if dtype == F16 else 1024
    sums = steps * 4 * 2.0 ** -23 + (32 + 1024) * 2.0 ** -24 + 2.0 ** -20
    score = SCALE * float(torch.einsum("crhd,psd->crhps", q.double().abs(), k.double().abs()).max())
    bound = h * want.abs() * (1 + 2.0 ** -8) + (2 * h + 2 * d * 2.0 ** -23 * score) * spread + sums * want.abs()
    assert (off.abs() <= bound).all(), float((off.abs() / bound).max())
    # On average the roundings cancel (a step is at most 2 h of a value: 2 h / sqrt(12) over the root of their number; four
    # times that). What is cut off does not: half of a unit each, which is at most 2^-24 of sums that grow from zero to their
    # value in so many steps.
    loss = float((off * want.sign() / want.abs()).mean())
    assert abs(loss) <= steps / 2 * 4 * 2.0 ** -24 + 4 * 2 * h / math.sqrt(12 * off.numel()), loss
