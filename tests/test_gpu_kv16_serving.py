"""GPU: append and attention together, as a server's steps run them: prompts in chunks, then a captured step of several
conversations whose pages are taken as they grow and given back, against plain arithmetic from the rows themselves."""
import math

import pytest
import torch

import kv16_ref as R
from kv16_cases import BF16, check, ints, normal

pytestmark = pytest.mark.gpu

HEADS, KVH, D, PAGE, WINDOW = 8, 2, 128, 16, 50


def test_conversations(xtg, cuda):
    gen = torch.Generator(device="cuda").manual_seed(1)
    prompts, steps = [37, 1, 70], 20
    seqs, width = len(prompts), 8
    freq = (10000.0 ** (-torch.arange(D // 2, dtype=torch.float64) / (D // 2))).float().cuda()
    free = list(range(40))
    pools = [xtg.kv16_pool(40, KVH, D, page=PAGE) for _ in range(2)]
    table = torch.full((seqs, width), -1, dtype=torch.int32)
    scale = 1 / math.sqrt(D)
    rows = [[normal(gen, n + steps, h, D, dtype=BF16) for h in (HEADS, KVH, KVH)] for n in prompts]   # q, k, v

    def take(i, upto):
        for j in range(-(-upto // PAGE)):
            if table[i, j] < 0 and (j + 1) * PAGE > upto - 1 - WINDOW - PAGE:
                table[i, j] = free.pop(0)

    def give_back(i, held):   # pages that no later row sees
        for j in range(max(0, (held - WINDOW) // PAGE)):
            if table[i, j] >= 0:
                free.append(int(table[i, j]))
                table[i, j] = -1

    def want(i, first, n):
        q, k, v = (x[:first + n] for x in rows[i])
        at = torch.arange(first + n, device="cuda")
        q, k = R.rotate(q, at, freq, False).to(BF16), R.rotate(k, at, freq, False).to(BF16)   # as the calls round them
        k, v = (x.transpose(0, 1)[None] for x in (k, v))
        one = torch.zeros(1, 1, dtype=torch.int32)
        # one page of everything
        ref = R.attention(q[first:], k, v, one, torch.tensor([first]), torch.tensor([0, n]), scale, WINDOW)
        tol = R.tolerance(ref, BF16, D, first + n)
        # a rotated value may round to the neighbour of the reference's: 2^-8 of q and of k in the scores, at most
        return ref[0], tol + ref[1] * 2 * 2.0 ** -8 * ref[2][..., None]

    d_table, d_pos, d_cu = torch.zeros(seqs, width, dtype=torch.int32, device="cuda"), ints([0] * seqs), ints(range(seqs + 1))
    # the prompts, in chunks of 32 rows
    for i, n in enumerate(prompts):
        for a in range(0, n, 32):
            m = min(32, n - a)
            take(i, a + m)
            where = (table[i:i + 1].cuda(), ints([a]), ints([0, m]))
            q, k, v = (x[a:a + m] for x in rows[i])
            q = xtg.kv16_append(*pools, k, v, *where, freq=freq, q=q)
            check(xtg.kv16_attention(q, *pools, *where, scale=scale, window=WINDOW), *want(i, a, m), f"prompt {i} from {a}")
            give_back(i, a + m)
    # the steps, captured once
    step = [torch.zeros(seqs, h, D, dtype=BF16, device="cuda") for h in (HEADS, KVH, KVH)]

    def run():
        q = xtg.kv16_append(*pools, step[1], step[2], d_table, d_pos, d_cu, freq=freq, q=step[0])
        return xtg.kv16_attention(q, *pools, d_table, d_pos, d_cu, scale=scale, window=WINDOW)
    side = torch.cuda.Stream()
    d_table.fill_(-1)   # the first run writes nothing
    with torch.cuda.stream(side):
        run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run()
    for t in range(steps):
        for i, n in enumerate(prompts):
            take(i, n + t + 1)
        d_table.copy_(table)
        d_pos.copy_(ints([n + t for n in prompts]))
        for x, j in zip(step, range(3)):
            x.copy_(torch.stack([rows[i][j][n + t] for i, n in enumerate(prompts)]))
        graph.replay()
        for i, n in enumerate(prompts):
            check(out[i:i + 1], *want(i, n + t, 1), f"step {t}, conversation {i}")
            give_back(i, n + t + 1)
