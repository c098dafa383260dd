"""Several conversations over one paged 4-bit key/value cache, as a server's attention layer uses it: prompts arrive in
chunks, then every step appends one token to each conversation; pages are taken from one pool as the conversations
grow, and given back when one ends or when a sliding window has passed them.

    python examples/kv4_serving.py [--device 0]

Each call's descriptor (page table, positions, row offsets) serves the store and the attention of its rows. The layer's
own projections are not the point here: seeded keys, values and queries stand for them. The result of every step is
compared with attention over the same keys and values unquantised in 32 bits, to show what 4 bits cost.
"""
import argparse
import importlib.util
import math
import os
import sys

import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def package():
    if "xtier_go_b200" not in sys.modules:
        pkg = os.path.join(ROOT, "xtier-go_b200")
        spec = importlib.util.spec_from_file_location("xtier_go_b200", os.path.join(pkg, "__init__.py"),
                                                      submodule_search_locations=[pkg])
        mod = importlib.util.module_from_spec(spec)
        sys.modules["xtier_go_b200"] = mod
        spec.loader.exec_module(mod)
    return sys.modules["xtier_go_b200"]


class PagedLayer:
    """One attention layer's cache for up to `seqs` conversations: the pool, the free pages and each conversation's table."""

    def __init__(self, x, seqs, pages, max_pages, kv_heads, head_dim, window=0):
        self.x, self.window = x, window
        self.pool = x.kv4_pool(pages, kv_heads, head_dim)
        self.err = torch.zeros(1, dtype=torch.int32, device="cuda")
        self.free = list(range(pages))
        self.table = torch.full((seqs, max_pages), -1, dtype=torch.int32)   # -1: nothing there
        self.length = [0] * seqs

    def step(self, rows, q, k, v, scale):
        """Append rows[i] tokens to conversation i (q, k, v hold them one conversation after another) and attend."""
        pos = torch.tensor(self.length, dtype=torch.int32)
        for i, n in enumerate(rows):
            for p in range(self.length[i] // self.x.KV4_PAGE, -(-(self.length[i] + n) // self.x.KV4_PAGE)):
                if n and self.table[i, p] < 0:
                    self.table[i, p] = self.free.pop()
            self.length[i] += n
        cu_rows = torch.tensor([0] + rows).cumsum(0).to(torch.int32)
        where = [t.cuda(non_blocking=True) for t in (self.table, pos, cu_rows)]
        self.x.kv4_store(self.pool, k, v, *where, err=self.err)
        out = self.x.kv4_attention(q, self.pool, *where, scale=scale, window=self.window, err=self.err)
        if self.window:   # pages that no later row sees
            for i, n in enumerate(self.length):
                for p in range(max(0, n - self.window) // self.x.KV4_PAGE):
                    self.give_back(i, p)
        return out

    def give_back(self, i, p):
        if self.table[i, p] >= 0:
            self.free.append(int(self.table[i, p]))
            self.table[i, p] = -1

    def end(self, i):
        for p in range(self.table.shape[1]):
            self.give_back(i, p)
        self.length[i] = 0


def plain(q, k, v, scale, window, pos):
    """Attention of one conversation's rows over its unquantised keys and values, in 32 bits."""
    n, heads, _ = q.shape
    group = heads // k.shape[1]
    k, v = (t.repeat_interleave(group, 1) for t in (k, v))
    s = torch.einsum("nhd,phd->hnp", q.float(), k) * scale
    p, t = torch.arange(k.shape[0], device=q.device), torch.arange(pos, pos + n, device=q.device)[:, None]
    s = s.masked_fill((p > t) | ((p <= t - window) if window else False), -math.inf)
    return torch.einsum("hnp,phd->nhd", torch.softmax(s, -1), v)


def serve(prompts=(700, 65, 1, 130), steps=24, chunk=64, heads=24, kv_heads=6, head_dim=128, window=0, seed=0):
    """The largest relative error of a step's rows against plain attention, the pages in use at the end."""
    x = package()
    gen = torch.Generator(device="cuda").manual_seed(seed)
    draw = lambda n, h: torch.randn((n, h, head_dim), generator=gen, device="cuda")
    seqs, scale = len(prompts), 1 / math.sqrt(head_dim)
    most = -(-(max(prompts) + 2 * steps) // x.KV4_PAGE)
    layer = PagedLayer(x, seqs, seqs * most, most, kv_heads, head_dim, window)
    held = [[torch.empty((0, kv_heads, head_dim), device="cuda")] * 2 for _ in prompts]
    left = list(prompts)
    worst = 0.0
    for step in range(steps):
        if step == steps // 2:   # one conversation ends, another takes its place
            layer.end(seqs - 1)
            held[-1], left[-1] = [held[-1][0][:0]] * 2, prompts[-1]
        rows = [min(chunk, n) or 1 for n in left]
        left = [max(0, n - r) for n, r in zip(left, rows)]
        total = sum(rows)
        q, k, v = draw(total, heads).bfloat16(), draw(total, kv_heads), draw(total, kv_heads)
        pos = list(layer.length)
        out = layer.step(rows, q, k.bfloat16(), v.bfloat16(), scale)
        at = 0
        for i, n in enumerate(rows):
            held[i] = [torch.cat([h, t[at:at + n]]) for h, t in zip(held[i], (k, v))]
            want = plain(q[at:at + n], *held[i], scale, window, pos[i])
            worst = max(worst, float((out[at:at + n].float() - want).norm() / want.norm()))
            at += n
    x.kv4_check(layer.err)
    return worst, seqs * most - len(layer.free)


if __name__ == "__main__":
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--device", type=int, default=0)
    torch.cuda.set_device(ap.parse_args().device)
    for window in (0, 256):
        worst, pages = serve(window=window)
        print(f"window {window or 'none'}: worst relative error of a step against 32-bit attention {worst:.3f}, "
              f"{pages} pages in use")
