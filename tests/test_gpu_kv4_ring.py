"""GPU: attention over the 4-bit cache where a CTA brings many more chunks than its ring holds. Sequences share pages that
are only read, so that a small pool gives every CTA several turns of the ring; a reference is worked out once for each
kind of sequence."""
import numpy as np
import pytest

import kv4_ref as R
from test_gpu_kv4 import MANTISSA, dtype_of, torch  # noqa: F401 (a fixture)

pytestmark = pytest.mark.gpu

STAGES = 24   # of the longest ring


class Shared:
    """Kinds of sequences, each of `rows` rows after position pos[kind], over one pool; a call takes `seqs` sequences, of
    the kinds in turn, with the same queries for all of a kind."""

    def __init__(self, torch, xtg, seed, rows, pos, table, heads, kvh, d, dtype, v_of=None):  # noqa: F811
        self.torch, self.xtg, self.dtype = torch, xtg, dtype
        rng = np.random.default_rng(seed)
        self.kinds, self.rows, self.heads = len(pos), rows, heads
        self.pos, self.table = np.array(pos, np.int32), np.array(table, np.int32)
        self.ref = R.Cache(int(self.table.max()) + 1, kvh, d)
        n = 64 * len(self.ref.words)
        k = rng.standard_normal((n, kvh, d)).astype(np.float32)
        v = rng.standard_normal((n, kvh, d)).astype(np.float32) if v_of is None else v_of(rng, (n, kvh, d))
        self.ref.store(k, v, np.arange(len(self.ref.words))[None], np.zeros(1, np.int32), np.array([0, n]))
        self.q = torch.from_numpy(rng.standard_normal((self.kinds * rows, heads, d)).astype(np.float32) * 2).to(
            dtype_of(torch, dtype))
        self.cu = np.arange(self.kinds + 1, dtype=np.int32) * rows
        self.pool = torch.from_numpy(self.ref.bytes).cuda().view(len(self.ref.words), kvh, 72 * d)

    def run(self, seqs, scale, window=0):
        """The call's rows [seqs][rows][heads][d]."""
        out, err = self.attend(seqs, scale, window)
        self.xtg.kv4_check(err)
        return out

    def attend(self, seqs, scale, window=0):
        torch = self.torch  # noqa: F811
        kind = torch.arange(seqs) % self.kinds
        q = self.q.view(self.kinds, self.rows, *self.q.shape[1:])[kind].flatten(0, 1).cuda()
        cu = torch.arange(seqs + 1, dtype=torch.int32, device="cuda") * self.rows
        err = torch.zeros(1, dtype=torch.int32, device="cuda")
        out = self.xtg.kv4_attention(q, self.pool, torch.from_numpy(self.table)[kind].cuda(),
                                     torch.from_numpy(self.pos)[kind].cuda(), cu, scale, window, err=err)
        return out.view(seqs, self.rows, *q.shape[1:]), err

    def check(self, out, scale, window=0):
        q = self.q.double().numpy()
        want, reach, top = self.ref.attention(q, self.table, self.pos, self.cu, scale, window)
        bound = R.attention_bound(want, reach, top, MANTISSA[self.dtype])
        shape = (self.kinds, self.rows, *q.shape[1:])
        want, bound = (self.torch.from_numpy(x).view(shape).cuda() for x in (want, bound))
        worst = 0.0
        for kind in range(self.kinds):
            off = (out[kind::self.kinds].double() - want[kind]).abs() / bound[kind]
            worst = max(worst, float(off.max()))
        assert worst <= 1, worst


@pytest.mark.parametrize("window", [0, 300])
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows", [1, 2, 5])   # 4, 8 and 20 query rows of a KV head: each size of a row block
@pytest.mark.parametrize("d", [64, 128, 256])
def test_many_parts(cuda, xtg, torch, d, rows, dtype, window):  # noqa: F811
    """Every CTA takes at least 3 turns of the ring over parts of 1 to 21 chunks, with an absent page in the middle."""
    pos = [1290, 70, 0, 639]
    table = np.random.default_rng(31).permutation(22)[None].repeat(4, 0)
    table[0, 9] = table[3, 8] = -1
    s = Shared(torch, xtg, 30, rows, pos, table, 8, 2, d, dtype)
    first = [max(0, p - window + 1) // 64 if window else 0 for p in pos]
    chunks = sum(-(-(p + rows) // 64) - f for p, f in zip(pos, first))   # of one sequence of each kind, per KV head
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    # a part's start counts up to 12 more chunks in the shares
    per_cta = chunks / (chunks + 4 * 12)
    seqs = 4 * -(-int(3 * STAGES * sms / per_cta) // (2 * chunks))
    s.check(s.run(seqs, 0.1, window), 0.1, window)
