"""GPU: attention over the 4-bit cache in parts of 131072 positions: what a sum over positions loses must not grow with
their number. The tables repeat a few pages, so that a reference is the softmax over these with their positions counted."""
import numpy as np
import pytest

import kv4_ref as R
from test_gpu_kv4 import MANTISSA, torch  # noqa: F401 (a fixture)
from test_gpu_kv4_ring import Shared

pytestmark = pytest.mark.gpu

LENGTH, SCALE = 131072, 0.05


def one_sign(rng, shape):
    """Values of one sign per head dim (the offsets of their groups lie in between): sums over positions that only grow."""
    sign = np.where(np.arange(shape[-1]) % 2, -1.0, 1.0)
    return (sign * (1.01 + 0.05 * rng.standard_normal(shape))).astype(np.float32)


def reference(s):
    """Attention of each kind's rows at LENGTH - rows, ..., in 64 bits, with its reach and top (kv4_ref)."""
    k, v = (np.stack([[s.ref.value(p, i, w)[0] for i in range(64)] for p in range(len(s.ref.words))]) for w in (0, 1))
    q = s.q.double().numpy().reshape(s.kinds, s.rows, s.heads, -1)
    a = np.einsum("crhd,psd->crhps", q, k) * SCALE
    out = np.zeros(q.shape)
    for c in range(s.kinds):
        for r in range(s.rows):
            seen = LENGTH - s.rows + r + 1
            times = np.zeros(k.shape[:2])
            np.add.at(times, s.table[c, :seen // 64], 1)
            if seen % 64:
                times[s.table[c, seen // 64], :seen % 64] += 1
            see = times > 0
            e = np.where(see, np.exp(np.where(see, a[c, r] - a[c, r][:, see].max(-1)[:, None, None], 0)) * times, 0)
            out[c, r] = np.einsum("hps,psd->hd", e, v) / e.sum((-1, -2))[:, None]
    reach = SCALE * np.einsum("crhd,psd->crhps", np.abs(q), np.abs(k)).max((-1, -2))
    return out, reach, np.abs(v).max((0, 1))


def check(torch, s):  # noqa: F811
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    out = s.run(s.kinds * -(-2 * sms // s.kinds), SCALE).double().cpu().numpy()
    want, reach, top = reference(s)
    bound = R.attention_bound(want, reach, top, MANTISSA[s.dtype])
    for kind in range(s.kinds):
        off = np.abs(out[kind::s.kinds] - want[kind]) / bound[kind]
        assert off.max() <= 1, off.max()   # NaN fails too


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows", [1, 2, 5])   # 4, 8 and 20 query rows of the KV head: each size of a row block
@pytest.mark.parametrize("d", [64, 128, 256])
def test_long_parts(cuda, xtg, torch, d, rows, dtype):  # noqa: F811
    table = (np.arange(LENGTH // 64) % 8)[None].repeat(4, 0)
    check(torch, Shared(torch, xtg, 32, rows, [LENGTH - rows] * 4, table, 4, 1, d, dtype, one_sign))


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("rows", [1, 2, 5])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_long_parts_of_unlike_scales(cuda, xtg, torch, d, rows, dtype):  # noqa: F811
    """Values near 1000 in one half of the part and near 10^-29 in the other, in both orders, and by turns."""
    def v_of(rng, shape):
        return (one_sign(rng, shape) * np.where(np.arange(shape[0]) < shape[0] // 2, 1e3, 1e-29)[:, None, None]).astype(
            np.float32)

    at = np.arange(LENGTH // 64)
    half = at >= len(at) // 2
    table = np.stack([at % 8 + 8 * half, at % 8 + 8 * ~half, at % 16])
    check(torch, Shared(torch, xtg, 33, rows, [LENGTH - rows] * 3, table, 4, 1, d, dtype, v_of))
