"""The 4-bit paged cache's definition in numpy: codes, scales and offsets by the quantiser's f32 steps, the values they
stand for and attention over them in 64 bits. Written from the definition (include/xtg_cuda.h, csrc/kv4.h), one
(slot, head dim) address at a time, without the library."""
import numpy as np

PAGE = 64


def bf16_bits(x, up=False):
    """f32 -> bf16 bits: to nearest (ties to even), or (up, for positive numbers) toward +infinity."""
    u = np.asarray(x, np.float32).view(np.uint32).astype(np.uint64)
    add = np.uint64(0xFFFF) if up else np.uint64(0x7FFF) + ((u >> np.uint64(16)) & np.uint64(1))
    return ((u + add) >> np.uint64(16)).astype(np.uint32)


def of_bits(b):
    return (np.asarray(b).astype(np.uint32) << np.uint32(16)).view(np.float32)


def quantise(x):
    """f32 [..., D] -> codes uint8 [..., D], parameter words uint32 [..., D / 64]."""
    x = np.asarray(x, np.float32)
    g = x.reshape(*x.shape[:-1], -1, 64)
    with np.errstate(all="ignore"):
        lo, hi = g.min(-1), g.max(-1)
        raw = ((hi - lo).astype(np.float32) * np.float32(1 / 15)).astype(np.float32)
        fine = np.isfinite(raw)
        s = np.maximum(of_bits(bf16_bits(np.where(fine, raw, 1), up=True)), np.float32(2.0 ** -100))
        z = of_bits(bf16_bits(np.where(fine, lo + np.float32(8) * s, 0)))
        fine &= np.isfinite(z)
        t = (g - z[..., None]).astype(np.float32) * (np.float32(1) / s)[..., None]
        codes = np.where(fine[..., None], np.rint(np.clip(t, -8, 7)) + 8, 0)
    word = np.where(fine, (s.view(np.uint32) & np.uint32(0xFFFF0000)) | bf16_bits(z), np.uint32(0xFFC00000))
    return codes.astype(np.uint8).reshape(x.shape), word.astype(np.uint32)


def places(d):
    """For each slot and head dim of a page: (word, shift) of K's code, of V's code; for each slot and group the word of
    K's and of V's parameters. Words of the block of 18 d words."""
    slot, dim = np.meshgrid(np.arange(PAGE), np.arange(d), indexing="ij")
    h = min(d, 128)
    kw = ((dim // h * PAGE + slot) * 4 + dim % 32 // 8) * (h // 32) + dim % h // 32
    ks = 4 * (dim % 8)
    vw = (((slot // 32 * (d // 32) + dim // 32) * 8 + dim % 8) * 4 + slot % 8 // 2) * 4 + dim % 32 // 8
    vs = 4 * (slot % 32 // 8 + 4 * (slot % 2))
    ps, pg = np.meshgrid(np.arange(PAGE), np.arange(d // 64), indexing="ij")
    par = pg * PAGE + ps
    return (kw, ks, 8 * d + par), (9 * d + vw, vs, 17 * d + par)


class Cache:
    """A pool [pages][kv_heads][18 d] of 32-bit words, with the operators over it."""

    def __init__(self, pages, kvh, d, fill=0):
        self.d, self.kvh = d, kvh
        self.words = np.full((pages, kvh, 18 * d), fill, np.uint32)

    @property
    def bytes(self):
        return self.words.view(np.uint8)

    def _where(self, table, seq, p):
        if p < 0 or p >= table.shape[1] * PAGE:
            return None
        page = table[seq, p // PAGE]
        return (page, p % PAGE) if 0 <= page < len(self.words) else None

    def store(self, k, v, table, pos, cu):
        for x, (word, shift, par) in zip((k, v), places(self.d)):
            codes, params = quantise(x)
            for s in range(len(pos)):
                for r in range(cu[s], cu[s + 1]):
                    at = self._where(table, s, int(pos[s]) + r - cu[s])
                    if at is None:
                        continue
                    page, slot = at
                    for h in range(self.kvh):
                        w = self.words[page, h]
                        w[par[slot]] = params[r, h]
                        nib = codes[r, h].astype(np.uint32) << shift[slot].astype(np.uint32)
                        clear = np.uint32(15) << shift[slot].astype(np.uint32)
                        # K: 8 dims share a word; V: a word has one nibble of this slot
                        np.bitwise_and.at(w, word[slot], ~clear)
                        np.bitwise_or.at(w, word[slot], nib)

    def value(self, page, slot, which):
        """[kv_heads][d] in 64 bits (which: 0 K, 1 V)."""
        word, shift, par = (x[slot] for x in places_of(self.d)[which])
        w = self.words[page]
        code = (w[:, word] >> shift.astype(np.uint32)) & 15
        p = w[:, par]
        s, z = of_bits(p >> 16).astype(np.float64), of_bits(p & 0xFFFF).astype(np.float64)
        return (code.astype(np.float64) - 8) * np.repeat(s, 64, -1) + np.repeat(z, 64, -1)

    def load(self, table, pos, cu):
        out = np.zeros((2, cu[-1], self.kvh, self.d))
        for s in range(len(pos)):
            for r in range(cu[s], cu[s + 1]):
                at = self._where(table, s, int(pos[s]) + r - cu[s])
                if at is not None:
                    out[0, r], out[1, r] = self.value(*at, 0), self.value(*at, 1)
        return out

    def attention(self, q, table, pos, cu, scale, window=0):
        """q [rows][heads][d] in 64 bits -> (out, reach): reach [rows][heads] = max_p scale sum_d |q_d K_pd| and
        [rows][heads][d] = max_p |V_pd|, for error bounds."""
        rows, heads, d = q.shape
        group = heads // self.kvh
        out, reach, top = np.zeros(q.shape), np.zeros((rows, heads)), np.zeros(q.shape)
        for s in range(len(pos)):
            n = cu[s + 1] - cu[s]
            if n <= 0:
                continue
            end = int(pos[s]) + n
            first = max(0, int(pos[s]) - window + 1) if window else 0
            held = [(p, self._where(table, s, p)) for p in range(first, end)]
            held = [(p, at) for p, at in held if at is not None]
            if not held:
                continue
            k = np.stack([self.value(*at, 0) for _, at in held])
            v = np.stack([self.value(*at, 1) for _, at in held])
            p = np.array([p for p, _ in held])
            for r in range(cu[s], cu[s + 1]):
                t = int(pos[s]) + r - int(cu[s])
                see = (p <= t) & ((p > t - window) if window else True)
                if not see.any():
                    continue
                for j in range(heads):
                    kk, vv, qq = k[see, j // group], v[see, j // group], q[r, j].astype(np.float64)
                    a = kk @ qq * scale
                    e = np.exp(a - a.max())
                    out[r, j] = e @ vv / e.sum()
                    reach[r, j] = abs(scale) * (np.abs(kk) @ np.abs(qq)).max()
                    top[r, j] = np.abs(vv).max(0)
        return out, reach, top


_places = {}


def places_of(d):
    if d not in _places:
        _places[d] = places(d)
    return _places[d]


def attention_bound(out, reach, top, mantissa):
    """How far a row may be from `out`. A score is sum q K in products of f16 planes (22 bits) summed in f32: within
    2^-19 of sum |q K| (22 bits, up to 16 sums of 16 products, the groups' f32 sums, the factor); its error enters the
    probability's exponent and the normaliser's. A probability (2^x, its two planes) and the sums over positions in
    f32 are within 2^-17 of the largest value together. Then one rounding to the output's type."""
    return (2 * reach[..., None] * 2.0 ** -19 + 2.0 ** -17) * top + 2.0 ** -mantissa * np.abs(out) + 1e-30
