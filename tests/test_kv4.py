"""CPU: the 4-bit cache's definition (tests/kv4_ref.py) on numbers worked out by hand, and the entry points' refusals,
which are decided on the host before any device work."""
import ctypes as C

import numpy as np
import pytest

import kv4_ref as R


def test_quantiser_by_hand():
    # 0 .. 63: lo 0, hi 63, (63 / 15 = 4.2) up to bf16 (steps of 2^-5): 4.21875; z = bf16(8 x 4.21875 = 33.75) = 33.75
    codes, words = R.quantise(np.arange(64, dtype=np.float32))
    assert R.of_bits(words >> 16)[0] == 4.21875 and R.of_bits(words & 0xFFFF)[0] == 33.75
    want = np.clip(np.rint((np.arange(64) - 33.75) / 4.21875), -8, 7) + 8
    assert np.array_equal(codes, want) and codes[0] == 0 and codes[63] == 15


@pytest.mark.parametrize("value", [0.0, 1.5, -3.0, 10.01])
def test_quantiser_of_a_constant(value):
    x = np.full(64, value, np.float32)
    codes, words = R.quantise(x)
    s, z = float(R.of_bits(words >> 16)[0]), float(R.of_bits(words & 0xFFFF)[0])
    assert s == 2.0 ** -100
    assert np.all(np.abs((codes - 8.0) * s + z - np.float64(x)) <= 2.0 ** -9 * abs(value))


@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
def test_quantiser_marks_a_group_with_no_finite_spread(bad):
    x = np.ones(128, np.float32)
    x[70] = bad
    codes, words = R.quantise(x)
    assert words[1] == 0xFFC00000 and not codes[64:].any() and words[0] != 0xFFC00000


def test_quantisation_error_is_half_a_step():
    x = np.random.default_rng(0).standard_normal((200, 128)).astype(np.float32)
    codes, words = R.quantise(x)
    s, z = (np.repeat(R.of_bits(b).astype(np.float64), 64, -1) for b in (words >> 16, words & 0xFFFF))
    err = np.abs((codes - 8.0) * s + z - x)
    # half a step, and at the ends what z's rounding (2^-9 |z|) cuts off; t's two f32 roundings
    assert np.all(err <= s * (0.5 + 1e-5) + 2.0 ** -8 * np.abs(z))


@pytest.mark.parametrize("d", [64, 128, 256])
def test_places_cover_the_block_once(d):
    seen = np.zeros((18 * d, 8), int)
    pars = np.zeros(18 * d, int)
    for word, shift, par in R.places(d):
        np.add.at(seen, (word, shift // 4), 1)
        np.add.at(pars, par, 1)
    codes = np.r_[0:8 * d, 9 * d:17 * d]
    assert (seen[codes] == 1).all() and seen.sum() == 2 * 64 * d
    assert pars.sum() == 2 * d and (np.delete(pars, codes) == 1).all()


# ---- refusals: every pointer is an address that is never read ----

GOOD = dict(pool=4096, pages=4, kv_heads=2, head_dim=128, table=4096, max_pages=2, seqs=1, pos=4096, cu_rows=4096,
            rows=3, err=None)


def call(xtg, entry, cache=None, **kw):
    c = xtg.Kv4(**dict(GOOD, **(cache or {})))
    err = C.create_string_buffer(512)
    L = xtg.lib()
    if entry == "store":
        a = dict(k=4096, v=4096, dtype=1, k_row=256, k_head=128, v_row=256, v_head=128)
        a.update(kw)
        rc = L.xtg_cuda_kv4_store(C.byref(c), a["k"], a["v"], a["dtype"], a["k_row"], a["k_head"], a["v_row"],
                                  a["v_head"], None, err, len(err))
    elif entry == "load":
        a = dict(k=4096, v=4096, dtype=1)
        a.update(kw)
        rc = L.xtg_cuda_kv4_load(C.byref(c), a["k"], a["v"], a["dtype"], None, err, len(err))
    else:
        a = dict(q=4096, out=4096, dtype=1, heads=4, q_row=512, q_head=128, scale=0.1, window=0, rows_per_seq=1,
                 workspace=4096, workspace_bytes=1 << 30)
        a.update(kw)
        rc = L.xtg_cuda_kv4_attention(C.byref(c), a["q"], a["out"], a["dtype"], a["heads"], a["q_row"], a["q_head"],
                                      a["scale"], a["window"], a["rows_per_seq"], a["workspace"],
                                      a["workspace_bytes"], None, err, len(err))
    return rc, err.value.decode()


@pytest.mark.parametrize("entry", ["store", "load", "attention"])
@pytest.mark.parametrize("cache,needle", [
    (dict(head_dim=96), "head_dim"), (dict(head_dim=0), "head_dim"), (dict(kv_heads=0), "KV heads"),
    (dict(kv_heads=-1), "KV heads"), (dict(kv_heads=1 << 20), "KV heads"), (dict(pages=0), "page"),
    (dict(max_pages=0), "page"), (dict(seqs=-1), "rows"), (dict(rows=-1), "rows"), (dict(rows=1 << 31), "rows"),
    (dict(seqs=1 << 30), "sequences"), (dict(pool=None), "null"), (dict(table=None), "null"), (dict(pos=None), "null"),
    (dict(cu_rows=None), "null"), (dict(pool=4096 + 8), "16-byte"),
])
def test_cache_refusals(xtg, entry, cache, needle):
    rc, why = call(xtg, entry, cache)
    assert rc == -1 and needle in why, why


@pytest.mark.parametrize("entry,kw,needle", [
    ("store", dict(k=None), "null"), ("store", dict(v=4096 + 8), "16-byte"), ("store", dict(dtype=3), "f32"),
    ("store", dict(k_row=250), "strides"), ("store", dict(v_head=-128), "strides"),
    ("store", dict(dtype=0, v_row=258), "strides"),
    ("load", dict(v=None), "null"), ("load", dict(k=4096 + 4), "16-byte"), ("load", dict(dtype=-1), "f32"),
    ("attention", dict(q=None), "null"), ("attention", dict(out=4096 + 8), "16-byte"),
    ("attention", dict(dtype=7), "f32"), ("attention", dict(heads=3), "multiple"), ("attention", dict(heads=0), "heads"),
    ("attention", dict(q_row=516), "strides"), ("attention", dict(window=-1), "window"),
    ("attention", dict(rows_per_seq=0), "rows_per_seq"), ("attention", dict(scale=float("nan")), "scale"),
    ("attention", dict(scale=float("inf")), "scale"), ("attention", dict(heads=1 << 30), "2^31"),
])
def test_row_refusals(xtg, entry, kw, needle):
    rc, why = call(xtg, entry, **kw)
    assert rc == -1 and needle in why, why


@pytest.mark.parametrize("entry", ["store", "load", "attention"])
@pytest.mark.parametrize("cache", [dict(rows=0), dict(seqs=0, table=None, pos=None, cu_rows=None)])
def test_nothing_to_do_is_no_error(xtg, entry, cache):
    assert call(xtg, entry, cache) == (0, "")


def test_workspace_refusals(xtg):
    L = xtg.lib()
    for bad in [(4, 0, 128, 1), (3, 2, 128, 1), (4, 2, 100, 1), (4, 2, 128, 0), (0, 2, 128, 1)]:
        assert L.xtg_cuda_kv4_workspace(*bad) == -1


def test_python_refuses_host_tensors(xtg):
    import torch
    pool = torch.zeros((2, 2, 72 * 128), dtype=torch.uint8)
    t = torch.zeros((1, 2), dtype=torch.int32)
    one = torch.zeros(1, dtype=torch.int32)
    with pytest.raises(xtg.XtgError, match="pool"):
        xtg.kv4_load(pool, t, one, torch.zeros(2, dtype=torch.int32), 0)
