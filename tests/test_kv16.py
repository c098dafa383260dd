"""CPU: the 16-bit caches' definition (tests/kv16_ref.py) on numbers worked out by hand, and the entry points' refusals, which
are decided on the host before any device work."""
import ctypes as C
import math

import pytest
import torch

import kv16_ref as R


def test_rotation_by_hand():
    x = torch.tensor([[[1.0, 0.0, 2.0, 0.0]]])   # pairs (1, 2), (0, 0); interleaved (1, 0), (2, 0)
    freq = torch.tensor([math.pi / 2 / 3, 0.0], dtype=torch.float64)
    y = R.rotate(x, torch.tensor([3]), freq, False)   # a quarter turn: (a, b) -> (-b, a)
    assert torch.allclose(y, torch.tensor([[[-2.0, 0.0, 1.0, 0.0]]], dtype=torch.float64))
    y = R.rotate(x, torch.tensor([3]), freq, True)
    assert torch.allclose(y, torch.tensor([[[0.0, 1.0, 2.0, 0.0]]], dtype=torch.float64))


def test_attention_by_hand():
    # two positions, scores 0 and ln 3: weights 1/4 and 3/4; the row at position 0 sees the first alone; a window of one the
    # row's own alone; a page that is not there nothing
    k = torch.zeros(1, 1, 16, 64)
    v = torch.zeros(1, 1, 16, 64)
    k[0, 0, 1, 0] = math.log(3)
    v[0, 0, 0, 5], v[0, 0, 1, 5] = 4.0, 8.0
    q = torch.zeros(2, 1, 64)
    q[:, 0, 0] = 1
    where = [torch.tensor([[0]]), torch.tensor([0]), torch.tensor([0, 2])]
    assert torch.allclose(R.attention(q, k, v, *where, 1.0)[0][:, 0, 5], torch.tensor([4.0, 7.0], dtype=torch.float64))
    assert torch.allclose(R.attention(q, k, v, *where, 1.0, 1)[0][:, 0, 5], torch.tensor([4.0, 8.0], dtype=torch.float64))
    where[0] = torch.tensor([[-1]])
    assert not R.attention(q, k, v, *where, 1.0)[0].any()


# ---- refusals: every pointer is an address that is never read ----

CACHE = dict(k=4096, v=4096, dtype=1, pages=4, page=64, kv_heads=2, head_dim=128, v_dim=128, k_page=2 * 64 * 128,
             k_head=64 * 128, k_slot=128, v_page=2 * 64 * 128, v_head=64 * 128, v_slot=128, table=4096, max_pages=2, seqs=1,
             pos=4096, cu_rows=4096, rows=3, err=None)
LATENT = dict(v=None, kv_heads=1, head_dim=576, v_dim=512, k_page=64 * 576, k_slot=576)
ROWS = dict(k=4096, v=4096, q=4096, q_out=4096, dtype=0, heads=4, k_row=256, k_head=128, v_row=256, v_head=128, q_row=512,
            q_head=128, freq=4096, rotary=128, first=0, interleaved=0)
ATTN = dict(q=4096, q_rot=None, out=4096, heads=4, q_row=512, q_head=128, r_row=0, r_head=0, scale=0.1, window=0,
            rows_per_seq=1, zero_rest=0, workspace=4096, workspace_bytes=1 << 40)


def call(xtg, entry, cache=None, rows=None):
    c = xtg.Kv16(**dict(CACHE, **(cache or {})))
    err = C.create_string_buffer(512)
    if entry == "append":
        r = xtg.Kv16Rows(**dict(ROWS, **(rows or {})))
        rc = xtg.lib().xtg_cuda_kv16_append(C.byref(c), C.byref(r), None, err, len(err))
    else:
        r = xtg.Kv16Attn(**dict(ATTN, **(rows or {})))
        rc = xtg.lib().xtg_cuda_kv16_attention(C.byref(c), C.byref(r), None, err, len(err))
    return rc, err.value.decode()


@pytest.mark.parametrize("entry", ["append", "attention"])
@pytest.mark.parametrize("cache,needle", [
    (dict(dtype=0), "bf16"), (dict(dtype=3), "bf16"), (dict(head_dim=96), "head_dim"), (dict(v_dim=64), "head_dim"),
    (dict(head_dim=256, v_dim=128), "head_dim"), (dict(v=None), "head_dim"), (dict(kv_heads=0), "KV heads"),
    (dict(LATENT, kv_heads=2), "KV heads"), (dict(LATENT, head_dim=512, v_dim=448), "head_dim"),
    (dict(kv_heads=1 << 20), "KV heads"), (dict(page=8), "page"), (dict(page=48), "page"), (dict(page=2048), "page"),
    (dict(pages=0), "page"), (dict(pages=1 << 31), "page"), (dict(max_pages=0), "page"), (dict(seqs=-1), "rows"),
    (dict(rows=-1), "rows"), (dict(rows=1 << 31), "rows"), (dict(max_pages=1 << 26), "2^31"), (dict(seqs=1 << 30), "sequences"),
    (dict(k=None), "null"), (dict(table=None), "null"), (dict(pos=None), "null"), (dict(cu_rows=None), "null"),
    (dict(k=4096 + 8), "16-byte"), (dict(v=4096 + 2), "16-byte"), (dict(k_slot=120), "strides"), (dict(k_slot=132), "strides"),
    (dict(v_head=0), "strides"), (dict(k_page=-64 * 128), "strides"), (dict(v_page=1 << 39), "strides"),
])
def test_cache_refusals(xtg, entry, cache, needle):
    rc, why = call(xtg, entry, cache)
    assert rc == -1 and needle in why, why


@pytest.mark.parametrize("entry,rows,needle", [
    ("append", dict(dtype=3), "f32"), ("append", dict(dtype=-1), "f32"), ("append", dict(k=None), "null"),
    ("append", dict(v=4096 + 8), "16-byte"), ("append", dict(q_out=None), "null"), ("append", dict(k_row=254), "strides"),
    ("append", dict(dtype=1, v_row=252), "strides"), ("append", dict(q_head=-128), "strides"),
    ("append", dict(rotary=120), "rotary"), ("append", dict(rotary=-16), "rotary"), ("append", dict(first=4), "first"),
    ("append", dict(first=16), "head"), ("append", dict(freq=None), "null"), ("append", dict(heads=0), "heads"),
    ("append", dict(heads=1 << 30), "2^31"),
    ("attention", dict(q=None), "null"), ("attention", dict(out=4096 + 8), "16-byte"), ("attention", dict(heads=3), "multiple"),
    ("attention", dict(heads=0), "heads"), ("attention", dict(q_row=516), "strides"), ("attention", dict(window=-1), "window"),
    ("attention", dict(rows_per_seq=0), "rows_per_seq"), ("attention", dict(scale=float("nan")), "scale"),
    ("attention", dict(scale=float("inf")), "scale"), ("attention", dict(heads=1 << 30), "32768"),
])
def test_row_refusals(xtg, entry, rows, needle):
    rc, why = call(xtg, entry, None, rows)
    assert rc == -1 and needle in why, why


def test_latent_refusals(xtg):
    rc, why = call(xtg, "attention", LATENT)
    assert rc == -1 and "null" in why   # no q_rot
    rc, why = call(xtg, "append", LATENT, dict(rotary=128))
    assert rc == -1 and "head" in why   # 64 dims turn


@pytest.mark.parametrize("entry", ["append", "attention"])
@pytest.mark.parametrize("cache", [dict(rows=0), dict(seqs=0, table=None, pos=None, cu_rows=None)])
def test_nothing_to_do_is_no_error(xtg, entry, cache):
    assert call(xtg, entry, cache, dict(q=None) if entry == "append" else None) == (0, "")


def test_workspace_refusals(xtg):
    L = xtg.lib()
    for bad in [(4, 0, 128, 128, 0, 1), (3, 2, 128, 128, 0, 1), (4, 2, 96, 96, 0, 1), (4, 2, 128, 128, 0, 0),
                (0, 2, 128, 128, 0, 1), (8, 1, 128, 64, 1, 1)]:
        assert L.xtg_cuda_kv16_workspace(*bad) == -1


def test_wait_polls_are_kept(xtg):
    L = xtg.lib()
    first = L.xtg_cuda_kv16_wait_polls(-1)
    assert first == 1 << 18
    assert L.xtg_cuda_kv16_wait_polls(7) == first and L.xtg_cuda_kv16_wait_polls(first) == 7


def test_python_refuses_host_tensors(xtg):
    pool = torch.zeros((2, 2, 64, 128), dtype=torch.bfloat16)
    t, one, cu = torch.zeros((1, 2), dtype=torch.int32), torch.zeros(1, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    rows = torch.zeros((1, 2, 128), dtype=torch.bfloat16)
    with pytest.raises(xtg.XtgError, match="pool"):
        xtg.kv16_append(pool, pool, rows, rows, t, one, cu)
    with pytest.raises(xtg.XtgError, match="pool"):
        xtg.kv16_attention(rows, pool, pool, t, one, cu, 1.0)
    with pytest.raises(xtg.XtgError, match="pool"):
        xtg.latent_attention(rows, rows, torch.zeros((2, 64, 576), dtype=torch.float16), t, one, cu, 1.0)
    with pytest.raises(xtg.XtgError, match="tensor"):
        xtg.latent_append(None, rows, rows, t, one, cu)
