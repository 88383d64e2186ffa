"""The host side of the 4-bit paged KV cache's entry points: sizes, refusals
before any launch, no-ops (no GPU)."""
import ctypes as C

import numpy as np
import pytest

import kv4_ref as ref

F32, F16, BF16, Q8_0 = 0, 1, 30, 8
P = 0x7f0000000000   # an aligned address that no refused call reads


def batch(sn, **kw):
    d = dict(tok_start=P, kv_len=P, pages=P, kc=P, vc=P, n_seq=2, n_tok=3, max_pages=4, n_pages=9, page_rows=16, nkv=2, hd=64)
    d.update(kw)
    return sn.Kv4Batch(**d)


def rows(sn, **kw):
    d = dict(p=P, ld=128, hs=64)
    d.update(kw)
    return sn.Heads(**d)


def attn(sn, **kw):
    d = dict(q=rows(sn, ld=256), out=rows(sn, ld=256), ws=P, ws_bytes=1 << 40, nq=4, max_q=2, max_kv=64, scale=0.125, type=F32)
    d.update(kw)
    return sn.Kv4AttnArgs(**d)


def prep(sn, **kw):
    d = dict(q=rows(sn, ld=256), q_out=rows(sn, ld=256), k=rows(sn), k_out=rows(sn), nq=4, rope_dims=32, rope_base=1e4, eps=1e-6, type=F32)
    d.update(kw)
    return sn.Kv4PrepArgs(**d)


def test_page_bytes(sn):
    f = sn.lib().sinter_kv4_page_bytes
    for rows_, nkv, hd in ((16, 1, 64), (64, 4, 256), (1024, 8, 128), (1 << 20, 1, 256)):
        assert f(rows_, nkv, hd) == ref.page_bytes(rows_, nkv, hd)
    for rows_, nkv, hd in ((8, 1, 64), (48, 1, 64), (1 << 21, 1, 64), (16, 0, 64), (16, 1, 96), (16, 1025, 64), (1 << 20, 32, 256), (0, 1, 64)):
        assert f(rows_, nkv, hd) == 0


BAD_BATCH = [dict(hd=96), dict(hd=0), dict(nkv=0), dict(nkv=2000), dict(n_seq=70000), dict(n_tok=2 ** 31), dict(tok_start=0), dict(kv_len=0),
             dict(tok_start=P + 2), dict(kv_len=P + 1)]
BAD_CACHE = [dict(page_rows=8), dict(page_rows=24), dict(page_rows=1 << 21), dict(max_pages=0), dict(n_pages=0), dict(n_pages=2 ** 31),
             dict(pages=0), dict(pages=P + 2), dict(kc=0), dict(vc=0), dict(kc=P + 8), dict(vc=P + 4)]
BAD_ROWS = [dict(p=0), dict(p=P + 8), dict(ld=126), dict(hs=62), dict(hs=32), dict(ld=32), dict(ld=64, hs=64), dict(ld=-128), dict(hs=66)]


def refused(sn, rc, word=None):
    assert rc == sn.ERR_ARG
    msg = sn.lib().sinter_last_error().decode()
    assert msg.startswith("kv4_") and (word is None or word in msg), msg


@pytest.mark.parametrize("kw", BAD_BATCH + BAD_CACHE)
def test_bad_batches(sn, kw):
    L, b = sn.lib(), batch(sn, **kw)
    refused(sn, L.sinter_kv4_append(C.byref(b), C.byref(rows(sn)), C.byref(rows(sn)), F32, None))
    refused(sn, L.sinter_kv4_read(C.byref(b), C.byref(rows(sn)), None, F32, None))
    refused(sn, L.sinter_kv4_attn(C.byref(b), C.byref(attn(sn)), None))
    assert L.sinter_kv4_attn_ws_bytes(C.byref(b), C.byref(attn(sn))) == 0
    if kw in BAD_BATCH:
        refused(sn, L.sinter_kv4_prep(C.byref(b), C.byref(prep(sn)), None))


@pytest.mark.parametrize("kw", BAD_ROWS)
def test_bad_rows(sn, kw):
    L, b, r = sn.lib(), batch(sn), rows(sn, **kw)
    for args in ((r, rows(sn)), (rows(sn), r)):
        refused(sn, L.sinter_kv4_append(C.byref(b), C.byref(args[0]), C.byref(args[1]), F32, None))
        if r.p:   # (a null array is left out of a read)
            refused(sn, L.sinter_kv4_read(C.byref(b), C.byref(args[0]), C.byref(args[1]), F32, None))
    q = dict(kw)
    if q.get("ld", 0) == 128:
        q["ld"] = 256
    wide = rows(sn, **{**dict(ld=256), **q})
    for name in ("q", "out") + (("gate",) if wide.p else ()):
        refused(sn, L.sinter_kv4_attn(C.byref(b), C.byref(attn(sn, **{name: wide})), None))
    for name in ("q", "q_out"):
        refused(sn, L.sinter_kv4_prep(C.byref(b), C.byref(prep(sn, **{name: wide})), None), "q:")
    for name in ("k", "k_out"):
        refused(sn, L.sinter_kv4_prep(C.byref(b), C.byref(prep(sn, **{name: r})), None), "k:")


def test_bad_types_and_nulls(sn):
    L, b = sn.lib(), batch(sn)
    for t in (Q8_0, -1, 2):
        refused(sn, L.sinter_kv4_append(C.byref(b), C.byref(rows(sn)), C.byref(rows(sn)), t, None), "type")
        refused(sn, L.sinter_kv4_read(C.byref(b), C.byref(rows(sn)), None, t, None), "type")
    for t in (Q8_0, 2):
        refused(sn, L.sinter_kv4_attn(C.byref(b), C.byref(attn(sn, type=t)), None), "type")
        refused(sn, L.sinter_kv4_prep(C.byref(b), C.byref(prep(sn, type=t)), None), "type")
    r = C.byref(rows(sn))
    for rc in (L.sinter_kv4_append(None, r, r, F32, None), L.sinter_kv4_append(C.byref(b), None, r, F32, None),
               L.sinter_kv4_append(C.byref(b), r, None, F32, None), L.sinter_kv4_read(None, r, r, F32, None),
               L.sinter_kv4_read(C.byref(b), None, None, F32, None), L.sinter_kv4_attn(None, C.byref(attn(sn)), None),
               L.sinter_kv4_attn(C.byref(b), None, None), L.sinter_kv4_prep(None, C.byref(prep(sn)), None),
               L.sinter_kv4_prep(C.byref(b), None, None)):
        refused(sn, rc)
    # 16-bit rows need strides of 8 elements
    refused(sn, L.sinter_kv4_append(C.byref(b), C.byref(rows(sn, ld=132)), r, BF16, None))


@pytest.mark.parametrize("kw", [dict(nq=0), dict(nq=3), dict(nq=1024, q=None), dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")),
                                dict(scale=float("inf")), dict(max_q=0), dict(max_kv=0), dict(max_kv=2 ** 31)])
def test_bad_attention(sn, kw):
    if "q" in kw:
        kw = dict(nq=1024, q=rows(sn, ld=65536), out=rows(sn, ld=65536))
    L, b = sn.lib(), batch(sn)
    refused(sn, L.sinter_kv4_attn(C.byref(b), C.byref(attn(sn, **kw)), None))
    assert L.sinter_kv4_attn_ws_bytes(C.byref(b), C.byref(attn(sn, **kw))) == 0


@pytest.mark.parametrize("bk,ak", [(dict(n_seq=65536), dict(max_kv=1 << 22)), (dict(n_tok=1 << 30), dict()),
                                   (dict(n_seq=65536, n_tok=1 << 20, nkv=256), dict(nq=1024, max_kv=4096))])
def test_attention_too_large(sn, bk, ak):
    """Counts that 32 bits, or a launch, do not hold."""
    L, b = sn.lib(), batch(sn, **bk)
    q = rows(sn, ld=1 << 20)
    refused(sn, L.sinter_kv4_attn(C.byref(b), C.byref(attn(sn, q=q, out=q, **ak)), None), "too large")


def test_too_many_tokens(sn):
    L, b = sn.lib(), batch(sn, n_tok=1 << 25)
    refused(sn, L.sinter_kv4_prep(C.byref(b), C.byref(prep(sn)), None), "too many")


def test_workspace(sn):
    L, b = sn.lib(), batch(sn)
    a = attn(sn, max_kv=5000)
    n = L.sinter_kv4_attn_ws_bytes(C.byref(b), C.byref(a))
    assert n > 0
    for kw in (dict(ws=0), dict(ws=P + 8), dict(ws_bytes=n - 1)):
        refused(sn, L.sinter_kv4_attn(C.byref(b), C.byref(attn(sn, **{**dict(max_kv=5000, ws_bytes=n), **kw})), None), "workspace")
    # short sequences are not split: no workspace
    assert L.sinter_kv4_attn_ws_bytes(C.byref(b), C.byref(attn(sn, max_kv=64))) == 0


@pytest.mark.parametrize("kw", [dict(rope_dims=12), dict(rope_dims=72), dict(rope_base=0.0), dict(rope_base=float("nan")), dict(eps=-1.0),
                                dict(eps=float("nan")), dict(q_norm=P + 4), dict(k_norm=P + 8), dict(nq=5000)])
def test_bad_prep(sn, kw):
    refused(sn, sn.lib().sinter_kv4_prep(C.byref(batch(sn)), C.byref(prep(sn, **kw)), None))


@pytest.mark.parametrize("kw", [dict(n_seq=0), dict(n_tok=0), dict(n_seq=0, tok_start=0, kv_len=0, pages=0, kc=0, vc=0)])
def test_nothing_to_do(sn, kw):
    L, b = sn.lib(), batch(sn, **kw)
    assert L.sinter_kv4_append(C.byref(b), C.byref(rows(sn)), C.byref(rows(sn)), F32, None) == 0
    assert L.sinter_kv4_read(C.byref(b), C.byref(rows(sn)), None, F32, None) == 0
    assert L.sinter_kv4_attn(C.byref(b), C.byref(attn(sn, ws=0)), None) == 0
    assert L.sinter_kv4_prep(C.byref(b), C.byref(prep(sn)), None) == 0
    assert L.sinter_kv4_attn_ws_bytes(C.byref(b), C.byref(attn(sn))) == 0


def test_prep_of_nothing(sn):
    none = sn.Heads()
    assert sn.lib().sinter_kv4_prep(C.byref(batch(sn)), C.byref(prep(sn, q=none, q_out=none, k=none, k_out=none)), None) == 0


def test_reference_round_trip():
    """The reference itself: what it stores is what the format gives back."""
    rng = np.random.default_rng(1)
    x = rng.standard_normal((5, 2, 64)).astype(np.float32)
    code, d = ref.quantise(x)
    v = ref.values(code, d)
    top = np.abs(x.reshape(5, 2, 2, 32)).max(-1)
    # half a step of d = max / 8, a whole one at the end that has no code 16, and the scale's own rounding
    assert (np.abs(v - x).reshape(5, 2, 2, 32).max(-1) <= top / 8 * (1 + 8 * 2.0 ** -11)).all()
    cache = np.zeros(ref.page_bytes(16, 2, 64) * 3, np.uint8)
    for r in range(5):
        for g in range(2):
            ref.put(cache, 1, r, g, 16, 2, 64, code[r, g], d[r, g])
            assert np.array_equal(ref.get(cache, 1, r, g, 16, 2, 64), v[r, g])
