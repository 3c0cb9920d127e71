"""The paged 8-bit KV cache's entry points refuse bad arguments on the host,
before any CUDA call (fake, aligned device addresses; no device)."""

from __future__ import annotations

import ctypes as C

import pytest

from siphon_b200 import lib as L


@pytest.fixture(scope="module")
def so():
    return L.SiphonCuda()


P = 0x10000          # an aligned, never dereferenced address


def cache(**kw):
    a = dict(k=P, v=P, k_scale=P, v_scale=P, n_pages=10, page=16, n_head_kv=2, head_dim=64)
    a.update(kw)
    return L.kv8_cache(**a)


def refused(so, rc, code, word):
    assert rc == code, (rc, so.last_error())
    assert word in so.last_error(), so.last_error()


def test_plan_checks(so):
    def call(past=P, fresh=P, n_seq=4, page=16, table=P, max_pages=8, free=P, n_pages=10, n_free=P, out=P, n_tok=4, cu=P,
             length=P, slot=P, pos=P):
        return so.lib.sicu_kv8_plan(past, fresh, n_seq, page, table, max_pages, free, n_pages, n_free, out, n_tok, cu,
                                    length, slot, pos, None)
    refused(so, call(page=48), L.SICU_EINVAL, "pages of 48")
    refused(so, call(n_seq=0), L.SICU_EINVAL, "requests")
    refused(so, call(n_seq=8193), L.SICU_EINVAL, "requests")
    refused(so, call(max_pages=0), L.SICU_EINVAL, "size")
    refused(so, call(n_tok=-1), L.SICU_EINVAL, "size")
    refused(so, call(n_pages=1 << 31), L.SICU_EINVAL, "size")
    for name in ("past", "fresh", "table", "free", "n_free", "out", "cu", "length", "slot", "pos"):
        refused(so, call(**{name: None}), L.SICU_EINVAL, "null")
    refused(so, call(slot=P + 8), L.SICU_EINVAL, "aligned")
    refused(so, call(), L.SICU_EINVAL, "sicu_init")


def test_release_checks(so):
    def call(drop=P, n_seq=4, page=16, max_pages=8):
        return so.lib.sicu_kv8_release(drop, P, n_seq, page, P, max_pages, P, 10, P, None)
    refused(so, call(drop=None), L.SICU_EINVAL, "null")
    refused(so, call(page=0), L.SICU_EINVAL, "pages of 0")
    refused(so, call(n_seq=10 ** 6), L.SICU_EINVAL, "requests")
    refused(so, call(), L.SICU_EINVAL, "sicu_init")


def test_store_and_load_checks(so):
    def store(c=None, type=L.T_F32, k=P, v=P, ks=0, vs=0, slot=P, pos=P, rope=None, n=3):
        return so.lib.sicu_kv8_store(C.byref(c or cache()), type, k, v, ks, vs, slot, pos,
                                     C.byref(rope) if rope else None, n, None)
    refused(so, so.lib.sicu_kv8_store(None, 0, P, P, 0, 0, P, P, None, 1, None), L.SICU_EINVAL, "null cache")
    refused(so, store(cache(page=24)), L.SICU_EINVAL, "pages of 24")
    refused(so, store(cache(head_dim=80)), L.SICU_ENOTSUP, "head size 80")
    refused(so, store(cache(n_head_kv=0)), L.SICU_EINVAL, "KV heads")
    refused(so, store(cache(n_pages=0)), L.SICU_EINVAL, "pages")
    refused(so, store(cache(k=None)), L.SICU_EINVAL, "null cache")
    refused(so, store(cache(v=P + 4)), L.SICU_EINVAL, "aligned")
    refused(so, store(type=12), L.SICU_ENOTSUP, "type")
    refused(so, store(k=None), L.SICU_EINVAL, "null")
    refused(so, store(k=P + 4), L.SICU_EINVAL, "aligned")
    refused(so, store(ks=127), L.SICU_EINVAL, "stride")          # below 2 heads of 64
    refused(so, store(vs=129), L.SICU_EINVAL, "aligned")         # rows off 16 bytes
    refused(so, store(slot=None), L.SICU_EINVAL, "null")
    refused(so, store(n=-1), L.SICU_EINVAL, "tokens")
    refused(so, store(rope=L.rope(P, P, 8, 68)), L.SICU_EINVAL, "rotated")
    refused(so, store(rope=L.rope(P, P, 8, 4)), L.SICU_EINVAL, "rotated")
    refused(so, store(rope=L.rope(P, None, 8, 64)), L.SICU_EINVAL, "null RoPE")
    refused(so, store(rope=L.rope(P + 4, P, 8, 64)), L.SICU_EINVAL, "aligned")
    refused(so, store(rope=L.rope(P, P, 0, 64)), L.SICU_EINVAL, "positions")
    refused(so, store(rope=L.rope(P, P, 8, 64), pos=None), L.SICU_EINVAL, "null")
    refused(so, store(), L.SICU_EINVAL, "sicu_init")

    def load(type=L.T_F32, slot=P, n=3, k=P, v=P):
        return so.lib.sicu_kv8_load(C.byref(cache()), type, slot, n, k, v, None)
    refused(so, load(type=2), L.SICU_ENOTSUP, "type")
    refused(so, load(slot=None), L.SICU_EINVAL, "null")
    refused(so, load(v=P + 2), L.SICU_EINVAL, "aligned")
    refused(so, load(n=-5), L.SICU_EINVAL, "tokens")
    refused(so, load(), L.SICU_EINVAL, "sicu_init")


def test_attention_checks(so):
    def call(c=None, q=P, out=P, ws=P, ws_bytes=1 << 20, **kw):
        a = dict(type=L.T_F32, n_head=4, n_tok=3, table=P, max_pages=8, length=P, cu=P, n_seq=2, max_new=2, max_len=100,
                 scale=0.1)
        a.update(kw)
        return so.lib.sicu_kv8_attention(C.byref(c or cache()), C.byref(L.kv8_attn(**a)), q, out, ws, ws_bytes, None)
    refused(so, call(cache(head_dim=100)), L.SICU_ENOTSUP, "head size")
    refused(so, call(type=8), L.SICU_ENOTSUP, "type")
    refused(so, call(n_head=3), L.SICU_EINVAL, "heads")
    refused(so, call(n_head=0), L.SICU_EINVAL, "heads")
    refused(so, call(n_seq=-1), L.SICU_EINVAL, "requests")
    refused(so, call(n_seq=9000), L.SICU_EINVAL, "requests")
    refused(so, call(n_tok=-1), L.SICU_EINVAL, "tokens")
    refused(so, call(max_len=129), L.SICU_EINVAL, "lengths")     # 8 pages of 16
    refused(so, call(max_new=4), L.SICU_EINVAL, "new tokens")
    refused(so, call(max_len=1), L.SICU_EINVAL, "new tokens")
    refused(so, call(n_tok=1 << 30), L.SICU_EINVAL, "too many rows")
    refused(so, call(window=-1), L.SICU_EINVAL, "window")
    refused(so, call(cap=-1.0), L.SICU_EINVAL, "cap")
    refused(so, call(cap=float("nan")), L.SICU_EINVAL, "cap")
    refused(so, call(q=None), L.SICU_EINVAL, "null")
    refused(so, call(out=P + 8), L.SICU_EINVAL, "aligned")
    refused(so, call(q_stride=255), L.SICU_EINVAL, "stride")
    refused(so, call(table=None), L.SICU_EINVAL, "null table")
    refused(so, call(cu=None), L.SICU_EINVAL, "null table")
    refused(so, call(rope=L.rope(P, P, 8, 66)), L.SICU_EINVAL, "rotated")
    refused(so, call(), L.SICU_EINVAL, "sicu_init")
    n = C.c_size_t(0)
    a = L.kv8_attn(L.T_F32, 4, 3, P, 8, P, P, 2, 2, 100, 0.1)
    refused(so, so.lib.sicu_kv8_attention_ws(C.byref(cache()), C.byref(a), None), L.SICU_EINVAL, "null")
    refused(so, so.lib.sicu_kv8_attention_ws(C.byref(cache()), None, C.byref(n)), L.SICU_EINVAL, "null")
    refused(so, so.lib.sicu_kv8_attention_ws(C.byref(cache()), C.byref(a), C.byref(n)), L.SICU_EINVAL, "sicu_init")
