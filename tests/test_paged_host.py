"""The paged and sampling entry points refuse bad arguments before any GPU work."""
from __future__ import annotations

import ctypes

import pytest

from tinyserve_b200 import _lib

P = 1 << 20  # stands for an aligned device pointer; never dereferenced here


def cache(**kw):
    a = dict(k_cache=P, v_cache=P, page_stride=16 * 64, head_stride=0, row_stride=64, num_pages=4, page_size=16,
             n_kv_heads=1, head_dim=64, dtype=_lib.DT_BF16, cache_fp8=0) | kw
    return _lib.TsbPagedCache(**a)


def batch(**kw):
    a = dict(page_table=P, cu_q=P, kv_lens=P, table_stride=4, table_width=4, n_seqs=1, n_tokens=2, max_q=2) | kw
    return _lib.TsbPagedBatch(**a)


def attention(c=None, b=None, q=P, ts=512, hs=64, nq=8, window=0, keep=0, out=P, ws=P, nbytes=1 << 30):
    return _lib.lib().tsb_paged_attention(ctypes.byref(c or cache()), ctypes.byref(b or batch()), q, ts, hs, nq,
                                          window, keep, None, 0.125, out, ws, nbytes, None)


@pytest.mark.parametrize("kw,code,text", [
    (dict(c=cache(head_dim=96)), _lib.TSB_ERR_UNSUPPORTED, "head_dim"),
    (dict(c=cache(dtype=_lib.DT_F32)), _lib.TSB_ERR_UNSUPPORTED, "dtype"),
    (dict(c=cache(cache_fp8=2)), _lib.TSB_ERR_INVALID, "cache_fp8"),
    (dict(c=cache(page_size=0)), _lib.TSB_ERR_INVALID, "page_size"),
    (dict(c=cache(row_stride=65)), _lib.TSB_ERR_INVALID, "strides"),
    (dict(c=cache(row_stride=72, cache_fp8=1)), _lib.TSB_ERR_INVALID, "strides"),
    (dict(c=cache(page_stride=-1024)), _lib.TSB_ERR_INVALID, "strides"),
    (dict(c=cache(k_cache=P + 2)), _lib.TSB_ERR_INVALID, "aligned"),
    (dict(c=cache(k_cache=None)), _lib.TSB_ERR_INVALID, "null"),
    (dict(nq=0), _lib.TSB_ERR_INVALID, "n_q_heads"),
    (dict(c=cache(n_kv_heads=3)), _lib.TSB_ERR_INVALID, "n_q_heads"),
    (dict(b=batch(n_tokens=-1)), _lib.TSB_ERR_INVALID, "batch"),
    (dict(b=batch(table_stride=3)), _lib.TSB_ERR_INVALID, "batch"),
    (dict(b=batch(table_width=1 << 29, table_stride=1 << 29)), _lib.TSB_ERR_UNSUPPORTED, "table"),
    (dict(b=batch(cu_q=None)), _lib.TSB_ERR_INVALID, "null"),
    (dict(q=None), _lib.TSB_ERR_INVALID, "null"), (dict(out=None), _lib.TSB_ERR_INVALID, "null"),
    (dict(q=P + 8), _lib.TSB_ERR_INVALID, "aligned"), (dict(ts=515), _lib.TSB_ERR_INVALID, "strides"),
    (dict(window=-1), _lib.TSB_ERR_INVALID, "window"), (dict(keep=-1), _lib.TSB_ERR_INVALID, "keep_first"),
    (dict(ws=None), _lib.TSB_ERR_INVALID, "null"), (dict(ws=P + 16), _lib.TSB_ERR_INVALID, "workspace"),
    (dict(nbytes=64), _lib.TSB_ERR_WORKSPACE, "workspace"),
])
def test_attention_refusals(kw, code, text):
    assert attention(**kw) == code
    assert text in _lib.last_error()


def test_empty_batches_are_done_at_once():
    assert attention(b=batch(n_tokens=0)) == _lib.TSB_OK
    assert attention(b=batch(n_seqs=0)) == _lib.TSB_OK


def test_workspace_sizes():
    L = _lib.lib()
    assert L.tsb_paged_workspace(64) > 0 and L.tsb_paged_workspace(128) > 0
    assert L.tsb_paged_workspace(80) == 0


def test_store_refusals():
    L = _lib.lib()

    def store(qkv=P, stride=640, nq=8, cos=P, table=_lib.DT_F32, out=P):
        return L.tsb_paged_kv_store(ctypes.byref(cache()), ctypes.byref(batch()), qkv, stride, nq, cos, P, table, 64,
                                    out, P, 1 << 30, None)

    for kw, code in ((dict(qkv=None), 1), (dict(cos=None), 1), (dict(out=None), 1), (dict(stride=632), 1),
                     (dict(stride=644), 1), (dict(qkv=P + 2), 1), (dict(table=7), 2), (dict(nq=0), 1)):
        assert store(**kw) == code, kw


def test_sample_refusals():
    L = _lib.lib()

    def sample(x=P, dt=0, rows=2, vocab=8, stride=8, noise=P, ns=8, tokens=P):
        return L.tsb_sample(x, dt, rows, vocab, stride, noise, ns, None, None, None, None, tokens, None, None)

    for kw, code in ((dict(dt=7), 2), (dict(rows=-1), 1), (dict(vocab=0), 1), (dict(stride=7), 1), (dict(ns=7), 1),
                     (dict(x=None), 1), (dict(tokens=None), 1)):
        assert sample(**kw) == code, kw
    assert sample(rows=0) == 0


def test_pointers_off_their_type_are_refused():
    """An element that crosses its own alignment would fault on the device."""
    L = _lib.lib()
    for dt, off in ((_lib.DT_F32, 2), (_lib.DT_BF16, 1), (_lib.DT_F16, 1)):
        assert L.tsb_sample(P + off, dt, 2, 8, 8, P, 8, None, None, None, None, P, None, None) == _lib.TSB_ERR_INVALID
        assert "aligned" in _lib.last_error()
    for at in range(5, 13):
        if at == 6:  # noise_stride
            continue
        a = [P, 0, 2, 8, 8, P, 8, P, P, P, P, P, P, None]
        a[at] = P + (4 if at == 11 else 2)
        assert L.tsb_sample(*a) == _lib.TSB_ERR_INVALID, at
        assert "aligned" in _lib.last_error()
    for name in ("page_table", "cu_q", "kv_lens"):
        assert attention(b=batch(**{name: P + 2})) == _lib.TSB_ERR_INVALID
        assert "aligned" in _lib.last_error()
    rc = L.tsb_paged_attention(ctypes.byref(cache()), ctypes.byref(batch()), P, 512, 64, 8, 0, 0, P + 2, 0.125, P, P,
                               1 << 30, None)
    assert rc == _lib.TSB_ERR_INVALID and "aligned" in _lib.last_error()


def test_store_refuses_pools_whose_rows_overlap():
    """An expanded pool has one place for several heads' (rows', pages') values; reading one is fine."""
    L = _lib.lib()

    def store(c):
        return L.tsb_paged_kv_store(ctypes.byref(c), ctypes.byref(batch()), P, 1280, 8, P, P, _lib.DT_F32, 64, P, P,
                                    1 << 30, None)

    ok = dict(n_kv_heads=2, page_stride=2 * 16 * 64, head_stride=16 * 64, row_stride=64)
    for kw in (dict(head_stride=0), dict(row_stride=0), dict(page_stride=0), dict(row_stride=32)):
        assert store(cache(**ok | kw)) == _lib.TSB_ERR_INVALID, kw
        assert "overlap" in _lib.last_error()
