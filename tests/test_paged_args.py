"""Argument checks of the paged KV caches and their page keeping.  CPU only: every
refusal comes before any HIP call, and calls with nothing to do return 0."""

import ctypes

import pytest

from joule_amd import _lib

pytestmark = pytest.mark.skipif(not _lib.LIB_PATH.exists(), reason="libjoule_amd.so not built")
P = 4096                                # stands for a device address, never read
PAGE_BYTES = 4 * 32 * 128 * 2


def _cache(**kw):
    a = dict(k=P, v=P, page_stride=2 * PAGE_BYTES, table=P, table_stride=4, n_pages=9, page=32, n_seq=2, maxT=100, n_kv=4, dtype=1)
    a.update(kw)
    return _lib.KvPaged(*(a[n] for n, _ in _lib.KvPaged._fields_))


def _rows(**kw):
    a = dict(q=P, k=P, v=P, q_token=1024, q_head=128, k_token=512, k_head=128, v_token=512, v_head=128, n_heads=8, dtype=0,
             q_out=P, cos=P, sin=P, q_norm=P, k_norm=P, eps=1e-6)
    a.update(kw)
    return _lib.KvRows(*(a[n] for n, _ in _lib.KvRows._fields_))


def _append(c, N=2, start=P, cu=None, **kw):
    return _lib.lib().jm_kv_paged_append(c, start, cu, N, ctypes.byref(_rows(**kw)), None)


def _attn(c, N=2, start=P, cu=None, q=P, q_token=1024, q_head=128, H=8, scale=0.1, max_rows=0, dtype=0, out=P):
    return _lib.lib().jm_kv_paged_attn(c, start, cu, N, q, q_token, q_head, H, scale, max_rows, dtype, out, None)


@pytest.mark.parametrize("call", [_append, _attn])
def test_cache_refusals(call):
    for kw, code in ((dict(page=0), -2), (dict(page=8), -2), (dict(page=48), -2), (dict(page=2048), -2), (dict(page=-16), -2),
                     (dict(maxT=0), -2), (dict(maxT=2 ** 31 - 1), -2), (dict(n_kv=0), -2), (dict(n_kv=1025), -2),
                     (dict(n_seq=-1), -2), (dict(n_pages=-1), -2), (dict(n_pages=0), -2), (dict(dtype=2), -1),
                     (dict(k=None), -1), (dict(v=None), -1), (dict(table=None), -1), (dict(k=P + 8), -1), (dict(table=P + 2), -1),
                     (dict(page_stride=PAGE_BYTES + 8), -1), (dict(page_stride=PAGE_BYTES - 16), -2),
                     (dict(page_stride=1 << 41), -1), (dict(page_stride=PAGE_BYTES, dtype=0), -2),
                     (dict(table_stride=3), -2), (dict(table_stride=-4), -2)):
        assert call(ctypes.byref(_cache(**kw))) == code, kw
        assert _lib.lib().jm_last_error()
    c = ctypes.byref(_cache())
    assert call(None) == -1
    assert call(c, N=-1) == -1
    assert call(c, N=3) == -2                       # without cu one token a sequence
    assert call(c, start=None) == -1
    assert call(c, start=P + 2) == -1
    assert call(c, N=5, cu=P + 1) == -1
    assert call(c, N=1 << 30, cu=P) == -2           # more than one launch's threads
    assert call(c, dtype=2) == -1 and call(c, dtype=-1) == -1
    # nothing to do: no pointer is looked at
    assert call(c, N=0, cu=P) == 0
    assert call(ctypes.byref(_cache(n_seq=0, k=None, v=None, table=None)), N=0, start=None) == 0


def test_row_refusals():
    c = ctypes.byref(_cache())
    for name in ("k", "v", "q_out"):
        assert _append(c, **{name: None}) == -1, name
    for name in ("q", "k", "v", "q_out"):
        assert _append(c, **{name: P + 8}) == -1, name              # float32: 16 bytes
        assert _append(c, dtype=1, **{name: P + 4}) == -1, name     # bf16: 8 bytes
    for name in ("q_token", "q_head", "k_token", "k_head", "v_token", "v_head"):
        assert _append(c, **{name: 130}) == -1, name
    for name in ("cos", "sin"):
        assert _append(c, **{name: None}) == -1, name               # together or not at all
    for name in ("cos", "sin", "q_norm", "k_norm"):
        assert _append(c, **{name: P + 8}) == -1, name
    for eps in (float("nan"), float("inf"), -1e-6):
        assert _append(c, eps=eps) == -1
    for H in (0, -1, 65):
        assert _append(c, n_heads=H) == -2
    assert _lib.lib().jm_kv_paged_append(c, P, None, 2, None, None) == -1


def test_attention_refusals():
    c = ctypes.byref(_cache())
    for name in ("q", "out"):
        assert _attn(c, **{name: None}) == -1
        assert _attn(c, **{name: P + 8}) == -1
        assert _attn(c, dtype=1, **{name: P + 4}) == -1
    for name in ("q_token", "q_head"):
        assert _attn(c, **{name: 130}) == -1
    for H in (0, -4, 3, 6, 68, 128):
        assert _attn(c, H=H) == -2, H
    for scale in (float("nan"), float("inf"), 3e38):
        assert _attn(c, scale=scale) == -1
    assert _attn(c, max_rows=-1) == -1
