"""Argument checks of the 4-bit KV cache and of sampling.  CPU only: every
refusal comes before any HIP call, and calls with nothing to do return 0."""

import ctypes

import pytest

from joule_amd import _lib

pytestmark = pytest.mark.skipif(not _lib.LIB_PATH.exists(), reason="libjoule_amd.so not built")
P = 4096                                # stands for a device address, never read


def _cache(**kw):
    a = dict(k=P, v=P, seq_stride=1 << 20, n_seq=2, maxT=100, n_kv=4, group=64)
    a.update(kw)
    return _lib.KvQ4(*(a[n] for n in ("k", "v", "seq_stride", "n_seq", "maxT", "n_kv", "group")))


def test_plane_bytes():
    L = _lib.lib()
    # rows up to a multiple of 64, 64 bytes of codes and 2 or 4 fp16 scales a row and head
    assert L.jm_kv_q4_bytes(100, 4, 64) == 128 * 4 * 68
    assert L.jm_kv_q4_bytes(64, 1, 32) == 64 * 72
    assert L.jm_kv_q4_bytes(65, 3, 32) == 128 * 3 * 72
    assert L.jm_kv_q4_bytes(2_000_000, 64, 64) == 2_000_000 * 64 * 68      # past 32 bits
    for bad in ((0, 4, 64), (-1, 4, 64), (100, 0, 64), (100, 4, 16), (100, 4, 128), (2 ** 31 - 1, 4, 64)):
        assert L.jm_kv_q4_bytes(*bad) == -2, bad
        assert L.jm_last_error()


def _write(c, N=2, start=P, cu=None, k=P, kt=512, kh=128, v=P, vt=512, vh=128, dtype=0):
    return _lib.lib().jm_kv_q4_write(c, start, cu, N, k, kt, kh, v, vt, vh, dtype, None)


def _read(c, N=2, start=P, cu=None, k=P, v=P, dtype=0):
    return _lib.lib().jm_kv_q4_read(c, start, cu, N, k, v, dtype, None)


def _attn(c, N=2, start=P, cu=None, q=P, qt=1024, qh=128, H=8, scale=0.1, dtype=0, out=P):
    return _lib.lib().jm_kv_q4_attn(c, start, cu, N, q, qt, qh, H, scale, dtype, out, None)


@pytest.mark.parametrize("call", [_write, _read, _attn])
def test_cache_refusals(call):
    for kw, code in ((dict(group=48), -2), (dict(group=0), -2), (dict(maxT=0), -2), (dict(n_kv=0), -2),
                     (dict(n_seq=-1), -2), (dict(k=None), -1), (dict(v=None), -1), (dict(k=P + 8), -1),
                     (dict(seq_stride=100), -1), (dict(seq_stride=128 * 4 * 68 - 16), -2)):
        c = _cache(**kw)
        assert call(ctypes.byref(c)) == code, kw
        assert _lib.lib().jm_last_error()
    c = ctypes.byref(_cache())
    assert call(None) == -1
    assert call(c, N=-1) == -1
    assert call(c, N=3) == -2                       # without cu one token a sequence
    assert call(c, N=2, start=None) == -1
    assert call(c, N=2, start=P + 2) == -1
    assert call(c, N=5, cu=P + 1) == -1
    assert call(c, N=1 << 30, cu=P) == -2           # N * n_kv past 32 bits
    assert call(c, dtype=2) == -1 and call(c, dtype=-1) == -1
    # nothing to do: no pointer is looked at
    assert call(c, N=0, cu=P) == 0
    assert call(ctypes.byref(_cache(n_seq=0, k=None, v=None)), N=0, start=None) == 0


def test_tensor_refusals():
    c = ctypes.byref(_cache())
    for call, name in ((_write, "k"), (_write, "v"), (_read, "k"), (_read, "v"), (_attn, "q"), (_attn, "out")):
        assert call(c, **{name: None}) == -1
        assert call(c, **{name: P + 8}) == -1       # float32: 16 bytes
        assert call(c, dtype=1, **{name: P + 4}) == -1      # bf16: 8 bytes
    for call, name in ((_write, "kt"), (_write, "kh"), (_write, "vt"), (_write, "vh"), (_attn, "qt"), (_attn, "qh")):
        assert call(c, **{name: 130}) == -1


def test_attention_refusals():
    c = ctypes.byref(_cache())
    for H in (0, -4, 3, 6, 12, 64):
        assert _attn(c, H=H) == -2, H
    for scale in (float("nan"), float("inf")):
        assert _attn(c, scale=scale) == -1


def _sample(how=None, logits=P, dtype=0, ld=100, B=1, V=100, u=P, tok=P, p=P):
    how = _lib.Sampling(1.0, 0, 1.0, 0.0) if how is None else how
    return _lib.lib().jm_sample(logits, dtype, ld, B, V, ctypes.byref(how) if how else None, u, tok, p, None)


def test_sample_refusals():
    nan = float("nan")
    for kw, code in ((dict(dtype=2), -1), (dict(B=-1), -1), (dict(V=0), -2), (dict(V=(1 << 20) + 1, ld=1 << 21), -2),
                     (dict(ld=99), -2), (dict(how=False), -1), (dict(logits=None), -1), (dict(u=None), -1),
                     (dict(tok=None), -1), (dict(logits=P + 2), -1), (dict(logits=P + 1, dtype=1), -1),
                     (dict(u=P + 2), -1), (dict(tok=P + 1), -1), (dict(p=P + 2), -1),
                     (dict(how=_lib.Sampling(nan, 0, 1.0, 0.0)), -1), (dict(how=_lib.Sampling(1.0, 0, nan, 0.0)), -1),
                     (dict(how=_lib.Sampling(1.0, 0, 1.0, nan)), -1),
                     (dict(how=_lib.Sampling(1.0, 0, 1.0, 0.0, P + 1)), -1)):
        assert _sample(**kw) == code, kw
        assert _lib.lib().jm_last_error()
    assert _sample(B=0, logits=None, u=None, tok=None) == 0


def test_kv_dtype_setting_refuses_a_null_store():
    assert _lib.lib().jm_store_set_kv_dtype(None, _lib.JM_DTYPE_Q4) == -1
