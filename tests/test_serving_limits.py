"""Sizes past what the 4-bit cache's kernels count or launch are refused before
any HIP call.  CPU only."""

import ctypes

import pytest

from joule_amd import _lib

pytestmark = pytest.mark.skipif(not _lib.LIB_PATH.exists(), reason="libjoule_amd.so not built")
P = 4096                                # stands for a device address, never read


def _cache(n_seq, maxT=100, n_kv=4):
    return ctypes.byref(_lib.KvQ4(P, P, 1 << 40, n_seq, maxT, n_kv, 64))


def test_rows_of_a_cache_are_counted_with_room_for_a_step():
    L = _lib.lib()
    for maxT in (2 ** 31 - 1, 2 ** 31 - 65, 2 ** 31 - 200, 2 ** 31 - 1000):
        assert L.jm_kv_q4_bytes(maxT, 1, 64) == -2, maxT
        assert L.jm_kv_q4_write(_cache(1, maxT), P, None, 1, P, 512, 128, P, 512, 128, 0, None) == -2
    rows = -(-2_147_000_000 // 64) * 64
    assert L.jm_kv_q4_bytes(2_147_000_000, 1, 64) == rows * 68


def test_more_rows_than_a_launch_takes():
    """2^32 threads, 16 a row and head to write and read, 256 a KV head and unit
    to attend."""
    L = _lib.lib()
    N = 1 << 26
    c = _cache(N)
    assert L.jm_kv_q4_write(c, P, None, N, P, 512, 128, P, 512, 128, 0, None) == -2
    assert L.jm_kv_q4_read(c, P, None, N, P, P, 0, None) == -2
    # tokens are rounded up to 4 a head
    c = _cache(1, n_kv=1 << 20)
    assert L.jm_kv_q4_write(c, P, P, 253, P, 512, 128, P, 512, 128, 0, None) == -2
    N = 1 << 24
    assert L.jm_kv_q4_attn(_cache(N), P, None, N, P, 1024, 128, 8, 0.1, 0, P, None) == -2
    assert b"launch" in L.jm_last_error()
    assert L.jm_kv_q4_attn(_cache(1 << 20), P, P, (1 << 26) - 64, P, 1024, 128, 4, 0.1, 1, P, None) == -2


def test_scales_that_overflow_with_the_exponentials_base():
    L = _lib.lib()
    for scale in (3e38, -3e38, float("inf"), float("nan")):
        assert L.jm_kv_q4_attn(_cache(2), P, None, 2, P, 1024, 128, 8, scale, 0, P, None) == -1
