"""Which kind of cache a store's calls take, where several decoders share the
store.  CPU only: the library is replaced by one that records the setting."""

import ctypes
from types import SimpleNamespace

import pytest
import torch

from joule_amd import _lib
from joule_amd.decoder import DecoderShape, HipDecoder
from joule_amd.dense import dense_ffn_shape


class _Lib:
    """The setting of each store, as jm_store_set_kv_dtype leaves it."""

    def __init__(self):
        self.kind = {}

    def jm_store_set_kv_dtype(self, store, dtype):
        self.kind[store.value] = dtype
        return 0


def _decoder(store):
    d = HipDecoder.__new__(HipDecoder)
    d.store, d.shape = store, DecoderShape(n_layers=1, moe=dense_ffn_shape(1024, 512), n_heads=8, n_kv=2, maxT=64)
    return d


def _caches(shape, dtype, group=64):
    return SimpleNamespace(data=torch.empty(0, dtype=dtype), shape=shape, group=group)


def test_decoders_over_one_store_set_their_own_kind(monkeypatch):
    """Each call's kind holds for it, whatever another decoder over the same
    store set in between: a 4-bit plane taken for a bf16 cache would be written
    past its end."""
    lib = _Lib()
    monkeypatch.setattr(_lib, "lib", lambda: lib)
    store = SimpleNamespace(_h=ctypes.c_void_p(1))
    a, b = _decoder(store), _decoder(store)
    kinds = [(torch.uint8, 64, _lib.JM_DTYPE_Q4), (torch.bfloat16, 0, _lib.JM_DTYPE_BF16),
             (torch.uint8, 32, _lib.JM_DTYPE_Q4_G32), (torch.float32, 0, _lib.JM_DTYPE_F32)]
    for da, ga, want_a in kinds:
        for db, gb, want_b in kinds:
            for _ in range(2):
                a._kv_dtype(_caches(a.shape, da, ga))
                assert lib.kind[1] == want_a
                b._kv_dtype(_caches(b.shape, db, gb))
                assert lib.kind[1] == want_b


def test_4_bit_caches_of_another_shape_are_refused(monkeypatch):
    monkeypatch.setattr(_lib, "lib", _Lib)
    d = _decoder(SimpleNamespace(_h=ctypes.c_void_p(1)))
    for kw in (dict(maxT=128), dict(n_kv=4), dict(n_layers=2)):
        shape = dict(n_layers=1, moe=dense_ffn_shape(1024, 512), n_heads=8, n_kv=2, maxT=64)
        with pytest.raises(ValueError):
            d._kv_dtype(_caches(DecoderShape(**{**shape, **kw}), torch.uint8))
