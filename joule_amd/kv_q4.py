"""4-bit KV caches: rows quantised as they are written, read back, and attended
over (include/joule_amd.h, "the 4-bit KV cache").

``Q4KVCacheSet`` stands beside ``KVCacheSet``: it holds the caches of B
sequences x L layers and goes wherever that one goes in ``HipDecoder``
(decode and prefill calls append to it and attend over it), with 68 or 72
bytes a row and head for k and v instead of bf16's 256.  A host that keeps its
own projections calls ``write``, ``read`` and ``attention`` itself.

A row of a head is the expert store's Q4 format (``q4_store.quantize`` of its
128 values); how the codes lie in memory is the library's own, so the planes
are read and written only through these calls.
"""

from __future__ import annotations

import ctypes

import torch

from . import _lib
from .decoder import DecoderShape, KVCache

HD = 128
_DTYPES = {torch.float32: _lib.JM_DTYPE_F32, torch.bfloat16: _lib.JM_DTYPE_BF16}


class Q4KVCacheSet:
    """4-bit caches for B sequences x L layers: one uint8 tensor
    [B, L, 2, plane bytes] and the KVCache[B*L] array (entry b*L + l) that
    points into it.  ``group`` values share a scale: 64, or 32 for closer
    values at 6 % more bytes."""

    def __init__(self, shape: DecoderShape, B: int, group: int = 64, device="cuda", data: torch.Tensor | None = None):
        if shape.hd != HD:
            raise ValueError(f"4-bit caches take a head dim of {HD}, got {shape.hd}")
        plane = int(_lib.lib().jm_kv_q4_bytes(int(shape.maxT), int(shape.n_kv), int(group)))
        if plane < 0:
            _lib.check(plane, "jm_kv_q4_bytes")
        L = shape.n_layers
        full = (B, L, 2, plane)
        if data is None:
            data = torch.zeros(full, dtype=torch.uint8, device=device)
        if data.dtype != torch.uint8 or tuple(data.shape) != full or not data.is_cuda or not data.is_contiguous() \
                or data.data_ptr() % 16:
            raise ValueError(f"cache must be a contiguous 16-byte aligned uint8 CUDA tensor {full}")
        self.shape, self.B, self.group, self.data = shape, B, group, data
        self._device = data.device
        base, seq = data.data_ptr(), L * 2 * plane
        self.table = (KVCache * (B * L))()
        for b in range(B):
            for l in range(L):
                self.table[b * L + l].k = base + b * seq + l * 2 * plane
                self.table[b * L + l].v = base + b * seq + l * 2 * plane + plane
        self._layers = [_lib.KvQ4(base + l * 2 * plane, base + l * 2 * plane + plane, seq, B, shape.maxT, shape.n_kv, group)
                        for l in range(L)]
        self._refs = [ctypes.byref(x) for x in self._layers]

    # ------------------------------------------------------------ arguments

    def _layer(self, l: int):
        if not 0 <= l < len(self._layers):
            raise ValueError(f"layer {l} outside [0, {len(self._layers)})")
        return self._refs[l]

    def _tokens(self, start, cu, n: int) -> None:
        """start [B] and cu [B + 1] (or None: one token a sequence)."""
        for t, name, size in ((start, "start", self.B), (cu, "cu", self.B + 1)):
            if t is None and name == "cu":
                continue
            if not isinstance(t, torch.Tensor) or t.dtype != torch.int32 or t.device != self._device \
                    or t.shape != (size,) or not t.is_contiguous():
                raise ValueError(f"{name} must be a contiguous int32 tensor [{size}] on {self._device}")
        if cu is None and n != self.B:
            raise ValueError(f"without cu there is one token a sequence: {n} tokens, {self.B} sequences")

    def _heads(self, t, name: str, n: int, heads: int, dtype=None) -> None:
        """t is [n, heads, 128] in float32 or bfloat16, its rows contiguous."""
        if not isinstance(t, torch.Tensor) or t.device != self._device or t.dtype not in _DTYPES \
                or (dtype is not None and t.dtype != dtype):
            raise ValueError(f"{name} must be a {'float32 or bfloat16' if dtype is None else dtype} tensor "
                             f"on {self._device}")
        if t.shape != (n, heads, HD):
            raise ValueError(f"{name} must be [{n}, {heads}, {HD}], got {list(t.shape)}")
        ts, hs, one = t.stride()
        if n and (one != 1 or ts % 4 or hs % 4 or t.data_ptr() % (16 if t.dtype == torch.float32 else 8)):
            raise ValueError(f"{name}: rows of {HD} contiguous values, strides and address multiples of 4 elements")

    def _out(self, t, name: str, shape: tuple, dtype):
        if t is None:
            return torch.empty(shape, dtype=dtype, device=self._device)
        self._heads(t, name, shape[0], shape[1], dtype)
        if not t.is_contiguous():
            raise ValueError(f"{name} must be contiguous")
        return t

    # ------------------------------------------------------------ operators

    def write(self, l: int, k: torch.Tensor, v: torch.Tensor, start: torch.Tensor, cu: torch.Tensor | None = None,
              stream=None) -> None:
        """Quantise k and v [N, KH, 128] (float32 or bfloat16; any strides of
        tokens and heads that are multiples of 4) into layer l's caches.

        Sequence s has the tokens cu[s] .. cu[s + 1] - 1, at its rows start[s],
        start[s] + 1, ... (int32 CUDA tensors, cu ascending); without cu every
        sequence has one token.  Tokens from cu[B] on, and rows outside
        [0, maxT), are skipped.  A group with a NaN, an infinity or a magnitude
        of 458640 or more reads back as NaN."""
        n = k.shape[0] if isinstance(k, torch.Tensor) and k.dim() == 3 else -1
        self._heads(k, "k", n, self.shape.n_kv)
        self._heads(v, "v", n, self.shape.n_kv, k.dtype)
        self._tokens(start, cu, n)
        with _lib.on(self._device, stream):
            _lib.check(_lib.lib().jm_kv_q4_write(
                self._layer(l), _lib.ptr(start), _lib.ptr(cu), n, _lib.ptr(k), *k.stride()[:2],
                _lib.ptr(v), *v.stride()[:2], _DTYPES[k.dtype], _lib.stream_handle()), "jm_kv_q4_write")

    def read(self, l: int, start: torch.Tensor, cu: torch.Tensor | None = None, n: int | None = None,
             dtype: torch.dtype = torch.float32, k: torch.Tensor | None = None, v: torch.Tensor | None = None,
             stream=None) -> tuple[torch.Tensor, torch.Tensor]:
        """(k, v) [n, KH, 128]: the values of the cache rows that ``write``
        with the same start and cu writes, exact in float32, rounded in
        bfloat16.  n is the number of tokens (with cu; without: B).  Rows of the
        outputs whose token is skipped keep what they held."""
        if n is None:
            if cu is not None:
                raise ValueError("with cu, n says how many tokens there are")
            n = self.B
        if n < 0:
            raise ValueError("n must be >= 0")
        if dtype not in _DTYPES:
            raise ValueError("dtype must be float32 or bfloat16")
        self._tokens(start, cu, n)
        with _lib.on(self._device, stream):
            k = self._out(k, "k", (n, self.shape.n_kv, HD), dtype)
            v = self._out(v, "v", (n, self.shape.n_kv, HD), dtype)
            _lib.check(_lib.lib().jm_kv_q4_read(
                self._layer(l), _lib.ptr(start), _lib.ptr(cu), n, _lib.ptr(k), _lib.ptr(v), _DTYPES[dtype],
                _lib.stream_handle()), "jm_kv_q4_read")
        return k, v

    def attention(self, l: int, q: torch.Tensor, start: torch.Tensor, cu: torch.Tensor | None = None,
                  out: torch.Tensor | None = None, scale: float | None = None, stream=None) -> torch.Tensor:
        """out [N, H, 128] = softmax(scale q . K) V of q [N, H, 128] (float32 or
        bfloat16) over layer l's rows 0 .. the token's own, which ``write`` has
        put there; H / KH is 1, 2, 4 or 8, scale 1 / sqrt(128) unless given.
        Tokens and rows as in ``write``; a token whose row is below 0 gets 0,
        other skipped tokens keep what out held.  out may be q."""
        n, H = (q.shape[0], q.shape[1]) if isinstance(q, torch.Tensor) and q.dim() == 3 else (-1, self.shape.n_heads)
        self._heads(q, "q", n, H)
        self._tokens(start, cu, n)
        with _lib.on(self._device, stream):
            out = self._out(out, "out", (n, H, HD), q.dtype)
            _lib.check(_lib.lib().jm_kv_q4_attn(
                self._layer(l), _lib.ptr(start), _lib.ptr(cu), n, _lib.ptr(q), *q.stride()[:2], H,
                HD ** -0.5 if scale is None else float(scale), _DTYPES[q.dtype], _lib.ptr(out),
                _lib.stream_handle()), "jm_kv_q4_attn")
        return out
