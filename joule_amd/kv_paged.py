"""Paged KV caches: a pool of pages that all sequences share, new rows normed and
rotated on their way in, and attention over the pages (include/joule_amd.h, "paged
KV caches").

``PagedKVCacheSet`` stands beside ``KVCacheSet`` and ``Q4KVCacheSet`` for hosts
that keep their own projections and serve sequences of very different lengths: a
sequence holds pages for the rows it has, not for the longest it may get, and
sequences may share the pages of a common prefix.
"""

from __future__ import annotations

import ctypes

import torch

from . import _lib
from .decoder import DecoderShape

HD = 128
_DTYPES = {torch.float32: _lib.JM_DTYPE_F32, torch.bfloat16: _lib.JM_DTYPE_BF16}


class PagedKVCacheSet:
    """Caches of B sequences x L layers in n_pages pages of ``page`` rows: one
    tensor ``data`` [L, n_pages, 2, n_kv, page, 128] (k, then v; bfloat16 or
    float32), and ``table`` [B, ceil(maxT / page)] (int32, CUDA), the same for all
    layers: row r of sequence b is row r % page of page table[b, r // page].

    An entry of the table outside [0, n_pages) is no page: rows there are not
    written, and attention does not see them.  ``reserve``, ``share`` and
    ``release`` keep the table, on the current stream, which is that of the calls; a
    host with an allocator of its own writes it instead.  They are for one host thread at a
    time, and not for a stream that is being captured; where one raises, it has changed
    nothing.  ``reserve`` and ``share`` wait for the stream's work where they give out pages
    (they copy page numbers from the host): in a serving loop, reserve for some rows ahead."""

    def __init__(self, shape: DecoderShape, B: int, n_pages: int, page: int = 16, dtype: torch.dtype = torch.bfloat16,
                 device="cuda", data: torch.Tensor | None = None):
        if shape.hd != HD:
            raise ValueError(f"paged caches take a head dim of {HD}, got {shape.hd}")
        if page < 16 or page > 1024 or page & (page - 1):
            raise ValueError(f"page must be a power of two from 16 to 1024, got {page}")
        if B < 0 or n_pages <= 0:
            raise ValueError("B must be >= 0 and n_pages positive")
        L, KH = shape.n_layers, shape.n_kv
        full = (L, n_pages, 2, KH, page, HD)
        if data is None:
            if dtype not in _DTYPES:
                raise ValueError("dtype must be float32 or bfloat16")
            data = torch.zeros(full, dtype=dtype, device=device)
        if data.dtype not in _DTYPES or tuple(data.shape) != full or not data.is_cuda or not data.is_contiguous() \
                or data.data_ptr() % 16:
            raise ValueError(f"cache must be a contiguous 16-byte aligned bfloat16 or float32 CUDA tensor {full}")
        self.shape, self.B, self.n_pages, self.page, self.data = shape, B, n_pages, page, data
        self._device, self._index = data.device, data.get_device()
        width = -(-shape.maxT // page)
        self.table = torch.full((B, width), -1, dtype=torch.int32, device=self._device)
        self._free = list(range(n_pages - 1, -1, -1))
        self._uses = [0] * n_pages
        self._pages: list[list[int]] = [[] for _ in range(B)]
        half = KH * page * HD * data.element_size()
        base = data.data_ptr()
        self._layers = [_lib.KvPaged(base + l * n_pages * 2 * half, base + (l * n_pages * 2 + 1) * half, 2 * half,
                                     self.table.data_ptr(), width, n_pages, page, B, shape.maxT, KH, _DTYPES[data.dtype])
                        for l in range(L)]
        self._refs = [ctypes.byref(x) for x in self._layers]

    # ---------------------------------------------------------------- pages

    def _sequence(self, b: int) -> list[int]:
        if not 0 <= b < self.B:
            raise ValueError(f"sequence {b} outside [0, {self.B})")
        return self._pages[b]

    def _writable(self) -> None:
        # (a captured write is done at each replay, and not now)
        with _lib.on(self._device):
            if torch.cuda.is_current_stream_capturing():
                raise RuntimeError("pages are given out and taken back outside a captured graph")

    def _publish(self, b: int, at: int, pages: list[int]) -> None:
        if pages:
            self.table[b, at:at + len(pages)] = torch.tensor(pages, dtype=torch.int32).to(self._device)

    def free_pages(self) -> int:
        """Pages that no sequence holds."""
        return len(self._free)

    def reserve(self, b: int, rows: int) -> None:
        """Pages for rows 0 .. rows - 1 of sequence b (those that it has stay).
        Raises without taking any where the pool has too few left."""
        have = self._sequence(b)
        if not 0 <= rows <= self.shape.maxT:
            raise ValueError(f"rows {rows} outside [0, maxT={self.shape.maxT}]")
        n = -(-rows // self.page) - len(have)
        if n <= 0:
            return
        if n > len(self._free):
            raise RuntimeError(f"sequence {b} needs {n} more pages, {len(self._free)} are free")
        self._writable()
        got = self._free[:-n - 1:-1]
        self._publish(b, len(have), got)
        del self._free[-n:]
        for p in got:
            self._uses[p] = 1
        have += got

    def share(self, src: int, dst: int, rows: int) -> None:
        """Sequence dst, which has no pages, begins with rows 0 .. rows - 1 of src:
        whole pages are held in common, a page that they fill in part is copied (in
        every layer), so that each may append its own rows behind them."""
        a, b = self._sequence(src), self._sequence(dst)
        if b:
            raise ValueError(f"sequence {dst} has pages already")
        if not 0 <= rows <= len(a) * self.page or rows > self.shape.maxT:
            raise ValueError(f"sequence {src} has pages for {len(a) * self.page} rows, not {rows}")
        whole = rows // self.page
        if rows % self.page and not self._free:
            raise RuntimeError("no page is free for the rows that are copied")
        got = a[:whole]
        if rows:
            self._writable()
        if rows % self.page:
            got.append(self._free[-1])
            self.data[:, got[-1]] = self.data[:, a[whole]]
        self._publish(dst, 0, got)
        if rows % self.page:
            self._free.pop()
        for p in got:
            self._uses[p] += 1
        b += got

    def release(self, b: int) -> None:
        """Give sequence b's pages back (those that others hold stay theirs)."""
        held = self._sequence(b)
        if held:
            self._writable()
            self.table[b] = -1
        for p in held:
            self._uses[p] -= 1
            if self._uses[p] == 0:
                self._free.append(p)
        held.clear()

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
            if not isinstance(t, torch.Tensor) or t.dtype != torch.int32 or t.get_device() != self._index \
                    or t.shape != (size,) or not t.is_contiguous():
                raise ValueError(f"{name} must be a contiguous int32 tensor [{size}] on {self._device}")
        if cu is None and n != self.B:
            raise ValueError(f"without cu there is one token a sequence: {n} tokens, {self.B} sequences")

    def _heads(self, t, name: str, n: int, heads: int, dtype=None) -> None:
        """t is [n, heads, 128] in float32 or bfloat16, its rows contiguous."""
        if not isinstance(t, torch.Tensor) or t.get_device() != self._index or t.dtype not in _DTYPES \
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

    def _vector(self, t, name: str, dtype, rows: int) -> None:
        """t is [rows or more, 128], or [128] where rows is 0."""
        if not isinstance(t, torch.Tensor) or t.dtype != dtype or t.get_device() != self._index or t.dim() != (2 if rows else 1) \
                or t.shape[-1] != HD or (rows and t.shape[0] < rows) or not t.is_contiguous() or t.data_ptr() % 16:
            raise ValueError(f"{name} must be a contiguous 16-byte aligned {dtype} tensor "
                             f"{[rows, HD] if rows else [HD]} on {self._device}")

    # ------------------------------------------------------------ operators

    def append(self, l: int, k: torch.Tensor, v: torch.Tensor, start: torch.Tensor, cu: torch.Tensor | None = None, *,
               q: torch.Tensor | None = None, cos: torch.Tensor | None = None, sin: torch.Tensor | None = None,
               q_norm: torch.Tensor | None = None, k_norm: torch.Tensor | None = None, eps: float = 1e-6,
               q_out: torch.Tensor | None = None, stream=None) -> torch.Tensor | None:
        """k and v [N, KH, 128] into layer l's pages, finished on the way; returns q
        [N, H, 128] finished likewise (None without q).  q, k and v are float32 or
        bfloat16, all of one type, with any strides of tokens and heads that are
        multiples of 4; the pages' type is their own.

        Sequence s has the tokens cu[s] .. cu[s + 1] - 1, at its rows start[s],
        start[s] + 1, ... (int32 CUDA tensors, cu ascending); without cu every
        sequence has one token.  Tokens from cu[B] on, and rows outside [0, maxT),
        are skipped, in q_out too; rows without a page are not written.

        q_norm, k_norm (bfloat16 [128]): each q and k head becomes x / sqrt(mean(x^2)
        + eps) times the weight.  cos, sin (float32 [maxT or more, 128],
        ``decoder.rope_tables``): then each is rotated by halves to its row.  In
        float32, rounded once.  q_out may be q."""
        n = k.shape[0] if isinstance(k, torch.Tensor) and k.dim() == 3 else -1
        KH = self.shape.n_kv
        self._heads(k, "k", n, KH)
        self._heads(v, "v", n, KH, k.dtype)
        self._tokens(start, cu, n)
        H = 0
        if q is not None:
            H = q.shape[1] if isinstance(q, torch.Tensor) and q.dim() == 3 else self.shape.n_heads
            self._heads(q, "q", n, H, k.dtype)
        elif q_out is not None or q_norm is not None:
            raise ValueError("q_out and q_norm need q")
        if (cos is None) != (sin is None):
            raise ValueError("cos and sin come together")
        if cos is not None:
            self._vector(cos, "cos", torch.float32, self.shape.maxT)
            self._vector(sin, "sin", torch.float32, self.shape.maxT)
        if q_norm is not None:
            self._vector(q_norm, "q_norm", torch.bfloat16, 0)
        if k_norm is not None:
            self._vector(k_norm, "k_norm", torch.bfloat16, 0)
        with _lib.on(self._device, stream):
            if q is not None:
                q_out = self._out(q_out, "q_out", (n, H, HD), q.dtype)
            rows = _lib.KvRows(None if q is None else q.data_ptr(), k.data_ptr(), v.data_ptr(),
                               *((0, 0) if q is None else q.stride()[:2]), *k.stride()[:2], *v.stride()[:2], H, _DTYPES[k.dtype],
                               None if q is None else q_out.data_ptr(), None if cos is None else cos.data_ptr(),
                               None if sin is None else sin.data_ptr(), None if q_norm is None else q_norm.data_ptr(),
                               None if k_norm is None else k_norm.data_ptr(), float(eps))
            _lib.check(_lib.lib().jm_kv_paged_append(self._layer(l), start.data_ptr(), None if cu is None else cu.data_ptr(), n,
                                                     ctypes.byref(rows),
                                                     _lib.stream_handle()), "jm_kv_paged_append")
        return q_out

    def attention(self, l: int, q: torch.Tensor, start: torch.Tensor, cu: torch.Tensor | None = None,
                  out: torch.Tensor | None = None, scale: float | None = None, max_rows: int = 0,
                  stream=None) -> torch.Tensor:
        """out [N, H, 128] = softmax(scale q . K) V of q [N, H, 128] (float32 or
        bfloat16) over layer l's rows 0 .. the token's own, which ``append`` has put
        there; H / KH is a whole number from 1 to 16, scale 1 / sqrt(128) unless
        given.  Tokens and rows as in ``append``; a token that sees no row (its own
        below 0, or none with a page) gets 0, other skipped tokens keep what out
        held.  max_rows: at least as many rows as the longest sequence has after the
        call (0: the pages that ``reserve`` and ``share`` gave it, maxT where the host
        writes the table); the call is cut by it, which only rounding shows.  out may be
        q.  With bfloat16 q a weight holds 16 bits, with float32 q 24."""
        n, H = (q.shape[0], q.shape[1]) if isinstance(q, torch.Tensor) and q.dim() == 3 else (-1, self.shape.n_heads)
        self._heads(q, "q", n, H)
        self._tokens(start, cu, n)
        if max_rows < 0:
            raise ValueError("max_rows must be >= 0")
        if max_rows == 0:
            max_rows = max((len(p) for p in self._pages), default=0) * self.page
        with _lib.on(self._device, stream):
            out = self._out(out, "out", (n, H, HD), q.dtype)
            _lib.check(_lib.lib().jm_kv_paged_attn(
                self._layer(l), start.data_ptr(), None if cu is None else cu.data_ptr(), n, q.data_ptr(), *q.stride()[:2], H,
                HD ** -0.5 if scale is None else float(scale), min(max_rows, self.shape.maxT), _DTYPES[q.dtype], out.data_ptr(),
                _lib.stream_handle()), "jm_kv_paged_attn")
        return out
