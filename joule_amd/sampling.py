"""The next token of each row of logits under temperature, top-k, top-p and
min-p, drawn with given random numbers (jm_sample in include/joule_amd.h, which
defines the draw: whole-number weights, so that a token never depends on an
order of summation)."""

from __future__ import annotations

import ctypes

import torch

from . import _lib
from .moe import check_tensor

_DTYPES = {torch.float32: _lib.JM_DTYPE_F32, torch.bfloat16: _lib.JM_DTYPE_BF16}


def sample(logits: torch.Tensor, u: torch.Tensor, temperature: float | torch.Tensor = 1.0,
           top_k: int | torch.Tensor = 0, top_p: float | torch.Tensor = 1.0, min_p: float | torch.Tensor = 0.0,
           out_tok: torch.Tensor | None = None, out_p: torch.Tensor | None = None,
           stream=None) -> tuple[torch.Tensor, torch.Tensor]:
    """(tokens int32 [B], probabilities float32 [B]) of logits [B, V] (float32
    or bfloat16, rows of any stride) with the random numbers u [B] (float32,
    in [0, 1)).  Each setting is a number for all rows or a CUDA tensor [B]
    (float32; top_k int32).

    The tokens are ordered by logit (ties: the lower index first) and weighted
    by exp(logit / temperature).  top_k keeps the first top_k (0: all), top_p
    of these those before which less than top_p of the weight lies (1: all),
    min_p of these those of at least min_p times the largest weight (0: all);
    the first always stays.  u in [0, 1) picks along that order: 0 is the
    argmax.  A temperature of 0 takes the argmax.  A NaN logit counts as
    -infinity; a row without any logit above -infinity gives token -1,
    probability 0."""
    if not isinstance(logits, torch.Tensor) or not logits.is_cuda or logits.dim() != 2 or logits.dtype not in _DTYPES:
        raise ValueError("logits must be a float32 or bfloat16 CUDA tensor [B, V]")
    B, V = logits.shape
    if logits.numel() and (logits.stride(1) != 1 or (B > 1 and logits.stride(0) < V)):
        raise ValueError("logits: rows must be contiguous and apart")
    dev = logits.device
    check_tensor(u, "u", (B,), torch.float32, dev)
    how = _lib.Sampling(1.0, 0, 1.0, 0.0)
    for name, value, dtype in (("temperature", temperature, torch.float32), ("top_k", top_k, torch.int32),
                               ("top_p", top_p, torch.float32), ("min_p", min_p, torch.float32)):
        if isinstance(value, torch.Tensor):
            check_tensor(value, name, (B,), dtype, dev)
            setattr(how, name + "_b", value.data_ptr())
        elif name == "top_k":
            if not -2 ** 31 <= int(value) < 2 ** 31:
                raise ValueError("top_k must fit 32 bits")
            how.top_k = int(value)
        else:
            setattr(how, name, float(value))
    with _lib.on(dev, stream):
        if out_tok is None:
            out_tok = torch.empty(B, dtype=torch.int32, device=dev)
        else:
            check_tensor(out_tok, "out_tok", (B,), torch.int32, dev)
        if out_p is None:
            out_p = torch.empty(B, dtype=torch.float32, device=dev)
        else:
            check_tensor(out_p, "out_p", (B,), torch.float32, dev)
        _lib.check(_lib.lib().jm_sample(_lib.ptr(logits), _DTYPES[logits.dtype], max(V, logits.stride(0)), B, V,
                                        ctypes.byref(how), _lib.ptr(u), _lib.ptr(out_tok), _lib.ptr(out_p),
                                        _lib.stream_handle()), "jm_sample")
    return out_tok, out_p
