"""Rows finished for a paged cache and attention over its pages, in float64, and how
far an output may be from them.

TEST INFRASTRUCTURE ONLY: the oracle of the tests.  The product path
(joule_amd) never imports it.

With p_t the weights, v_t the values, o the output and A_t = |scale| sum_i |q_i k_ti|, an
error of e_t in the logarithm of each weight and of f_t relative in each weight's
product moves dimension d by at most  sum_t p_t (e_t + f_t) (|v_td| + |o_d|) .  What the
library's header states gives, n being the rows that a token sees:

  every form     e_t = 2^-17 A_t + 2^-20: a float32 sum of 128 products (at most 2^-24
                 of A_t each), the scale and the exponential; f_t = (n + 64) 2^-24: a
                 float32 sum of n products and of n weights
  bf16           weights in two parts, 2^-17; the output, 2^-8 of it
  bf16 prompt    a looser bound, of weights rounded once, 2^-8 (their sum that of the
                 rounded ones: a common factor drops out, the difference of two values is
                 what counts, which |v| + |o| covers)
"""

from __future__ import annotations

import numpy as np

HD = 128


def finish(x: np.ndarray, rows: np.ndarray, w, cos, sin, eps: float) -> np.ndarray:
    """Heads x [N, heads, 128] normed by w (or None) and rotated to their rows by
    the tables (or None)."""
    x = x.astype(np.float64)
    if w is not None:
        x = x / np.sqrt((x * x).mean(axis=-1, keepdims=True) + eps) * w.astype(np.float64)
    if cos is not None:
        c, s = cos[rows].astype(np.float64)[:, None], sin[rows].astype(np.float64)[:, None]
        x = x * c + np.concatenate([-x[..., HD // 2:], x[..., :HD // 2]], axis=-1) * s
    return x


def attend(q: np.ndarray, k: np.ndarray, v: np.ndarray, see: np.ndarray, scale: float, form: str):
    """(o, bound) [n, 128] of query rows q [n, 128] over rows k, v [T, 128]; see [n, T]
    says which each sees (rows that none sees may hold anything).  0 where none."""
    used = see.any(axis=0)
    q, k, v, see = q.astype(np.float64), k[used].astype(np.float64), v[used].astype(np.float64), see[:, used]
    a = np.where(see, q @ k.T * scale, -np.inf)
    top = a.max(axis=1, keepdims=True, initial=-np.inf)
    p = np.where(see, np.exp(a - np.where(np.isfinite(top), top, 0.0)), 0.0)
    p /= np.where(see.any(axis=1), p.sum(axis=1), 1.0)[:, None]
    o = p @ v
    n = see.sum(axis=1, keepdims=True)
    e = 2.0 ** -17 * (np.abs(q) @ np.abs(k).T * abs(scale)) + 2.0 ** -20 + (n + 64) * 2.0 ** -24
    if form != "f32":
        e = e + (2.0 ** -17 if form == "bf16" else 2.0 ** -8)
    off = (p * e) @ np.abs(v) + (p * e).sum(axis=1, keepdims=True) * np.abs(o)
    if form != "f32":
        off += 2.0 ** -8 * np.abs(o)
    return o, off
