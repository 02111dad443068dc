"""softmax(scale q . K) V in float64 over the values that a 4-bit cache holds,
and how far an output may be from it.

TEST INFRASTRUCTURE ONLY: the oracle of the tests.  The product path
(joule_amd) never imports it.

The bound is a sum over the rows that a token sees, each row weighted as the
softmax weights it, so that rows without weight do not loosen it.  With p_t the
weights, v_t the values, o the output and A_t = |scale| sum_i |q_i k_ti|, an error
of e_t in the logarithm of each weight and of f_t relative in each product moves
dimension d by at most  sum_t p_t (e_t (|v_td| + |o_d|) + f_t |v_td|).  What the
library's header states of its arithmetic gives, with room for the float32
roundings of 128 products, of the exponential and of the sums:

  every form     e_t = 2^-18 A_t + 2^-19, q to 2^-30 of its largest; products below
                 the range of fp16: 2^-29 of the largest p_t |v_t| a row
  bf16           weights to fp16 once: f_t = 2^-11; the output: 2^-8 of it
  bf16 prompts   also K and V to fp16, 2^-11 of the value and 2^-15 of the largest
                 scale of the 16 rows (of 2^8 times the row's own, where that is
                 less); the products then 2^-20 of the largest
"""

from __future__ import annotations

import numpy as np

FORMS = ("f32", "bf16", "bf16 prompt")


def weights(q: np.ndarray, k: np.ndarray, seen: int, scale: float) -> np.ndarray:
    """The softmax weights [seen] of one query row over rows 0 .. seen - 1."""
    a = k[:seen] @ q * scale
    p = np.exp(a - a.max())
    return p / p.sum()


def attend(q: np.ndarray, k: np.ndarray, v: np.ndarray, seen: int, scale: float) -> np.ndarray:
    """One query row [hd] over rows 0 .. seen - 1 of k and v [T, hd] (float64); 0
    where it sees none."""
    if seen <= 0:
        return np.zeros(v.shape[1])
    return weights(q, k, seen, scale) @ v[:seen]


def _rows16(x: np.ndarray, seen: int) -> np.ndarray:
    """2^-15 of the largest scale of each row's 16 rows, or of 2^8 times its own
    (rows that are not finite, behind those seen, do not count)."""
    s = np.abs(x).max(axis=1) / 6.9
    s = np.where(np.isfinite(s), s, 0.0)
    n = -(-len(s) // 16) * 16
    block = np.concatenate([s, np.zeros(n - len(s))]).reshape(-1, 16).max(axis=1).repeat(16)[:len(s)]
    return 2.0 ** -15 * np.minimum(block, 2.0 ** 8 * s)[:seen]


def bound(q: np.ndarray, k: np.ndarray, v: np.ndarray, seen: int, scale: float, form: str) -> np.ndarray:
    """How far each dimension of attend()'s result may be off."""
    if seen <= 0:
        return np.zeros(v.shape[1])
    p = weights(q, k, seen, scale)
    av, aq = np.abs(v[:seen]), np.abs(q)
    out = np.abs(p @ v[:seen])
    A = np.abs(k[:seen]) @ aq * abs(scale)
    e = 2.0 ** -18 * A + 2.0 ** -19 + 2.0 ** -30 * aq.max() * np.abs(k[:seen]).sum(axis=1) * abs(scale)
    f = 2.0 ** -19
    least = 2.0 ** -29
    off = np.zeros(v.shape[1])
    if form != "f32":
        f += 2.0 ** -11
        off += 2.0 ** -8 * out
    if form == "bf16 prompt":
        e = e + 2.0 ** -11 * A + _rows16(k, seen) * aq.sum() * abs(scale)
        f += 2.0 ** -11
        least = 2.0 ** -20
        off += p @ _rows16(v, seen)
    big = (p * av.max(axis=1)).max()
    return off + p @ ((e[:, None] + f) * av) + (p @ e) * out + seen * least * big
