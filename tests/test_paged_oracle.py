"""The bounds that the paged caches are tested with: roundings of the kind that they allow
stay inside, mistakes do not.  CPU only."""

import numpy as np
import pytest
import torch

from joule_amd.decoder import rope_tables
from oracle.paged import attend, finish

HD = 128


def case(n, T, seed=0):
    rng = np.random.default_rng(seed)
    k, v = (rng.standard_normal((T, HD)).astype(np.float32) for _ in range(2))
    k[:, 3::17] *= 2.0
    k, v = (torch.from_numpy(x).bfloat16().float().numpy() for x in (k, v))
    q = rng.standard_normal((n, HD)).astype(np.float32)
    q += 0.4 * k[T - n:]
    see = np.arange(T) <= T - n + np.arange(n)[:, None]
    return torch.from_numpy(q).bfloat16().float().numpy(), k, v, see


def rounded(x, bits):
    """x to `bits` bits of significand."""
    m, e = np.frexp(x)
    return np.ldexp(np.round(m * 2.0 ** bits) / 2.0 ** bits, e)


@pytest.mark.parametrize("form,bits,out", [("f32", 24, 24), ("bf16", 17, 8), ("bf16 prompt", 8, 8)])
@pytest.mark.parametrize("n,T", [(1, 1), (1, 900), (40, 300)])
def test_roundings_stay_inside(form, bits, out, n, T):
    q, k, v, see = case(n, T)
    want, tol = attend(q, k, v, see, HD ** -0.5, form)
    s = (q @ k.T).astype(np.float32) * np.float32(HD ** -0.5)
    s[~see] = -np.inf
    # (the reference need not be the largest score: up to 2^10 below it)
    p = rounded(np.exp2((s - s.max(axis=1, keepdims=True)) * 1.4426950408889634 + 9.3), bits)
    o = rounded(p @ v / p.sum(axis=1, keepdims=True), out)
    assert (np.abs(o - want) <= tol).all()


@pytest.mark.parametrize("form", ["f32", "bf16", "bf16 prompt"])
def test_mistakes_do_not(form):
    q, k, v, see = case(40, 300)
    want, tol = attend(q, k, v, see, HD ** -0.5, form)
    early, late, hole = see.copy(), see.copy(), see.copy()
    early[:, :1] = False                                # a row too few
    late[:, 1:] |= see[:, :-1]                          # the row behind the token's own
    hole[:, 160:176] = False
    other = k.copy()
    other[100:116] = k[116:132]                         # 16 rows of another place
    for wrong in (attend(q, k, v, late, HD ** -0.5, form), attend(q, k, v, hole, HD ** -0.5, form),
                  attend(q, k, v, see, 0.97 * HD ** -0.5, form), attend(q, other, v, see, HD ** -0.5, form),
                  attend(np.roll(q, 1, axis=0), k, v, see, HD ** -0.5, form), attend(q, k, np.roll(v, 1, axis=1), see, HD ** -0.5, form)):
        assert (np.abs(wrong[0] - want) > tol).any(axis=1).sum() > 20
    wrong = attend(q, k, v, early, HD ** -0.5, form)
    assert (np.abs(wrong[0] - want) > tol).any()


def test_what_sees_nothing_and_what_is_not_seen():
    q, k, v, see = case(4, 50)
    see[2] = False
    k[-1], v[-1], see[:, -1] = np.nan, np.inf, False
    o, tol = attend(q, k, v, see, 0.1, "f32")
    assert np.isfinite(o).all() and np.isfinite(tol).all() and not o[2].any() and not tol[2].any()


def test_rotation_keeps_lengths_and_norms_are_one():
    cos, sin = rope_tables(40, HD, 1e4)
    x = np.random.default_rng(1).standard_normal((40, 3, HD)).astype(np.float32)
    r = np.arange(40)
    y = finish(x, r, None, cos, sin, 0.0)
    assert np.allclose((y * y).sum(-1), (x.astype(np.float64) ** 2).sum(-1), rtol=1e-6)
    assert np.allclose(y[0], x[0], rtol=1e-6)
    y = finish(x, r, np.ones(HD, np.float32), cos, sin, 0.0)
    assert np.allclose((y * y).mean(-1), 1.0, rtol=1e-6)
    # the angle between two rows depends on their distance alone
    z = finish(np.broadcast_to(x[:1], x.shape), r, None, cos, sin, 0.0)
    assert np.allclose((z[5] * z[9]).sum(-1), (z[30] * z[34]).sum(-1), rtol=1e-5)
