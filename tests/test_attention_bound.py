"""What the bound of the 4-bit attention's tests lets pass: for each of their
shapes, and rows drawn as they draw them, ranges left out, an output of 0, a mask
off by one row and a score scale off by a hundredth have to be past it.  CPU only."""

import numpy as np
import pytest

from oracle.attention import FORMS, attend, bound

HD = 128
SCALE = HD ** -0.5


def rows(rng, T):
    """k and v of T rows as the GPU tests draw them."""
    k, v = rng.standard_normal((T, HD)), rng.standard_normal((T, HD))
    k[:, 3::17] *= 2.0
    return k, v


def query(rng, k, own):
    """A query that looks at its own row and at the one behind."""
    return rng.standard_normal(HD) + 0.4 * k[own:own + 2].sum(axis=0)


def past(wrong, want, tol):
    return bool((np.abs(wrong - want) > tol).any())


# (tokens, first row) of the GPU tests' sequences; prompts from 64 rows of queries
SHAPES = [(1, 300), (1, 5000), (5, 900), (64, 1500), (129, 2000), (300, 97), (70, 700), (90, 1800)]


@pytest.mark.parametrize("n,start,form", [(n, s, f) for n, s in SHAPES for f in FORMS if f == "f32" or (f == "bf16") == (n < 64)])
def test_what_the_bound_rejects(n, start, form):
    rng = np.random.default_rng(n + start)
    T = start + n
    k, v = rows(rng, T)
    for i in {0, n // 2, n - 1}:
        seen = start + i + 1
        q = query(rng, k, start + i)
        want, tol = attend(q, k, v, seen, SCALE), bound(q, k, v, seen, SCALE, form)
        assert past(np.zeros(HD), want, tol)
        # ranges of rows left out: the first and last quarters, one half, one tile of 32 in 8
        for lo, hi in ((0, seen // 4), (seen - seen // 4, seen), (seen // 4, 3 * seen // 4)):
            keep = np.r_[0:lo, hi:seen]
            assert past(attend(q, k[keep], v[keep], len(keep), SCALE), want, tol)
        keep = [t for t in range(seen) if t // 32 % 8 != 3 or seen < 128]
        if len(keep) < seen:
            assert past(attend(q, k[keep], v[keep], len(keep), SCALE), want, tol)
        # the own row unseen, and one row too many
        assert past(attend(q, k, v, seen - 1, SCALE), want, tol)
        if seen < T:
            assert past(attend(q, k, v, seen + 1, SCALE), want, tol)
        assert past(attend(q, k, v, seen, SCALE * 1.1), want, tol)


def test_rows_without_weight_do_not_loosen_it():
    rng = np.random.default_rng(1)
    k, v = rows(rng, 400)
    q = rng.standard_normal(HD)
    for form in FORMS[:2]:
        alone = bound(q, k[1:], v[1:], 399, SCALE, form)
        k2, v2 = k.copy(), v.copy()
        k2[0], v2[0] = -40.0 * q, 1e5
        assert (bound(q, k2, v2, 400, SCALE, form) <= 1.01 * alone).all()
