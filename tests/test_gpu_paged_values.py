"""Paged attention at the ends of the number range: rows of K that are not finite, seen by
their tokens; scores that only a scale near 0 keeps small."""

import numpy as np
import pytest
import torch

from oracle.paged import attend
from test_gpu_paged import CALLS, DEEP, DT, HD, TYPES, check, form_of, held, ints, prepared, put

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dt,cached", TYPES)
@pytest.mark.parametrize("H,KH,counts,start", CALLS)
@pytest.mark.parametrize("maxT", [1500, DEEP])
@pytest.mark.parametrize("scale", [HD ** -0.5, -0.2])
def test_tokens_that_see_an_infinite_or_nan_k(H, KH, counts, start, maxT, scale, dt, cached):
    """A NaN: NaN.  An infinity: NaN where the score is +infinity; where it is -infinity, what
    the other rows give (float32 q over bf16 pages, in parts: that, or NaN)."""
    cu = np.concatenate([[0], np.cumsum(counts)]).tolist()
    for value in (float("inf"), -float("inf"), float("nan")):
        c, q = prepared(H, KH, counts, start, cached, maxT)
        for b, (s, n) in enumerate(zip(start, counts)):
            if n:
                k, v = (x[s // 2:s // 2 + 1].copy() for x in held(c, b, s + n))
                k[:, :, 3] = value
                put(c, b, k, v, first=s // 2)
        qd = torch.from_numpy(q).cuda().to(DT[dt])
        got = c.attention(0, qd, ints(start), ints(cu), scale=scale)
        torch.cuda.synchronize()
        g64, q64 = got.double().cpu().numpy(), qd.double().cpu().numpy()
        form, seen = form_of(c, dt, len(q), H, KH, len(counts)), [0, 0]
        for b, (s, n) in enumerate(zip(start, counts)):
            if not n:
                continue
            k, v = held(c, b, s + n)
            pick = np.array(sorted({*range(s // 2 - s, min(n, 6)), n - 1}))
            pick = pick[(pick >= 0) & (s + pick >= s // 2)]             # tokens that see the row
            see = np.arange(s + n) <= s + pick[:, None]
            for h in range(H):
                x, y = g64[cu[b] + pick, h], q64[cu[b] + pick, h]
                low = y[:, 3] * value * scale < 0                       # (a NaN is not)
                others = see.copy()
                others[:, s // 2] = False
                kk = k[:, h * KH // H].copy()
                kk[s // 2] = 0.0
                want, tol = attend(y, kk, v[:, h * KH // H], others, scale, form)
                nan = np.isnan(x).all(axis=1)
                near = (np.abs(x - want) <= tol).all(axis=1) & (others.any(axis=1))
                assert nan[~low].all()
                # (a token whose only row this is has no other, NaN)
                alone = ~others.any(axis=1)
                assert (near | nan if dt == "f32" and cached == "bf16" else np.where(alone, nan, near))[low].all()
                seen[0] += int(low.sum())
                seen[1] += int((~low).sum())
        assert seen[1] and (seen[0] or np.isnan(value))


@pytest.mark.parametrize("dt,cached", TYPES)
@pytest.mark.parametrize("H,KH,counts,start", [(4, 2, [1], [40]), (8, 1, [2], [500]), (2, 2, [100, 130], [0, 333]), (16, 2, [300], [600])])
@pytest.mark.parametrize("maxT", [1500, DEEP])
@pytest.mark.parametrize("scale", [0.0, -0.0, 1e-36, -1e-33, 2e-38, -1e-41])
def test_large_scores_under_a_scale_near_0(H, KH, counts, start, maxT, scale, dt, cached):
    """Products of 2^105 and more: a scale of 0 gives the mean all the same, one of 1e-33
    what the formula gives."""
    c, q = prepared(H, KH, counts, start, cached, maxT)
    c.data[:, :, 0] *= 2.0 ** 105
    check(c, q, start, counts, dt, scale=scale)


@pytest.mark.parametrize("dt,cached", TYPES)
@pytest.mark.parametrize("H,KH,counts,start", CALLS)
@pytest.mark.parametrize("maxT", [1500, DEEP])
def test_the_largest_values_allowed(H, KH, counts, start, maxT, dt, cached):
    """V up to 2^100, under weights that pass the reference."""
    c, q = prepared(H, KH, counts, start, cached, maxT)
    v = c.data[:, :, 1]
    v *= 2.0 ** 99 / float(v[v.isfinite()].abs().max())
    for x in (1.0, 8.0):
        check(c, q * x, start, counts, dt)


@pytest.mark.parametrize("dt,cached", TYPES)
def test_rows_at_the_ends_of_their_type(dt, cached):
    """A token a sequence, at rows that int32 just holds: past the cache, and below 0."""
    c, q = prepared(8, 2, [1, 1, 1, 1], [0, 0, 40, 0], cached, 900)
    start = [2 ** 31 - 1, -2 ** 31, 40, 2 ** 31 - 1]
    out = torch.full((4, 8, HD), 7.0, dtype=DT[dt], device="cuda")
    qd, k = torch.from_numpy(q).cuda().to(DT[dt]), torch.ones(4, 2, HD, dtype=DT[dt], device="cuda")
    got = c.attention(0, qd, ints(start), out=out)
    want = c.attention(0, qd, ints([0, 0, 40, 0]))
    assert bool((got[[0, 3]] == 7.0).all()) and not bool(got[1].any()) and torch.equal(got[2], want[2])
    before = c.data.clone()
    c.append(0, k, k, ints(start), q=torch.ones_like(out), q_out=out.fill_(7.0))
    assert bool((out[[0, 1, 3]] == 7.0).all()) and bool((out[2] == 1.0).all())
    bits = torch.int32 if cached == "f32" else torch.int16              # (the pages hold NaN elsewhere)
    assert 0 < int((c.data.view(bits) != before.view(bits)).sum()) <= 2 * 2 * HD
