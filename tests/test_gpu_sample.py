"""Sampling (jm_sample) against its definition in numpy's float64.

Tokens have to be equal.  The definition's weights are whole numbers of 2^-40
of the largest; another exponential, right to a few 2^-53, changes a weight by
one in about 2^-10 of the tokens, so a running sum of n weights by less than n,
and a token only if its random number lies within n 2^-40 of the kept weight of
a border: below 10^-6 a row here, for inputs that are fixed.  Probabilities are
rounded to float32 once: 2^-23."""

import numpy as np
import pytest
import torch

from joule_amd import _lib
from joule_amd.sampling import sample

pytestmark = pytest.mark.gpu

ONE = 2.0 ** 40


def _want(logits, u, temperature, top_k, top_p, min_p):
    B, V = logits.shape
    tok, prob = np.zeros(B, np.int32), np.zeros(B)
    per = [np.broadcast_to(np.asarray(x, t), (B,)) for x, t in ((temperature, np.float32), (top_k, np.int64),
                                                                (top_p, np.float32), (min_p, np.float32))]
    for b in range(B):
        T, k, p, mp = (float(x[b]) for x in per)
        l = logits[b].astype(np.float64)
        l = np.where(np.isnan(l), -np.inf, l)
        if l.max() == -np.inf:
            tok[b] = -1
            continue
        k = 1 if T <= 0 else V if k <= 0 else min(int(k), V)
        T = 1.0 if T <= 0 else T
        order = np.argsort(-l, kind="stable")
        s = l[order]
        with np.errstate(invalid="ignore", over="ignore"):
            w = np.where(s == s[0], ONE, np.rint(np.exp((s - s[0]) / T) * ONE))
        w = np.nan_to_num(w, nan=0.0)[:k]
        if p < 1:
            n = np.count_nonzero(np.cumsum(w) - w < p * w.sum())
            w = w[:max(1, n)]
        if mp > 0:
            w = w[:max(1, np.count_nonzero(w >= mp * ONE))]
        x = u[b] if u[b] > 0 else 0.0
        at = np.floor(float(x) * w.sum()) if x < 1 else w.sum() - 1
        i = int(np.searchsorted(np.cumsum(w), min(at, w.sum() - 1), side="right"))
        tok[b], prob[b] = order[i], w[i] / w.sum()
    return tok, prob


def _logits(seed, B, V, spread=1.4):
    rng = np.random.default_rng(seed)
    rank = np.argsort(rng.random((B, V)), axis=1)
    return (-spread * np.log(rank + 2.7) + 0.7 * rng.standard_normal((B, V)) + 9.0).astype(np.float32)


def _check(logits, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, dtype=torch.float32):
    t = torch.from_numpy(logits).cuda().to(dtype)
    dev = lambda x, d: torch.from_numpy(np.asarray(x, d)).cuda() if isinstance(x, (list, np.ndarray)) else x  # noqa: E731
    print(f"[sample] {list(t.shape)} {dtype}", flush=True)
    tok, p = sample(t, torch.from_numpy(np.asarray(u, np.float32)).cuda(), dev(temperature, np.float32), dev(top_k, np.int32),
                    dev(top_p, np.float32), dev(min_p, np.float32))
    want, prob = _want(t.float().cpu().numpy(), np.asarray(u, np.float32), temperature, top_k, top_p, min_p)
    got = tok.cpu().numpy()
    assert np.array_equal(got, want), (got, want)
    assert np.allclose(p.cpu().numpy(), prob, rtol=2.0 ** -23, atol=1e-38)


SETTINGS = [dict(), dict(temperature=0.7), dict(top_k=1), dict(top_k=50), dict(top_k=1000), dict(top_p=0.9), dict(top_p=0.01),
            dict(min_p=0.1), dict(temperature=0.8, top_k=50, top_p=0.95), dict(temperature=1.3, top_p=0.8, min_p=0.02),
            dict(temperature=1.5, top_k=300, top_p=0.99, min_p=0.001), dict(temperature=0.0), dict(temperature=-1.0, top_p=0.5),
            dict(temperature=0.01), dict(temperature=50.0), dict(temperature=50.0, top_k=5000, top_p=0.999)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("B,V", [(1, 1), (2, 2), (3, 63), (2, 1025), (5, 4099), (9, 50304), (3, 151936)])
def test_matches_the_definition(B, V, dtype):
    logits = _logits(B + V, B, V)
    rng = np.random.default_rng(3)
    for how in SETTINGS:
        _check(logits, rng.random(B), **how, dtype=dtype)


def test_settings_of_each_row():
    B, V = 64, 20011
    rng = np.random.default_rng(1)
    pick = lambda v: rng.choice(v, B)  # noqa: E731
    _check(_logits(7, B, V), rng.random(B), pick([0.0, 0.5, 1.0, 2.0]), pick([0, -3, 1, 7, 40, 3000, V, V + 5, 2 ** 31 - 1]),
           pick([1.0, 2.0, 0.9, 0.3, 0.0, -1.0]), pick([0.0, -1.0, 0.05, 0.5, 1.0, 3.0]))


def test_small_top_k_of_many_rows():
    """Rows in chunks of many tokens a thread, of which few are counted: sorted
    either way, tied, with all that is kept in one place, and mostly -infinity."""
    B, V = 258, 40001
    x = _logits(21, B, V)
    rng = np.random.default_rng(22)
    for b in range(B):
        if b % 6 == 1:
            x[b] = np.sort(x[b])
        elif b % 6 == 2:
            x[b] = -np.sort(-x[b])
        elif b % 6 == 3:
            x[b] = np.rint(x[b] * 0.5)
        elif b % 6 == 4:
            x[b, 64 * 1024 // 4:64 * 1024 // 4 + 80] += 30.0
        elif b % 6 == 5:
            x[b, rng.random(V) < 0.999] = -np.inf
    k = rng.choice(np.asarray([1, 2, 20, 63, 64, 65, 400], np.int32), B)
    _check(x, rng.random(B).astype(np.float32), temperature=0.9, top_k=k, top_p=rng.choice(np.asarray([1.0, 0.9], np.float32), B))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_more_rows_than_one_launch_takes(dtype):
    B, V = 2100, 77
    rng = np.random.default_rng(23)
    x = torch.from_numpy(_logits(24, B, V)).to(dtype).float().numpy()
    pick = lambda v, t: rng.choice(np.asarray(v, t), B)  # noqa: E731
    _check(x, rng.random(B).astype(np.float32), pick([0.0, 0.7, 1.3], np.float32), pick([0, 1, 9], np.int32),
           pick([1.0, 0.8], np.float32), pick([0.0, 0.1], np.float32), dtype)


@pytest.mark.parametrize("how", [dict(), dict(top_k=5), dict(top_p=0.6), dict(min_p=0.5), dict(top_k=700, top_p=0.9)])
@pytest.mark.parametrize("V", [5, 1000, 40001])
def test_ties_go_to_the_lower_index(V, how):
    rng = np.random.default_rng(V)
    logits = np.stack([np.zeros(V), rng.integers(0, 3, V), -rng.integers(0, 2, V) * 0.0, rng.integers(-1, 1, V) * 30.0]).astype(np.float32)
    logits[2, ::2] = -0.0
    for u in ([0.0] * 4, [0.5] * 4, [0.99999994] * 4, rng.random(4)):
        _check(logits, u, **how)


def test_random_numbers_at_and_past_the_ends():
    logits = np.repeat(_logits(2, 1, 3001), 8, axis=0)
    u = [0.0, 0.99999994, 1.0, 5.0, -1.0, float("nan"), float("inf"), 1e-30]
    for how in (dict(), dict(top_k=20), dict(top_p=0.5), dict(temperature=0.0)):
        _check(logits, u, **how)


def test_masks_infinities_and_nan():
    V = 2049
    low = np.finfo(np.float32).min
    x = _logits(4, 10, V)
    x[0] = -np.inf                          # nothing left
    x[1] = np.nan
    x[2, :] = -np.inf
    x[2, 77] = -3.0                         # one left
    x[3, :] = low                           # the type's lowest value as a mask
    x[3, [5, 900]] = 4.0
    x[4, :] = low                           # ... over everything
    x[5, 1::2] = -np.inf
    x[6, ::3] = np.nan
    x[7, [9, 2000]] = np.inf
    x[8] = np.inf
    x[9, :] = low
    x[9, 3] = -low
    for u in np.linspace(0, 0.999, 7):
        for how in (dict(), dict(top_k=3), dict(top_p=0.7, temperature=0.6), dict(min_p=0.2), dict(temperature=0.0)):
            _check(x, [u] * 10, **how)


def test_one_logit_far_above_and_many_far_below():
    """Weights of a few units of 2^-40, and none at all."""
    V = 30000
    x = np.full((6, V), -26.0, np.float32) + np.random.default_rng(1).random((6, V)).astype(np.float32)
    x[:, 123] = [0.0, 1.0, 2.0, 3.0, 10.0, 100.0]
    for u in (0.5, 0.99999994):
        for how in (dict(), dict(top_k=100), dict(top_p=0.9999999), dict(temperature=3.0, top_p=0.99), dict(min_p=1.2e-12),
                    dict(min_p=3e-12), dict(min_p=1e-30), dict(min_p=4e-11, temperature=1.1)):
            _check(x, [u] * 6, **how)


def test_strided_rows_unaligned_start_and_given_outputs():
    big = torch.from_numpy(_logits(5, 7, 1500)).cuda()
    x = big[:, 3:1204]
    u = torch.rand(7, device="cuda", generator=torch.Generator("cuda").manual_seed(1))
    tok, p = torch.full((7,), -5, dtype=torch.int32, device="cuda"), torch.empty(7, device="cuda")
    a = sample(x, u, 0.9, 40, 0.9, out_tok=tok, out_p=p)
    assert a[0].data_ptr() == tok.data_ptr() and a[1].data_ptr() == p.data_ptr()
    want, prob = _want(x.cpu().numpy(), u.cpu().numpy(), 0.9, 40, 0.9, 0.0)
    assert np.array_equal(tok.cpu().numpy(), want) and np.allclose(p.cpu().numpy(), prob, rtol=2.0 ** -23)
    h = x.bfloat16()
    odd = torch.empty(7, 1203, dtype=torch.bfloat16, device="cuda")[:, 1:1202]
    odd.copy_(h)
    assert torch.equal(sample(odd, u, 0.9, 40, 0.9)[0], sample(h, u, 0.9, 40, 0.9)[0])


def test_frequencies_follow_the_distribution():
    """Evenly spaced random numbers give each token its share to within one draw."""
    n = 2000
    l = np.array([2.0, 1.0, -1.0, 1.5, 0.0], np.float32)
    u = (np.arange(n) + 0.5) / n
    tok, _ = sample(torch.from_numpy(np.repeat(l[None], n, 0)).cuda(), torch.from_numpy(u.astype(np.float32)).cuda())
    share = np.bincount(tok.cpu().numpy(), minlength=5)
    p = np.exp(l.astype(np.float64)) / np.exp(l.astype(np.float64)).sum()
    assert np.abs(share - p * n).max() <= 1.0


def test_captured_replayed_and_on_other_streams():
    B, V = 6, 40000
    x, u = torch.from_numpy(_logits(9, B, V)).cuda(), torch.rand(B, device="cuda")
    tok, p = torch.empty(B, dtype=torch.int32, device="cuda"), torch.empty(B, device="cuda")
    run = lambda: sample(x, u, 0.8, 0, 0.95, out_tok=tok, out_p=p)  # noqa: E731
    run()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            run()
        graphs.append(g)
    for i in range(6):
        x.copy_(torch.from_numpy(_logits(20 + i, B, V)).cuda())
        u.copy_(torch.rand(B, device="cuda"))
        graphs[i % 2].replay()
        torch.cuda.synchronize()
        got = tok.clone(), p.clone()
        want, _ = _want(x.cpu().numpy(), u.cpu().numpy(), 0.8, 0, 0.95, 0.0)
        assert np.array_equal(got[0].cpu().numpy(), want)
        run()
        assert torch.equal(tok, got[0]) and torch.equal(p, got[1])
        other = sample(x, u, 0.8, 0, 0.95, stream=side)
        side.synchronize()
        assert torch.equal(other[0], tok)


def test_python_refusals():
    x, u = torch.zeros(2, 10, device="cuda"), torch.zeros(2, device="cuda")
    for i, f in enumerate([lambda: sample(x[0], u), lambda: sample(x.half(), u), lambda: sample(x.cpu(), u),
                           lambda: sample(x, u[:1]), lambda: sample(x, u.double()), lambda: sample(x, u.cpu()),
                           lambda: sample(x.t().contiguous().t(), u), lambda: sample(x[:1].expand(2, 10), u),
                           lambda: sample(x, u, temperature=u.double()), lambda: sample(x, u, top_k=u),
                           lambda: sample(x, u, top_p=u[:1]), lambda: sample(x, u, out_tok=u), lambda: sample(x, u, out_p=u[:1]),
                           lambda: sample(x, u, temperature=float("nan")), lambda: sample(x, u, top_k=2 ** 40)]):
        with pytest.raises((ValueError, OverflowError, _lib.JouleError)):
            f()
            pytest.fail(f"call {i} was taken")
    tok, p = sample(x[:0], u[:0])
    assert tok.shape == (0,) and p.shape == (0,)
