"""Sampling at settings and rows where the places of the borders are easily
missed.  Tokens have to be those of the definition (tests/test_gpu_sample.py)."""

import numpy as np
import pytest
import torch

from joule_amd.sampling import sample
from test_gpu_sample import _check, _logits

pytestmark = pytest.mark.gpu

INF = float("inf")


@pytest.mark.parametrize("T", [1e3, 1e6, 1e9, 1e10, 1e11, 1e12, 1e15, 1e20, 1e38, INF])
@pytest.mark.parametrize("spread", [1.4, 1e-6])
def test_min_p_at_high_temperatures(T, spread):
    """Next to a min_p of 1 the border lies where a weight is no longer the whole
    2^40, which a high temperature puts far from the largest logit, or past all of
    them.  Weights there are rounded from exponentials right to a few 2^-53: 1 part
    in 2^12 of the distance that decides one, so tokens are compared at random
    numbers that are not within that of a border."""
    B, V = 4, 5000
    x = _logits(31, B, V, spread)
    if spread < 1:
        x = (9.0 + (x - 9.0) * 1e-5).astype(np.float32)
    for min_p in (1.0, 1.0 - 2.0 ** -24, 0.999, 0.5, 0.0):
        for u in (0.0, 0.3, 0.71, 0.99):
            _check(x, [u] * B, temperature=T, min_p=min_p)
            _check(x, [u] * B, temperature=T, min_p=min_p, top_k=300, top_p=0.9)


def test_min_p_where_logits_differ_beyond_float32():
    x = np.full((3, 3000), 3e38, np.float32)
    x[:, 1::3] = -3e38
    x[1, 2::3] = 1.0
    x[2, ::3] = -np.inf
    for T in (1.0, 1e30, 1e38, INF):
        for min_p in (1.0, 0.5, 0.0):
            for u in (0.0, 0.5, 0.9):
                _check(x, [u] * 3, temperature=T, min_p=min_p)


@pytest.mark.parametrize("min_p", [0.001, 0.02, 0.2, 0.9])
def test_a_border_among_logits_that_differ_beyond_float32(min_p):
    """At temperatures of 10^37 and more, weights that count lie on both sides of
    such a difference."""
    rng = np.random.default_rng(8)
    x = (rng.random((3, 7000)) * 6.6e38 - 3.3e38).astype(np.float32)
    for T in (3e37, 1e38, 3e38):
        for u in (0.0, 0.4, 0.97):
            _check(x, [u] * 3, temperature=T, min_p=min_p)


def test_small_top_k_with_the_largest_logit_at_a_chunks_end():
    """The last token of a chunk belongs to one part of the row, from whose maxima
    the bound on the k-th logit comes; where it counted for several, the bound
    passed all but that token and the row was selected by its keys."""
    B, V = 128, 151936
    g = torch.Generator(device="cuda").manual_seed(5)
    x = torch.randn(B, V, generator=g, device="cuda") * 2
    chunk = V // 4
    for at in (chunk - 1, 2 * chunk - 1, V - 1, 0):
        y = x.clone()
        y[:, at] = 40.0
        u = torch.rand(B, generator=g, device="cuda")
        for k in (2, 16, 50):
            tok, p = sample(y, u, 30.0, k)
            w, order = y.double().topk(k, dim=1)
            w = torch.round(torch.exp((w - w[:, :1]) / 30.0) * 2.0 ** 40)
            run = w.cumsum(dim=1)
            i = (run <= torch.floor(u.double()[:, None] * run[:, -1:])).sum(dim=1, keepdim=True)
            assert torch.equal(order.gather(1, i).squeeze(1).int(), tok)
            assert torch.allclose((w.gather(1, i) / run[:, -1:]).squeeze(1).float(), p, rtol=2.0 ** -22, atol=0)
