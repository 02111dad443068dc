"""4-bit attention where its arithmetic could leave the definition."""

import numpy as np
import pytest

from test_gpu_kv_q4_bound import cache, check, rows, run, write

pytestmark = pytest.mark.gpu

HD = 128
COUNTS = [([1, 1], [40, 700]), ([3, 2], [40, 700]), ([100, 130], [0, 333])]


@pytest.mark.parametrize("scale", [0.0, -0.0, 1e-38, 1e-30, 1e-9, -0.3, -HD ** -0.5, 1.0])
@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("counts,start", COUNTS)
def test_scales_of_any_sign_and_zero(counts, start, dt, scale):
    """A scale of 0 gives the mean of the rows that a token sees, a negative one
    turns the order round."""
    run(4, 1, counts, start, 64, dt, scale=scale)


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("counts,start", COUNTS)
def test_queries_of_zero_and_of_the_smallest_values(counts, start, dt):
    for value in (0.0, 1e-38, 1e-40):
        c = cache(2, 900, 1, 4)
        for b, (s, n) in enumerate(zip(start, counts)):
            k, v = rows(b + 1, s + n, 1)
            write(c, b, k, v)
        q = np.random.default_rng(3).standard_normal((sum(counts), 4, HD)).astype(np.float32) * np.float32(value)
        for scale in (HD ** -0.5, 1e-8, 0.0):
            check(c, q, start, counts, dt, scale)
