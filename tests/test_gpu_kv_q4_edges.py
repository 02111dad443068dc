"""4-bit attention where its arithmetic could leave the definition."""

import numpy as np
import pytest
import torch

from test_gpu_kv_q4_bound import cache, check, ints, queries, rows, run, write

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


@pytest.mark.parametrize("maxT", [0, 3000])
@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("n,start", [(1, 0), (1, 700), (3, 0), (5, 700), (130, 0), (130, 333)])
def test_an_infinite_query_gives_nan(n, start, dt, maxT):
    """Also where every score that it makes is -infinity, whose softmax is
    undefined: never the 0 of a token that sees no row."""
    H, KH, T = 4, 2, start + n
    c = cache(1, maxT or T, KH, H)
    k, v = rows(5, T, KH)
    k[:, :, 77] = -2.0                  # an infinity there makes every score -infinity
    k[:, :, 78] = 2.0                   # ... +infinity
    write(c, 0, k, v)
    for at, value in ((77, np.inf), (78, np.inf), (78, -np.inf), (5, np.inf)):
        q = queries(6, k, start, n, H)
        q[:, 1, at] = value
        q[n // 2, 2, at] = value
        got = c.attention(0, torch.from_numpy(q).cuda().to({"f32": torch.float32, "bf16": torch.bfloat16}[dt]), ints([start]), ints([0, n]))
        assert bool(got[:, 1].isnan().all()) and bool(got[n // 2, 2].isnan().all())
        got[:, 1] = 0.0
        got[n // 2, 2] = 0.0
        assert bool(got.isfinite().all())


@pytest.mark.parametrize("maxT", [200, 3000])
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n", [1, 3, 130])
def test_a_token_without_rows_gets_0_whatever_its_query(n, dt, maxT):
    c = cache(2, maxT, 2, 8)
    k, v = rows(5, 180, 2)
    write(c, 0, k, v)
    q = torch.from_numpy(queries(6, k, 0, 2 * n, 8)).cuda().to(dt)
    q[0, 0], q[0, 1, 5], q[0, 2, 5], q[n, 3] = float("nan"), float("inf"), -float("inf"), float("nan")
    got = c.attention(0, q, ints([-1, -200]), ints([0, n, 2 * n]))
    assert not bool(got[0].any()) and not bool(got[n:].any())
    assert bool(got.isfinite().all())


def _without_weight(T, big, at):
    """Rows of 1e-3 that share the weight, and row `at` of `big` with none."""
    rng = np.random.default_rng(4)
    q = rng.standard_normal((1, 2, HD)).astype(np.float32)
    k, v = rows(9, T, 1)
    v *= 1e-3
    k[at, 0] = -30.0 * (q[0, 0] + q[0, 1])
    v[at, 0] = big
    return q, k, v


@pytest.mark.parametrize("big", [1.0, 1e3, 1e5, 4e5])
@pytest.mark.parametrize("at", [0, 37, 390])
@pytest.mark.parametrize("maxT", [400, 3000])
def test_a_large_v_without_weight_leaves_the_others_whole(maxT, at, big):
    """Single tokens, float32 and bf16, and prompts, float32: the weights of the
    others keep their bits, next to the large row and after it."""
    T = 400
    q, k, v = _without_weight(T, big, at)
    c = cache(1, maxT, 1, 2)
    write(c, 0, k, v)
    for dt in ("f32", "bf16"):
        check(c, q, [T - 1], [1], dt)
    # 100 tokens with the last one's query
    check(c, np.repeat(q, 100, axis=0), [T - 100], [100], "f32", only=[70, 99] if at > 300 else [0, 70, 99])


@pytest.mark.parametrize("group", [64, 32])
@pytest.mark.parametrize("maxT", [400, 3000, 40000])
@pytest.mark.parametrize("big", [3.0, 1e3, 1e5, 4e5])
def test_a_large_v_without_weight_in_bf16_prompts(big, maxT, group):
    T = 400
    for at in (0, 37, 390):
        q, k, v = _without_weight(T, big, at)
        c = cache(1, maxT, 1, 2, group)
        write(c, 0, k, v)
        check(c, np.repeat(q, 100, axis=0), [T - 100], [100], "bf16", only=[70, 99] if at > 300 else [0, 70, 99])


@pytest.mark.parametrize("H,KH,n,start", [(2, 1, 100, 0), (8, 1, 60, 333), (8, 2, 150, 10), (4, 4, 130, 64)])
@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("maxT", [0, 3000, 40000])
def test_rows_of_later_tokens_may_hold_anything(H, KH, n, start, dt, maxT):
    """A prompt's row with a K or V far above the others: tokens before it are
    as exact as without it."""
    for which, big in (("v", 3e5), ("k", 3e5), ("v", 300.0), ("k", 300.0)):
        k, v = rows(17, start + n + 1, KH)
        at = start + n // 2
        (v if which == "v" else k)[at] *= big / 3
        c = cache(1, maxT or start + n, KH, H)
        write(c, 0, k[:start + n], v[:start + n])
        q = queries(18, rows(17, start + n + 1, KH)[0], start, n, H)
        check(c, q, [start], [n], dt, only=sorted({0, n // 4, n // 2 - 2, n // 2 - 1}))


@pytest.mark.parametrize("group", [64, 32])
@pytest.mark.parametrize("maxT", [0, 3000, 40000])
def test_rows_of_every_magnitude_in_bf16_prompts(maxT, group):
    """K and V from 1e-7 to 1e5 within 16 rows, subnormal scales among them, and
    sequences without such rows beside."""
    H, KH, counts, start = 4, 2, [120, 0, 90, 100], [50, 3, 400, 0]
    c = cache(4, maxT or 490, KH, H, group)
    q = []
    for b, (s, n) in enumerate(zip(start, counts)):
        k, v = rows(b + 40, s + n + 1, KH)
        if b != 3:
            v *= 10.0 ** (np.arange(s + n + 1) % 13 - 7.0)[:, None, None]
        if b == 2:
            k *= 10.0 ** (np.arange(s + n + 1) % 5 - 3.0)[:, None, None]
        write(c, b, k[:s + n], v[:s + n])
        q.append(queries(b + 60, rows(b + 40, s + n + 1, KH)[0], s, n, H))
    check(c, np.concatenate(q), start, counts, "bf16")


def test_non_finite_rows_beside_large_ones_in_bf16_prompts():
    """A NaN in V reaches the group's outputs of those that see it, also where rows
    differ far; the others are as they were."""
    H, KH, n, s = 4, 1, 100, 60
    k, v = rows(71, s + n + 1, KH)
    v[s + 10] *= 1e5
    clean = cache(1, s + n, KH, H)
    write(clean, 0, k[:s + n], v[:s + n])
    q = queries(72, k, s, n, H)
    want = check(clean, q, [s], [n], "bf16", only=[0, 9, 50])
    bad = v.copy()
    bad[s + 40, 0, 3] = np.nan
    c = cache(1, s + n, KH, H)
    write(c, 0, k[:s + n], bad[:s + n])
    got = c.attention(0, torch.from_numpy(q).cuda().bfloat16(), ints([s]), ints([0, n]))
    assert torch.equal(got[:40], want[:40]) and bool(got[40:, :, 64:].isfinite().all())
    assert bool(got[40:, :, :64].isnan().all())


@pytest.mark.parametrize("counts,start", [([1, 1], [37, 90]), ([4, 2], [37, 90]), ([70, 66], [37, 90]), ([200], [37])])
@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("maxT", [237, 3000])
def test_infinite_and_other_scales_behind_a_tokens_own_row(counts, start, dt, maxT):
    """What rows that were never written hold, as fp16: infinities, the largest
    values, the smallest; over caches just filled and with room."""
    res = []
    for bits in (0x7C00, 0x7BFF, 0x0001, 0xFC00, 0x0000):
        c = cache(len(counts), maxT, 2, 8)
        c.data.view(torch.int16).fill_(bits - 0x10000 if bits & 0x8000 else bits)
        q = []
        for b, (s, n) in enumerate(zip(start, counts)):
            k, v = rows(b + 90, s + n + 1, 2)
            write(c, b, k[:s + n], v[:s + n])
            q.append(queries(b + 95, k, s, n, 8))
        res.append(check(c, np.concatenate(q), start, counts, dt))
    for r in res[1:]:
        assert torch.equal(r, res[0])


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("n", [1, 5, 130])
def test_rows_moved_into_a_wider_cache(n, dt):
    """Read from a cache of 300 rows and written into one of 5000: the same values,
    in planes laid out otherwise, and attention over them."""
    k, v = rows(3, 300, 2)
    a, b = cache(2, 300, 2, 8), cache(2, 5000, 2, 8)
    write(a, 0, k, v)
    write(a, 1, k[:200] * 3, v[:200])
    cu = ints([0, 300, 500])
    zero = ints([0, 0])
    ka, va = a.read(0, zero, cu, 500)
    b.write(0, ka, va, zero, cu)
    for x, y in zip(b.read(0, zero, cu, 500), (ka, va)):
        assert torch.equal(x, y)
    q = np.concatenate([queries(4, k, 299 - n, n, 8), queries(5, k, 199 - n, n, 8)])
    check(b, q, [300 - n, 200 - n], [n, n], dt)


@pytest.mark.parametrize("counts,start", [([1] * 5, [900, 3, 250, 64, 511]), ([5], [900]), ([200], [300])])
@pytest.mark.parametrize("apart", [False, True])
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
def test_the_same_call_gives_the_same_bits(counts, start, apart, dt):
    c = cache(len(counts), 1100, 2, 8)
    for b, (s, n) in enumerate(zip(start, counts)):
        k, v = rows(b + 7, s + n, 2)
        if apart:
            v[::50] *= 1e4
        write(c, b, k, v)
    q = torch.from_numpy(np.random.default_rng(2).standard_normal((sum(counts), 8, HD)).astype(np.float32)).cuda().to(dt)
    cu = ints(np.concatenate([[0], np.cumsum(counts)]).tolist())
    want = c.attention(0, q, ints(start), cu)
    for _ in range(5):
        assert torch.equal(c.attention(0, q, ints(start), cu), want)


@pytest.mark.parametrize("apart", [False, True])
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("maxT", [400, 5000])
def test_prompts_in_place_and_captured(maxT, dt, apart):
    """The output over q, and two graphs replayed in turn between eager calls."""
    H, KH, n, s = 8, 2, 150, 240
    c = cache(1, maxT, KH, H)
    k, v = rows(7, s + n, KH)
    if apart:
        v[::50] *= 1e4
    write(c, 0, k, v)
    start, cu = ints([s]), ints([0, n])
    new = lambda seed: torch.from_numpy(np.random.default_rng(seed).standard_normal((n, H, HD)).astype(np.float32)).cuda().to(dt)  # noqa: E731
    q = new(1)
    want = c.attention(0, q, start, cu)
    same = q.clone()
    assert torch.equal(c.attention(0, same, start, cu, out=same), want) and torch.equal(same, want)
    out = torch.empty_like(q)
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            c.attention(0, q, start, cu, out=out)
        graphs.append(g)
    for i in range(6):
        q.copy_(new(10 + i))
        out.zero_()
        graphs[i % 2].replay()
        torch.cuda.synchronize()
        got = out.clone()
        assert torch.equal(c.attention(0, q, start, cu), got)


@pytest.mark.parametrize("group", [64, 32])
def test_the_largest_magnitude_that_a_group_holds(group):
    """Scales round to 65504 below 65520, to infinity from there: 7 times that
    is the first magnitude that reads back as NaN."""
    x = torch.zeros(6, 1, HD, device="cuda")
    x[:, 0, 1] = torch.tensor([458528.0, 458600.0, 458639.96875, 458640.0, 458700.0, -458640.0], device="cuda")
    x[:, 0, 2] = -65504.0
    c = cache(1, 6, 1, 1, group)
    c.write(0, x, -x, ints([0]), ints([0, 6]))
    for got, sign in zip(c.read(0, ints([0]), ints([0, 6]), 6), (1.0, -1.0)):
        assert bool((got[:3, 0, 1] == sign * 458528.0).all()) and bool((got[:3, 0, 2] == -sign * 65504.0).all())
        assert bool(got[3:, 0, :group].isnan().all()) and bool((got[3:, 0, group:] == 0.0).all())


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("counts", [[2, 3], [90, 60]])
def test_tokens_before_the_first_sequence_are_skipped(counts, dt):
    """cu may begin behind 0, as the ends of a packed batch's padding do."""
    lead, N = 5, 5 + sum(counts)
    start, cu = [20, 3], [lead, lead + counts[0], N]
    k, v = rows(33, N, 2)
    c = cache(2, 200, 2, 8)
    for b in range(2):
        write(c, b, *rows(b + 60, start[b], 2))
    c.write(0, torch.from_numpy(k).cuda(), torch.from_numpy(v).cuda(), ints(start), ints(cu))
    out = torch.full((N, 2, HD), 7.0, device="cuda")
    c.read(0, ints(start), ints(cu), N, k=out, v=out.clone())
    assert bool((out[:lead] == 7.0).all()) and not bool((out[lead:] == 7.0).all(dim=2).any())
    q = np.random.default_rng(1).standard_normal((N, 8, HD)).astype(np.float32)
    d = {"f32": torch.float32, "bf16": torch.bfloat16}[dt]
    got = torch.full((N, 8, HD), 7.0, dtype=d, device="cuda")
    c.attention(0, torch.from_numpy(q).cuda().to(d), ints(start), ints(cu), out=got)
    assert bool((got[:lead] == 7.0).all())
    want = check(c, q[lead:], start, counts, dt)
    assert torch.equal(got[lead:], want)
