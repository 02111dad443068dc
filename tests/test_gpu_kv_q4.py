"""The 4-bit KV cache (jm_kv_q4_write, jm_kv_q4_read, jm_kv_q4_attn) on the GPU.

Rows are compared bit for bit with the format's own numpy form
(q4_store.quantize / dequantize); attention with softmax(scale q K^T) V in
float64 over the values the cache holds, row by row within a bound computed
from the inputs:
  * float32: q and the weights reach the matrix cores as two fp16 halves (22
    bits), products are summed in float32.  With A = max_t sum_i |q_i k_ti| scale
    a score is off by at most 2^-20 A + its own float32 roundings, a few 2^-24 A,
    a weight by that much relative, the output by twice that times the largest
    |v|: (2^-18 A + 2^-17) max|v| holds with room;
  * bfloat16: K, V and weights may be rounded to fp16 (2^-11 each), so
    (2^-9 A + 2^-8) max|v|, and the output's own rounding, 2^-8 of it.
"""

import numpy as np
import pytest
import torch

from joule_amd import _lib
from joule_amd.decoder import DecoderShape
from joule_amd.dense import dense_ffn_shape
from joule_amd.kv_q4 import Q4KVCacheSet
from joule_amd.q4_store import dequantize, quantize

pytestmark = pytest.mark.gpu

HD = 128
DT = {"f32": torch.float32, "bf16": torch.bfloat16}


def _cache(B, maxT, KH, H=None, group=64, layers=1):
    shape = DecoderShape(n_layers=layers, moe=dense_ffn_shape(1024, 512), n_heads=H or KH, n_kv=KH, maxT=maxT)
    c = Q4KVCacheSet(shape, B, group=group)
    c.data.fill_(0xFF)                  # rows never written hold NaN scales
    return c


def _randn(seed, *shape, scale=1.0):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return torch.randn(shape, generator=g, device="cuda") * scale


def _int(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _held(x, group):
    """float32 values of the format for rows x [n, KH, HD]."""
    a = x.float().cpu().numpy()
    return dequantize(*quantize(a, group), a.size, group).reshape(a.shape)


def _rows(seed, n, KH, dt):
    x = _randn(seed, n, KH, HD)
    x[:, :, 3::17] *= 6.0
    return x.to(dt)


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("group", [64, 32])
@pytest.mark.parametrize("KH,counts,start", [(1, [1], [0]), (4, [1, 1, 1], [5, 0, 62]), (3, [7, 0, 65, 1], [0, 9, 3, 99]),
                                             (8, [130], [1])])
def test_rows_are_the_formats(dt, group, KH, counts, start):
    print(f"[kv q4] rows {dt} g{group} KH={KH} {counts}", flush=True)
    B, n = len(counts), sum(counts)
    c = _cache(B, 150, KH, group=group, layers=2)
    k, v = _rows(1, n, KH, DT[dt]), _rows(2, n, KH, DT[dt])
    cu = _int(np.concatenate([[0], np.cumsum(counts)]).tolist())
    c.write(1, k, v, _int(start), None if counts == [1] * B else cu)
    for out in (torch.float32, torch.bfloat16):
        gk, gv = c.read(1, _int(start), cu, n, dtype=out)
        for g, x in ((gk, k), (gv, v)):
            want = torch.from_numpy(_held(x, group)).to(out)
            assert torch.equal(g.cpu(), want)
    # nothing else moved: the other layer is as it was, and so is the rest of this one
    assert bool((c.data[:, 0] == 0xFF).all())
    touched = int((c.data[:, 1] != 0xFF).sum())
    assert touched <= 2 * n * KH * (64 + 256 // group)
    for b, (s, m) in enumerate(zip(start, counts)):
        for r in (s - 1, s + m):
            if 0 <= r < 150:
                other = [0] * B
                other[b] = r
                one = [0] * (b + 1) + [1] * (B - b)
                k1, v1 = c.read(1, _int(other), _int(one), 1)
                assert bool(k1.isnan().all()) and bool(v1.isnan().all())


@pytest.mark.parametrize("group", [64, 32])
def test_values_where_rounding_matters(group):
    """Quotients at and next to halves, tiny and huge groups, zeros, every
    magnitude of fp16's scales, NaN and infinities."""
    rng = np.random.default_rng(5)
    n, KH = 64, 4
    x = rng.standard_normal((n, KH, HD)).astype(np.float32)
    g = x.reshape(-1, group)
    half = (rng.integers(-15, 16, g.shape) / 2).astype(np.float32)          # k + 0.5 and k steps
    s = np.exp2(rng.integers(-22, 12, (g.shape[0], 1))).astype(np.float32) * rng.integers(1024, 2048, (g.shape[0], 1)) / 1024
    g[::3] = (half * s)[::3]
    g[::3, 0] = (7 * s)[::3, 0]                                             # the scale is s itself
    g[1::6] = np.nextafter(half * s, np.inf, dtype=np.float32)[1::6]
    g[4] = 0.0
    g[7] = 1e-9
    g[10] = -3e-7
    g[13] = 1e-38
    g[16, 5] = np.nan
    g[19, 6] = np.inf
    g[22] = 458000.0
    g[25] = 1e30
    c = _cache(1, n, KH, group=group)
    t = torch.from_numpy(x).cuda()
    c.write(0, t, -t, _int([0]), _int([0, n]))
    k, v = c.read(0, _int([0]), _int([0, n]), n)
    with np.errstate(invalid="ignore", over="ignore"):
        for got, src in ((k, t), (v, -t)):
            got, want = got.cpu().numpy(), _held(src, group)
            fine = np.isfinite(want)
            assert np.array_equal(got[fine], want[fine])
            assert not np.isfinite(got[~fine]).any()
    bad = ~np.isfinite(k.cpu().numpy().reshape(-1, group))
    assert bad[[16, 19, 25]].all() and bad.sum() == 3 * group


@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_strided_rows_skips_and_padding(dt):
    """k and v as slices of one fused tensor, heads before tokens, rows outside
    the cache, tokens behind the last sequence."""
    B, KH, maxT, n = 3, 2, 40, 12
    fused = _rows(3, n + 4, 3 * KH, DT[dt])
    k, v = fused[:, KH:2 * KH], fused[:, 2 * KH:]
    c = _cache(B, maxT, KH)
    start, cu = _int([-2, 38, 3]), _int([0, 5, 9, n])        # two rows below 0, two past the end
    c.write(0, k, v, start, cu)
    gk, gv = (torch.full((n + 4, KH, HD), 7.0, dtype=DT[dt], device="cuda") for _ in range(2))
    c.read(0, start, cu, n + 4, dtype=DT[dt], k=gk, v=gv)
    lives = [i for i in range(n) if not (i < 2 or 7 <= i < 9)]
    dead = [i for i in range(n + 4) if i not in lives]
    for g, x in ((gk, k), (gv, v)):
        want = torch.from_numpy(_held(x, 64)).to(DT[dt])
        assert torch.equal(g.cpu()[lives], want[lives])
        assert bool((g[dead] == 7.0).all())
    # heads first in memory
    hk = k[:n].transpose(0, 1).contiguous().transpose(0, 1)
    d = _cache(B, maxT, KH)
    d.write(0, hk, v[:n], start, cu)
    assert torch.equal(c.data, d.data)


# ---------------------------------------------------------------- attention


def _want(c, q, start, counts, H, scale=HD ** -0.5):
    """(float64 output, A, max|v|) of each token and head."""
    KH, t0 = c.shape.n_kv, 0
    out = np.zeros((q.shape[0], H, HD))
    A, vmax = np.zeros((q.shape[0], H, 1)), np.zeros((q.shape[0], H, 1))
    qd = q.double().cpu().numpy()
    for b, (s, n) in enumerate(zip(start, counts)):
        T = s + n
        if n == 0 or T <= 0:
            t0 += n
            continue
        cu = [0] * (b + 1) + [T] * (c.B - b)
        k, v = (x.double().cpu().numpy() for x in c.read(0, _int([0] * c.B), _int(cu), T))
        for i in range(n):
            m = s + i + 1
            if m <= 0:
                continue
            for h in range(H):
                kh = h * KH // H
                kk, vv, x = k[:m, kh], v[:m, kh], qd[t0 + i, h]
                a = kk @ x * scale
                p = np.exp(a - a.max())
                out[t0 + i, h] = p @ vv / p.sum()
                A[t0 + i, h] = (np.abs(kk) @ np.abs(x)).max() * abs(scale)
                vmax[t0 + i, h] = np.abs(vv).max()
        t0 += n
    return out, A, vmax


def _close(got, want, A, vmax, dt):
    got = got.double().cpu().numpy()
    if dt == "f32":
        tol = (2.0 ** -18 * A + 2.0 ** -17) * vmax
    else:
        tol = (2.0 ** -9 * A + 2.0 ** -8) * vmax + 2.0 ** -8 * np.abs(want)
    off = np.abs(got - want) - tol
    assert (off <= 0).all(), f"off by {np.abs(got - want).max():.3g}, {off.max():.3g} past the bound"


def _fill(c, ends, dt, seed=11):
    for b, T in enumerate(ends):
        if T > 0:
            cu = [0] * (b + 1) + [T] * (c.B - b)
            c.write(0, _rows(seed + 2 * b, T, c.shape.n_kv, DT[dt]), _rows(seed + 2 * b + 1, T, c.shape.n_kv, DT[dt]),
                    _int([0] * c.B), _int(cu))


def _check(H, KH, counts, start, group, dt, maxT=None, qscale=1.0):
    print(f"[kv q4] attention H={H} KH={KH} {counts} at {start} g{group} {dt}", flush=True)
    ends = [s + n for s, n in zip(start, counts)]
    c = _cache(len(counts), maxT or max(max(ends), 1), KH, H, group)
    _fill(c, ends, dt)
    N = sum(counts)
    q = (_randn(99, N, H, HD) * qscale).to(DT[dt])
    cu = np.concatenate([[0], np.cumsum(counts)]).tolist()
    got = c.attention(0, q, _int(start), None if all(n == 1 for n in counts) else _int(cu))
    torch.cuda.synchronize()
    _close(got, *_want(c, q, start, counts, H), dt)
    return c, q, got


@pytest.mark.parametrize("dt,group", [("f32", 64), ("bf16", 64), ("f32", 32), ("bf16", 32)])
@pytest.mark.parametrize("H,KH,start", [(1, 1, [0]), (8, 1, [0, 1, 15]), (4, 2, [30, 31, 32, 33]), (16, 4, [63, 64, 127]),
                                        (8, 8, [128, 200]), (32, 4, [777]), (16, 2, [1500, 3, 700]), (8, 1, [5000, 1])])
def test_single_tokens(H, KH, start, dt, group):
    _check(H, KH, [1] * len(start), start, group, dt)


@pytest.mark.parametrize("dt,group", [("f32", 64), ("bf16", 32)])
@pytest.mark.parametrize("H,KH,counts,start", [(4, 4, [5, 3], [0, 40]), (8, 1, [2, 0, 7], [31, 5, 62]), (4, 2, [9, 1, 4], [300, 0, 90]),
                                               (16, 4, [17, 2], [0, 128]), (2, 1, [8, 8, 8], [0, 1, 24])])
def test_drafts(H, KH, counts, start, dt, group):
    _check(H, KH, counts, start, group, dt)


@pytest.mark.parametrize("dt,group", [("f32", 64), ("f32", 32), ("bf16", 64), ("bf16", 32)])
@pytest.mark.parametrize("H,KH,counts,start", [(8, 1, [64], [0]), (4, 1, [33, 100], [0, 31]), (2, 2, [129], [5]), (4, 2, [70, 0, 65, 1], [0, 7, 200, 300]),
                                               (8, 2, [300], [97])])
def test_prompts(H, KH, counts, start, dt, group):
    _check(H, KH, counts, start, group, dt)


@pytest.mark.parametrize("dt,group", [("f32", 64), ("bf16", 64), ("f32", 32), ("bf16", 32)])
@pytest.mark.parametrize("H,KH,counts,start", [(8, 2, [1, 1, 1, 1], [0, 31, 1027, 2900]), (2, 2, [1], [40]), (4, 1, [3, 0, 2, 5], [0, 7, 1500, 2040]),
                                               (8, 8, [7, 1], [900, 2600])])
def test_few_tokens_of_long_caches(H, KH, counts, start, dt, group):
    """Caches whose rows are cut into ranges, some of them without a row."""
    _check(H, KH, counts, start, group, dt, maxT=3001)


@pytest.mark.parametrize("dt,group", [("f32", 64), ("bf16", 32)])
@pytest.mark.parametrize("H,KH,counts,start", [(8, 1, [64], [1500]), (4, 2, [40, 0, 90], [900, 5, 1800]), (2, 2, [129], [2000]), (8, 8, [70], [700])])
def test_prompts_behind_long_prefixes(H, KH, counts, start, dt, group):
    _check(H, KH, counts, start, group, dt, maxT=4000)


@pytest.mark.parametrize("counts", [[1, 1], [3, 2], [40, 70]])
def test_rows_below_zero_see_nothing(counts):
    """A token whose row is below 0 gets 0; the sequence's later ones see what
    there is."""
    start = [-2, -1]
    c, _, got = _check(4, 2, counts, start, 64, "f32", maxT=80)
    t0 = 0
    for s, n in zip(start, counts):
        assert bool((got[t0:t0 + min(n, -s)] == 0).all())
        t0 += n


@pytest.mark.parametrize("counts", [[1, 1, 1], [2, 3, 1], [50, 40, 30]])
def test_skipped_tokens_keep_what_out_held(counts):
    """Tokens behind the last sequence, and rows past the cache's end."""
    H, KH, maxT, start = 4, 2, 64, [3, 64, 20]
    c = _cache(3, maxT, KH, H)
    _fill(c, [maxT] * 3, "f32")
    n = sum(counts)
    q = _randn(5, n + 6, H, HD)
    out = torch.full_like(q, 9.0)
    cu = np.concatenate([[0], np.cumsum(counts)]).tolist()
    c.attention(0, q, _int(start), _int(cu), out=out)
    dead = list(range(cu[1], cu[2])) + list(range(n, n + 6)) + [cu[2] + i for i in range(counts[2]) if 20 + i >= maxT] \
        + [i for i in range(counts[0]) if 3 + i >= maxT]
    live = [i for i in range(n) if i not in dead]
    assert bool((out[dead] == 9.0).all())
    keep = [counts[0], 0, counts[2]]
    want, A, vmax = _want(c, q[[*range(cu[1]), *range(cu[2], cu[3])]], [3, 0, 20], keep, H)
    pick = [i if i < cu[1] else i - counts[1] for i in live]
    _close(out[live], want[pick], A[pick], vmax[pick], "f32")


@pytest.mark.parametrize("counts,start", [([1, 1], [37, 90]), ([4, 2], [37, 90]), ([70, 66], [37, 90])])
@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_what_is_not_seen_may_be_anything(counts, start, dt):
    """Rows behind a token's own, and the other sequence, filled with NaN or
    infinite scales or the largest codes: no output changes."""
    H, KH, maxT = 8, 2, 200
    ends = [s + n for s, n in zip(start, counts)]
    res = []
    for fill in (0xFF, 0x00, 0x7C):
        c = _cache(3, maxT, KH, H)
        c.data.fill_(fill)
        _fill(c, ends, dt)
        N = sum(counts)
        q = _randn(7, N, H, HD).to(DT[dt])
        cu = [0, counts[0], N, N]
        res.append(c.attention(0, q, _int(start + [50]), _int(cu)))
    assert bool(res[0].isfinite().all())
    assert torch.equal(res[0], res[1]) and torch.equal(res[0], res[2])


@pytest.mark.parametrize("counts", [[1], [3], [100]])
def test_a_row_of_nan_reaches_those_that_see_it(counts):
    H, KH, s = 4, 2, 50
    n = counts[0]
    c = _cache(1, 200, KH, H)
    _fill(c, [s + n], "f32")
    q = _randn(8, n, H, HD)
    clean = c.attention(0, q, _int([s]), _int([0, n]))
    bad = torch.full((1, KH, HD), float("nan"), device="cuda")
    at = s + n // 2                     # only tokens n // 2 .. see it
    c.write(0, bad, bad, _int([at]))
    got = c.attention(0, q, _int([s]), _int([0, n]))
    assert torch.equal(got[:n // 2], clean[:n // 2])
    assert bool(got[n // 2:].isnan().all())


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("counts", [[1], [3], [100]])
def test_a_row_of_nan_counts_however_small_its_weight(counts, dt):
    """A visible V of NaN makes the output NaN, also where float32 has no weight
    as small as the row's, and far from the rows with weight."""
    H, KH, n = 2, 1, 1500
    for at in (3, 700, 1300):
        c = _cache(1, 2000, KH, H=H)
        k, v = torch.ones(n, KH, HD, device="cuda"), _rows(8, n, KH, DT["f32"])
        k[at] = -1.0
        v[at, :, 5] = float("nan")
        c.write(0, k.to(DT[dt]), v.to(DT[dt]), _int([0]), _int([0, n]))
        q = torch.full((counts[0], H, HD), 40.0, dtype=DT[dt], device="cuda")   # scores of 450 and -450
        got = c.attention(0, q, _int([n - counts[0]]), _int([0, counts[0]]))
        assert bool(got[..., :64].isnan().all())
        assert not bool(got[..., 64:].isnan().any())


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("counts", [[1], [3], [100]])
def test_a_query_of_nan_gives_nan(counts, dt):
    H, KH, n = 2, 1, 1500
    c = _cache(1, 2000, KH, H=H)
    _fill(c, [n], dt)
    q = _randn(12, counts[0], H, HD).to(DT[dt])
    q[0, 1, 77] = float("nan")
    got = c.attention(0, q, _int([n - counts[0]]), _int([0, counts[0]]))
    assert bool(got[0, 1].isnan().all())
    got[0, 1] = 0.0
    assert bool(got.isfinite().all())


@pytest.mark.parametrize("qscale", [1e-30, 1e-4, 30.0, 1e4])
@pytest.mark.parametrize("counts,start", [([1], [300]), ([70], [100])])
def test_magnitudes_of_q_and_of_the_rows(qscale, counts, start):
    """Scores from all alike to one that takes everything; V rows from 1e-6 to
    1e4 in one sequence."""
    H, KH = 4, 1
    ends = start[0] + counts[0]
    c = _cache(1, ends, KH, H)
    k, v = _rows(1, ends, KH, DT["f32"]), _rows(2, ends, KH, DT["f32"])
    v *= 10.0 ** (torch.arange(ends, device="cuda") % 11 - 6).float()[:, None, None]
    c.write(0, k, v, _int([0]), _int([0, ends]))
    q = _randn(3, counts[0], H, HD) * qscale
    got = c.attention(0, q, _int(start), _int([0, counts[0]]))
    _close(got, *_want(c, q, start, counts, H), "f32")


def test_small_rows_after_a_large_one():
    """A row with a huge V and no weight leaves the others' precision alone."""
    H, KH, T = 2, 1, 400
    c = _cache(1, T, KH, H)
    k, v = _rows(1, T, KH, DT["f32"]), _rows(2, T, KH, DT["f32"]) * 1e-3
    q = _randn(3, 1, H, HD)
    k[0] = -40.0 * q[0, 0]              # head 0 never looks at it
    v[0] = 1e4
    c.write(0, k, v, _int([0]), _int([0, T]))
    got = c.attention(0, q[:, :2], _int([T - 1])).double().cpu().numpy()
    want, A, vmax = _want(c, q, [T - 1], [1], H)
    rest = np.abs(c.read(0, _int([0]), _int([0, T]), T)[1].cpu().numpy()[1:]).max()
    assert np.abs(got - want)[0, 0].max() <= (2.0 ** -18 * A[0, 0, 0] + 2.0 ** -17) * rest


@pytest.mark.parametrize("counts", [[1], [130]])
def test_a_few_rows_of_v_far_above_the_others(counts):
    """The others hold no more than the weights' sum, which has to be whole: an
    output is the few rows' share of it times their value, and relative to that
    off by the weights' errors alone (2^-9 A of each score and 2^-11 of each weight
    on both sides of the quotient) and the output's rounding."""
    H, KH, n = 2, 1, 400
    for first in (0, 128, 384):
        c = _cache(1, 600, KH, H=H)
        k, v = _rows(31, n, KH, torch.bfloat16), torch.zeros(n, KH, HD, dtype=torch.bfloat16, device="cuda")
        v[first:first + 4] = 3e4
        c.write(0, k, v, _int([0]), _int([0, n]))
        st = [n - counts[0]]
        q = (_randn(32, counts[0], H, HD) * 0.05).to(torch.bfloat16)
        got = c.attention(0, q, _int(st), _int([0, counts[0]])).double().cpu().numpy()
        want, A, _ = _want(c, q, st, counts, H)
        assert (np.abs(got - want) <= (2.0 ** -8 * A + 2.0 ** -8 + 2.0 ** -10) * np.abs(want)).all()


def test_strided_q_in_place_and_scale():
    H, KH, T = 8, 2, 90
    c = _cache(2, T, KH, H)
    _fill(c, [T, T], "f32")
    fused = _randn(4, 2, H + 4, HD)
    start = _int([70, 89])
    a = c.attention(0, fused[:, 2:2 + H], start, scale=0.3)
    want, A, vmax = _want(c, fused[:, 2:2 + H], [70, 89], [1, 1], H, scale=0.3)
    _close(a, want, A, vmax, "f32")
    q = fused[:, 2:2 + H].contiguous()
    b = c.attention(0, q, start, out=q, scale=0.3)
    assert b.data_ptr() == q.data_ptr() and torch.equal(a, b)
    n = 2 * 66
    q = _randn(5, n, H, HD)
    a = c.attention(0, q, _int([4, 0]), _int([0, 66, n]))
    c.attention(0, q, _int([4, 0]), _int([0, 66, n]), out=q)
    assert torch.equal(a, q)


def test_long_cache_past_32_bits():
    """A cache set whose planes lie more than 4 GiB apart, and rows past 2^16."""
    KH, H, T = 2, 4, 70000
    shape = DecoderShape(n_layers=240, moe=dense_ffn_shape(1024, 512), n_heads=H, n_kv=KH, maxT=T)
    c = Q4KVCacheSet(shape, 2)
    assert c.data.numel() > 2 ** 32
    k, v = _rows(1, 300, KH, DT["f32"]), _rows(2, 300, KH, DT["f32"])
    s = T - 300
    c.write(239, k, v, _int([0, s]), _int([0, 0, 300]))
    gk, gv = c.read(239, _int([0, s]), _int([0, 0, 300]), 300)
    assert np.array_equal(gk.cpu().numpy(), _held(k, 64)) and np.array_equal(gv.cpu().numpy(), _held(v, 64))
    assert not bool(c.data[:, :239].any()) and not bool(c.data[0].any())
    # every other row holds 0: equal weights but for the last 300
    q = _randn(3, 2, H, HD)
    got = c.attention(239, q, _int([10, T - 1])).double().cpu().numpy()
    assert not got[0].any()
    kd, vd, qd = gk.double().cpu().numpy(), gv.double().cpu().numpy(), q.double().cpu().numpy()
    for h in range(H):
        e = np.exp(kd[:, h // 2] @ qd[1, h] * HD ** -0.5)
        want = e @ vd[:, h // 2] / (e.sum() + s)
        assert np.abs(got[1, h] - want).max() <= 2.0 ** -17 * np.abs(vd).max()


def test_captured_and_replayed_and_other_streams():
    H, KH, T = 8, 2, 700
    c = _cache(2, T, KH, H)
    _fill(c, [T, T], "f32")
    k, v, q = _rows(1, 2, KH, DT["f32"]), _rows(2, 2, KH, DT["f32"]), _randn(3, 2, H, HD)
    start = _int([650, 600])
    out, rk, rv = torch.empty_like(q), torch.empty_like(k), torch.empty_like(v)

    def step():
        c.write(0, k, v, start)
        c.attention(0, q, start, out=out)
        c.read(0, start, k=rk, v=rv)

    step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):                  # two graphs, each with a workspace of its own
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            step()
        graphs.append(g)
    for i in range(4):
        k.copy_(_rows(10 + i, 2, KH, DT["f32"]))
        v.copy_(_rows(20 + i, 2, KH, DT["f32"]))
        q.copy_(_randn(30 + i, 2, H, HD))
        start.copy_(_int([600 + i, 20 + 100 * i]))
        graphs[i % 2].replay()
        torch.cuda.synchronize()
        got = [x.clone() for x in (out, rk, rv)]
        step()
        torch.cuda.synchronize()
        for a, b in zip(got, (out, rk, rv)):
            assert torch.equal(a, b)
        other = c.attention(0, q, start, stream=side)
        side.synchronize()
        assert torch.equal(other, out)


def test_the_same_call_gives_the_same_bits():
    for counts, start in (([1] * 5, [900, 3, 250, 64, 511]), ([200], [300])):
        c = _cache(len(counts), 1000, 2, 8)
        _fill(c, [s + n for s, n in zip(start, counts)], "f32")
        q = _randn(1, sum(counts), 8, HD)
        cu = _int(np.concatenate([[0], np.cumsum(counts)]).tolist())
        a = c.attention(0, q, _int(start), cu)
        for _ in range(5):
            assert torch.equal(a, c.attention(0, q, _int(start), cu))


def test_python_refusals():
    c = _cache(2, 64, 2, 4)
    k, q, start = _rows(1, 2, 2, torch.float32), _randn(2, 2, 4, HD), _int([0, 1])
    bad = [lambda: c.write(1, k, k, start), lambda: c.write(-1, k, k, start), lambda: c.write(0, k[:, :1], k, start),
           lambda: c.write(0, k, k.bfloat16(), start), lambda: c.write(0, k.half(), k.half(), start),
           lambda: c.write(0, k.cpu(), k, start), lambda: c.write(0, k, k, start.long()),
           lambda: c.write(0, k, k, start.cpu()), lambda: c.write(0, k, k, start[:1]),
           lambda: c.write(0, k, k, start, _int([0, 2])), lambda: c.write(0, k[:1], k[:1], start),
           lambda: c.write(0, k.transpose(1, 2).contiguous().transpose(1, 2), k, start),
           lambda: c.read(0, start, _int([0, 1, 2])), lambda: c.read(0, start, n=3), lambda: c.read(0, start, dtype=torch.float16),
           lambda: c.read(0, start, k=k[:, :, :64]), lambda: c.read(0, start, k=k.transpose(0, 1).contiguous().transpose(0, 1)),
           lambda: c.attention(0, q[0], start), lambda: c.attention(0, q, start, out=q.bfloat16()),
           lambda: c.attention(0, q[:, :, :64], start), lambda: c.attention(0, torch.empty(3, 4, HD, device="cuda"), start),
           lambda: c.attention(0, torch.empty(2 * 4 * HD + 2, device="cuda")[2:].view(2, 4, HD), start),
           lambda: Q4KVCacheSet(c.shape, 2, group=16), lambda: Q4KVCacheSet(c.shape, 2, data=c.data[:1])]
    for i, f in enumerate(bad):
        with pytest.raises((ValueError, _lib.JouleError)):
            f()
            pytest.fail(f"call {i} was taken")
    with pytest.raises(_lib.JouleError):
        c.attention(0, torch.empty(2, 6, HD, device="cuda"), start)
    # nothing to do
    none = torch.empty(0, 2, HD, device="cuda")
    c.write(0, none, none, start, _int([0, 0, 0]))
    assert c.attention(0, torch.empty(0, 4, HD, device="cuda"), start, _int([0, 0, 0])).shape == (0, 4, HD)
    assert c.read(0, start, _int([0, 0, 0]), 0)[0].shape == (0, 2, HD)
