"""Paged KV caches: rows appended and attention over the pages, against float64
(oracle/paged.py, which derives the bounds)."""

import numpy as np
import pytest
import torch

from joule_amd.decoder import DecoderShape, rope_tables
from joule_amd.dense import dense_ffn_shape
from joule_amd.kv_paged import PagedKVCacheSet
from oracle.paged import attend, finish

pytestmark = pytest.mark.gpu

HD = 128
DT = {"f32": torch.float32, "bf16": torch.bfloat16}
HALF = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8}           # half a step of a value, relative


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


DEEP = 2 ** 19          # a maxT whose calls are cut as if the prefixes were as long


def cache(B, maxT, KH, page=16, dtype="bf16", layers=1, extra=3, seed=0, rows=None):
    """Caches of NaN, every sequence's pages (for maxT rows, or for `rows`) anywhere in
    the pool."""
    shape = DecoderShape(n_layers=layers, moe=dense_ffn_shape(1024, 512), n_heads=KH, n_kv=KH, maxT=maxT)
    width = -(-(rows or maxT) // page)
    c = PagedKVCacheSet(shape, B, B * width + extra, page=page, dtype=DT[dtype])
    c.data.fill_(float("nan"))
    order = np.random.default_rng(seed).permutation(B * width + extra)[:B * width]
    c.table[:, :width] = ints(order.reshape(B, width).tolist())
    return c


def put(c, b, k, v, l=0, first=0):
    """Rows first .. of sequence b, by plain indexing."""
    r = np.arange(first, first + len(k))
    table = c.table.cpu().numpy()
    page = torch.from_numpy(table[b, r // c.page].astype(np.int64)).cuda()
    at = torch.from_numpy(r % c.page).cuda()
    for i, x in enumerate((k, v)):
        c.data[l, page, i, :, at] = torch.as_tensor(x, device="cuda").to(c.data.dtype)


def held(c, b, n, l=0):
    """k and v [n, KH, 128] in float32 of rows 0 .. n - 1; NaN without a page."""
    t = c.table[b, :-(-n // c.page)].long()
    x = c.data[l, t.clamp(0, c.n_pages - 1)].float()
    x[(t < 0) | (t >= c.n_pages)] = float("nan")
    x = x.permute(1, 0, 3, 2, 4).reshape(2, -1, c.shape.n_kv, HD)[:, :n].cpu().numpy()
    return x[0], x[1]


def rows(seed, T, KH):
    rng = np.random.default_rng(seed)
    k, v = (rng.standard_normal((T, KH, HD)).astype(np.float32) for _ in range(2))
    k[:, :, 3::17] *= 2.0
    return k, v


def queries(seed, k, start, n, H):
    """n tokens from row `start` on, each looking at its own row and the one before."""
    rng = np.random.default_rng(seed)
    KH = k.shape[1]
    q = rng.standard_normal((n, H, HD)).astype(np.float32)
    for i in range(n):
        at = max(start + i - 1, 0)
        for h in range(H):
            q[i, h] += 0.4 * np.nan_to_num(k[at:start + i + 1, h * KH // H]).sum(axis=0)
    return q


def form_of(c, dt, n, H, KH, n_seq, max_rows=0):
    """As the entry point decides for a call with cu: a prompt where a sequence has 32 query
    rows a KV head, and the rows (512 at least) that the units of 16 query rows pass over
    are 450000."""
    units = min(n_seq * -(-(-(-n // n_seq)) // (16 * KH // H)), n)
    prompt = n * (H // KH) >= 32 * n_seq and units * KH * max(min(max_rows or c.shape.maxT, c.shape.maxT), 512) >= 450000
    return "f32" if dt == "f32" else "bf16 prompt" if c.data.dtype == torch.bfloat16 and prompt else "bf16"


def check(c, q, start, counts, dt, scale=HD ** -0.5, out=None, max_rows=0, only=None, one=False):
    """attention() of tokens q [N, H, 128] (numpy) against float64; returns the output."""
    H, KH = q.shape[1], c.shape.n_kv
    qd = torch.from_numpy(q).cuda().to(DT[dt])
    cu = np.concatenate([[0], np.cumsum(counts)]).tolist()
    print(f"[paged] H={H} KH={KH} {counts} at {start} of {c.shape.maxT} page {c.page} {dt}/{c.data.dtype} scale {scale} max_rows {max_rows}",
          flush=True)
    got = c.attention(0, qd, ints(start), None if one else ints(cu), scale=scale, out=out, max_rows=max_rows)
    torch.cuda.synchronize()
    g64, q64 = got.double().cpu().numpy(), qd.float().cpu().numpy()
    table = c.table.cpu().numpy()
    form = "bf16" if one and dt == "bf16" else form_of(c, dt, len(q), H, KH, len(counts), max_rows)
    for b, (s, n) in enumerate(zip(start, counts)):
        T = s + n
        if n == 0 or T <= 0:
            continue
        k, v = held(c, b, T)
        t = np.arange(T)
        paged = (table[b, t // c.page] >= 0) & (table[b, t // c.page] < c.n_pages)
        pick = np.array(sorted({0, n - 1, *np.random.default_rng(n).integers(0, n, 30).tolist()}))
        if only == "before":                    # tokens in front of the middle one
            pick = np.array(sorted({*pick[pick < n // 2].tolist(), max(n // 2 - 1, 0)})) if n > 1 else np.array([], int)
            if len(pick) == 0:
                continue
        pick = pick[s + pick < c.shape.maxT]
        see = paged & (t <= s + pick[:, None])
        for h in range(H):
            want, tol = attend(q64[cu[b] + pick, h], k[:, h * KH // H], v[:, h * KH // H], see, scale, form)
            off = np.abs(g64[cu[b] + pick, h] - want)
            worst = np.nanmax(off / np.maximum(tol, 1e-300))
            assert (off <= tol).all(), f"sequence {b} head {h}: {worst:.3g} bounds off, by {np.nanmax(off):.3g}"
    return got


def run(H, KH, counts, start, dt, cached, page=16, maxT=None, **kw):
    T = max(s + n for s, n in zip(start, counts))
    c = cache(len(counts), maxT or T, KH, page, cached, rows=max(T, 1) if maxT == DEEP else None)
    q = []
    for b, (s, n) in enumerate(zip(start, counts)):
        k, v = rows(7 * b + 1, max(s + n, 1), KH)
        if s + n > 0:
            put(c, b, k[:s + n], v[:s + n])
        q.append(queries(b + 100, k, s, n, H))
    return check(c, np.concatenate(q), start, counts, dt, **kw)


# ------------------------------------------------------------------ append


def append_case(H, KH, counts, start, dt, cached, page, norm, rope, maxT=None, l=0, layers=1, inplace=False, strided=False):
    T = maxT or max(max(s + n for s, n in zip(start, counts)), 1)
    c = cache(len(counts), T, KH, page, cached, layers=layers)
    N = sum(counts)
    rng = np.random.default_rng(N + H)
    x = [torch.from_numpy(rng.standard_normal((N, h, HD)).astype(np.float32)).cuda().to(DT[dt]) for h in (H, KH, KH)]
    if strided:
        full = torch.zeros((N, H + 2 * KH + 1, HD + 4), dtype=DT[dt], device="cuda")
        out, at = [], 0
        for y in x:
            z = full[:, at:at + y.shape[1], :HD]
            z.copy_(y)
            out.append(z)
            at += y.shape[1]
        x = out
    q, k, v = x
    w = [torch.from_numpy((1 + 0.3 * rng.standard_normal(HD)).astype(np.float32)).cuda().bfloat16() for _ in range(2)] if norm else [None, None]
    tables = rope_tables(T, HD, 1e4) if rope else (None, None)
    cos, sin = (None if t is None else torch.from_numpy(t).cuda() for t in tables)
    cu = np.concatenate([[0], np.cumsum(counts)])
    before = c.data.clone()
    want_in = [t.float().cpu().numpy() for t in (q, k, v)]
    print(f"[append] H={H} KH={KH} {counts} at {start} page {page} {dt}/{cached} norm {norm} rope {rope}", flush=True)
    got = c.append(l, k, v, ints(start), ints(cu.tolist()), q=q, cos=cos, sin=sin, q_norm=w[0], k_norm=w[1], eps=1e-5,
                   q_out=q if inplace else None)
    torch.cuda.synchronize()
    row = np.concatenate([np.arange(s, s + n) for s, n in zip(start, counts)]).astype(np.int64)
    seq = np.repeat(np.arange(len(counts)), counts)
    live = (row >= 0) & (row < T)
    r = np.clip(row, 0, T - 1)
    wn = [None if y is None else y.float().cpu().numpy() for y in w]
    wq, wk = (finish(want_in[i], r, wn[i], tables[0], tables[1], 1e-5) for i in range(2))
    # 12 float32 roundings of values of at most |x| + |partner|, in the sum of squares half of
    # 128 more; then the type's own
    room = [(12 + 64 * norm) * 2.0 ** -24 * (np.abs(y) + np.abs(np.roll(y, HD // 2, axis=-1)) + 1e-30) for y in (wq, wk)]
    g = got.double().cpu().numpy()
    assert (np.abs(g - wq) <= room[0] + HALF[dt] * np.abs(wq))[live].all()
    table = c.table.cpu().numpy()
    page_of = table[np.where(live, seq, 0), np.where(live, row, 0) // page]
    ok = live & (page_of >= 0) & (page_of < c.n_pages)
    idx = (torch.from_numpy(page_of[ok].astype(np.int64)).cuda(), torch.from_numpy(row[ok] % page).cuda())
    gk, gv = (c.data[l, idx[0], i, :, idx[1]].double().cpu().numpy() for i in range(2))
    assert (np.abs(gk - wk[ok]) <= room[1][ok] + HALF[cached] * np.abs(wk[ok])).all()
    assert np.array_equal(gv, torch.from_numpy(want_in[2][ok]).to(DT[cached]).double().numpy())
    # nothing else was touched
    for i in range(2):
        before[l, idx[0], i, :, idx[1]] = c.data[l, idx[0], i, :, idx[1]]
    assert torch.equal(before.view(torch.uint8), c.data.view(torch.uint8))
    return c, got


@pytest.mark.parametrize("dt,cached", [("f32", "bf16"), ("bf16", "bf16"), ("f32", "f32"), ("bf16", "f32")])
@pytest.mark.parametrize("norm,rope", [(False, False), (True, False), (False, True), (True, True)])
@pytest.mark.parametrize("H,KH,counts,start,page", [(1, 1, [1], [0], 16), (8, 2, [3, 0, 40], [14, 7, 0], 16), (28, 4, [17, 33], [31, 64], 32),
                                                    (16, 16, [1, 1, 1], [5, 100, 31], 64), (5, 1, [130], [60], 128)])
def test_append(H, KH, counts, start, page, norm, rope, dt, cached):
    append_case(H, KH, counts, start, dt, cached, page, norm, rope)


@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_append_in_place_strided_and_in_a_later_layer(dt):
    append_case(8, 2, [3, 5], [0, 20], dt, "bf16", 16, True, True, inplace=True)
    append_case(8, 2, [3, 5], [0, 20], dt, "bf16", 16, True, True, strided=True)
    append_case(7, 1, [9], [11], dt, "f32", 32, False, True, layers=3, l=2)


@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_append_skips_rows_outside(dt):
    append_case(4, 2, [5, 6, 3], [-2, 28, 500], dt, "bf16", 16, True, True, maxT=30)


# --------------------------------------------------------------- attention

TYPES = [("f32", "bf16"), ("bf16", "bf16"), ("f32", "f32"), ("bf16", "f32")]


@pytest.mark.parametrize("dt,cached", TYPES)
@pytest.mark.parametrize("H,KH,page", [(1, 1, 16), (8, 2, 32), (28, 4, 16), (16, 1, 64), (12, 4, 128), (5, 5, 16)])
@pytest.mark.parametrize("start", [[0], [15, 16, 17], [30, 700, 31, 63], [2500, 3]])
def test_single_tokens(H, KH, page, start, dt, cached):
    run(H, KH, [1] * len(start), start, dt, cached, page, one=True)


@pytest.mark.parametrize("dt,cached", TYPES)
@pytest.mark.parametrize("H,KH,counts,start", [(8, 2, [5, 0, 3], [900, 4, 12]), (7, 1, [2, 9], [15, 1300]), (2, 2, [16, 17], [0, 40]),
                                               (16, 1, [4], [2222])])
def test_few_tokens(H, KH, counts, start, dt, cached):
    run(H, KH, counts, start, dt, cached)


@pytest.mark.parametrize("dt,cached", TYPES)
@pytest.mark.parametrize("H,KH", [(3, 1), (5, 1), (9, 1), (11, 1), (13, 1), (15, 1), (10, 2), (28, 4)])
@pytest.mark.parametrize("counts,start", [([1, 1], [1039, 746]), ([1, 0, 2, 7, 1], [2100, 5, 1500, 900, 1039]), ([40, 133], [700, 1515])])
def test_ranges_of_heads_that_do_not_fill_a_unit(H, KH, counts, start, dt, cached):
    """Units of 9 to 15 query rows (of 117 to 126 in a long cache) whose outputs are joined."""
    run(H, KH, counts, start, dt, cached, 64)
    run(H, KH, counts, start, dt, cached, 64, maxT=DEEP)


@pytest.mark.parametrize("dt,cached", TYPES)
@pytest.mark.parametrize("H,KH,counts,start,page", [(8, 1, [64], [1500], 16), (2, 2, [129], [2000], 64), (6, 2, [300], [97], 32),
                                                    (8, 8, [130], [700], 16), (4, 2, [130, 0, 90], [900, 5, 1800], 128), (7, 1, [201], [0], 16)])
def test_prompts(H, KH, counts, start, page, dt, cached):
    run(H, KH, counts, start, dt, cached, page, maxT=4000)
    run(H, KH, counts, start, dt, cached, page)
    run(H, KH, counts, start, dt, cached, page, maxT=DEEP)


@pytest.mark.parametrize("dt,cached", TYPES)
@pytest.mark.parametrize("H,KH,counts,start,page", [(64, 64, [260], [100], 32), (128, 128, [260], [77], 16), (128, 32, [130], [400], 16),
                                                    (112, 16, [70, 140], [0, 250], 64), (40, 40, [90, 33, 99, 1], [200, 31, 0, 409], 16)])
def test_prompts_of_many_heads(H, KH, counts, start, page, dt, cached):
    """In one range of rows, without a kernel that joins them."""
    run(H, KH, counts, start, dt, cached, page, maxT=600)
    run(H, KH, counts, start, dt, cached, page)


@pytest.mark.parametrize("dt,cached", TYPES)
@pytest.mark.parametrize("counts,start", [([1], [777]), ([5], [777]), ([70], [700])])
@pytest.mark.parametrize("max_rows", [1, 700, 1025, 5000, 100000, 2 ** 31 - 1])
def test_max_rows_only_cuts(counts, start, max_rows, dt, cached):
    """Any bound gives the same, too small or too large."""
    run(4, 2, counts, start, dt, cached, maxT=120000, max_rows=max_rows)


# ------------------------------------------------- what is not finite, what is not there

CALLS = [(4, 2, [1], [40]), (8, 1, [2], [500]), (4, 2, [5, 0, 3], [40, 9, 700]), (2, 2, [100, 130], [0, 333]), (7, 1, [150], [77]),
         (16, 2, [300], [600])]


def prepared(H, KH, counts, start, cached, maxT, page=16, seed=0):
    c = cache(len(counts), maxT, KH, page, cached, seed=seed, rows=1500 if maxT == DEEP else None)
    q = []
    for b, (s, n) in enumerate(zip(start, counts)):
        k, v = rows(7 * b + 1, max(s + n, 1), KH)
        if s + n > 0:
            put(c, b, k[:s + n], v[:s + n])
        q.append(queries(b + 100, k, s, n, H))
    return c, np.concatenate(q)


@pytest.mark.parametrize("dt,cached", TYPES)
@pytest.mark.parametrize("H,KH,counts,start", CALLS)
@pytest.mark.parametrize("maxT", [0, 1500, DEEP])
def test_rows_of_later_tokens_may_hold_anything(H, KH, counts, start, maxT, dt, cached):
    """NaN and infinities in K and V of a token's row do not reach the tokens before
    it; the tokens from it on get what the formula gives."""
    T = maxT or max(s + n for s, n in zip(start, counts))
    cu = np.concatenate([[0], np.cumsum(counts)])
    for value in (float("nan"), float("inf"), -float("inf"), 3e38):
        c, q = prepared(H, KH, counts, start, cached, T)
        late = []
        for b, (s, n) in enumerate(zip(start, counts)):
            if not n:
                continue
            k, v = (x[s + n // 2:s + n // 2 + 1].copy() for x in held(c, b, s + n))
            v[:, :, 5], v[:, 0, 77] = value, -value
            put(c, b, k, v, first=s + n // 2)
            late += range(int(cu[b]) + n // 2, int(cu[b]) + n)
        got = check(c, q, start, counts, dt, only="before")
        if value != 3e38:
            x = got[late].float()
            assert not bool(x[:, :, 5].isfinite().any()) and not bool(x[:, 0, 77].isfinite().any())
            x[:, :, 5] = 0.0
            x[:, :, 77] = 0.0
            assert bool(x.isfinite().all())
        # the same in K
        for b, (s, n) in enumerate(zip(start, counts)):
            if n:
                k, v = (x[s + n // 2:s + n // 2 + 1].copy() for x in held(c, b, s + n))
                k[:, :, 3] = value
                put(c, b, k, v, first=s + n // 2)
        check(c, q, start, counts, dt, only="before")


@pytest.mark.parametrize("dt,cached", TYPES)
@pytest.mark.parametrize("H,KH,counts,start", CALLS)
@pytest.mark.parametrize("maxT", [1500, DEEP])
def test_pages_that_are_not_there(H, KH, counts, start, maxT, dt, cached):
    """Rows of pages given back, of numbers outside the pool and of pages still to
    come are not seen; a token that sees none gets 0."""
    for gone in ([0], [1, 2], [3], [0, 1, 2, 3, 4, 5], list(range(400))):
        c, q = prepared(H, KH, counts, start, cached, maxT)
        for b in range(c.B):
            for i, p in enumerate(gone):
                if p < c.table.shape[1]:
                    c.table[b, p] = [-1, c.n_pages, 2 ** 31 - 1, -2 ** 31][i % 4]
        # (the pages of NaN behind the rows, and those that others hold, are not read in their place)
        got = check(c, q, start, counts, dt)
        if len(gone) == 400:
            assert not bool(got.any())


@pytest.mark.parametrize("dt,cached", TYPES)
@pytest.mark.parametrize("H,KH,counts,start", [(4, 2, [1, 1], [-1, 20]), (4, 2, [3, 5], [-2, -9]), (4, 2, [100, 130], [-40, 900]), (4, 2, [70, 70], [-200, 960]),
                                               (64, 64, [300, 70], [-200, 960])])
def test_tokens_without_rows_and_rows_outside(H, KH, counts, start, dt, cached):
    """A row below 0: 0.  A row past the cache, and tokens behind the last sequence:
    left as they were."""
    T = 1000
    c, q = prepared(H, KH, counts, [min(s, T - n) for s, n in zip(start, counts)], cached, T)
    q = np.concatenate([q, q[:3]])
    out = torch.full((len(q), H, HD), 7.0, dtype=DT[dt], device="cuda")
    cu = np.concatenate([[0], np.cumsum(counts)])
    qd = torch.from_numpy(q).cuda().to(DT[dt])
    qd[0, 0, 5] = float("nan")
    got = c.attention(0, qd, ints(start), ints(cu.tolist()), out=out)
    torch.cuda.synchronize()
    assert got.data_ptr() == out.data_ptr()
    for b, (s, n) in enumerate(zip(start, counts)):
        r = torch.arange(s, s + n, device="cuda")
        x = got[int(cu[b]):int(cu[b + 1])]
        assert not bool(x[r < 0].any())
        assert bool((x[r >= T] == 7.0).all())
        assert bool(x[(r >= 0) & (r < T)].isfinite().all())
    assert bool((got[int(cu[-1]):] == 7.0).all())


@pytest.mark.parametrize("scale", [0.0, -0.0, 1e-38, 1e-9, -0.3, -HD ** -0.5, 1.0])
@pytest.mark.parametrize("dt,cached", TYPES)
def test_scales_of_any_sign_and_zero(dt, cached, scale):
    for H, KH, counts, start in CALLS:
        run(H, KH, counts, start, dt, cached, scale=scale)
        run(H, KH, counts, start, dt, cached, scale=scale, maxT=DEEP)


@pytest.mark.parametrize("dt,cached", TYPES)
@pytest.mark.parametrize("H,KH,counts,start", CALLS)
@pytest.mark.parametrize("maxT", [1500, DEEP])
def test_an_infinite_query_gives_nan(H, KH, counts, start, maxT, dt, cached):
    c, q = prepared(H, KH, counts, start, cached, maxT)
    q[:, 1, 77] = np.inf
    q[0, 0, 5] = -np.inf
    cu = np.concatenate([[0], np.cumsum(counts)])
    got = c.attention(0, torch.from_numpy(q).cuda().to(DT[dt]), ints(start), ints(cu.tolist()))
    assert bool(got[:, 1].isnan().all()) and bool(got[0, 0].isnan().all())
    got[:, 1] = 0.0
    got[0, 0] = 0.0
    assert bool(got.isfinite().all())


@pytest.mark.parametrize("dt,cached", TYPES)
@pytest.mark.parametrize("H,KH,counts,start", CALLS)
@pytest.mark.parametrize("maxT", [1500, DEEP])
def test_weights_far_apart(H, KH, counts, start, maxT, dt, cached):
    """Scores of hundreds: one row has all the weight, the reference rises often."""
    c, q = prepared(H, KH, counts, start, cached, maxT)
    check(c, q * 30.0, start, counts, dt)
    check(c, q * 1e-4, start, counts, dt)
