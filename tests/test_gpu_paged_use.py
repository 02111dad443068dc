"""Paged KV caches as a server uses them: prompts, steps and drafts after one another,
pages given out, shared and taken back, other streams, replayed graphs, host threads,
pools past 4 GiB."""

import threading

import numpy as np
import pytest
import torch

from joule_amd import _lib
from joule_amd.decoder import DecoderShape, rope_tables
from joule_amd.dense import dense_ffn_shape
from joule_amd.kv_paged import PagedKVCacheSet
from oracle.paged import attend, finish
from test_gpu_paged import DT, HALF, TYPES, cache, check, held, ints, prepared, put, queries, rows, run

pytestmark = pytest.mark.gpu

HD = 128


def shape_of(KH, H, maxT, layers=1):
    return DecoderShape(n_layers=layers, moe=dense_ffn_shape(1024, 512), n_heads=H, n_kv=KH, maxT=maxT)


# -------------------------------------------------------------- one after the other


class Server:
    """A host of one layer: every call appends its tokens and attends, and is checked
    against float64 over all the rows that its sequences were given."""

    def __init__(self, H, KH, B, n_pages, page, dt, cached, maxT=4000):
        self.H, self.KH, self.dt, self.cached = H, KH, dt, cached
        self.c = PagedKVCacheSet(shape_of(KH, H, maxT), B, n_pages, page=page, dtype=DT[cached])
        self.c.data.fill_(float("nan"))
        self.rng = np.random.default_rng(H * B + page)
        self.tables = rope_tables(maxT, HD, 1e4)
        self.cos, self.sin = (torch.from_numpy(t).cuda() for t in self.tables)
        self.w = [torch.from_numpy((1 + 0.3 * self.rng.standard_normal(HD)).astype(np.float32)).cuda().bfloat16() for _ in range(2)]
        self.k = [np.zeros((0, KH, HD)) for _ in range(B)]              # what the rows should hold, float64
        self.v = [np.zeros((0, KH, HD)) for _ in range(B)]

    def call(self, counts, draft=0):
        """counts[b] new tokens of each sequence; with draft, the last `draft` of them are
        refused afterwards: the next call writes over them."""
        start = [len(k) for k in self.k]
        for b, n in enumerate(counts):
            if n:
                self.c.reserve(b, start[b] + n)
        N = sum(counts)
        x = [torch.from_numpy(self.rng.standard_normal((N, h, HD)).astype(np.float32)).cuda().to(DT[self.dt])
             for h in (self.H, self.KH, self.KH)]
        cu = np.concatenate([[0], np.cumsum(counts)]).tolist()
        at, upto = ints(start), ints(cu)
        print(f"[server] {counts} at {start}", flush=True)
        q = self.c.append(0, x[1], x[2], at, upto, q=x[0], cos=self.cos, sin=self.sin, q_norm=self.w[0], k_norm=self.w[1])
        out = self.c.attention(0, q, at, upto)
        torch.cuda.synchronize()
        row = np.concatenate([np.arange(s, s + n) for s, n in zip(start, counts)]).astype(np.int64)
        wk = finish(x[1].float().cpu().numpy(), row, self.w[1].float().cpu().numpy(), *self.tables, 1e-6)
        q64, o64, v64 = q.double().cpu().numpy(), out.double().cpu().numpy(), x[2].float().cpu().numpy()
        for b, n in enumerate(counts):
            if not n:
                continue
            gk, gv = held(self.c, b, start[b] + n)
            # rows of this call and of all before it, rounded once
            self.k[b] = np.concatenate([self.k[b], wk[cu[b]:cu[b + 1]]])
            self.v[b] = np.concatenate([self.v[b], v64[cu[b]:cu[b + 1]]])
            room = 80 * 2.0 ** -24 * (np.abs(self.k[b]) + np.abs(np.roll(self.k[b], HD // 2, axis=-1)) + 1e-30)
            assert (np.abs(gk - self.k[b]) <= room + HALF[self.cached] * np.abs(self.k[b])).all()
            assert np.array_equal(gv, torch.from_numpy(self.v[b]).to(DT[self.cached]).float().numpy())
            t = np.arange(start[b] + n)
            pick = np.unique(np.r_[0, n - 1, self.rng.integers(0, n, 6)])
            for h in range(self.H):
                g = h * self.KH // self.H
                want, tol = attend(q64[cu[b] + pick, h], gk[:, g], gv[:, g], t <= start[b] + pick[:, None], HD ** -0.5,
                                   "f32" if self.dt == "f32" else "bf16 prompt")
                off = np.abs(o64[cu[b] + pick, h] - want)
                assert (off <= tol).all(), f"sequence {b} head {h}: {np.nanmax(off / tol):.3g} bounds off"
            if draft:
                self.k[b], self.v[b] = self.k[b][:-draft], self.v[b][:-draft]


@pytest.mark.parametrize("dt,cached", TYPES)
@pytest.mark.parametrize("H,KH,page", [(8, 2, 16), (7, 1, 64), (4, 4, 32)])
def test_prompts_steps_drafts_sharing_and_release(H, KH, page, dt, cached):
    s = Server(H, KH, 4, 2000 // page + 12, page, dt, cached)
    total = s.c.free_pages()
    s.call([300, 0, 77, 1])
    for _ in range(3):
        s.call([1, 0, 1, 1])
    s.call([5, 0, 4, 4], draft=3)                       # two, one and one token of the draft are kept
    s.call([1, 0, 1, 1])
    # the second sequence begins with most of the first's rows, and each goes its own way
    before = s.c.free_pages()
    n = len(s.k[0]) - 3
    s.c.share(0, 1, n)
    assert before - s.c.free_pages() == (1 if n % page else 0)
    s.k[1], s.v[1] = s.k[0][:n].copy(), s.v[0][:n].copy()
    s.call([1, 2, 0, 0])
    s.call([40, 130, 0, 1])
    # the first leaves; what the second has in common stays
    s.c.release(0)
    s.k[0], s.v[0] = s.k[0][:0], s.v[0][:0]
    assert bool((s.c.table[0] == -1).all())
    s.call([0, 1, 1, 1])
    # another takes its place, on pages that others held
    s.call([500, 1, 200, 0])
    s.call([1, 1, 1, 1])
    for b in range(4):
        s.c.release(b)
    assert s.c.free_pages() == total and bool((s.c.table == -1).all())


def test_page_keeping():
    c = PagedKVCacheSet(shape_of(2, 4, 100), 3, 6, page=16)
    assert c.table.shape == (3, 7) and c.free_pages() == 6
    c.reserve(0, 0)
    c.reserve(0, 33)
    assert c.free_pages() == 3
    first = c.table[0].tolist()
    c.reserve(0, 20)                                    # it has them
    c.reserve(0, 48)
    assert c.table[0].tolist() == first and first[3:] == [-1] * 4 and len(set(first[:3])) == 3
    with pytest.raises(RuntimeError, match="4 more pages, 3 are free"):
        c.reserve(1, 64)
    assert c.free_pages() == 3 and bool((c.table[1] == -1).all())
    c.data.fill_(0.0)
    c.data[:, first[1]] = 2.0
    c.share(0, 1, 31)                                   # one whole page, and 15 rows of the next, copied
    second = c.table[1].tolist()
    assert second[0] == first[0] and second[1] not in first and second[2:] == [-1] * 5 and c.free_pages() == 2
    assert bool((c.data[:, second[1]] == 2.0).all())
    c.share(0, 2, 32)
    assert c.table[2].tolist()[:3] == first[:2] + [-1] and c.free_pages() == 2
    for what in (lambda: c.share(0, 1, 16), lambda: c.share(1, 0, 16)):
        with pytest.raises(ValueError, match="has pages already"):
            what()
    c.release(0)
    assert c.free_pages() == 3                          # the third page; two are held in common
    c.release(0)
    c.release(2)
    assert c.free_pages() == 4
    with pytest.raises(ValueError, match="has pages for 32 rows, not 33"):
        c.share(1, 0, 33)
    c.reserve(0, 64)
    with pytest.raises(RuntimeError, match="no page is free"):
        c.share(1, 2, 17)
    assert bool((c.table[2] == -1).all())
    c.release(1)
    c.release(0)
    assert c.free_pages() == 6
    for b in (-1, 3):
        for what in (lambda: c.reserve(b, 1), lambda: c.release(b), lambda: c.share(b, 0, 0), lambda: c.share(0, b, 0)):
            with pytest.raises(ValueError, match="outside"):
                what()
    for n in (-1, 101):
        with pytest.raises(ValueError, match="maxT"):
            c.reserve(0, n)


# ------------------------------------------------------------- sizes, places, strides


@pytest.mark.parametrize("dt,cached", TYPES)
@pytest.mark.parametrize("page", [128, 256, 512, 1024])
def test_large_pages(page, dt, cached):
    run(8, 2, [1, 1, 1], [2, 1023, 2999], dt, cached, page, one=True)
    run(8, 2, [40, 0, 200], [1000, 5, 900], dt, cached, page, maxT=5000)
    run(16, 1, [70], [2030], dt, cached, page, maxT=2 ** 19)


@pytest.mark.parametrize("dt,cached", TYPES)
def test_a_pool_past_4_gib(dt, cached):
    """Pages whose byte offsets pass 32 bits, and sequences of pages from both ends."""
    KH, page = 8, 64
    size = 2 * KH * page * HD * (4 if cached == "f32" else 2)
    n_pages = 2 ** 32 // size + 200
    data = torch.zeros(1, n_pages, 2, KH, page, HD, dtype=DT[cached], device="cuda")
    for counts, start in (([1, 1], [900, 63]), ([130, 90], [700, 20])):
        c = PagedKVCacheSet(shape_of(KH, 4 * KH, 1000), 2, n_pages, page=page, data=data)
        order = torch.cat([torch.arange(8, device="cuda"), torch.arange(n_pages - 24, n_pages, device="cuda")])
        c.table.copy_(order[torch.randperm(32, generator=torch.Generator().manual_seed(1)).cuda()].view(2, 16).int())
        rng = np.random.default_rng(5)
        k, v, q = [], [], []
        for b, (s, n) in enumerate(zip(start, counts)):
            x, y = rows(b + 3, s + n, KH)
            put(c, b, x[:s], y[:s])
            k.append(torch.from_numpy(x[s:])), v.append(torch.from_numpy(y[s:]))
            q.append(queries(b, x, s, n, 4 * KH))
        cu = ints([0, counts[0], sum(counts)])
        c.append(0, torch.cat(k).cuda(), torch.cat(v).cuda(), ints(start), cu)
        check(c, np.concatenate(q), start, counts, dt)
        for b, (s, n) in enumerate(zip(start, counts)):
            gk, gv = held(c, b, s + n)
            assert np.array_equal(gk[s:], k[b].to(DT[cached]).float().numpy()) and np.array_equal(gv[s:], v[b].to(DT[cached]).float().numpy())
        # the pages of nobody are as they were
        assert not bool(data[0, 8:n_pages - 24:997].any())
    del data


@pytest.mark.parametrize("dt,cached", TYPES)
@pytest.mark.parametrize("counts,start", [([1, 1], [700, 30]), ([5, 3], [700, 30]), ([200, 60], [100, 30])])
@pytest.mark.parametrize("maxT", [1000, 2 ** 19])
def test_strided_queries_and_out_in_place(counts, start, maxT, dt, cached):
    H, KH = 8, 2
    c, q = prepared(H, KH, counts, start, cached, maxT)
    cu = ints(np.concatenate([[0], np.cumsum(counts)]).tolist())
    qd = torch.from_numpy(q).cuda().to(DT[dt])
    want = c.attention(0, qd, ints(start), cu).clone()
    wide = torch.full((len(q), H + 3, HD + 4), float("nan"), dtype=DT[dt], device="cuda")
    wide[:, 1:H + 1, :HD] = qd
    assert torch.equal(c.attention(0, wide[:, 1:H + 1, :HD], ints(start), cu), want)
    t = torch.full((H, len(q), HD), 0.0, dtype=DT[dt], device="cuda")
    t.copy_(qd.transpose(0, 1))
    assert torch.equal(c.attention(0, t.transpose(0, 1), ints(start), cu), want)
    assert c.attention(0, qd, ints(start), cu, out=qd).data_ptr() == qd.data_ptr()
    assert torch.equal(qd, want)


@pytest.mark.parametrize("dt", ["f32", "bf16"])
def test_no_tokens_and_no_sequences(dt):
    for B in (0, 2):
        c = PagedKVCacheSet(shape_of(2, 4, 64), B, 3)
        e = [torch.empty(0, h, HD, dtype=DT[dt], device="cuda") for h in (4, 2, 2)]
        start, cu = ints([0] * B), ints([0] * (B + 1))
        assert c.append(0, e[1], e[2], start, cu, q=e[0]).shape == (0, 4, HD)
        assert c.append(0, e[1], e[2], start, cu) is None
        assert c.attention(0, e[0], start, cu).shape == (0, 4, HD)
    c = PagedKVCacheSet(shape_of(2, 4, 64), 0, 3)
    k = torch.ones(3, 2, HD, dtype=DT[dt], device="cuda")
    out = torch.full((3, 4, HD), 7.0, dtype=DT[dt], device="cuda")
    # tokens behind the last of no sequences
    c.append(0, k, k, ints([]), ints([0]))
    c.attention(0, torch.ones_like(out), ints([]), ints([0]), out=out)
    assert not bool(c.data.any()) and bool((out == 7.0).all())


@pytest.mark.parametrize("dt,cached", TYPES)
@pytest.mark.parametrize("many", [False, True])
def test_append_without_pages_and_behind_the_last_sequence(many, dt, cached):
    """Rows without a page are not written, their q is finished all the same; tokens from
    cu[B] on are left out, in q_out too."""
    H, KH, counts, start = 8, 2, [700, 900] if many else [20, 40], [5, 100]
    T = 1200
    c = cache(2, T, KH, 16, cached)
    c.table[0, 1], c.table[1, 7], c.table[1, 8] = -1, c.n_pages, 2 ** 31 - 1
    N = sum(counts) + 3
    g = torch.Generator(device="cuda").manual_seed(4)
    q, k, v = (torch.randn(N, h, HD, generator=g, device="cuda").to(DT[dt]) for h in (H, KH, KH))
    cos, sin = (torch.from_numpy(t).cuda() for t in rope_tables(T, HD, 1e4))
    out = torch.full_like(q, 7.0)
    before = c.data.clone()
    cu = [0, counts[0], sum(counts)]
    got = c.append(0, k, v, ints(start), ints(cu), q=q, cos=cos, sin=sin, q_out=out)
    torch.cuda.synchronize()
    assert got.data_ptr() == out.data_ptr() and bool((out[sum(counts):] == 7.0).all())
    row = np.concatenate([np.arange(s, s + n) for s, n in zip(start, counts)])
    want = finish(q[:cu[-1]].float().cpu().numpy(), row, None, cos.cpu().numpy(), sin.cpu().numpy(), 0.0)
    off = np.abs(out[:cu[-1]].double().cpu().numpy() - want)
    room = 12 * 2.0 ** -24 * (np.abs(want) + np.abs(np.roll(want, HD // 2, axis=-1)) + 1e-30)
    assert (off <= room + HALF[dt] * np.abs(want)).all()
    for b in range(2):
        _, gv = held(c, b, start[b] + counts[b])
        w = v[cu[b]:cu[b + 1]].to(DT[cached]).float().cpu().numpy()
        paged = np.isfinite(gv[start[b]:, 0, 0])
        gone = {0: [1], 1: [7, 8]}[b]
        assert np.array_equal(~paged, np.isin(np.arange(start[b], start[b] + counts[b]) // 16, gone))
        assert np.array_equal(gv[start[b]:][paged], w[paged])
    # nothing but the rows of the call was touched: put those back and compare
    table = c.table.cpu().numpy()
    for b in range(2):
        r = np.arange(start[b], start[b] + counts[b])
        r = r[~np.isin(r // 16, {0: [1], 1: [7, 8]}[b])]
        p, at = torch.from_numpy(table[b, r // 16].astype(np.int64)).cuda(), torch.from_numpy(r % 16).cuda()
        for i in range(2):
            c.data[0, p, i, :, at] = before[0, p, i, :, at]
    assert torch.equal(before.view(torch.uint8), c.data.view(torch.uint8))


@pytest.mark.parametrize("dt,cached", TYPES)
def test_more_sequences_than_a_wave_has_lanes(dt, cached):
    """130 sequences, some of them empty: a token each, drafts, ragged prompts."""
    B = 130
    rng = np.random.default_rng(8)
    start = rng.integers(0, 60, B).tolist()
    for counts in ([1] * B, rng.integers(0, 5, B).tolist(), rng.integers(0, 90, B).tolist()):
        counts[0], counts[64], counts[65], counts[-1] = 1, 1, 1, max(counts[-1], 1)
        for maxT in (300, 2 ** 19):
            run(8, 2, counts, start, dt, cached, maxT=maxT, one=max(counts) == 1)


@pytest.mark.parametrize("dt,cached", TYPES)
@pytest.mark.parametrize("maxT", [1500, 2 ** 19])
def test_tokens_in_front_of_the_first_sequence(maxT, dt, cached):
    """cu[0] above 0: tokens of nobody, left as they were; and a call of fewer sequences'
    tokens than there are rows for."""
    H, KH, counts, start = 8, 2, [40, 0, 200], [30, 9, 700]
    c, q = prepared(H, KH, counts, start, cached, maxT)
    cu = np.concatenate([[0], np.cumsum(counts)])
    qd = torch.from_numpy(q).cuda().to(DT[dt])
    pad = torch.full((7, H, HD), float("nan"), dtype=DT[dt], device="cuda")
    # (a call of as many tokens, which is cut alike)
    want = c.attention(0, torch.cat([qd, pad, pad]), ints(start), ints(cu.tolist()))[:-14]
    out = torch.full((len(q) + 14, H, HD), 7.0, dtype=DT[dt], device="cuda")
    got = c.attention(0, torch.cat([pad, qd, pad]), ints(start), ints((cu + 7).tolist()), out=out)
    assert bool((got[:7] == 7.0).all()) and bool((got[-7:] == 7.0).all()) and torch.equal(got[7:-7], want)
    k = torch.full((len(q) + 14, KH, HD), 3.0, dtype=DT[dt], device="cuda")
    before = c.data.clone()
    out.fill_(7.0)
    c.append(0, k, k, ints(start), ints((cu + 7).tolist()), q=torch.ones_like(out), q_out=out)
    assert bool((out[:7] == 7.0).all()) and bool((out[-7:] == 7.0).all()) and bool((out[7:-7] == 1.0).all())
    for b, (s, n) in enumerate(zip(start, counts)):
        gk, gv = held(c, b, s + n)
        assert (gk[s:] == 3.0).all() and (gv[s:] == 3.0).all()
    bits = torch.int32 if cached == "f32" else torch.int16              # (the pages hold NaN elsewhere)
    assert int((c.data.view(bits) != before.view(bits)).sum()) <= 2 * 240 * KH * HD


def test_tensors_past_32_bits():
    """q, k, v and the outputs of more than 2^32 bytes and 2^31 values, in sequences of 150
    tokens that share one page table's pages: the last of them against float64."""
    H, KH, n, B = 32, 2, 150, 3600
    T, page = 200, 64
    g = torch.Generator(device="cuda").manual_seed(3)
    c = PagedKVCacheSet(shape_of(KH, H, T), B, 4 * B, page=page)
    c.table.copy_(torch.arange(4 * B, device="cuda").int().view(B, 4))
    N = n * B
    assert N * H * HD > 2 ** 31
    q = torch.randn(N, H, HD, generator=g, device="cuda", dtype=torch.bfloat16)
    kv = torch.randn(2, N, KH, HD, generator=g, device="cuda", dtype=torch.bfloat16)
    start, cu = ints([b % 50 for b in range(B)]), ints([n * b for b in range(B + 1)])
    c.data.fill_(0.5)
    got = c.append(0, kv[0], kv[1], start, cu, q=q)
    assert torch.equal(got[-1000:], q[-1000:]) and torch.equal(got[:1000], q[:1000])
    out = c.attention(0, q, start, cu, out=got)
    for b in (0, B // 2, B - 1):
        s = b % 50
        gk, gv = held(c, b, s + n)
        assert np.array_equal(gv[s:], kv[1, n * b:n * (b + 1)].float().cpu().numpy())
        t = np.arange(s + n)
        pick = np.array([0, 1, 77, n - 1])
        for h in (0, 13, H - 1):
            i = h * KH // H
            want, tol = attend(q[n * b + pick, h].float().cpu().numpy(), gk[:, i], gv[:, i], t <= s + pick[:, None], HD ** -0.5, "bf16 prompt")
            assert (np.abs(out[n * b + pick, h].double().cpu().numpy() - want) <= tol).all()


# -------------------------------------------------- streams, graphs, threads, devices


def test_another_stream():
    c, q = prepared(8, 2, [60, 200], [1000, 700], "bf16", 1500)
    qd, start, cu = torch.from_numpy(q).cuda(), ints([1000, 700]), ints([0, 60, 260])
    k = torch.randn(260, 2, HD, device="cuda")
    c.append(0, k, k, start, cu)
    want = c.attention(0, qd, start, cu)
    put_back = c.data.clone()
    torch.cuda.synchronize()
    st = torch.cuda.Stream()
    for _ in range(3):
        c.data.fill_(float("nan"))
        st.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(st):
            c.data.copy_(put_back)
            c.append(0, k, k, start, cu)                # the current stream
            got = c.attention(0, qd, start, cu)
        st.synchronize()
        assert torch.equal(got, want)
        c.append(0, k, k, start, cu, stream=st)         # a stream by name
        got = c.attention(0, qd, start, cu, stream=st)
        st.synchronize()
        assert torch.equal(got, want)


@pytest.mark.parametrize("dt,cached", TYPES)
@pytest.mark.parametrize("counts,start", [([1, 1, 1], [700, 30, 2000]), ([60, 200, 3], [1000, 700, 0])])
def test_graphs_replayed(counts, start, dt, cached):
    """A step captured: append and attention in ranges, replayed with new tokens, other
    places and other pages, eager work and an attention of other sizes between; two graphs
    that are both alive."""
    H, KH, T = 16, 2, 4000
    c = cache(3, T, KH, 32, cached)
    c.data.normal_(generator=torch.Generator(device="cuda").manual_seed(1))
    N = sum(counts)
    g = torch.Generator(device="cuda").manual_seed(2)
    at, cu = ints(start), ints(np.concatenate([[0], np.cumsum(counts)]).tolist())
    bufs = [[torch.empty(N, h, HD, dtype=DT[dt], device="cuda") for h in (H, KH, KH)] for _ in range(2)]
    outs = [torch.empty(N, H, HD, dtype=DT[dt], device="cuda") for _ in range(2)]
    fill = lambda b: [x.normal_(generator=g) for x in b]
    step = lambda b, o: c.attention(0, c.append(0, b[1], b[2], at, cu, q=b[0]), at, cu, out=o, max_rows=T)
    for b, o in zip(bufs, outs):
        fill(b)
        step(b, o)
    torch.cuda.synchronize()
    graphs = []
    for b, o in zip(bufs, outs):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            step(b, o)
        graphs.append(gr)
    for i in range(6):
        for b in bufs:
            fill(b)
        at.copy_(ints([(s + 17 * i) % (T - 300) for s in start]))
        c.table.copy_(c.table.flatten()[torch.randperm(c.table.numel(), generator=torch.Generator().manual_seed(i)).cuda()].view_as(c.table))
        held_before = c.data.clone()
        got = []
        for gr, o in zip(graphs, outs):
            o.fill_(float("nan"))
            gr.replay()
            got.append(o.clone())
        after = c.data.clone()
        c.data.copy_(held_before)
        other = c.attention(0, torch.randn(3, H, HD, generator=g, device="cuda"), at)        # takes the workspace again
        for b, o, x in zip(bufs, outs, got):
            o.fill_(float("nan"))
            step(b, o)
            torch.cuda.synchronize()
            assert torch.equal(o, x), i
        assert torch.equal(after.view(torch.uint8), c.data.view(torch.uint8))
        assert bool(other.isfinite().all())


def test_graphs_on_two_streams_at_once():
    """Two captured calls with ranges do not share what their kernels hand on."""
    c, _ = prepared(16, 2, [1], [3999], "bf16", 4000)
    c.data.nan_to_num_(0.0)
    g = torch.Generator(device="cuda").manual_seed(2)
    qs = [torch.randn(1, 16, HD, generator=g, device="cuda") for _ in range(2)]
    start = ints([3999])
    want = [c.attention(0, q, start).clone() for q in qs]
    assert not torch.equal(*want)
    graphs, outs = [], []
    for q in qs:
        gr = torch.cuda.CUDAGraph()
        outs.append(torch.empty_like(q))
        with torch.cuda.graph(gr):
            for _ in range(20):
                c.attention(0, q, start, out=outs[-1])
        graphs.append(gr)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(5):
        for gr, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                gr.replay()
        torch.cuda.synchronize()
        for o, w in zip(outs, want):
            assert torch.equal(o, w)


def test_host_threads_on_one_stream():
    c, _ = prepared(8, 2, [1, 1], [2999, 1500], "bf16", 3000)
    c.data.nan_to_num_(0.0)
    g = torch.Generator(device="cuda").manual_seed(2)
    start = ints([2999, 1500])
    qs = [torch.randn(2, 8, HD, generator=g, device="cuda") for _ in range(2)]
    want = [c.attention(0, q, start) for q in qs]
    torch.cuda.synchronize()
    out = [[] for _ in qs]
    go = threading.Barrier(len(qs))

    def work(i):
        go.wait()
        for _ in range(50):
            out[i].append(c.attention(0, qs[i], start))

    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(qs))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert all(torch.equal(o, w) for got, w in zip(out, want) for o in got)


# ---------------------------------------------------------------- refused calls


def test_python_refusals():
    c = PagedKVCacheSet(shape_of(2, 8, 100), 2, 9, page=32)
    q, k = torch.zeros(2, 8, HD, device="cuda"), torch.zeros(2, 2, HD, device="cuda")
    at, cos = ints([0, 0]), torch.zeros(100, HD, device="cuda")
    w = torch.ones(HD, dtype=torch.bfloat16, device="cuda")
    ok = dict(q=q, cos=cos, sin=cos, q_norm=w, k_norm=w)
    c.append(0, k, k, at, **ok)
    c.attention(0, q, at)
    bad = torch.zeros(2, 2, HD + 1, device="cuda")
    for a in ((-1, k, k, at), (1, k, k, at), (0, k.cpu(), k, at), (0, k, k.bfloat16(), at), (0, k.half(), k.half(), at),
              (0, k[:, :1], k, at), (0, k, k, at.long()), (0, k, k, at[:1]), (0, k[:1], k[:1], at), (0, k, k, at, at),
              (0, k, k, at.cpu()), (0, bad[:, :, 1:], k, at), (0, bad[:, :, :HD], k, at), (0, [1.0], k, at), (0, k, None, at),
              (0, k.transpose(0, 1).contiguous().transpose(1, 2), k, at)):
        with pytest.raises(ValueError):
            c.append(*a)
    for kw in (dict(cos=cos), dict(sin=cos), dict(ok, cos=cos[:99]), dict(ok, cos=cos.bfloat16()), dict(ok, sin=cos.cpu()),
               dict(ok, cos=cos[:, :64]), dict(ok, q_norm=w.float()), dict(ok, k_norm=w[:64]), dict(ok, k_norm=w[None]),
               dict(ok, q=q.bfloat16()), dict(ok, q=q[:1]), dict(ok, q_out=q[:1]), dict(ok, q_out=q.bfloat16()), dict(q_norm=w), dict(q_out=q),
               dict(ok, q_out=torch.zeros(2, 8, 2 * HD, device="cuda")[:, :, :HD]), dict(ok, q=torch.zeros(2, 16, 64, device="cuda"))):
        with pytest.raises(ValueError):
            c.append(0, k, k, at, **kw)
    with pytest.raises(_lib.JouleError, match="eps"):
        c.append(0, k, k, at, **ok, eps=-1.0)
    with pytest.raises(_lib.JouleError, match="16 times n_kv"):
        c.append(0, k, k, at, q=torch.zeros(2, 33, HD, device="cuda"))
    for a, kw in (((2, q, at), {}), ((0, q.cpu(), at), {}), ((0, q[:1], at), {}), ((0, q.half(), at), {}), ((0, q, at, at), {}),
                  ((0, q, at), dict(max_rows=-1)), ((0, q, at), dict(out=q[:1])), ((0, q, at), dict(out=q.bfloat16())),
                  ((0, q, at.float()), {}), ((0, None, at), {}), ((0, q, None), {})):
        with pytest.raises(ValueError):
            c.attention(*a, **kw)
    for H in (7, 34):
        with pytest.raises(_lib.JouleError, match="whole number"):
            c.attention(0, torch.zeros(2, H, HD, device="cuda"), at)
    for scale in (float("nan"), float("inf"), 3e38):
        with pytest.raises(_lib.JouleError, match="scale"):
            c.attention(0, q, at, scale=scale)
    shape = shape_of(2, 8, 100)
    for kw in (dict(page=8), dict(page=24), dict(page=2048), dict(n_pages=0), dict(B=-1), dict(dtype=torch.float16),
               dict(data=c.data[:, :3]), dict(data=c.data.cpu()), dict(data=c.data.half()), dict(data=c.data.transpose(3, 4))):
        a = dict(shape=shape, B=2, n_pages=9, page=32)
        a.update(kw)
        with pytest.raises(ValueError):
            PagedKVCacheSet(**a)
