"""Operators of a serving loop over a paged key-value cache, measured one by one:
rows of new tokens finished (per-head RMSNorm, rotary position) and appended to
their sequences' pages, and attention over the pages.

A case is a dict of plain values.  ``kind`` is the operator:

* ``append``  the tokens' q and k heads are normed and rotated where the case
              says so, q comes out, and k and v go into the cache;
* ``attn``    query tokens of some sequences over their pages: one token each (a
              decode step), several (a draft being checked), or a chunk of a
              prompt; a token sees the rows up to its own.

The cache of a layer is a pool [pages, 2, KV heads, page, 128] (k, then v) and a
table [sequences, pages a sequence]: row r of sequence s is row r % page of page
table[s, r // page].

The rotation is by halves, with tables cos and sin [rows, 128]: dimension d < 64
becomes x[d] cos[d] - x[d + 64] sin[d], dimension d + 64 becomes x[d + 64]
cos[d + 64] + x[d] sin[d + 64].  The norm is x / sqrt(mean(x^2) + eps) times its
weight.

``own`` set, ``run`` makes the framework's calls; else it computes the same in
elementary torch operations.
"""

from __future__ import annotations

import math

import numpy as np
import torch

own = False

HD = 128                        # head dimension
EPS = 1e-6
DT = {"f32": torch.float32, "bf16": torch.bfloat16}


def listed() -> list[dict]:
    return [
        # one step of the benchmark's decode batch: a token a sequence, with the
        # QK-norm of the model it decodes, into bf16 pages
        {"name": "append_step_b8", "kind": "append", "seqs": 8, "new": 1, "context": 2048, "heads": 32, "kv": 4,
         "page": 16, "dtype": "f32", "cache": "bf16", "norm": True, "rope": True},
        # prompts of three users entering the cache together
        {"name": "append_prompts_b3", "kind": "append", "seqs": 3, "new": 1531, "context": 130, "heads": 32, "kv": 8,
         "page": 64, "dtype": "bf16", "cache": "bf16", "norm": False, "rope": True},
        # long prompts of a busy server
        {"name": "append_prompts_b12", "kind": "append", "seqs": 12, "new": 3001, "context": 0, "heads": 32, "kv": 8,
         "page": 32, "dtype": "bf16", "cache": "bf16", "norm": True, "rope": True},
        # one user's chat, where round trips count
        {"name": "attn_b1_c777", "kind": "attn", "seqs": 1, "new": 1, "context": 777, "heads": 32, "kv": 4,
         "page": 16, "dtype": "f32", "cache": "bf16"},
        # the benchmark's decode batch and context over float32 pages, the
        # reference's own type
        {"name": "attn_b8_c2048", "kind": "attn", "seqs": 8, "new": 1, "context": 2048, "heads": 32, "kv": 4,
         "page": 16, "dtype": "f32", "cache": "f32"},
        # one user behind a book
        {"name": "attn_b1_c131k", "kind": "attn", "seqs": 1, "new": 1, "context": 131001, "heads": 32, "kv": 8,
         "page": 64, "dtype": "bf16", "cache": "bf16"},
        # a busy server with long conversations of very different lengths
        {"name": "attn_b32_c16k", "kind": "attn", "seqs": 32, "new": 1, "context": 16003, "heads": 32, "kv": 8,
         "page": 16, "dtype": "bf16", "cache": "bf16"},
        # drafts of up to 5 tokens being checked, a head of its own per KV head
        {"name": "attn_draft_b6", "kind": "attn", "seqs": 6, "new": 5, "context": 3001, "heads": 16, "kv": 16,
         "page": 32, "dtype": "f32", "cache": "bf16"},
        # a prompt's first chunk
        {"name": "attn_prompt_t509", "kind": "attn", "seqs": 1, "new": 509, "context": 0, "heads": 32, "kv": 4,
         "page": 16, "dtype": "f32", "cache": "bf16"},
        # two prompts over float32 pages
        {"name": "attn_prompt_b2_f32", "kind": "attn", "seqs": 2, "new": 1021, "context": 260, "heads": 16, "kv": 16,
         "page": 32, "dtype": "f32", "cache": "f32"},
        # a later chunk of a long prompt
        {"name": "attn_chunk_t2047", "kind": "attn", "seqs": 1, "new": 2047, "context": 4099, "heads": 32, "kv": 8,
         "page": 64, "dtype": "bf16", "cache": "bf16"},
        # prompts of many users at once, 7 query heads a KV head
        {"name": "attn_prompts_b5", "kind": "attn", "seqs": 5, "new": 1201, "context": 400, "heads": 28, "kv": 4,
         "page": 128, "dtype": "bf16", "cache": "bf16"},
    ]


def _log_int(rng, lo: int, hi: int) -> int:
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng) -> dict:
    kv = rng.choice([1, 2, 4, 8, 16])
    ratio = rng.choice([1, 2, 3, 4, 5, 7, 8, 16] if kv <= 4 else [1, 2, 4, 5, 8] if kv == 8 else [1, 2])
    c = {"kind": rng.choice(["append", "attn", "attn"]), "heads": kv * ratio, "kv": kv, "page": rng.choice([16, 32, 64, 128])}
    c["dtype"], c["cache"] = rng.choice([("bf16", "bf16"), ("bf16", "bf16"), ("f32", "bf16"), ("f32", "bf16"), ("f32", "f32"),
                                         ("bf16", "f32")])
    wide = 2 if c["cache"] == "f32" else 1
    if c["kind"] == "append":
        new = rng.choice([1, _log_int(rng, 2, 9), _log_int(rng, 10, 3000)])
        c.update(new=new, context=_log_int(rng, 1, 4000) - 1, norm=rng.random() < 0.5, rope=rng.random() < 0.8,
                 seqs=_log_int(rng, 1, max(1, min(64, 1_200_000 // (new * (c["heads"] + 2 * kv) * wide)))))
        return c
    kind = rng.choice(["step", "step", "draft", "prompt", "prompt"])
    if kind == "step":
        ctx = _log_int(rng, 1, 40000)
        c.update(new=1, context=ctx, seqs=_log_int(rng, 1, max(1, min(64, 4_000_000 // (ctx * kv * wide)))))
    elif kind == "draft":
        ctx = _log_int(rng, 1, 16000)
        c.update(new=rng.randint(2, 9), context=ctx, seqs=_log_int(rng, 1, max(1, min(32, 2_000_000 // (ctx * kv * wide)))))
    else:
        new, ctx = _log_int(rng, 10, 2000), _log_int(rng, 1, 4000) - 1
        pairs = 300_000_000 // (8 if c["cache"] == "f32" else 4 if c["dtype"] == "f32" else 1)
        while new > 10 and new * (ctx + new) * c["heads"] > pairs:
            new = new * 3 // 4
        c.update(new=new, context=ctx, seqs=rng.randint(1, max(1, min(6, pairs // (new * (ctx + new) * c["heads"])))))
    return c


# ------------------------------------------------------------------- inputs


def _gen(seed: int) -> torch.Generator:
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _randn(gen, *shape, dtype=torch.float32) -> torch.Tensor:
    return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32).to(dtype)


def _counts(case):
    """(start, n) of the sequences: where their new tokens begin, and how many
    there are.  The first has the most of both; one of several others has none."""
    S, n, c = case["seqs"], case["new"], case["context"]
    rng = np.random.default_rng([S, n, c])
    start = c - rng.integers(0, c // 2 + 1, S)
    count = n - rng.integers(0, n, S) if n > 1 else np.ones(S, np.int64)
    if n > 1 and S > 3:
        count[rng.integers(1, S)] = 0
    start[0], count[0] = c, n
    return start.astype(np.int32), count.astype(np.int32)


def _table(case, ends, seed: int):
    """(table [sequences, pages a sequence], pages of the pool): every sequence's
    pages lie anywhere in the pool."""
    need = -(-ends.astype(np.int64) // case["page"])
    total = int(need.sum()) + 3
    order = np.random.default_rng(seed + 5).permutation(total).astype(np.int32)
    table = np.full((len(ends), int(need.max())), -1, np.int32)
    at = 0
    for s, n in enumerate(need):
        table[s, :n] = order[at:at + n]
        at += n
    return table, total


def _pool(gen, case, pages: int) -> torch.Tensor:
    """Pages full of rows: N(0, 1), a few of k's channels large, as keys have
    them.  What lies behind a sequence's rows is what was there before."""
    pool = torch.empty((pages, 2, case["kv"], case["page"], HD), dtype=DT[case["cache"]], device="cuda")
    for p in range(0, pages, 4096):
        pool[p:p + 4096] = _randn(gen, *pool[p:p + 4096].shape)
    pool[:, 0, :, :, 5::29] *= 5.0
    return pool


def _rope(rows: int):
    """cos, sin [rows, 128] of the base 1e6, both halves of the head alike."""
    inv = 1.0 / (1e6 ** (np.arange(0, HD, 2) / HD))
    a = np.arange(rows)[:, None] * inv
    a = np.concatenate([a, a], axis=1)
    return [torch.from_numpy(f(a).astype(np.float32)).cuda() for f in (np.cos, np.sin)]


def _heads(gen, case, N: int):
    """What the projections give: q, k and v of the tokens, and the norm weights."""
    dt = DT[case["dtype"]]
    q, k, v = (_randn(gen, N, h, HD, dtype=dt) for h in (case["heads"], case["kv"], case["kv"]))
    k[:, :, 5::29] *= 5.0
    w = [(1.0 + 0.2 * _randn(gen, HD)).to(torch.bfloat16) for _ in range(2)]
    return q, k, v, w


def prepare(case: dict, seed: int) -> dict:
    gen = _gen(seed * 7 + 1)
    start, count = _counts(case)
    ends = start + count
    table, pages = _table(case, ends, seed)
    pool = _pool(gen, case, pages)
    N = int(count.sum())
    cu = np.concatenate([[0], np.cumsum(count)]).astype(np.int32)
    s = {"kind": case["kind"], "N": N, "new": int(count.max()), "page": case["page"], "pool": pool, "rows": int(ends.max()),
         "table": torch.from_numpy(table).cuda(), "start": torch.from_numpy(start).cuda(), "cu": torch.from_numpy(cu).cuda()}
    if case["kind"] == "append":
        q, k, v, w = _heads(gen, case, N)
        cos, sin = _rope(s["rows"]) if case["rope"] else (None, None)
        s.update(q=q, k=k, v=v, w=w if case["norm"] else (None, None), cos=cos, sin=sin)
    else:
        s.update(q=_randn(gen, N, case["heads"], HD, dtype=DT[case["dtype"]]))
    if own:
        from joule_amd.decoder import DecoderShape
        from joule_amd.dense import dense_ffn_shape
        from joule_amd.kv_paged import PagedKVCacheSet

        shape = DecoderShape(n_layers=1, moe=dense_ffn_shape(1024, 512), n_heads=case["heads"], n_kv=case["kv"], maxT=s["rows"])
        s["cache"] = PagedKVCacheSet(shape, case["seqs"], pages, page=case["page"], data=pool.unsqueeze(0))
        s["cache"].table.copy_(s["table"])
    return s


# ---------------------------------------------------------------------- run


def _place(s):
    """The sequence of each token, and its number there."""
    t = torch.arange(s["N"], device="cuda")
    seq = torch.searchsorted(s["cu"], t, right=True) - 1
    return seq, t - s["cu"][seq]


def _finish(x, w, cos, sin):
    """Heads normed (w given) and rotated (cos, sin given), in 32 bits."""
    x = x.float()
    if w is not None:
        x = x / torch.sqrt((x * x).mean(dim=-1, keepdim=True) + EPS) * w.float()
    if cos is not None:
        half = torch.cat([-x[..., HD // 2:], x[..., :HD // 2]], dim=-1)
        x = x * cos.unsqueeze(1) + half * sin.unsqueeze(1)
    return x


def _plain_append(s):
    seq, i = _place(s)
    row = s["start"][seq].long() + i
    at = s["table"][seq, row // s["page"]].long(), row % s["page"]
    cos, sin = (None, None) if s["cos"] is None else (s["cos"][row], s["sin"][row])
    pool = s["pool"]
    q = _finish(s["q"], s["w"][0], cos, sin).to(s["q"].dtype)
    pool[at[0], 0, :, at[1]] = _finish(s["k"], s["w"][1], cos, sin).to(pool.dtype)
    pool[at[0], 1, :, at[1]] = s["v"].to(pool.dtype)
    return q, pool


def _plain_attention(s):
    q, pool, P = s["q"], s["pool"], s["page"]
    N, H, _ = q.shape
    S, KH, T = s["table"].shape[0], pool.shape[2], s["rows"]
    seq, i = _place(s)
    # the tokens of each sequence side by side, padded to the longest
    qp = torch.zeros((S, s["new"], H, HD), device="cuda")
    qp[seq, i] = q.float()
    qp = qp.view(S, s["new"], KH, H // KH, HD).transpose(1, 2).reshape(S * KH, -1, HD)
    pages = s["table"].clamp(min=0).long()

    def rows(which):
        x = pool[pages, which].transpose(1, 2).reshape(S, KH, -1, HD)
        return x[:, :, :T].reshape(S * KH, T, HD).float()

    p = torch.matmul(qp * HD ** -0.5, rows(0).transpose(1, 2)).view(S, KH, s["new"], H // KH, T)
    last = s["start"][:, None] + torch.arange(s["new"], device="cuda")
    p = p.masked_fill(torch.arange(T, device="cuda") > last[:, None, :, None, None], float("-inf"))
    p = torch.exp(p - p.amax(dim=-1, keepdim=True))
    p = p / p.sum(dim=-1, keepdim=True)
    o = torch.matmul(p.view(S * KH, -1, T), rows(1))
    o = o.view(S, KH, s["new"], H // KH, HD).transpose(1, 2).reshape(S, s["new"], H, HD)
    return o[seq, i].to(q.dtype)


def run(state: dict):
    s = state
    if s["kind"] == "append":
        if not own:
            return _plain_append(s)
        q = s["cache"].append(0, s["k"], s["v"], s["start"], s["cu"], q=s["q"], cos=s["cos"], sin=s["sin"], q_norm=s["w"][0],
                              k_norm=s["w"][1], eps=EPS)
        return q, s["pool"]
    if not own:
        return _plain_attention(s)
    return s["cache"].attention(0, s["q"], s["start"], s["cu"], max_rows=s["rows"])


# --------------------------------------------------------------------- work


def work(case: dict) -> dict:
    start, count = _counts(case)
    N, H, kv = float(count.sum()), case["heads"], case["kv"]
    size, cached = (4 if case[k] == "f32" else 2 for k in ("dtype", "cache"))
    if case["kind"] == "append":
        rows = float((start + count).max() - start.min()) if case["rope"] else 0.0
        return {"bytes": N * HD * ((2 * H + 2 * kv) * size + 2 * kv * cached) + 8.0 * rows * HD,
                "flops": N * HD * (H + kv) * (3.0 * case["rope"] + 4.0 * case["norm"])}
    pairs = float(sum(int(n) * int(s) + int(n) * (int(n) + 1) // 2 for s, n in zip(start, count)))
    seen = float(sum(int(s) + int(n) for s, n in zip(start, count) if n))
    return {"bytes": seen * 2 * kv * HD * cached + 2.0 * N * H * HD * size, "flops": 4.0 * pairs * H * HD}


# ----------------------------------------------------------- float64 results


def _turned(x, rows, tables, w):
    """x [N, heads, 128] in 64 bits: normed by w, rotated to its rows."""
    x = x.double()
    if w is not None:
        x = x * torch.rsqrt(x.pow(2).sum(-1, keepdim=True) / HD + EPS) * w.double()
    if tables is None:
        return x
    a, b = x.split(HD // 2, dim=-1)
    c, s = (t[rows].double().unsqueeze(1).split(HD // 2, dim=-1) for t in tables)
    return torch.cat([a * c[0] - b * s[0], b * c[1] + a * s[1]], dim=-1)


def exact(case: dict, seed: int):
    gen = _gen(seed * 7 + 1)
    start, count = _counts(case)
    table, pages = _table(case, start + count, seed)
    pool = _pool(gen, case, pages)
    P, N, H, kv = case["page"], int(count.sum()), case["heads"], case["kv"]
    if case["kind"] == "append":
        q, k, v, w = _heads(gen, case, N)
        row = np.concatenate([np.arange(s, s + n) for s, n in zip(start.tolist(), count.tolist())])
        seq = np.repeat(np.arange(len(count)), count)
        page = torch.from_numpy(table[seq, row // P].astype(np.int64)).cuda()
        line, row = torch.from_numpy(row % P).cuda(), torch.from_numpy(row).cuda()
        tables = _rope(int((start + count).max())) if case["rope"] else None
        w = w if case["norm"] else (None, None)
        pool = pool.double()
        pool[page, 0, :, line] = _turned(k, row, tables, w[1])
        pool[page, 1, :, line] = v.double()
        return _turned(q, row, tables, w[0]), pool
    q = _randn(gen, N, H, HD, dtype=DT[case["dtype"]]).double()
    out, t0 = torch.empty_like(q), 0
    for b, (s, n) in enumerate(zip(start.tolist(), count.tolist())):
        if n == 0:
            continue
        held = pool[torch.from_numpy(table[b, :-(-(s + n) // P)].astype(np.int64)).cuda()]
        future = torch.arange(s + n, device="cuda") > s + torch.arange(n, device="cuda").unsqueeze(1)
        for g in range(kv):
            k, v = (held[:, i, g].reshape(-1, HD)[:s + n].double() for i in range(2))
            for h in range(g * H // kv, (g + 1) * H // kv):
                a = q[t0:t0 + n, h] @ k.T.contiguous() / math.sqrt(HD)
                out[t0:t0 + n, h] = torch.softmax(a.masked_fill(future, float("-inf")), dim=1) @ v
        t0 += n
    return out
