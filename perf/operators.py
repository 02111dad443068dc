"""Operators of a serving loop around the decoder, measured one by one: the 4-bit
KV cache (rows quantised as they are written, and read back), attention over
it, and the sampling of the next token.

A case is a dict of plain values.  ``kind`` is the operator:

* ``kv``      rows of k and v of some sequences go into their 4-bit caches and
              come back as the values that the cache holds for them
              (``write``), or rows that are there come back;
* ``attn``    query tokens of some sequences over their 4-bit caches: one
              token each (a decode step), several (a draft being checked), or
              a chunk of a prompt; a token sees the rows up to its own;
* ``sample``  the next token of each row of logits under temperature, top-k,
              top-p and min-p, from one random number a row.

A 4-bit row is the framework's Q4 format along the head: groups of 64 or 32
values, each with a scale fp16(fp32(absmax / 7)), the values
clip(round(v / scale), -8, 7) * scale.

Sampling is defined on whole numbers, so that no order of summation changes a
token: w = round(2^40 exp((l - max l) / temperature)), the tokens in the order
of their logits (ties: the lower index first).  top-k keeps the first k; top-p
those before whose weights less than top_p of what top-k kept lies; min-p those
of a weight of at least min_p 2^40.  The token drawn is the first whose running
sum passes floor(u * sum of the kept weights); its probability is its weight
over that sum.  A temperature of 0 takes the first token.

``own`` set, ``run`` makes the framework's calls; else it computes the same in
elementary torch operations.
"""

from __future__ import annotations

import math

import numpy as np
import torch

own = False

HD = 128                        # head dimension
ONE = float(2 ** 40)            # the weight of the largest logit
DT = {"f32": torch.float32, "bf16": torch.bfloat16}


def listed() -> list[dict]:
    return [
        # one step of the benchmark's decode batch: a row a sequence, where
        # launches count
        {"name": "kv_step_b8", "kind": "kv", "write": True, "seqs": 8, "rows": 1, "context": 2048, "kv": 4,
         "group": 64, "dtype": "f32"},
        # prompts of three users entering the cache together, the smaller group
        {"name": "kv_prompts_b3", "kind": "kv", "write": True, "seqs": 3, "rows": 1531, "context": 130, "kv": 8,
         "group": 32, "dtype": "bf16"},
        # whole conversations read back, to move them to a wider cache
        {"name": "kv_restore_b16", "kind": "kv", "write": False, "seqs": 16, "rows": 7001, "context": 0, "kv": 8,
         "group": 64, "dtype": "bf16"},
        # one user's chat, where round trips count
        {"name": "attn_b1_c777", "kind": "attn", "seqs": 1, "new": 1, "context": 777, "heads": 32, "kv": 4,
         "group": 64, "dtype": "f32"},
        # the benchmark's decode batch and context
        {"name": "attn_b8_c2048", "kind": "attn", "seqs": 8, "new": 1, "context": 2048, "heads": 32, "kv": 4,
         "group": 64, "dtype": "f32"},
        # a busy server with long conversations of very different lengths
        {"name": "attn_b32_c16k", "kind": "attn", "seqs": 32, "new": 1, "context": 16003, "heads": 32, "kv": 8,
         "group": 32, "dtype": "bf16"},
        # drafts of up to 5 tokens being checked, a head of its own per KV head
        {"name": "attn_draft_b6", "kind": "attn", "seqs": 6, "new": 5, "context": 3001, "heads": 16, "kv": 16,
         "group": 64, "dtype": "f32"},
        # a prompt's first chunk
        {"name": "attn_prompt_t509", "kind": "attn", "seqs": 1, "new": 509, "context": 0, "heads": 32, "kv": 4,
         "group": 64, "dtype": "f32"},
        # a later chunk of a long prompt
        {"name": "attn_chunk_t2047", "kind": "attn", "seqs": 1, "new": 2047, "context": 4099, "heads": 32, "kv": 8,
         "group": 64, "dtype": "bf16"},
        # one user's next token with the settings chats use
        {"name": "sample_b1", "kind": "sample", "rows": 1, "vocab": 151936, "dtype": "f32", "set": "chat"},
        # a few rows of a smaller vocabulary over the whole distribution
        {"name": "sample_b7_full", "kind": "sample", "rows": 7, "vocab": 50304, "dtype": "f32", "set": "full"},
        # a busy server, every request with settings of its own
        {"name": "sample_b128_mixed", "kind": "sample", "rows": 128, "vocab": 151936, "dtype": "f32", "set": "mixed"},
    ]


def _log_int(rng, lo: int, hi: int) -> int:
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng) -> dict:
    kind = rng.choice(["kv", "kv", "attn", "attn", "attn", "sample", "sample"])
    if kind == "sample":
        vocab = _log_int(rng, 1000, 151936)
        return {"kind": "sample", "rows": _log_int(rng, 1, 128), "vocab": vocab, "dtype": rng.choice(["f32", "f32", "bf16"]),
                "set": rng.choice(["chat", "full", "nucleus", "mixed"])}
    c = {"kind": kind, "kv": rng.choice([2, 4, 8, 16]), "group": rng.choice([64, 64, 32]),
         "dtype": rng.choice(["f32", "bf16"])}
    if kind == "kv":
        rows = _log_int(rng, 1, 7000)
        c.update(write=rng.random() < 0.7, rows=rows, context=_log_int(rng, 1, 4000) - 1,
                 seqs=_log_int(rng, 1, max(1, min(64, 120_000 // (rows * c["kv"] // 8 + 1)))))
        return c
    c["heads"] = c["kv"] * rng.choice([1, 2, 4, 8] if c["kv"] < 16 else [1, 2])
    new = rng.choice([1, 1, 2, 0])
    if new == 1:                # a decode step
        ctx = _log_int(rng, 1, 16000)
        c.update(new=1, context=ctx, seqs=_log_int(rng, 1, max(1, min(64, 4_000_000 // (ctx * c["kv"])))))
    elif new == 2:              # a draft
        ctx = _log_int(rng, 1, 16000)
        c.update(new=rng.randint(2, 9), context=ctx, seqs=_log_int(rng, 1, max(1, min(32, 2_000_000 // (ctx * c["kv"])))))
    else:                       # prompts
        new = _log_int(rng, 10, 2000)
        c.update(new=new, context=_log_int(rng, 1, 4000) - 1, seqs=rng.randint(1, max(1, min(6, 2000 // new))))
    return c


# ------------------------------------------------------------------- inputs


def _gen(seed: int) -> torch.Generator:
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _randn(gen, *shape) -> torch.Tensor:
    return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32)


def _counts(case):
    """(start, n) of the sequences: where their rows or tokens begin, and how
    many there are.  The first has the most of both; one of the others has
    none."""
    S, n, c = case["seqs"], case.get("rows", case.get("new")), case["context"]
    rng = np.random.default_rng([S, n, c])
    start = c - rng.integers(0, c // 2 + 1, S)
    count = n - rng.integers(0, n, S) if n > 1 else np.ones(S, np.int64)
    if n > 1 and S > 3:
        count[rng.integers(1, S)] = 0
    start[0], count[0] = c, n
    return start.astype(np.int32), count.astype(np.int32)


def _rows(gen, n: int, kv: int):
    """k and v of n rows [n, kv, HD]: N(0, 1), a few of k's channels large, as
    keys have them."""
    k, v = _randn(gen, n, kv, HD), _randn(gen, n, kv, HD)
    k[:, :, 5::29] *= 5.0
    return k, v


class _PlainCache:
    """The caches of S sequences as two tensors each for k and v: nibbles
    [S, T, kv, HD / 2], the even value low, and fp16 scales [S, T, kv, HD / group]."""

    def __init__(self, S: int, T: int, kv: int, group: int):
        self.group = group
        self.q = [torch.zeros((S, T, kv, HD // 2), dtype=torch.uint8, device="cuda") for _ in range(2)]
        self.s = [torch.zeros((S, T, kv, HD // group), dtype=torch.float16, device="cuda") for _ in range(2)]

    def write(self, seq, pos, k, v):
        for i, x in enumerate((k, v)):
            x = x.float().unflatten(-1, (HD // self.group, self.group))
            top = x.abs().amax(dim=-1).clamp(min=1e-12)
            s = (top / torch.full_like(top, 7.0)).to(torch.float16)
            q = torch.nan_to_num((x / s.float().unsqueeze(-1)).round().clamp(-8, 7), nan=0.0)
            q = (q + 8).to(torch.uint8).flatten(-2)
            self.q[i][seq, pos] = q[..., 0::2] | (q[..., 1::2] << 4)
            self.s[i][seq, pos] = s

    def values(self, i: int, at) -> torch.Tensor:
        """The values of k (i = 0) or v at an index of (sequence, row)."""
        p, s = self.q[i][at], self.s[i][at]
        q = torch.stack([p & 15, p >> 4], dim=-1).flatten(-2).float() - 8.0
        return (q.unflatten(-1, (HD // self.group, self.group)) * s.float().unsqueeze(-1)).flatten(-2)


def _cache(S: int, T: int, kv: int, heads: int, group: int):
    """An empty cache: the framework's handle, or the plain one."""
    if not own:
        return _PlainCache(S, T, kv, group)
    from joule_amd.decoder import DecoderShape
    from joule_amd.dense import dense_ffn_shape
    from joule_amd.kv_q4 import Q4KVCacheSet

    shape = DecoderShape(n_layers=1, moe=dense_ffn_shape(1024, 512), n_heads=heads, n_kv=kv, maxT=T)
    return Q4KVCacheSet(shape, S, group=group)


def _fill(cache, seq: int, n: int, k, v):
    """Rows 0 .. n - 1 of one sequence."""
    if not own:
        cache.write(torch.full((n,), seq, device="cuda"), torch.arange(n, device="cuda"), k, v)
        return
    count = torch.zeros(cache.B, dtype=torch.int32, device="cuda")
    count[seq] = n
    cu = torch.cat([torch.zeros_like(count[:1]), count.cumsum(0, dtype=torch.int32)])
    cache.write(0, k, v, torch.zeros_like(count), cu)


def _logits(gen, case):
    """Logits as language has them: the probabilities of a Zipf law over a
    random order of the tokens, noise on top; a fifth of the rows with a mask
    of -inf over half of the vocabulary."""
    B, V = case["rows"], case["vocab"]
    rank = torch.rand((B, V), generator=gen, device="cuda").argsort(dim=1).float()
    l = -1.4 * torch.log(rank + 2.7) + 0.7 * _randn(gen, B, V) + 12.0
    masked = (torch.arange(B, device="cuda") % 5 == 4).unsqueeze(1) & (torch.arange(V, device="cuda") % 2 == 1)
    return l.masked_fill(masked, float("-inf")).to(DT[case["dtype"]])


def _settings(case, seed: int) -> dict:
    B, kind = case["rows"], case["set"]
    if kind == "chat":
        return {"temperature": 0.8, "top_k": 50, "top_p": 0.95, "min_p": 0.0}
    if kind == "full":
        return {"temperature": 1.0, "top_k": 0, "top_p": 1.0, "min_p": 0.0}
    if kind == "nucleus":
        return {"temperature": 1.1, "top_k": 0, "top_p": 0.9, "min_p": 0.02}
    rng = np.random.default_rng(seed + 29)
    pick = lambda v, t: torch.from_numpy(rng.choice(np.asarray(v, t), B)).cuda()  # noqa: E731
    return {"temperature": pick([0.0, 0.3, 0.7, 1.0, 1.5], np.float32), "top_k": pick([0, 0, 1, 20, 50, 1000], np.int32),
            "top_p": pick([1.0, 0.95, 0.8, 0.3], np.float32), "min_p": pick([0.0, 0.0, 0.05, 0.3], np.float32)}


def prepare(case: dict, seed: int) -> dict:
    gen = _gen(seed * 7 + 1)
    s = {"kind": case["kind"]}
    if case["kind"] == "sample":
        s.update(logits=_logits(gen, case), u=torch.rand(case["rows"], generator=gen, device="cuda"),
                 settings=_settings(case, seed))
        return s
    start, count = _counts(case)
    S, kv, dt = case["seqs"], case["kv"], DT[case["dtype"]]
    ends = start + count
    cache = _cache(S, int(ends.max()), kv, case.get("heads", kv), case["group"])
    N = int(count.sum())
    cu = np.concatenate([[0], np.cumsum(count)]).astype(np.int32)
    s.update(cache=cache, N=N, new=int(count.max()), start=torch.from_numpy(start).cuda(), cu=torch.from_numpy(cu).cuda())
    if case["kind"] == "kv" and case["write"]:
        k, v = _rows(gen, N, kv)
        s.update(write=True, k=k.to(dt), v=v.to(dt), dtype=dt)
        return s
    for b in range(S):
        k, v = _rows(gen, int(ends[b]), kv)
        _fill(cache, b, int(ends[b]), k.to(dt), v.to(dt))
    if case["kind"] == "kv":
        s.update(write=False, dtype=dt)
    else:
        s.update(q=_randn(gen, N, case["heads"], HD).to(dt))
    return s


# ---------------------------------------------------------------------- run


def _place(s):
    """The sequence of each token or row, and its number there."""
    t = torch.arange(s["N"], device="cuda")
    seq = torch.searchsorted(s["cu"], t, right=True) - 1
    return seq, t - s["cu"][seq]


def _plain_attention(s):
    q, cache = s["q"], s["cache"]
    N, H, _ = q.shape
    S, T, KH, _ = cache.q[0].shape
    seq, i = _place(s)
    # the tokens of each sequence side by side, padded to the longest
    qp = torch.zeros((S, s["new"], H, HD), device="cuda")
    qp[seq, i] = q.float()
    qp = qp.view(S, s["new"], KH, H // KH, HD).transpose(1, 2).reshape(S * KH, -1, HD)
    k = cache.values(0, slice(None)).transpose(1, 2).reshape(S * KH, T, HD)
    p = torch.matmul(qp * HD ** -0.5, k.transpose(1, 2)).view(S, KH, s["new"], H // KH, T)
    del k
    last = s["start"][:, None] + torch.arange(s["new"], device="cuda")
    p = p.masked_fill(torch.arange(T, device="cuda") > last[:, None, :, None, None], float("-inf"))
    p = torch.exp(p - p.amax(dim=-1, keepdim=True))
    p = p / p.sum(dim=-1, keepdim=True)
    v = cache.values(1, slice(None)).transpose(1, 2).reshape(S * KH, T, HD)
    o = torch.matmul(p.view(S * KH, -1, T), v).view(S, KH, s["new"], H // KH, HD).transpose(1, 2).reshape(S, s["new"], H, HD)
    return o[seq, i].to(q.dtype)


def _plain_sample(logits, u, temperature, top_k, top_p, min_p):
    B, V = logits.shape
    col = lambda x, t: torch.as_tensor(x, device="cuda", dtype=t).expand(B).unsqueeze(1)  # noqa: E731
    T, k = col(temperature, torch.float32).double(), col(top_k, torch.int64)
    p, mp = col(top_p, torch.float32).double(), col(min_p, torch.float32).double()
    k = torch.where(T <= 0, torch.ones_like(k), torch.where(k <= 0, torch.full_like(k, V), k))
    T = torch.where(T <= 0, torch.ones_like(T), T)
    l, order = torch.sort(logits.float(), dim=1, descending=True, stable=True)
    l = l.double()
    w = torch.round(torch.exp((l - l[:, :1]) / T) * ONE).to(torch.int64)
    keep = torch.arange(V, device="cuda") < k
    run = (w * keep).cumsum(dim=1)
    keep = keep & ((run - w).double() < p * run[:, -1:].double()) & (w.double() >= mp * ONE)
    keep[:, 0] = True
    run = (w * keep).cumsum(dim=1)
    total = run[:, -1:]
    at = torch.minimum((u.double().unsqueeze(1) * total.double()).floor().to(torch.int64), total - 1)
    at = (run <= at).sum(dim=1, keepdim=True)
    return order.gather(1, at).squeeze(1).to(torch.int32), (w.gather(1, at).double() / total.double()).squeeze(1).float()


def run(state: dict):
    s = state
    if s["kind"] == "sample":
        if own:
            from joule_amd.sampling import sample

            return sample(s["logits"], s["u"], **s["settings"])
        return _plain_sample(s["logits"], s["u"], **s["settings"])
    cache = s["cache"]
    if s["kind"] == "attn":
        return cache.attention(0, s["q"], s["start"], s["cu"]) if own else _plain_attention(s)
    if own:
        if s["write"]:
            cache.write(0, s["k"], s["v"], s["start"], s["cu"])
        return cache.read(0, s["start"], s["cu"], s["N"], dtype=s["dtype"])
    seq, i = _place(s)
    pos = s["start"][seq] + i
    if s["write"]:
        cache.write(seq, pos, s["k"], s["v"])
    return [cache.values(j, (seq, pos)).to(s["dtype"]) for j in range(2)]


# --------------------------------------------------------------------- work


def work(case: dict) -> dict:
    size = 4 if case["dtype"] == "f32" else 2
    if case["kind"] == "sample":
        n = float(case["rows"]) * case["vocab"]
        return {"bytes": size * n + 24.0 * case["rows"], "flops": 3.0 * n}
    start, count = _counts(case)
    N, kv = float(count.sum()), case["kv"]
    row = 2 * kv * (HD // 2 + 2 * HD // case["group"])      # bytes of a row's k and v in the cache
    if case["kind"] == "kv":
        return {"bytes": N * (row + 2 * kv * HD * size * (2 if case["write"] else 1)), "flops": 4.0 * N * kv * HD}
    pairs = float(sum(int(n) * int(s) + int(n) * (int(n) + 1) // 2 for s, n in zip(start, count)))
    cached = float(sum(int(s) + int(n) for s, n in zip(start, count) if n))
    return {"bytes": cached * row + 2.0 * N * case["heads"] * HD * size, "flops": 4.0 * pairs * case["heads"] * HD}


# ----------------------------------------------------------- float64 results


def _quantised(x, group: int):
    """The values that a 4-bit row holds for x, in 64 bits."""
    g = x.double().unflatten(-1, (HD // group, group))
    top = torch.clamp(g.abs().max(dim=-1, keepdim=True).values, min=1e-12)
    s = (top / 7.0).float().to(torch.float16).double()
    q = torch.round((g / s).float().double())
    return (torch.clamp(q, -8, 7) * s).flatten(-2)


def _exact_sample(case, seed):
    gen = _gen(seed * 7 + 1)
    B, V = case["rows"], case["vocab"]
    logits = _logits(gen, case).double().cpu().numpy()
    u = torch.rand(B, generator=gen, device="cuda").double().cpu().numpy()
    given = {k: np.broadcast_to(v.cpu().numpy() if torch.is_tensor(v) else np.float32(v), (B,)).astype(np.float64)
             for k, v in _settings(case, seed).items()}
    tok, prob = np.zeros(B, np.int32), np.zeros(B)
    for b in range(B):
        T, k, p, mp = (given[n][b] for n in ("temperature", "top_k", "top_p", "min_p"))
        k = 1 if T <= 0 else V if k <= 0 else int(k)
        order = np.argsort(-logits[b], kind="stable")[:k]
        l = logits[b][order]
        w = np.rint(np.exp((l - l[0]) / (T if T > 0 else 1.0)) * ONE)
        before = np.cumsum(w) - w
        n = max(1, int(np.count_nonzero((before < p * w.sum()) & (w >= mp * ONE))))
        w = w[:n]
        at = int(np.searchsorted(np.cumsum(w), math.floor(u[b] * w.sum()), side="right"))
        tok[b], prob[b] = order[min(at, n - 1)], w[min(at, n - 1)] / w.sum()
    return tok, prob


def exact(case: dict, seed: int):
    if case["kind"] == "sample":
        return _exact_sample(case, seed)
    gen = _gen(seed * 7 + 1)
    start, count = _counts(case)
    N, kv, dt, G = int(count.sum()), case["kv"], DT[case["dtype"]], case["group"]
    if case["kind"] == "kv" and case["write"]:
        return [_quantised(x.to(dt), G) for x in _rows(gen, N, kv)]
    seqs = []
    for b in range(case["seqs"]):
        seqs.append([_quantised(x.to(dt), G).to(torch.float32) for x in _rows(gen, int(start[b] + count[b]), kv)])
    if case["kind"] == "kv":
        return [torch.cat([r[j][int(s):int(s + n)] for r, s, n in zip(seqs, start, count)]).double() for j in range(2)]
    H = case["heads"]
    q = _randn(gen, N, H, HD).to(dt).double()
    out, t0 = torch.empty_like(q), 0
    for (k, v), s, n in zip(seqs, start.tolist(), count.tolist()):
        future = torch.arange(s + n, device="cuda") > s + torch.arange(n, device="cuda").unsqueeze(1)
        for h in range(H):
            kh = h * kv // H
            a = q[t0:t0 + n, h] @ k[:, kh].double().T.contiguous() / math.sqrt(HD)
            out[t0:t0 + n, h] = torch.softmax(a.masked_fill(future, float("-inf")), dim=1) @ v[:, kh].double()
        t0 += n
    return out
