"""4-bit attention against float64 within a bound that weights each row as the
softmax does (oracle/attention.py; tests/test_attention_bound.py shows on the CPU
that rows left out, an output of 0, a mask off by one row and a scale off by a
tenth are past it at these shapes)."""

import numpy as np
import pytest
import torch

from joule_amd.decoder import DecoderShape
from joule_amd.dense import dense_ffn_shape
from joule_amd.kv_q4 import Q4KVCacheSet
from oracle.attention import attend, bound

pytestmark = pytest.mark.gpu

HD = 128
DT = {"f32": torch.float32, "bf16": torch.bfloat16}


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def cache(B, maxT, KH, H, group=64):
    """A cache whose rows hold NaN scales until they are written."""
    c = Q4KVCacheSet(DecoderShape(n_layers=1, moe=dense_ffn_shape(1024, 512), n_heads=H, n_kv=KH, maxT=maxT), B, group=group)
    c.data.fill_(0xFF)
    return c


def write(c, b, k, v):
    """Rows 0 .. of sequence b."""
    n = len(k)
    if n:
        cu = [0] * (b + 1) + [n] * (c.B - b)
        c.write(0, torch.from_numpy(np.ascontiguousarray(k)).cuda(), torch.from_numpy(np.ascontiguousarray(v)).cuda(), ints([0] * c.B), ints(cu))


def held(c, b, n):
    """The values of rows 0 .. n - 1 of sequence b."""
    cu = [0] * (b + 1) + [n] * (c.B - b)
    return [x.double().cpu().numpy() for x in c.read(0, ints([0] * c.B), ints(cu), n)]


def rows(seed, T, KH):
    rng = np.random.default_rng(seed)
    k, v = (rng.standard_normal((T, KH, HD)).astype(np.float32) for _ in range(2))
    k[:, :, 3::17] *= 2.0
    return k, v


def queries(seed, k, start, n, H):
    """n tokens from row `start` on, each looking at its own row and the next."""
    rng = np.random.default_rng(seed)
    KH = k.shape[1]
    q = rng.standard_normal((n, H, HD)).astype(np.float32)
    for i in range(n):
        for h in range(H):
            q[i, h] += 0.4 * k[start + i:start + i + 2, h * KH // H].sum(axis=0)
    return q


def form_of(dt, n, H, KH, n_seq):
    """As the entry point decides: prompts from 96 query rows a KV head and sequence."""
    return "f32" if dt == "f32" else "bf16 prompt" if n * (H // KH) >= 96 * n_seq else "bf16"


def check(c, q, start, counts, dt, scale=HD ** -0.5, out=None, only=None):
    """attention() of tokens q [N, H, HD] (numpy float32) against float64, at some
    16 tokens of each sequence; returns the output."""
    H, KH = q.shape[1], c.shape.n_kv
    qd = torch.from_numpy(q).cuda().to(DT[dt])
    cu = np.concatenate([[0], np.cumsum(counts)]).tolist()
    print(f"[kv q4 bound] H={H} KH={KH} {counts} at {start} of {c.shape.maxT} g{c.group} {dt} scale {scale}", flush=True)
    got = c.attention(0, qd, ints(start), None if all(n == 1 for n in counts) else ints(cu), scale=scale, out=out)
    torch.cuda.synchronize()
    g64, q64 = got.double().cpu().numpy(), qd.double().cpu().numpy()
    form = form_of(dt, len(q), H, KH, len(counts))
    for b, (s, n) in enumerate(zip(start, counts)):
        if n == 0 or s + n <= 0:
            continue
        k, v = held(c, b, s + n)
        pick = only if only is not None else sorted({0, n - 1, *np.random.default_rng(n).integers(0, n, 14).tolist()})
        for i in pick:
            for h in range(H):
                kk, vv, x = k[:, h * KH // H], v[:, h * KH // H], q64[cu[b] + i, h]
                want, tol = attend(x, kk, vv, s + i + 1, scale), bound(x, kk, vv, s + i + 1, scale, form)
                off = np.abs(g64[cu[b] + i, h] - want)
                assert (off <= tol).all(), f"sequence {b} token {i} head {h}: {np.nanmax(off / tol):.3g} bounds off, by {np.nanmax(off):.3g}"
    return got


def run(H, KH, counts, start, group, dt, maxT=None, scale=HD ** -0.5):
    c = cache(len(counts), maxT or max(s + n for s, n in zip(start, counts)), KH, H, group)
    q = []
    for b, (s, n) in enumerate(zip(start, counts)):
        k, v = rows(7 * b + 1, s + n + 1, KH)
        write(c, b, k[:s + n], v[:s + n])
        q.append(queries(b + 100, k, s, n, H))
    return check(c, np.concatenate(q), start, counts, dt, scale)


@pytest.mark.parametrize("dt,group", [("f32", 64), ("bf16", 64), ("f32", 32), ("bf16", 32)])
@pytest.mark.parametrize("H,KH,counts,start", [(8, 1, [64], [1500]), (2, 2, [129], [2000]), (8, 2, [300], [97]), (8, 8, [130], [700]),
                                               (4, 2, [130, 0, 90], [900, 5, 1800])])
def test_prompts(H, KH, counts, start, dt, group):
    run(H, KH, counts, start, group, dt, maxT=4000)
    run(H, KH, counts, start, group, dt)


@pytest.mark.parametrize("dt,group", [("f32", 64), ("bf16", 64), ("f32", 32), ("bf16", 32)])
@pytest.mark.parametrize("H,KH,counts,start", [(8, 1, [1], [5000]), (16, 4, [1, 1], [300, 900]), (8, 8, [5, 3], [900, 20]), (4, 1, [2, 0, 5], [300, 7, 900])])
def test_few_tokens(H, KH, counts, start, dt, group):
    run(H, KH, counts, start, group, dt, maxT=6000)
    run(H, KH, counts, start, group, dt)


@pytest.mark.parametrize("dt", ["f32", "bf16"])
@pytest.mark.parametrize("counts,start", [([1], [777]), ([3], [777]), ([64], [700]), ([200], [500])])
@pytest.mark.parametrize("maxT", [1024, 1025, 4096, 32768, 131072, 300001])
def test_caches_with_room_for_more_rows(counts, start, dt, maxT):
    """The call is cut by the rows that a cache has room for: ranges without a
    row, and both forms for prompts, over the same rows."""
    run(8, 2, counts, start, 64, dt, maxT=maxT)
