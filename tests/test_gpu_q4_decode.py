"""The decoder over 4-bit caches and its sampled tokens: steps and prompts
against the oracle with caches that hold the Q4 format's values, then the whole
loop of a server (prompts, sampled steps, the cache read back)."""

import numpy as np
import pytest
import torch

from joule_amd.checkpoint import HipNativeDecoder
from joule_amd.decoder import DecoderShape, DecoderWeights, HipDecoder, KVCacheSet
from joule_amd.dense import DenseFfnStore, dense_ffn_shape
from joule_amd.kv_q4 import Q4KVCacheSet
from joule_amd.q4_store import dequantize, quantize
from joule_amd.sampling import sample
from joule_amd.synth import activations, decoder_weights
from oracle import decoder as D

pytestmark = pytest.mark.gpu

TOL = 1e-3          # the decoder's bar: max relative error against the oracle, per token
DIM, M = 1024, 512


class _Q4Rows(np.ndarray):
    """A cache whose rows become the format's values as they are assigned."""

    group = 64

    def __setitem__(self, pos, row):
        v = np.asarray(row, np.float32)
        np.ndarray.__setitem__(self, pos, dequantize(*quantize(v, self.group), v.size, self.group).reshape(v.shape))


def _model(H, KH, qk, maxT, layers, group, B, graph=False, V=0):
    shape = DecoderShape(n_layers=layers, moe=dense_ffn_shape(DIM, M), n_heads=H, n_kv=KH, maxT=maxT, qk_norm_type=qk, V=V)
    weights = DecoderWeights(shape, **decoder_weights(shape, norm_jitter=0.1))
    w = {k: v.float().cpu().numpy() for k, v in weights.t.items()}
    oracle = D.OracleDecoder(layers, DIM, H, KH, 128, shape.eps, qk, False, w, None, kv_bf16=False)
    kv = Q4KVCacheSet(shape, B, group=group)
    kv_h = []
    for b in range(B):
        kv_h.append([])
        for l in range(layers):
            pair = []
            for _ in range(2):
                r = np.zeros((maxT, KH, 128), np.float32).view(_Q4Rows)
                r.group = group
                pair.append(r)
            kv_h[b].append(tuple(pair))
    return HipDecoder(DenseFfnStore(DIM, M, layers), weights, graph=graph), oracle, kv, kv_h


def _preload(kv, kv_h, rows, seed=3):
    """Rows 0 .. rows - 1 of every sequence and layer."""
    KH, L = kv.shape.n_kv, kv.shape.n_layers
    rng = np.random.default_rng(seed)
    for b in range(kv.B):
        cu = torch.tensor([0] * (b + 1) + [rows] * (kv.B - b), dtype=torch.int32, device="cuda")
        for l in range(L):
            k, v = (rng.standard_normal((rows, KH, 128)).astype(np.float32) for _ in range(2))
            for dst, src in zip(kv_h[b][l], (k, v)):
                for r in range(rows):
                    dst[r] = src[r]
            kv.write(l, torch.from_numpy(k).cuda(), torch.from_numpy(v).cuda(), torch.zeros(kv.B, dtype=torch.int32, device="cuda"), cu)


def _rel(got, want):
    return (np.abs(got - want).max(axis=1) / np.abs(want).max(axis=1)).max()


def _rows_agree(kv, kv_h, b, l, r0, n):
    """The rows that the step wrote: the oracle's values, but for one step of
    the scale where the two sides' float32 rounding differs at a border (the
    projections differ by about 1e-6 of a value, a step is 1/7 of the largest),
    and for one unit of fp16 in a scale (7 steps of 2^-11)."""
    start = torch.zeros(kv.B, dtype=torch.int32, device="cuda")
    start[b] = r0
    cu = torch.tensor([0] * (b + 1) + [n] * (kv.B - b), dtype=torch.int32, device="cuda")
    for got, want in zip(kv.read(l, start, cu, n), kv_h[b][l]):
        got, want = got.cpu().numpy(), np.asarray(want[r0:r0 + n])
        step = np.abs(want).reshape(n, -1, kv.group).max(axis=2).repeat(kv.group, axis=1).reshape(want.shape) / 7
        assert (np.abs(got - want) <= 1.01 * step).all()
        assert (np.abs(got - want) > 0.01 * step).mean() <= 1e-2


@pytest.mark.parametrize("H,KH,qk,group,graph", [(8, 8, 1, 64, False), (8, 4, 0, 32, True), (8, 2, 2, 64, True), (8, 1, 1, 32, False)])
def test_steps_match_oracle(H, KH, qk, group, graph):
    B, layers = 3, 2
    print(f"[q4 decode] H={H} KH={KH} qk={qk} g{group}", flush=True)
    dec, oracle, kv, kv_h = _model(H, KH, qk, 256, layers, group, B, graph)
    _preload(kv, kv_h, 140)
    for step in range(3):
        pos = [140 + step, 5 + step, 63 + step]
        x = activations(B, DIM, seed=40 + step)
        got = dec.decode_layers_batch(torch.from_numpy(x).cuda(), pos, kv).cpu().numpy()
        want = oracle.decode_layers_batch(x, pos, kv_h)
        assert _rel(got, want) <= TOL
        for b, p in enumerate(pos):
            for l in range(layers):
                _rows_agree(kv, kv_h, b, l, p, 1)
    dec.store.close()


@pytest.mark.parametrize("H,KH,qk,group,T,p0", [(8, 8, 1, 64, 70, 0), (8, 2, 1, 64, 130, 37), (8, 1, 2, 32, 40, 5), (8, 4, 0, 64, 9, 100)])
def test_prompts_match_oracle(H, KH, qk, group, T, p0):
    """The positions of one prompt as one batch over one sequence's caches."""
    print(f"[q4 prompt] H={H} KH={KH} qk={qk} T={T} p0={p0}", flush=True)
    dec, oracle, kv, kv_h = _model(H, KH, qk, 256, 1, group, 2)
    _preload(kv, kv_h, 110)
    x = activations(T, DIM, seed=T)
    got = dec.decode_layers_batch(torch.from_numpy(x).cuda(), list(range(p0, p0 + T)), kv, seqs=[1] * T).cpu().numpy()
    want = np.concatenate([oracle.decode_layers_batch(x[i:i + 1], [p0 + i], [kv_h[1]]) for i in range(T)])
    assert _rel(got, want) <= TOL
    _rows_agree(kv, kv_h, 1, 0, p0, T)
    _rows_agree(kv, kv_h, 0, 0, 0, 110)
    dec.store.close()


@pytest.mark.parametrize("H,KH,group,T", [(8, 1, 64, 24), (8, 4, 32, 90)])
def test_a_prompt_behind_a_long_prefix(H, KH, group, T):
    """Its cache rows are cut into ranges, whose partial outputs the step's
    workspace holds."""
    p0 = 900
    print(f"[q4 prompt] H={H} KH={KH} T={T} p0={p0}", flush=True)
    dec, oracle, kv, kv_h = _model(H, KH, 1, 1100, 1, group, 1)
    _preload(kv, kv_h, p0)
    x = activations(T, DIM, seed=T)
    got = dec.decode_layers_batch(torch.from_numpy(x).cuda(), list(range(p0, p0 + T)), kv, seqs=[0] * T).cpu().numpy()
    want = np.concatenate([oracle.decode_layers_batch(x[i:i + 1], [p0 + i], [kv_h[0]]) for i in range(T)])
    assert _rel(got, want) <= TOL
    _rows_agree(kv, kv_h, 0, 0, p0, T)
    dec.store.close()


def test_caches_of_each_kind_in_turn_over_one_graph():
    """A store's decoder goes from bf16 caches to 4-bit ones and back: the
    recorded step is not replayed over the wrong kind."""
    dec, _, q4, _ = _model(8, 2, 1, 128, 1, 64, 2, graph=True)
    bf = KVCacheSet(dec.shape, 2)
    x = torch.from_numpy(activations(2, DIM, seed=1)).cuda()
    first = {}
    for _ in range(3):
        for name, kv in (("bf16", bf), ("q4", q4)):
            got = dec.decode_layers_batch(x, [0, 0], kv)
            torch.cuda.synchronize()
            first.setdefault(name, got.clone())
            assert torch.equal(got, first[name])
    assert not torch.equal(first["bf16"], first["q4"])
    other = DecoderShape(n_layers=1, moe=dense_ffn_shape(DIM, M), n_heads=8, n_kv=2, maxT=256)
    with pytest.raises(ValueError):
        dec.decode_layers_batch(x, [0, 0], Q4KVCacheSet(other, 2))
    dec.store.close()


@pytest.mark.parametrize("group", [64, 32])
def test_a_servers_loop(group):
    """Prompts of two sequences, then steps whose tokens are drawn and fed
    back: every step's tokens are those drawn from the step's logits, the tokens
    of a second loop over the same numbers are the same, and what the caches
    hold afterwards serves a step from a copy."""
    V, B = 997, 2
    dec, _, kv, _ = _model(8, 2, 1, 128, 2, group, B, graph=True, V=V)
    g = torch.Generator(device="cuda").manual_seed(4)
    dec.weights.t["embed"] = torch.randn(V, DIM, generator=g, device="cuda").to(torch.bfloat16)
    dec._w = dec.weights.kernel_w()
    dec.set_lm_head((torch.randn(V, DIM, generator=g, device="cuda") * 0.1).to(torch.bfloat16))
    prompts = [torch.randint(0, V, (n,), generator=g, device="cuda", dtype=torch.int32) for n in (37, 50)]
    u = torch.rand(12, B, generator=g, device="cuda")
    how = dict(temperature=0.9, top_k=100, top_p=0.95, min_p=0.01)

    def loop():
        for b, t in enumerate(prompts):
            dec.prefill_layers(t, kv, b)
        tok, out = torch.stack([p[-1] for p in prompts]), []
        for i in range(12):
            tok, p = dec.decode_layers_batch_sample(dec.embed(tok), [37 + i, 50 + i], kv, u[i], **how)
            assert bool((tok >= 0).all()) and bool((tok < V).all()) and bool((p > 0).all())
            out.append(tok.clone())
        return torch.stack(out)

    a, b = loop(), loop()
    assert torch.equal(a, b)
    # one step by hand: the logits, then the draw
    x = dec.embed(a[-1].contiguous())
    logits = torch.empty(B, V, device="cuda")
    dec.decode_layers_batch(x, [49, 62], kv, logits=logits)
    tok, p = sample(logits, u[0], **how)
    tok2, p2 = dec.decode_layers_batch_sample(x, [49, 62], kv, u[0], **how)
    assert torch.equal(tok, tok2) and torch.equal(p, p2)
    # greedy sampling is the argmax step
    am = dec.decode_layers_batch_argmax(x, [49, 62], kv)
    assert torch.equal(am, dec.decode_layers_batch_sample(x, [49, 62], kv, u[0], temperature=0.0)[0])
    # the rows move to a wider cache and back, and serve the same step
    moved = Q4KVCacheSet(dec.shape, B, group=group)
    n = torch.tensor([0, 49, 49 + 62], dtype=torch.int32, device="cuda")
    zero = torch.zeros(B, dtype=torch.int32, device="cuda")
    for l in range(2):
        k, v = kv.read(l, zero, n, 111)
        moved.write(l, k, v, zero, n)
        for s, t in zip(moved.read(l, zero, n, 111), (k, v)):
            assert torch.equal(s, t)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    tok3, p3 = dec.decode_layers_batch_sample(x, [49, 62], moved, u[0], stream=side, **how)
    side.synchronize()
    assert torch.equal(tok, tok3) and torch.equal(p, p3)
    dec.store.close()


def test_native_decoder_takes_4_bit_caches(tmp_path):
    """HipNativeDecoder over a small checkpoint with 4-bit caches: prompts,
    greedy and sampled steps."""
    import json

    from safetensors.torch import save_file

    V, L, H, KH = 320, 2, 8, 2
    g = torch.Generator().manual_seed(0)
    rnd = lambda *s: (torch.randn(*s, generator=g) * 0.03).to(torch.bfloat16)  # noqa: E731
    t = {"model.embed_tokens.weight": rnd(V, DIM) * 30, "model.norm.weight": torch.ones(DIM, dtype=torch.bfloat16), "lm_head.weight": rnd(V, DIM)}
    for l in range(L):
        p = f"model.layers.{l}."
        t[p + "input_layernorm.weight"] = torch.ones(DIM, dtype=torch.bfloat16)
        t[p + "post_attention_layernorm.weight"] = torch.ones(DIM, dtype=torch.bfloat16)
        for n, r, c in (("q", H * 128, DIM), ("k", KH * 128, DIM), ("v", KH * 128, DIM), ("o", DIM, H * 128)):
            t[p + f"self_attn.{n}_proj.weight"] = rnd(r, c)
        for n, r, c in (("gate", M, DIM), ("up", M, DIM), ("down", DIM, M)):
            t[p + f"mlp.{n}_proj.weight"] = rnd(r, c)
    save_file(t, str(tmp_path / "model.safetensors"))
    (tmp_path / "config.json").write_text(json.dumps(dict(
        model_type="llama", hidden_size=DIM, intermediate_size=M, num_hidden_layers=L, num_attention_heads=H,
        num_key_value_heads=KH, head_dim=128, rms_norm_eps=1e-6, rope_theta=1e4, vocab_size=V)))
    out = []
    for group in (0, 64, 32):
        nd = HipNativeDecoder(tmp_path, max_tokens=64, max_batch=2, kv_group=group)
        nd.prefill_batch([[1, 2, 3], [4, 5]])
        am = nd.decode_batch_argmax([7, 8], [3, 2])
        assert am == nd.decode_batch_sample([7, 8], [3, 2], [0.9, 0.1], temperature=0.0)
        s = nd.decode_batch_sample(am, [4, 3], [0.3, 0.7], temperature=0.8, top_k=20)
        assert all(0 <= i < V for i in s)
        out.append(nd.kv.data.dtype)
        nd.dec.store.close()
    assert out == [torch.bfloat16, torch.uint8, torch.uint8]
