"""Two host threads that share a stream: calls that keep what one kernel hands
to the next in the stream's workspace."""

import threading

import pytest
import torch

from joule_amd.decoder import DecoderShape
from joule_amd.dense import dense_ffn_shape
from joule_amd.kv_q4 import Q4KVCacheSet
from joule_amd.sampling import sample

pytestmark = pytest.mark.gpu

HD = 128


def _in_threads(jobs, rounds):
    """Every job `rounds` times in a thread of its own, all on the current
    stream: the outputs of each."""
    out = [[] for _ in jobs]
    go = threading.Barrier(len(jobs))

    def work(i):
        go.wait()
        for _ in range(rounds):
            out[i].append(jobs[i]())

    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(jobs))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    return out


def test_threads_on_one_stream_get_their_own_answers():
    g = torch.Generator(device="cuda").manual_seed(3)
    rows = [(torch.randn(b, v, generator=g, device="cuda") * 2, torch.rand(b, generator=g, device="cuda"))
            for b, v in ((1, 151936), (3, 50000), (17, 20000))]
    jobs = [lambda x=x, u=u: sample(x, u, 0.9, 0, 0.95) for x, u in rows]
    # attention in ranges, merged by a second kernel
    c = Q4KVCacheSet(DecoderShape(n_layers=1, moe=dense_ffn_shape(1024, 512), n_heads=8, n_kv=2, maxT=3000), 2)
    kv = torch.randn(2, 3000, 2, HD, generator=g, device="cuda")
    c.write(0, kv[0], kv[1], torch.zeros(2, dtype=torch.int32, device="cuda"), torch.tensor([0, 3000, 3000], dtype=torch.int32, device="cuda"))
    start = torch.tensor([2900, 0], dtype=torch.int32, device="cuda")
    for seed in range(2):
        q = torch.randn(2, 8, HD, generator=g, device="cuda")
        jobs.append(lambda q=q: (c.attention(0, q, start),))
    want = [j() for j in jobs]
    torch.cuda.synchronize()
    for got, w in zip(_in_threads(jobs, 40), want):
        for r in got:
            for a, b in zip(r, w):
                assert torch.equal(a, b)
