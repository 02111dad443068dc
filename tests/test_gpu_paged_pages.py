"""Pages given out and taken back while a graph is being captured: refused, and the capture
goes on."""

import pytest
import torch

from joule_amd.kv_paged import PagedKVCacheSet
from test_gpu_paged import HD, ints
from test_gpu_paged_use import shape_of

pytestmark = pytest.mark.gpu


def test_page_keeping_inside_a_capture():
    c = PagedKVCacheSet(shape_of(2, 4, 200), 2, 8, page=16)
    c.reserve(0, 40)
    c.data.normal_(generator=torch.Generator(device="cuda").manual_seed(1))
    q, start, cu = torch.randn(1, 4, HD, device="cuda"), ints([39, 0]), ints([0, 1, 1])
    want = c.attention(0, q, start, cu, max_rows=200)
    torch.cuda.synchronize()
    table, out, gr = c.table.clone(), torch.zeros_like(q), torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        for what in (lambda: c.reserve(1, 20), lambda: c.reserve(0, 60), lambda: c.share(0, 1, 39), lambda: c.release(0)):
            with pytest.raises(RuntimeError, match="captur"):
                what()
        c.attention(0, q, start, cu, out=out, max_rows=200)
    assert c.free_pages() == 5 and torch.equal(c.table, table)
    c.share(0, 1, 39)
    for _ in range(3):
        out.zero_()
        gr.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
    c.release(0)
    c.release(1)
    assert c.free_pages() == 8 and bool((c.table == -1).all())
