"""The keeping of pages where the table cannot be written: nothing is taken, held or given
back, and the next call finds everything as it was.  CPU only (the table and the pool
stand in for the device's)."""

import contextlib
import copy

import pytest
import torch

from joule_amd import _lib
from joule_amd.decoder import DecoderShape
from joule_amd.dense import dense_ffn_shape
from joule_amd.kv_paged import PagedKVCacheSet


class Table:
    """A table whose writes fail while `broken` is set."""

    def __init__(self, B, width):
        self.t, self.broken = torch.full((B, width), -1, dtype=torch.int32), False

    def __setitem__(self, at, x):
        if self.broken:
            raise RuntimeError("the table cannot be written")
        self.t[at] = x


@pytest.fixture
def pages(monkeypatch):
    monkeypatch.setattr(_lib, "on", lambda *a: contextlib.nullcontext())
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    c = object.__new__(PagedKVCacheSet)
    c.shape = DecoderShape(n_layers=1, moe=dense_ffn_shape(1024, 512), n_heads=2, n_kv=2, maxT=100)
    c.B, c.n_pages, c.page, c._device = 3, 8, 16, torch.device("cpu")
    c.data, c.table = torch.zeros(1, 8, 2, 2, 16, 128), Table(3, 7)
    c._free, c._uses, c._pages = list(range(7, -1, -1)), [0] * 8, [[] for _ in range(3)]
    c.reserve(0, 40)
    return c


def kept(c):
    return copy.deepcopy((c._free, c._uses, c._pages, c.table.t.tolist()))


def tries(c):
    return {"reserve": lambda: c.reserve(1, 33), "grow": lambda: c.reserve(0, 64), "share": lambda: c.share(0, 1, 32),
            "share a part": lambda: c.share(0, 1, 39), "release": lambda: c.release(0)}


@pytest.mark.parametrize("what", ["reserve", "grow", "share", "share a part", "release"])
def test_a_table_that_cannot_be_written(pages, what):
    before = kept(pages)
    pages.table.broken = True
    with pytest.raises(RuntimeError, match="cannot be written"):
        tries(pages)[what]()
    assert kept(pages) == before
    pages.table.broken = False
    tries(pages)[what]()                                # it does what it would have done
    for b in range(3):
        pages.release(b)
    assert sorted(pages._free) == list(range(8)) and not any(pages._uses) and bool((pages.table.t == -1).all())


def test_a_page_that_cannot_be_copied(pages):
    class Pool:
        def __getitem__(self, at):
            raise RuntimeError("out of memory")

    before, data = kept(pages), pages.data
    pages.data = Pool()
    with pytest.raises(RuntimeError, match="out of memory"):
        pages.share(0, 1, 39)
    assert kept(pages) == before
    pages.data = data
    pages.share(0, 1, 39)
    assert pages._pages[1][:2] == pages._pages[0][:2] and pages.free_pages() == 4


@pytest.mark.parametrize("what", ["reserve", "grow", "share", "share a part", "release"])
def test_refused_while_a_graph_is_captured(pages, what, monkeypatch):
    """The write would be the graph's, to be done at every replay, and not have been done now."""
    before = kept(pages)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    with pytest.raises(RuntimeError, match="captur"):
        tries(pages)[what]()
    assert kept(pages) == before


def test_nothing_to_write_is_not_refused(pages, monkeypatch):
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    before = kept(pages)
    pages.reserve(0, 48)
    pages.share(1, 2, 0)
    pages.release(1)
    assert kept(pages) == before
