"""PagedKVCache.reorder over rows of many pages: what it counts grows with the pages, not with their square (no GPU: the
copies are stood in for)."""
import importlib

import pytest
import torch


class Page(int):
    """A page number that counts how often it is compared."""
    compared = 0

    def __eq__(self, other):
        Page.compared += 1
        return int(self) == other

    __hash__ = int.__hash__


@pytest.fixture
def copies(te, monkeypatch):
    calls = []
    monkeypatch.setattr(importlib.import_module(te.__name__ + ".kv_cache"), "copy_pages",
                        lambda k, v, src, dst, **kw: calls.append((src.tolist(), dst.tolist())))
    return calls


@pytest.mark.parametrize("evictable", [False, True])
@pytest.mark.parametrize("spare", [0, 4000])
def test_reorder_of_many_pages(te, copies, evictable, spare):
    """16 rows of 128 pages, half of them dropped: once with pages to spare, once with none, where the dropped rows' are
    enough. Any page is compared a few times at most (looked up for the dropped, shared ones among them counted once)."""
    rows, width = 16, 128
    c = te.PagedKVCache(1, 1, 8, rows=rows, max_len=16 * width, pages=rows * width + spare, page_size=16, device="cpu", evictable=evictable)
    c._free = [Page(p) for p in c._free]
    c.grow(16 * width - 1)
    # rows in pairs go on from one; the odd ones are dropped
    parents = [b // 2 * 2 for b in range(rows)]
    for step in range(3):
        Page.compared = 0
        kept = [c._owned[p] for p in parents]
        c.reorder(parents)
        assert Page.compared <= 4 * rows * width
        full = 0 if evictable else width - 1
        for b, p in enumerate(parents):
            assert len(c._owned[b]) == width and [int(x) for x in c._owned[b][:full]] == [int(x) for x in kept[b][:full]]
        have = [int(p) for own in c._owned for p in own]
        free = sorted(int(p) for p in c._free)
        assert all(c._refs[p] == n for p, n in zip(*[t.tolist() for t in torch.tensor(have).unique(return_counts=True)]))
        assert sorted(free + list(set(have))) == list(range(rows * width + spare))


def test_shared_pages_of_dropped_rows_come_back_once_all_are_dropped(te, copies):
    """Pages that two dropped rows share count once towards the room; those that a row which stays shares too, not at all."""
    c = te.PagedKVCache(1, 1, 8, rows=4, max_len=64, pages=7, page_size=16, device="cpu")
    c.grow([64, 0, 33, 0])                       # 4 and 3 pages: the pool is empty
    c.reorder([0, 0, 2, 3])                      # four full pages shared
    assert len(c._free) == 0 and copies == []
    with pytest.raises(ValueError, match="1 pages needed, 0 free"):
        c.reorder([0, 3, 2, 2])                  # row 1's pages are row 0's too
    c.reorder([3, 3, 2, 2])                      # both are dropped: four pages come back, one is taken
    assert len(c._free) == 3 and c.lengths == [0, 0, 33, 33] and len(copies) == 1
