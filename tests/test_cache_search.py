"""PagedKVCache's bookkeeping for prompts, drafts and beams (no GPU: the calls that move tokens are stood in for)."""
import pytest
import torch


@pytest.fixture
def moved(te, monkeypatch):
    """What the cache asks to be copied or kept."""
    import importlib
    module = importlib.import_module(te.__name__ + ".kv_cache")
    calls = []
    monkeypatch.setattr(module, "copy_pages", lambda k, v, src, dst, counts=None, scores=None, pos=None: calls.append(
        ("copy", src.tolist(), dst.tolist(), counts.tolist())))

    def keep(k, v, table, lens, starts, path, scores=None, pos=None):
        calls.append(("keep", starts.tolist(), path.tolist()))
        return (lens - starts.diff() + (path >= 0).sum(1)).int()

    monkeypatch.setattr(module, "keep_kv", keep)
    return calls


def _cache(te, pages=12, rows=3, **kw):
    return te.PagedKVCache(2, 1, 8, rows=rows, max_len=64, pages=pages, page_size=16, device="cpu", **kw)


def _whole(c):
    """Every page is free or counted as often as rows have it."""
    have = [p for own in c._owned for p in own]
    assert all(c._refs[p] == have.count(p) for p in range(len(c._refs)))
    assert sorted(c._free) == [p for p in range(len(c._refs)) if p not in have]
    assert c.lens.tolist() == c.lengths and c.next_pos.tolist() == c.seen
    for b, own in enumerate(c._owned):
        assert len(own) == -(-c.lengths[b] // c.page_size)
        assert c.table[b].tolist() == own + [-1] * (c.table.shape[1] - len(own))
        # a page that a row will write to is its own
        assert all(c._refs[p] == 1 for p in own[c.lengths[b] // c.page_size:])


def test_depths_set_the_positions(te, moved):
    c = _cache(te)
    c.grow([5, 0, 2])
    c.grow([4, 1, 3], depths=[0, 1, 1, 2, 0, 0, 1, 2])
    assert c._positions.tolist() == [5, 6, 6, 7, 0, 2, 3, 4] and c._starts.tolist() == [0, 4, 5, 8]
    assert c.lengths == [9, 1, 5] and c.seen == [8, 1, 5]
    for bad in ([0, 1, 1], [0, 1, 1, 2, 0, 0, 1, -1]):
        with pytest.raises(ValueError):
            c.grow([4, 1, 3], depths=bad)
    c.grow(1, depths=[3, 0, 0])
    assert c._positions.tolist() == [11, 1, 5] and c._starts.tolist() == [0, 1, 2, 3]
    _whole(c)


def test_keep(te, moved):
    c = _cache(te)
    c.grow([14, 3, 0])
    c.grow([6, 2, 1], depths=[0, 1, 1, 2, 2, 3, 0, 0, 0])
    free = len(c._free)
    for bad in ([[0, 1], [0]], [[0, 6], [], []], [[1, 0], [], []], [[0, 0], [], []], [[-1], [], []]):
        with pytest.raises(ValueError):
            c.keep(bad)
    assert moved == [] and c.lengths == [20, 5, 1]
    c.keep([[0, 2], [1], []])
    assert moved == [("keep", [0, 6, 8, 9], [[0, 2], [1, -1], [-1, -1]])]
    assert c.lengths == c.seen == [16, 4, 0] and len(c._free) == free + 2
    _whole(c)
    with pytest.raises(ValueError):
        c.keep([[], [], []])
    with pytest.raises(ValueError):
        c.append(0, *(torch.zeros((3, 1, 8)) for _ in range(3)))
    c.grow(1)
    c.keep([[0], [], [0]])
    assert c.lengths == [17, 4, 1] and moved[-1] == ("keep", [0, 1, 2, 3], [[0], [-1], [0]])
    _whole(c)
    c.grow([2, 0, 0])
    c.keep([[], [], []])
    assert c.lengths == [17, 4, 1]
    _whole(c)


def test_reorder_shares_full_pages(te, moved):
    c = _cache(te)
    c.grow([37, 16, 3])
    own = [list(o) for o in c._owned]
    c.reorder([0, 0, 0])
    assert c.lengths == [37, 37, 37] and [o[:2] for o in c._owned] == [own[0][:2]] * 3 and c._owned[0] == own[0]
    (kind, src, dst, counts), = moved
    assert kind == "copy" and src == [own[0][2]] * 2 and counts == [5, 5] and dst == [c._owned[1][2], c._owned[2][2]]
    assert not set(src) & set(dst)
    _whole(c)
    c.grow(1)
    c.release(0)
    _whole(c)
    assert c._refs[own[0][0]] == 2
    c.reorder([1, 2, 0])
    assert c.lengths == [38, 38, 0] and len(moved) == 1          # each row has one heir: nothing is copied
    _whole(c)


def test_reorder_of_whole_pages_copies_nothing(te, moved):
    c = _cache(te)
    c.grow([32, 1, 0])
    c.reorder([0, 0, 2])
    assert moved == [] and c._owned[0] == c._owned[1] and c.lengths == [32, 32, 0]
    _whole(c)
    c.grow([1, 2, 0])
    assert c._owned[0][2] != c._owned[1][2]
    _whole(c)
    c.keep([[], [0], []])
    assert c.lengths == [32, 33, 0]
    _whole(c)


def test_reorder_of_an_evictable_cache_copies_all(te, moved):
    c = _cache(te, evictable=True)
    c.grow([20, 2, 0])
    own = [list(o) for o in c._owned]
    c.reorder([0, 0, 1])
    (_, src, dst, counts), = moved
    assert src == own[0] and counts == [16, 4] and dst == c._owned[1] and c._owned[2] == own[1]
    assert all(n <= 1 for n in c._refs)
    _whole(c)


def test_reorder_refuses(te, moved):
    c = _cache(te, pages=3)
    c.grow([17, 10, 0])
    before = [list(o) for o in c._owned], list(c._free), list(c._refs), c.table.clone()
    for bad in ([0, 0], [0, 1, 3], [0, -1, 2], [0, 1, 2, 0]):
        with pytest.raises(ValueError):
            c.reorder(bad)
    with pytest.raises(ValueError, match="pages"):
        c.reorder([0, 1, 0])
    assert moved == [] and c.lengths == [17, 10, 0]
    assert before[:3] == ([list(o) for o in c._owned], list(c._free), list(c._refs)) and torch.equal(c.table, before[3])
    # the dropped row's page is enough
    c.reorder([0, 0, 2])
    assert c.lengths == [17, 17, 0]
    _whole(c)


@pytest.mark.parametrize("evictable", [False, True])
def test_many_steps(te, moved, evictable):
    """Random steps of growing, keeping, forking and releasing: pages are neither lost nor given twice."""
    import random
    rng = random.Random(5)
    c = _cache(te, pages=20, rows=4, evictable=evictable)
    for _ in range(300):
        try:
            what = rng.randrange(4)
            if what == 0:
                c.grow([rng.randrange(7) for _ in range(4)])
            elif what == 1 and c._drafts:
                c.keep([sorted(rng.sample(range(n), rng.randint(0, n))) for n in c._drafts[0]])
            elif what == 2:
                c.reorder([rng.randrange(4) for _ in range(4)])
            else:
                c.release(rng.randrange(4))
        except ValueError:
            pass
        _whole(c)
