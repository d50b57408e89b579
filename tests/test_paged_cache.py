"""PagedKVCache's bookkeeping (no GPU)."""
import pytest


def _cache(te, **kw):
    return te.PagedKVCache(1, 1, 8, rows=3, max_len=40, pages=9, page_size=16, device="cpu", **kw)


@pytest.mark.parametrize("row", [-1, -3, 3, 100])
def test_release_of_a_row_that_is_none(te, row):
    """It raises and changes nothing: counted from the end, a row would lose its positions and keep its tokens."""
    c = _cache(te)
    c.grow([1, 20, 17])
    free = list(c._free)
    with pytest.raises(ValueError):
        c.release(row)
    assert c.lengths == c.seen == [1, 20, 17] and c._free == free
    assert c.lens.tolist() == c.next_pos.tolist() == [1, 20, 17]
    c.grow(1)
    assert c._positions.tolist() == [1, 20, 17]


@pytest.mark.parametrize("row", [0, 1, 2])
def test_release_empties_its_row_alone(te, row):
    c = _cache(te)
    c.grow([1, 20, 17])
    c.release(row)
    left = [0 if b == row else n for b, n in enumerate([1, 20, 17])]
    assert c.lengths == c.seen == left and c.lens.tolist() == c.next_pos.tolist() == left
    assert (c.table[row] == -1).all() and len(c._free) == 9 - sum(-(-n // 16) for n in left)
