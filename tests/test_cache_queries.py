"""PagedKVCache.attend_new takes a query for each token that grow() made room for, neither more nor fewer (no GPU: the
attention is stood in for)."""
import importlib

import pytest
import torch


@pytest.fixture
def asked(te, monkeypatch):
    """The queries that reach the attention, and whose."""
    calls = []
    module = importlib.import_module(te.__name__ + ".kv_cache")
    monkeypatch.setattr(module, "tree_attention", lambda q, *a, starts=None, **kw: calls.append(
        (q.shape[0], None if starts is None else starts.tolist())) or q)
    return calls


@pytest.mark.parametrize("counts,starts", [(1, None), (2, [0, 2, 4, 6]), ([5, 0, 2], [0, 5, 5, 7]), ([1, 1, 1], None), ([0, 0, 0], [0] * 4)])
def test_as_many_queries_as_tokens(te, asked, counts, starts):
    """After a step of one token each (no starts) twice as many queries would be two new tokens a row, one of them older;
    elsewhere fewer would move the rows' first slots, more would get zeros."""
    c = te.PagedKVCache(2, 1, 8, rows=3, max_len=64, pages=12, page_size=16, device="cpu")
    c.grow(4)
    c.grow(counts)
    n = 3 * counts if isinstance(counts, int) else sum(counts)
    for bad in {0, n - 1, n + 1, 2 * n, 3, 6} - {n, -1}:
        with pytest.raises(ValueError, match="query for each"):
            c.attend_new(0, torch.zeros((bad, 2, 8)))
    for shape in ((n, 8), (n, 2, 2, 8)):
        with pytest.raises(ValueError, match="query for each"):
            c.attend_new(0, torch.zeros(shape))
    assert asked == []
    assert c.attend_new(1, torch.zeros((n, 2, 8))).shape == (n, 2, 8) and asked == [(n, starts)]
