"""PagedKVCache on a GPU: steps in which some of the rows wait."""
import pytest
import torch

pytestmark = pytest.mark.gpu
F16, F32 = torch.float16, torch.float32


def _step(cache, counts, g, dev, heads=2, d=64):
    cache.grow(counts)
    n = sum([counts] * len(cache.lengths) if isinstance(counts, int) else counts)
    q, k, v = (torch.randn((n, h, d), generator=g, device=dev, dtype=F16) for h in (2 * heads, heads, heads))
    cache.append(0, q, k, v)
    return torch.randn((len(cache.lengths), 2 * heads, d), generator=g, device=dev, dtype=F16)


def _of(plane, cache, row):
    j = torch.arange(cache.lengths[row], device=plane.device)
    return plane[cache.table[row].long()[j // cache.page_size], :, j % cache.page_size]


@pytest.mark.parametrize("prompt", [[40, 3, 17, 0], [700, 3, 17, 0]])
@pytest.mark.parametrize("y", [F16, F32])
def test_scores_of_waiting_rows_stay(te, gpu_device, prompt, y):
    """Rows that a step gives no token keep their scores, whatever query they are asked with; every row's answer, and the
    other rows' scores, are those of a call on its own tensors."""
    make = lambda evictable: te.PagedKVCache(1, 2, 64, rows=4, max_len=800, page_size=16, device=gpu_device, evictable=evictable)
    cache, plain = make(True), make(False)
    seeds = [torch.Generator(device=gpu_device).manual_seed(1) for _ in range(2)]
    for counts in (prompt, [0, 1, 0, 2], 1, [0, 0, 0, 0], [1, 0, 0, 0]):
        q, q2 = _step(cache, counts, seeds[0], gpu_device), _step(plain, counts, seeds[1], gpu_device)
        assert torch.equal(q, q2)
        was = cache.scores[0].clone()
        twin = cache.scores[0].clone()
        out = cache.attend(0, q, out_dtype=y)
        want = te.paged_attention(q, cache.k[0], cache.v[0], cache.table, cache.lens, max_len=max(cache.lengths), scores=twin, out_dtype=y)
        assert torch.equal(out, want) and torch.equal(out, plain.attend(0, q, out_dtype=y))
        for b in range(4):
            waits = isinstance(counts, list) and counts[b] == 0
            old = _of(was if waits else twin, cache, b)
            assert torch.equal(_of(cache.scores[0], cache, b), old), (counts, b)


def test_waiting_rows_after_an_eviction_and_a_release(te, gpu_device):
    g = torch.Generator(device=gpu_device).manual_seed(2)
    cache = te.PagedKVCache(1, 2, 64, rows=4, max_len=100, page_size=16, device=gpu_device, evictable=True)
    cache.attend(0, _step(cache, [40, 30, 17, 2], g, gpu_device))
    cache.attend(0, _step(cache, [1, 0, 1, 0], g, gpu_device))
    cache.evict(20, 5)
    assert cache.lens.tolist() == [20, 20, 18, 2]
    was, q = cache.scores[0].clone(), torch.randn((4, 4, 64), generator=g, device=gpu_device, dtype=F16)
    out = cache.attend(0, q, out_dtype=F32)
    assert torch.equal(out, te.paged_attention(q, cache.k[0], cache.v[0], cache.table, cache.lens, out_dtype=F32))
    assert torch.equal(_of(cache.scores[0], cache, 1), _of(was, cache, 1)) and not torch.equal(_of(cache.scores[0], cache, 0), _of(was, cache, 0))
    cache.release(0)
    was = cache.scores[0].clone()
    out = cache.attend(0, q, out_dtype=F32)
    assert (out[0] == 0).all() and (out[1:] != 0).any(-1).all()
    assert torch.equal(_of(cache.scores[0], cache, 3), _of(was, cache, 3))
