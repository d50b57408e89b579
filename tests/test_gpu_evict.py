"""evict_kv in forms beside test_gpu_kv.py's, against the definition: moves are copies, so everything is
compared bit for bit."""
import pytest
import torch

import serve_ref as ref

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("keep", [1 << 20, 2 ** 30])
def test_keep_beyond_every_row(te, gpu_device, keep):
    """Nothing is evicted; into other pages everything is copied. Scratch goes by the rows, not by `keep`."""
    lengths = [70, 0, 33, 16]
    P = ref.Pages(lengths, 2, 16, 64, torch.float16, 1, idle=None)
    need = -(-max(lengths) // 16)
    out = (P.pages + torch.arange(need * len(lengths))).int().view(len(lengths), need)
    grow = lambda t: torch.cat([t, torch.zeros_like(t[:1]).expand(out.numel(), *t.shape[1:])])
    P.k, P.v, P.scores, P.pos = (grow(t) for t in (P.k, P.v, P.scores, P.pos))
    k, v, table, lens, scores, pos = P.to(gpu_device)
    new = te.evict_kv(k, v, scores, pos, table, lens, keep, 5, out_table=out.to(gpu_device))
    assert new.tolist() == lengths
    for b, n in enumerate(lengths):
        page, slot = P.slots(b, n)
        to = out[b].long()[torch.arange(n) // 16]
        for got, old in ((k, P.k), (v, P.v), (scores, P.scores), (pos, P.pos)):
            assert torch.equal(got.cpu()[to, :, slot], old[page, :, slot])
    before = [t.clone() for t in (k, v, scores, pos)]
    assert te.evict_kv(k, v, scores, pos, table, lens, keep, 5).tolist() == lengths
    assert all(torch.equal(a, b) for a, b in zip(before, (k, v, scores, pos)))


def _order(pages, b, h, present, n, recent):
    """Row b's tokens on existing pages, the ones to keep first: the newest, the heaviest, the lowest slot."""
    at = lambda plane, j: plane[int(pages.table[b, j // pages.page]), h, j % pages.page].item()
    new = lambda j: at(pages.pos, j) >= n - recent
    return sorted(present, key=lambda j: (not new(j), 0.0 if new(j) else -at(pages.scores, j), j))


def _moves(pages, b, h, n, keep, recent, room=None):
    """[(from, to)] of the kept tokens of a row and head, and the new length. room: slots of the other pages (None: in place)."""
    present = [j for j in range(n) if 0 <= int(pages.table[b, j // pages.page]) < pages.pages]
    if room is None:
        if n <= keep:
            return [], n
        kept = set(_order(pages, b, h, present, n, recent)[:sum(j < keep for j in present)])
        free = [j for j in present if j < keep and j not in kept]
        return list(zip(sorted(j for j in kept if j >= keep), free)), keep
    count = min(keep, room, len(present))
    kept = set(_order(pages, b, h, present, n, recent)[:count])
    above = sorted(j for j in kept if j >= count)
    return [(j if j in kept else above.pop(0), j) for j in range(count)], count


def _check(te, dev, lengths, missing, keep, recent, apart, room=None, page=16, heads=2, d=64, ties=False, seed=0):
    """missing: (row, page of the row, the id it gets there). room: slots of the out table."""
    P = ref.Pages(lengths, heads, page, d, torch.float16, seed, idle=None)
    P.pos = torch.zeros_like(P.pos)
    for b, n in enumerate(lengths):
        pg, sl = P.slots(b, n)
        P.pos[pg, :, sl] = torch.arange(n).int()[:, None].expand(-1, heads)
    if ties:
        P.scores = P.scores.floor()
    for b, i, idn in missing:
        P.table[b, i] = idn
    out, rooms = None, None
    if apart:
        rooms = -(-min(keep, max(lengths)) // page) * page if room is None else room
        out = (P.pages + torch.randperm(rooms // page * len(lengths), generator=P.g)).int().view(len(lengths), -1)
        grow = lambda t: torch.cat([t, t[:1].expand(out.numel(), *t.shape[1:])])
        P.k, P.v, P.scores, P.pos = (grow(t) for t in (P.k, P.v, P.scores, P.pos))
        P.pages += out.numel()
        old_pages, P.pages = P.pages, P.pages - out.numel()
    planes = (P.k, P.v, P.scores, P.pos)
    want, lens_want = [t.clone() for t in planes], []
    for b, n in enumerate(lengths):
        for h in range(heads):
            moves, new = _moves(P, b, h, n, keep, recent, rooms)
            for a, z in moves:
                to = int((P.table if out is None else out)[b, z // page])
                for w, t in zip(want, planes):
                    w[to, h, z % page] = t[int(P.table[b, a // page]), h, a % page]
        lens_want.append(new)
    k, v, table, lens, scores, pos = P.to(dev)
    if not apart:
        old_pages = P.pages
    assert k.shape[0] == old_pages
    # an id is no page where the pool has none: the ids in `missing` lie outside the grown pool too
    got = te.evict_kv(k, v, scores, pos, table, lens, keep, recent, out_table=None if out is None else out.to(dev))
    assert got.tolist() == lens_want
    for name, a, w in zip(("k", "v", "scores", "pos"), (k, v, scores, pos), want):
        assert torch.equal(a.cpu(), w), name


MISSING = [(0, 1, -1), (0, 5, 1 << 20), (1, 0, -7), (3, 2, -1), (4, 0, 2 ** 31 - 1), (4, 1, -1)]


@pytest.mark.parametrize("apart", [False, True])
@pytest.mark.parametrize("keep,recent", [(1, 0), (16, 3), (40, 10), (64, 64), (100, 7), (300, 0)])
@pytest.mark.parametrize("ties", [False, True])
def test_missing_pages(te, gpu_device, apart, keep, recent, ties):
    """Tokens on pages that do not exist are absent: never kept in another's place, never moved, and their slots take
    nothing in place; into other pages the present ones close up."""
    _check(te, gpu_device, [130, 100, 33, 70, 32, 0, 200], MISSING, keep, recent, apart, ties=ties, seed=keep)


@pytest.mark.parametrize("apart", [False, True])
def test_missing_pages_of_long_rows(te, gpu_device, apart):
    """More moves than the selection makes itself, rows of each of its forms, segments among them."""
    for lengths, keep in (([1500, 900], 700), ([3000], 1000), ([9000], 5000), ([20000], 8000), ([40000], 30000)):
        missing = [(0, 0, -1), (0, 3, -1), (0, lengths[0] // 128 - 1, -1)]
        _check(te, gpu_device, lengths, missing, keep, 50, apart, page=128, heads=1, d=8, ties=True)


def test_no_page_at_all(te, gpu_device):
    for apart in (False, True):
        _check(te, gpu_device, [40, 40], [(0, 0, -1), (0, 1, -1), (0, 2, -1)], 10, 2, apart)
        _check(te, gpu_device, [40, 40], [(0, 0, -1), (0, 1, -1), (0, 2, -1)], 64, 2, apart)


@pytest.mark.parametrize("room", [16, 32, 48])
def test_out_table_with_less_room_than_keep(te, gpu_device, room):
    """What the out table has slots for is kept, the worthiest; the lengths count no more."""
    _check(te, gpu_device, [130, 20, 0, 64], [], 60, 12, True, room=room)
    _check(te, gpu_device, [130, 20, 0, 64], [(0, 2, -1), (3, 0, -1)], 60, 12, True, room=room)
