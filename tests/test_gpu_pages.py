"""copy_pages and keep_kv against plain restatements (search_ref), to the bit."""
import pytest
import torch

import search_ref as ref
from serve_ref import Pages

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16
SHAPES = [(8, 128, 64, F16, "hs"), (3, 64, 16, BF16, "hs"), (2, 80, 32, F16, "sh"), (1, 256, 16, BF16, "sh"), (1, 8, 1024, F16, "hs"),
          (2, 136, 128, F16, "hs"), (5, 24, 16, F16, "hs")]


def same(got, want, what=""):
    got, want = got.cpu(), want
    if got.is_floating_point():
        assert torch.equal(got.isnan(), want.isnan()), what
        got, want = got.nan_to_num(0), want.nan_to_num(0)
    assert torch.equal(got, want), what


def _layers(P, count, dev):
    """`count` layers of P's pool, with planes of their own: lists of k, v, scores, pos on the CPU and on the device."""
    def more(t):
        if t.is_floating_point():
            turned = t if t.is_contiguous() else t.transpose(1, 2)
            fresh = torch.randn(turned.shape, generator=P.g).to(t.dtype)
            return fresh if t.is_contiguous() else fresh.transpose(1, 2)
        return torch.randint(0, 1000, t.shape, generator=P.g).int()

    def move(t):
        return t.to(dev) if t.is_contiguous() else t.transpose(1, 2).to(dev).transpose(1, 2)

    host = [[more(t) for _ in range(count)] for t in (P.k, P.v, P.scores, P.pos)]
    return host, [[move(t) for t in ts] for ts in host]


@pytest.mark.parametrize("heads,d,page,dtype,layout", SHAPES)
@pytest.mark.parametrize("layers", [1, 3, 40])
def test_copies(te, gpu_device, heads, d, page, dtype, layout, layers):
    if layers == 40 and page * d * heads > 20000:
        layers = 33
    P = Pages([page * 3, page * 4 + 1], heads, page, d, dtype, d, layout=layout, idle=None)
    host, dev = _layers(P, layers, gpu_device)
    src, dst = [0, 3, 2, 7], [1, 8, 4, 5]
    for counts in (None, [1, page, 0, page // 2 + 1], [page - 1, 2 * page, -3, 7]):
        want = [ref.copy_pages([t[i] for t in host], src, dst, counts) for i in range(layers)]
        ints = lambda v: None if v is None else torch.tensor(v, dtype=torch.int32, device=gpu_device)
        k, v, s, z = ([t.clone() if t.is_contiguous() else t.transpose(1, 2).clone().transpose(1, 2) for t in ts] for ts in dev)
        assert te.copy_pages(k, v, ints(src), ints(dst), counts=ints(counts), scores=s, pos=z) is None
        for i in range(layers):
            for got, w in zip((k[i], v[i], s[i], z[i]), want[i]):
                same(got, w, (i, counts))


def test_copies_of_one_layer_and_without_planes(te, gpu_device):
    P = Pages([100], 2, 16, 64, F16, 1, idle=None)
    k, v, _, _, scores, pos = P.to(gpu_device)
    src, dst = (torch.tensor(t, dtype=torch.int32, device=gpu_device) for t in ([0, 1], [5, 6]))
    te.copy_pages(k, v, src, dst)
    want = ref.copy_pages([P.k, P.v], [0, 1], [5, 6])
    same(k, want[0]), same(v, want[1]), same(scores, P.scores), same(pos, P.pos)
    te.copy_pages((k,), (v,), src, dst, scores=[None], pos=[pos])
    same(scores, P.scores), same(pos, ref.copy_pages([P.pos], [0, 1], [5, 6])[0])


def test_layers_in_one_tensor(te, gpu_device):
    """Stacked layers, contiguous or a slice of a larger stack, give what a list of them gives."""
    P = Pages([60, 33], 2, 16, 64, F16, 9, idle=None, spare=6)
    host, _ = _layers(P, 5, gpu_device)
    stack = [torch.stack(t).to(gpu_device) for t in host]
    every = [torch.cat([t, t])[::2] for t in stack]      # layers 0, 2, 4, 1, 3, two strides apart
    ints = lambda t: torch.tensor(t, dtype=torch.int32, device=gpu_device)
    src, dst, starts, path = ints([0, 1]), ints([3, 2]), ints([0, 10, 20]), ints([[0, 3, 8, -1], [1, 2, 5, 9]])
    for k, v, s, z in (stack, every):
        lists = [[u.clone() for u in t] for t in (k, v, s, z)]
        te.copy_pages(k, v, src, dst, scores=s, pos=z)
        te.copy_pages(lists[0], lists[1], src, dst, scores=lists[2], pos=lists[3])
        table, lens = P.table.to(gpu_device), P.lens.to(gpu_device)
        a = te.keep_kv(k, v, table, lens, starts, path, scores=s, pos=z)
        assert torch.equal(a, te.keep_kv(lists[0], lists[1], table, lens, starts, path, scores=lists[2], pos=lists[3]))
        for got, want in zip((k, v, s, z), lists):
            assert torch.equal(got.nan_to_num(0), torch.stack(want).nan_to_num(0))
    k, v, s, z = stack
    for bad in (lambda: te.copy_pages(k, v[:4], src, dst), lambda: te.copy_pages(k, list(v), src, dst), lambda: te.copy_pages(list(k), v, src, dst),
                lambda: te.copy_pages(k, v, src, dst, scores=s[0]), lambda: te.copy_pages(k, v, src, dst, pos=list(z)), lambda: te.copy_pages(k[:0], v[:0], src, dst),
                lambda: te.copy_pages(k[0], v, src, dst), lambda: te.copy_pages(list(k), list(v), src, dst, scores=s)):
        with pytest.raises((ValueError, RuntimeError)):
            bad()


def test_copies_of_pages_that_are_none(te, gpu_device):
    """Ids outside the pool, and a page onto itself, copy nothing; no pages at all are no error."""
    P = Pages([100], 2, 16, 64, F16, 2, idle=None)
    k, v, *_ = P.to(gpu_device)
    bad = torch.tensor([-1, P.pages, 2 ** 31 - 1, 3, 0, 1, -2 ** 31], dtype=torch.int32, device=gpu_device)
    to = torch.tensor([0, 1, 2, 3, -1, P.pages, 4], dtype=torch.int32, device=gpu_device)
    te.copy_pages(k, v, bad, to)
    te.copy_pages(k, v, bad[:0], to[:0])
    same(k, P.k), same(v, P.v)


def test_copies_many_pages(te, gpu_device):
    P = Pages([16 * 600], 1, 16, 8, F16, 3, idle=None)
    k, v, *_ = P.to(gpu_device)
    order = torch.randperm(P.pages, generator=P.g)
    src, dst = order[:300].tolist(), order[300:600].tolist()
    te.copy_pages(k, v, *(torch.tensor(t, dtype=torch.int32, device=gpu_device) for t in (src, dst)))
    want = ref.copy_pages([P.k, P.v], src, dst)
    same(k, want[0]), same(v, want[1])


def _keep(te, dev, lengths, new, paths, heads=2, d=64, page=16, dtype=F16, layout="hs", layers=1, seed=0, planes=True, width=None, lens=None):
    P = Pages(lengths, heads, page, d, dtype, seed, layout=layout, idle=None)
    host, on = _layers(P, layers, dev)
    k, v, s, z = on
    starts = [3]
    for n in new:
        starts.append(starts[-1] + n)
    width = max([len(p) for p in paths] + [0]) if width is None else width
    path = torch.tensor([p + [-1] * (width - len(p)) for p in paths], dtype=torch.int32).view(len(paths), width)
    lens = lengths if lens is None else lens
    dl = torch.tensor(lens, dtype=torch.int32, device=dev)
    got = te.keep_kv(k, v, P.table.to(dev), dl, torch.tensor(starts, dtype=torch.int32, device=dev), path.to(dev),
                     scores=s if planes else None, pos=z if planes else None)
    for i in range(layers):
        want, new_lens = ref.keep([t[i] for t in host], P.table, page, lens, starts, paths)
        for j, (a, w) in enumerate(zip((k[i], v[i], s[i], z[i]), want)):
            same(a, w if planes or j < 2 else host[j][i], (i, j))
    assert got.dtype == torch.int32 and got.tolist() == new_lens and dl.tolist() == lens
    return got


@pytest.mark.parametrize("heads,d,page,dtype,layout", SHAPES)
@pytest.mark.parametrize("layers", [1, 4, 34])
def test_paths(te, gpu_device, heads, d, page, dtype, layout, layers):
    new = [9, 0, 1, 1, 5, 26, 26]
    paths = [[0, 2, 5, 8], [], [0], [], [4], list(range(26)), [3, 4, 20, 25]]
    _keep(te, gpu_device, [page + 9, 5, 1, 40, 5, 50, 26], new, paths, heads, d, page, dtype, layout, layers, seed=d)


@pytest.mark.parametrize("n", [17, 70, 255, 256, 257, 700])
def test_long_paths(te, gpu_device, n):
    """Moves over more tokens than a group holds: a slot is read before it is written over."""
    g = torch.Generator().manual_seed(n)
    some = torch.randperm(n, generator=g)[:n * 2 // 3].sort().values.tolist()
    paths = [list(range(1, n)), some, [n - 1], list(range(n)), list(range(n // 2, n))]
    for d in (64, 8, 256):
        _keep(te, gpu_device, [n, n + 5, n + 16, n, n + 100], [n] * 5, paths, heads=1, d=d, seed=n, layers=2)


def test_paths_that_end_early(te, gpu_device):
    """At the first entry that is not above the last, negative or not below the row's new tokens."""
    paths = [[0, 2, 2, 5], [3, 1, 4, 5], [0, 6, 1, 2], [-1, 0, 1, 2], [5, 2 ** 31 - 1, 1, 1], [1, 2, -5, 3], [0, 1, 2, 3]]
    _keep(te, gpu_device, [20, 33, 16, 6, 40, 17, 50], [6] * 7, paths)
    _keep(te, gpu_device, [20, 33], [6, 2], [[], []], width=3)
    _keep(te, gpu_device, [20, 33], [6, 2], [[], []], width=0)
    _keep(te, gpu_device, [20, 33], [6, 2], [[0, 3], [1]], planes=False)


def test_slots_that_are_not_there(te, gpu_device):
    """Lengths below the new tokens' number, and past the table."""
    _keep(te, gpu_device, [20, 33, 40], [10, 10, 10], [[0, 3, 9], [2, 5, 7], [1, 2, 3]], lens=[4, 0, 48 + 5])
    _keep(te, gpu_device, [20], [10], [[4, 6, 7]], lens=[2 ** 31 - 1])


def test_missing_pages(te, gpu_device):
    P = Pages([60, 60], 2, 16, 64, F16, 5, idle=None)
    P.table[0, 2], P.table[1, 1] = -1, P.pages + 3
    k, v, table, lens, scores, pos = P.to(gpu_device)
    starts, paths = [0, 40, 80], [[0, 5, 13, 30, 39], [7, 9, 20, 38]]
    path = torch.tensor([p + [-1] * (5 - len(p)) for p in paths], dtype=torch.int32, device=gpu_device)
    got = te.keep_kv(k, v, table, lens, torch.tensor(starts, dtype=torch.int32, device=gpu_device), path, scores=scores, pos=pos)
    want, new = ref.keep([P.k, P.v, P.scores, P.pos], P.table, 16, [60, 60], starts, paths)
    for a, w in zip((k, v, scores, pos), want):
        same(a, w)
    assert got.tolist() == new


def test_graph(te, gpu_device):
    """Copies and paths in a captured graph: every replay, with eager calls between, equals the eager call."""
    P = Pages([60, 33], 2, 16, 64, F16, 6, idle=None, spare=6)
    (k, v, table, lens, scores, pos), twin = P.to(gpu_device), P.to(gpu_device)
    ints = lambda t: torch.tensor(t, dtype=torch.int32, device=gpu_device)
    free = [p for p in range(P.pages) if p not in set(P.table.flatten().tolist())]
    src, dst, starts, path = ints(P.table[0, :2].tolist()), ints(free[:2]), ints([0, 10, 20]), ints([[0, 3, 8, -1], [1, 2, 5, 9]])

    def step(k, v, lens, scores, pos):
        te.copy_pages([k], [v], src, dst, scores=[scores], pos=[pos])
        return te.keep_kv([k], [v], table, lens, starts, path, scores=[scores], pos=[pos])

    step(*(t.clone() for t in (k, v, lens, scores, pos)))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(k, v, lens, scores, pos)
    a, b = (k, v, scores, pos), (twin[0], twin[1], twin[4], twin[5])
    for i, (p, at) in enumerate((([[0, 3, 8, -1], [1, 2, 5, 9]], [60, 33]), ([[9, -1, -1, -1], [-1, 2, 5, 9]], [57, 33]), ([[0, 1, 2, 3], [4, 5, 6, 7]], [48, 31]))):
        path.copy_(ints(p))
        lens.copy_(ints(at))
        graph.replay()
        want = step(twin[0], twin[1], ints(at), twin[4], twin[5])
        torch.cuda.synchronize()
        assert torch.equal(out, want) and all(torch.equal(s, t) for s, t in zip(a, b)), i


def test_writes_count(te, gpu_device):
    P = Pages([40], 2, 16, 64, F16, 7, idle=None)
    k, v, table, lens, scores, pos = P.to(gpu_device)
    one = torch.zeros(1, dtype=torch.int32, device=gpu_device)
    starts, path = torch.tensor([0, 4], dtype=torch.int32, device=gpu_device), one[None]
    own = {"k": k, "v": v, "table": table, "lens": lens, "scores": scores, "pos": pos, "starts": starts, "path": path, "one": one}

    def counted(call):
        before = {n: u._version for n, u in own.items()}
        call()
        return {n for n, u in own.items() if u._version != before[n]}

    assert counted(lambda: te.copy_pages([k], [v], one, one)) == {"k", "v"}
    assert counted(lambda: te.copy_pages(k, v, one, one, scores=scores, pos=[pos])) == {"k", "v", "scores", "pos"}
    assert counted(lambda: te.keep_kv([k], [v], table, lens, starts, path, scores=[scores])) == {"k", "v", "scores"}


def test_refusals(te, gpu_device):
    P = Pages([40, 3], 2, 16, 64, F16, 8, idle=None)
    k, v, table, lens, scores, pos = P.to(gpu_device)
    one = torch.zeros(1, dtype=torch.int32, device=gpu_device)
    starts, path = torch.tensor([0, 4, 5], dtype=torch.int32, device=gpu_device), torch.zeros((2, 3), dtype=torch.int32, device=gpu_device)
    cp = lambda k=k, v=v, src=one, dst=one, **kw: te.copy_pages(k, v, src, dst, **kw)
    kp = lambda k=k, v=v, table=table, lens=lens, starts=starts, path=path, **kw: te.keep_kv(k, v, table, lens, starts, path, **kw)
    bad = [lambda: cp([]), lambda: cp([k], [v, v]), lambda: cp([k, k], [v, v], scores=scores), lambda: cp([k, k], [v, v], pos=[pos]),
           lambda: cp([k, k[:-1]], [v, v[:-1]]), lambda: cp([k, k.bfloat16()], [v, v.bfloat16()]), lambda: cp(k.cpu(), v.cpu()),
           lambda: cp(src=one.long()), lambda: cp(dst=path[0]), lambda: cp(counts=path[0]), lambda: cp(dst=None), lambda: cp(src=None),
           lambda: cp(src=path), lambda: cp(scores=scores.half()), lambda: cp(pos=pos[:-1]), lambda: cp(k.float(), v.float()),
           lambda: cp("x", v), lambda: cp([k.clone().requires_grad_()], [v]), lambda: cp([k, None], [v, v]),
           lambda: kp(path=path[:1]), lambda: kp(path=path.long()), lambda: kp(path=path.cpu()), lambda: kp(path=path[0]), lambda: kp(path=path.t()[:2]),
           lambda: kp(starts=starts[:2]), lambda: kp(starts=None), lambda: kp(path=None), lambda: kp(table=None), lambda: kp(lens=None),
           lambda: kp(lens=lens[:1]), lambda: kp(table=table.long()), lambda: kp([], [])]
    for i, f in enumerate(bad):
        with pytest.raises((ValueError, RuntimeError)):
            f()
            pytest.fail(f"call {i} was not refused")
    assert kp(table=table[:0], lens=lens[:0], starts=starts[:1], path=path[:0]).shape == (0,)
