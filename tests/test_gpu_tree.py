"""tree_attention against its float64 restatement (search_ref), at the lengths, trees, pages, head layouts, strides and
masks where it can go wrong.

Tolerances. As the attention of one token (test_gpu_kv): a logit's error, relative to its weight, is at most 2e-4 for these
inputs, so out, a mean of values, is off by 2e-4 x max |v| before its rounding. Where q, cache and out are of one 16-bit
type, a weight may be rounded once to that type besides, half a step relative to itself: 2^-11 (f16) or 2^-8 (bf16) of
max |v| at most."""
import pytest
import torch

import search_ref as ref
import serve_ref
from serve_ref import Pages, close

pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
TYPES = [(F16, F16, F16), (BF16, BF16, BF16), (F32, F16, F32), (F32, BF16, F32), (BF16, F16, BF16), (F16, BF16, F16)]


def _starts(new, first=0):
    s = [first]
    for n in new:
        s.append(s[-1] + n)
    return torch.tensor(s, dtype=torch.int32)


def _parents(new, g, back=4):
    """Random trees: each token continues one of the last few before it, or the cached tokens."""
    out = []
    for n in new:
        out += [int(torch.randint(max(-1, i - back), i, (1,), generator=g)) if i else -1 for i in range(n)]
    return torch.tensor(out, dtype=torch.int32)


def _error(P, x, cache, y):
    top = float(P.v.double().nan_to_num(0, 0, 0).abs().max())
    return (2e-4 + ((2.0 ** -11 if cache == F16 else 2.0 ** -8) if x == cache == y else 0.0)) * top


def _tree(te, dev, lengths, new, heads, group, d, page, x=F16, cache=F16, y=F16, seed=0, parents="tree", layout="hs", idle=float("nan"),
          scale=None, max_len=None, strided=False, uniform=False, qscale=2.0):
    P = Pages(lengths, heads, page, d, cache, seed, idle=idle, layout=layout)
    starts = _starts(new)
    if parents == "tree":
        parents = _parents(new, P.g)
    q = (torch.randn((sum(new), heads * group, d), generator=P.g) * qscale).to(x)
    k, v, table, lens, _, _ = P.to(dev)
    dq = q.to(dev)
    if strided:    # heads of a wider buffer, tokens an odd distance apart
        wide = torch.zeros((sum(new), heads * group * d + 3), dtype=x, device=dev)
        wide[:, 1:-2] = dq.flatten(1)
        dq = wide[:, 1:-2].unflatten(1, (-1, d))
    got = te.tree_attention(dq, k, v, table, lens, starts=None if uniform else starts.to(dev),
                            parents=None if parents is None else parents.to(dev), scale=scale, max_len=max_len, out_dtype=y)
    want = ref.tree(q, P, starts, parents, scale, max_len=max_len)
    close(got, want, y, _error(P, x, cache, y), "out")
    return got


LENGTHS = [0, 1, 15, 17, 33, 64, 130, 130, 500]
NEW = [0, 1, 15, 1, 7, 64, 130, 0, 40]


@pytest.mark.parametrize("heads,group,d,page", [(2, 4, 128, 64), (3, 3, 64, 16), (2, 1, 128, 16), (1, 16, 128, 32), (1, 17, 64, 16),
                                                (1, 40, 32, 128), (2, 2, 80, 32), (1, 5, 96, 16), (1, 4, 256, 64), (1, 3, 136, 1024),
                                                (2, 2, 8, 16), (1, 6, 192, 256)])
@pytest.mark.parametrize("x,cache,y", TYPES)
def test_trees(te, gpu_device, heads, group, d, page, x, cache, y):
    _tree(te, gpu_device, LENGTHS, NEW, heads, group, d, page, x, cache, y, seed=d + group)


@pytest.mark.parametrize("heads,group,d,page", [(2, 4, 128, 64), (3, 3, 64, 16), (1, 17, 64, 32), (2, 2, 80, 32), (1, 2, 256, 64), (1, 1, 8, 16)])
@pytest.mark.parametrize("x,cache,y", TYPES[:4])
def test_prompts(te, gpu_device, heads, group, d, page, x, cache, y):
    """From an empty cache and behind one; one token; none."""
    _tree(te, gpu_device, [200, 1, 0, 129, 64, 65], [200, 1, 0, 129, 60, 1], heads, group, d, page, x, cache, y, parents=None, seed=d)


@pytest.mark.parametrize("heads,group,d", [(2, 4, 128), (1, 9, 64), (1, 2, 256), (1, 3, 80)])
@pytest.mark.parametrize("x,cache,y", TYPES[:4])
def test_long_rows_in_chunks(te, gpu_device, heads, group, d, x, cache, y):
    _tree(te, gpu_device, [3000], [5], heads, group, d, 64, x, cache, y, seed=d)
    _tree(te, gpu_device, [2500], [50], heads, group, d, 16, x, cache, y, seed=d + 1)
    _tree(te, gpu_device, [1300, 1, 513, 0, 2049], [33, 1, 13, 0, 2], heads, group, d, 16, x, cache, y, seed=d + 2, layout="sh")


@pytest.mark.parametrize("x,cache,y", TYPES[:4])
def test_a_long_prompt(te, gpu_device, x, cache, y):
    _tree(te, gpu_device, [1111], [1111], 1, 2, 64, 16, x, cache, y, parents=None, seed=1)
    _tree(te, gpu_device, [1700, 30], [300, 30], 1, 4, 128, 64, x, cache, y, parents=None, seed=2)


@pytest.mark.parametrize("n", [1, 2, 3, 8, 16, 31, 32, 33])
def test_as_many_tokens_for_each_row(te, gpu_device, n):
    """Without starts; one token each is the attention of one token."""
    got = _tree(te, gpu_device, [n, 40, 700, 64], [n] * 4, 2, 3, 64, 16, uniform=True, seed=n)
    if n == 1:
        P = Pages([1, 40, 700, 64], 2, 16, 64, F16, 1)
        q = (torch.randn((4, 6, 64), generator=P.g) * 2).half().to(gpu_device)
        k, v, table, lens, _, _ = P.to(gpu_device)
        got = te.tree_attention(q, k, v, table, lens, out_dtype=F32)
        close(got.cpu(), te.paged_attention(q, k, v, table, lens, out_dtype=F32).cpu(), F32, 4e-4 * 5)


@pytest.mark.parametrize("n", [1, 2, 17, 64, 100, 300])
def test_a_chain_of_parents_is_a_prompt(te, gpu_device, n):
    P = Pages([n + 37, n], 2, 16, 64, F16, n)
    q = torch.randn((2 * n, 6, 64), generator=P.g).half().to(gpu_device)
    k, v, table, lens, _, _ = P.to(gpu_device)
    chain = (torch.arange(2 * n) % n - 1).int().to(gpu_device)
    a = te.tree_attention(q, k, v, table, lens, parents=chain)
    assert torch.equal(a, te.tree_attention(q, k, v, table, lens))


def test_parents_that_are_none(te, gpu_device):
    """Itself, a later token, a negative number, one far outside: the token continues the cached tokens."""
    new, lengths = [9, 5], [40, 5]
    parents = torch.tensor([5, 1, -7, 2, 2 ** 31 - 1, 3, -2 ** 31, 6, 9, 0, 0, 1, 4, 99], dtype=torch.int32)
    for y in (F16, F32):
        _tree(te, gpu_device, lengths, new, 2, 2, 64, 16, y=y, parents=parents)


def test_padding(te, gpu_device):
    """Tokens before the first row's and behind the last one's get zeros, whatever they and their memory hold."""
    P = Pages([50, 9], 2, 16, 64, F16, 3)
    starts, k_v = torch.tensor([3, 10, 14], dtype=torch.int32), P.to(gpu_device)[:4]
    for extra in (0, 1, 200):
        for par in (None, torch.tensor([7] * 3 + [-1, 0, 1, 0, 3, 3, 5] + [-1, 0, 0, 2] + [0] * extra, dtype=torch.int32)):
            q = torch.randn((14 + extra, 4, 64), generator=P.g).half()
            q[:3], q[14:] = float("nan"), float("inf")
            out = torch.full(q.shape, 7.0, device=gpu_device)
            te.tree_attention(q.to(gpu_device), *k_v, starts=starts.to(gpu_device), parents=None if par is None else par.to(gpu_device), out=out)
            close(out, ref.tree(q.nan_to_num(0, 0, 0), P, starts, par), F32, 1e-3)
            assert (out[:3] == 0).all() and (out[14:] == 0).all()


def test_slots_that_are_not_there(te, gpu_device):
    """Lengths below the new tokens' number, past the table, past max_len: those tokens get zeros, the others what they see."""
    P = Pages([60, 60, 60], 2, 16, 64, F16, 4, idle=0.0)
    starts = _starts([20, 30, 10])
    for lens, max_len in (([5, 64 + 7, 60], None), ([0, -3, 2 ** 31 - 1], None), ([60, 60, 60], 45), ([60, 60, 60], 0), ([60, 60, 60], 30)):
        for parents in (None, _parents([20, 30, 10], P.g)):
            q = torch.randn((60, 4, 64), generator=P.g).half()
            k, v, table, _, _, _ = P.to(gpu_device)
            got = te.tree_attention(q.to(gpu_device), k, v, table, torch.tensor(lens, dtype=torch.int32, device=gpu_device),
                                    starts=starts.to(gpu_device), parents=None if parents is None else parents.to(gpu_device),
                                    max_len=max_len, out_dtype=F32)
            close(got, ref.tree(q, P, starts, parents, lens=lens, max_len=max_len), F32, 1e-3)


def test_starts_that_are_none(te, gpu_device):
    """Starts outside the tokens or in no order touch nothing outside; the rows that are in order keep their results."""
    P = Pages([30, 20, 40], 1, 16, 64, F16, 5, idle=0.0)
    q = torch.randn((12, 2, 64), generator=P.g).half()
    k, v, table, lens, _, _ = P.to(gpu_device)
    for s in ([-5, 4, 8, 12], [0, 4, 2, 12], [0, 4, 8, 99], [2 ** 31 - 1, 0, 0, 0], [0, 0, 0, 2 ** 31 - 1]):
        got = te.tree_attention(q.to(gpu_device), k, v, table, lens, starts=torch.tensor(s, dtype=torch.int32, device=gpu_device))
        assert got.shape == q.shape and got.isfinite().all()
    s = torch.tensor([0, 4, 8, 99], dtype=torch.int32)
    got = te.tree_attention(q.to(gpu_device), k, v, table, lens, starts=s.to(gpu_device), out_dtype=F32)
    close(got[:8], ref.tree(q, P, torch.tensor([0, 4, 8, 8]))[:8], F32, 1e-3)


@pytest.mark.parametrize("rows,longest", [(63, 90), (65, 700), (200, 300), (700, 40)])
def test_many_rows(te, gpu_device, rows, longest):
    g = torch.Generator().manual_seed(rows)
    new = torch.randint(0, 6, (rows,), generator=g).tolist()
    new[0], new[-1], new[5] = 3, 2, 30
    lengths = [n + int(torch.randint(0, longest, (1,), generator=g)) for n in new]
    lengths[0], lengths[-1] = longest, longest
    _tree(te, gpu_device, lengths, new, 1, 2, 16, 16, F16, F16, F32, seed=rows)
    _tree(te, gpu_device, lengths, new, 1, 2, 16, 16, F16, F16, F16, seed=rows, parents=None)


@pytest.mark.parametrize("idle", [float("inf"), float("-inf"), float("nan"), 65504.0])
def test_reads_nothing_of_idle_memory(te, gpu_device, idle):
    for x, cache, y in TYPES[:3]:
        _tree(te, gpu_device, LENGTHS, NEW, 2, 4, 128, 64, x, cache, y, idle=idle)


def test_strides_and_layouts(te, gpu_device):
    for x, cache, y in TYPES:
        _tree(te, gpu_device, LENGTHS, NEW, 2, 3, 128, 32, x, cache, y, strided=True, layout="sh")
    got = _tree(te, gpu_device, LENGTHS, NEW, 2, 3, 80, 32, strided=True)
    assert got.is_contiguous()


def test_scale_and_max_len(te, gpu_device):
    for max_len in (500, 501, 20000):
        _tree(te, gpu_device, LENGTHS, NEW, 2, 4, 64, 16, F16, F16, F32, max_len=max_len, scale=0.31)


@pytest.mark.parametrize("y", [F16, F32])
def test_peaked_and_flat(te, gpu_device, y):
    """All logits equal; logits far apart in every order (the running maximum moves often), and huge."""
    _tree(te, gpu_device, [777, 33], [40, 3], 1, 4, 128, 16, F16, F16, y, qscale=0.0)
    P = Pages([1500], 1, 16, 64, F16, 1)
    q = torch.ones((50, 2, 64)).half()
    page, slot = P.slots(0, 1500)
    ramp = torch.linspace(-300, 300, 1500)                     # logits 8 x ramp: from -2400 to 2400
    for order in (torch.arange(1500), torch.arange(1499, -1, -1), torch.randperm(1500, generator=P.g)):
        P.k[page, 0, slot] = ramp[order][:, None].expand(-1, 64).half()
        k, v, table, lens, _, _ = P.to(gpu_device)
        for parents in (None, _parents([50], P.g)):
            want = ref.tree(q, P, [0, 50], parents)
            got = te.tree_attention(q.to(gpu_device), k, v, table, lens, parents=None if parents is None else parents.to(gpu_device), out_dtype=y)
            close(got, want, y, 1e-3 * float(P.v.nan_to_num(0).abs().max()))


@pytest.mark.parametrize("size,scale", [(1e7, 1e-8), (1e-9, 1e8), (3e4, 1e-5)])
def test_extreme_queries(te, gpu_device, size, scale):
    """fp32 queries outside f16's range in either direction keep their precision."""
    _tree(te, gpu_device, [200, 31], [20, 31], 2, 4, 128, 16, F32, F16, F32, qscale=size, scale=scale)


def test_infinite_logits_and_nan(te, gpu_device):
    """A key of -inf has no weight; one token's NaN stays within its row and head."""
    P = Pages([100, 50], 2, 16, 64, F16, 2)
    page, slot = P.slots(0, 100)
    P.k[page[40], 0, slot[40]] = float("-inf")
    P.k[page[95], 0, slot[95]] = float("-inf")
    page1, slot1 = P.slots(1, 50)
    P.k[page1[7], 1, slot1[7]] = float("nan")
    q = torch.rand((30, 4, 64), generator=P.g).half() + 0.01
    k, v, table, lens, _, _ = P.to(gpu_device)
    starts = torch.tensor([0, 20, 30], dtype=torch.int32)
    for parents in (None, _parents([20, 10], P.g)):
        want = ref.tree(q, P, starts, parents)
        got = te.tree_attention(q.to(gpu_device), k, v, table, lens, starts=starts.to(gpu_device),
                                parents=None if parents is None else parents.to(gpu_device)).cpu()
        assert got[20:, 2:].isnan().all()
        close(got[:20], want[:20].nan_to_num(0), F16, 3e-3)       # (a token that sees a -inf key alone gives no NaN)
        close(got[20:, :2], want[20:, :2], F16, 3e-3)


@pytest.mark.parametrize("first", [200, 1200])
def test_missing_pages(te, gpu_device, first):
    """Tokens on pages that do not exist count as absent, cached and new ones; where nothing is left, zeros."""
    P = Pages([first, 90, 20], 2, 16, 64, F16, 4)
    P.table[0, 3], P.table[0, 6], P.table[1, 5] = -1, P.pages, 2 ** 31 - 1
    P.table[2] = -5
    new = [40, 30, 7]
    q = torch.randn((77, 6, 64), generator=P.g).half()
    k, v, table, lens, _, _ = P.to(gpu_device)
    for parents in (None, _parents(new, P.g)):
        for y in (F16, F32):
            got = te.tree_attention(q.to(gpu_device), k, v, table, lens, starts=_starts(new).to(gpu_device),
                                    parents=None if parents is None else parents.to(gpu_device), out_dtype=y)
            close(got, ref.tree(q, P, _starts(new), parents), y, 3e-3)
            assert (got[70:] == 0).all()


@pytest.mark.parametrize("length,n", [(300, 20), (1700, 5), (1700, 60)])
def test_shared_pages_and_repeats(te, gpu_device, length, n):
    P = Pages([length, length], 2, 32, 128, F16, 6)
    P.table[1, :5] = P.table[0, :5]
    q = torch.randn((2 * n, 8, 128), generator=P.g).half()
    k, v, table, lens, _, _ = P.to(gpu_device)
    for y in (F16, F32):
        runs = [te.tree_attention(q.to(gpu_device), k, v, table, lens, out_dtype=y) for _ in range(3)]
        close(runs[0], ref.tree(q, P, [0, n, 2 * n]), y, 3e-3)
        assert torch.equal(runs[0], runs[1]) and torch.equal(runs[0], runs[2])


def test_pool_past_32_bit_offsets(te, gpu_device):
    """A pool of more than 2^31 elements, its last pages in use."""
    heads, page, d = 8, 64, 128
    pages = 2 ** 31 // (heads * page * d) + 5
    k, v = (torch.empty((pages, heads, page, d), dtype=F16, device=gpu_device) for _ in range(2))
    small = Pages([150], heads, page, d, F16, 7, spare=0)
    ids = torch.tensor([pages - 1, pages - 3, 0], dtype=torch.int32)
    k[ids.long().to(gpu_device)] = small.k[small.table[0].long()].to(gpu_device)
    v[ids.long().to(gpu_device)] = small.v[small.table[0].long()].to(gpu_device)
    for n in (3, 30):
        q = torch.randn((n, 32, d), generator=small.g).half()
        got = te.tree_attention(q.to(gpu_device), k, v, ids[None].to(gpu_device), small.lens.to(gpu_device))
        close(got, ref.tree(q, small, [0, n]), F16, 3e-3)


def test_workspace_of_the_caller(te, gpu_device):
    P = Pages([3000], 1, 16, 64, F16, 3)
    q = torch.randn((4, 4, 64), generator=P.g).half().to(gpu_device)
    k, v, table, lens, _, _ = P.to(gpu_device)
    ws = torch.full((1 << 24,), 255, dtype=torch.uint8, device=gpu_device)
    out = torch.empty((4, 4, 64), dtype=F32, device=gpu_device)
    got = te.tree_attention(q, k, v, table, lens, workspace=ws, out=out)
    assert got is out and torch.equal(out, te.tree_attention(q, k, v, table, lens, out_dtype=F32))


def test_workspaces_that_do_not_do(te, gpu_device):
    P = Pages([3000], 1, 16, 64, F16, 3)
    q = torch.zeros((4, 4, 64), dtype=F16, device=gpu_device)
    k, v, table, lens, _, _ = P.to(gpu_device)
    for ws, status in ((torch.empty(64, dtype=torch.uint8, device=gpu_device), 10), (torch.empty((1 << 24) + 8, dtype=torch.uint8, device=gpu_device)[8:], 8)):
        with pytest.raises(te.TrellisError) as e:
            te.tree_attention(q, k, v, table, lens, workspace=ws)
        assert e.value.status == status


@pytest.mark.parametrize("group", [129, 300])
@pytest.mark.parametrize("x,cache,y", TYPES[:3])
def test_groups_of_more_heads_than_a_block_holds(te, gpu_device, group, x, cache, y):
    _tree(te, gpu_device, [40, 3, 700], [3, 1, 5], 1, group, 32, 16, x, cache, y, seed=group)
    _tree(te, gpu_device, [40, 9], [7, 9], 1, group, 64, 16, x, cache, y, seed=group, parents=None)


@pytest.mark.parametrize("y", [F16, F32])
def test_starts_in_no_order_of_long_rows(te, gpu_device, y):
    """Rows that are cut into chunks: nothing outside out is touched, and the next call is right."""
    P = Pages([900, 20, 1300], 2, 16, 64, F16, 5, idle=0.0)
    q = torch.randn((12, 4, 64), generator=P.g).half()
    k, v, table, lens, _, _ = P.to(gpu_device)
    for s in ([0, 12, 0, 12], [12, 0, 12, 0], [0, 4, 2, 12], [-5, 4, 8, 12], [0, 4, 8, 99], [2 ** 31 - 1, 0, 0, 0], [5, 5, 5, 5]):
        wide = torch.full((12 + 128, 4, 64), 7.0, dtype=y, device=gpu_device)
        te.tree_attention(q.to(gpu_device), k, v, table, lens, starts=torch.tensor(s, dtype=torch.int32, device=gpu_device), out=wide[64:76])
        torch.cuda.synchronize()
        assert (wide[:64] == 7).all() and (wide[76:] == 7).all() and wide.isfinite().all(), s
    assert (wide[64:76] == 0).all()     # no row has a token
    s = torch.tensor([0, 4, 5, 12], dtype=torch.int32)
    got = te.tree_attention(q.to(gpu_device), k, v, table, lens, starts=s.to(gpu_device), out_dtype=y)
    close(got, ref.tree(q, P, s), y, 3e-3)


@pytest.mark.parametrize("y", [F16, F32])
def test_graphs_and_streams(te, gpu_device, y):
    """Two calls at once on two streams, and replays of a captured call whose rows and chunks change between them, with
    eager calls in between, give what one eager call gives."""
    P = Pages([2000, 700, 64], 2, 16, 64, F16, 8, idle=None)
    k, v, table, lens, _, _ = P.to(gpu_device)
    ints = lambda t: torch.tensor(t, dtype=torch.int32, device=gpu_device)
    starts, parents = ints([0, 20, 25, 40]), _parents([20, 5, 15], P.g).to(gpu_device)
    qs = [torch.randn((40, 8, 64), generator=P.g).half().to(gpu_device) for _ in range(2)]
    call = lambda q, starts=starts, lens=lens: te.tree_attention(q, k, v, table, lens, starts=starts, parents=parents, out_dtype=y)
    eager = [call(q) for q in qs]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(3):
        with torch.cuda.stream(side):
            a = call(qs[0])
        b = call(qs[1])
        torch.cuda.synchronize()
        assert torch.equal(a, eager[0]) and torch.equal(b, eager[1])
    q = qs[0].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call(q)
    for i, (s, n) in enumerate((([0, 20, 25, 40], [2000, 700, 64]), ([0, 1, 40, 40], [40, 700, 0]), ([0, 0, 0, 0], [9, 9, 9]), ([3, 8, 30, 33], [5, 650, 3]))):
        q.copy_(qs[i % 2])
        starts.copy_(ints(s))
        lens.copy_(ints(n))
        graph.replay()
        want = call(qs[i % 2], ints(s), ints(n))
        torch.cuda.synchronize()
        assert torch.equal(out, want), i


def test_writes_count(te, gpu_device):
    P = Pages([40], 2, 16, 64, F16, 7, idle=None)
    k, v, table, lens, _, _ = P.to(gpu_device)
    q, ws = torch.zeros((4, 4, 64), dtype=F16, device=gpu_device), torch.zeros(1 << 20, dtype=torch.uint8, device=gpu_device)
    own = {"q": q, "k": k, "v": v, "table": table, "lens": lens, "out": torch.zeros_like(q), "ws": ws}
    before = {n: t._version for n, t in own.items()}
    te.tree_attention(q, k, v, table, lens, out=own["out"], workspace=ws)
    assert {n for n, t in own.items() if t._version != before[n]} == {"out", "ws"}


def test_refusals(te, gpu_device):
    dev = gpu_device
    P = Pages([20, 3], 2, 16, 64, F16, 0, idle=None)
    k, v, table, lens, _, _ = P.to(dev)
    q, par, st = torch.zeros((4, 4, 64), dtype=F16, device=dev), torch.zeros(4, dtype=torch.int32, device=dev), _starts([2, 2]).to(dev)
    call = lambda q=q, k=k, v=v, table=table, lens=lens, **kw: te.tree_attention(q, k, v, table, lens, **kw)
    bad = [lambda: call(q[:3]), lambda: call(q[..., :32]), lambda: call(q.double()), lambda: call(q[:, :3]), lambda: call(q.cpu()),
           lambda: call(k=k.float(), v=v.float()), lambda: call(v=v[:, :1]), lambda: call(table=table.long()), lambda: call(lens=lens[:1]),
           lambda: call(starts=st[:2]), lambda: call(starts=st.long()), lambda: call(starts=st.cpu()), lambda: call(parents=par[:3]),
           lambda: call(parents=par.float()), lambda: call(out=q[:2]), lambda: call(out=q.double()), lambda: call(max_len=-1),
           lambda: call(q.clone().requires_grad_()), lambda: call(out_dtype=torch.int8), lambda: call(scale="x"), lambda: call(table=None),
           lambda: call(lens=None), lambda: call(table=table[:0], lens=lens[:0]), lambda: call(q[0])]
    for i, f in enumerate(bad):
        with pytest.raises((ValueError, RuntimeError)):
            f()
            pytest.fail(f"call {i} was not refused")
    assert call(q[:0]).shape == (0, 4, 64) and call(q[:0], table=table[:0], lens=lens[:0]).shape == (0, 4, 64)
    assert call(q[:0], starts=_starts([0, 0]).to(dev), parents=par[:0]).shape == (0, 4, 64)
