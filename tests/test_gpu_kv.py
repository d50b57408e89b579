"""append_kv, paged_attention and evict_kv against float64 restatements (serve_ref), at the lengths, pages, head
layouts, strides and masks where they can go wrong.

Tolerances. append: 64 x 2^-24 of a row's largest value before the one rounding (as the norms), 4 more roundings
for the rotation. Attention: a logit of size S carries (d + 3) 2^-24 of sum |q k| (below 40 for these inputs), and
2^-21 of it from q in two f16 terms: at most 2e-4 for d = 256, an error of the weights relative to themselves; out
is a mean of values, so 2e-4 x max |v| (the sums' own roundings are far below that). bf16 results in two terms a
weight: 2^-16 more. Scores are sums of weights, at most one a head: 2e-4 x group plus fp32's rounding of the sum."""
import pytest
import torch

import serve_ref as ref

pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
FP = 80 * 2.0 ** -24
LENGTHS = [0, 1, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 129, 500]


# ------------------------------------------------------------------ append


def _append(te, dev, new, before, heads, group, d, page, x, cache, qdt, rot, normed, positions=None, layout="hs", seed=0,
            fused=False):
    lengths = [a + b for a, b in zip(before, new)]
    P = ref.Pages(lengths, heads, page, d, cache, seed, idle=None, layout=layout)
    g, t, hq = P.g, sum(new), heads * group
    if fused:      # slices of one buffer, an element off alignment
        buf = torch.randn((t, (hq + 2 * heads) * d + 1), generator=g).to(x)
        parts = lambda u: [u[:, 1:][:, i * d:j * d].unflatten(1, (-1, d)) for i, j in ((0, hq), (hq, hq + heads), (hq + heads, hq + 2 * heads))]
        q, k, v = parts(buf)
        dq, dk, dv = parts(buf.to(dev))
    else:
        q, k, v = (torch.randn((t, h, d), generator=g).to(x) for h in (hq, heads, heads))
        dq, dk, dv = q.to(dev), k.to(dev), v.to(dev)
    qw, kw = (torch.rand(d, generator=g) + 0.5, torch.rand(d, generator=g) + 0.5) if normed else (None, None)
    table = torch.rand((max(lengths) + 40, rot // 2), generator=g) * 6 if rot else None
    cos, sin = (table.cos(), table.sin()) if rot else (None, None)
    starts = None if all(n == 1 for n in new) and len(new) == t else torch.tensor([sum(new[:i]) for i in range(len(new) + 1)], dtype=torch.int32)
    dk_p, dv_p, dt, dl, ds, dpos = P.to(dev)
    up = lambda u: None if u is None else u.to(dev)
    got = te.append_kv(dq, dk, dv, dk_p, dv_p, dt, dl, starts=up(starts), positions=up(positions), q_norm=up(qw),
                       k_norm=up(kw), eps=1e-5, cos=up(cos), sin=up(sin), scores=ds, pos=dpos, q_dtype=qdt)
    want_q = torch.zeros((t, hq, d), dtype=torch.float64)
    K, V, S, Z = P.k.double().clone(), P.v.double().clone(), P.scores.clone(), P.pos.clone()
    i = 0
    for b, n in enumerate(new):
        for j in range(n):
            slot = before[b] + j
            at = slot if positions is None else int(positions[i])
            qq, kk = q[i].double(), k[i].double()
            if normed:
                qq, kk = ref.rms(qq, qw, 1e-5), ref.rms(kk, kw, 1e-5)
            if rot:
                c, s = (cos[at].double(), sin[at].double()) if 0 <= at < cos.shape[0] else (torch.full((rot // 2,), float("nan")),) * 2
                qq, kk = ref.rotate(qq, c, s), ref.rotate(kk, c, s)
            want_q[i] = qq
            pg, sl = int(P.table[b, slot // page]), slot % page
            K[pg, :, sl], V[pg, :, sl], S[pg, :, sl], Z[pg, :, sl] = kk, v[i].double(), 0.0, at
            i += 1
    ref.close(got, want_q, qdt, FP * want_q.abs().nan_to_num(0).amax(-1, keepdim=True), "q'")
    ref.close(dk_p, K, cache, FP * K.abs().nan_to_num(0).amax(-1, keepdim=True), "k")
    ref.close(dv_p, V, cache, 0.0, "v")
    assert torch.equal(ds.cpu(), S) and torch.equal(dpos.cpu(), Z)


@pytest.mark.parametrize("heads,group,d,rot,page", [(8, 4, 128, 128, 64), (3, 3, 64, 64, 16), (1, 1, 8, 0, 16), (2, 2, 80, 80, 32),
                                                    (1, 16, 96, 32, 128), (2, 1, 256, 256, 16), (1, 2, 136, 64, 1024), (2, 3, 24, 16, 16)])
@pytest.mark.parametrize("x,cache,qdt", [(F32, F16, F16), (BF16, BF16, BF16), (F16, F16, F32), (F16, BF16, BF16), (BF16, F16, F32)])
def test_append(te, gpu_device, heads, group, d, rot, page, x, cache, qdt):
    _append(te, gpu_device, [1] * 5, [0, 1, 15, 16, 40], heads, group, d, page, x, cache, qdt, rot, True, seed=d)
    _append(te, gpu_device, [0, 3, 1, 0, 70, 0], [4, 0, 31, 0, 15, 0], heads, group, d, page, x, cache, qdt, rot, False, seed=d + 1)


def test_append_many_rows(te, gpu_device):
    """More rows than a wave looks at at once, most of them with few tokens or none."""
    g = torch.Generator().manual_seed(11)
    for rows in (63, 64, 65, 200):
        new = torch.randint(0, 4, (rows,), generator=g).tolist()
        new[0], new[-1] = 0, 2
        before = torch.randint(0, 40, (rows,), generator=g).tolist()
        _append(te, gpu_device, new, before, 2, 2, 64, 16, F16, F16, F16, 64, True, seed=rows)


def test_append_layouts(te, gpu_device):
    for x in (F32, F16):
        _append(te, gpu_device, [2, 0, 19], [5, 3, 7], 2, 4, 128, 16, x, F16, F16, 128, True, fused=True)
        _append(te, gpu_device, [2, 0, 19], [5, 3, 7], 3, 1, 64, 32, x, BF16, F32, 32, True, layout="sh")


def test_append_positions_of_an_evicted_cache(te, gpu_device):
    """Positions apart from the slots; one that the rotary table does not hold makes NaN of its own token alone."""
    _append(te, gpu_device, [1, 1, 1], [3, 9, 30], 2, 2, 64, 16, F32, F16, F16, 64, True, positions=torch.tensor([60, 0, 33], dtype=torch.int32))
    _append(te, gpu_device, [1, 1], [3, 9], 2, 2, 64, 16, F32, F16, F32, 64, True, positions=torch.tensor([99, 5], dtype=torch.int32))
    _append(te, gpu_device, [1, 1], [3, 9], 2, 2, 64, 16, F32, F16, F32, 64, True, positions=torch.tensor([4, -1], dtype=torch.int32))


def test_append_padding_writes_nothing(te, gpu_device):
    """Tokens past the last row, of an empty row, past the table and on pages that do not exist are not stored."""
    P = ref.Pages([5, 20, 9, 0], 2, 16, 64, F16, 3, idle=None)
    P.table[2, 0] = P.pages + 7          # no page
    lens = torch.tensor([5, P.width * 16 + 1, 9, 0], dtype=torch.int32)
    k, v, table, _, scores, pos = P.to(gpu_device)
    t = torch.randn((6, 2, 64), device=gpu_device)
    starts = torch.tensor([0, 1, 2, 3, 4], dtype=torch.int32, device=gpu_device)
    got = te.append_kv(t, t, t, k, v, table, lens.to(gpu_device), starts=starts, scores=scores, pos=pos).cpu()
    K = P.k.clone()
    K[P.table[0, 0].long(), :, 4] = t[0].half().cpu()
    assert torch.equal(k.cpu(), K)
    assert torch.equal(got[0], t[0].cpu()) and (got[1:] == 0).all()
    assert int((pos.cpu() != P.pos).sum()) <= 2 and int((scores.cpu() != P.scores).sum()) == 2


# ------------------------------------------------------------------ attention


def _attend(te, dev, lengths, heads, group, d, page, x, cache, y, seed=0, layout="hs", idle=float("nan"), scale=None,
            scored=True, max_len=None, strided=False, qscale=2.0):
    P = ref.Pages(lengths, heads, page, d, cache, seed, idle=idle, layout=layout)
    q = (torch.randn((len(lengths), heads * group, d), generator=P.g) * qscale).to(x)
    k, v, table, lens, scores, _ = P.to(dev)
    dq = q.to(dev)
    if strided:    # heads of a wider buffer, rows an odd distance apart
        wide = torch.zeros((len(lengths), heads * group * d + 3), dtype=x, device=dev)
        wide[:, 1:-2] = dq.flatten(1)
        dq = wide[:, 1:-2].unflatten(1, (-1, d))
    got = te.paged_attention(dq, k, v, table, lens, scale=scale, max_len=max_len, scores=scores if scored else None, out_dtype=y)
    seen = None if max_len is None else [min(n, max_len) for n in lengths]
    want, want_scores = ref.attend(q, P, scale, seen)
    top = float(P.v.double().nan_to_num(0, 0, 0).abs().max())
    bf = 2.0 ** -16 if cache == BF16 else 0.0
    ref.close(got, want, y, (2e-4 + bf) * top, "out")
    if scored:
        err = (scores.double().cpu() - want_scores).abs()
        assert float((err - 2e-4 * group - 2 ** -23 * want_scores).max()) <= 0, float(err.max())
    return got


@pytest.mark.parametrize("heads,group,d,page", [(8, 4, 128, 64), (3, 3, 64, 16), (2, 1, 128, 16), (1, 16, 128, 32), (1, 17, 64, 16),
                                                (2, 40, 32, 128), (2, 2, 80, 32), (1, 5, 96, 16), (2, 4, 256, 64), (1, 3, 136, 1024),
                                                (2, 2, 8, 16), (1, 6, 192, 256)])
@pytest.mark.parametrize("x,cache,y", [(F16, F16, F16), (BF16, BF16, BF16), (F32, F16, F32), (F32, BF16, F32), (BF16, F16, BF16), (F16, BF16, F16)])
def test_attention(te, gpu_device, heads, group, d, page, x, cache, y):
    _attend(te, gpu_device, LENGTHS, heads, group, d, page, x, cache, y, seed=d + group)


@pytest.mark.parametrize("heads,group,d,page", [(8, 4, 128, 64), (3, 3, 64, 16), (1, 17, 64, 32), (2, 40, 32, 128), (2, 2, 80, 32),
                                                (1, 5, 96, 16), (2, 2, 256, 64), (1, 3, 136, 1024), (1, 1, 8, 16)])
@pytest.mark.parametrize("x,cache,y", [(F16, F16, F16), (BF16, BF16, BF16), (F32, F16, F32), (F32, BF16, F32)])
def test_attention_chunks_of_uneven_rows(te, gpu_device, heads, group, d, page, x, cache, y):
    """Rows in several chunks (longer than 512 tokens), some in one, some empty."""
    _attend(te, gpu_device, [0, 1300, 1, 513, 127, 0, 900], heads, group, d, page, x, cache, y, seed=d)
    _attend(te, gpu_device, [1, 2049, 0], heads, group, d, page, x, cache, y, seed=d, scored=False, layout="sh")


@pytest.mark.parametrize("rows,longest", [(65, 1400), (200, 900), (512, 600), (513, 600), (700, 40)])
def test_attention_many_rows(te, gpu_device, rows, longest):
    """More rows than a wave looks at at once, and more than are split at all."""
    g = torch.Generator().manual_seed(rows)
    lengths = torch.randint(0, longest, (rows,), generator=g).tolist()
    lengths[0], lengths[63], lengths[-1] = longest, 0, longest
    _attend(te, gpu_device, lengths, 1, 2, 16, 16, F16, F16, F32, seed=rows)
    _attend(te, gpu_device, [0] * (rows - 1) + [longest], 2, 1, 8, 16, F16, F16, F16, seed=rows)


@pytest.mark.parametrize("length", [1, 2, 100, 128, 129, 1000, 4097, 9001])
def test_attention_split_over_one_row(te, gpu_device, length):
    """One row: every split of the length, and its join."""
    for heads, group, d in ((1, 4, 128), (2, 20, 64)):
        _attend(te, gpu_device, [length], heads, group, d, 16, F16, F16, F32, seed=length)


def test_attention_many_ragged_rows(te, gpu_device):
    g = torch.Generator().manual_seed(5)
    lengths = torch.randint(0, 700, (70,), generator=g).tolist()
    _attend(te, gpu_device, lengths, 2, 4, 64, 32, F16, F16, F16)
    _attend(te, gpu_device, [0] * 70, 2, 4, 64, 32, F16, F16, F16)
    _attend(te, gpu_device, [0, 3000, 0, 1], 2, 4, 128, 64, BF16, BF16, F32)


@pytest.mark.parametrize("idle", [float("inf"), float("-inf"), float("nan"), 65504.0])
def test_attention_reads_nothing_of_idle_memory(te, gpu_device, idle):
    _attend(te, gpu_device, LENGTHS, 2, 4, 128, 64, F16, F16, F16, idle=idle)
    _attend(te, gpu_device, LENGTHS, 2, 4, 128, 64, F32, F16, F32, idle=idle)


def test_attention_strides_and_layouts(te, gpu_device):
    for x in (F32, F16, BF16):
        _attend(te, gpu_device, LENGTHS, 2, 3, 128, 32, x, F16, F16, strided=True, layout="sh")
    got = _attend(te, gpu_device, LENGTHS, 2, 3, 80, 32, F16, F16, F16, strided=True)
    assert got.is_contiguous()


def test_attention_max_len_and_scale(te, gpu_device):
    """Tokens past max_len are not seen; a longer max_len than any row changes nothing but the split."""
    for max_len in (0, 1, 40, 64, 511, 20000):
        _attend(te, gpu_device, LENGTHS, 2, 4, 64, 16, F16, F16, F32, max_len=max_len, scale=0.31)


def test_attention_peaked_and_flat(te, gpu_device):
    """Logits far apart (one weight takes all, the running maximum moves often), all equal, and huge."""
    _attend(te, gpu_device, [777, 33], 1, 4, 128, 16, F16, F16, F16, qscale=0.0)
    P = ref.Pages([1500], 1, 16, 64, F16, 1)
    q = torch.ones((1, 2, 64)).half()
    page, slot = P.slots(0, 1500)
    ramp = torch.linspace(-300, 300, 1500)                     # logits 8 x ramp: from -2400 to 2400
    for order in (torch.arange(1500), torch.arange(1499, -1, -1), torch.randperm(1500, generator=P.g)):
        P.k[page, 0, slot] = ramp[order][:, None].expand(-1, 64).half()
        k, v, table, lens, _, _ = P.to(gpu_device)
        for y in (F16, F32):
            want, _ = ref.attend(q, P)
            ref.close(te.paged_attention(q.to(gpu_device), k, v, table, lens, out_dtype=y), want, y, 1e-3 * float(P.v.nan_to_num(0).abs().max()))


def test_attention_extreme_queries(te, gpu_device):
    """fp32 queries outside f16's range in either direction keep their precision (they are scaled by a power of 2)."""
    for size, scale in ((1e7, 1e-8), (1e-9, 1e8), (3e4, 1e-5)):
        _attend(te, gpu_device, [200, 31], 2, 4, 128, 16, F32, F16, F32, qscale=size, scale=scale)


def test_attention_infinite_logits(te, gpu_device):
    """A key of -inf has no weight, and one token's NaN makes its own row's heads NaN, nothing else."""
    P = ref.Pages([100, 50], 2, 16, 64, F16, 2)
    page, slot = P.slots(0, 100)
    P.k[page[40], 0, slot[40]] = float("-inf")
    page1, slot1 = P.slots(1, 50)
    P.k[page1[7], 1, slot1[7]] = float("nan")
    q = torch.rand((2, 4, 64), generator=P.g).half() + 0.01
    k, v, table, lens, _, _ = P.to(gpu_device)
    got = te.paged_attention(q.to(gpu_device), k, v, table, lens).cpu()
    want, _ = ref.attend(q, P)
    assert got[1, 2:].isnan().all()
    ref.close(got[0], want[0], F16, 1e-3)
    ref.close(got[1, :2], want[1, :2], F16, 1e-3)


@pytest.mark.parametrize("first", [200, 1200])
def test_attention_missing_pages(te, gpu_device, first):
    """Tokens on pages that do not exist count as absent; a row of only such tokens gives zeros."""
    P = ref.Pages([first, 90, 20], 2, 16, 64, F16, 4)
    P.table[0, 3], P.table[0, 6], P.table[1, 5] = -1, P.pages, 2 ** 31 - 1
    P.table[2] = -5
    q = torch.randn((3, 6, 64), generator=P.g).half()
    k, v, table, lens, scores, _ = P.to(gpu_device)
    got = te.paged_attention(q.to(gpu_device), k, v, table, lens, scores=scores, out_dtype=F32)
    want, want_scores = ref.attend(q, P)
    ref.close(got, want, F32, 1e-3)
    assert float((scores.double().cpu() - want_scores).abs().max()) < 1e-3 and (got[2] == 0).all()


@pytest.mark.parametrize("length", [300, 1700])
def test_attention_shared_pages_and_repeats(te, gpu_device, length):
    """Rows may share pages (a common prefix) without scores; the same call twice is bit-identical."""
    P = ref.Pages([length, length], 2, 32, 128, F16, 6)
    P.table[1, :5] = P.table[0, :5]
    q = torch.randn((2, 8, 128), generator=P.g).half()
    k, v, table, lens, _, _ = P.to(gpu_device)
    runs = [te.paged_attention(q.to(gpu_device), k, v, table, lens, out_dtype=F32) for _ in range(3)]
    ref.close(runs[0], ref.attend(q, P)[0], F32, 1e-3)
    assert torch.equal(runs[0], runs[1]) and torch.equal(runs[0], runs[2])


def test_attention_pool_past_32_bit_offsets(te, gpu_device):
    """A pool of more than 2^31 elements, its last pages in use."""
    heads, page, d = 8, 64, 128
    pages = 2 ** 31 // (heads * page * d) + 5
    k, v = (torch.empty((pages, heads, page, d), dtype=F16, device=gpu_device) for _ in range(2))
    small = ref.Pages([150], heads, page, d, F16, 7, spare=0)
    ids = torch.tensor([pages - 1, pages - 3, 0], dtype=torch.int32)
    k[ids.long().to(gpu_device)] = small.k[small.table[0].long()].to(gpu_device)
    v[ids.long().to(gpu_device)] = small.v[small.table[0].long()].to(gpu_device)
    q = torch.randn((1, 32, d), generator=small.g).half()
    lens = small.lens.to(gpu_device)
    got = te.paged_attention(q.to(gpu_device), k, v, ids[None].to(gpu_device), lens)
    ref.close(got, ref.attend(q, small)[0], F16, 1e-3)
    new = torch.randn((1, heads, d), generator=small.g).half().to(gpu_device)
    te.append_kv(q.to(gpu_device), new, new, k, v, ids[None].to(gpu_device), torch.tensor([65], dtype=torch.int32, device=gpu_device))
    assert torch.equal(k[pages - 3, :, 0], new[0]) and torch.equal(v[pages - 3, :, 0], new[0])


# ------------------------------------------------------------------ eviction


def _evict(te, dev, lengths, keep, recent, heads=2, page=16, d=64, dtype=F16, seed=0, values="spread", apart=False, next_pos=None,
           layout="hs", max_len=None):
    P = ref.Pages(lengths, heads, page, d, dtype, seed, layout=layout)
    g = P.g
    for b, n in enumerate(lengths):
        pg, sl = P.slots(b, n)
        for h in range(heads):
            s = torch.rand(n, generator=g) ** 4 * 30
            if values == "ties":
                s = torch.randint(0, 3, (n,), generator=g).float()
            elif values == "equal":
                s = torch.zeros(n)
            elif values == "odd":
                s = torch.randn(n, generator=g)
                s[::7] = float("inf")
                s[3::11] = float("-inf")
                s[5::13] = float("nan")
                s[6::9] = -0.0
                s[2::9] = 0.0
            P.scores[pg, h, sl] = s
            P.pos[pg, h, sl] = (torch.randperm(n, generator=g) if next_pos else torch.arange(n)).int() + (next_pos[b] - n if next_pos else 0)
    k, v, table, lens, scores, pos = P.to(dev)
    out = None
    if apart:      # fresh pages behind the pool's
        more = -(-keep // page) * len(lengths)
        grow = lambda t: torch.cat([t, t[:1].expand(more, *t.shape[1:])])
        P.k, P.v, P.scores, P.pos = (grow(t) for t in (P.k, P.v, P.scores, P.pos))
        k, v, table, lens, scores, pos = P.to(dev)
        out = (P.pages + torch.randperm(more, generator=g)).int().view(len(lengths), -1)
        P.pages += more
    got = te.evict_kv(k, v, scores, pos, table, lens, keep, recent, max_len=max_len, out_table=None if out is None else out.to(dev),
                      next_pos=None if next_pos is None else torch.tensor(next_pos, dtype=torch.int32, device=dev))
    planes, want = ref.evict(P, keep, recent, next_pos, out)
    assert got.tolist() == want and lens.tolist() == lengths
    for name, a, b in zip(("k", "v", "scores", "pos"), (k, v, scores, pos), planes):
        a, b = a.cpu(), b
        assert torch.equal(torch.nan_to_num(a, -1.0), torch.nan_to_num(b, -1.0)) and torch.equal(a.isnan(), b.isnan()), name


@pytest.mark.parametrize("values", ["spread", "ties", "equal", "odd"])
@pytest.mark.parametrize("apart", [False, True])
@pytest.mark.parametrize("keep,recent", [(1, 0), (1, 1), (16, 3), (33, 33), (64, 10), (200, 0), (1000, 7)])
def test_evict(te, gpu_device, values, apart, keep, recent):
    _evict(te, gpu_device, [0, 1, 16, 17, 33, 34, 64, 65, 201, 333], keep, recent, values=values, apart=apart, seed=keep)


@pytest.mark.parametrize("values", ["spread", "ties", "equal"])
def test_evict_very_long_rows(te, gpu_device, values):
    """More tokens than the selection holds at once (32768), and the last lengths that it does."""
    _evict(te, gpu_device, [33000], 20000, 100, heads=1, d=8, page=1024, values=values)
    _evict(te, gpu_device, [33000, 70000], 3000, 0, heads=1, d=8, page=1024, values=values, apart=True)
    _evict(te, gpu_device, [32768, 16385, 16384, 4097, 4096, 2048], 2040, 7, heads=1, d=8, page=1024, values=values)
    _evict(te, gpu_device, [70000], 69990, 9, heads=1, d=8, page=1024, values=values)


@pytest.mark.parametrize("values", ["spread", "ties", "odd"])
def test_evict_long_rows(te, gpu_device, values):
    _evict(te, gpu_device, [5000, 2049, 1024], 1024, 100, heads=1, d=8, values=values)
    _evict(te, gpu_device, [5000, 2049, 1024], 700, 700, heads=1, d=8, values=values, apart=True)
    _evict(te, gpu_device, [1025, 1030], 1024, 128, heads=1, d=8, values=values)


def test_evict_shapes(te, gpu_device):
    for heads, page, d, dtype, layout in ((3, 64, 128, BF16, "hs"), (1, 128, 256, F16, "sh"), (2, 32, 80, F16, "sh"), (1, 1024, 136, BF16, "hs")):
        _evict(te, gpu_device, [70, 41, 0, 300], 40, 9, heads=heads, page=page, d=d, dtype=dtype, layout=layout)
        _evict(te, gpu_device, [70, 41, 0, 300], 40, 9, heads=heads, page=page, d=d, dtype=dtype, apart=True)


def test_evict_after_an_eviction(te, gpu_device):
    """Positions in no order and ahead of the slots, as an earlier eviction leaves them."""
    _evict(te, gpu_device, [70, 41, 8], 40, 12, next_pos=[900, 41, 30])
    _evict(te, gpu_device, [70, 41, 8], 40, 0, next_pos=[900, 41, 30], values="ties")


def test_evict_more_recent_than_kept_places(te, gpu_device):
    """Every token recent (positions past next_pos): the lowest slots stay."""
    _evict(te, gpu_device, [70], 40, 40, next_pos=[10])


def test_evict_max_len_bounds_what_is_seen(te, gpu_device):
    P = ref.Pages([100], 1, 16, 8, F16, 0, idle=None)
    k, v, table, lens, scores, pos = P.to(gpu_device)
    assert te.evict_kv(k, v, scores, pos, table, lens, 30, 0, max_len=20).tolist() == [20]
    assert torch.equal(k.cpu(), P.k) and torch.equal(scores.cpu(), P.scores)


# ------------------------------------------------------------------ together


@pytest.mark.parametrize("longest,keep", [(100, 50), (1400, 1000)])
def test_steps_in_a_graph_and_on_a_stream(te, gpu_device, longest, keep):
    """append, attention with scores, eviction of one decode step captured in a HIP graph: every replay, with eager
    work between, equals the eager step on a copy of the same state."""
    dev = gpu_device
    P = ref.Pages([60, 33, 1] if longest <= 512 else [longest - 40, 700, 1], 2, 16, 64, F16, 9, idle=0.0, room=40)
    state = P.to(dev)
    twin = [t.clone() for t in state]
    g = torch.Generator(device=dev).manual_seed(1)
    x = [torch.zeros((3, h, 64), dtype=F16, device=dev) for h in (4, 2, 2)]

    def step(s, x):
        k, v, table, lens, scores, pos = s
        lens.add_(1)
        q = te.append_kv(*x, k, v, table, lens, scores=scores, pos=pos)
        out = te.paged_attention(q, k, v, table, lens, scores=scores, max_len=longest, out_dtype=F32)
        lens.copy_(te.evict_kv(k, v, scores, pos, table, lens, keep, 5, max_len=longest))
        return out

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        warm = [t.clone() for t in state]
        step(warm, x)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(state, x)
    for i in range(4):
        fresh = [torch.randn(t.shape, generator=g, device=dev, dtype=F16) for t in x]
        for t, f in zip(x, fresh):
            t.copy_(f)
        graph.replay()
        want = step(twin, fresh)
        torch.cuda.synchronize()
        assert torch.equal(out, want), i
        for a, b in zip(state, twin):
            assert torch.equal(a, b), i


def test_workspace_of_the_caller(te, gpu_device):
    P = ref.Pages([3000], 1, 16, 64, F16, 3)
    q = torch.randn((1, 4, 64), generator=P.g).half().to(gpu_device)
    k, v, table, lens, _, _ = P.to(gpu_device)
    ws = torch.full((1 << 22,), 255, dtype=torch.uint8, device=gpu_device)
    out = torch.empty((1, 4, 64), dtype=F32, device=gpu_device)
    got = te.paged_attention(q, k, v, table, lens, workspace=ws, out=out)
    assert got is out and torch.equal(out, te.paged_attention(q, k, v, table, lens, out_dtype=F32))
    with pytest.raises(te.TrellisError) as e:
        te.paged_attention(q, k, v, table, lens, workspace=ws[:256])
    assert e.value.status == 10


def test_paged_cache_and_the_example(te, gpu_device):
    """A small decoder through its blocks for some tokens against plain float64 torch; with a budget, the cached
    lengths stay within it and the outputs are finite. f16 activations round at every linear: 2e-2."""
    import importlib.util
    import os
    spec = importlib.util.spec_from_file_location("decode_block", os.path.join(os.path.dirname(os.path.dirname(__file__)), "examples", "decode_block.py"))
    ex = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(ex)
    g = torch.Generator(device=gpu_device).manual_seed(2)
    h = [torch.randn((3, 128), generator=g, device=gpu_device) for _ in range(20)]
    dec = ex.Decoder(2, 128, 256, 4, 2, 64, 3, 32, page_size=16)
    past = {}
    for x in h:
        got, want = dec.step(x), ex.reference_step(dec, x, past)
        assert float((got - want).norm() / want.norm()) < 2e-2
    dec = ex.Decoder(2, 128, 256, 4, 2, 64, 3, 32, budget=8, recent=4, page_size=16)
    for x in h:
        y = dec.step(x)
    assert dec.cache.lengths == [8, 8, 8] and dec.cache.seen == [20, 20, 20]
    assert dec.cache.lens.tolist() == [8, 8, 8] and y.isfinite().all()


# ------------------------------------------------------------------ refusals


def test_refusals(te, gpu_device):
    dev = gpu_device
    P = ref.Pages([20, 3], 2, 16, 64, F16, 0, idle=None)
    k, v, table, lens, scores, pos = P.to(dev)
    q, t = torch.zeros((2, 4, 64), dtype=F16, device=dev), torch.zeros((2, 2, 64), dtype=F16, device=dev)
    w, c = torch.ones(64, device=dev), torch.ones((9, 32), device=dev)
    att = lambda q=q, k=k, v=v, table=table, lens=lens, **kw: te.paged_attention(q, k, v, table, lens, **kw)
    app = lambda q=q, kk=t, vv=t, table=table, lens=lens, **kw: te.append_kv(q, kk, vv, k, v, table, lens, **kw)
    ev = lambda keep=4, recent=1, table=table, **kw: te.evict_kv(k, v, scores, pos, table, lens, keep, recent, **kw)
    bad = [lambda: att(q[:1]), lambda: att(q[..., :32]), lambda: att(q.double()), lambda: att(q[:, :3]), lambda: att(q.cpu()),
           lambda: att(k=k.float(), v=v.float()), lambda: att(v=v[:, :1]), lambda: att(v=v.bfloat16()), lambda: att(table=table.long()),
           lambda: att(table=table.cpu()), lambda: att(lens=lens.long()), lambda: att(lens=lens[:1]), lambda: att(scores=scores.half()),
           lambda: att(scores=scores[:-1]), lambda: att(out=q[:1]), lambda: att(out=q.double()), lambda: att(max_len=-1),
           lambda: att(k=k[..., :60], v=v[..., :60], q=q[..., :60]), lambda: att(k=k[:, :, :8], v=v[:, :, :8]),
           lambda: att(k=k[:, :, :, 1:57], v=v[:, :, :, 1:57], q=q[..., :56].contiguous()), lambda: att(q.clone().requires_grad_()),
           lambda: app(kk=t[:1]), lambda: app(kk=t.float()), lambda: app(q_norm=w), lambda: app(q_norm=w, k_norm=w[:32]),
           lambda: app(cos=c), lambda: app(cos=c, sin=c[:4]), lambda: app(cos=c[:, :12], sin=c[:, :12]),
           lambda: app(cos=torch.ones((9, 40), device=dev), sin=torch.ones((9, 40), device=dev)), lambda: app(cos=c.half(), sin=c.half()),
           lambda: app(starts=lens), lambda: app(positions=lens[:1]), lambda: app(q[:1], t[:1], t[:1]), lambda: app(q_dtype=torch.int8),
           lambda: app(q=q[:, :3]), lambda: ev(keep=0, recent=0), lambda: ev(recent=5), lambda: ev(recent=-1), lambda: ev(out_table=table[:1]),
           lambda: ev(out_table=table.long()), lambda: ev(next_pos=lens.long()), lambda: te.evict_kv(k, v, None, pos, table, lens, 4, 1),
           lambda: te.evict_kv(k, v, scores, None, table, lens, 4, 1)]
    for i, f in enumerate(bad):
        with pytest.raises((ValueError, RuntimeError)):
            f()
            pytest.fail(f"call {i} was not refused")
    # empty batches are no error
    assert att(q[:0], table=table[:0], lens=lens[:0]).shape == (0, 4, 64)
    assert app(q[:0], t[:0], t[:0], table=table[:0], lens=lens[:0]).shape == (0, 4, 64)
    none = torch.zeros(3, dtype=torch.int32, device=dev)
    assert app(q[:0], t[:0], t[:0], starts=none).shape == (0, 4, 64)
