"""Prompts, drafts and beams together on a GPU: PagedKVCache's attend_new, keep and reorder with tree_attention and
beam_select, against contiguous float64 caches; a step of them in a captured graph; the examples.

Tolerances: the attention's of test_gpu_tree."""
import importlib.util
import os
import random

import pytest
import torch

import search_ref as ref
import serve_ref

pytestmark = pytest.mark.gpu
F16, F32 = torch.float16, torch.float32


def _example(name):
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", name + ".py")
    spec = importlib.util.spec_from_file_location(name, path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


class Twin:
    """The same sequences as lists of float64 keys and values, one list a row."""

    def __init__(self, rows):
        self.kv = [[] for _ in range(rows)]

    def attend(self, q, counts, parents):
        """Of the rows' last counts[b] tokens, as PagedKVCache.attend_new."""
        out, t = torch.zeros(q.shape, dtype=torch.float64), 0
        for b, n in enumerate(counts):
            base = len(self.kv[b]) - n
            for i, line in enumerate(ref.ancestors(None if parents is None else parents[t:t + n], n)):
                seen = self.kv[b][:base] + [self.kv[b][base + j] for j in sorted(line)]
                k, v = (torch.stack([s[m] for s in seen]) for m in (0, 1))        # [n, heads, d]
                group = q.shape[1] // k.shape[1]
                k, v = k.repeat_interleave(group, 1), v.repeat_interleave(group, 1)
                p = torch.softmax((k * q[t + i].double()).sum(-1) * q.shape[-1] ** -0.5, 0)
                out[t + i] = (p[..., None] * v).sum(0)
            t += n
        return out


@pytest.mark.parametrize("evictable", [False, True])
@pytest.mark.parametrize("page", [16, 64])
def test_random_steps(te, gpu_device, evictable, page):
    """Rows that take prompts, drafts of which some stay, fork, and end: every attention equals the twin's."""
    rng, rows, heads, d = random.Random(page), 4, 2, 64
    g = torch.Generator().manual_seed(page)
    cache = te.PagedKVCache(2, heads, d, rows=rows, max_len=400, pages=60, page_size=page, device=gpu_device, evictable=evictable)
    twins = [Twin(rows), Twin(rows)]
    for step in range(40):
        counts = [rng.choice([0, 1, 1, 5, 20]) if len(twins[0].kv[b]) < 300 else 0 for b in range(rows)]
        if step % 5 == 4:
            counts = [1] * rows
        n, drafts = sum(counts), step % 2 == 0
        if n == 0:
            continue
        parents, depths = None, None
        if drafts:
            parents, depths = [], []
            for c in counts:
                one = []
                for i in range(c):
                    p = rng.randint(max(-1, i - 3), i - 1) if i else -1
                    one.append(0 if p < 0 else one[p] + 1)
                    parents.append(p)
                depths += one
        cache.grow(counts, depths)
        assert not drafts or cache._positions.tolist() == [s - max(one, default=-1) - 1 + x for s, one in zip(
            cache.seen, [depths[sum(counts[:b]):sum(counts[:b + 1])] for b in range(rows)]) for x in one]
        for layer, twin in enumerate(twins):
            q, k, v = (torch.randn((n, h, d), generator=g).half() for h in (2 * heads, heads, heads))
            got = cache.append(layer, *(t.to(gpu_device) for t in (q, k, v)))
            assert torch.equal(got.cpu(), q)
            t = 0
            for b, c in enumerate(counts):
                twin.kv[b] += [(k[t + i].double(), v[t + i].double()) for i in range(c)]
                t += c
            out = cache.attend_new(layer, got, parents=None if parents is None else torch.tensor(parents, dtype=torch.int32, device=gpu_device), out_dtype=F32)
            serve_ref.close(out, twin.attend(q, counts, parents), F32, 2e-4 * 5, f"step {step}, layer {layer}")
        if drafts:
            paths, t = [], 0
            for c in counts:      # a line of the tree from a root
                path = []
                for i in range(c):
                    if parents[t + i] == (path[-1] if path else -1) and rng.random() < 0.8:
                        path.append(i)
                paths.append(path)
                t += c
            cache.keep(paths)
            for twin in twins:
                for b, (c, path) in enumerate(zip(counts, paths)):
                    base = len(twin.kv[b]) - c
                    twin.kv[b] = twin.kv[b][:base] + [twin.kv[b][base + i] for i in path]
        if step % 3 == 2:
            new = [rng.randrange(rows) for _ in range(rows)]
            cache.reorder(new)
            for twin in twins:
                twin.kv = [list(twin.kv[p]) for p in new]
        if step % 7 == 6:
            row = rng.randrange(rows)
            cache.release(row)
            for twin in twins:
                twin.kv[row] = []
        assert cache.lengths == [len(kv) for kv in twins[0].kv] == cache.lens.tolist()


def test_a_waiting_rows_scores_follow_it(te, gpu_device):
    """An evictable cache's rows that fork take their scores and positions with them."""
    g = torch.Generator(device=gpu_device).manual_seed(1)
    cache = te.PagedKVCache(1, 2, 64, rows=3, max_len=60, page_size=16, device=gpu_device, evictable=True)
    new = lambda n: (torch.randn((n, h, 64), generator=g, device=gpu_device, dtype=F16) for h in (4, 2, 2))
    cache.grow([20, 3, 0])
    cache.append(0, *new(23))
    cache.attend(0, next(new(3)))
    of = lambda plane, b: plane[cache.table[b, :2].long()].transpose(0, 1).flatten(1, 2)[:, :20]
    was = of(cache.scores[0], 0).clone(), of(cache.pos[0], 0).clone()
    cache.reorder([0, 0, 1])
    for b in (0, 1):
        assert torch.equal(of(cache.scores[0], b), was[0]) and torch.equal(of(cache.pos[0], b), was[1])
    cache.attend(0, next(new(3)))
    cache.evict(8, 2)
    assert cache.lengths == [8, 8, 3]


def test_a_search_step_in_a_graph(te, gpu_device):
    """append, tree_attention, beam_select, keep_kv and copy_pages of a step captured in a HIP graph: every replay, with
    eager calls between, equals the eager step on a copy of the same state."""
    dev = gpu_device
    P = serve_ref.Pages([1400, 70], 2, 16, 64, F16, 9, idle=0.0, room=40, spare=8)
    state, twin = P.to(dev), P.to(dev)
    g = torch.Generator(device=dev).manual_seed(1)
    ints = lambda t: torch.tensor(t, dtype=torch.int32, device=dev)
    starts, parents, path = ints([0, 7, 12]), ints([-1, 0, 0, 1, 3, 2, 5, -1, 0, 1, 1, 3]), ints([[0, 1, 3], [0, 2, -1]])
    used = set(P.table.flatten().tolist())
    free = [p for p in range(P.pages) if p not in used][:2]
    src, dst = ints(P.table[:, 0].tolist()), ints(free)
    x = [torch.zeros((12, h, 64), dtype=F16, device=dev) for h in (4, 2, 2)]
    head = torch.randn((64 * 4, 997), generator=g, device=dev, dtype=F16)

    def step(s, x):
        k, v, table, lens, scores, pos = s
        lens.add_(starts.diff())
        q = te.append_kv(*x, k, v, table, lens, starts=starts, scores=scores, pos=pos)
        out = te.tree_attention(q, k, v, table, lens, starts=starts, parents=parents, max_len=1440)
        chosen = te.beam_select((out.flatten(1) @ head).view(2, 6, -1), torch.zeros((2, 6), device=dev), 4)
        lens.copy_(te.keep_kv([k], [v], table, lens, starts, path, scores=[scores], pos=[pos]))
        te.copy_pages(k, v, src, dst, scores=scores, pos=pos)
        return (out, *chosen)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step([t.clone() for t in state], x)
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
        for a, b in zip((*out, *state), (*want, *twin)):
            assert torch.equal(a, b), i
    assert state[3].tolist() == [1400 + 4 * 3, 70 + 4 * 2]


def test_decoder_takes_prompts_and_drafts(te, gpu_device):
    """The example's decoder: a prompt in one pass, then a drafted tree, equal to the plain float64 decoder that takes their
    lines token by token. f16 activations round at every linear: 2e-2."""
    ex = _example("decode_block")
    g = torch.Generator(device=gpu_device).manual_seed(2)
    dec = ex.Decoder(2, 128, 256, 4, 2, 64, 1, 64, page_size=16)
    h = [torch.randn((1, 128), generator=g, device=gpu_device) for _ in range(18)]
    past = {}
    want = [ex.reference_step(dec, x, past) for x in h[:9]]
    got = dec.forward(torch.cat(h[:9]), [9])
    for a, b in zip(got, want):
        assert float((a - b[0]).norm() / b.norm()) < 2e-2
    # the tree's line 0, 2, 3, 5 is h[9], h[10], h[11], h[12]
    tree = [h[9], h[14], h[10], h[11], h[15], h[12]]
    got = dec.forward(torch.cat(tree), [6], [0, 1, 1, 2, 2, 3], torch.tensor([-1, 0, 0, 2, 1, 3], dtype=torch.int32, device=gpu_device))
    for i, x in zip((0, 2, 3, 5), h[9:13]):
        b = ex.reference_step(dec, x, past)
        assert float((got[i] - b[0]).norm() / b.norm()) < 2e-2
    dec.cache.keep([[0, 2, 3, 5]])
    b = ex.reference_step(dec, h[13], past)
    assert dec.cache.lengths == dec.cache.seen == [13] and float((dec.step(h[13]) - b).norm() / b.norm()) < 2e-2


def test_search_example(te, gpu_device):
    """Drafts give the tokens that decoding one by one gives, in fewer passes; beams come best first, each with the score
    that its line has when it is decoded alone."""
    ex = _example("search_block")
    rng = random.Random(1)
    prompt = [rng.randrange(512) for _ in range(11)]
    plain = ex.decode(ex.Model(1, 64), prompt, 16)
    drafted, passes = ex.decode_drafted(ex.Model(1, 64), prompt, 16, ex.noisy_drafter(plain, 8, 512, rng))
    assert drafted == plain and passes < 12
    lines, scores = ex.beam_search(ex.Model(3, 64), prompt, 3, 6)
    assert len({tuple(line) for line in lines}) == 3 and scores == sorted(scores, reverse=True)
    for line, score in zip(lines, scores):
        model, total = ex.Model(1, 64), 0.0
        logits = model(prompt, [len(prompt)])[-1]
        for token in line:
            total += float(torch.log_softmax(logits.double(), 0)[token])
            logits = model([token], 1)[0]
        assert abs(total - score) < 0.05 * 6      # logits of size 3, off by 2e-2 of that and less a step
