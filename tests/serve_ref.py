"""Plain float64 restatements of the operators between the packed linears, in loops over rows and heads on the
CPU, for the tests; and a paged cache laid out at random."""
import torch

EPS = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}   # half an ulp, relative
TINY = {torch.float32: 0.0, torch.float16: 2.0 ** -25, torch.bfloat16: 0.0}               # of f16's subnormals


def rms(x, w, eps=1e-6):
    x = x.double()
    return x / (x.pow(2).mean(-1, keepdim=True) + eps).sqrt() * w.double()


def residual_norm(x, residual, weight, post_weight=None, gate=None, scale=1.0, eps=1e-6):
    b = x.double() if post_weight is None else rms(x, post_weight, eps)
    if gate is not None:
        b = b * gate.double()
    h = scale * b if residual is None else residual.double() + scale * b
    return rms(h, weight, eps), h


def rotate(x, cos, sin):
    """x [..., d] float64; cos, sin [r/2]."""
    r = cos.shape[-1]
    a, b = x[..., :r], x[..., r:2 * r]
    return torch.cat([a * cos - b * sin, b * cos + a * sin, x[..., 2 * r:]], -1)


class Pages:
    """A pool and tables on the CPU: row b's n tokens on pages of their own, in no order; idle memory holds
    `idle`. layout "hs": [pages, heads, page, d]; "sh": the same view of memory [pages, page, heads, d]."""

    def __init__(self, lengths, heads, page, d, dtype, seed=0, idle=float("nan"), layout="hs", spare=2, room=0):
        self.g = g = torch.Generator().manual_seed(seed)
        self.lengths, self.heads, self.page, self.d = lengths, heads, page, d
        need = [-(-(n + room) // page) for n in lengths]
        self.pages = sum(need) + spare
        ids = torch.randperm(self.pages, generator=g).int()
        self.width = max(1, max(need, default=1))
        self.table = torch.full((len(lengths), self.width), -1, dtype=torch.int32)
        at = 0
        for b, k in enumerate(need):
            self.table[b, :k] = ids[at:at + k]
            at += k
        shape = (self.pages, heads, page, d) if layout == "hs" else (self.pages, page, heads, d)
        turn = (lambda t: t) if layout == "hs" else (lambda t: t.transpose(1, 2))
        self.k, self.v = (turn(torch.randn(shape, generator=g).to(dtype)) for _ in range(2))
        self.scores = torch.rand((self.pages, heads, page), generator=g) * 3
        self.pos = torch.randint(0, 1000, (self.pages, heads, page), generator=g).int()
        self.lens = torch.tensor(lengths, dtype=torch.int32)
        if idle is not None:
            live = torch.zeros((self.pages, page), dtype=torch.bool)
            for b, n in enumerate(lengths):
                for j in range(n):
                    live[self.table[b, j // page], j % page] = True
            for p in (self.k, self.v):
                p.transpose(1, 2)[~live] = idle

    def slots(self, b, n):
        """Page and slot-in-page index tensors of row b's first n tokens."""
        j = torch.arange(n)
        return self.table[b].long()[j // self.page], j % self.page

    def to(self, device):
        """The tensors on the device (strides kept): k, v, table, lens, scores, pos."""
        def move(t):
            if t.is_contiguous():
                return t.to(device)
            return t.transpose(1, 2).to(device).transpose(1, 2)
        return [move(t) for t in (self.k, self.v, self.table, self.lens, self.scores, self.pos)]


def attend(q, pages, scale=None, lengths=None):
    """(out float64 [rows, hq, d], scores float64 of the planes after)."""
    rows, hq, d = q.shape
    group = hq // pages.heads
    out, scores = torch.zeros((rows, hq, d), dtype=torch.float64), pages.scores.double().clone()
    for b, n in enumerate(pages.lengths if lengths is None else lengths):
        page, slot = pages.slots(b, n)
        there = (page >= 0) & (page < pages.pages)
        page, slot = page[there], slot[there]
        if page.numel() == 0:
            continue
        for h in range(pages.heads):
            k, v = pages.k[page, h, slot].double(), pages.v[page, h, slot].double()
            s = q[b, h * group:(h + 1) * group].double() @ k.t() * (d ** -0.5 if scale is None else scale)
            p = torch.softmax(s, -1)
            out[b, h * group:(h + 1) * group] = p @ v
            scores[page, h, slot] += p.sum(0)
    return out, scores


def evict(pages, keep, recent, next_pos=None, out_table=None):
    """The planes (k, v, scores, pos) and lengths after, by the definition."""
    planes = [t.clone() for t in (pages.k, pages.v, pages.scores, pages.pos)]
    to = pages.table if out_table is None else out_table
    for b, n in enumerate(pages.lengths):
        page, slot = pages.slots(b, n)
        for h in range(pages.heads):
            score, pos = pages.scores[page, h, slot].tolist(), pages.pos[page, h, slot].tolist()
            first = (n if next_pos is None else next_pos[b]) - recent
            worth = lambda i: (2, 0.0) if pos[i] >= first else (1, 0.0) if score[i] != score[i] else (0, score[i])
            order = sorted(range(n), key=lambda i: (-worth(i)[0], -worth(i)[1], i))
            kept = set(order[:keep])
            above = [i for i in range(keep, n) if i in kept]
            for j in range(min(n, keep)):
                src = j if j in kept else above.pop(0)
                if out_table is None and src == j:
                    continue
                for plane, old in zip(planes, (pages.k, pages.v, pages.scores, pages.pos)):
                    plane[to[b, j // pages.page].long(), h, j % pages.page] = old[page[src], h, slot[src]]
    return planes, [min(n, keep) for n in pages.lengths]


def close(got, want, dtype, abs_err, what=""):
    """|got - want| within abs_err (computed in fp32) plus one rounding of the result to dtype."""
    got, want = got.double().cpu(), want.double()
    assert torch.equal(torch.isnan(got), torch.isnan(want)), f"{what}: NaN in other places"
    ok = ~torch.isnan(want)
    err = (got - want).abs()
    bound = abs_err + 1.01 * EPS[dtype] * (want.abs() + abs_err) + TINY[dtype]
    bad = ok & (err > bound)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float((err - bound)[ok].max()):.3e} over"
