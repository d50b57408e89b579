"""Plain float64 restatements of the operators that carry several hypotheses over a paged cache, in loops on the CPU, for
the tests."""
import math

import torch

NONE = -math.inf


def counted(starts, rows):
    return [int(starts[b + 1]) - int(starts[b]) for b in range(rows)]


def ancestors(parents, n):
    """Token i's own number and its ancestors'; parents None: a chain."""
    out = []
    for i in range(n):
        p = i - 1 if parents is None else int(parents[i])
        out.append([i] + (out[p] if 0 <= p < i else []))
    return out


def tree(q, pages, starts, parents=None, scale=None, lens=None, max_len=None):
    """out float64 [tokens, hq, d] of serve_ref.Pages `pages`; lens: instead of the pages' lengths."""
    tokens, hq, d = q.shape
    group, out = hq // pages.heads, torch.zeros(q.shape, dtype=torch.float64)
    lens = pages.lengths if lens is None else lens
    cap = pages.width * pages.page if max_len is None else min(max_len, pages.width * pages.page)
    for b, n in enumerate(counted(starts, len(lens))):
        base, seen = lens[b] - n, max(0, min(lens[b], cap))
        t0 = int(starts[b])
        lines = ancestors(None if parents is None else parents[t0:t0 + n], n)
        for i in range(n):
            if not 0 <= base + i < seen:
                continue
            slots = list(range(max(0, base))) + sorted(base + j for j in lines[i] if base + j >= 0)
            j = torch.tensor(slots, dtype=torch.long)
            page = pages.table[b].long()[j // pages.page]
            there = (page >= 0) & (page < pages.pages)
            page, slot = page[there], j[there] % pages.page
            if page.numel() == 0:
                continue
            for h in range(pages.heads):
                k, v = pages.k[page, h, slot].double(), pages.v[page, h, slot].double()
                s = q[t0 + i, h * group:(h + 1) * group].double() @ k.t() * (d ** -0.5 if scale is None else scale)
                out[t0 + i, h * group:(h + 1) * group] = torch.softmax(s, -1) @ v
    return out


def beams(logits, scores, k, ended=None, end_token=0):
    """(scores float64, beams, tokens) [batch, k]."""
    batch, n, vocab = logits.shape
    out = torch.full((batch, k), NONE, dtype=torch.float64)
    frm, token = torch.zeros((batch, k), dtype=torch.int32), torch.full((batch, k), end_token, dtype=torch.int32)
    for b in range(batch):
        offers = []
        for j in range(n):
            score = float(scores[b, j])
            if ended is not None and bool(ended[b, j]):
                offers.append((score, j, end_token))
                continue
            x = logits[b, j].double()
            x = torch.where(x.isnan(), NONE, x)
            top = x.max()
            if top == NONE:
                continue
            c = score + (x - (top + (x - top).exp().sum().log()))
            order = torch.argsort(c, descending=True, stable=True)[:k]
            offers += [(float(c[v]), j, int(v)) for v in order]
        offers = sorted((o for o in offers if o[0] > NONE), key=lambda o: (-o[0], o[1], o[2]))[:k]
        for i, (c, j, v) in enumerate(offers):
            out[b, i], frm[b, i], token[b, i] = c, j, v
    return out, frm, token


def copy_pages(planes, src, dst, counts=None):
    """Copies of the planes [pages, heads, page, ...] after."""
    after = [p.clone() for p in planes]
    for i, (s, d) in enumerate(zip(src, dst)):
        pages, page = planes[0].shape[0], planes[0].shape[2]
        if not (0 <= s < pages and 0 <= d < pages) or s == d:
            continue
        n = page if counts is None else max(0, min(counts[i], page))
        for new, old in zip(after, planes):
            new[d, :, :n] = old[s, :, :n]
    return after


def path_of(path, n):
    kept = []
    for p in path:
        if p >= n or p <= (kept[-1] if kept else -1):
            break
        kept.append(p)
    return kept


def keep(planes, table, page, lens, starts, paths):
    """(the planes after, the new lengths)."""
    after, pages, new = [p.clone() for p in planes], planes[0].shape[0], []
    cap = table.shape[1] * page
    for b, n in enumerate(counted(starts, len(lens))):
        n = max(0, n)
        base, kept = lens[b] - n, path_of(paths[b], n)
        new.append(max(0, base + len(kept)))
        for i, p in enumerate(kept):
            s, d = base + p, base + i
            if d < 0 or s >= cap:
                continue
            sp, dp = int(table[b, s // page]), int(table[b, d // page])
            if 0 <= sp < pages and 0 <= dp < pages:
                for a, old in zip(after, planes):
                    a[dp, :, d % page] = old[sp, :, s % page]
    return after, new
