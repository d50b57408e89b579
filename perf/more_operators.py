"""The operators that carry several hypotheses over a paged key-value cache, as a serving loop runs them: attention
of several new tokens a row (drafted tokens in a tree, or a prompt), beam search's selection over beams and
vocabulary, copies of pages (forks), and the closing up of the drafted tokens that stay.

Sizes are those of the models that the benchmark names (Qwen3-8B: 32 query heads over 8 key-value heads of 128,
vocabulary 151936; SmolLM2-135M: 9 over 3 heads of 64, vocabulary 49152) or generic. `run` computes the operators in
elementary torch operations, or, where `own` is true, through the package's entry points.
"""
from __future__ import annotations

import math
import random

import torch

own = False

DEV = "cuda"
DTYPES = {"f16": torch.float16, "f32": torch.float32, "bf16": torch.bfloat16}
SIZE = {"f16": 2, "f32": 4, "bf16": 2}


def _tree(name, batch, length, new, **more):
    """`length`: the longest sequence, its `new` drafted tokens among it; `ragged` spreads both over the rows."""
    c = {"name": name, "op": "tree", "batch": batch, "length": length, "new": new, "ragged": False, "hq": 32, "hkv": 8,
         "d": 128, "page": 64, "x": "f16", "cache": "f16", "y": "f16"}
    c.update(more)
    return c


def _prompt(name, batch, tokens, before, **more):
    """`tokens` of all rows' prompts, unevenly split, behind `before` cached ones each."""
    c = {"name": name, "op": "prompt", "batch": batch, "tokens": tokens, "before": before, "hq": 32, "hkv": 8, "d": 128,
         "page": 64, "x": "f16", "cache": "f16", "y": "f16"}
    c.update(more)
    return c


def _beam(name, batch, beams, vocab, k, **more):
    c = {"name": name, "op": "beam", "batch": batch, "beams": beams, "vocab": vocab, "k": k, "x": "f32", "ended": False}
    c.update(more)
    return c


def _copy(name, layers, pages, **more):
    c = {"name": name, "op": "copy", "layers": layers, "pages": pages, "partial": False, "planes": False, "hkv": 8, "d": 128,
         "page": 64, "cache": "f16"}
    c.update(more)
    return c


def _keep(name, layers, batch, length, new, path, **more):
    """`path`: the longest run of drafted tokens that stays, of `new` behind up to `length` cached ones."""
    c = {"name": name, "op": "keep", "layers": layers, "batch": batch, "length": length, "new": new, "path": path,
         "planes": False, "hkv": 8, "d": 128, "page": 64, "cache": "f16"}
    c.update(more)
    return c


def listed():
    return [
        # the smallest check of drafted tokens: a small model's first answer tokens, f32 in and out
        _tree("tree_small_b1", 1, 149, 7, hq=9, hkv=3, d=64, page=16, x="f32", y="f32"),
        # a serving batch of uneven lengths, each row with a tree of its own; one row waits, one has its draft alone
        _tree("tree_b32", 32, 8192, 26, ragged=True),
        # one long sequence with a large tree: the work has to be split over its length
        _tree("tree_long_b1", 1, 32717, 63, x="bf16", cache="bf16", y="bf16"),
        # prompts of five sequences at once, of uneven lengths, into an empty cache
        _prompt("prompt_6007", 5, 6007, 0),
        # the next part of a long prompt
        _prompt("prompt_part_b1", 1, 1024, 8192, x="bf16", cache="bf16", y="bf16"),
        # one sequence of the small model, its likeliest token and that token's log-probability: the call itself counts
        _beam("beam_greedy_b1", 1, 1, 49152, 1),
        # a small batch of the 8B model's logits with four beams each, twice as many candidates as beams
        _beam("beam_b16", 16, 4, 151936, 8, x="f16"),
        # a large one, bf16, some of whose beams have ended
        _beam("beam_b64", 64, 8, 151936, 16, x="bf16", ended=True),
        # a small model's sequence forked into four beams: the page that each fills further, as far as it is filled
        _copy("copy_fork_small", 6, 3, partial=True, hkv=3, d=64, page=16, cache="bf16"),
        # sequences of the 8B model copied page by page in a third of its layers, with scores and positions
        _copy("copy_pages_40", 12, 40, planes=True),
        # after a check of drafted tokens: a few of each row's stay
        _keep("keep_step_b16", 12, 16, 333, 26, 6),
        # long drafts of a small model's batch, scores and positions with them
        _keep("keep_long_b48", 30, 48, 219, 200, 90, planes=True, hkv=3, d=64, page=16, cache="bf16"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["tree", "tree", "tree", "prompt", "prompt", "beam", "beam", "beam", "copy", "keep"])
    low = rng.choice(["f16", "bf16"])
    hkv, group = rng.choice([1, 2, 3, 4, 8]), rng.choice([1, 2, 3, 4, 4, 6, 8, 16])
    d, page = rng.choice([64, 64, 80, 96, 128, 128, 128, 256]), rng.choice([16, 32, 64, 64, 128])
    types = {"x": rng.choice([low, low, low, "f32"]), "cache": low, "y": rng.choice([low, low, low, "f32"])}
    heads = {"hq": hkv * group, "hkv": hkv, "d": d, "page": page}
    hd = hkv * group * d
    if op == "tree":
        batch, length, new = _log_int(rng, 1, 64), _log_int(rng, 1, 32768), _log_int(rng, 1, 128)
        length = max(1, min(length, 32 * 8192 * 8 * 128 // 2 // (batch * hkv * d)))
        # no more products than the largest part of a prompt, nor larger logits for the plain form
        new = max(1, min(new, length, 100_000_000_000 // (4 * batch * length * hd), 1_400_000_000 // (batch * length * hkv * group)))
        c = _tree("", batch, length, new, ragged=rng.random() < 0.6, **heads, **types)
    elif op == "prompt":
        batch, before = _log_int(rng, 1, 16), rng.choice([0, _log_int(rng, 1, 8192)])
        tokens = _log_int(rng, batch, 6007)
        while True:
            c = _prompt("", batch, tokens, before, **heads, **types)
            most = max(_prompts(c))
            pairs = sum(n * before + n * (n + 1) // 2 for n in _prompts(c))
            if 4 * pairs * hd <= 100_000_000_000 and batch * most * (before + most) * hkv * group <= 1_400_000_000:
                break
            tokens = max(batch, tokens * 3 // 4)
    elif op == "beam":
        batch, beams, vocab = _log_int(rng, 1, 64), _log_int(rng, 1, 16), _log_int(rng, 1000, 151936)
        x = rng.choice(["f16", "bf16", "f32"])
        vocab = min(vocab, 64 * 8 * 151936 * 2 // (batch * beams * SIZE[x]))
        c = _beam("", batch, beams, vocab, rng.choice([1, beams, 2 * beams, _log_int(rng, 1, 64)]), x=x, ended=rng.random() < 0.4)
    elif op == "copy":
        c = _copy("", _log_int(rng, 1, 36), _log_int(rng, 1, 200), partial=rng.random() < 0.5, planes=rng.random() < 0.3,
                  hkv=hkv, d=d, page=page, cache=low)
        c["pages"] = max(1, min(c["pages"], 12 * 40 * 8 * 64 * 128 // (c["layers"] * hkv * page * d)))
    else:
        batch, new = _log_int(rng, 1, 48), _log_int(rng, 1, 256)
        c = _keep("", _log_int(rng, 1, 36), batch, _log_int(rng, 1, 400), new, rng.randint(1, new), planes=rng.random() < 0.3,
                  hkv=hkv, d=d, page=page, cache=low)
        each = c["layers"] * hkv * d
        c["batch"] = max(1, min(batch, 30 * 48 * 480 * 3 * 64 // (each * (c["length"] + new + page))))
    del c["name"]
    return c


# ------------------------------------------------------------------ the rows


def _prompts(case):
    """The rows' new tokens: a ragged split of all of them."""
    n, total = case["batch"], case["tokens"]
    rng = random.Random(1000 * n + total)
    cuts = sorted(rng.randint(0, total - n) for _ in range(n - 1))
    return [b - a + 1 for a, b in zip([0] + cuts, cuts + [total - n])]


def _rows(case):
    """The rows' lengths and how many tokens of each are new. Ragged: the first row full, one that waits, one with
    nothing but its draft, and the rest spread."""
    n = case["batch"]
    if case["op"] == "prompt":
        new = _prompts(case)
        return [case["before"] + k for k in new], new
    top, most = case["length"], case["new"]
    rng = random.Random(1000 * n + top)
    if case["op"] == "keep":
        new = [most] + [rng.randint(0, most) for _ in range(n - 1)]
        return [rng.randint(0, top) + k for k in new], new
    if not case["ragged"]:
        return [top] * n, [most] * n
    lengths = ([top, rng.randint(0, top), most] + [rng.randint(most, top) for _ in range(n)])[:n]
    return lengths, ([most, 0, most] + [rng.randint(1, most) for _ in range(n)])[:n]


def _parents(case):
    """Trees as a drafter makes them: each token continues one of the last few before it."""
    rng = random.Random(case["length"])
    return [[-1 if i == 0 else rng.randint(max(0, i - 8), i - 1) for i in range(n)] for n in _rows(case)[1]]


def _paths(case):
    """What stays of each row's draft: from its first token on, in order, up to `path` of them."""
    rng = random.Random(case["length"] + 1)
    return [sorted(rng.sample(range(n), min(n, rng.randint(1, case["path"])))) for n in _rows(case)[1]]


def _pages(case, lengths, g):
    """Page ids in no order, as an allocator that frees and reuses them hands them out (-1 past a row's own); one page
    more than the table holds exists. Returns the table and the count of pages."""
    need = [-(-n // case["page"]) for n in lengths]
    total, widest = sum(need) + 1, max(1, max(need))
    ids = torch.randperm(total - 1, generator=g, device=DEV).int()
    table = torch.full((len(need), widest), -1, dtype=torch.int32, device=DEV)
    at = 0
    for b, k in enumerate(need):
        table[b, :k] = ids[at:at + k]
        at += k
    return table, total


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    s = {"case": case}
    if case["op"] == "beam":
        shape = (case["batch"], case["beams"], case["vocab"])
        # a model's logits: a few tokens stand out; some tokens are banned
        x = torch.randn(shape, generator=g, device=DEV) * 3
        x[..., :: 97] = -math.inf
        s["logits"] = x.to(DTYPES[case["x"]])
        s["scores"] = -torch.rand(shape[:2], generator=g, device=DEV) * 20
        s["ended"] = None
        if case["ended"]:
            s["ended"] = (torch.arange(shape[0] * shape[1], device=DEV) % 5 == 3).view(shape[:2])
        return s
    hkv, page, d = case["hkv"], case["page"], case["d"]
    dtype = DTYPES[case["cache"]]

    def pool(*n):
        return torch.randn((*n, hkv, page, d), generator=g, device=DEV, dtype=dtype)

    if case["op"] == "copy":
        n = case["pages"]
        total = 2 * n + 5
        ids = torch.randperm(total, generator=g, device=DEV).int()
        s["src"], s["dst"] = ids[:n].clone(), ids[n:2 * n].clone()
        s["counts"] = torch.randint(1, page, (n,), generator=g, device=DEV).int() if case["partial"] else None
    else:
        lengths, new = _rows(case)
        s["table"], total = _pages(case, lengths, g)
        s["lens"] = _ints(lengths)
        starts = [sum(new[:i]) for i in range(len(new) + 1)]
        s["starts"] = _ints(starts)
    if case["op"] in ("copy", "keep"):
        s["k"], s["v"] = pool(case["layers"], total), pool(case["layers"], total)
        plane = (case["layers"], total, hkv, page)
        s["scores"] = torch.rand(plane, generator=g, device=DEV) if case["planes"] else None
        s["pos"] = torch.randint(0, 9999, plane, generator=g, device=DEV).int() if case["planes"] else None
        if case["op"] == "keep":
            paths = _paths(case)
            s["path"] = _ints([p + [-1] * (case["path"] - len(p)) for p in paths])
        return s
    s["k_pages"], s["v_pages"] = pool(total), pool(total)
    s["q"] = (torch.randn((starts[-1], case["hq"], d), generator=g, device=DEV) * 2).to(DTYPES[case["x"]])
    s["parents"] = _ints([p for row in _parents(case) for p in row]) if case["op"] == "tree" else None
    # memory that no token has been written to holds anything
    slot = torch.arange(s["table"].shape[1] * page, device=DEV)
    idle = (slot >= s["lens"][:, None]).view(case["batch"], -1, 1, page, 1)
    at = s["table"].long().clamp_min(0)
    owned = (s["table"] >= 0)[:, :, None, None, None]
    for p in (s["k_pages"], s["v_pages"]):
        p[at[owned.flatten(1)]] = torch.where(idle & owned, math.nan, p[at])[owned.flatten(1)]
    return s


# ------------------------------------------------------------------ one pass


def run(s):
    return {"tree": _run_tree, "prompt": _run_tree, "beam": _run_beam, "copy": _run_copy, "keep": _run_keep}[s["case"]["op"]](s)


def _te():
    import importlib
    return importlib.import_module("trellis-everywhere_amd")


def _run_tree(s):
    c = s["case"]
    if own:
        most = c["length"] if c["op"] == "tree" else s["table"].shape[1] * c["page"]
        return _te().tree_attention(s["q"], s["k_pages"], s["v_pages"], s["table"], s["lens"], starts=s["starts"],
                                    parents=s["parents"], max_len=most, out_dtype=DTYPES[c["y"]])
    hkv, d, page, batch = c["hkv"], c["d"], c["page"], c["batch"]
    starts, lens = s["starts"].long(), s["lens"].long()
    n = starts.diff()
    t = torch.arange(s["q"].shape[0], device=DEV)
    row = torch.searchsorted(starts, t, right=True) - 1
    nth = t - starts[row]
    most = int(_most_new(c))
    q = torch.zeros((batch, most, c["hq"], d), device=DEV)
    q[row, nth] = s["q"].float()
    # what each new token sees of its row's new tokens
    i = torch.arange(most, device=DEV)
    if s["parents"] is None:
        sees = (i[:, None] >= i).expand(batch, -1, -1)
    else:
        parent = torch.full((batch, most), -1, dtype=torch.long, device=DEV)
        parent[row, nth] = s["parents"].long()
        hop = (parent[:, :, None] == i).float()
        sees = torch.eye(most, device=DEV) + hop
        for _ in range(most.bit_length()):
            hop = torch.matmul(hop, hop)
            sees = sees + torch.matmul(hop, sees)
        sees = sees > 0
    # slots of the rows' pages, in a [pages, heads, page] plane
    at = torch.where(s["table"] >= 0, s["table"], 0).long()
    head = torch.arange(hkv, device=DEV).view(1, -1, 1, 1)
    at = ((at[:, None, :, None] * hkv + head) * page + torch.arange(page, device=DEV)).flatten(2)
    slot = torch.arange(at.shape[-1], device=DEV)
    rel = slot - (lens - n)[:, None]                                                         # [B, L]
    seen = torch.gather(sees, 2, rel.clamp(0, most - 1)[:, None].expand(-1, most, -1))
    seen = ((rel < 0)[:, None] | seen) & (slot < lens[:, None])[:, None]                     # [B, T, L]
    live = (slot < lens[:, None])[:, None, :, None]
    k = torch.where(live, s["k_pages"].view(-1, d)[at].float(), 0.0)
    q = q.view(batch, most, hkv, -1, d).transpose(1, 2)                                      # [B, hkv, T, G, d]
    group = q.shape[3]
    p = torch.matmul(q.reshape(batch, hkv, -1, d), k.transpose(-1, -2).contiguous()) / math.sqrt(d)
    del k
    p = p.view(batch, hkv, most, group, -1)
    p = torch.where(seen[:, None, :, None], p, -math.inf)
    p = torch.exp(p - p.amax(-1, keepdim=True).clamp_min(-3e38))
    p = p / p.sum(-1, keepdim=True).clamp_min(1e-38)
    v = torch.where(live, s["v_pages"].view(-1, d)[at].float(), 0.0)
    out = torch.matmul(p.view(batch, hkv, most * group, -1), v).view(batch, hkv, most, group, d)
    return out.transpose(1, 2).reshape(batch, most, c["hq"], d)[row, nth].to(DTYPES[c["y"]])


def _most_new(case):
    return max(1, max(_rows(case)[1]))


def _run_beam(s):
    c = s["case"]
    if own:
        scores, beams, tokens = _te().beam_select(s["logits"], s["scores"], c["k"], ended=s["ended"], end_token=2)
        return {"scores": scores, "beams": beams, "tokens": tokens}
    # in 64 bits: candidates of two beams may lie next to each other
    x = s["logits"].double()
    top = x.amax(-1, keepdim=True)
    x = x - top - torch.exp(x - top).sum(-1, keepdim=True).log() + s["scores"].double()[..., None]
    if s["ended"] is not None:
        alone = torch.arange(c["vocab"], device=DEV) == 2
        x = torch.where(s["ended"][..., None], torch.where(alone, s["scores"].double()[..., None], -math.inf), x)
    # each beam's first k, then theirs; equal ones by the lowest index
    k = min(c["k"], c["vocab"])
    value, token = torch.sort(x, dim=-1, descending=True, stable=True)
    value, token = value[..., :k].flatten(1), token[..., :k].flatten(1)
    value, order = torch.sort(value, dim=-1, descending=True, stable=True)
    value, order = value[:, :c["k"]], order[:, :c["k"]]
    none = value == -math.inf
    return {"scores": value.float(), "beams": torch.where(none, 0, order // k).int(),
            "tokens": torch.where(none, 2, token.gather(1, order)).int()}


def _run_copy(s):
    if own:
        _te().copy_pages(s["k"], s["v"], s["src"], s["dst"], counts=s["counts"], scores=s["scores"], pos=s["pos"])
    else:
        src, dst = s["src"].long(), s["dst"].long()
        page = s["case"]["page"]
        taken = torch.arange(page, device=DEV) < (page if s["counts"] is None else s["counts"][:, None, None])   # [n, 1, page]
        for name in ("k", "v", "scores", "pos"):
            p = s[name]
            if p is not None:
                p[:, dst] = torch.where(taken[..., None] if p.dim() == 5 else taken, p[:, src], p[:, dst])
    return {n: s[n] for n in ("k", "v", "scores", "pos")}


def _run_keep(s):
    if own:
        lens = _te().keep_kv(s["k"], s["v"], s["table"], s["lens"], s["starts"], s["path"], scores=s["scores"], pos=s["pos"])
    else:
        page, table = s["case"]["page"], s["table"].long()
        base = s["lens"].long() - s["starts"].long().diff()
        path = s["path"].long()
        row, nth = (path >= 0).nonzero(as_tuple=True)
        src, dst = base[row] + path[row, nth], base[row] + nth
        frm, to = (table[row, src // page], src % page), (table[row, dst // page], dst % page)
        for name in ("k", "v", "scores", "pos"):
            p = s[name]
            if p is not None:
                p[:, to[0], :, to[1]] = p[:, frm[0], :, frm[1]]
        lens = (base + (path >= 0).sum(1)).int()
    return {"lens": lens, **{n: s[n] for n in ("k", "v", "scores", "pos")}}


# ------------------------------------------------------------------ what a pass cannot do without


def work(case):
    c = case
    if c["op"] == "beam":
        rows = c["batch"] * c["beams"]
        if c["ended"]:
            rows -= sum(i % 5 == 3 for i in range(rows))
        return {"bytes": rows * c["vocab"] * SIZE[c["x"]] + 5 * c["batch"] * c["beams"] + 12 * c["batch"] * c["k"],
                "flops": 4 * rows * c["vocab"]}
    each = c["hkv"] * (4 * c["d"] + (8 if c.get("planes") else 0))      # bytes of a token in one layer
    if c["op"] == "copy":
        tokens = c["pages"] * c["page"] // (2 if c["partial"] else 1)
        return {"bytes": 2 * c["layers"] * tokens * each, "flops": 0}
    if c["op"] == "keep":
        moves = sum(i != j for p in _paths(c) for i, j in enumerate(p))
        return {"bytes": 2 * c["layers"] * moves * each + 4 * c["batch"] * c["path"], "flops": 0}
    lengths, new = _rows(c)
    if c["op"] == "prompt":
        pairs = sum(n * c["before"] + n * (n + 1) // 2 for n in new)
    else:
        pairs = 0
        for m, n, parents in zip(lengths, new, _parents(c)):
            depth = []
            for p in parents:
                depth.append(1 if p < 0 else depth[p] + 1)
            pairs += n * (m - n) + sum(depth)
    read = sum(m for m, n in zip(lengths, new) if n)
    row = sum(new) * c["hq"] * c["d"] * (SIZE[c["x"]] + SIZE[c["y"]])
    return {"bytes": read * each + row + 4 * read // c["page"], "flops": 4 * pairs * c["hq"] * c["d"]}


# ------------------------------------------------------------------ the definitions in 64 bits


def exact(case, seed):
    s = prepare(case, seed)
    return {"tree": _exact_tree, "prompt": _exact_tree, "beam": _exact_beam, "copy": _exact_copy, "keep": _exact_keep}[case["op"]](s)


def _exact_tree(s):
    c = s["case"]
    group, page = c["hq"] // c["hkv"], c["page"]
    lengths, new = _rows(c)
    parents = _parents(c) if c["op"] == "tree" else None
    out, t = [], 0
    for b, (m, n) in enumerate(zip(lengths, new)):
        if n == 0:
            continue
        hidden = torch.ones((n, m), dtype=torch.bool)
        hidden[:, :m - n] = False
        if parents is None:
            hidden[:, m - n:] = torch.ones((n, n), dtype=torch.bool).triu(1)
        else:
            for i in range(n):
                j = i
                while j >= 0:
                    hidden[i, m - n + j] = False
                    j = parents[b][j]
        hidden = hidden.to(DEV)
        ids = s["table"][b, :-(-m // page)].long()
        got = torch.zeros((n, c["hq"], c["d"]), dtype=torch.float64, device=DEV)
        for h in range(c["hkv"]):
            k = s["k_pages"][ids, h].reshape(-1, c["d"])[:m].double()
            v = s["v_pages"][ids, h].reshape(-1, c["d"])[:m].double()
            for i in range(h * group, (h + 1) * group):
                p = (s["q"][t:t + n, i].double() @ k.t()) * c["d"] ** -0.5
                got[:, i] = torch.softmax(p.masked_fill(hidden, -math.inf), -1) @ v
        out.append(got)
        t += n
    return torch.cat(out)


def _exact_beam(s):
    c = s["case"]
    out = []
    for b in range(c["batch"]):
        offers = []
        for j in range(c["beams"]):
            score = s["scores"][b, j].double()
            if s["ended"] is not None and bool(s["ended"][b, j]):
                offers.append(score.view(1))
            else:
                offers.append(torch.log_softmax(s["logits"][b, j].double(), -1) + score)
        offers = torch.cat(offers)
        offers = torch.cat([offers, torch.full((c["k"],), -math.inf, dtype=torch.float64, device=DEV)])
        out.append(offers.topk(c["k"]).values)
    return {"scores": torch.stack(out), "beams": None, "tokens": None}


def _exact_copy(s):
    c = s["case"]
    counts = [c["page"]] * c["pages"] if s["counts"] is None else s["counts"].tolist()
    planes = {n: None if s[n] is None or n == "pos" else s[n].double() for n in ("k", "v", "scores", "pos")}
    for p in planes.values():
        if p is not None:
            for i, j, n in zip(s["src"].tolist(), s["dst"].tolist(), counts):
                p[:, j, :, :n] = p[:, i, :, :n]
    return planes


def _exact_keep(s):
    c = s["case"]
    planes = {n: None if s[n] is None or n == "pos" else s[n].double() for n in ("k", "v", "scores", "pos")}
    table = s["table"].tolist()
    lengths, new = _rows(c)
    for p in planes.values():
        if p is None:
            continue
        old = p.clone()
        for b, (m, n, path) in enumerate(zip(lengths, new, _paths(c))):
            for to, frm in enumerate(path):
                i, j = m - n + to, m - n + frm
                p[:, table[b][i // c["page"]], :, i % c["page"]] = old[:, table[b][j // c["page"]], :, j % c["page"]]
        del old
    return {"lens": None, **planes}
