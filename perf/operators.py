"""The operators between a decoder block's packed linears, as a serving loop runs them: the norms around a
block with its residual, the append of new tokens to a paged key-value cache, attention of one new token
over that cache, and the cache's eviction by accumulated attention weight.

Sizes are those of the models that the benchmark names (Qwen3-8B: 32 query heads over 8 key-value heads of
128, width 4096; SmolLM2-135M: 9 over 3 heads of 64, width 576) or generic. `run` computes the operators in
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
EPS = 1e-6
THETA = 1e6


def _norm(name, rows, width, **more):
    c = {"name": name, "op": "norm", "rows": rows, "width": width, "x": "f32", "residual": "f32", "y": "f16",
         "post": False, "gate": "none", "scale": 1.0}
    c.update(more)
    return c


def _append(name, batch, tokens, **more):
    """`tokens`: new tokens in all; equal to `batch` for one each, otherwise ragged prompts."""
    c = {"name": name, "op": "append", "batch": batch, "tokens": tokens, "before": 1000, "hq": 32, "hkv": 8,
         "d": 128, "rot": 128, "page": 64, "x": "f32", "cache": "f16", "q": "f16", "qk_norm": True}
    c.update(more)
    return c


def _attend(name, batch, length, **more):
    """`length`: the longest sequence; `ragged` spreads the others from none to it."""
    c = {"name": name, "op": "attend", "batch": batch, "length": length, "ragged": False, "hq": 32, "hkv": 8,
         "d": 128, "page": 64, "x": "f16", "cache": "f16", "y": "f16", "scores": False}
    c.update(more)
    return c


def _evict(name, batch, length, keep, recent, **more):
    c = {"name": name, "op": "evict", "batch": batch, "length": length, "keep": keep, "recent": recent,
         "ragged": False, "apart": False, "hkv": 8, "d": 128, "page": 64, "cache": "f16"}
    c.update(more)
    return c


def listed():
    return [
        # one decoded token of the 8B model: the o projection's output joins the residual and is normed for
        # gate/up. The call itself counts
        _norm("norm_b1", 1, 4096),
        # a few sequences through a model with a norm on both sides of the block and a gate for each
        # row, bf16 throughout, a width that fills no vector evenly
        _norm("norm_gated_b37", 37, 1531, x="bf16", residual="bf16", y="bf16", post=True, gate="row", scale=0.25),
        # a long prompt's activations between two groups of linears
        _norm("norm_prompt_8192", 8192, 4096, x="f16", residual="f32"),
        # one decoded token of the 8B model: q and k normed and rotated, k and v into their pages
        _append("append_b1", 1, 1),
        # a serving batch of the small model, heads of 64, no norms of q and k, bf16
        _append("append_small_b48", 48, 48, hq=9, hkv=3, d=64, rot=64, page=16, x="bf16", cache="bf16", q="bf16",
                qk_norm=False, before=333),
        # prompts of five sequences at once, of uneven lengths
        _append("append_prompt_6007", 5, 6007, x="f16", before=0),
        # the shortest attention: a small model's first answer tokens, f32 in and out
        _attend("attend_small_b1", 1, 149, hq=9, hkv=3, d=64, page=16, x="f32", y="f32"),
        # one sequence of the 8B model with a long cache: the work has to be split over its length
        _attend("attend_long_b1", 1, 32717),
        # a serving batch of uneven lengths, from an empty slot to a full one
        _attend("attend_b64", 64, 8192, ragged=True),
        # the same with the weights accumulated for eviction, bf16
        _attend("attend_scored_b16", 16, 4099, ragged=True, scores=True, x="bf16", cache="bf16", y="bf16"),
        # a cache held at its budget: each step's token pushes one out, in place
        _evict("evict_step_b16", 16, 1025, 1024, 128),
        # a prompt's cache cut to a budget, into pages of its own (its old pages may be shared)
        _evict("evict_prompt_b4", 4, 16000, 2048, 256, ragged=True, apart=True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm", "append", "attend", "attend", "evict"])
    low = rng.choice(["f16", "bf16"])
    hkv, group = rng.choice([1, 2, 3, 4, 8]), rng.choice([1, 2, 3, 4, 4, 6, 8, 16])
    d, page = rng.choice([64, 64, 80, 96, 128, 128, 128, 256]), rng.choice([16, 32, 64, 64, 128])
    if op == "norm":
        width = _log_int(rng, 500, 12288)
        if rng.random() < 0.5:
            width = max(8, width // 64 * 64)
        c = _norm("", max(1, min(_log_int(rng, 1, 8192), (1 << 25) // width)), width, x=rng.choice([low, "f32"]),
                  residual=rng.choice([low, "f32"]), y=rng.choice([low, "f32"]), post=rng.random() < 0.4,
                  gate=rng.choice(["none", "none", "width", "row"]), scale=rng.choice([1.0, 0.5, 0.22]))
    elif op == "append":
        batch = _log_int(rng, 1, 64)
        tokens = batch if rng.random() < 0.5 else _log_int(rng, batch + 1, 6007)
        c = _append("", batch, tokens, hq=hkv * group, hkv=hkv, d=d, rot=rng.choice([d, d, d // 2 // 16 * 16]),
                    page=page, x=rng.choice([low, "f32"]), cache=low, q=rng.choice([low, "f32"]),
                    qk_norm=rng.random() < 0.5, before=_log_int(rng, 1, 4000) if tokens == batch else 0)
        if c["tokens"] * (c["hq"] + 2 * c["hkv"]) * d > 6007 * 48 * 128:
            c["tokens"] = max(c["batch"], 6007 * 48 * 128 // ((c["hq"] + 2 * c["hkv"]) * d))
    elif op == "attend":
        batch, length = _log_int(rng, 1, 64), _log_int(rng, 1, 32768)
        length = max(1, min(length, 64 * 8192 * 8 * 128 // 2 // (batch * hkv * d)))
        c = _attend("", batch, length, ragged=rng.random() < 0.6, hq=hkv * group, hkv=hkv, d=d, page=page,
                    x=rng.choice([low, low, "f32"]), cache=low, y=rng.choice([low, low, "f32"]),
                    scores=rng.random() < 0.3)
    else:
        batch, length = _log_int(rng, 1, 32), _log_int(rng, 64, 16000)
        length = max(64, min(length, 4 * 16000 * 8 * 128 // (batch * hkv * d)))
        apart = rng.random() < 0.5
        # in place a pass leaves the next less to move: a step's few tokens then
        keep = _log_int(rng, 16, length) if apart else max(16, length - _log_int(rng, 1, 16))
        c = _evict("", batch, length, keep, _log_int(rng, 1, keep), ragged=apart and rng.random() < 0.6,
                   apart=apart, hkv=hkv, d=d, page=page, cache=low)
    del c["name"]
    return c


# ------------------------------------------------------------------ inputs


def _lengths(case):
    """The rows' lengths: the longest first, then (if ragged) an empty one, one token, and the rest spread."""
    n, top = case["batch"], case["length"]
    if not case["ragged"]:
        return [top] * n
    rng = random.Random(1000 * n + top)
    return ([top, 0, 1] + [rng.randint(0, top) for _ in range(n)])[:n]


def _prompts(case):
    """The rows' new tokens: one each, or a ragged split of all of them."""
    n, total = case["batch"], case["tokens"]
    if total == n:
        return [1] * n
    rng = random.Random(1000 * n + total)
    cuts = sorted(rng.randint(0, total - n) for _ in range(n - 1))
    return [b - a + 1 for a, b in zip([0] + cuts, cuts + [total - n])]


def _pages(case, lengths, g, copies=1):
    """Page ids in no order, as an allocator that frees and reuses them hands them out (-1 past a row's own);
    one page more than the tables hold exists. Returns the tables and the count of pages."""
    need = [-(-n // case["page"]) for n in lengths]
    total, widest = sum(need) * copies + 1, max(1, max(need))
    ids = torch.randperm(total - 1, generator=g, device=DEV).int() if total > 1 else torch.zeros(0, dtype=torch.int32, device=DEV)
    tables, at = [], 0
    for _ in range(copies):
        rows = []
        for k in need:
            rows.append(torch.cat([ids[at:at + k], torch.full((widest - k,), -1, dtype=torch.int32, device=DEV)]))
            at += k
        tables.append(torch.stack(rows))
    return tables, total


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)

    def randn(*shape, dtype="f32", scale=1.0):
        return (torch.randn(shape, generator=g, device=DEV) * scale).to(DTYPES[dtype])

    def weight(n):
        return torch.rand(n, generator=g, device=DEV) + 0.5

    s = {"case": case}
    if case["op"] == "norm":
        rows, width = case["rows"], case["width"]
        s["x"] = randn(rows, width, dtype=case["x"])
        s["residual"] = randn(rows, width, dtype=case["residual"], scale=4.0)
        s["weight"] = weight(width)
        s["post"] = weight(width) if case["post"] else None
        s["gate"] = None if case["gate"] == "none" else randn(
            *((rows, width) if case["gate"] == "row" else (width,)), dtype=case["x"])
        return s

    def pool(n):
        return torch.randn((n, case["hkv"], case["page"], case["d"]), generator=g, device=DEV, dtype=DTYPES[case["cache"]])

    hkv, page, d = case["hkv"], case["page"], case["d"]
    if case["op"] == "append":
        new = _prompts(case)
        lengths = [case["before"] + n for n in new]
        (s["table"],), n_pages = _pages(case, lengths, g)
        s["k_pages"], s["v_pages"] = pool(n_pages), pool(n_pages)
        s["pos"] = torch.zeros((n_pages, hkv, page), dtype=torch.int32, device=DEV)
        s["scores"] = torch.rand((n_pages, hkv, page), generator=g, device=DEV)
        s["lens"] = _ints(lengths)
        ends = [sum(new[:i]) for i in range(len(new) + 1)]
        s["starts"] = None if case["tokens"] == case["batch"] else _ints(ends)
        t, hq = case["tokens"], case["hq"]
        s["q"], s["k"] = randn(t, hq, d, dtype=case["x"]), randn(t, hkv, d, dtype=case["x"])
        s["v"] = randn(t, hkv, d, dtype=case["x"])
        s["q_norm"], s["k_norm"] = (weight(d), weight(d)) if case["qk_norm"] else (None, None)
        # the rotary table of a model whose context holds these positions
        freq = THETA ** (-torch.arange(0, case["rot"], 2, dtype=torch.float64, device=DEV) / case["rot"])
        angle = torch.arange(max(lengths), dtype=torch.float64, device=DEV)[:, None] * freq
        s["cos"], s["sin"] = angle.cos().float(), angle.sin().float()
        return s

    lengths = _lengths(case)
    tables, n_pages = _pages(case, lengths, g, copies=2 if case.get("apart") else 1)
    s["table"], s["lens"] = tables[0], _ints(lengths)
    s["k_pages"], s["v_pages"] = pool(n_pages), pool(n_pages)
    slot = torch.arange(tables[0].shape[1] * page, device=DEV)
    if case["op"] == "attend":
        s["q"] = randn(case["batch"], case["hq"], d, dtype=case["x"], scale=2.0)
        # memory that no token has been written to holds anything
        idle = (slot >= s["lens"][:, None]).view(case["batch"], -1, 1, page, 1)
        at = tables[0].long().clamp_min(0)
        owned = (tables[0] >= 0)[:, :, None, None, None]
        for p in (s["k_pages"], s["v_pages"]):
            p[at[owned.flatten(1)]] = torch.where(idle & owned, math.nan, p[at])[owned.flatten(1)]
        s["scores"] = torch.rand((n_pages, hkv, page), generator=g, device=DEV) if case["scores"] else None
        return s
    # accumulated weights: most tokens little, a few much; some equal (tokens that no head looked at)
    w = torch.rand((n_pages, hkv, page), generator=g, device=DEV)
    s["scores"] = torch.where(w < 0.2, 0.0, w.pow(4) * 30)
    # positions: every token's own slot, as in a cache that nothing was evicted from
    s["pos"] = torch.zeros((n_pages, hkv, page), dtype=torch.int32, device=DEV)
    owned = tables[0] >= 0
    s["pos"][tables[0][owned].long()] = slot.int().view(1, -1, 1, page).expand(case["batch"], -1, hkv, page)[owned]
    s["out_table"] = tables[1][:, :-(-min(case["keep"], case["length"]) // page)].contiguous() if case["apart"] else None
    return s


# ------------------------------------------------------------------ one pass


def run(s):
    return {"norm": _run_norm, "append": _run_append, "attend": _run_attend, "evict": _run_evict}[s["case"]["op"]](s)


def _te():
    import importlib
    return importlib.import_module("trellis-everywhere_amd")


def _rms(x, weight):
    return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * weight


def _run_norm(s):
    c = s["case"]
    if own:
        y, h = _te().residual_norm(s["x"], s["residual"], s["weight"], post_weight=s["post"], gate=s["gate"],
                                   scale=c["scale"], eps=EPS, out_dtype=DTYPES[c["y"]])
        return {"y": y, "h": h}
    b = s["x"].float()
    if s["post"] is not None:
        b = _rms(b, s["post"])
    if s["gate"] is not None:
        b = b * s["gate"].float()
    h = s["residual"].float() + c["scale"] * b
    return {"y": _rms(h, s["weight"]).to(DTYPES[c["y"]]), "h": h.to(s["residual"].dtype)}


def _rotate(x, cos, sin):
    r = cos.shape[-1]
    a, b, rest = x[..., :r], x[..., r:2 * r], x[..., 2 * r:]
    return torch.cat([a * cos - b * sin, b * cos + a * sin, rest], -1)


def _slots(table, hkv, page, n_pages):
    """Flat slot numbers [rows, heads, width x page] of the tables' pages in a [pages, heads, page] plane; a
    page that a table does not have counts as the plane's last, which no table has."""
    at = torch.where(table >= 0, table, n_pages - 1).long()
    head = torch.arange(hkv, device=DEV).view(1, -1, 1, 1)
    inner = torch.arange(page, device=DEV).view(1, 1, 1, -1)
    return ((at[:, None, :, None] * hkv + head) * page + inner).flatten(2)


def _run_append(s):
    c = s["case"]
    if own:
        q = _te().append_kv(s["q"], s["k"], s["v"], s["k_pages"], s["v_pages"], s["table"], s["lens"],
                            starts=s["starts"], q_norm=s["q_norm"], k_norm=s["k_norm"], eps=EPS, cos=s["cos"],
                            sin=s["sin"], scores=s["scores"], pos=s["pos"], q_dtype=DTYPES[c["q"]])
        return {"q": q, "k_pages": s["k_pages"], "v_pages": s["v_pages"], "pos": s["pos"], "scores": s["scores"]}
    t = torch.arange(c["tokens"], device=DEV)
    starts = torch.arange(c["batch"] + 1, device=DEV) if s["starts"] is None else s["starts"].long()
    row = torch.searchsorted(starts, t, right=True) - 1
    place = s["lens"].long()[row] - (starts[row + 1] - t)
    q, k = s["q"].float(), s["k"].float()
    if s["q_norm"] is not None:
        q, k = _rms(q, s["q_norm"]), _rms(k, s["k_norm"])
    cos, sin = s["cos"][place][:, None], s["sin"][place][:, None]
    q, k = _rotate(q, cos, sin), _rotate(k, cos, sin)
    page, inner = s["table"].long()[row, place // c["page"]], place % c["page"]
    s["k_pages"][page, :, inner] = k.to(s["k_pages"].dtype)
    s["v_pages"][page, :, inner] = s["v"].to(s["v_pages"].dtype)
    s["pos"][page, :, inner] = place.int()[:, None].expand(-1, c["hkv"])
    s["scores"][page, :, inner] = torch.zeros((), device=DEV)
    return {"q": q.to(DTYPES[c["q"]]), "k_pages": s["k_pages"], "v_pages": s["v_pages"], "pos": s["pos"], "scores": s["scores"]}


def _run_attend(s):
    c = s["case"]
    if own:
        out = _te().paged_attention(s["q"], s["k_pages"], s["v_pages"], s["table"], s["lens"], max_len=c["length"],
                                    scores=s["scores"], out_dtype=DTYPES[c["y"]])
        return {"out": out, "scores": s["scores"]}
    hkv, d = c["hkv"], c["d"]
    at = _slots(s["table"], hkv, c["page"], s["k_pages"].shape[0])
    live = (torch.arange(at.shape[-1], device=DEV) < s["lens"][:, None])[:, None, None]      # [B, 1, 1, L]
    k = s["k_pages"].view(-1, d)[at].float()
    logits = torch.matmul(s["q"].float().view(c["batch"], hkv, -1, d), k.transpose(-1, -2)) / math.sqrt(d)
    del k
    logits = torch.where(live, logits, -math.inf)
    top = logits.amax(-1, keepdim=True).clamp_min(-3e38)
    p = torch.exp(logits - top)
    p = p / p.sum(-1, keepdim=True).clamp_min(1e-38)
    v = torch.where(live.transpose(-1, -2), s["v_pages"].view(-1, d)[at].float(), 0.0)
    out = torch.matmul(p, v).view(c["batch"], c["hq"], d).to(DTYPES[c["y"]])
    if s["scores"] is not None:
        s["scores"].view(-1).index_add_(0, at.flatten(), p.sum(2).flatten())
    return {"out": out, "scores": s["scores"]}


def _run_evict(s):
    c = s["case"]
    keep = c["keep"]
    if own:
        lens = _te().evict_kv(s["k_pages"], s["v_pages"], s["scores"], s["pos"], s["table"], s["lens"], keep,
                              c["recent"], out_table=s["out_table"], max_len=c["length"])
    else:
        hkv, page, n_pages = c["hkv"], c["page"], s["k_pages"].shape[0]
        at = _slots(s["table"], hkv, page, n_pages)
        width = at.shape[-1]
        slot = torch.arange(width, device=DEV)
        n = s["lens"].long().view(-1, 1, 1)
        scores, pos = s["scores"].view(-1)[at], s["pos"].view(-1)[at]
        key = torch.where(pos >= n - c["recent"], math.inf, scores)
        key = torch.where(slot < n, key, -math.inf)
        order = torch.sort(key, dim=-1, descending=True, stable=True).indices[..., :keep]
        kept = torch.zeros(at.shape, dtype=torch.bool, device=DEV).scatter_(-1, order, True) & (slot < n)
        top = min(keep, width)
        # the kept tokens above `keep`, in order, fill the holes below it, in order
        above = torch.where(kept & (slot >= keep), slot, width).sort(-1).values
        hole = ~kept[..., :top]
        nth = hole.cumsum(-1) - 1
        source = torch.where(hole, above.gather(-1, nth.clamp_min(0)).clamp_max(width - 1), slot[:top])
        target = at if s["out_table"] is None else _slots(s["out_table"], hkv, page, n_pages)
        to = target[..., :top]
        live = slot[:top] < n.clamp_max(keep)
        frm = torch.where(live, at.gather(-1, source), to)
        d = c["d"]
        for plane in (s["k_pages"].view(-1, d), s["v_pages"].view(-1, d), s["scores"].view(-1), s["pos"].view(-1)):
            plane[to] = plane[frm]
        lens = s["lens"].clamp_max(keep)
    return {"lens": lens, "k_pages": s["k_pages"], "v_pages": s["v_pages"], "scores": s["scores"], "pos": s["pos"]}


# ------------------------------------------------------------------ what a pass cannot do without


def work(case):
    c = case
    if c["op"] == "norm":
        n = c["rows"] * c["width"]
        each = SIZE[c["x"]] + 2 * SIZE[c["residual"]] + SIZE[c["y"]]
        gate = {"none": 0, "width": c["width"], "row": n}[c["gate"]] * SIZE[c["x"]]
        return {"bytes": n * each + gate + 4 * c["width"] * (2 if c["post"] else 1), "flops": n * (12 if c["post"] else 7)}
    if c["op"] == "append":
        t, heads = c["tokens"], c["hq"] + 2 * c["hkv"]
        moved = t * c["d"] * (heads * SIZE[c["x"]] + c["hq"] * SIZE[c["q"]] + 2 * c["hkv"] * SIZE[c["cache"]])
        return {"bytes": moved + t * (4 * c["rot"] + 8 * c["hkv"] + 8), "flops": 10 * t * (c["hq"] + c["hkv"]) * c["d"]}
    n = sum(_lengths(c))
    if c["op"] == "attend":
        row = c["batch"] * c["hq"] * c["d"] * (SIZE[c["x"]] + SIZE[c["y"]])
        cache = n * c["hkv"] * (2 * c["d"] * SIZE[c["cache"]] + (8 if c["scores"] else 0))
        return {"bytes": cache + row + 4 * n // c["page"], "flops": 4 * n * c["hq"] * c["d"]}
    moves = sum(min(m, c["keep"]) if c["apart"] else max(0, min(m - c["keep"], c["keep"])) for m in _lengths(c))
    return {"bytes": c["hkv"] * (8 * n + 2 * moves * (2 * c["d"] * SIZE[c["cache"]] + 8)), "flops": c["hkv"] * n}


# ------------------------------------------------------------------ the definitions in 64 bits


def exact(case, seed):
    s = prepare(case, seed)
    return {"norm": _exact_norm, "append": _exact_append, "attend": _exact_attend, "evict": _exact_evict}[case["op"]](s)


def _unit(x, weight):
    x = x.double()
    return x / ((x ** 2).sum(-1, keepdim=True) / x.shape[-1] + EPS).sqrt() * weight.double()


def _exact_norm(s):
    b = s["x"].double() if s["post"] is None else _unit(s["x"], s["post"])
    g = 1.0 if s["gate"] is None else s["gate"].double()
    h = s["residual"].double() + s["case"]["scale"] * g * b
    return {"y": _unit(h, s["weight"]), "h": h}


def _exact_append(s):
    c = s["case"]
    new, half, page = _prompts(c), c["rot"] // 2, c["page"]
    k_pages, v_pages, scores = s["k_pages"].double(), s["v_pages"].double(), s["scores"].double()
    q_out, t = [], 0
    for b, n in enumerate(new):
        first = c["before"]
        place = torch.arange(first, first + n, device=DEV)
        angle = torch.complex(s["cos"][place].double(), s["sin"][place].double())[:, None]

        def turned(x, weight):
            x = x.double() if weight is None else _unit(x, weight)
            z = torch.complex(x[..., :half], x[..., half:2 * half]) * angle
            return torch.cat([z.real, z.imag, x[..., 2 * half:]], -1)

        q_out.append(turned(s["q"][t:t + n], s["q_norm"]))
        ids = s["table"][b].long()[place // page]
        k_pages[ids, :, place % page] = turned(s["k"][t:t + n], s["k_norm"])
        v_pages[ids, :, place % page] = s["v"][t:t + n].double()
        scores[ids, :, place % page] = 0.0
        t += n
    return {"q": torch.cat(q_out), "k_pages": k_pages, "v_pages": v_pages, "pos": None, "scores": scores}


def _exact_attend(s):
    c = s["case"]
    out = torch.zeros((c["batch"], c["hq"], c["d"]), dtype=torch.float64, device=DEV)
    scores = None if s["scores"] is None else s["scores"].double()
    group, page = c["hq"] // c["hkv"], c["page"]
    for b, n in enumerate(_lengths(c)):
        if n == 0:
            continue
        ids = s["table"][b, :-(-n // page)].long()
        for h in range(c["hkv"]):
            k = s["k_pages"][ids, h].reshape(-1, c["d"])[:n].double()
            v = s["v_pages"][ids, h].reshape(-1, c["d"])[:n].double()
            rows = slice(h * group, (h + 1) * group)
            p = torch.softmax((k @ s["q"][b, rows].double().t()).t() * c["d"] ** -0.5, -1)
            out[b, rows] = p @ v
            if scores is not None:
                j = torch.arange(n, device=DEV)
                scores[ids[j // page], h, j % page] += p.sum(0)
    return {"out": out, "scores": scores}


def _exact_evict(s):
    c = s["case"]
    keep, page = c["keep"], c["page"]
    planes = {k: s[k].double().cpu() for k in ("k_pages", "v_pages", "scores")}
    scores, pos, table = s["scores"].cpu(), s["pos"].cpu(), s["table"].cpu().long()
    to = table if s["out_table"] is None else s["out_table"].cpu().long()
    for b, n in enumerate(_lengths(c)):
        j = torch.arange(n)
        for h in range(c["hkv"]):
            score, place = scores[table[b, j // page], h, j % page], pos[table[b, j // page], h, j % page]
            # by (newest first, then score), lowest slot first among equals
            rank = sorted(range(n), key=lambda i, sc=score.tolist(), pl=place.tolist(): (
                pl[i] < n - c["recent"], -sc[i] if pl[i] < n - c["recent"] else 0.0, i))
            chosen = set(rank[:keep])
            spare = [i for i in range(keep, n) if i in chosen]
            source = [i if i in chosen else spare.pop(0) for i in range(min(n, keep))]
            frm, dst = torch.tensor(source, dtype=torch.long), torch.arange(len(source))
            for plane in planes.values():
                moved = plane[table[b, frm // page], h, frm % page]
                plane[to[b, dst // page], h, dst % page] = moved
    return {"lens": None, "pos": None, **planes}
