"""What the attention kernel's arithmetic may err by, from each result's own quantities, and a restatement of that
arithmetic on the CPU into which a mistake can be planted.

The kernel, per query head: q as NQ terms of the cache's type (exact products, fp32 sums), logits times scale log2(e),
weights 2^(s - m) in fp32, as NP terms of the cache's type against v (exact products, fp32 sums), their fp32 sum. u is
2^-24, half an ulp of fp32; a matrix instruction's additions, whose rounding is not documented, count 2 u each.

  q's split     f16: two terms leave 2^-22 of an element and, below f16's normal range, 2^-25 in units in which the
                row's largest is at least 2^14: 2^-39 of it. bf16: three terms leave 2^-26. If q has the type, only
                the 2^-39.
  logit j       scale sum_i (split of q_i) |k_i| + 2 u NQ (products) A_j + 4 u |S_j|,  A_j = scale sum |q_i k_i|
                (scale, log2(e), their product and the logit are rounded)
  weight j      u |S_j - max| (s - m) + 2 u (2^x) + 2 u a rescale, of which a row of up to 32 tokens has none, another one
                for each 128 tokens (a wave's tiles) and 6 where waves and chunks join
  its split     f16: 2^-22 of it and 2^-36 of the largest (2^-25 where that is at least 2^11); bf16: 2^-26 in three terms
  sums          2 u NP n of sum p |v| and u n of the weights' sum; the division 2 u."""
import math

import torch

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
U = 2.0 ** -24


def terms(x, cache, y):
    """(NQ, NP) where q or out is of another type than the cache's, or out is fp32."""
    assert x != cache or y == F32
    return (2, 2) if cache == F16 else (3, 3)


def inputs(lengths, heads, group, d, x, cache, seed, keys="dense", outlier=0.0):
    """q [rows, hq, d], and (k, v) [heads, n, d] of each row. keys "one": one nonzero dim each, so that a logit is one
    product. outlier: one dim of every query this much larger than the others, facing keys as much smaller."""
    g = torch.Generator().manual_seed(seed)
    q = torch.randn((len(lengths), heads * group, d), generator=g)
    big = torch.arange(d) == d // 2
    if outlier:
        q[..., big] = outlier * (1 + torch.rand((len(lengths), heads * group, 1), generator=g))
    kv = []
    for n in lengths:
        k, v = torch.randn((heads, n, d), generator=g), torch.randn((heads, n, d), generator=g)
        if keys == "one":
            at = torch.randint(0, d, (heads, n, 1), generator=g)
            k = torch.zeros_like(k).scatter_(-1, at, k.gather(-1, at) * d ** 0.5)
            v = v * (torch.rand(v.shape, generator=g) < 0.5)
        if outlier:
            k[..., big] *= 0.05 / outlier
        kv.append((k.to(cache), v.to(cache)))
    return q.to(x), kv


def exact(q, k, v, scale):
    """One query head in float64: out, weights, logits."""
    s = k.double() @ q.double() * scale
    p = torch.softmax(s, 0)
    return p @ v.double(), p, s


def bound(q, k, v, scale, x, cache, y):
    """Per element of one query head's out: the most that the kernel's arithmetic may err by, before out's rounding."""
    out, p, s = exact(q, k, v, scale)
    nq, np_ = terms(x, cache, y)
    n, q, k, v = k.shape[0], q.double().abs(), k.double().abs(), v.double().abs()
    left = torch.zeros_like(q) if x == cache else q * (2.0 ** -22 if cache == F16 else 2.0 ** -26)
    if cache == F16:
        left = left + 2.0 ** -39 * q.max()
    logit = scale * (k @ left) + 2 * U * nq * (k * q != 0).sum(-1) * (scale * (k @ q)) + 4 * U * s.abs()
    scales = 0 if n <= 32 else -(-n // 128) + 6
    weight = logit + U * (s.max() - s) + 2 * U + 2 * U * scales
    split = (2.0 ** -22 * p + 2.0 ** -36 * p.max()) if cache == F16 else 2.0 ** -26 * p
    pv = p @ v
    return (p * weight) @ v + (p @ weight) * out.abs() + split @ v + 2 * U * np_ * n * pv + U * (n + 2) * out.abs()


def split(x, dtype, count):
    parts = []
    for _ in range(count):
        part = x.to(dtype).float()
        parts.append(part)
        x = x - part
    return parts


def kernel(q, k, v, scale, x, cache, y, mistake=None):
    """The kernel's arithmetic on one query head. mistake: "q" or "p" (the last term of the split is lost), "low" (q's
    largest element to [0.5, 1) before its split)."""
    nq, np_ = terms(x, cache, y)
    up = 15 if cache == F16 and mistake != "low" else 0
    e = math.frexp(float(q.abs().max()))[1] if float(q.abs().max()) else 0
    parts = split(torch.ldexp(q.float(), torch.tensor(up - e)), cache, nq - (mistake == "q"))
    acc = sum((k.double() @ t.double()).float() for t in parts)
    fold = torch.ldexp(torch.tensor(scale, dtype=F32) * torch.tensor(1.44269504, dtype=F32), torch.tensor(e - up))
    s = acc * fold
    w = torch.exp2((s - (s.max() - 11)).double()).float()
    o = sum((t.double() @ v.double()).float() for t in split(w, cache, np_ - (mistake == "p")))
    return o * (1 / w.sum())
