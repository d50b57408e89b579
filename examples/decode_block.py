"""Decoding through decoder blocks that run in this package alone: packed linears, the norms around them,
and a paged key-value cache with its attention and eviction.

    python examples/decode_block.py                      # a small model, checked against plain torch
    python examples/decode_block.py --blocks 4 --hidden 4096 --ffn 12288 --heads 32 --kv-heads 8 --tokens 64

The weights are random packed words (what an encoder's output looks like). The blocks are pre-norm with
per-head norms of q and k and rotary positions:

    y = norm(h);  q, k, v = linear(y);  h += o(attention(rot(norm(q)), cache))
    y = norm(h);  gate, up = linear(y); h += down(silu(gate) * up)
"""
from __future__ import annotations

import argparse
import importlib
import os
import sys
import time

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
te = importlib.import_module("trellis-everywhere_amd")


def packed(n, k, g, device, K=3):
    """A packed linear of random words: unit-variance weights in z-space, scaled to keep |W x| ~ |x|."""
    bits = torch.randint(-2 ** 31, 2 ** 31 - 1, (n // 16 * (k // 16), 8 * K), generator=g, device=device, dtype=torch.int32)
    signs = [torch.randint(0, 2, (m,), generator=g, device=device).float() * 2 - 1 for m in (k, n)]
    return te.PackedLinear.from_device(n, k, K, bits, signs[0], signs[1], torch.full((k,), k ** -0.5, device=device),
                                       torch.ones(n, device=device))


class DecoderBlock:
    def __init__(self, hidden, ffn, heads, kv_heads, head_dim, g, device):
        self.heads, self.kv_heads, self.head_dim = heads, kv_heads, head_dim
        self.linears = {name: packed(n, k, g, device) for name, n, k in (
            ("q", heads * head_dim, hidden), ("k", kv_heads * head_dim, hidden), ("v", kv_heads * head_dim, hidden),
            ("o", hidden, heads * head_dim), ("gate", ffn, hidden), ("up", ffn, hidden), ("down", hidden, ffn))}
        pick = lambda names: [self.linears[n] for n in names]
        self.qkv, self.gate_up = te.PackedGroup(pick("qkv")), te.PackedGroup(pick(("gate", "up")))
        weight = lambda n: torch.rand(n, generator=g, device=device) + 0.5
        self.attn_norm, self.ffn_norm = weight(hidden), weight(hidden)
        self.q_norm, self.k_norm = weight(head_dim), weight(head_dim)


class Decoder:
    """`rows` sequences decoded together, their cache held at `budget` tokens each if given."""

    def __init__(self, blocks, hidden, ffn, heads, kv_heads, head_dim, rows, max_len, budget=None, recent=16,
                 page_size=16, seed=0, device="cuda"):
        g = torch.Generator(device=device)
        g.manual_seed(seed)
        self.blocks = [DecoderBlock(hidden, ffn, heads, kv_heads, head_dim, g, device) for _ in range(blocks)]
        self.final_norm = torch.ones(hidden, device=device)
        freq = 1e6 ** (-torch.arange(0, head_dim, 2, dtype=torch.float64, device=device) / head_dim)
        angle = torch.arange(max_len, dtype=torch.float64, device=device)[:, None] * freq
        self.cos, self.sin = angle.cos().float(), angle.sin().float()
        self.budget, self.recent = budget, recent
        self.cache = te.PagedKVCache(blocks, kv_heads, head_dim, rows=rows, max_len=budget + 1 if budget else max_len,
                                     page_size=page_size, device=device, evictable=budget is not None)

    def step(self, h):
        """One token's hidden states h [rows, hidden] (f32) through the blocks; the normed output [rows, hidden]."""
        return self.forward(h, 1)

    @torch.no_grad()
    def forward(self, h, counts, depths=None, parents=None):
        """Hidden states of counts[b] new tokens for each row b (an int: for every row), row by row, h [tokens, hidden]
        (f32): prompts, or (depths, parents: PagedKVCache.grow and attend_new) drafted tokens in a tree."""
        cache, n = self.cache, h.shape[0]
        cache.grow(counts, depths)
        several = not isinstance(counts, int) or counts > 1 or depths is not None
        first = self.blocks[0]
        y = te.rms_norm(h, first.attn_norm, out_dtype=torch.float16)
        for i, b in enumerate(self.blocks):
            q, k, v = (t.view(n, -1, b.head_dim) for t in b.qkv([y, y, y], out_dtype=torch.float16))
            q = cache.append(i, q, k, v, q_norm=b.q_norm, k_norm=b.k_norm, cos=self.cos, sin=self.sin)
            x = (cache.attend_new(i, q, parents=parents) if several else cache.attend(i, q)).view(n, -1)
            y, h = te.residual_norm(b.linears["o"](x), h, b.ffn_norm, out_dtype=torch.float16)
            gate, up = b.gate_up([y, y])
            x = b.linears["down"]((torch.nn.functional.silu(gate) * up).half())
            last = i + 1 == len(self.blocks)
            y, h = te.residual_norm(x, h, self.final_norm if last else self.blocks[i + 1].attn_norm,
                                    out_dtype=torch.float32 if last else torch.float16)
        if self.budget:
            cache.evict(self.budget, min(self.recent, self.budget))
        return y


def reference_step(dec, h, past):
    """The same step in plain float64 torch over a contiguous cache `past` (no eviction)."""
    def norm(x, w):
        return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6) * w.double()

    h = h.double()
    rows = h.shape[0]
    for i, b in enumerate(dec.blocks):
        eye = lambda name: past.setdefault((i, name), dec_dense(b.linears[name]))
        y = norm(h, b.attn_norm)
        q, k, v = ((y @ eye(n).t()).view(rows, -1, b.head_dim) for n in "qkv")
        q, k = norm(q, b.q_norm), norm(k, b.k_norm)
        at = past.get((i, "len"), 0)
        c, s = dec.cos[at].double(), dec.sin[at].double()
        half = b.head_dim // 2
        turn = lambda x: torch.cat([x[..., :half] * c - x[..., half:] * s, x[..., half:] * c + x[..., :half] * s], -1)
        k, v = turn(k)[:, :, None], v[:, :, None]
        if at:
            k, v = torch.cat([past[i, "K"], k], 2), torch.cat([past[i, "V"], v], 2)
        past[i, "K"], past[i, "V"], past[i, "len"] = k, v, at + 1
        group = b.heads // b.kv_heads
        w = torch.softmax((k.repeat_interleave(group, 1) * turn(q)[:, :, None]).sum(-1) * b.head_dim ** -0.5, -1)
        x = (w[..., None] * v.repeat_interleave(group, 1)).sum(2).reshape(rows, -1)
        h = h + x @ eye("o").t()
        y = norm(h, b.ffn_norm)
        h = h + (torch.nn.functional.silu(y @ eye("gate").t()) * (y @ eye("up").t())) @ eye("down").t()
    return norm(h, dec.final_norm)


def dec_dense(lin):
    """W_hat of a packed linear in float64, column by column through the linear itself."""
    return lin(torch.eye(lin.k_in, device=lin.device)).t().double().contiguous()


def main():
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    for name, default in (("blocks", 2), ("hidden", 256), ("ffn", 512), ("heads", 8), ("kv-heads", 2), ("head-dim", 128),
                          ("rows", 4), ("tokens", 40), ("budget", 0)):
        ap.add_argument("--" + name, type=int, default=default)
    a = ap.parse_args()
    dec = Decoder(a.blocks, a.hidden, a.ffn, a.heads, a.kv_heads, a.head_dim, a.rows, a.tokens, budget=a.budget or None)
    g = torch.Generator(device="cuda")
    g.manual_seed(1)
    h = [torch.randn((a.rows, a.hidden), generator=g, device="cuda") for _ in range(a.tokens)]
    check = a.hidden <= 1024 and not a.budget
    past, worst = {}, 0.0
    torch.cuda.synchronize()
    began = time.perf_counter()
    out = [dec.step(x) for x in h]
    torch.cuda.synchronize()
    took = time.perf_counter() - began
    if check:
        for x, y in zip(h, out):
            want = reference_step(dec, x, past)
            worst = max(worst, float((y - want).norm() / want.norm()))
        print(f"against float64 torch: largest relative error of {a.tokens} tokens {worst:.2e}")
    print(f"{a.tokens} tokens x {a.rows} rows through {a.blocks} blocks: {1e6 * took / a.tokens:.0f} us a token, "
          f"cached {dec.cache.lengths}")
    if check and not worst < 2e-2:
        sys.exit("the decoder differs from the reference")


if __name__ == "__main__":
    main()
