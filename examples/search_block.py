"""Searching with the decoder of decode_block.py: beam search, and decoding with drafted tokens.

    python examples/search_block.py                 # both, on a small model
    python examples/search_block.py --beams 8 --draft 16

Beam search: each step's logits through beam_select, and the cache's rows follow the beams (PagedKVCache.reorder).
Drafts: a drafter proposes a tree of tokens behind the last one; one pass checks them all (tree_attention under
PagedKVCache.attend_new), the line of the tree that the model itself would have taken stays (PagedKVCache.keep). The
result is the one of decoding token by token. The drafter here knows the model's own continuation and errs at random.
"""
from __future__ import annotations

import argparse
import importlib
import importlib.util
import os
import random
import sys

import torch

HERE = os.path.dirname(os.path.abspath(__file__))
sys.path.insert(0, os.path.dirname(HERE))
te = importlib.import_module("trellis-everywhere_amd")
_spec = importlib.util.spec_from_file_location("decode_block", os.path.join(HERE, "decode_block.py"))
block = importlib.util.module_from_spec(_spec)
_spec.loader.exec_module(block)


class Model:
    """Token ids in, logits out: a random embedding, the decoder's blocks, a packed head."""

    def __init__(self, rows, max_len, vocab=512, hidden=128, seed=0, device="cuda"):
        self.dec = block.Decoder(2, hidden, 2 * hidden, 4, 2, 64, rows, max_len, page_size=16, seed=seed, device=device)
        g = torch.Generator(device=device).manual_seed(seed + 1)
        self.table = torch.randn((vocab, hidden), generator=g, device=device)
        self.head = block.packed(vocab, hidden, g, device)
        self.cache, self.device = self.dec.cache, device

    def __call__(self, tokens, counts, depths=None, parents=None):
        """Logits [tokens, vocab] of each row's new tokens (ids, row by row)."""
        ids = torch.as_tensor(tokens, dtype=torch.long, device=self.device)
        if parents is not None:
            parents = torch.tensor(parents, dtype=torch.int32, device=self.device)
        return self.head(self.dec.forward(self.table[ids], counts, depths, parents)) * 3


def likeliest(logits):
    """The largest logit's token of each row."""
    return te.beam_select(logits[:, None], torch.zeros((logits.shape[0], 1), device=logits.device), 1)[2].flatten().tolist()


def decode(model, prompt, steps):
    """Token by token: the prompt in one pass, then each step's likeliest token."""
    out = [likeliest(model(prompt, [len(prompt)])[-1:])[0]]
    while len(out) < steps:
        out.append(likeliest(model([out[-1]], 1))[0])
    return out


def decode_drafted(model, prompt, steps, drafter):
    """The same by checking drafts. drafter(tokens so far) gives (ids, parents) of a tree whose first token, number 0,
    is the last one decided; returns the tokens and how many passes they took."""
    out, passes = [likeliest(model(prompt, [len(prompt)])[-1:])[0]], 1
    while len(out) < steps:
        ids, parents = drafter(out)
        depths = []
        for p in parents:
            depths.append(0 if p < 0 else depths[p] + 1)
        best, passes = likeliest(model(ids, [len(ids)], depths, parents)), passes + 1
        path = [0]
        while True:     # the child that the model would have taken
            child = [i for i, p in enumerate(parents) if p == path[-1] and ids[i] == best[path[-1]]]
            if not child:
                break
            path.append(child[0])
        model.cache.keep([path])
        out += [ids[i] for i in path[1:]] + [best[path[-1]]]
    return out[:steps], passes


def beam_search(model, prompt, beams, steps):
    """The beams' tokens [beams, steps] and scores; the model's cache has a row for each beam."""
    logits = model(prompt, [len(prompt)] + [0] * (beams - 1))[-1:]
    scores = torch.zeros((1, 1), device=logits.device)
    scores, _, tokens = te.beam_select(logits[None], scores, beams)
    model.cache.reorder([0] * beams)
    lines = [[t] for t in tokens[0].tolist()]
    while len(lines[0]) < steps:
        logits = model([line[-1] for line in lines], 1)
        scores, parents, tokens = te.beam_select(logits[None], scores, beams)
        parents = parents[0].tolist()
        model.cache.reorder(parents)
        lines = [lines[p] + [t] for p, t in zip(parents, tokens[0].tolist())]
    return lines, scores[0].tolist()


def noisy_drafter(truth, size, vocab, rng, right=0.8):
    """Drafts of `size` tokens that follow `truth` most of the time, with wrong branches beside it."""
    def draft(out):
        ids, parents = [out[-1]], [-1]
        on, at = 0, len(out)       # the node that is still right, and the next token there
        while len(ids) < size:
            good = at < len(truth) and rng.random() < right
            ids.append(truth[at] if good else rng.randrange(vocab))
            parents.append(on if good else rng.randrange(len(ids) - 1))
            if good:
                on, at = len(ids) - 1, at + 1
        return ids, parents
    return draft


def main():
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    for name, default in (("beams", 4), ("draft", 12), ("steps", 24), ("prompt", 20)):
        ap.add_argument("--" + name, type=int, default=default)
    a = ap.parse_args()
    rng = random.Random(0)
    prompt = [rng.randrange(512) for _ in range(a.prompt)]
    longest = a.prompt + a.steps + a.draft + 1
    plain = decode(Model(1, longest), prompt, a.steps)
    drafted, passes = decode_drafted(Model(1, longest), prompt, a.steps, noisy_drafter(plain, a.draft, 512, rng))
    print(f"token by token: {plain}")
    print(f"by drafts of {a.draft}: {passes} passes for {a.steps} tokens, {'the same' if drafted == plain else 'OTHER TOKENS'}")
    lines, scores = beam_search(Model(a.beams, longest), prompt, a.beams, a.steps)
    for line, score in zip(lines, scores):
        print(f"{score:9.3f}  {line}")


if __name__ == "__main__":
    main()
