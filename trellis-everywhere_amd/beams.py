"""Beam search's selection (trellis_beam_select): the step between a model's logits and the next tokens of its beams,
whose cached sequences PagedKVCache.reorder() then follows. No reference counterpart: it samples one sequence
(web/model.js:77-102). For serving: forward only. Arguments are checked in csrc/bind.cpp.
"""
from __future__ import annotations

import torch

from . import _capi


def beam_select(logits: torch.Tensor, scores: torch.Tensor, k: int, *, ended: torch.Tensor | None = None,
                end_token: int = 0, workspace: torch.Tensor | None = None):
    """The k best continuations of each batch element's beams, best first:

        c(j, v) = scores[j] + log_softmax(logits[j])[v]          (beam j, token v)
        an ended beam offers (j, end_token) alone, at scores[j]; its logits are not read

    equal candidates by the lower beam, then the lower token. A candidate that is -inf or NaN is none (a banned token has
    logit -inf, a beam not yet in use score -inf); where fewer than k are left, the rest are (-inf, beam 0, end_token).

    logits: [batch, beams, vocab] float32, float16 or bfloat16, any batch and beam strides, below +inf
    scores: float32 [batch, beams]; ended: bool [batch, beams]; beams and k up to 64
    Returns (scores float32, beams int32, tokens int32), each [batch, k]. The scores are formed in 64 bits on fp32
    exponentials' sums (within 5e-6, mostly some 1e-7: two beams' candidates nearer than twice that may change places; a
    beam's own keep the order of their logits) and rounded once (below float32's lowest value to -inf). k = 1 of one beam is
    the likeliest token and its log-probability.
    workspace: scratch for a caller that keeps its own, as for paged_attention."""
    r = _capi.serve().beam_select(logits, scores, k, ended, end_token, workspace)
    if r.__class__ is int:
        _capi.check(r)
    return r
