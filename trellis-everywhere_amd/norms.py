"""The norms around a decoder block with its residual (trellis_residual_norm): what runs between one
packed linear's output and the next one's input (the reference's RMSNORM and ADD dispatches,
within web/model.js:77-102). For serving: forward only. Arguments are checked in csrc/bind.cpp.
"""
from __future__ import annotations

import torch

from . import _capi


def rms_norm(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6,
             out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """x * rsqrt(mean(x^2) + eps) * weight over the last dim (float32, float16 or bfloat16 x of any
    leading shape, float32 weight), computed in fp32 and rounded once to out_dtype (x's if None)."""
    y = _capi.serve().residual_norm(x, None, weight, None, None, 1.0, eps, out_dtype, None)
    if y.__class__ is int:
        _capi.check(y)
    return y


def residual_norm(x: torch.Tensor, residual: torch.Tensor, weight: torch.Tensor, *,
                  post_weight: torch.Tensor | None = None, gate: torch.Tensor | None = None,
                  scale: float = 1.0, eps: float = 1e-6, out_dtype: torch.dtype | None = None,
                  residual_out: torch.Tensor | None = None):
    """A block's output x joins the residual stream, and the stream is normed for the next block:

        b = x, or rms_norm(x, post_weight)           (post_weight: a norm after the block)
        h = residual + scale * gate * b              (gate: x's dtype, broadcast against x)
        y = rms_norm(h, weight)                      (of h before it is rounded)

    Returns (y, h): y in out_dtype (x's if None), h in the residual's dtype, written to residual_out
    if given (the residual itself, for a stream that is updated in place)."""
    if residual is None:
        raise ValueError("residual must be a tensor (rms_norm is the norm without one)")
    yh = _capi.serve().residual_norm(x, residual, weight, post_weight, gate, scale, eps, out_dtype, residual_out)
    if yh.__class__ is int:
        _capi.check(yh)
    return yh
