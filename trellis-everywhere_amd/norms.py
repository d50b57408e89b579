"""The norms around a decoder block with its residual (trellis_residual_norm): what runs between one
packed linear's output and the next one's input (the reference's RMSNORM and ADD dispatches,
web/model.js:79, 96-97, 101). For serving: forward only.
"""
from __future__ import annotations

import torch

from . import _capi
from .packed_linear import _stream

_DT = {torch.float32: _capi.DT_F32, torch.float16: _capi.DT_F16, torch.bfloat16: _capi.DT_BF16}


def refuse_grad(*tensors) -> None:
    """The operators record no gradient: a tensor that wants one is refused, not silently detached."""
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise ValueError("forward only: call it under torch.no_grad() or detach the inputs")


def _rows(t: torch.Tensor) -> torch.Tensor:
    """[rows, width] with unit column stride."""
    if t.dim() != 2:
        t = t.reshape(-1, t.shape[-1])
    return t if t.stride(1) == 1 or t.shape[1] == 1 else t.contiguous()


def _weight(name, w, width, dev):
    if w.dtype != torch.float32 or w.shape != (width,) or w.device != dev or not w.is_contiguous():
        raise ValueError(f"{name} must be a contiguous float32 [{width}] tensor on {dev}")
    return w.data_ptr()


def _call(x, residual, weight, post_weight, gate, scale, eps, out_dtype, residual_out):
    refuse_grad(x, residual, weight, post_weight, gate)
    dev, shape, dt = x.device, x.shape, x.dtype
    if dev.type != "cuda":
        raise ValueError(f"the norms run on a GPU, not {dev}")
    if x.dim() == 0:
        raise ValueError("x must have at least one dim")
    width = shape[-1]
    xdt, ydt = _DT.get(dt), _DT.get(out_dtype if out_dtype is not None else dt)
    if xdt is None or ydt is None:
        raise ValueError(f"x dtype {dt} and out dtype {out_dtype} must be float32, float16 or bfloat16")
    x2 = _rows(x)
    rows = x2.shape[0]
    r_ptr = ldr = h_ptr = ldh = g_ptr = ldg = rdt = 0
    g_inner, h = 1, None
    if residual is not None:
        if residual.shape != shape or residual.device != dev:
            raise ValueError(f"residual must be {tuple(shape)} on {dev}")
        rdt = _DT.get(residual.dtype)
        if rdt is None:
            raise ValueError(f"residual dtype {residual.dtype} not supported")
        r2 = _rows(residual)
        if residual_out is None:
            h = torch.empty(shape, dtype=residual.dtype, device=dev)
        else:
            h = residual_out
            if h.shape != shape or h.dtype != residual.dtype or h.device != dev:
                raise ValueError("residual_out must have the residual's shape, dtype and device")
        h2 = h if h.dim() == 2 else h.view(-1, width)
        if h2.stride(1) != 1 and width != 1:
            raise ValueError("residual_out must have unit column stride")
        r_ptr, ldr, h_ptr, ldh = r2.data_ptr(), r2.stride(0), h2.data_ptr(), h2.stride(0)
    if gate is not None:
        if gate.dtype != dt or gate.device != dev:
            raise ValueError(f"gate must be {dt} on {dev}")
        g2 = gate.expand(shape)
        if g2.dim() != 2:
            g2 = g2.reshape(-1, width)
        g_inner = 0 if g2.stride(1) == 0 or width == 1 else 1
        if g_inner and g2.stride(1) != 1:
            g2 = g2.contiguous()
        g_ptr, ldg = g2.data_ptr(), g2.stride(0)
    w_ptr = _weight("weight", weight, width, dev)
    p_ptr = 0 if post_weight is None else _weight("post_weight", post_weight, width, dev)
    y = torch.empty(shape, dtype=dt if out_dtype is None else out_dtype, device=dev)
    st = _capi.load().trellis_residual_norm(
        x2.data_ptr(), x2.stride(0), xdt, r_ptr, ldr, rdt, g_ptr, ldg, g_inner, p_ptr, w_ptr, scale, eps,
        h_ptr, ldh, y.data_ptr(), width, ydt, rows, width, _stream(dev))
    if st:
        _capi.check(st)
    return y, h


def rms_norm(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6,
             out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """x * rsqrt(mean(x^2) + eps) * weight over the last dim (float32, float16 or bfloat16 x of any
    leading shape, float32 weight), computed in fp32 and rounded once to out_dtype (x's if None)."""
    return _call(x, None, weight, None, None, 1.0, eps, out_dtype, None)[0]


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
    return _call(x, residual, weight, post_weight, gate, scale, eps, out_dtype, residual_out)
