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
    for t in tensors:
        if t is not None and t.requires_grad and torch.is_grad_enabled():
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
    # (most of a small call's time is this function's: attributes are read once, and a tensor that is already
    # [rows, width] and contiguous, as a decode loop's are, goes through without a view)
    refuse_grad(x, residual, weight, post_weight, gate)
    dev, shape, dt = x.device, x.shape, x.dtype
    if dev.type != "cuda":
        raise ValueError(f"the norms run on a GPU, not {dev}")
    if not shape:
        raise ValueError("x must have at least one dim")
    if out_dtype is None:
        out_dtype = dt
    width, xdt, ydt = shape[-1], _DT.get(dt), _DT.get(out_dtype)
    if xdt is None or ydt is None:
        raise ValueError(f"x dtype {dt} and out dtype {out_dtype} must be float32, float16 or bfloat16")
    plain = len(shape) == 2 and x.is_contiguous()
    x2 = x if plain else _rows(x)
    rows, ldx = x2.shape[0], width if plain else x2.stride(0)
    r_ptr = ldr = h_ptr = ldh = g_ptr = ldg = rdt = 0
    g_inner, h = 1, None
    if residual is not None:
        rt = residual.dtype
        rdt = _DT.get(rt)
        if rdt is None:
            raise ValueError(f"residual dtype {rt} not supported")
        if residual.shape != shape or residual.device != dev:
            raise ValueError(f"residual must be {tuple(shape)} on {dev}")
        r2 = residual if plain and residual.is_contiguous() else _rows(residual)
        r_ptr, ldr = r2.data_ptr(), r2.stride(0)
        if residual_out is None:
            h = torch.empty_like(x, dtype=rt) if plain else torch.empty(shape, dtype=rt, device=dev)
            h_ptr, ldh = h.data_ptr(), width
        else:
            h = residual_out
            if h.shape != shape or h.dtype != rt or h.device != dev:
                raise ValueError("residual_out must have the residual's shape, dtype and device")
            h2 = h if len(shape) == 2 else h.view(-1, width)
            if h2.stride(1) != 1 and width != 1:
                raise ValueError("residual_out must have unit column stride")
            h_ptr, ldh = h2.data_ptr(), h2.stride(0)
    if gate is not None:
        if gate.dtype != dt or gate.device != dev:
            raise ValueError(f"gate must be {dt} on {dev}")
        if not plain or gate.shape != shape or not gate.is_contiguous():
            gate = gate.expand(shape)
            if len(shape) != 2:
                gate = gate.reshape(-1, width)
            g_inner = 0 if gate.stride(1) == 0 or width == 1 else 1
            if g_inner and gate.stride(1) != 1:
                gate = gate.contiguous()
        g_ptr, ldg = gate.data_ptr(), gate.stride(0)
    w_ptr = _weight("weight", weight, width, dev)
    p_ptr = 0 if post_weight is None else _weight("post_weight", post_weight, width, dev)
    y = torch.empty_like(x, dtype=out_dtype) if plain else torch.empty(shape, dtype=out_dtype, device=dev)
    st = _capi.load().trellis_residual_norm(
        x2.data_ptr(), ldx, xdt, r_ptr, ldr, rdt, g_ptr, ldg, g_inner, p_ptr, w_ptr, scale, eps, h_ptr, ldh,
        y.data_ptr(), width, ydt, rows, width, _stream(dev))
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
