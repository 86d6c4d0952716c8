"""Root-mean-square norm of rows with the residual's addition, in one launch, forward and backward, and with its output in 8 bits
(``scenerf_hip_rms_*``, csrc/norm.hip).

The reference's ResnetFC adds its branches without a norm (scenerf/models/resnetfc.py:57-64, 150-160); deeper or narrower-typed nets
want one in front of every block.  The addition belongs to the same pass over the row::

    y, h = rms_norm(x, weight, residual=h)             # h = x + h, y = h / sqrt(mean(h^2) + eps) * weight
    q, scale, h = rms_norm_8bit(x, weight, residual=h) # y as rows of e4m3 with one fp32 scale each: what linear_8bit reads

float32, bfloat16, float16; the row's sum, the norm and every value up to its one rounding are held in 32 bits (y is made from the
unrounded h).  CUDA tensors only: anything else raises, there is no fallback.
"""
from __future__ import annotations

from typing import Optional, Tuple, Union

import torch
import torch.autograd.forward_ad as forward_ad
import torch.nn as nn
from torch.autograd.function import once_differentiable

from .rowops import MAX_ROWS, RMS, TYPE_CODES, check_float, check_tensors, no_gradient, no_tangent, rows_forward, rows_of, run_rows, together, vector_of


def _check(what, x, weight, residual, eps) -> None:
    shape = x.shape
    if forward_ad._current_level >= 0:
        no_tangent(what, x, weight, residual)
    if not together(x, weight, residual):
        check_tensors(what, x.device, x.dtype, ("weight", weight), ("residual", residual))
    check_float(what, "x", x.dtype)
    if len(shape) < 1 or shape[-1] < 1:
        raise ValueError("%s: x must have at least one column (got %s)" % (what, tuple(shape)))
    if weight.shape != (shape[-1],):
        raise ValueError("%s: weight must be (%d,) (got %s)" % (what, shape[-1], tuple(weight.shape)))
    if residual is not None and residual.shape != shape:
        raise ValueError("%s: residual must be %s (got %s); expand it first if it is to be broadcast" % (what, tuple(shape), tuple(residual.shape)))
    if not eps >= 0.0:
        raise ValueError("%s: eps must not be negative (got %r)" % (what, eps))
    if x.numel() // shape[-1] > MAX_ROWS:
        raise ValueError("%s: more than 2^31 - 1025 rows" % what)


def rms_step_back(h: torch.Tensor, weight: torch.Tensor, rstd: torch.Tensor, eps: float, dy: torch.Tensor, dh: Optional[torch.Tensor],
                  need_x: bool, need_w: bool, residual: Optional[torch.Tensor] = None, sums: bool = False):
    """(gradient of h, gradient of weight), None where not needed; h as the forward stored it (or its x, with its ``residual``), ``dh`` what
    else flows into it.  ``sums``: the weight's in fp32, not rounded to its type."""
    if forward_ad._current_level >= 0:
        no_tangent("rms_norm's step back", dy, dh)
    width, dev = h.shape[-1], h.device
    h2, dy2, w = rows_of(h, width), rows_of(dy, width), vector_of(weight, width)
    dh2 = rows_of(dh, width) if dh is not None else None
    r2 = rows_of(residual, width) if residual is not None else None
    dx = dy.new_empty(dy.shape) if need_x else None
    dw = torch.empty(width, dtype=torch.float32 if sums else dy.dtype, device=dev) if need_w else None
    run_rows("rms", True, RMS.pack(
        TYPE_CODES[h.dtype], width, h2.shape[0], eps, int(sums), h2.data_ptr(), h2.stride(0), 0 if r2 is None else r2.data_ptr(),
        0 if r2 is None else r2.stride(0), w.data_ptr(), 0, 0, 0, 0, rstd.data_ptr(),
        dy2.data_ptr(), dy2.stride(0), 0 if dh2 is None else dh2.data_ptr(), 0 if dh2 is None else dh2.stride(0),
        0 if dx is None else dx.data_ptr(), 0 if dw is None else dw.data_ptr(), 0, 0), dev, "rms_norm backward")
    return dx, dw


class _RmsNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, residual, eps):
        y, _, h, rstd, x2 = rows_forward("rms_norm", x, weight, residual, eps, keep_rstd=True)
        ctx.eps, ctx.has_residual = eps, residual is not None
        ctx.set_materialize_grads(False)
        if residual is None:
            ctx.save_for_backward(x2, weight, rstd, None)
            return y
        if x.dtype == torch.float32:
            ctx.save_for_backward(h, weight, rstd, None)
        else:
            # 16 bits: the gradients are made from x + residual once more, not from h as it was stored, whose rounding made dweight half as
            # inexact again as its own does (153,600 x 512 bf16, passes in a row: 118 us from h, 147 so)
            ctx.save_for_backward(x2, weight, rstd, residual)
        return y, h

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dh=None):
        h, weight, rstd, residual = ctx.saved_tensors
        need_h = ctx.needs_input_grad[0] or (ctx.has_residual and ctx.needs_input_grad[2])
        if dy is None:               # only h was used
            dx, dw = dh, torch.zeros_like(weight) if ctx.needs_input_grad[1] and dh is not None else None
        else:
            dx, dw = rms_step_back(h, weight, rstd, ctx.eps, dy, dh, need_h, ctx.needs_input_grad[1], residual)
        return dx if ctx.needs_input_grad[0] else None, dw, dx if ctx.has_residual and ctx.needs_input_grad[2] else None, None


def rms_norm(x: torch.Tensor, weight: torch.Tensor, *, residual: Optional[torch.Tensor] = None,
             eps: float = 1e-6) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """``y = h / sqrt(mean(h^2) + eps) * weight`` over the last dimension, h = x (+ residual): x and residual (..., width), weight
    (width,), all of one type.  Returns y, or ``(y, h)`` where a residual is added: h is the next residual stream.  Differentiable once,
    in reverse, in x, weight and residual (one gradient serves x and residual); none of x, residual and h may change before the backward pass."""
    _check("rms_norm", x, weight, residual, eps)
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad or (residual is not None and residual.requires_grad)):
        return _RmsNorm.apply(x, weight, residual, float(eps))
    y, _, h, _, _ = rows_forward("rms_norm", x, weight, residual, float(eps))
    return y if residual is None else (y, h)


def rms_norm_8bit(x: torch.Tensor, weight: torch.Tensor, *, residual: Optional[torch.Tensor] = None, eps: float = 1e-6):
    """``rms_norm`` with y as rows of e4m3: returns ``(q, scale)``, or ``(q, scale, h)`` where a residual is added; q (..., width)
    float8_e4m3fn, scale (...) float32 = max(max|y| / 448, 2^-126), made from the unrounded y (``quantize_rows`` says what q and scale
    stand for).  Forward only."""
    _check("rms_norm_8bit", x, weight, residual, eps)
    no_gradient("rms_norm_8bit", x, weight, residual)
    q, scale, h, _, _ = rows_forward("rms_norm_8bit", x, weight, residual, float(eps), quantize=True)
    return (q, scale) if residual is None else (q, scale, h)


class RMSNorm(nn.Module):
    """``rms_norm`` with its weight: ``forward(x)`` -> y, ``forward(x, residual)`` -> (y, h)."""

    def __init__(self, width: int, eps: float = 1e-6):
        super().__init__()
        self.weight, self.eps = nn.Parameter(torch.ones(width)), eps

    def forward(self, x: torch.Tensor, residual: Optional[torch.Tensor] = None):
        return rms_norm(x, self.weight, residual=residual, eps=self.eps)
