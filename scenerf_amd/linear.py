"""A linear layer with its epilogue in one launch, forward and backward, and its 8-bit form (``scenerf_hip_linear_*``, csrc/linear.hip).

The reference's ResnetFC is ``nn.Linear`` + activation + addition, each a pass over the rows (scenerf/models/resnetfc.py:49-64, 146-163).
Here one call is one product with all of that behind its sums::

    y = linear(x, weight, bias, activation="gelu", residual=h)        # act(x @ weight.T + bias) + h, differentiable in every input
    q, s = quantize_rows(x)                                           # rows in e4m3 with one fp32 scale each
    y = linear_8bit(q, s, wq, ws, bias, activation="gelu", residual=h)

float32 (fp32 matrix instructions), bfloat16 and float16 operands, 32-bit sums (``linear_8bit`` with a bfloat16 result: see there), every output rounded once.  Rows are whatever precedes
the last dimension, zero rows included; a row's elements must be neighbours in memory (other layouts are copied first), its pitch is
free.  CUDA tensors only: anything else raises, there is no fallback.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch
import torch.autograd.forward_ad as forward_ad
from torch.autograd.function import once_differentiable

from . import _capi
from .rowops import LINEAR, MAX_ROWS, TYPE_CODES, check_float, check_tensors, no_gradient, no_tangent, rows_forward, rows_of, run_on, run_rows, together, vector_of


def _activation(name: str) -> int:
    code = _capi.ACTIVATIONS.get(name)
    if code is None:
        raise ValueError("activation must be one of %s (got %r)" % (", ".join(sorted(_capi.ACTIVATIONS)), name))
    return code


def _check_shapes(what, x, weight, bias, residual):
    if weight.dim() != 2 or weight.shape[0] < 1 or weight.shape[1] < 1:
        raise ValueError("%s: weight must be (n, k) with n, k >= 1 (got %s)" % (what, tuple(weight.shape)))
    n, k = weight.shape
    xs = x.shape
    if len(xs) < 1 or xs[-1] != k:
        raise ValueError("%s: x must end in %d features (got %s)" % (what, k, tuple(xs)))
    shape = (xs[0], n) if len(xs) == 2 else xs[:-1] + (n,)
    if bias is not None and bias.shape != (n,):
        raise ValueError("%s: bias must be (%d,) (got %s)" % (what, n, tuple(bias.shape)))
    if residual is not None and residual.shape != shape:
        raise ValueError("%s: residual must be %s (got %s); expand it first if it is to be broadcast" % (what, tuple(shape), tuple(residual.shape)))
    if x.numel() // k > MAX_ROWS:
        raise ValueError("%s: more than 2^31 - 1025 rows" % what)
    return shape


def _in_pieces(x2: torch.Tensor, w2: torch.Tensor, back: bool = False):
    """(x's pointer, its pitch, w's pointer, its pitch, padded, what holds them): the two as the kernels read them fast, 16 bytes at a time --
    as they are, or both copied into one buffer with zeros behind each row.  Up to 8 rows are read from any address; the step ``back`` is not."""
    es, rows = x2.element_size(), x2.shape[0]
    xp, wp, ldx, ldw = x2.data_ptr(), w2.data_ptr(), x2.stride(0), w2.stride(0)
    if (rows <= 8 and not back) or not (w2.shape[1] | ldx | ldw) * es & 15 | (xp | wp) & 15:
        return xp, ldx, wp, ldw, 0, (x2, w2)
    (n, k), dev, dtype = w2.shape, x2.device, x2.dtype
    pitch = -(-k * es // 16) * 16 // es
    both = torch.empty((rows + n) * pitch, dtype=dtype, device=dev)
    to = both.data_ptr()
    run_on(dev, _capi.load().scenerf_hip_linear_pad, (_capi.T_E4M3 if es == 1 else TYPE_CODES[dtype], k, xp if rows else None, ldx, rows,
                                                      to if rows else None, wp, ldw, n, to + rows * pitch * es), "linear (padding)")
    return to, pitch, to + rows * pitch * es, pitch, 1, (both, None)


def _forward(what, pieces, rows, n, k, bias, residual, shape, in_type, out_dtype, dev, act, keep_z, scales=None):
    y = torch.empty(shape, dtype=out_dtype, device=dev)
    z = y.new_empty((rows, n)) if keep_z else None
    if bias is not None:
        bias = vector_of(bias, n)
    r = rows_of(residual, n) if residual is not None else None
    xp, ldx, wp, ldw, padded, _ = pieces
    run_rows("linear", False, LINEAR.pack(
        in_type, TYPE_CODES[out_dtype], act, n, k, padded, rows, xp, ldx, wp, ldw, 0 if scales is None else scales[0].data_ptr(),
        0 if scales is None else scales[1].data_ptr(), 0 if bias is None else bias.data_ptr(), 0 if r is None else r.data_ptr(),
        0 if r is None else r.stride(0), y.data_ptr(), 0 if z is None else z.data_ptr(), 0, 0, 0, 0, 0, 0, 0), dev, what)
    return y, z


def linear_step(x: torch.Tensor, weight: torch.Tensor, bias, residual, act: int, shape, keep_z: bool):
    """(y, what ``linear_step_back`` needs) of a layer that will be differentiated; no checks, no autograd."""
    n, k = weight.shape
    x2 = rows_of(x, k)
    rows = x2.shape[0]
    pieces = _in_pieces(x2, rows_of(weight, k), True)
    y, z = _forward("linear", pieces, rows, n, k, bias, residual, shape, TYPE_CODES[x.dtype], x.dtype, x.device, act, keep_z)
    # (x and w or the one copy of both, z; then numbers)
    return y, (*pieces[5], z, rows, n, k, pieces[1], pieces[4], act)


def linear_step_back(saved, dy: torch.Tensor, x_shape, need_x: bool, need_w: bool, need_b: bool, sums: bool = False):
    """(dx, dweight, dbias), None where not needed.  ``sums``: dweight and dbias in fp32, not rounded to their type."""
    if forward_ad._current_level >= 0:
        no_tangent("linear's step back", dy)
    x2, w2, z, rows, n, k, pitch, padded, act = saved
    dev = dy.device
    # (dy is of x's type: autograd sees to it; new_empty takes less of the host's time than empty)
    dx = dy.new_empty(x_shape) if need_x else None
    kind = torch.float32 if sums else dy.dtype
    dw = dy.new_empty((n, k), dtype=kind) if need_w else None
    db = dy.new_empty(n, dtype=kind) if need_b else None
    dy2 = rows_of(dy, n)
    code, xp = TYPE_CODES[x2.dtype], x2.data_ptr()
    if padded:
        ldx, wp, ldw = pitch, xp + rows * pitch * x2.element_size(), pitch
    else:       # (where a hook on saved tensors has moved them, their pitch may be another)
        ldx, wp, ldw = x2.stride(0), w2.data_ptr(), w2.stride(0)
    run_rows("linear", True, LINEAR.pack(
        code, _capi.T_F32 if sums else code, act, n, k, padded, rows, xp, ldx, wp, ldw, 0, 0, 0, 0, 0, 0, 0 if z is None else z.data_ptr(), dy2.data_ptr(), dy2.stride(0),
        0 if dx is None else dx.data_ptr(), 0 if dw is None else dw.data_ptr(), 0 if db is None else db.data_ptr(), 0, 0), dev, "linear backward")
    return dx, dw, db


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, act, shape):
        y, saved = linear_step(x, weight, bias, residual, act, shape, act != _capi.ACTIVATIONS["none"] and any(ctx.needs_input_grad[:3]))
        ctx.save_for_backward(*saved[:3])
        ctx.rest, ctx.x_shape = saved[3:], x.shape
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        need = ctx.needs_input_grad
        grads = (None, None, None)
        if any(need[:3]):
            grads = linear_step_back(ctx.saved_tensors + ctx.rest, dy, ctx.x_shape, *need[:3])
        return grads + (dy if need[3] else None, None, None)


def linear(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, *, activation: str = "none",
           residual: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``act(x @ weight.T + bias) + residual``: x (..., k), weight (n, k), bias (n,), residual (..., n), all of one type -> (..., n).

    ``activation``: "none", "relu", "gelu" (the exact one, by erf) or "silu".  Sums, bias, activation and addition are in 32 bits; the
    result is rounded once.  Differentiable once, in reverse, in x, weight, bias and residual; where an activation is asked for and a gradient will
    be, the sums in front of it are kept in the operands' type; in 16 bits the gradient behind the activation is rounded to it as well in front
    of the two products that x's and weight's gradients are."""
    act = _activation(activation)
    dtype = x.dtype
    if forward_ad._current_level >= 0:
        no_tangent("linear", x, weight, bias, residual)
    if not together(x, weight, bias, residual):
        check_tensors("linear", x.device, dtype, ("weight", weight), ("bias", bias), ("residual", residual))
    code = check_float("linear", "x", dtype)
    shape = _check_shapes("linear", x, weight, bias, residual)
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad or (bias is not None and bias.requires_grad)
                                    or (residual is not None and residual.requires_grad)):
        return _Linear.apply(x, weight, bias, residual, act, shape)
    n, k = weight.shape
    x2 = rows_of(x, k)
    return _forward("linear", _in_pieces(x2, rows_of(weight, k)), x2.shape[0], n, k, bias, residual, shape, code, dtype, x.device, act, False)[0]


def linear_8bit(x: torch.Tensor, x_scale: torch.Tensor, weight: torch.Tensor, weight_scale: torch.Tensor, bias: Optional[torch.Tensor] = None,
                *, activation: str = "none", residual: Optional[torch.Tensor] = None, out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """``linear`` on rows in 8 bits: x (..., k) and weight (n, k) float8_e4m3fn, x_scale (...) and weight_scale (n,) float32 as
    ``quantize_rows`` makes them; the sums of the 8-bit products are scaled by ``x_scale[row] * weight_scale[col]`` in front of the bias.
    bias, residual and the result are of ``out_dtype``.  Forward only.

    Sums are in 32 bits where ``out_dtype`` is float32 or float16 (products at half the 8-bit rate) and for up to 8 rows.  For more rows with
    a bfloat16 result the 8-bit matrix instructions add groups of 8 neighbouring products to 2^-13 of the group's largest: a sum may be off by 7 * 2^-13 of
    its terms' magnitudes, which shows where it cancels, and a row computed alone may differ by that much from the same row among others."""
    act = _activation(activation)
    dev = x.device
    if forward_ad._current_level >= 0:
        no_tangent("linear_8bit", x_scale, weight_scale, bias, residual)
    check_tensors("linear_8bit", dev, torch.float8_e4m3fn, ("x", x), ("weight", weight))
    check_float("linear_8bit", "out_dtype", out_dtype)
    check_tensors("linear_8bit", dev, torch.float32, ("x_scale", x_scale), ("weight_scale", weight_scale))
    check_tensors("linear_8bit", dev, out_dtype, ("bias", bias), ("residual", residual))
    shape = _check_shapes("linear_8bit", x, weight, bias, residual)
    if x_scale.shape != x.shape[:-1] or weight_scale.shape != (weight.shape[0],):
        raise ValueError("linear_8bit: x_scale must be %s and weight_scale (%d,) (got %s, %s)" % (
            tuple(x.shape[:-1]), weight.shape[0], tuple(x_scale.shape), tuple(weight_scale.shape)))
    no_gradient("linear_8bit", x_scale, weight_scale, bias, residual)
    n, k = weight.shape
    x2 = rows_of(x, k)
    return _forward("linear_8bit", _in_pieces(x2, rows_of(weight, k)), x2.shape[0], n, k, bias, residual, shape, _capi.T_E4M3, out_dtype, dev, act,
                    False, (vector_of(x_scale, x2.shape[0]), vector_of(weight_scale, n)))[0]


def quantize_rows(x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """Rows in 8 bits: x (..., width) float32 / bfloat16 / float16 -> (q (..., width) float8_e4m3fn, scale (...) float32) with
    scale = max(max|row| / 448, 2^-126) and q = x / scale rounded to nearest even: x is q * scale up to half a step of e4m3.  A row that
    holds a NaN or an infinity gets a scale that is not finite, and stands for no number."""
    if forward_ad._current_level >= 0:
        no_tangent("quantize_rows", x)
    check_tensors("quantize_rows", x.device, x.dtype)
    check_float("quantize_rows", "x", x.dtype)
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError("quantize_rows: x must have at least one column (got %s)" % (tuple(x.shape),))
    no_gradient("quantize_rows", x)
    return rows_forward("quantize_rows", x, None, None, 0.0, quantize=True)[:2]
