"""A linear layer with its epilogue in one launch, forward and backward, and its 8-bit form (``scenerf_hip_linear_*``, csrc/linear.hip).

The reference's ResnetFC is ``nn.Linear`` + activation + addition, each a pass over the rows (scenerf/models/resnetfc.py:49-64, 146-163).
Here one call is one product with all of that behind its sums::

    y = linear(x, weight, bias, activation="gelu", residual=h)        # act(x @ weight.T + bias) + h, differentiable in every input
    q, s = quantize_rows(x)                                           # rows in e4m3 with one fp32 scale each
    y = linear_8bit(q, s, wq, ws, bias, activation="gelu", residual=h)

float32 (fp32 matrix instructions), bfloat16 and float16 operands, 32-bit sums, every output rounded once.  Rows are whatever precedes
the last dimension, zero rows included; a row's elements must be neighbours in memory (other layouts are copied first), its pitch is
free.  CUDA tensors only: anything else raises, there is no fallback.
"""
from __future__ import annotations

import ctypes as C
from typing import Optional, Tuple

import torch
from torch.autograd.function import once_differentiable

from . import _capi

TYPE_CODES = {torch.float32: _capi.T_F32, torch.bfloat16: _capi.T_BF16, torch.float16: _capi.T_F16}
MAX_ROWS = 2 ** 31 - 1025


def rows_of(t: torch.Tensor, width: int) -> torch.Tensor:
    """``t`` as (rows, width) with neighbouring elements inside a row: a view where the layout allows it."""
    if t.dim() != 2:
        t = t.reshape(-1, width)
    return t if width == 1 or t.stride(1) == 1 else t.contiguous()


def require_cuda(what: str, dev: torch.device, **tensors) -> None:
    if dev.type != "cuda":
        raise RuntimeError("%s runs on the GPU only (no CPU fallback): got a tensor on %s" % (what, dev))
    for name, t in tensors.items():
        if t is not None and t.device != dev:
            raise RuntimeError("%s: %s is on %s, the first argument on %s" % (what, name, t.device, dev))


def require_type(what: str, dtype: torch.dtype, **tensors) -> None:
    for name, t in tensors.items():
        if t is not None and t.dtype != dtype:
            raise RuntimeError("%s: %s is %s, expected %s" % (what, name, t.dtype, dtype))


def run_on(dev: torch.device, fn, args, what: str) -> None:
    """``fn(args, stream)`` on ``dev``'s current stream, with ``dev`` current."""
    if dev.index == torch.cuda.current_device():
        _capi.check(fn(C.byref(args), torch.cuda.current_stream(dev).cuda_stream), what)
    else:
        with torch.cuda.device(dev):
            _capi.check(fn(C.byref(args), torch.cuda.current_stream(dev).cuda_stream), what)


def give_workspace(fn, args, backward: bool, dev: torch.device, what: str) -> Optional[torch.Tensor]:
    """A workspace of the calling stream's own, for one call: two captured graphs, or two streams, never share one."""
    need = fn(C.byref(args), int(backward))
    if need < 0:
        _capi.check(1, what)
    if need == 0:
        return None
    ws = torch.empty(need, dtype=torch.uint8, device=dev)
    args.workspace, args.workspace_bytes = ws.data_ptr(), need
    return ws


def no_gradient(what: str, *tensors) -> None:
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise RuntimeError("%s has no gradient: call it under torch.no_grad() or on detached tensors" % what)


def _activation(name: str) -> int:
    code = _capi.ACTIVATIONS.get(name)
    if code is None:
        raise ValueError("activation must be one of %s (got %r)" % (", ".join(sorted(_capi.ACTIVATIONS)), name))
    return code


def _check_shapes(what, x, weight, bias, residual):
    if weight.dim() != 2 or weight.shape[0] < 1 or weight.shape[1] < 1:
        raise ValueError("%s: weight must be (n, k) with n, k >= 1 (got %s)" % (what, tuple(weight.shape)))
    n, k = weight.shape
    if x.dim() < 1 or x.shape[-1] != k:
        raise ValueError("%s: x must end in %d features (got %s)" % (what, k, tuple(x.shape)))
    shape = x.shape[:-1] + (n,)
    if bias is not None and tuple(bias.shape) != (n,):
        raise ValueError("%s: bias must be (%d,) (got %s)" % (what, n, tuple(bias.shape)))
    if residual is not None and residual.shape != shape:
        raise ValueError("%s: residual must be %s (got %s); expand it first if it is to be broadcast" % (what, tuple(shape), tuple(residual.shape)))
    if x.numel() // k > MAX_ROWS:
        raise ValueError("%s: more than 2^31 - 1025 rows" % what)
    return shape


def _args(x2, w2, in_type, out_type, activation) -> "_capi.Linear":
    p = _capi.Linear(in_type, out_type, activation, w2.shape[0], w2.shape[1], x2.shape[0])
    p.x, p.ldx, p.w, p.ldw = x2.data_ptr(), x2.stride(0), w2.data_ptr(), w2.stride(0)
    return p


def _forward(what, x2, w2, bias, residual, shape, in_type, out_dtype, act, keep_z, scales=None):
    n, dev = w2.shape[0], x2.device
    y = torch.empty(shape, dtype=out_dtype, device=dev)
    z = torch.empty((x2.shape[0], n), dtype=out_dtype, device=dev) if keep_z else None
    p = _args(x2, w2, in_type, TYPE_CODES[out_dtype], act)
    hold = []
    if scales is not None:
        p.x_scale, p.w_scale = scales[0].data_ptr(), scales[1].data_ptr()
    if bias is not None:
        bias = bias.contiguous()
        p.bias = bias.data_ptr()
    if residual is not None:
        r = rows_of(residual, n)
        hold.append(r)
        p.residual, p.ld_residual = r.data_ptr(), r.stride(0)
    p.y = y.data_ptr()
    if z is not None:
        p.z = z.data_ptr()
    lib = _capi.load()
    hold.append(give_workspace(lib.scenerf_hip_linear_workspace, p, False, dev, what))
    run_on(dev, lib.scenerf_hip_linear_forward, p, what)
    return y, z


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, act, shape):
        x2, w2 = rows_of(x, weight.shape[1]), rows_of(weight, weight.shape[1])
        keep_z = act != _capi.ACTIVATIONS["none"] and any(ctx.needs_input_grad[:3])
        y, z = _forward("linear", x2, w2, bias, residual, shape, TYPE_CODES[x.dtype], x.dtype, act, keep_z)
        ctx.save_for_backward(x2, w2, z)
        ctx.act, ctx.x_shape = act, x.shape
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x2, w2, z = ctx.saved_tensors
        need_x, need_w, need_b, need_r = ctx.needs_input_grad[:4]
        dev, (n, k) = dy.device, w2.shape
        dx = torch.empty(ctx.x_shape, dtype=x2.dtype, device=dev) if need_x else None
        dw = torch.empty((n, k), dtype=x2.dtype, device=dev) if need_w else None
        db = torch.empty((n,), dtype=x2.dtype, device=dev) if need_b else None
        if need_x or need_w or need_b:
            dy2 = rows_of(dy, n)
            p = _args(x2, w2, TYPE_CODES[x2.dtype], TYPE_CODES[x2.dtype], ctx.act)
            p.dy, p.ld_dy = dy2.data_ptr(), dy2.stride(0)
            p.z, p.dx, p.dw, p.db = _capi.ptr(z), _capi.ptr(dx), _capi.ptr(dw), _capi.ptr(db)
            lib = _capi.load()
            ws = give_workspace(lib.scenerf_hip_linear_workspace, p, True, dev, "linear backward")
            run_on(dev, lib.scenerf_hip_linear_backward, p, "linear backward")
            del ws
        return dx, dw, db, (dy if need_r else None), None, None


def linear(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None, *, activation: str = "none",
           residual: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``act(x @ weight.T + bias) + residual``: x (..., k), weight (n, k), bias (n,), residual (..., n), all of one type -> (..., n).

    ``activation``: "none", "relu", "gelu" (the exact one, by erf) or "silu".  Sums, bias, activation and addition are in 32 bits; the
    result is rounded once.  Differentiable once in x, weight, bias and residual; where an activation is asked for and a gradient will
    be, the sums in front of it are kept in the operands' type."""
    act = _activation(activation)
    require_cuda("linear", x.device, weight=weight, bias=bias, residual=residual)
    if x.dtype not in TYPE_CODES:
        raise RuntimeError("linear: x must be float32, bfloat16 or float16 (got %s)" % x.dtype)
    require_type("linear", x.dtype, weight=weight, bias=bias, residual=residual)
    shape = _check_shapes("linear", x, weight, bias, residual)
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad or (bias is not None and bias.requires_grad)
                                    or (residual is not None and residual.requires_grad)):
        return _Linear.apply(x, weight, bias, residual, act, shape)
    k = weight.shape[1]
    return _forward("linear", rows_of(x, k), rows_of(weight, k), bias, residual, shape, TYPE_CODES[x.dtype], x.dtype, act, False)[0]


def linear_8bit(x: torch.Tensor, x_scale: torch.Tensor, weight: torch.Tensor, weight_scale: torch.Tensor, bias: Optional[torch.Tensor] = None,
                *, activation: str = "none", residual: Optional[torch.Tensor] = None, out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """``linear`` on rows in 8 bits: x (..., k) and weight (n, k) float8_e4m3fn, x_scale (...) and weight_scale (n,) float32 as
    ``quantize_rows`` makes them; the sums of the 8-bit products are scaled by ``x_scale[row] * weight_scale[col]`` in front of the bias.
    bias, residual and the result are of ``out_dtype``.  Forward only."""
    act = _activation(activation)
    require_cuda("linear_8bit", x.device, x_scale=x_scale, weight=weight, weight_scale=weight_scale, bias=bias, residual=residual)
    if out_dtype not in TYPE_CODES:
        raise RuntimeError("linear_8bit: out_dtype must be float32, bfloat16 or float16 (got %s)" % out_dtype)
    require_type("linear_8bit", torch.float8_e4m3fn, x=x, weight=weight)
    require_type("linear_8bit", torch.float32, x_scale=x_scale, weight_scale=weight_scale)
    require_type("linear_8bit", out_dtype, bias=bias, residual=residual)
    shape = _check_shapes("linear_8bit", x, weight, bias, residual)
    if x_scale.shape != x.shape[:-1] or tuple(weight_scale.shape) != (weight.shape[0],):
        raise ValueError("linear_8bit: x_scale must be %s and weight_scale (%d,) (got %s, %s)" % (
            tuple(x.shape[:-1]), weight.shape[0], tuple(x_scale.shape), tuple(weight_scale.shape)))
    no_gradient("linear_8bit", x_scale, weight_scale, bias, residual)
    k = weight.shape[1]
    return _forward("linear_8bit", rows_of(x, k), rows_of(weight, k), bias, residual, shape, _capi.T_E4M3, out_dtype, act, False,
                    (x_scale.contiguous(), weight_scale.contiguous()))[0]


def quantize_rows(x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """Rows in 8 bits: x (..., width) float32 / bfloat16 / float16 -> (q (..., width) float8_e4m3fn, scale (...) float32) with
    scale = max(max|row| / 448, 2^-126) and q = x / scale rounded to nearest even: x is q * scale up to half a step of e4m3.  A row that
    holds a NaN or an infinity gets a scale that is not finite, and stands for no number."""
    from .norm import rows_forward
    require_cuda("quantize_rows", x.device)
    if x.dtype not in TYPE_CODES:
        raise RuntimeError("quantize_rows: x must be float32, bfloat16 or float16 (got %s)" % x.dtype)
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError("quantize_rows: x must have at least one column (got %s)" % (tuple(x.shape),))
    no_gradient("quantize_rows", x)
    got = rows_forward("quantize_rows", x, None, None, 0.0, quantize=True)
    return got["q"], got["scale"]
