"""What the row operators (``linear``, ``norm``) share: checks, layouts, workspaces and the call itself."""
from __future__ import annotations

import ctypes as C
from typing import Optional

import torch

from . import _capi

TYPE_CODES = {torch.float32: _capi.T_F32, torch.bfloat16: _capi.T_BF16, torch.float16: _capi.T_F16}
MAX_ROWS = 2 ** 31 - 1025


def rows_of(t: torch.Tensor, width: int) -> torch.Tensor:
    """``t`` as (rows, width) with neighbouring elements inside a row: a view where the layout allows it."""
    if t.dim() != 2:
        t = t.reshape(-1, width)
    return t if width == 1 or t.stride(1) == 1 else t.contiguous()


def check_tensors(what: str, dev: torch.device, dtype: torch.dtype, *named) -> None:
    """``named``: (name, tensor or None) pairs that have to be on ``dev`` and of ``dtype``."""
    if dev.type != "cuda":
        raise RuntimeError("%s runs on the GPU only (no CPU fallback): got a tensor on %s" % (what, dev))
    for name, t in named:
        if t is not None:
            if t.device != dev:
                raise RuntimeError("%s: %s is on %s, the first argument on %s" % (what, name, t.device, dev))
            if t.dtype != dtype:
                raise RuntimeError("%s: %s is %s, expected %s" % (what, name, t.dtype, dtype))


def check_float(what: str, name: str, dtype: torch.dtype) -> int:
    code = TYPE_CODES.get(dtype)
    if code is None:
        raise RuntimeError("%s: %s must be float32, bfloat16 or float16 (got %s)" % (what, name, dtype))
    return code


def run_on(dev: torch.device, fn, args: tuple, what: str) -> None:
    """``fn(*args, stream)`` on ``dev``'s current stream, with ``dev`` current."""
    index = dev.index
    if index == torch.cuda.current_device():
        # (torch.cuda.current_stream(dev).cuda_stream without the Stream object: a fifth of a small call's host time)
        rc = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    else:
        with torch.cuda.device(dev):
            rc = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    if rc:
        _capi.check(rc, what)


def give_workspace(fn, args, backward: int, dev: torch.device, what: str) -> Optional[torch.Tensor]:
    """A workspace of the calling stream's own, for one call: two captured graphs, or two streams, never share one."""
    need = fn(C.byref(args), backward)
    if need == 0:
        return None
    if need < 0:
        _capi.check(1, what)
    ws = torch.empty(need, dtype=torch.uint8, device=dev)
    args.workspace, args.workspace_bytes = ws.data_ptr(), need
    return ws


def no_gradient(what: str, *tensors) -> None:
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                raise RuntimeError("%s has no gradient: call it under torch.no_grad() or on detached tensors" % what)


def rows_forward(what, x, weight, residual, eps, *, quantize=False, keep_rstd=False):
    """(q or y, scale or None, h or None, rstd or None, x as rows) of scenerf_hip_rms_forward."""
    shape, dtype, dev = x.shape, x.dtype, x.device
    width = shape[-1]
    x2 = rows_of(x, width)
    rows = x2.shape[0]
    if weight is not None and not weight.is_contiguous():
        weight = weight.contiguous()
    r2 = rows_of(residual, width) if residual is not None else None
    h = torch.empty(shape, dtype=dtype, device=dev) if residual is not None else None
    out = torch.empty(shape, dtype=torch.float8_e4m3fn if quantize else dtype, device=dev)
    scale = torch.empty(shape[:-1], dtype=torch.float32, device=dev) if quantize else None
    rstd = torch.empty((rows,), dtype=torch.float32, device=dev) if keep_rstd else None
    p = _capi.Rms(TYPE_CODES[dtype], width, rows, eps, x2.data_ptr(), x2.stride(0), None if r2 is None else r2.data_ptr(),
                  0 if r2 is None else r2.stride(0), None if weight is None else weight.data_ptr(), None if h is None else h.data_ptr(),
                  None if quantize else out.data_ptr(), out.data_ptr() if quantize else None, None if scale is None else scale.data_ptr(),
                  None if rstd is None else rstd.data_ptr())
    run_on(dev, _capi.load().scenerf_hip_rms_forward, (C.byref(p),), what)
    return out, scale, h, rstd, x2
