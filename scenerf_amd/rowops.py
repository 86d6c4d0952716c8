"""What the row operators (``linear``, ``norm``) share: checks, layouts, workspaces and the call itself."""
from __future__ import annotations

import ctypes as C
import struct
from typing import Any, Dict

import torch
import torch.autograd.forward_ad as forward_ad

from . import _capi

TYPE_CODES = {torch.float32: _capi.T_F32, torch.bfloat16: _capi.T_BF16, torch.float16: _capi.T_F16}
MAX_ROWS = 2 ** 31 - 1025


def rows_of(t: torch.Tensor, width: int) -> torch.Tensor:
    """``t`` as (rows, width) with neighbouring elements inside a row: a view where the layout allows it."""
    if t.dim() != 2:
        t = t.reshape(-1, width)
    if width == 1:          # (the imaginary part of a conjugate holds the other sign in its memory: every second element, so wider rows are copied)
        return t.resolve_neg()
    return t if t.stride(1) == 1 else t.contiguous()


def vector_of(t: torch.Tensor, n: int = 1) -> torch.Tensor:
    """``t`` of ``n`` elements as neighbours, as it is where the layout allows it (``rows_of`` says why one alone is looked at)."""
    return (t.resolve_neg() if n == 1 else t).contiguous()


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


def together(x: torch.Tensor, *others) -> bool:
    """All on x's GPU and of x's type: the usual call, without what ``check_tensors`` needs to say otherwise."""
    dtype, dev = x.dtype, x.device
    for t in others:
        if t is not None and (t.dtype is not dtype or t.device != dev):
            return False
    return x.is_cuda


# The arguments of one call, laid out as scenerf_linear / scenerf_rms: packed bytes cost a small call half of what the structures do
# (tests/test_rowops_refusals.py holds them to the structures' offsets).  The last two fields are the workspace and its bytes.
LINEAR = struct.Struct("@6i19q")
RMS = struct.Struct("@2iqfi18q")
_WORKSPACE = struct.Struct("@2q")
_entries: Dict[str, Any] = {}


def _entry(name: str, backward: bool):
    """(the call, its workspace query) of ``scenerf_hip_<name>_*`` on packed bytes."""
    key = name + ("_backward" if backward else "_forward")
    got = _entries.get(key)
    if got is None:
        lib = _capi.load()
        run, query = lib["scenerf_hip_" + key], lib["scenerf_hip_%s_workspace" % name]
        run.argtypes, run.restype = [C.c_char_p, C.c_void_p], C.c_int
        query.argtypes, query.restype = [C.c_char_p, C.c_int], C.c_int64
        got = _entries[key] = (run, query)
    return got


def run_on(dev: torch.device, fn, args: tuple, what: str) -> None:
    """``fn(*args, stream)`` on ``dev``'s current stream, with ``dev`` current."""
    if dev.index != torch._C._cuda_getDevice():
        with torch.cuda.device(dev):
            return run_on(dev, fn, args, what)
    _capi.check(fn(*args, torch._C._cuda_getCurrentRawStream(dev.index)), what)


def run_rows(name: str, backward: bool, args: bytes, dev: torch.device, what: str) -> None:
    """One call on ``dev``'s current stream, with ``dev`` current and a workspace of the calling stream's own where the call needs one: two
    captured graphs, or two streams, never share it."""
    index = dev.index
    if index != torch._C._cuda_getDevice():
        with torch.cuda.device(dev):
            return run_rows(name, backward, args, dev, what)
    run, query = _entry(name, backward)
    # (torch.cuda.current_stream(dev).cuda_stream without the Stream object)
    stream = torch._C._cuda_getCurrentRawStream(index)
    rc = _capi.NEEDS_WORKSPACE if backward else run(args, stream)     # (few forward calls need one, nearly all backward calls do)
    if rc == _capi.NEEDS_WORKSPACE:
        need = query(args, 1 if backward else 0)
        if need < 0:
            _capi.check(1, what)
        if need:
            ws = torch.empty(need, dtype=torch.uint8, device=dev)
            args = args[:-_WORKSPACE.size] + _WORKSPACE.pack(ws.data_ptr(), need)
        rc = run(args, stream)
    if rc:
        _capi.check(rc, what)


def no_tangent(what: str, *tensors) -> None:
    """Refuses dual tensors: nothing else about them says that a derivative is asked for, and grad mode does not concern them.  Called where
    ``forward_ad._current_level`` is not negative: there are none outside a level, and a small call feels the function."""
    for t in tensors:
        if t is not None and forward_ad.unpack_dual(t).tangent is not None:
            raise RuntimeError("%s has no forward-mode derivative (got a dual tensor)" % what)


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
    if weight is not None:
        weight = vector_of(weight, width)
    r2 = rows_of(residual, width) if residual is not None else None
    h = x.new_empty(shape) if residual is not None else None
    out = torch.empty(shape, dtype=torch.float8_e4m3fn, device=dev) if quantize else x.new_empty(shape)
    scale = torch.empty(shape[:-1], dtype=torch.float32, device=dev) if quantize else None
    rstd = torch.empty((rows,), dtype=torch.float32, device=dev) if keep_rstd else None
    run_rows("rms", False, RMS.pack(
        TYPE_CODES[dtype], width, rows, eps, 0, x2.data_ptr(), x2.stride(0), 0 if r2 is None else r2.data_ptr(), 0 if r2 is None else r2.stride(0),
        0 if weight is None else weight.data_ptr(), 0 if h is None else h.data_ptr(), 0 if quantize else out.data_ptr(),
        out.data_ptr() if quantize else 0, 0 if scale is None else scale.data_ptr(), 0 if rstd is None else rstd.data_ptr(),
        0, 0, 0, 0, 0, 0, 0, 0), dev, what)
    return out, scale, h, rstd, x2
