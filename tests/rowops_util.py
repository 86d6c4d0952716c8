"""Oracle of the row operators: their definitions in 64 bits on the CPU or the GPU, each with an elementwise bound of what a kernel with 32-bit
sums and one rounding to the output's type may be off by.

Half a step of a type is ``finfo(t).eps / 2`` relative, half its smallest subnormal absolute.  A sum of k products in 32 bits, in any
order, is off by at most about k 2^-24 times the sum of the products' magnitudes; (k + 8) 2^-23 leaves a factor of two for the matrix
instructions' own order and for bias and addition."""
import math

import torch


def half(t):
    return torch.finfo(t).eps / 2


def least(t):
    return torch.finfo(t).smallest_normal * torch.finfo(t).eps / 2


# largest |act'| and |act''|: gelu 1.129, 2 phi(0) = 0.798; silu 1.0998, 0.5
SLOPE = {"none": 1.0, "relu": 1.0, "gelu": 1.13, "silu": 1.1}
BEND = {"none": 0.0, "relu": 0.0, "gelu": 0.8, "silu": 0.5}


def act64(z, name):
    if name == "relu":
        return torch.where(z < 0, torch.zeros_like(z), z)
    if name == "gelu":
        return 0.5 * z * torch.special.erfc(-z / math.sqrt(2))
    if name == "silu":
        return z * torch.sigmoid(z)
    return z


def slope64(z, name):
    if name == "relu":
        return (z > 0).double()
    if name == "gelu":
        return 0.5 * torch.special.erfc(-z / math.sqrt(2)) + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    if name == "silu":
        p = torch.sigmoid(z)
        return p * (1 + z * (1 - p))
    return torch.ones_like(z)


def linear64(x, w, b=None, act="none", r=None, dy=None, scales=None, out_dtype=None, whole_dz=False):
    """{name: (value, bound)} of y and, with dy, of dx, dw, db, dr.  ``whole_dz``: dz with what its rounding leaves out as an operand of its own,
    so that the rest's rounding alone is left."""
    t = out_dtype or x.dtype
    u, tiny = half(t), least(t)
    X, W = x.double(), w.double()
    k, n = W.shape[1], W.shape[0]
    lead = X.shape[:-1]
    X = X.reshape(-1, k)
    if scales is not None:
        X, W = X * scales[0].double().reshape(-1, 1), W * scales[1].double().reshape(-1, 1)
    z, size = X @ W.t(), X.abs() @ W.abs().t()
    if b is not None:
        z, size = z + b.double(), size + b.double().abs()
    ez = (k + 8) * 2.0 ** -23 * size
    if scales is not None and t != torch.float32:
        # the 8-bit matrix instructions add groups of 8 neighbouring products with their bits below 2^-13 of the largest one's exponent cut
        # off (measured with single powers of two): at most 7 of a group lose less than 2^-13 of it each, and a group's largest is no
        # more than the sum of its magnitudes.  Results in 32 bits do not go through them.
        ez = ez + 7 * 2.0 ** -13 * size
    y = act64(z, act)
    arith = 2.0 ** -21 * z.abs() if act in ("gelu", "silu") else 0.0      # expf / erff / the division, a few ulp each
    if r is not None:
        y = y + r.double().reshape(-1, n)
    ey = SLOPE[act] * ez + arith + (u + 2.0 ** -23) * y.abs() + tiny
    out = {"y": (y.reshape(*lead, n), ey.reshape(*lead, n))}
    if dy is None:
        return out
    g = dy.double().reshape(-1, n)
    dz = g * slope64(z, act)
    # the slope at the kept z (rounded to t); dz itself is rounded to t where it is an operand
    esum = g.abs() * (BEND[act] * (ez + u * z.abs() + tiny) + (2.0 ** -20 if act in ("gelu", "silu") else 0.0))
    edz = esum if act == "none" else esum + (u * u * dz.abs() if whole_dz else u * dz.abs()) + tiny
    m = X.shape[0]
    dx = dz @ W
    out["dx"] = (dx.reshape(*lead, k), (edz @ W.abs() + (n + 8) * 2.0 ** -23 * (dz.abs() @ W.abs()) + u * dx.abs() + tiny).reshape(*lead, k))
    dw = dz.t() @ X
    out["dw"] = (dw, edz.t() @ X.abs() + (m + 8) * 2.0 ** -23 * (dz.abs().t() @ X.abs()) + u * dw.abs() + tiny)
    if b is not None:
        db = dz.sum(0)
        out["db"] = (db, esum.sum(0) + (m + 8) * 2.0 ** -23 * dz.abs().sum(0) + u * db.abs() + tiny)
    if r is not None:
        out["dr"] = (dy.double(), torch.zeros_like(dy, dtype=torch.float64))
    return out


def rms64(x, w, eps, r=None, dy=None, dh=None):
    """{name: (value, bound)} of h, y, rstd and, with dy, of dx, dw.  mean(h^2) of d squares is off by (d + 8) 2^-23 relative, rstd by half of
    that; the gradients are made from h as it is stored."""
    t, d = x.dtype, x.shape[-1]
    u, tiny = half(t), least(t)
    h = x.double().reshape(-1, d)
    if r is not None:
        h = h + r.double().reshape(-1, d)
    rstd = 1 / torch.sqrt((h * h).mean(1, keepdim=True) + eps)
    e = (d + 16) * 2.0 ** -23
    xhat = h * rstd
    W = w.double()
    y = xhat * W
    out = {"y": (y, (u + e) * y.abs() + 2.0 ** -23 * (rstd * W).abs() * h.abs() + tiny), "h": (h, (u + 2.0 ** -23) * h.abs() + tiny)}
    if dy is not None:
        g = dy.double().reshape(-1, d)
        a = g * W
        stored = u if r is not None else 0.0
        dot = (a * xhat).mean(1, keepdim=True)
        mag = (a * xhat).abs().mean(1, keepdim=True)
        dx = rstd * (a - xhat * dot)
        ex = rstd * (e * a.abs() + xhat.abs() * mag * (3 * e + 2 * stored))
        if dh is not None:
            dx = dx + dh.double().reshape(-1, d)
        out["dx"] = (dx, ex + (u + 2.0 ** -22) * dx.abs() + tiny + (2.0 ** -23 * dh.double().reshape(-1, d).abs() if dh is not None else 0.0))
        dw = (g * xhat).sum(0)
        out["dw"] = (dw, (g * xhat).abs().sum(0) * ((h.shape[0] + 8) * 2.0 ** -23 + e + stored) + u * dw.abs() + tiny)
    return {k: (v.reshape(x.shape) if v.shape != (d,) else v, b.reshape(x.shape) if b.shape != (d,) else b) for k, (v, b) in out.items()}


def hold(got, want, name=""):
    """``got`` within the bound, element by element; NaN and infinities where the oracle has them."""
    value, bound = want
    value, bound = value.to(got.device), bound.to(got.device)
    assert got.shape == value.shape, "%s: shape %s, expected %s" % (name, tuple(got.shape), tuple(value.shape))
    g = got.double()
    fine = torch.isfinite(value)
    assert torch.equal(torch.isnan(g), torch.isnan(value)), "%s: NaN elsewhere" % name
    top = torch.finfo(got.dtype).max
    far = ((g - value).abs() > bound) & fine & (value.abs() <= top)
    if bool(far.any()):
        i = int(((g - value).abs() / bound).nan_to_num(0).masked_fill(~far, 0).argmax())
        raise AssertionError("%s: %d of %d elements are off; worst: got %r, expected %r, bound %r" % (
            name, int(far.sum()), g.numel(), float(g.reshape(-1)[i]), float(value.reshape(-1)[i]), float(bound.reshape(-1)[i])))
