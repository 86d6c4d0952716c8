"""A ResnetFC with an RMS norm in front of every block (``ResnetFC(norm="rms")``), made of the row operators.

    zs = [lin_z.0; lin_z.1; ..] z                      one product: the latent rows are read once for all blocks
    h  = lin_in x
    per block b:  a, h = rms_norm(zs[b], residual=h);  h = h + fc_1(act(fc_0 a))      addition and norm in one pass, the second
                                                                                      addition in fc_1's epilogue
    out = lin_out rms_norm(h)

The blocks run in the model's precision; lin_in (whose inputs are coordinates in metres beside sines) and lin_out (whose outputs are
densities) always in fp32.  The reference's net has the same layers without the norms (scenerf/models/resnetfc.py:133-164).
"""
from __future__ import annotations

import ctypes as C
from typing import List, Optional

import torch

from . import _capi
from .linear import linear, linear_8bit, linear_step, linear_step_back, quantize_rows
from .norm import rms_norm, rms_norm_8bit, rms_step_back
from .rowops import rows_forward

NONE = _capi.ACTIVATIONS["none"]


class NetParams(list):
    """The parameters of such a net in ``ResnetFC.ordered_params`` order, and what else an evaluation needs to know."""

    def __init__(self, params, n_blocks: int, activation: str, eps: float, eight_bit: bool):
        super().__init__(params)
        self.n_blocks, self.activation, self.eps, self.eight_bit = n_blocks, activation, eps, eight_bit


class _Layers:
    """The parameters by their place in the net, the blocks' in ``dtype``."""

    def __init__(self, params, n_blocks: int, dtype: torch.dtype):
        cast = (lambda t: t) if dtype == torch.float32 else (lambda t: t.to(dtype))
        self.w_in, self.b_in, self.w_out, self.b_out = params[:4]
        per = [params[4 + 6 * b:10 + 6 * b] for b in range(n_blocks)]
        self.fc0 = [(cast(p[0]), cast(p[1])) for p in per]
        self.fc1 = [(cast(p[2]), cast(p[3])) for p in per]
        self.w_z, self.b_z = cast(torch.cat([p[4] for p in per], 0)), cast(torch.cat([p[5] for p in per], 0))
        self.norms = [cast(t) for t in params[4 + 6 * n_blocks:4 + 7 * n_blocks]]
        self.norm_out = cast(params[4 + 7 * n_blocks])


def evaluate(params: NetParams, z: torch.Tensor, x: torch.Tensor) -> torch.Tensor:
    """The net on rows z (..., d_latent) and x (..., d_in) of one type, through autograd."""
    nb, lead = params.n_blocks, z.shape[:-1]
    net = _Layers(params, nb, z.dtype)
    H = net.fc0[0][0].shape[0]
    zs = linear(z.reshape(-1, z.shape[-1]), net.w_z, net.b_z).view(-1, nb, H).unbind(1)
    h = linear(x.reshape(-1, x.shape[-1]).float(), net.w_in, net.b_in).to(z.dtype)
    for b in range(nb):
        a, h = rms_norm(zs[b], net.norms[b], residual=h, eps=params.eps)
        t = linear(a, *net.fc0[b], activation=params.activation)
        h = linear(t, *net.fc1[b], residual=h)
    a = rms_norm(h, net.norm_out, eps=params.eps)
    return linear(a.float(), net.w_out, net.b_out).view(*lead, net.w_out.shape[0]).to(z.dtype)


class PackedNormedMLP:
    """Such a net inside a render session: what ``PackedMLP`` is for the fused kernels' nets, where the chunk touches it.  Gradients leave
    their kernels in fp32 and are summed over the session's chunks in one flat buffer of it (one all-reduce per net), laid out like the parameters."""
    normed = True

    def __init__(self, params: List[torch.Tensor], spec: NetParams, d_out: int, cfg, trainable: bool):
        ps = [t.detach().float().contiguous() for t in params]
        nb, H = spec.n_blocks, ps[0].shape[0]
        for i, t in enumerate(ps):
            if not t.is_cuda:
                raise RuntimeError("ResnetFC parameter %d must be a CUDA tensor (the render pass has no CPU path)" % i)
        if len(ps) != 5 + 7 * nb or ps[0].shape[1] != 42 or tuple(ps[2].shape) != (d_out, H):
            raise RuntimeError("ResnetFC(norm='rms'): parameter shapes do not match d_in=42, d_hidden=%d, d_out=%d, %d blocks" % (H, d_out, nb))
        self.shapes = [t.shape for t in ps]
        self.spec, self.n_blocks, self.d_hidden, self.d_out, self.device, self.trainable = spec, nb, H, d_out, ps[0].device, trainable
        self.dtype = torch.bfloat16 if cfg.precision_code else torch.float32
        self.act = _capi.ACTIVATIONS[spec.activation]
        self.net = _Layers(ps, nb, self.dtype)
        self.w_in = torch.zeros((H, _capi.D_XENC), dtype=torch.float32, device=self.device)      # the encoding's rows end in zeros: 42 -> 48
        self.w_in[:, :42] = ps[0]
        self.eight = None
        if spec.eight_bit and not trainable:
            n = self.net
            self.eight = dict(w_z=quantize_rows(n.w_z), fc0=[quantize_rows(w) for w, _ in n.fc0], fc1=[quantize_rows(w) for w, _ in n.fc1])
        self.gflat: Optional[torch.Tensor] = None
        self.gc, self.gviews = None, {}
        self.w_z_t: List[torch.Tensor] = []
        if trainable:       # per pyramid level the columns of [Wz_0; Wz_1; ..] as rows: the feature maps' gradients are dzs Wz
            self.w_z_t = [w.t().contiguous() for w in self.net.w_z.split([c for c, _, _ in cfg.map_shapes()], 1)]

    def launch_pack(self, upto: int = 2) -> None:
        pass

    def wait_ready(self, backward: bool = False) -> None:
        if backward and not self.trainable:
            raise RuntimeError("this ResnetFC session was opened without gradients")

    # ---- forward on gathered rows
    def forward(self, xenc: torch.Tensor, Z: torch.Tensor, keep: bool):
        """(logits (M, d_out) fp32, what ``backward`` needs or None)."""
        if keep:
            return self._forward_kept(xenc, Z)
        n, nb, H, dt = self.net, self.n_blocks, self.d_hidden, self.dtype
        M = Z.shape[0]
        h = linear(xenc, self.w_in, n.b_in).to(dt)
        e, act, eps = self.eight, self.spec.activation, self.spec.eps
        if e is not None:
            zs = linear_8bit(*quantize_rows(Z), *e["w_z"], n.b_z, out_dtype=dt).view(M, nb, H)
            for b in range(nb):
                q, s, h = rms_norm_8bit(zs[:, b], n.norms[b], residual=h, eps=eps)
                t = linear_8bit(q, s, *e["fc0"][b], n.fc0[b][1], activation=act, out_dtype=dt)
                h = linear_8bit(*quantize_rows(t), *e["fc1"][b], n.fc1[b][1], residual=h, out_dtype=dt)
        else:
            zs = linear(Z, n.w_z, n.b_z).view(M, nb, H)
            for b in range(nb):
                a, h = rms_norm(zs[:, b], n.norms[b], residual=h, eps=eps)
                h = linear(linear(a, *n.fc0[b], activation=act), *n.fc1[b], residual=h)
        return linear(rms_norm(h, n.norm_out, eps=eps).float(), n.w_out, n.b_out), None

    def _norm(self, x, weight, residual):
        """y, h and what ``_norm_back`` needs: in 16 bits x and residual, whose sum h is rounded as it is stored."""
        y, _, h, rstd, x2 = rows_forward("rms_norm", x, weight, residual, self.spec.eps, keep_rstd=True)
        return y, h, (x2, weight, rstd, residual) if h is None or self.dtype != torch.float32 else (h, weight, rstd, None)

    def _norm_back(self, saved, dy, dh):
        return rms_step_back(*saved[:3], self.spec.eps, dy, dh, True, True, saved[3], sums=True)

    def _forward_kept(self, xenc, Z):
        n, nb, H, dt = self.net, self.n_blocks, self.d_hidden, self.dtype
        M = Z.shape[0]
        h, s_in = linear_step(xenc, self.w_in, n.b_in, None, NONE, (M, H), False)
        h = h.to(dt)
        zs, s_z = linear_step(Z, n.w_z, n.b_z, None, NONE, (M, nb * H), False)
        zs = zs.view(M, nb, H)
        blocks = []
        for b in range(nb):
            a, h, s_n = self._norm(zs[:, b], n.norms[b], h)
            t, s_0 = linear_step(a, *n.fc0[b], None, self.act, (M, H), True)
            h, s_1 = linear_step(t, *n.fc1[b], h, NONE, (M, H), False)
            blocks.append((s_n, s_0, s_1))
        a, _, s_norm = self._norm(h, n.norm_out, None)
        out, s_out = linear_step(a.float(), n.w_out, n.b_out, None, NONE, (M, self.d_out), False)
        return out, (s_in, s_z, blocks, s_norm, s_out)

    # ---- backward: parameter gradients into the sink; returns the gradient of zs (M, n_blocks * d_hidden)
    def backward(self, saved, d_logits: torch.Tensor) -> torch.Tensor:
        s_in, s_z, blocks, s_norm, s_out = saved
        nb, H, dt = self.n_blocks, self.d_hidden, self.dtype
        M = d_logits.shape[0]
        grads: List[Optional[torch.Tensor]] = [None] * len(self.shapes)
        dzs = torch.empty((M, nb, H), dtype=dt, device=d_logits.device)
        da, grads[2], grads[3] = linear_step_back(s_out, d_logits.contiguous(), (M, H), True, True, True, sums=True)
        dh, grads[4 + 7 * nb] = self._norm_back(s_norm, da.to(dt), None)
        for b in range(nb - 1, -1, -1):
            s_n, s_0, s_1 = blocks[b]
            at = 4 + 6 * b
            dt_, grads[at + 2], grads[at + 3] = linear_step_back(s_1, dh, (M, H), True, True, True, sums=True)
            da, grads[at], grads[at + 1] = linear_step_back(s_0, dt_, (M, H), True, True, True, sums=True)
            dh, grads[4 + 6 * nb + b] = self._norm_back(s_n, da, dh)
            dzs[:, b] = dh
        dzs = dzs.view(M, nb * H)
        _, dwz, dbz = linear_step_back(s_z, dzs, None, False, True, True, sums=True)
        for b in range(nb):
            grads[8 + 6 * b], grads[9 + 6 * b] = dwz[b * H:(b + 1) * H], dbz[b * H:(b + 1) * H]
        _, dwi, grads[1] = linear_step_back(s_in, dh.float(), None, False, True, True, sums=True)
        grads[0] = dwi[:, :42]
        self.grad_sink()
        torch._foreach_add_(self.gviews["all"], grads)
        return dzs

    def grad_sink(self):
        if self.gc is None:
            if self.gflat is None:
                self.gflat = torch.zeros(sum(s.numel() for s in self.shapes), dtype=torch.float32, device=self.device)
            self.gviews = {"all": [v.view(s) for v, s in zip(self.gflat.split([s.numel() for s in self.shapes]), self.shapes)]}
            self.gc = self.gviews
        return self.gc

    def unpack_grads(self) -> List[Optional[torch.Tensor]]:
        """Gradients in ``ResnetFC.ordered_params`` order (None if no chunk ran a backward)."""
        return list(self.gviews["all"]) if self.gviews else [None] * len(self.shapes)

    def feature_grads(self, ccfg, run, dzs: torch.Tensor, gmaps, stream) -> None:
        ptrs = (C.c_void_p * _capi.N_SCALES)(*[w.data_ptr() for w in self.w_z_t])
        _capi.check(_capi.load().scenerf_hip_resnetfc_feature_grads(C.byref(ccfg), C.byref(ptrs), self.n_blocks * self.d_hidden, run.tile_mask.data_ptr(),
                                                                    run.tap_texel.data_ptr(), run.tap_weight.data_ptr(), run.M, dzs.data_ptr(), gmaps,
                                                                    stream), "resnetfc_feature_grads")
