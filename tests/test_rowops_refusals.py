"""What the row operators refuse, without a GPU: the C entries' own checks and the Python entries' (no kernel runs)."""
import ctypes as C

import pytest
import torch

from scenerf_amd import _capi
from scenerf_amd.linear import linear, linear_8bit, quantize_rows
from scenerf_amd.norm import rms_norm, rms_norm_8bit


def test_there_is_no_cpu_path():
    x, w = torch.ones(3, 4), torch.ones(5, 4)
    q, s = x.to(torch.float8_e4m3fn), torch.ones(3)
    for call in (lambda: linear(x, w), lambda: linear_8bit(q, s, w.to(torch.float8_e4m3fn), torch.ones(5)), lambda: quantize_rows(x),
                 lambda: rms_norm(x, torch.ones(4)), lambda: rms_norm_8bit(x, torch.ones(4))):
        with pytest.raises(RuntimeError, match="GPU only"):
            call()
    with pytest.raises(ValueError, match="activation"):
        linear(x, w, activation="tanh")


def _linear(**kw):
    p = _capi.Linear(in_type=0, out_type=0, activation=0, n=4, k=8, rows=3)
    p.x = p.w = p.y = 4096
    p.ldx = p.ldw = 8
    for k, v in kw.items():
        setattr(p, k, v)
    return p


def _said(rc):
    assert rc != 0
    return _capi.load().scenerf_hip_last_error().decode()


def test_linear_entry_refuses():
    lib = _capi.load()
    assert "NULL argument" in _said(lib.scenerf_hip_linear_forward(None, None))
    assert "types must be" in _said(lib.scenerf_hip_linear_forward(C.byref(_linear(in_type=7)), None))
    assert "types must be" in _said(lib.scenerf_hip_linear_forward(C.byref(_linear(out_type=3)), None))
    assert "differ" in _said(lib.scenerf_hip_linear_forward(C.byref(_linear(in_type=1)), None))
    assert "activation" in _said(lib.scenerf_hip_linear_forward(C.byref(_linear(activation=4)), None))
    for bad in (dict(n=0), dict(k=0), dict(n=-1), dict(rows=-1), dict(rows=2 ** 31), dict(ldx=-8)):
        assert lib.scenerf_hip_linear_forward(C.byref(_linear(**bad)), None) != 0
        assert lib.scenerf_hip_linear_workspace(C.byref(_linear(**bad)), 0) == -1
    assert "NULL x" in _said(lib.scenerf_hip_linear_forward(C.byref(_linear(x=None)), None))
    assert "x_scale" in _said(lib.scenerf_hip_linear_forward(C.byref(_linear(in_type=3)), None))
    assert "nothing to compute" in _said(lib.scenerf_hip_linear_backward(C.byref(_linear(dy=4096)), None))
    assert "NULL dy" in _said(lib.scenerf_hip_linear_backward(C.byref(_linear(dx=4096)), None))
    assert "z is NULL" in _said(lib.scenerf_hip_linear_backward(C.byref(_linear(dx=4096, dy=4096, activation=2)), None))
    assert "no gradients" in _said(lib.scenerf_hip_linear_backward(C.byref(_linear(in_type=3, dx=4096, dy=4096)), None))
    p = _linear(dx=4096, db=4096, dy=4096, z=4096, activation=2, ld_dy=4)
    need = lib.scenerf_hip_linear_workspace(C.byref(p), 1)
    assert need > 0
    assert "workspace" in _said(lib.scenerf_hip_linear_backward(C.byref(p), None))
    p.workspace, p.workspace_bytes = 4096, need - 1
    assert "workspace" in _said(lib.scenerf_hip_linear_backward(C.byref(p), None))
    p.workspace, p.workspace_bytes = 4096 + 8, need
    assert "workspace" in _said(lib.scenerf_hip_linear_backward(C.byref(p), None))


def test_linear_entry_with_no_rows_does_nothing():
    lib = _capi.load()
    assert lib.scenerf_hip_linear_forward(C.byref(_linear(rows=0, x=None, y=None)), None) == 0
    assert lib.scenerf_hip_linear_workspace(C.byref(_linear(rows=0)), 0) == 0
    assert lib.scenerf_hip_linear_workspace(C.byref(_linear(rows=0, dx=4096, dw=4096, db=4096)), 1) >= 0


def _rms(**kw):
    p = _capi.Rms(type=0, width=8, rows=3, eps=1e-6)
    p.x = p.weight = p.y = 4096
    p.ldx = 8
    for k, v in kw.items():
        setattr(p, k, v)
    return p


def test_rms_entry_refuses():
    lib = _capi.load()
    assert "NULL argument" in _said(lib.scenerf_hip_rms_forward(None, None))
    for bad in (dict(type=3), dict(width=0), dict(rows=-1), dict(rows=2 ** 31), dict(eps=-1.0), dict(eps=float("nan")), dict(ldx=-1), dict(x=None), dict(y=None),
                dict(h=4096), dict(q=4096), dict(scale=4096), dict(weight=None, rstd=4096)):
        assert lib.scenerf_hip_rms_forward(C.byref(_rms(**bad)), None) != 0, bad
    assert "nothing to compute" in _said(lib.scenerf_hip_rms_backward(C.byref(_rms(dy=4096, rstd=4096)), None))
    assert "NULL" in _said(lib.scenerf_hip_rms_backward(C.byref(_rms(dx=4096, rstd=4096)), None))
    p = _rms(dx=4096, dweight=4096, dy=4096, rstd=4096)
    need = lib.scenerf_hip_rms_workspace(C.byref(p), 1)
    assert need >= 32 and "workspace" in _said(lib.scenerf_hip_rms_backward(C.byref(p), None))
    assert lib.scenerf_hip_rms_forward(C.byref(_rms(rows=0, x=None, y=None)), None) == 0


def test_the_net_with_norms():
    from scenerf_amd.model import ResnetFC, SceneRF
    m = ResnetFC(n_blocks=2, d_hidden=32, norm="rms")
    assert not m.is_standard and m.activation == "gelu" and not ResnetFC(norm="rms").is_standard and ResnetFC().activation == "relu"
    p = m.ordered_params()
    assert len(p) == 4 + 6 * 2 + 3 and {id(t) for t in p} == {id(t) for t in m.parameters()} and tuple(p[-1].shape) == (32,)
    for bad in (dict(norm="layer"), dict(norm="rms", activation="tanh"), dict(activation="gelu"), dict(norm="rms", norm_eps=0.0)):
        with pytest.raises(ValueError):
            ResnetFC(**bad)
    with pytest.raises(RuntimeError, match="render_rays_batch"):
        ResnetFC()(torch.zeros(1, 2522))
    with pytest.raises((RuntimeError, ValueError)):        # no CPU path
        m(torch.zeros(1, 2522))
    r = SceneRF(som_sigma=2.0, std=2.0, add_fov_hor=20, add_fov_ver=8, precision="bf16")
    r.mlp = m
    with pytest.raises(NotImplementedError):
        r.render_image(None, None, {})


def test_packed_arguments_are_the_structures():
    from scenerf_amd.rowops import LINEAR, RMS
    for packer, kind in ((LINEAR, _capi.Linear), (RMS, _capi.Rms)):
        assert packer.size == C.sizeof(kind)
        values = [2.5 if t is C.c_float else i + 1 for i, (_, t) in enumerate(kind._fields_)]
        got = kind.from_buffer_copy(packer.pack(*values))
        assert [getattr(got, name) for name, _ in kind._fields_] == values


def test_a_call_without_its_workspace_says_so():
    lib = _capi.load()
    p = _capi.Linear(in_type=0, out_type=0, activation=0, n=4, k=8, rows=3)
    p.dy, p.x, p.w, p.db, p.ld_dy, p.ldx, p.ldw = 16, 16, 16, 16, 4, 8, 8
    assert lib.scenerf_hip_linear_workspace(C.byref(p), 1) > 0
    assert lib.scenerf_hip_linear_backward(C.byref(p), None) == _capi.NEEDS_WORKSPACE
    p.workspace, p.workspace_bytes = 16, 1
    assert lib.scenerf_hip_linear_backward(C.byref(p), None) == _capi.NEEDS_WORKSPACE
    r = _capi.Rms(type=0, width=8, rows=3, eps=1e-6)
    r.x, r.weight, r.rstd, r.dy, r.dweight = 16, 16, 16, 16, 16
    assert lib.scenerf_hip_rms_backward(C.byref(r), None) == _capi.NEEDS_WORKSPACE


@pytest.mark.parametrize("kind", [0, 1, 2])
def test_a_step_back_of_no_rows_has_nothing_to_write(kind):
    """Frozen parameters and no rows: the one gradient asked for, x's, is empty and its pointer NULL."""
    lib = _capi.load()
    p = _linear(in_type=kind, out_type=kind, rows=0, x=None, y=None, activation=2)
    assert lib.scenerf_hip_linear_workspace(C.byref(p), 1) == 0
    assert lib.scenerf_hip_linear_backward(C.byref(p), None) == 0
    r = _rms(type=kind, rows=0, x=None, y=None)
    assert lib.scenerf_hip_rms_workspace(C.byref(r), 1) == 0
    assert lib.scenerf_hip_rms_backward(C.byref(r), None) == 0


def test_forward_mode_derivatives_are_refused():
    """A dual tensor asks for no gradient and has an address like any: without a refusal its tangent would be lost without a word."""
    import torch.autograd.forward_ad as fwd
    x, w, b = torch.ones(3, 4), torch.ones(5, 4), torch.ones(5)
    q, s, wq = x.to(torch.float8_e4m3fn), torch.ones(3), w.to(torch.float8_e4m3fn)
    one = torch.ones(4)
    with fwd.dual_level():
        def dual(t):
            return fwd.make_dual(t, torch.ones_like(t))
        for call in (lambda: linear(dual(x), w), lambda: linear(x, dual(w), b), lambda: linear(x, w, dual(b)), lambda: linear(x, w, residual=dual(torch.ones(3, 5))),
                     lambda: linear_8bit(q, dual(s), wq, b), lambda: linear_8bit(q, s, wq, dual(b)), lambda: linear_8bit(q, s, wq, b, dual(b)),
                     lambda: linear_8bit(q, s, wq, b, residual=dual(torch.ones(3, 5))), lambda: quantize_rows(dual(x)),
                     lambda: rms_norm(dual(x), one), lambda: rms_norm(x, dual(one)), lambda: rms_norm(x, one, residual=dual(x)),
                     lambda: rms_norm_8bit(dual(x), one), lambda: rms_norm_8bit(x, dual(one)), lambda: rms_norm_8bit(x, one, residual=dual(x))):
            with pytest.raises(RuntimeError, match="forward-mode"):
                call()
            with torch.no_grad(), pytest.raises(RuntimeError, match="forward-mode"):
                call()
        with pytest.raises(RuntimeError, match="GPU only"):         # inside a level, but without a tangent
            linear(x, w)


@pytest.mark.parametrize("back", ["linear", "rms_norm"])
def test_a_step_back_of_a_dual_tensor_is_refused(back):
    """Forward mode over a step back: the incoming gradient alone has a tangent."""
    import torch.autograd.forward_ad as fwd
    from scenerf_amd.linear import linear_step_back
    from scenerf_amd.norm import rms_step_back
    with fwd.dual_level():
        dy = fwd.make_dual(torch.ones(3, 4), torch.ones(3, 4))
        with pytest.raises(RuntimeError, match="forward-mode"):
            if back == "linear":
                linear_step_back((torch.ones(3, 4), torch.ones(4, 4), None, 3, 4, 4, 4, 0, 0), dy, (3, 4), True, True, True)
            else:
                rms_step_back(torch.ones(3, 4), torch.ones(4), torch.ones(3), 1e-6, dy, None, True, True)


def test_gradients_in_32_bits_are_asked_for_by_their_type():
    lib = _capi.load()
    back = dict(dx=4096, dw=4096, dy=4096, ld_dy=4)
    assert lib.scenerf_hip_linear_workspace(C.byref(_linear(in_type=1, out_type=0, **back)), 1) >= 4 * 8 * 4
    assert "differ" in _said(lib.scenerf_hip_linear_backward(C.byref(_linear(in_type=1, out_type=2, **back)), None))
    assert "differ" in _said(lib.scenerf_hip_linear_backward(C.byref(_linear(in_type=0, out_type=1, **back)), None))
    assert "differ" in _said(lib.scenerf_hip_linear_forward(C.byref(_linear(in_type=2, out_type=0)), None))
    assert "dweight_f32" in _said(lib.scenerf_hip_rms_backward(C.byref(_rms(dweight=4096, dy=4096, rstd=4096, dweight_f32=2)), None))


def test_a_lazily_negated_tensor_is_read_as_it_reads():
    """The imaginary part of a conjugate holds its numbers with the other sign and a flag: what the kernels are given an address of has none."""
    from scenerf_amd.rowops import rows_of, vector_of
    c = torch.complex(torch.ones(5, 1), torch.full((5, 1), 3.0)).conj()
    assert c.imag.is_neg()
    got = rows_of(c.imag, 1)
    assert not got.is_neg() and torch.equal(got, torch.full((5, 1), -3.0))
    wide = torch.complex(torch.ones(4, 8), torch.full((4, 8), 3.0)).conj().imag
    assert not rows_of(wide, 8).is_neg() and rows_of(wide, 8).stride(1) == 1 and torch.equal(rows_of(wide, 8), wide)
    one = c.imag[0]
    assert one.is_neg() and one.is_contiguous() and not vector_of(one).is_neg() and torch.equal(vector_of(one), torch.full((1,), -3.0))
    plain = torch.ones(7)
    assert vector_of(plain) is plain and vector_of(torch.ones(7, 2)[:, 0]).is_contiguous()


def test_a_net_without_norms_says_where_it_is_evaluated():
    from scenerf_amd.model import ResnetFC
    for call in (lambda m: m(), lambda m: m(torch.zeros(1, 2522)), lambda m: m(zx=torch.zeros(1, 2522)), lambda m: m(points=1, views=2)):
        with pytest.raises(RuntimeError, match="render_rays_batch"):
            call(ResnetFC(d_hidden=16, n_blocks=1))
    for call in (lambda m: m(), lambda m: m(torch.zeros(1, 2522), 1), lambda m: m(points=1)):
        with pytest.raises(TypeError):
            call(ResnetFC(d_hidden=16, n_blocks=1, norm="rms"))
