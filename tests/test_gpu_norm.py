"""rms_norm / rms_norm_8bit (scenerf_amd.norm) against their definitions in 64 bits (rowops_util: bounds per element)."""
import pytest
import torch

from rowops_util import hold, rms64
from test_gpu_linear import DEV, TYPES, gen, normal

pytestmark = pytest.mark.gpu
# rows x width: one element, odd widths, a wave's chunk and its neighbours, the widest row in registers and wider ones
SIZES = [(1, 1), (1, 512), (3, 7), (5, 63), (8, 64), (130, 65), (33, 511), (1000, 512), (9, 513), (17, 515), (64, 1536), (5, 2480), (3, 4095),
         (3, 4096), (3, 4097), (2, 4104), (2, 10000), (4801, 130)]


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("m,d", SIZES)
def test_forward_and_gradients(m, d, dtype):
    from scenerf_amd.norm import rms_norm
    g = gen("rms", m, d, dtype)
    x, r, w = normal(g, m, d, dtype=dtype, scale=2.0), normal(g, m, d, dtype=dtype), (1 + 0.1 * normal(g, d)).to(dtype)
    dy, dh = normal(g, m, d, dtype=dtype), normal(g, m, d, dtype=dtype)
    want = rms64(x, w, 1e-6)
    hold(rms_norm(x, w), want["y"], "y")
    x, r, w = (t.requires_grad_(True) for t in (x, r, w))
    y, h = rms_norm(x, w, residual=r, eps=1e-5)
    dx, dr, dw = torch.autograd.grad((y, h), (x, r, w), (dy, dh))
    want = rms64(x.detach(), w.detach(), 1e-5, r.detach(), dy, dh)
    for name, got in (("y", y), ("h", h), ("dx", dx), ("dx", dr), ("dw", dw)):
        hold(got.detach(), want[name], name)
    y = rms_norm(x, w)
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    want = rms64(x.detach(), w.detach(), 1e-6, None, dy)
    for name, got in (("y", y), ("dx", dx), ("dw", dw)):
        hold(got.detach(), want[name], "no residual " + name)


def test_gradients_against_differences():
    from scenerf_amd.norm import rms_norm
    g = gen("rmsdiff")
    x, r, w = normal(g, 11, 37), normal(g, 11, 37), normal(g, 37)
    c, e2 = normal(g, 11, 37), normal(g, 11, 37)
    leaves = [t.requires_grad_(True) for t in (x, r, w)]
    y, h = rms_norm(x, w, residual=r, eps=1e-3)
    grads = torch.autograd.grad((y * c).sum() + (h * e2).sum(), leaves)
    for i in range(3):
        d = normal(g, *leaves[i].shape).double()
        ends = []
        for s in (1e-4, -1e-4):
            v = [t.detach().double() for t in leaves]
            v[i] = v[i] + s * d
            hh = v[0] + v[1]
            yy = hh / torch.sqrt((hh * hh).mean(1, keepdim=True) + 1e-3) * v[2]
            ends.append(float((yy * c.double()).sum() + (hh * e2.double()).sum()))
        want, got = (ends[0] - ends[1]) / 2e-4, float((grads[i].double() * d).sum())
        # differences: 1e-8 / 6 of the third derivative (under 100 per element at rows of norm about 1); the kernels: 2^-18 of the terms
        assert abs(got - want) <= 2.0 ** -18 * float((grads[i].double() * d).abs().sum()) + 2e-6 * float(c.abs().sum()), (i, got, want)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_layouts_and_missing_gradients(dtype):
    from scenerf_amd.norm import rms_norm
    g = gen("rmslay", dtype)
    zs = normal(g, 60, 3, 128, dtype=dtype).requires_grad_(True)        # three blocks' parts side by side
    r, w = normal(g, 60, 128, dtype=dtype), normal(g, 128, dtype=dtype)
    parts = zs.unbind(1)
    dy = normal(g, 60, 128, dtype=dtype)
    y, h = rms_norm(parts[1], w, residual=r)
    got = torch.autograd.grad(y, zs, dy)[0]                             # h unused
    want = rms64(zs.detach()[:, 1], w, 1e-6, r, dy)
    hold(y.detach(), want["y"], "y")
    hold(got[:, 1].contiguous(), want["dx"], "dx")
    assert not got[:, 0].any() and not got[:, 2].any()
    y, h = rms_norm(parts[2], w, residual=r)
    got = torch.autograd.grad(h, zs, dy)[0]                             # y unused: the addition's gradient alone
    assert torch.equal(got[:, 2], dy)
    odd = normal(g, 61, 131, dtype=dtype)[:, 3:]                        # rows that are not aligned
    hold(rms_norm(odd, w), rms64(odd, w, 1e-6)["y"], "unaligned")
    t = normal(g, 128, 61, dtype=dtype).t()
    hold(rms_norm(t, w), rms64(t, w, 1e-6)["y"], "transposed")
    one = normal(g, 1, 128, dtype=dtype).expand(9, 128)
    hold(rms_norm(one, w, residual=one)[0], rms64(one, w, 1e-6, one)["y"], "one row, expanded")
    x = normal(g, 2, 3, 128, dtype=dtype).requires_grad_(True)
    hold(torch.autograd.grad(rms_norm(x, w).sum(), x)[0], rms64(x.detach(), w, 1e-6, None, torch.ones_like(x))["dx"], "three dimensions, dy of ones")
    e = torch.empty(0, 128, dtype=dtype, device=DEV).requires_grad_(True)
    w2 = w.clone().requires_grad_(True)
    de, dw = torch.autograd.grad(rms_norm(e, w2).sum(), (e, w2))
    assert de.shape == (0, 128) and not dw.any()


def test_rows_that_are_zero_or_not_numbers():
    from scenerf_amd.norm import rms_norm, rms_norm_8bit
    for d in (512, 515, 5000):
        x = torch.ones(5, d, device=DEV, dtype=torch.bfloat16)
        w = torch.full((d,), 2.0, device=DEV, dtype=torch.bfloat16)
        x[1], x[2, d - 1], x[3, 0] = 0, float("nan"), float("inf")
        y = rms_norm(x, w)
        assert bool((y[0] == 2).all()) and not y[1].any() and bool(torch.isnan(y[2]).all()) and bool((y[4] == 2).all())
        assert bool(torch.isnan(y[3, 0])) and not y[3, 1:].any()
        q, s = rms_norm_8bit(x, w)
        back = q.float() * s[:, None]
        assert bool((back[0] == back[4]).all()) and abs(float(back[0, 0]) - 2) <= 2 * 2.0 ** -4 and not back[1].any()
        assert bool(torch.isnan(back[2:4]).all())


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("m,d", SIZES)
def test_8bit_output(m, d, dtype):
    from scenerf_amd.norm import rms_norm_8bit
    g = gen("rms8", m, d, dtype)
    x, r, w = normal(g, m, d, dtype=dtype), normal(g, m, d, dtype=dtype), (1 + 0.1 * normal(g, d)).to(dtype)
    for res in (None, r):
        got = rms_norm_8bit(x, w, residual=res)
        q, s = got[:2]
        y = rms64(x, w, 1e-6, res)["y"][0]
        scale = (y.abs().amax(1) / 448).clamp(min=2.0 ** -126)
        e = (d + 32) * 2.0 ** -23
        assert bool(((s.double() - scale).abs() <= e * scale).all())
        v = y / s.double()[:, None]
        assert bool(((q.double() - v).abs() <= (2.0 ** -4 + 2 * e) * v.abs() + 2.0 ** -10 * (1 + e)).all())
        if res is not None:
            hold(got[2], rms64(x, w, 1e-6, res)["h"], "h")


def test_a_chain_as_a_block_runs_it():
    """rms_norm -> linear with activation -> linear onto the residual stream, and the same in 8 bits."""
    from scenerf_amd.linear import linear, linear_8bit, quantize_rows
    from scenerf_amd.norm import rms_norm, rms_norm_8bit
    g = gen("chain")
    bf = torch.bfloat16
    x, h0 = normal(g, 700, 128, dtype=bf), normal(g, 700, 128, dtype=bf)
    gain, w0, w1 = (1 + 0.1 * normal(g, 128)).to(bf), normal(g, 256, 128, dtype=bf, scale=128 ** -0.5), normal(g, 128, 256, dtype=bf, scale=256 ** -0.5)
    b0, b1, dy = normal(g, 256, dtype=bf), normal(g, 128, dtype=bf), normal(g, 700, 128, dtype=bf)
    leaves = [t.requires_grad_(True) for t in (x, h0, gain, w0, b0, w1, b1)]

    def block(norm, lin, x, h0, gain, w0, b0, w1, b1):
        a, h = norm(x, gain, h0)
        return lin(lin(a, w0, b0, "gelu", None), w1, b1, "none", h)

    y = block(lambda x, w, r: rms_norm(x, w, residual=r), lambda x, w, b, act, r: linear(x, w, b, activation=act, residual=r), *leaves)
    grads = torch.autograd.grad(y, leaves, dy)

    def norm64(x, w, r):
        h = x + r
        return h / torch.sqrt((h * h).mean(-1, keepdim=True) + 1e-6) * w, h

    def lin64(x, w, b, act, r):
        z = x @ w.t() + b
        z = torch.nn.functional.gelu(z) if act == "gelu" else z
        return z if r is None else z + r
    wide = [t.detach().double().requires_grad_(True) for t in leaves]
    y64 = block(norm64, lin64, *wide)
    grads64 = torch.autograd.grad(y64, wide, dy.double())
    # at most 6 roundings of 2^-8 on the way to any output, each amplified by at most 1.2 (unit-variance layers); in the 2-norm they add in squares
    room = 6 ** 0.5 * 1.2 * 2.0 ** -8
    for got, want in zip((y.detach(),) + grads, (y64.detach(),) + grads64):
        assert float((got.double() - want).norm() / want.norm()) <= room
    with torch.no_grad():
        q, s, h = rms_norm_8bit(x, gain, residual=h0)
        t = linear_8bit(q, s, *quantize_rows(w0), b0, activation="gelu")
        y8 = linear_8bit(*quantize_rows(t), *quantize_rows(w1), b1, residual=h)
    # four operands in e4m3: at most 2^-4 each on a branch of about half the result's size
    assert float((y8.double() - y64.detach()).norm() / y64.detach().norm()) <= 4 ** 0.5 * 2.0 ** -4


def test_graph_replays():
    from scenerf_amd.norm import rms_norm
    g = gen("rmsgraph")
    x, r, w = (t.requires_grad_(True) for t in (normal(g, 333, 512, dtype=torch.bfloat16), normal(g, 333, 512, dtype=torch.bfloat16),
                                                normal(g, 512, dtype=torch.bfloat16)))
    dy = normal(g, 333, 512, dtype=torch.bfloat16)

    def step():
        y, h = rms_norm(x, w, residual=r)
        return (y, h) + torch.autograd.grad((y, h), (x, w), (dy, dy))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        out = [t.detach() for t in step()]
    for _ in range(3):
        with torch.no_grad():
            x.copy_(normal(g, 333, 512, dtype=torch.bfloat16))
        gr.replay()
        eager = [t.detach() for t in step()]
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, eager))


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("m,d", [(257, 1030), (300, 1536), (260, 2047), (400, 2480), (257, 3000), (300, 4096), (256, 4096), (1, 1025), (520, 5000)])
def test_wide_rows_few_and_many(m, d, dtype):
    """A workgroup a row and a wave a row, either side of the choice between them."""
    from scenerf_amd.norm import rms_norm, rms_norm_8bit
    g = gen("wide", m, d, dtype)
    x, r, w = normal(g, m, d, dtype=dtype), normal(g, m, d, dtype=dtype), (1 + 0.2 * normal(g, d)).to(dtype)
    dy, dh = normal(g, m, d, dtype=dtype), normal(g, m, d, dtype=dtype)
    leaves = [t.requires_grad_(True) for t in (x, r, w)]
    y, h = rms_norm(x, w, residual=r)
    dx, dr, dw = torch.autograd.grad((y, h), leaves, (dy, dh))
    want = rms64(x.detach(), w.detach(), 1e-6, r.detach(), dy, dh)
    for name, t in (("y", y), ("h", h), ("dx", dx), ("dx", dr), ("dw", dw)):
        hold(t.detach(), want[name], name)
    q, s, h8 = rms_norm_8bit(x.detach(), w.detach(), residual=r.detach())
    assert torch.equal(h8, h.detach())
    exact, bound = want["y"]
    top = exact.abs().amax(1)
    assert bool(((s.double() - top / 448).abs() <= (top / 448) * (d + 24) * 2.0 ** -23).all())
    # half a step of e4m3 at the value, or of its smallest values, on top of the unrounded y's own error
    room = 2.0 ** -4 * exact.abs() + s.double()[:, None] * 2.0 ** -10 + (d + 24) * 2.0 ** -22 * exact.abs()
    assert bool(((q.double() * s.double()[:, None] - exact).abs() <= room * (1 + 2.0 ** -10)).all())


def test_wide_8bit_rows_whose_weighted_values_overflow():
    """h w beyond the largest fp32, h rstd w inside it: the scale comes from y."""
    from scenerf_amd.norm import rms_norm_8bit
    g = gen("overflow")
    x, w = normal(g, 3, 5000) * 1e10, torch.ones(5000, device=DEV)
    w[7] = 1e30
    q, s = rms_norm_8bit(x, w)
    y = rms64(x, w, 1e-6)["y"][0]
    assert bool(torch.isfinite(s).all()) and bool(((s.double() / (y.abs().amax(1) / 448) - 1).abs() <= 2.0 ** -10).all())
    assert bool(((q[:, 7].double() * s.double() - y[:, 7]).abs() <= 2.0 ** -4 * y[:, 7].abs()).all())


def test_rows_past_32_bit_offsets():
    """More than 2^31 elements, the gradient on the last rows alone: their own call is the oracle."""
    from scenerf_amd.norm import rms_norm, rms_norm_8bit
    g = gen("large rms")
    m, d, last, bf = 4_200_000, 520, 300, torch.bfloat16
    x = torch.empty(m, d, dtype=bf, device=DEV).normal_(generator=g).requires_grad_(True)
    r = torch.empty(m, d, dtype=bf, device=DEV).normal_(generator=g)
    w = (1 + 0.1 * normal(g, d)).to(bf).requires_grad_(True)
    y, h = rms_norm(x, w, residual=r)
    dy = torch.zeros(m, d, dtype=bf, device=DEV)
    dy[-last:] = normal(g, last, d, dtype=bf)
    dx, dw = torch.autograd.grad(y, (x, w), dy)
    want = rms64(x.detach()[-last:], w.detach(), 1e-6, r[-last:], dy[-last:])
    for name, t in (("y", y.detach()[-last:]), ("h", h.detach()[-last:]), ("dx", dx[-last:]), ("dw", dw)):
        hold(t, want[name], name)
    assert not bool(dx[:-last].any())
    del dx, dy, y, h
    with torch.no_grad():
        q, s, _ = rms_norm_8bit(x, w, residual=r)
        one = rms_norm_8bit(x[-last:], w, residual=r[-last:])
    assert torch.equal(q[-last:].view(torch.uint8), one[0].view(torch.uint8)) and torch.equal(s[-last:], one[1])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("m,d", [(1, 16), (1, 5000), (3, 515), (32, 272), (120, 512), (4801, 515), (700, 4100)])
def test_gradients_are_made_from_the_unrounded_sum(m, d, dtype):
    """16 bits: the gradients against the formula at x + residual, with bounds that know no rounding of h."""
    from scenerf_amd.norm import rms_norm
    g = gen("unrounded", m, d, dtype)
    x, r, dy, dh = (normal(g, m, d, dtype=dtype) for _ in range(4))
    w = (1 + 0.2 * normal(g, d)).to(dtype)
    leaves = [t.requires_grad_(True) for t in (x, r, w)]
    dx, dr, dw = torch.autograd.grad(rms_norm(x, w, residual=r), leaves, (dy, dh))
    # in 32 bits x + r is off by 2^-24 at most: the oracle without a residual, on that sum, rounded as the outputs are
    want = rms64(x.detach().double() + r.detach().double(), w.detach().double(), 1e-6, None, dy.double(), dh.double())
    u, tiny, e = torch.finfo(dtype).eps / 2, torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2, (d + 64) * 2.0 ** -22
    for name, got in (("dx", dx), ("dx", dr), ("dw", dw)):
        value, _ = want[name]
        h64 = x.detach().double() + r.detach().double()
        rstd = 1 / torch.sqrt((h64 * h64).mean(1, keepdim=True) + 1e-6)
        if name == "dx":
            a = (dy.double() * w.detach().double()).abs()
            size = rstd * (a + (h64 * rstd).abs() * (a * (h64 * rstd).abs()).mean(1, keepdim=True)) + dh.double().abs()
        else:
            size = (dy.double() * h64 * rstd).abs().sum(0) * (1 + m)
        hold(got, (value, u * value.abs() + e * size + tiny), name)


@pytest.mark.parametrize("m,d", [(3, 1030), (3, 5000), (300, 4096), (5, 512)])
def test_8bit_rows_whose_weighted_values_underflow(m, d):
    """h w below the smallest fp32, h rstd w well above it: the scale comes from y."""
    from scenerf_amd.norm import rms_norm_8bit
    g = gen("underflow", m, d)
    x, w = normal(g, m, d) * 1e-18, (1 + 0.1 * normal(g, d)) * 1e-25
    for rows in (slice(None), slice(0, 1)):
        q, s = rms_norm_8bit(x[rows], w, eps=0.0)
        y = rms64(x[rows], w, 0.0)["y"][0]
        assert bool(((s.double() / (y.abs().amax(1) / 448) - 1).abs() <= (d + 32) * 2.0 ** -23).all())
        back = q.double() * s.double()[:, None]
        assert bool(((back - y).abs() <= (2.0 ** -4 + 2.0 ** -10) * y.abs() + s.double()[:, None] * 2.0 ** -9).all())
    x[1] = 0                                        # (and a row of zeros stays one)
    q, s = rms_norm_8bit(x, w, eps=1e-30)
    assert not bool(q[1].float().any()) and float(s[1]) == 2.0 ** -126


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("m,d", [(1, 5000), (3, 515), (32, 272), (120, 512), (4801, 515), (700, 4100)])
def test_gradients_do_not_know_the_rounded_sum(m, d, dtype):
    """16 bits, in the 2-norm: the gradients are off by their own rounding and 32-bit sums, and an oracle made from h as it is stored is not."""
    from scenerf_amd.norm import rms_norm
    g = gen("unrounded norm", m, d, dtype)
    x, r = normal(g, m, d, dtype=dtype), normal(g, m, d, dtype=dtype)
    w = (1 + 0.2 * normal(g, d)).to(dtype)
    h64 = x.double() + r.double()
    leaves = [t.requires_grad_(True) for t in (x, r, w)]
    # for dx a dy along h, so that the mean term weighs as much as the first; for dw one across it, so that its sum does not outgrow h's roundings
    noise = normal(g, m, d)
    along, across = (h64 + 0.5 * noise.double()).to(dtype), noise.to(dtype)
    dx, dr = torch.autograd.grad(rms_norm(x, w, residual=r)[0], leaves[:2], along)
    dw, = torch.autograd.grad(rms_norm(x, w, residual=r)[0], leaves[2:], across)
    assert torch.equal(dx, dr)

    def oracle(h, dy):
        rstd = 1 / torch.sqrt((h64 * h64).mean(1, keepdim=True) + 1e-6)
        a, xhat = dy.double() * w.detach().double(), h * rstd
        terms = dy.double() * xhat
        return {"dx": (rstd * (a - xhat * (a * xhat).mean(1, keepdim=True)), rstd * (a.abs() + xhat.abs() * (a * xhat).abs().mean(1, keepdim=True))),
                "dw": (terms.sum(0), (terms * terms).sum(0).sqrt())}
    for name, got, dy in (("dx", dx, along), ("dw", dw, across)):
        value, size = oracle(h64, dy)[name]
        stored, _ = oracle(h64.to(dtype).double(), dy)[name]
        own = float((value.to(dtype).double() - value).norm())
        # a value off by e before it is rounded is off by at most 2 e more behind it; the errors of 32-bit sums of m and d terms add in squares
        lim = own + 2 * 4 * (m ** 0.5 + d ** 0.5) * 2.0 ** -24 * float(size.norm())
        assert float((got.double() - value).norm()) <= lim, (name, float((got.double() - value).norm()), own, lim)
        worse = float((stored.to(dtype).double() - value).norm())
        assert worse > 1.1 * lim, (name, worse, lim)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("m,d", [(0, 24), (1, 16), (33, 515), (4801, 130), (700, 4100)])
def test_the_weights_gradient_as_it_is_summed(m, d, dtype):
    """``sums``: dweight in fp32, whose rounding is the gradient that autograd gets.  Against 64 bits: 32-bit sums' errors of m and d terms, in squares."""
    from scenerf_amd.norm import rms_step_back
    from scenerf_amd.rowops import rows_forward
    g = gen("norm sums", m, d, dtype)
    x, r, dy = (normal(g, m, d, dtype=dtype) for _ in range(3))
    w = (1 + 0.2 * normal(g, d)).to(dtype)
    _, _, h, rstd, x2 = rows_forward("rms_norm", x, w, r, 1e-6, keep_rstd=True)
    dx, dw = rms_step_back(x2, w, rstd, 1e-6, dy, None, True, True, r, sums=True)
    dx2, rounded = rms_step_back(x2, w, rstd, 1e-6, dy, None, True, True, r)
    assert dw.dtype == torch.float32 and rounded.dtype == dtype and torch.equal(dw.to(dtype), rounded) and torch.equal(dx, dx2)
    h64 = x.double() + r.double()
    terms = dy.double() * h64 / torch.sqrt((h64 * h64).mean(1, keepdim=True) + 1e-6)
    lim = 4 * (m ** 0.5 + d ** 0.5) * 2.0 ** -24 * float((terms * terms).sum(0).sqrt().norm())
    assert float((dw.double() - terms.sum(0)).norm()) <= lim
