"""ResnetFC(norm="rms"): the row operators together as a net runs them, on its own (against 64 bits) and inside the render pass (against the
pipeline's oracle with this net in the place of its own)."""
import math

import pytest
import torch

import scenerf_oracle as orc
from scenerf_amd import synth
from scenerf_amd.model import ResnetFC, SceneRF

pytestmark = pytest.mark.gpu
DEV = "cuda"
ACT = {"relu": torch.relu, "gelu": torch.nn.functional.gelu, "silu": torch.nn.functional.silu}


def net_state(seed, d_out, n_blocks, d_hidden, out_scale=1.0):
    sd = synth.mlp_state(seed, d_out, d_hidden=d_hidden, n_blocks=n_blocks, out_scale=out_scale)
    g = torch.Generator().manual_seed(seed)
    for b in range(n_blocks):
        sd["blocks.%d.norm.weight" % b] = 1 + 0.2 * torch.randn(d_hidden, generator=g)
        sd["blocks.%d.fc_1.weight" % b] = torch.randn(d_hidden, d_hidden, generator=g) * d_hidden ** -0.5
    sd["norm_out.weight"] = 1 + 0.2 * torch.randn(d_hidden, generator=g)
    return sd


def net(seed, d_out, n_blocks, d_hidden, activation="gelu", out_scale=1.0):
    m = ResnetFC(d_out=d_out, n_blocks=n_blocks, d_hidden=d_hidden, norm="rms", activation=activation)
    m.load_state_dict(net_state(seed, d_out, n_blocks, d_hidden, out_scale))
    return m.to(DEV)


def plain(p, zx, activation="gelu", eps=1e-6, **_):
    """The net from its formula, in the type of ``zx``: what the oracle's own net is replaced with."""
    lin = lambda x, name: x @ p[name + ".weight"].to(zx.dtype).t() + p[name + ".bias"].to(zx.dtype)
    norm = lambda h, name: h / torch.sqrt((h * h).mean(-1, keepdim=True) + eps) * p[name + ".weight"].to(zx.dtype)
    z, x = zx[..., :2480], zx[..., 2480:]
    h = lin(x, "lin_in")
    for b in range(sum(1 for k in p if k.endswith(".fc_0.weight"))):
        h = h + lin(z, "lin_z.%d" % b)
        h = h + lin(ACT[activation](lin(norm(h, "blocks.%d.norm" % b), "blocks.%d.fc_0" % b)), "blocks.%d.fc_1" % b)
    return lin(norm(h, "norm_out"), "lin_out")


def room(dtype, n_blocks, rows):
    """Relative error in the 2-norm.  32 bits: a sum of k products of either sign is off by about sqrt(k) 2^-24; 3 layers a block, lin_in and
    lin_out, there and back, each amplified by at most 2 (norms and gains near 1).  16 bits: at most 8 roundings a block (three weights, their
    inputs, the stream) and as many back, 4 at the ends, each off by 2^-8 (fp16: 2^-11), amplified by 1.2; they add in squares."""
    u = torch.finfo(dtype).eps / 2
    if dtype == torch.float32:
        return 2 * (6 * n_blocks + 4) * max(2480, rows) ** 0.5 * u
    return (16 * n_blocks + 8) ** 0.5 * 1.2 * u


def off(got, want):
    got, want = got.detach().double(), want.detach().double()
    return float((got - want).norm() / want.norm())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("rows,n_blocks,d_hidden,activation", [(1, 1, 16, "relu"), (131, 2, 80, "silu"), (700, 3, 128, "gelu"), (300, 1, 512, "gelu")])
def test_the_net_and_its_gradients_against_64_bits(rows, n_blocks, d_hidden, activation, dtype):
    m = net(3, 4, n_blocks, d_hidden, activation)
    g = torch.Generator(device=DEV).manual_seed(rows)
    zx = torch.randn(rows, 2480 + 42, generator=g, device=DEV).to(dtype).requires_grad_(True)
    dy = torch.randn(rows, 4, generator=g, device=DEV).to(dtype)
    y = m(zx)
    assert y.shape == (rows, 4) and y.dtype == dtype
    names, params = zip(*m.named_parameters())
    got = torch.autograd.grad(y, (zx,) + params, dy)
    p64 = {k: v.detach().double().requires_grad_(True) for k, v in zip(names, params)}
    zx64 = zx.detach().double().requires_grad_(True)
    y64 = plain(p64, zx64, activation)
    want = torch.autograd.grad(y64, (zx64,) + tuple(p64[k] for k in names), dy.double())
    lim = room(dtype, n_blocks, rows)
    if activation == "relu" and dtype != torch.float32:      # a unit whose input is rounded across 0 has its whole slope wrong
        lim = None
    assert off(y, y64) <= room(dtype, n_blocks, rows)
    for name, a, b in zip(("zx",) + names, got, want):
        assert bool(torch.isfinite(a).all()), name
        assert lim is None or off(a, b) <= lim, (name, off(a, b), lim)


def test_no_rows_one_row_and_more_dimensions():
    m = net(5, 2, 2, 32)
    zx = torch.randn(3, 4, 2522, device=DEV)
    with torch.no_grad():
        y = m(zx)
        assert y.shape == (3, 4, 2) and m(zx[:0]).shape == (0, 4, 2) and m(zx[0, 0]).shape == (2,)
        assert off(m(zx[1, 2]), y[1, 2]) <= room(torch.float32, 2, 1) and torch.equal(m(zx.view(12, 2522)).view(3, 4, 2), y)
    got = torch.autograd.grad(m(zx[:0].requires_grad_(True)).sum(), list(m.parameters()))
    assert all(float(t.abs().max()) == 0.0 for t in got)
    with pytest.raises(ValueError):
        m(zx[..., :2500])
    with pytest.raises(TypeError):
        m(zx, zx)


def packed(m, precision, trainable):
    from scenerf_amd.normed import PackedNormedMLP
    cfg = SceneRF(som_sigma=2.0, std=2.0, add_fov_hor=20, add_fov_ver=8, precision=precision).render_cfg
    p = m.ordered_params()
    return PackedNormedMLP(list(p), p, m.d_out, cfg, trainable)


@pytest.mark.parametrize("precision", ["fp32", "bf16"])
@pytest.mark.parametrize("rows,n_blocks,d_hidden,d_out", [(1, 1, 16, 2), (257, 2, 144, 4), (1000, 3, 512, 2)])
def test_the_passes_of_a_session_against_64_bits(rows, n_blocks, d_hidden, d_out, precision):
    m = net(7, d_out, n_blocks, d_hidden)
    pk = packed(m, precision, True)
    g = torch.Generator(device=DEV).manual_seed(rows)
    Z = torch.randn(rows, 2480, generator=g, device=DEV).to(pk.dtype)
    xenc = torch.zeros(rows, 48, device=DEV)
    xenc[:, :42] = torch.randn(rows, 42, generator=g, device=DEV)
    dy = torch.randn(rows, d_out, generator=g, device=DEV)
    y, saved = pk.forward(xenc, Z, True)
    bare, nothing = pk.forward(xenc, Z, False)
    assert nothing is None and torch.equal(y, bare) and y.dtype == torch.float32
    names = dict(m.named_parameters())
    p64 = {k: v.detach().double().requires_grad_(True) for k, v in names.items()}
    order = [next(k for k, v in names.items() if v is t) for t in m.ordered_params()]
    z64 = Z.double().requires_grad_(True)
    y64 = plain(p64, torch.cat([z64, xenc[:, :42].double()], 1))
    want = torch.autograd.grad(y64, [z64] + [p64[k] for k in order], dy.double())
    lim = room(pk.dtype, n_blocks, rows)
    assert off(y, y64) <= lim
    dzs = pk.backward(saved, dy)
    assert off(dzs.float() @ pk.net.w_z.float(), want[0]) <= lim
    once = [t.clone() for t in pk.unpack_grads()]
    for name, a, b in zip(order, once, want[1:]):
        assert a.shape == names[name].shape and off(a, b) <= lim, (name, off(a, b), lim)
    pk.backward(saved, dy)       # a second chunk of the session adds to the first's
    for a, b in zip(pk.unpack_grads(), once):
        assert torch.equal(a, 2 * b)


def test_eight_bits():
    """no_grad passes in e4m3: both operands of each of the 3 products a block are off by at most 2^-4, in squares."""
    m = net(9, 4, 2, 256)
    m.eight_bit = True
    g = torch.Generator(device=DEV).manual_seed(1)
    Z, xenc = torch.randn(515, 2480, generator=g, device=DEV).to(torch.bfloat16), torch.zeros(515, 48, device=DEV)
    xenc[:, :42] = torch.randn(515, 42, generator=g, device=DEV)
    for precision in ("bf16", "fp32"):
        pk = packed(m, precision, False)
        assert pk.eight is not None and packed(m, precision, True).eight is None
        y, _ = pk.forward(xenc, Z.to(pk.dtype), False)
        y64 = plain({k: v.detach().double() for k, v in m.named_parameters()}, torch.cat([Z.double(), xenc[:, :42].double()], 1))
        assert 1e-3 < off(y, y64) <= (2 * 3 * 2) ** 0.5 * 2.0 ** -4


KW = dict(sphere_W=376, sphere_H=114, n_pts_uni=32, n_pts_per_gaussian=8)


def render_case(R, seed=0):
    maps = synth.feature_maps(376, 114, 13 + seed, smooth=True)
    nu, ng = synth.sampling_noise(R, 32, 32, 15 + seed)
    return maps, synth.stride2_pixels((1220, 370), R, 14 + seed), nu, ng, synth.kitti_cam_K(), synth.rel_pose(2.0, 10.0)


def model(precision, main, head, **kw):
    m = SceneRF(som_sigma=2.0, std=2.0, add_fov_hor=20, add_fov_ver=8, precision=precision, **KW, **kw)
    m.mlp, m.mlp_gaussian = main, head
    return m.to(DEV)


def loss_of(out):
    return out["depth"].mean() + out["color"].mean() + out["loss_kl"].mean() + out["gaussian_means"].mean()


@pytest.mark.parametrize("precision", ["fp32", "bf16"])
@pytest.mark.parametrize("R", [1, 40])
def test_render_and_its_gradients_against_the_oracle(R, precision, monkeypatch):
    """Both nets with norms, one chunk; the oracle takes the head's offsets, the sphere pixels and the two discrete choices of the RaySOM from
    the render, so what is left between them is the nets' arithmetic.  Tolerances: the render suite's for outputs and gradient norms."""
    monkeypatch.setattr(orc, "resnetfc_forward", plain)
    maps, pix, nu, ng, K, T = render_case(R)
    m = model(precision, net(31, 4, 2, 64), net(32, 2, 1, 48, out_scale=4.0))
    m.debug_aux = True
    x = {k: v.to(DEV).requires_grad_(True) for k, v in maps.items()}
    out = m.render_rays_batch(K.to(DEV), T.to(DEV), x, sampled_pixels=pix.to(DEV), ray_batch_size=R, noise=(nu.to(DEV), ng.to(DEV)))
    aux = {k: v.detach().cpu() for k, v in m.last_aux.items() if torch.is_tensor(v)}
    loss_of(out).backward()
    po = {k: v.detach().cpu().requires_grad_(True) for k, v in m.mlp.named_parameters()}
    pg = {k: v.detach().cpu().requires_grad_(True) for k, v in m.mlp_gaussian.named_parameters()}
    xm = {k: v.clone().requires_grad_(True) for k, v in maps.items()}
    ref = orc.render_chunk(orc.OracleConfig.kitti(**KW), po, pg, K, T, xm, pix, nu, ng, head_offsets=aux["offsets"].reshape(R, 4, 2),
                           sphere_idx=(aux["sphere_idx"].long(), aux["sphere_idx_g"].long()),
                           som_choices=(aux["bmu"].reshape(R, -1).long(), aux["kl_mask"].reshape(R, -1).bool()))
    loss_of(ref).backward()
    tol = dict(depth=1e-4, color=1e-5, grad=1e-2) if precision == "fp32" else dict(depth=2e-2, color=2e-2, grad=1.5e-1)
    assert float(((out["depth"].detach().cpu() - ref["depth"].detach()).abs() / (1 + ref["depth"].detach().abs())).max()) <= tol["depth"]
    assert float((out["color"].detach().cpu() - ref["color"].detach()).abs().max()) <= tol["color"]
    for mod, want in ((m.mlp, po), (m.mlp_gaussian, pg)):
        for k, v in mod.named_parameters():
            assert off(v.grad.cpu(), want[k].grad) <= tol["grad"], (k, off(v.grad.cpu(), want[k].grad))
    for k, v in x.items():
        if float(xm[k].grad.norm()) > 0:
            assert off(v.grad.cpu(), xm[k].grad) <= tol["grad"], (k, off(v.grad.cpu(), xm[k].grad))


def test_chunks_add_up_and_no_grad_renders_the_same():
    """Two chunks (the last one ragged) against one: same outputs, gradients equal up to the order of their sums; a net with norms beside one
    without; ``no_grad`` gives the trained pass's outputs bit for bit."""
    R = 37
    maps, pix, nu, ng, K, T = render_case(R, 3)
    plain_head = ResnetFC(d_out=2, n_blocks=1, d_hidden=64)
    plain_head.load_state_dict(synth.mlp_state(5, 2, d_hidden=64, n_blocks=1, out_scale=4.0))
    m = model("fp32", net(33, 4, 2, 64), plain_head)
    x = {k: v.to(DEV).requires_grad_(True) for k, v in maps.items()}
    leaves = list(m.parameters()) + [x["1_1"], x["1_4"]]
    leaves = [t for t in leaves if t.requires_grad]

    def render(chunk):
        return m.render_rays_batch(K.to(DEV), T.to(DEV), x, sampled_pixels=pix.to(DEV), ray_batch_size=chunk, noise=(nu.to(DEV), ng.to(DEV)))
    grads = {}
    for chunk in (R, 20):
        out = render(chunk)
        grads[chunk] = torch.autograd.grad(loss_of(out), leaves, allow_unused=True)
        with torch.no_grad():
            still = render(chunk)
        for k in ("depth", "color", "weights", "gaussian_means"):
            assert torch.equal(out[k].detach(), still[k]), k
    for a, b in zip(grads[R], grads[20]):
        assert (a is None) == (b is None)
        if a is not None and float(a.norm()) > 0:
            assert off(b, a) <= 64 * 2480 ** 0.5 * 2.0 ** -24


def test_a_captured_training_step_replays():
    """One captured step (both nets with norms, bf16, AdamW inside) against eager steps from the same start."""
    from scenerf_amd.graph import GraphedStep
    from scenerf_amd.optim import FusedAdamW
    R = 96
    maps, pix, nu, ng, K, T = render_case(R, 5)

    def start():
        m = model("bf16", net(41, 4, 2, 128), net(42, 2, 1, 64, out_scale=4.0), device_rng=True)
        params = list(m.mlp.parameters()) + list(m.mlp_gaussian.parameters())
        opt = FusedAdamW(params, lr=1e-4, weight_decay=0.0, capturable=True)
        return m, opt, params, {k: v.to(DEV).requires_grad_(True) for k, v in maps.items()}
    args = (K.to(DEV), T.to(DEV))
    noise = (nu.to(DEV), ng.to(DEV))

    def eager(steps):
        m, opt, params, x = start()
        losses = []
        for _ in range(steps):
            opt.zero_grad(set_to_none=True)
            loss = loss_of(m.render_rays_batch(*args, x, sampled_pixels=pix.to(DEV), ray_batch_size=R, noise=noise))
            loss.backward()
            opt.step()
            losses.append(float(loss.detach()))
        return losses, [p.detach().clone() for p in params]
    losses, ref = eager(5)
    m, opt, params, x = start()
    begin = [p.detach().clone() for p in params]
    gs = GraphedStep(m, opt, loss_of, *args, x, pix.to(DEV), ray_batch_size=R, warmup=2, noise=noise)
    got = []
    for _ in range(3):
        got.append(float(gs()))
        torch.randn(1000, 1000, device=DEV).sum().item()       # eager work of the program's own between replays
    spread = math.sqrt(sum(float((a - b.detach()).norm()) ** 2 for a, b in zip(ref, params)))
    moved = math.sqrt(sum(float((a - b.detach()).norm()) ** 2 for a, b in zip(begin, params)))
    # the same kernels on the same inputs: the nets' gradients have no order of their own (no atomics); the compositing's sums may differ in the last
    # place, and an entry of almost no gradient turns that into a step of the whole learning rate
    assert moved > 0 and spread <= 0.2 * moved, (spread, moved)
    for a, b in zip(got, losses[2:]):
        assert abs(a - b) <= 2e-3 * (1 + abs(b)), (got, losses)


def test_one_reduction_of_the_gradients_per_net():
    """Data parallel: the hook gets one flat buffer per net, and what it leaves there is what the parameters receive."""
    from scenerf_amd.renderer import RenderSession
    R = 8
    maps, pix, nu, ng, K, T = render_case(R, 7)
    m = model("bf16", net(51, 4, 1, 32), net(52, 2, 1, 32, out_scale=4.0))
    seen = []

    def halve(flat):
        seen.append(flat.numel())
        flat.mul_(0.5)

    def grads(sync):
        sess = RenderSession(m.render_cfg, {k: v.to(DEV) for k, v in maps.items()}, m.mlp.ordered_params(), m.mlp_gaussian.ordered_params(), grad_sync=sync)
        out = sess.render_chunk(pix.to(DEV), K.to(DEV), torch.inverse(K).to(DEV), T.to(DEV), nu.to(DEV), ng.to(DEV))
        return torch.autograd.grad(loss_of(out), list(m.mlp.parameters()) + list(m.mlp_gaussian.parameters()))
    whole, half = grads(None), grads(halve)
    assert sorted(seen) == sorted(sum(p.numel() for p in n.parameters()) for n in (m.mlp, m.mlp_gaussian))
    for a, b in zip(whole, half):
        assert off(2 * b, a) <= 2.0 ** -8


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
@pytest.mark.parametrize("rows,n_blocks,d_hidden", [(33, 1, 16), (257, 2, 144), (1000, 3, 512)])
def test_a_session_trains_as_the_net_on_its_own_does(rows, n_blocks, d_hidden, dtype):
    """The same operators on the same rows: every gradient behind lin_in (whose rows are padded in a session) has the same bits, in the type that
    the net's own step rounds it to."""
    m = net(11, 4, n_blocks, d_hidden)
    pk = packed(m, "fp32" if dtype == torch.float32 else "bf16", True)
    g = torch.Generator(device=DEV).manual_seed(rows)
    Z, dy = torch.randn(rows, 2480, generator=g, device=DEV).to(dtype), torch.randn(rows, 4, generator=g, device=DEV).to(dtype)
    xenc = torch.zeros(rows, 48, device=DEV)
    xenc[:, :42] = torch.randn(rows, 42, generator=g, device=DEV).to(dtype).float()
    y, saved = pk.forward(xenc, Z, True)
    own = m(torch.cat([Z, xenc[:, :42].to(dtype)], 1))
    assert torch.equal(y.to(dtype), own.detach())
    want = torch.autograd.grad(own, m.ordered_params(), dy)
    pk.backward(saved, dy.float())
    names = {id(v): k for k, v in m.named_parameters()}
    for p, a, b in zip(m.ordered_params(), pk.unpack_grads(), want):
        kind = torch.float32 if names[id(p)].startswith("lin_out") else dtype
        if not names[id(p)].startswith("lin_in"):
            assert torch.equal(a.to(kind), b.to(kind)), (names[id(p)], off(a, b))


@pytest.mark.parametrize("chunks", [1, 6])
def test_a_session_sums_its_chunks_in_32_bits(chunks):
    """bf16: lin_z's gradients are sums over every chunk's rows of dzs and Z, both in hand here; a rounding to bf16 a chunk would put them 2^-9 off.
    Errors of 32-bit sums of n terms add in squares: sqrt(n) 2^-24 of the terms' norm, four times over."""
    rows, nb, H = 700, 2, 144
    m = net(13, 4, nb, H)
    pk = packed(m, "bf16", True)
    g = torch.Generator(device=DEV).manual_seed(chunks)
    dw, db = torch.zeros(nb * H, 2480, dtype=torch.float64, device=DEV), torch.zeros(nb * H, dtype=torch.float64, device=DEV)
    size_w, size_b = torch.zeros_like(dw), torch.zeros_like(db)
    for _ in range(chunks):
        Z = torch.randn(rows, 2480, generator=g, device=DEV).to(pk.dtype)
        xenc = torch.zeros(rows, 48, device=DEV)
        xenc[:, :42] = torch.randn(rows, 42, generator=g, device=DEV)
        _, saved = pk.forward(xenc, Z, True)
        dzs = pk.backward(saved, torch.randn(rows, 4, generator=g, device=DEV)).double()
        dw, db = dw + dzs.t() @ Z.double(), db + dzs.sum(0)
        size_w, size_b = size_w + (dzs ** 2).t() @ Z.double() ** 2, size_b + (dzs ** 2).sum(0)
    order = {id(t): i for i, t in enumerate(m.ordered_params())}
    got = pk.unpack_grads()
    for b in range(nb):
        for p, want, size in ((m.lin_z[b].weight, dw, size_w), (m.lin_z[b].bias, db, size_b)):
            a = got[order[id(p)]]
            want, size = want[b * H:(b + 1) * H], size[b * H:(b + 1) * H]
            assert a.dtype == torch.float32
            lim = 4 * (chunks * rows) ** 0.5 * 2.0 ** -24 * float(size.sqrt().norm())
            assert float((a.double() - want).norm()) <= lim, (float((a.double() - want).norm()), lim)
