"""linear / linear_8bit / quantize_rows (scenerf_amd.linear) against their definitions in 64 bits (rowops_util: bounds per element)."""
import pytest
import torch

from rowops_util import hold, linear64

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = [torch.float32, torch.bfloat16, torch.float16]
ACTS = ["none", "relu", "gelu", "silu"]


def normal(g, *shape, dtype=torch.float32, scale=1.0):
    return (torch.randn(*shape, generator=g, device=DEV) * scale).to(dtype)


def gen(*key):
    return torch.Generator(device=DEV).manual_seed(sum(ord(c) * (i + 1) for i, c in enumerate(repr(key))))


def whole(g, *shape, dtype, top=2):
    return torch.randint(-top, top + 1, shape, generator=g, device=DEV).to(dtype)


# rows x k x n: one element, one row, odd everything, tile edges (63 .. 65, 127 .. 129, 255 .. 257), short and long sums
SIZES = [(1, 1, 1), (1, 2480, 1536), (2, 42, 515), (7, 48, 4), (33, 130, 2), (63, 64, 65), (64, 63, 64), (65, 257, 63), (129, 128, 127),
         (255, 42, 512), (257, 512, 256), (300, 1000, 24), (513, 31, 130), (1024, 512, 512), (4801, 96, 130)]


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("m,k,n", SIZES)
def test_forward(m, k, n, dtype):
    from scenerf_amd.linear import linear
    g = gen("fwd", m, k, n, dtype)
    x, w, b, r = normal(g, m, k, dtype=dtype), normal(g, n, k, dtype=dtype, scale=k ** -0.5), normal(g, n, dtype=dtype), normal(g, m, n, dtype=dtype)
    for act in ACTS:
        hold(linear(x, w, b, activation=act, residual=r), linear64(x, w, b, act, r)["y"], act)
    hold(linear(x, w), linear64(x, w)["y"], "bare")
    hold(linear(x, w, b), linear64(x, w, b)["y"], "bias")
    hold(linear(x, w, residual=r, activation="gelu"), linear64(x, w, None, "gelu", r)["y"], "residual")


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("m,k,n", SIZES)
def test_gradients_against_the_formula(m, k, n, dtype):
    from scenerf_amd.linear import linear
    g = gen("bwd", m, k, n, dtype)
    for act in ("none", "gelu", "silu"):
        x, w, b, r = normal(g, m, k, dtype=dtype), normal(g, n, k, dtype=dtype, scale=k ** -0.5), normal(g, n, dtype=dtype), normal(g, m, n, dtype=dtype)
        leaves = [t.requires_grad_(True) for t in (x, w, b, r)]
        dy = normal(g, m, n, dtype=dtype)
        y = linear(x, w, b, activation=act, residual=r)
        grads = torch.autograd.grad(y, leaves, dy)
        want = linear64(x.detach(), w.detach(), b.detach(), act, r.detach(), dy)
        hold(y.detach(), want["y"], act + " y")
        for name, got in zip(("dx", "dw", "db", "dr"), grads):
            hold(got, want[name], "%s %s" % (act, name))


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("m,k,n", [(1, 5, 3), (65, 42, 130), (300, 64, 257)])
def test_relu_gradients_on_whole_numbers(m, k, n, dtype):
    """Whole x and w and a bias of halves: every sum is exact and none is 0, so relu's slope is decided and only the results' own rounding is left."""
    from scenerf_amd.linear import linear
    g = gen("relu", m, k, n, dtype)
    x, w, dy = whole(g, m, k, dtype=dtype), whole(g, n, k, dtype=dtype), whole(g, m, n, dtype=dtype)
    b = whole(g, n, dtype=dtype) + 0.5
    x, w, b = (t.requires_grad_(True) for t in (x, w, b))
    y = linear(x, w, b, activation="relu")
    grads = torch.autograd.grad(y, (x, w, b), dy)
    want = linear64(x.detach(), w.detach(), b.detach(), "relu", None, dy)
    for name, got in zip(("y", "dx", "dw", "db"), (y.detach(),) + grads):
        value, exact = want[name][0], want[name][0].to(dtype)
        assert torch.equal(got, exact), (name, float((got.double() - value).abs().max()))


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("m,k,n", [(70001, 96, 264), (66003, 200, 136), (70001, 64, 129)])
def test_more_tiles_than_workgroups(m, k, n, dtype):
    """A workgroup goes through several tiles (results that leave in 16-byte pieces) or many workgroups queue (the odd width)."""
    from scenerf_amd.linear import linear
    g = gen("tiles", m, k, n, dtype)
    x, w, b, r = normal(g, m, k, dtype=dtype), normal(g, n, k, dtype=dtype, scale=k ** -0.5), normal(g, n, dtype=dtype), normal(g, m, n, dtype=dtype)
    for act in ACTS:
        hold(linear(x, w, b, activation=act, residual=r), linear64(x, w, b, act, r)["y"], act)
    hold(linear(x, w), linear64(x, w)["y"], "bare")
    x, w, b = (t.requires_grad_(True) for t in (x, w, b))
    dy = normal(g, m, n, dtype=dtype)
    y = linear(x, w, b, activation="silu")
    want = linear64(x.detach(), w.detach(), b.detach(), "silu", None, dy)
    for name, got in zip(("y", "dx", "dw", "db"), (y.detach(),) + torch.autograd.grad(y, (x, w, b), dy)):
        hold(got, want[name], name)


def test_gradients_against_differences():
    """fp32, 64-bit oracle: (L(p + e d) - L(p - e d)) / 2 e of the definition equals <gradient, d> of the kernels."""
    from scenerf_amd.linear import linear
    g = gen("diff")
    for act in ("gelu", "silu"):
        x, w, b, r = normal(g, 37, 19), normal(g, 23, 19), normal(g, 23), normal(g, 37, 23)
        c = normal(g, 37, 23)
        leaves = [t.requires_grad_(True) for t in (x, w, b, r)]
        grads = torch.autograd.grad((linear(x, w, b, activation=act, residual=r) * c).sum(), leaves)
        for i, name in enumerate("xwbr"):
            d = normal(g, *leaves[i].shape).double()
            e = 1e-4
            ends = []
            for s in (e, -e):
                v = [t.detach().double() for t in leaves]
                v[i] = v[i] + s * d
                ends.append(float((linear64(v[0], v[1], v[2], act, v[3])["y"][0] * c.double()).sum()))
            want = (ends[0] - ends[1]) / (2 * e)
            got = float((grads[i].double() * d).sum())
            # differences: e^2 / 6 of the third derivative (under 10 per element); the kernels: 2^-20 of the terms' magnitudes
            room = 2.0 ** -18 * float((grads[i].double() * d).abs().sum()) + 1e-6 * float(c.abs().sum())
            assert abs(got - want) <= room, (act, name, got, want, room)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_layouts(dtype):
    """Columns of wider tensors (aligned and not), transposed operands, a residual and a dy that one row stands for, more than two dimensions."""
    from scenerf_amd.linear import linear
    g = gen("layout", dtype)
    for off, wide in ((8, 96), (3, 91), (1, 72)):
        big, wbig = normal(g, 70, wide, dtype=dtype), normal(g, 40, wide, dtype=dtype)
        x, w = big[:, off:off + 64], wbig[:, off:off + 64]
        r = normal(g, 70, 40 + off, dtype=dtype)[:, off:]
        x.requires_grad_(True)
        y = linear(x, w, residual=r)
        hold(y.detach(), linear64(x.detach(), w, None, "none", r)["y"], "sliced")
        dy = normal(g, 70, 40 + off, dtype=dtype)[:, off:]
        hold(torch.autograd.grad(y, x, dy)[0], linear64(x.detach(), w, None, "none", r, dy)["dx"], "sliced dx")
    x, w = normal(g, 64, 70, dtype=dtype).t(), normal(g, 64, 40, dtype=dtype).t()
    hold(linear(x, w), linear64(x, w)["y"], "transposed")
    x3, r1 = normal(g, 3, 5, 64, dtype=dtype), normal(g, 40, dtype=dtype).expand(3, 5, 40)
    hold(linear(x3, w.contiguous(), residual=r1), linear64(x3, w, None, "none", r1)["y"], "three dimensions, one residual row")
    x3.requires_grad_(True)
    got = torch.autograd.grad(linear(x3, w.contiguous(), activation="silu").sum(), x3)[0]
    hold(got, linear64(x3.detach(), w, None, "silu", None, torch.ones(3, 5, 40, dtype=dtype, device=DEV))["dx"], "dy of ones, expanded")
    v = normal(g, 64, dtype=dtype)
    hold(linear(v, w.contiguous()), linear64(v, w)["y"], "a single vector")
    few = normal(g, 1, 64, dtype=dtype).expand(70, 64)
    hold(linear(few, w.contiguous()), linear64(few, w)["y"], "x of one row, expanded")


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_no_rows_and_partial_gradients(dtype):
    from scenerf_amd.linear import linear
    g = gen("none", dtype)
    x, w, b = normal(g, 0, 12, dtype=dtype), normal(g, 9, 12, dtype=dtype), normal(g, 9, dtype=dtype)
    assert linear(x, w, b, activation="gelu").shape == (0, 9)
    x, w, b = (t.requires_grad_(True) for t in (x, w, b))
    dx, dw, db = torch.autograd.grad(linear(x, w, b, activation="gelu").sum(), (x, w, b))
    assert dx.shape == (0, 12) and not dw.any() and not db.any() and dw.shape == (9, 12) and db.shape == (9,)
    x, r = normal(g, 50, 12, dtype=dtype), normal(g, 50, 9, dtype=dtype)
    dy = normal(g, 50, 9, dtype=dtype)
    want = linear64(x, w.detach(), b.detach(), "gelu", r, dy)
    for only, names in (((w,), ["dw"]), ((b,), ["db"]), ((w, b), ["dw", "db"])):
        for t in (w, b):
            t.requires_grad_(any(t is o for o in only))
        for name, got in zip(names, torch.autograd.grad(linear(x, w, b, activation="gelu", residual=r), only, dy)):
            hold(got, want[name], name)
    w.requires_grad_(False), b.requires_grad_(False)
    r.requires_grad_(True)
    hold(torch.autograd.grad(linear(x, w, b, activation="gelu", residual=r), r, dy)[0], want["dr"], "dr alone")


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_values_that_are_not_numbers_stay_in_their_rows(dtype):
    from scenerf_amd.linear import linear
    g = gen("nan", dtype)
    x, w = normal(g, 70, 72, dtype=dtype), normal(g, 40, 72, dtype=dtype)
    x[3, 5], x[66, 0], x[69, 71] = float("nan"), float("inf"), float("-inf")
    r = normal(g, 70, 40, dtype=dtype)
    r[10, 7] = float("nan")
    for act in ACTS:
        y = linear(x, w, activation=act, residual=r)
        bad = torch.zeros(70, 40, dtype=torch.bool, device=DEV)
        bad[3], bad[66], bad[69], bad[10, 7] = True, True, True, True
        assert bool(torch.isfinite(y[~bad]).all()) and bool(torch.isnan(y[3]).all()) and bool(torch.isnan(y[10, 7]))
        ok = [i for i in range(70) if i not in (3, 10, 66, 69)]
        hold(y[ok], linear64(x[ok], w, None, act, r[ok])["y"], act)


@pytest.mark.parametrize("out", TYPES, ids=str)
@pytest.mark.parametrize("m,k,n", SIZES)
def test_8bit(m, k, n, out):
    from scenerf_amd.linear import linear_8bit, quantize_rows
    g = gen("8bit", m, k, n, out)
    q, s = quantize_rows(normal(g, m, k))
    wq, ws = quantize_rows(normal(g, n, k, scale=k ** -0.5))
    b, r = normal(g, n, dtype=out), normal(g, m, n, dtype=out)
    for act in ACTS:
        hold(linear_8bit(q, s, wq, ws, b, activation=act, residual=r, out_dtype=out),
             linear64(q.float(), wq.float(), b, act, r, scales=(s, ws), out_dtype=out)["y"], act)
    hold(linear_8bit(q, s, wq, ws, out_dtype=out), linear64(q.float(), wq.float(), scales=(s, ws), out_dtype=out)["y"], "bare")


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("m,d", [(1, 1), (3, 7), (5, 512), (17, 515), (9, 2480), (4, 4096), (3, 4100), (2, 9000), (3, 4099)])
def test_quantize_rows(m, d, dtype):
    from scenerf_amd.linear import quantize_rows
    g = gen("q", m, d, dtype)
    x = normal(g, m, d, dtype=dtype, scale=3.0)
    x[m - 1] = 0
    q, s = quantize_rows(x)
    scale = (x.double().abs().amax(1) / 448).clamp(min=2.0 ** -126)
    assert bool(((s.double() - scale).abs() <= 2.0 ** -23 * scale).all()) and not q[m - 1].float().any()
    # half a step of e4m3 is 2^-4 of the value, or half its smallest subnormal 2^-9; the quotient is off by 2^-22
    v = x.double() / s.double()[:, None]
    assert bool(((q.double() - v).abs() <= (2.0 ** -4 + 2.0 ** -20) * v.abs() + 2.0 ** -10 * (1 + 2.0 ** -20)).all())
    assert float(q.float().abs().max()) <= 448


def test_quantize_rows_of_values_that_are_not_numbers():
    from scenerf_amd.linear import quantize_rows
    x = torch.ones(4, 600, device=DEV)
    x[1, 599], x[2, 3] = float("nan"), float("-inf")
    x[3] = 1e-44
    q, s = quantize_rows(x)
    assert float(s[0]) == torch.tensor(1.0).div(448).item() and not bool(torch.isfinite(s[1:3]).any())
    assert bool(torch.isnan(q.float() * s[:, None])[1:3].all()) and float(s[3]) == 2.0 ** -126 and not bool(torch.isnan(q[3].float()).any())


def test_another_stream_and_a_replayed_graph():
    """Captured twice, replayed in turn between eager calls: each replay equals the eager result bit for bit."""
    from scenerf_amd.linear import linear
    g = gen("graph")
    sets, graphs = [], []
    for m, k, n in ((300, 128, 64), (1, 2480, 1536)):
        x, w, b = normal(g, m, k, dtype=torch.bfloat16), normal(g, n, k, dtype=torch.bfloat16, scale=k ** -0.5), normal(g, n, dtype=torch.bfloat16)
        x, w, b = (t.requires_grad_(True) for t in (x, w, b))
        dy = normal(g, m, n, dtype=torch.bfloat16)

        def step(x=x, w=w, b=b, dy=dy):
            y = linear(x, w, b, activation="gelu")
            return (y,) + torch.autograd.grad(y, (x, w, b), dy)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            first = step()
        torch.cuda.current_stream().wait_stream(side)
        eager = [t.detach().clone() for t in step()]
        assert all(torch.equal(a.detach(), e) for a, e in zip(first, eager))
        del first
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            out = [t.detach() for t in step()]
        sets.append((x, step, out))
        graphs.append(gr)
    for rep in range(4):
        for (x, step, out), gr in zip(sets, graphs):
            with torch.no_grad():
                x.copy_(normal(g, *x.shape, dtype=x.dtype))
            gr.replay()
        for x, step, out in sets:
            eager = [t.detach() for t in step()]
            torch.cuda.synchronize()
            assert all(torch.equal(a, e) for a, e in zip(out, eager)), rep


def test_rows_past_32_bit_offsets():
    """x and y of more than 2^31 elements: the last rows equal the same rows on their own."""
    from scenerf_amd.linear import linear
    g = gen("large")
    m, k, n = 1_100_000, 2048, 16
    x = torch.empty(m, k, dtype=torch.bfloat16, device=DEV).normal_(generator=g)
    w = normal(g, n, k, dtype=torch.bfloat16, scale=k ** -0.5)
    y = linear(x, w)
    hold(y[-300:], linear64(x[-300:], w)["y"], "last rows")
    del y
    wt = normal(g, 2048, 16, dtype=torch.bfloat16)
    y = linear(x[:, :16], wt, activation="relu")
    hold(y[-300:], linear64(x[-300:, :16], wt, None, "relu")["y"], "last rows of a large result")


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("k", [1, 3, 4, 5, 7, 8, 9, 15, 16, 17, 31, 257, 511, 513, 1023, 1030, 2049])
def test_few_rows_of_any_length(k, dtype):
    """1 to 9 rows whose last 16 bytes overlap the piece in front of them; starts that nothing is aligned to; 8 bits too."""
    from scenerf_amd.linear import linear, linear_8bit, quantize_rows
    g = gen("few", k, dtype)
    for m in (1, 2, 3, 4, 5, 8, 9):
        n = 2 * m + 5
        x, w = normal(g, m, k + 3, dtype=dtype)[:, 1:k + 1], normal(g, n, k + 1, dtype=dtype, scale=k ** -0.5)[:, 1:]
        b, r = normal(g, n, dtype=dtype), normal(g, m, n, dtype=dtype)
        hold(linear(x, w, b, activation="silu", residual=r), linear64(x, w, b, "silu", r)["y"], "%d rows" % m)
        q, s = quantize_rows(x)
        wq, ws = quantize_rows(w)
        hold(linear_8bit(q, s, wq, ws, b, residual=r, out_dtype=dtype), linear64(q.float(), wq.float(), b, "none", r, scales=(s, ws), out_dtype=dtype)["y"],
             "%d rows in 8 bits" % m)


@pytest.mark.parametrize("k,pitch", [(48, 48), (48, 64), (42, 42)])
def test_saved_tensors_moved_by_hooks(k, pitch):
    """torch.autograd.graph.save_on_cpu hands the backward pass other copies, with another pitch, of what the forward saved."""
    from scenerf_amd.linear import linear
    g = gen("hooks", k, pitch)
    bf = torch.bfloat16
    x, w, b = normal(g, 300, pitch, dtype=bf)[:, :k].requires_grad_(True), normal(g, 130, k, dtype=bf, scale=k ** -0.5).requires_grad_(True), None
    dy = normal(g, 300, 130, dtype=bf)
    want = torch.autograd.grad(linear(x, w, b, activation="gelu"), (x, w), dy)
    with torch.autograd.graph.save_on_cpu():
        y = linear(x, w, b, activation="gelu")
    got = torch.autograd.grad(y, (x, w), dy)
    full = linear64(x.detach(), w.detach(), b, "gelu", None, dy)
    hold(got[0], full["dx"], "dx")
    hold(got[1], full["dw"], "dw")
    assert want[0].shape == got[0].shape


# sizes from which the plan takes each of its tiles, whole and in splits, forward and for both gradients, rows and columns that end inside one
TILES = [(9001, 42, 1541), (9001, 1541, 48), (16385, 4104, 130), (20011, 264, 48), (20011, 42, 263), (1001, 4104, 776), (20011, 199, 520),
         (300, 16392, 520), (300, 2056, 1543), (5003, 16392, 130), (2049, 2056, 520), (1001, 1032, 1544), (33000, 2048, 264)]


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("m,k,n", TILES)
def test_every_tile(m, k, n, dtype):
    from scenerf_amd.linear import linear
    g = gen("tile", m, k, n, dtype)
    x, w, b, r = normal(g, m, k, dtype=dtype), normal(g, n, k, dtype=dtype, scale=k ** -0.5), normal(g, n, dtype=dtype), normal(g, m, n, dtype=dtype)
    dy = normal(g, m, n, dtype=dtype)
    want = linear64(x, w, b, "gelu", r, dy)
    with torch.no_grad():
        hold(linear(x, w, b, activation="gelu", residual=r), want["y"], "y")
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    y = linear(*leaves, activation="gelu", residual=r)
    hold(y.detach(), want["y"], "y")
    for name, got in zip(("dx", "dw", "db"), torch.autograd.grad(y, leaves, dy)):
        hold(got, want[name], name)


@pytest.mark.parametrize("out", TYPES, ids=str)
@pytest.mark.parametrize("m,k,n", [(20011, 42, 263), (300, 16392, 1544), (9001, 42, 1541), (9001, 16392, 130), (20011, 1544, 520), (300, 4104, 48)])
def test_every_tile_in_8_bits(m, k, n, out):
    from scenerf_amd.linear import linear_8bit, quantize_rows
    g = gen("tile8", m, k, n, out)
    q, s = quantize_rows(normal(g, m, k))
    wq, ws = quantize_rows(normal(g, n, k, scale=k ** -0.5))
    b, r = normal(g, n, dtype=out), normal(g, m, n, dtype=out)
    hold(linear_8bit(q, s, wq, ws, b, activation="silu", residual=r, out_dtype=out),
         linear64(q.float(), wq.float(), b, "silu", r, scales=(s, ws), out_dtype=out)["y"])


@pytest.mark.parametrize("k,n", [(2048, 16), (16, 2048)])
def test_gradients_past_32_bit_offsets(k, n):
    """x, dx (or y, z, dy and dz) of more than 2^31 elements; a gradient that reaches the last rows alone, so that their own call is the oracle."""
    from scenerf_amd.linear import linear
    g = gen("large back", k, n)
    m, last, bf = 1_100_000, 300, torch.bfloat16
    x = torch.empty(m, k, dtype=bf, device=DEV).normal_(generator=g).requires_grad_(True)
    w, b = normal(g, n, k, dtype=bf, scale=k ** -0.5).requires_grad_(True), normal(g, n, dtype=bf).requires_grad_(True)
    dy = torch.zeros(m, n, dtype=bf, device=DEV)
    dy[-last:] = normal(g, last, n, dtype=bf)
    dx, dw, db = torch.autograd.grad(linear(x, w, b, activation="silu"), (x, w, b), dy)
    want = linear64(x.detach()[-last:], w.detach(), b.detach(), "silu", None, dy[-last:])
    hold(dx[-last:], want["dx"], "dx")
    hold(dw, want["dw"], "dw")
    hold(db, want["db"], "db")
    assert not bool(dx[:-last].any())


@pytest.mark.parametrize("m", [5, 300])
def test_8bit_rows_and_columns_that_are_not_numbers(m):
    """A row of x, or of w, that quantize_rows could not hold spoils its own row, or column, of the result and no other."""
    from scenerf_amd.linear import linear_8bit, quantize_rows
    g = gen("nan8", m)
    x, w = normal(g, m, 200), normal(g, 70, 200, scale=200 ** -0.5)
    clean = linear_8bit(*quantize_rows(x), *quantize_rows(w), activation="gelu")
    x[m - 2, 3], w[69, 199] = float("inf"), float("nan")
    y = linear_8bit(*quantize_rows(x), *quantize_rows(w), activation="gelu")
    assert not bool(torch.isfinite(y[m - 2]).any()) and not bool(torch.isfinite(y[:, 69]).any())
    keep = [i for i in range(m) if i != m - 2]
    assert torch.equal(y[keep][:, :69], clean[keep][:, :69])


@pytest.mark.parametrize("m,k,n", [(300, 520, 136), (5003, 1032, 130), (20011, 200, 520)])
def test_the_same_bits_every_time(m, k, n):
    from scenerf_amd.linear import linear
    g = gen("bits", m, k, n)
    bf = torch.bfloat16
    x, w, b, dy = (t.requires_grad_(True) for t in (normal(g, m, k, dtype=bf), normal(g, n, k, dtype=bf), normal(g, n, dtype=bf), normal(g, m, n, dtype=bf)))

    def once():
        y = linear(x, w, b, activation="gelu")
        return (y.detach(),) + torch.autograd.grad(y, (x, w, b), dy.detach())
    first = once()
    for _ in range(5):
        assert all(torch.equal(a, c) for a, c in zip(first, once()))


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_rows_far_apart(dtype):
    """A pitch of more than 4 MiB: beyond the tiles' 32-bit offsets."""
    from scenerf_amd.linear import linear
    g = gen("far", dtype)
    big = torch.empty(40, 2_200_000, dtype=dtype, device=DEV)
    x = big[:, 64:168]
    x.copy_(normal(g, 40, 104, dtype=dtype))
    w, b, dy = normal(g, 72, 104, dtype=dtype, scale=0.1).requires_grad_(True), normal(g, 72, dtype=dtype).requires_grad_(True), normal(g, 40, 72, dtype=dtype)
    x.requires_grad_(True)
    y = linear(x, w, b, activation="gelu")
    want = linear64(x.detach(), w.detach(), b.detach(), "gelu", None, dy)
    hold(y.detach(), want["y"], "y")
    for name, t in zip(("dx", "dw", "db"), torch.autograd.grad(y, (x, w, b), dy)):
        hold(t, want[name], name)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("m,k,n", [(1, 3, 5), (9, 42, 515), (200, 1001, 130), (5000, 42, 65)])
def test_the_c_entries_on_rows_as_they_are(m, k, n, dtype):
    """The entries without scenerf_hip_linear_pad's copies: rows of any length and start, element by element."""
    import ctypes as C

    from scenerf_amd import _capi
    g = gen("c", m, k, n, dtype)
    lib = _capi.load()
    code = {torch.float32: _capi.T_F32, torch.bfloat16: _capi.T_BF16, torch.float16: _capi.T_F16}[dtype]
    x, w = normal(g, m, k + 1, dtype=dtype)[:, 1:], normal(g, n, k + 3, dtype=dtype, scale=k ** -0.5)[:, 3:]
    b, r, dy = normal(g, n, dtype=dtype), normal(g, m, n + 1, dtype=dtype)[:, :n], normal(g, m, n + 1, dtype=dtype)[:, 1:]
    y, z, dx, dw, db = (torch.empty(*s, dtype=dtype, device=DEV) for s in ((m, n), (m, n), (m, k), (n, k), (n,)))
    p = _capi.Linear(code, code, _capi.ACTIVATIONS["silu"], n, k, 0, m, x.data_ptr(), x.stride(0), w.data_ptr(), w.stride(0), None, None, b.data_ptr(),
                     r.data_ptr(), r.stride(0), y.data_ptr(), z.data_ptr(), dy.data_ptr(), dy.stride(0), dx.data_ptr(), dw.data_ptr(), db.data_ptr())
    stream = torch.cuda.current_stream().cuda_stream
    for backward, fn in ((0, lib.scenerf_hip_linear_forward), (1, lib.scenerf_hip_linear_backward)):
        need = lib.scenerf_hip_linear_workspace(C.byref(p), backward)
        assert need >= 0
        ws = torch.empty(need + 16, dtype=torch.uint8, device=DEV)
        p.workspace, p.workspace_bytes = ws.data_ptr(), need
        assert fn(C.byref(p), stream) == 0, lib.scenerf_hip_last_error()
    want = linear64(x, w, b, "silu", r, dy)
    for name, t in (("y", y), ("dx", dx), ("dw", dw), ("db", db)):
        hold(t, want[name], name)


def test_threads_on_their_own_streams():
    """Four host threads, each with a stream, a shape and a graph of its own: what each gets is what it gets alone."""
    import threading

    from scenerf_amd.linear import linear, linear_8bit, quantize_rows
    from scenerf_amd.norm import rms_norm
    bf = torch.bfloat16
    shapes = [(300, 520, 136), (5003, 72, 515), (4, 512, 512), (1001, 1032, 264)]

    def work(i, reps, out):
        m, k, n = shapes[i]
        g = gen("threads", i)
        x, w, dy = normal(g, m, k, dtype=bf).requires_grad_(True), normal(g, n, k, dtype=bf, scale=k ** -0.5).requires_grad_(True), normal(g, m, n, dtype=bf)
        gain = torch.ones(k, device=DEV, dtype=bf)
        for _ in range(reps):
            y = linear(rms_norm(x, gain), w, activation="gelu")
            grads = torch.autograd.grad(y, (x, w), dy)
            with torch.no_grad():
                y8 = linear_8bit(*quantize_rows(x), *quantize_rows(w))
            out.append([t.detach().clone() for t in (y, *grads, y8)])
    alone = []
    for i in range(4):
        work(i, 1, alone)
    torch.cuda.synchronize()
    together = [[] for _ in range(4)]

    def run(i):
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            work(i, 10, together[i])
            s.synchronize()
    threads = [threading.Thread(target=run, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for i in range(4):
        assert len(together[i]) == 10
        for got in together[i]:
            assert all(torch.equal(a, b) for a, b in zip(got, alone[i]))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("m,k,n", [(1, 16, 16), (1, 300, 1000), (5, 43, 544), (33, 512, 130), (60, 2480, 130), (300, 12, 512), (4801, 64, 40), (20011, 42, 96), (1, 512, 3)])
def test_few_gradients_are_made_from_the_whole_dz(m, k, n, dtype):
    """Below 32,768 dz (16,384 dx, dw) their rounding to 16 bits is made good by a second operand: the bounds know no rounding of dz."""
    from scenerf_amd.linear import linear
    g = gen("whole dz", m, k, n, dtype)
    leaves = [t.requires_grad_(True) for t in (normal(g, m, k, dtype=dtype), normal(g, n, k, dtype=dtype, scale=k ** -0.5), normal(g, n, dtype=dtype))]
    dy = normal(g, m, n, dtype=dtype)
    for act in ("gelu", "silu"):
        want = linear64(*(t.detach() for t in leaves), act, None, dy, whole_dz=True)
        dx, dw, db = torch.autograd.grad(linear(*leaves, activation=act), leaves, dy)
        hold(db, want["db"], "db")
        if m * n < 32768 or m * k < 16384:
            hold(dx, want["dx"], "dx")
        if m * n < 32768 or n * k < 16384:
            hold(dw, want["dw"], "dw")
    dy[0, 0] = float("inf")
    dx, dw, db = torch.autograd.grad(linear(*leaves, activation="silu"), leaves, dy)
    assert not bool(torch.isfinite(db[0])) and bool(torch.isfinite(db[1:]).all()) and bool(torch.isfinite(dx[1:]).all()) and bool(torch.isfinite(dw[1:]).all())


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_no_rows_through_frozen_parameters(dtype):
    from scenerf_amd.linear import linear
    from scenerf_amd.norm import rms_norm
    g = gen("frozen", dtype)
    w, b = normal(g, 9, 12, dtype=dtype), normal(g, 9, dtype=dtype)
    for act in ACTS:
        x = normal(g, 0, 12, dtype=dtype).requires_grad_(True)
        assert torch.autograd.grad(linear(x, w, b, activation=act).sum(), x)[0].shape == (0, 12)
    x = normal(g, 0, 12, dtype=dtype).requires_grad_(True)
    assert torch.autograd.grad(rms_norm(x, normal(g, 12, dtype=dtype)).sum(), x)[0].shape == (0, 12)


@pytest.mark.parametrize("act", ["relu", "gelu", "silu"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("m,n", [(3, 24), (70, 72), (300, 520), (5, 33)])
def test_sums_past_the_range_of_their_type(m, n, dtype, act):
    """Sums that are finite in 32 bits and not in the operands' type: the activation is at its limit there and so is its slope, 0 or 1."""
    from scenerf_amd.linear import linear
    g = gen("past", m, n, dtype, act)
    k = 16
    x, w, dy = normal(g, m, k, dtype=dtype), normal(g, n, k, dtype=dtype, scale=k ** -0.5), normal(g, m, n, dtype=dtype)
    # three features alone reach the far columns: fp16 256 * 300 = 76,800; bf16 (1 + 127 / 128 + 3 / 512) 2^127, between the largest
    # bf16, (1 + 127 / 128) 2^127, and the largest of 32 bits
    big, weights = (2.0 ** 8, (300.0, 0.0, 0.0)) if dtype == torch.float16 else (2.0 ** 64, (2.0 ** 63, 2.0 ** 63 * 127 / 128, 2.0 ** 63 * 3 / 512))
    x[:, :3], w[:, :3] = big, 0
    low, high = list(range(0, n, 3)), list(range(1, n, 3))
    near = [j for j in range(n) if j % 3 == 2]
    w[low, :], w[high, :] = 0, 0
    for f, v in enumerate(weights):
        w[low, f], w[high, f] = -v, v
    leaves = [t.requires_grad_(True) for t in (x, w)]
    y = linear(x, w, activation=act)
    z = x.detach().double() @ w.detach().double().t()
    top = torch.finfo(dtype).max
    assert bool((z[:, low] < -top).all()) and bool((z[:, high] > top).all()) and float(z.abs().max()) < torch.finfo(torch.float32).max
    assert not bool(y.detach()[:, low].any())
    dx, dw = torch.autograd.grad(y, leaves, dy)
    # the far columns' slopes are 0 and 1 exactly; of dx the products with the three features' weights cancel or overflow: the others are held
    part = linear64(x.detach()[:, 3:], w.detach()[near, 3:], None, act, None, dy[:, near])
    hold(dx[:, 3:], part["dx"], "dx")
    hold(dw[near, 3:], part["dw"], "dw of the near columns")
    assert not bool(dw[low].any())
    far = linear64(x.detach()[:, 3:], w.detach()[high, 3:], None, "none", None, dy[:, high])
    hold(dw[high, 3:], far["dw"], "dw of the columns whose slope is 1")


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("m,d", [(1000, 512), (70, 515), (300, 2480), (40, 2481), (257, 4096), (33, 5000), (9, 4101)])
def test_quantize_rows_to_the_bit(m, d, dtype):
    """q is x / scale rounded once: values of 16 bits lie on e4m3's ties often, where the last bit of the quotient decides."""
    from scenerf_amd.linear import quantize_rows
    g = gen("ties", m, d, dtype)
    x = normal(g, m, d, dtype=dtype)
    q, s = quantize_rows(x)
    x, q, s = x.cpu().float(), q.cpu(), s.cpu()
    assert torch.equal(s, (x.abs().amax(1) / 448).clamp(min=2.0 ** -126))
    want = (x / s[:, None]).to(torch.float8_e4m3fn)
    assert torch.equal(q.view(torch.uint8), want.view(torch.uint8)), int((q.float() != want.float()).sum())


@pytest.mark.parametrize("out", [torch.float32, torch.float16], ids=str)
@pytest.mark.parametrize("m,k,n", [(1, 64, 16), (8, 512, 72), (9, 512, 72), (64, 40, 33), (300, 1024, 520), (5003, 1024, 130), (20011, 264, 48)])
def test_8bit_sums_that_cancel(m, k, n, out):
    """Large products that cancel beside small ones 2^-16 of their size.  Every partial sum, in any order, is a whole number of 2^-6 below 2^17, so
    exact in 32 bits, and the result below 2^4, exact in fp16 too: the same bits whatever number of rows a call has."""
    from scenerf_amd.linear import linear_8bit
    g = gen("cancel", m, k, n)
    small = torch.randint(-1, 2, (m, k), generator=g, device=DEV) * 2.0 ** -6
    sign = 1 - 2 * torch.randint(0, 2, (n, k), generator=g, device=DEV).float()
    at = torch.arange(0, k // 16 * 16, 8, device=DEV)          # one of each 8 neighbours, the next one's of the other sign
    small[:, at] = 256.0
    sign[:, at] = torch.where(at // 8 % 2 == 0, 4.0, -4.0)
    x, w = small.to(torch.float8_e4m3fn), sign.to(torch.float8_e4m3fn)
    assert torch.equal(x.float(), small) and torch.equal(w.float(), sign)
    sx, sw = torch.ones(m, device=DEV), torch.ones(n, device=DEV)
    want = small.double() @ sign.double().t()
    assert float(want.abs().max()) < 16
    got = linear_8bit(x, sx, w, sw, out_dtype=out)
    assert torch.equal(got.double(), want), float((got.double() - want).abs().max())
    alone = linear_8bit(x[m - 1:], sx[:1], w, sw, out_dtype=out)
    assert torch.equal(alone[0], got[m - 1])


@pytest.mark.parametrize("act", ["gelu", "silu"])
@pytest.mark.parametrize("m,k,n", [(4, 24, 40), (300, 64, 136), (5003, 72, 130), (20011, 264, 264)])
def test_fp16_gradients_of_large_dy(m, k, n, act):
    """dy near the type's largest value and a slope above 1: dz is past it, dx and db are not."""
    from scenerf_amd.linear import linear
    g = gen("large dy", m, k, n, act)
    h = torch.float16
    # sums around where the slope is largest: gelu 1.129 at 1.41, silu 1.0998 at 2.4
    x, w, b = normal(g, m, k, dtype=h, scale=0.1), normal(g, n, k, dtype=h, scale=0.01), torch.full((n,), 1.41 if act == "gelu" else 2.4, dtype=h, device=DEV)
    dy = torch.zeros(m, n, dtype=h, device=DEV)
    rows = torch.arange(m, device=DEV)
    dy[rows, rows % n] = torch.where(rows % 2 == 0, 65000.0, -64000.0).to(h)       # one a row
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    dx, dw, db = torch.autograd.grad(linear(*leaves, activation=act), leaves, dy)
    want = linear64(*(t.detach() for t in leaves), act, None, dy)
    assert float((dy.double() * 1.09).abs().max()) > 65504 * 1.05
    for name, got in (("dx", dx), ("dw", dw), ("db", db)):
        hold(got, want[name], name)
    assert bool(torch.isfinite(dx).all())


@pytest.mark.parametrize("act", ["gelu", "silu"])
@pytest.mark.parametrize("m,k,n", [(300, 64, 136), (5003, 72, 130), (20011, 264, 264), (9001, 42, 1541)])
def test_fp16_gradients_of_small_dy(m, k, n, act):
    """dy around 2^-18, 60 times the smallest fp16: dz in fp16 itself would keep five bits.  Roundings are independent and add in squares: of dz, of z
    in the slope and of the results together they are less than two half steps in the 2-norm."""
    from scenerf_amd.linear import linear
    g = gen("small dy", m, k, n, act)
    h = torch.float16
    # (w large, so that dx is not small itself; x small, so that z is of size 1)
    x, w, b = normal(g, m, k, dtype=h, scale=2.0 ** -10), normal(g, n, k, dtype=h, scale=2.0 ** 9 * k ** -0.5), normal(g, n, dtype=h)
    x[:, 0] = 0
    x[:, 0] += 1
    w[:, 0] = 0
    dy = (normal(g, m, n) * 2.0 ** -18).to(h)
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    dx, dw, db = torch.autograd.grad(linear(*leaves, activation=act), leaves, dy)
    want = linear64(*(t.detach() for t in leaves), act, None, dy)
    assert float(want["dx"][0][:, 1:].abs().mean()) > 2.0 ** -13
    for name, got, v in (("dx", dx[:, 1:], want["dx"][0][:, 1:]), ("dw", dw[:, 0], want["dw"][0][:, 0])):
        rounded = v.to(h).double()
        lim = 2 * 2.0 ** -11 * float(v.norm()) + float((rounded - v).norm())
        assert float((got.double() - v).norm()) <= lim, (name, float((got.double() - v).norm()) / float(v.norm()))


@pytest.mark.parametrize("m,k,n", [(40, 72, 24), (5003, 72, 520)])
def test_an_fp16_step_replays_with_dy_of_any_size(m, k, n):
    """The power of two that dz is held by is found anew in every replay: dy of sizes 2^-18 to 2^14 in turn, each replay equal to the eager step."""
    from scenerf_amd.linear import linear
    g = gen("fp16 graph", m, k, n)
    h = torch.float16
    x, w, b = (t.requires_grad_(True) for t in (normal(g, m, k, dtype=h), normal(g, n, k, dtype=h, scale=k ** -0.5), normal(g, n, dtype=h)))
    dy = normal(g, m, n, dtype=h)

    def step():
        return torch.autograd.grad(linear(x, w, b, activation="silu"), (x, w, b), dy)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        out = [t.detach() for t in step()]
    for size in (-18, 0, 13, -10, 14):
        dy.copy_((normal(g, m, n) * 2.0 ** size).clamp(-65504, 65504).to(h))
        gr.replay()
        eager = [t.detach() for t in step()]
        torch.cuda.synchronize()
        assert all(torch.equal(a, e) if bool(torch.isfinite(e).all()) else torch.equal(a.nan_to_num(), e.nan_to_num()) for a, e in zip(out, eager)), size
    dy.zero_()
    gr.replay()
    assert all(not bool(t.any()) for t in out)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("m,k,n", TILES)
def test_every_tile_on_whole_numbers(m, k, n, dtype):
    """Sums that are exact in 32 bits, so that one product too few, or one twice, at the end of a tile, a split or a strip changes the result."""
    from scenerf_amd.linear import linear
    g = gen("whole tiles", m, k, n, dtype)
    x, w, dy = whole(g, m, k, dtype=dtype), whole(g, n, k, dtype=dtype), whole(g, m, n, dtype=dtype)
    b = whole(g, n, dtype=dtype) + 0.5
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    z = x.detach().double() @ w.detach().double().t() + b.detach().double()
    for act in ("none", "relu"):
        on = (z > 0).double() if act == "relu" else torch.ones_like(z)
        dz = dy.double() * on
        want = {"y": z * on, "dx": dz @ w.detach().double(), "dw": dz.t() @ x.detach().double(), "db": dz.sum(0)}
        y = linear(*leaves, activation=act)
        for name, got in zip(("y", "dx", "dw", "db"), (y.detach(),) + torch.autograd.grad(y, leaves, dy)):
            assert float(want[name].abs().max()) < 2 ** 22
            assert torch.equal(got, want[name].float().to(dtype)), (act, name, int((got.double() != want[name].float().to(dtype).double()).sum()))


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("m,k,n", TILES)
def test_every_tile_on_a_dy_of_few_rows(m, k, n, dtype):
    """dy is not 0 in the last rows and around every 256th alone: a row of these that a split or strip drops is most of a sum, not one of thousands."""
    from scenerf_amd.linear import linear
    g = gen("few dy", m, k, n, dtype)
    x, w, dy = whole(g, m, k, dtype=dtype), whole(g, n, k, dtype=dtype), torch.zeros(m, n, dtype=dtype, device=DEV)
    rows = torch.tensor(sorted({r for c in range(0, m + 256, 256) for r in (c - 1, c) if 0 <= r < m} | set(range(max(0, m - 9), m))), device=DEV)
    dy[rows] = whole(g, len(rows), n, dtype=dtype)
    leaves = [t.requires_grad_(True) for t in (x, w)]
    dx, dw = torch.autograd.grad(linear(*leaves), leaves, dy)
    assert torch.equal(dx, (dy.double() @ w.detach().double()).float().to(dtype))
    assert torch.equal(dw, (dy[rows].double().t() @ x.detach()[rows].double()).float().to(dtype))


@pytest.mark.parametrize("out", TYPES, ids=str)
@pytest.mark.parametrize("m,k,n", [(20011, 42, 263), (300, 16392, 1544), (9001, 42, 1541), (9001, 16392, 130), (20011, 1544, 520), (300, 4104, 48), (5, 2480, 96)])
def test_every_tile_in_8_bits_on_whole_numbers(m, k, n, out):
    from scenerf_amd.linear import linear_8bit
    g = gen("whole 8", m, k, n)
    x, w = whole(g, m, k, dtype=torch.float32), whole(g, n, k, dtype=torch.float32)
    x[:, k - 17:], w[:, k - 17:] = 2, 2         # (the end of the contraction weighs most)
    got = linear_8bit(x.to(torch.float8_e4m3fn), torch.ones(m, device=DEV), w.to(torch.float8_e4m3fn), torch.ones(n, device=DEV), out_dtype=out)
    assert torch.equal(got, (x.double() @ w.double().t()).float().to(out))


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("m,k,n", [(0, 24, 40), (1, 16, 16), (40, 72, 24), (300, 42, 515), (1001, 1032, 264), (20011, 264, 48), (9001, 42, 1541), (2049, 2056, 520)])
def test_weight_gradients_as_they_are_summed(m, k, n, dtype):
    """``sums``: dweight and dbias in fp32.  Whole numbers: exact, where 16 bits would round them; otherwise 32-bit sums' bounds, and the rounded ones'
    own bits."""
    from scenerf_amd import _capi
    from scenerf_amd.linear import linear_step, linear_step_back
    g = gen("sums", m, k, n, dtype)

    def back(x, w, b, dy, act, sums):
        y, saved = linear_step(x, w, b, None, _capi.ACTIVATIONS[act], (m, n), act != "none")
        return linear_step_back(saved, dy, (m, k), True, True, True, sums=sums)
    x, w, dy, b = whole(g, m, k, dtype=dtype), whole(g, n, k, dtype=dtype), whole(g, m, n, dtype=dtype), whole(g, n, dtype=dtype) + 0.5
    on = (x.double() @ w.double().t() + b.double() > 0).double()
    for act, dz in (("none", dy.double()), ("relu", dy.double() * on)):
        dx, dw, db = back(x, w, b, dy, act, True)
        assert dx.dtype == dtype and dw.dtype == db.dtype == torch.float32
        assert torch.equal(dw.double(), dz.t() @ x.double()) and torch.equal(db.double(), dz.sum(0))
        assert torch.equal(dx, (dz @ w.double()).float().to(dtype))
    x, w, b, dy = normal(g, m, k, dtype=dtype), normal(g, n, k, dtype=dtype, scale=k ** -0.5), normal(g, n, dtype=dtype), normal(g, m, n, dtype=dtype)
    for act in ("gelu", "silu"):
        dx, dw, db = back(x, w, b, dy, act, True)
        rounded = back(x, w, b, dy, act, False)
        assert torch.equal(dx, rounded[0]) and torch.equal(dw.to(dtype), rounded[1]) and torch.equal(db.to(dtype), rounded[2])
        if m:
            want = linear64(x, w, b, act, None, dy)
            hold(dw, want["dw"], act + " dw")
            hold(db, want["db"], act + " db")


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("act", ["relu", "gelu", "silu"])
def test_slopes_of_kept_values_that_are_not_finite(dtype, act):
    """The step back from a z of infinities, NaN and the type's ends: 0 and 1 at the infinities, NaN at NaN, and no other column knows."""
    from scenerf_amd import _capi
    from scenerf_amd.linear import linear_step_back
    g = gen("slopes", dtype, act)
    m, k, n = 40, 24, 16
    x, w, dy = normal(g, m, k, dtype=dtype), normal(g, n, k, dtype=dtype), normal(g, m, n, dtype=dtype)
    z = normal(g, m, n, dtype=dtype)
    top = torch.finfo(dtype).max
    for j, v in enumerate((float("inf"), float("-inf"), top, -top, float("nan"))):
        z[:, j] = v
    dx, dw, db = linear_step_back((x, w, z, m, n, k, k, 0, _capi.ACTIVATIONS[act]), dy, (m, k), True, True, True)
    ones = linear64(x, w[[0, 2]], torch.zeros(2, dtype=dtype, device=DEV), "none", None, dy[:, [0, 2]])
    hold(dw[[0, 2]], ones["dw"], "slope 1")
    hold(db[[0, 2]], ones["db"], "slope 1")
    assert not bool(dw[[1, 3]].any()) and not bool(db[[1, 3]].any())
    if act == "relu":                                # (a comparison: NaN is not above 0)
        assert not bool(dw[4].any()) and bool(torch.isfinite(dx).all())
    else:
        assert bool(torch.isnan(dw[4]).all()) and bool(torch.isnan(db[4])) and bool(torch.isnan(dx).all())
    assert bool(torch.isfinite(dw[5:]).all()) and bool(torch.isfinite(db[5:]).all())


@pytest.mark.parametrize("m,d", [(40, 512), (9, 4101), (300, 515)])
def test_quantize_rows_of_any_size_to_the_bit(m, d):
    """Rows from the smallest fp32 numbers to the largest, each row of one size."""
    from scenerf_amd.linear import quantize_rows
    g = gen("sizes", m, d)
    x = normal(g, m, d) * torch.exp2(torch.linspace(-140, 120, m, device=DEV))[:, None]
    q, s = quantize_rows(x)
    x, q, s = x.cpu(), q.cpu(), s.cpu()
    assert torch.equal(s, (x.abs().amax(1) / 448).clamp(min=2.0 ** -126))
    want = (x / s[:, None]).to(torch.float8_e4m3fn)
    assert torch.equal(q.view(torch.uint8), want.view(torch.uint8)), int((q.float() != want.float()).sum())


@pytest.mark.parametrize("act", ["gelu", "silu"])
def test_fp32_activations_to_the_last_bits(act):
    """One feature times 1: z is x itself, and what is left is the activation's own error.  In the 2-norm over normal z: no more than 1.25 times what
    32 bits with a correctly rounded erf and exp come to, and twice that in the slope, whose value and density both carry the exponential's."""
    from scenerf_amd.linear import linear
    g = gen("last bits", act)
    x = normal(g, 200000, 1).requires_grad_(True)
    w = torch.ones(16, 1, device=DEV)
    dy = torch.zeros(200000, 16, device=DEV)
    dy[:, 3] = 1
    y = linear(x, w, activation=act)
    dx, = torch.autograd.grad(y, x, dy)

    def formulas(z, erf, exp):
        if act == "gelu":
            c = 0.5 * (1 + erf(z * 0.5 ** 0.5))
            return z * c, c + z * exp(-0.5 * z * z) / (2 * torch.pi) ** 0.5
        p = 1 / (1 + exp(-z))
        return z * p, p * (1 + z * (1 - p))
    z = x.detach()
    want = formulas(z.double(), torch.erf, torch.exp)
    # erf and exp correctly rounded to 32 bits, every operation in 32 bits
    plain = formulas(z, lambda v: torch.erf(v.double()).float(), lambda v: torch.exp(v.double()).float())
    for got, ours, exact, factor in ((y.detach()[:, :1], plain[0], want[0], 1.25), (dx, plain[1], want[1], 2.0)):
        limit = factor * float((ours.double() - exact).norm())
        assert float((got.double() - exact).norm()) <= limit, (factor * float((got.double() - exact).norm()) / limit)
    assert torch.equal(y.detach(), y.detach()[:, :1].expand(-1, 16))
