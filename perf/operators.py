"""What the row operators of a ResnetFC cost: the linear layer with its epilogue, its 8-bit form, the RMS norm and rows in 8 bits.

``own`` false: the operators' plain form in elementary torch operations; true: the framework's entry points (scenerf_amd.linear,
scenerf_amd.norm).  Rows are samples: 1,200 rays x 128 samples = 153,600 in a training render, 1,200 x 4 = 4,800 in the gaussian head,
4,096 x 64 = 262,144 in the 1 x 128 net; widths are the ResnetFC's (d_in 42, d_hidden 128 and 512, d_latent 2,480, three lin_z side by
side 1,536)."""
import math

import torch

own = False

TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
SIZE = {"float32": 4, "bfloat16": 2, "float16": 2}
E4M3_MAX = 448.0
SCALE_MIN = 2.0 ** -126
EPS = 1e-6
DEVICE = "cuda"


def listed():
    lin = {"op": "linear", "train": False, "activation": "none", "bias": True, "residual": False, "sliced": False}
    low = {"op": "linear_8bit", "activation": "none", "bias": True, "residual": False, "dtype": "bfloat16"}
    nrm = {"op": "rms_norm", "train": True, "residual": True, "sliced": False}
    return [
        # one sample's latent vector through the three lin_z at once: the call's own latency, and the weights read once
        dict(lin, name="linear one row", dtype="bfloat16", rows=1, k=2480, n=1536),
        # the same product for every sample of a training render: the largest one of the net
        dict(lin, name="linear lin_z", dtype="bfloat16", rows=153600, k=2480, n=1536),
        # a training step through a hidden layer of the radiance net, with the residual stream added
        dict(lin, name="linear train hidden", dtype="bfloat16", rows=153600, k=512, n=512, train=True, activation="gelu", residual=True),
        # a training step through an input layer: 42 features (rows of 84 bytes), an odd number of rows and of outputs
        dict(lin, name="linear train ragged", dtype="float16", rows=4801, k=42, n=515, train=True, activation="silu"),
        # the narrow net trained in full precision
        dict(lin, name="linear train float32", dtype="float32", rows=262144, k=128, n=128, train=True, activation="silu", residual=True),
        # one sample through a hidden layer in 8 bits
        dict(low, name="linear_8bit one row", rows=1, k=512, n=512, activation="gelu", residual=True),
        # a frame's chunk of samples through the lin_z in 8 bits
        dict(low, name="linear_8bit lin_z", rows=153600, k=2480, n=1536),
        # the normalisation in front of each block of a training render
        dict(nrm, name="rms_norm train", dtype="bfloat16", rows=153600, width=512),
        # the gaussian head's rows of a net of odd width, out of a wider tensor, in full precision
        dict(nrm, name="rms_norm ragged", dtype="float32", rows=4801, width=515, train=False, sliced=True),
        # one sample on its way to an 8-bit layer
        {"name": "rms_norm_8bit one row", "op": "rms_norm_8bit", "dtype": "bfloat16", "rows": 1, "width": 512, "residual": True, "sliced": False},
        # a chunk of samples on its way to an 8-bit layer
        {"name": "rms_norm_8bit", "op": "rms_norm_8bit", "dtype": "bfloat16", "rows": 153600, "width": 512, "residual": True, "sliced": False},
        # gathered features to 8 bits, half precision, an odd number of rows
        {"name": "quantize_rows", "op": "quantize_rows", "dtype": "float16", "rows": 40001, "width": 2480, "sliced": False},
    ]


def _spread(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["linear", "linear", "linear", "linear_8bit", "rms_norm", "rms_norm", "rms_norm_8bit", "quantize_rows"])
    dtype = rng.choice(["bfloat16", "bfloat16", "float16", "float32"])
    rows = rng.choice([1, _spread(rng, 1, 64), _spread(rng, 1, 153600), _spread(rng, 4096, 153600)])
    most = max(c["rows"] * c["k"] * c["n"] for c in listed() if "k" in c)
    if op in ("linear", "linear_8bit"):
        # widths of nets of 16 to 2,048, the odd ones of inputs and outputs among them
        k, n = (rng.choice([16 * _spread(rng, 1, 128), _spread(rng, 1, 2560)]) for _ in range(2))
        case = {"op": op, "activation": rng.choice(["none", "relu", "gelu", "silu"]), "bias": rng.random() < 0.8,
                "residual": rng.random() < 0.5, "dtype": dtype if op == "linear" else rng.choice(["bfloat16", "float16", "float32"])}
        if op == "linear":
            case["train"], case["sliced"] = rng.random() < 0.5, rng.random() < 0.3
            if case["train"] and case["activation"] == "relu":
                # a step through relu jumps at 0, where a sum's last bit decides: such steps are held to exact sums in the tests
                case["activation"] = "gelu"
        share = 1 if op == "linear_8bit" else (3 if case["train"] else 1) * (12 if dtype == "float32" else 1)
        return dict(case, rows=max(1, min(rows, most // (share * k * n))), k=k, n=n)
    width = rng.choice([16 * _spread(rng, 1, 256), _spread(rng, 1, 4096)])
    rows = max(1, min(rows, 153600 * 1024 // width))
    case = {"op": op, "dtype": dtype, "rows": rows, "width": width, "sliced": rng.random() < 0.4}
    if op != "quantize_rows":
        case["residual"] = rng.random() < 0.6
    if op == "rms_norm":
        case["train"] = rng.random() < 0.6
    return case


def _normal(g, rows, cols, dtype, sliced=False, scale=1.0):
    """Normal values; ``sliced``: columns of a wider tensor, as the blocks' parts of one lin_z product are."""
    t = torch.randn(rows, cols + 24 if sliced else cols, generator=g, device=DEVICE, dtype=torch.float32).mul_(scale).to(dtype)
    return t[:, 8:8 + cols] if sliced else t


def _to_8bit(t):
    scale = (t.abs().amax(1, keepdim=True) / E4M3_MAX).clamp(min=SCALE_MIN)
    return (t / scale).to(torch.float8_e4m3fn), scale.squeeze(1)


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    s, dt, rows = {"case": case}, TYPES[case["dtype"]], case["rows"]
    if case["op"] in ("linear", "linear_8bit"):
        k, n = case["k"], case["n"]
        s["bias"] = torch.randn(n, generator=g, device=DEVICE).mul_(0.1).to(dt) if case["bias"] else None
        s["residual"] = _normal(g, rows, n, dt, case.get("sliced", False)) if case["residual"] else None
        if case["op"] == "linear_8bit":
            s["x"], s["x_scale"] = _to_8bit(_normal(g, rows, k, torch.float32))
            s["weight"], s["weight_scale"] = _to_8bit(_normal(g, n, k, torch.float32, scale=math.sqrt(2.0 / k)))
            return s
        s["x"] = _normal(g, rows, k, dt, case["sliced"])
        s["weight"] = _normal(g, n, k, dt, scale=math.sqrt(2.0 / k))
        if case["train"]:
            s["dy"] = _normal(g, rows, n, dt)
    else:
        d = case["width"]
        # a residual stream: rows of different sizes
        size = torch.exp(0.5 * torch.randn(rows, 1, generator=g, device=DEVICE))
        s["x"] = _normal(g, rows, d + 24 if case["sliced"] else d, torch.float32).mul_(size).to(dt)
        s["x"] = s["x"][:, 8:8 + d] if case["sliced"] else s["x"]
        if case["op"] == "quantize_rows":
            return s
        s["residual"] = _normal(g, rows, d, dt) if case["residual"] else None
        s["weight"] = (1.0 + 0.1 * torch.randn(d, generator=g, device=DEVICE)).to(dt)
        if case.get("train"):
            s["dy"] = _normal(g, rows, d, dt)
            s["dh"] = _normal(g, rows, d, dt) if case["residual"] else None
    if case.get("train"):
        for name in ("x", "weight", "bias", "residual"):
            if s.get(name) is not None:
                s[name] = s[name].detach().requires_grad_(True)
    return s


def _act(z, name):
    if name == "relu":
        return z.clamp(min=0)
    if name == "gelu":
        return 0.5 * z * (1 + torch.erf(z * math.sqrt(0.5)))
    if name == "silu":
        return z / (1 + torch.exp(-z))
    return z


def _slope(z, name):
    if name == "relu":
        return (z > 0).to(z.dtype)
    if name == "gelu":
        return 0.5 * (1 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    if name == "silu":
        p = 1 / (1 + torch.exp(-z))
        return p * (1 + z * (1 - p))
    return torch.ones_like(z)


def _plain_linear(s):
    c, dt = s["case"], TYPES[s["case"]["dtype"]]
    x, w = s["x"].float(), s["weight"].float()
    z = torch.mm(x, w.t())
    if c["op"] == "linear_8bit":
        z = z * s["x_scale"][:, None] * s["weight_scale"][None, :]
    if s["bias"] is not None:
        z = z + s["bias"].float()
    y = _act(z, c["activation"])
    if s["residual"] is not None:
        y = y + s["residual"].float()
    out = {"y": y.to(dt)}
    if c.get("train"):
        dz = s["dy"].float()
        if c["activation"] != "none":
            dz = dz * _slope(z, c["activation"])
        out["dx"], out["dweight"] = torch.mm(dz, w).to(dt), torch.mm(dz.t(), x).to(dt)
        if s["bias"] is not None:
            out["dbias"] = dz.sum(0).to(dt)
        if s["residual"] is not None:
            out["dresidual"] = s["dy"]
    return out


def _plain_rows(s):
    c, dt = s["case"], TYPES[s["case"]["dtype"]]
    h, out = s["x"].float(), {}
    if c["op"] != "quantize_rows":
        if s["residual"] is not None:
            h = h + s["residual"].float()
            out["h"] = h.to(dt)
        rstd = 1 / torch.sqrt((h * h).mean(1, keepdim=True) + EPS)
        w = s["weight"].float()
        xhat = h * rstd
        y = xhat * w
    else:
        y = h
    if c["op"] != "rms_norm":
        scale = (y.abs().amax(1) / E4M3_MAX).clamp(min=SCALE_MIN)
        out["q"], out["scale"] = (y / scale[:, None]).to(torch.float8_e4m3fn), scale
        return out
    out["y"] = y.to(dt)
    if c["train"]:
        dy = s["dy"].float()
        dyw = dy * w
        dh = (dyw - xhat * (dyw * xhat).mean(1, keepdim=True)) * rstd
        if s["residual"] is not None:
            dh = dh + s["dh"].float()
        out["dx"], out["dweight"] = dh.to(dt), (dy * xhat).sum(0).to(dt)
        if s["residual"] is not None:
            out["dresidual"] = out["dx"]
    return out


def _own(s):
    from scenerf_amd.linear import linear, linear_8bit, quantize_rows
    from scenerf_amd.norm import rms_norm, rms_norm_8bit
    c, r = s["case"], s.get("residual")
    if c["op"] == "quantize_rows":
        q, scale = quantize_rows(s["x"])
        return {"q": q, "scale": scale}
    if c["op"] == "rms_norm_8bit":
        got = rms_norm_8bit(s["x"], s["weight"], residual=r, eps=EPS)
        return dict(zip(("q", "scale", "h"), got))
    if c["op"] == "linear_8bit":
        return {"y": linear_8bit(s["x"], s["x_scale"], s["weight"], s["weight_scale"], s["bias"], activation=c["activation"], residual=r,
                                 out_dtype=TYPES[c["dtype"]])}
    if c["op"] == "linear":
        out = {"y": linear(s["x"], s["weight"], s["bias"], activation=c["activation"], residual=r)}
        ends, grads = [out["y"]], [s.get("dy")]
    else:
        got = rms_norm(s["x"], s["weight"], residual=r, eps=EPS)
        out = {"y": got} if r is None else {"y": got[0], "h": got[1]}
        ends, grads = ([got], [s.get("dy")]) if r is None else (list(got), [s.get("dy"), s.get("dh")])
    if c["train"]:
        names = [n for n in ("x", "weight", "bias", "residual") if s.get(n) is not None]
        out.update(zip(["d" + n for n in names], torch.autograd.grad(ends, [s[n] for n in names], grads)))
        out = {n: v.detach() for n, v in out.items()}
    return out


def run(state):
    if own:
        return _own(state)
    with torch.no_grad():
        return _plain_linear(state) if "k" in state["case"] else _plain_rows(state)


def work(case):
    rows = case["rows"]
    if "k" in case:
        k, n, es = case["k"], case["n"], SIZE[case["dtype"]]
        xs = 1 if case["op"] == "linear_8bit" else es
        moved = xs * (rows * k + n * k) + es * rows * n * (2 if case["residual"] else 1) + (es * n if case["bias"] else 0)
        if case["op"] == "linear_8bit":
            moved += 4 * (rows + n)
        if not case.get("train"):
            return {"bytes": moved, "flops": 2 * rows * k * n}
        # the step back: dy in; dx, dweight, dbias out
        return {"bytes": moved + es * (rows * n + rows * k + n * k + (n if case["bias"] else 0)), "flops": 6 * rows * k * n}
    d, es = case["width"], SIZE[case["dtype"]]
    if case["op"] == "quantize_rows":
        return {"bytes": rows * (d * (es + 1) + 4), "flops": 3 * rows * d}
    moved = es * rows * d * (3 if case["residual"] else 1) + es * d
    if case["op"] == "rms_norm_8bit":
        return {"bytes": moved + rows * (d + 4), "flops": 7 * rows * d}
    moved += es * rows * d
    if not case["train"]:
        return {"bytes": moved, "flops": 5 * rows * d}
    return {"bytes": moved + es * rows * d * (3 if case["residual"] else 2) + es * d, "flops": 16 * rows * d}


def exact(case, seed):
    """The definition in 64 bits, the gradients by torch's own differentiation of it."""
    s = prepare(case, seed)
    wide = {n: v.detach().double() for n, v in s.items() if torch.is_tensor(v)}
    leaves = [n for n in ("x", "weight", "bias", "residual") if n in wide] if case.get("train") else []
    for n in leaves:
        wide[n].requires_grad_(True)
    out = {}
    if "k" in case:
        x, w = wide["x"], wide["weight"]
        if case["op"] == "linear_8bit":
            x, w = x * wide["x_scale"].unsqueeze(1), w * wide["weight_scale"].unsqueeze(1)
        z = torch.nn.functional.linear(x, w, wide.get("bias"))
        y = {"none": lambda t: t, "relu": torch.relu, "gelu": torch.nn.functional.gelu, "silu": torch.nn.functional.silu}[case["activation"]](z)
        out["y"] = y + wide["residual"] if "residual" in wide else y
        ends = {"y": "dy"}
    else:
        h, ends = wide["x"], {"y": "dy"}
        if "residual" in wide:
            h = h + wide["residual"]
            out["h"] = h
            ends["h"] = "dh"
        y = h
        if case["op"] != "quantize_rows":
            y = h / torch.sqrt(h.pow(2).mean(dim=1, keepdim=True) + EPS) * wide["weight"]
        if case["op"] == "rms_norm":
            out["y"] = y
        else:
            scale = torch.clamp(y.abs().max(dim=1).values / E4M3_MAX, min=SCALE_MIN)
            out["q"], out["scale"] = y / scale.unsqueeze(1), scale
    if leaves:
        grads = torch.autograd.grad([out[e] for e in ends], [wide[n] for n in leaves], [wide[g] for g in ends.values()])
        out.update(zip(["d" + n for n in leaves], grads))
    return {n: v.detach() for n, v in out.items()}
