"""Measured cases of the normalisation and weight-update operators.

* LayerNorm over the last axis, forward and backward (``yl_layernorm_fwd``,
  ``yl_layernorm_bwd``): the rows of a Linear's input, or the channels of every
  pixel of an NHWC activation.
* Newton-Schulz orthogonalisation of matrices (``yl_newton_schulz``).
* One Muon step over a table of weight matrices (``yl_muon_multi``).

``run`` computes a case in plain torch operations, or, where ``own`` is true,
through the library's C entry points on the same device buffers.
"""
import ctypes
import math

import torch

own = False

NS_COEFFS = (3.4445, -4.7750, 2.0315)
NS_STEPS = 5
NS_EPS = 1e-7
LN_EPS = 1e-5
MUON = {"lr": 0.02, "momentum": 0.95, "weight_decay": 0.01}

# The motion U-Net's hidden weights (levels 128 / 256 / 384, time MLP 512) as
# matrices of oc rows and k*k*ic columns.
UNET = (
    "512x128,512x512,4*128x512,4*256x512,2*384x512,"
    "8*128x1152,256x1152,6*256x2304,256x128,384x2304,3*384x3456,384x256,"
    "256x3456,256x4608,256x512,2*128x2304,128x256"
)
# Four transformer blocks of width 1024: q, k, v, o and a feed-forward pair.
BLOCKS = "16*1024x1024,4*4096x1024,4*1024x4096"


def _shapes(text):
    out = []
    for part in text.split(","):
        times, _, shape = part.rpartition("*")
        r, c = shape.split("x")
        out += [(int(r), int(c))] * int(times or 1)
    return out


def listed():
    return [
        # the time MLP's hidden rows at a batch of 32: latency of one small call
        {"name": "ln_fwd_time_mlp", "op": "ln_fwd", "rows": 32, "cols": 512, "pad": 0},
        # odd rows inside a wider buffer
        {"name": "ln_fwd_ragged", "op": "ln_fwd", "rows": 4097, "cols": 1021, "pad": 6},
        # the 128 channels of every pixel of eight 480x856 frames, NHWC
        {"name": "ln_fwd_frames", "op": "ln_fwd", "rows": 8 * 480 * 856, "cols": 128, "pad": 0},
        # the time MLP's backward: latency
        {"name": "ln_bwd_time_mlp", "op": "ln_bwd", "rows": 32, "cols": 512, "pad": 0,
         "addend": False},
        # the 256 channels of eight 60x107 latents, with the residual's gradient added
        {"name": "ln_bwd_latents", "op": "ln_bwd", "rows": 8 * 60 * 107, "cols": 256, "pad": 0,
         "addend": True},
        # long rows of a large batch of tokens
        {"name": "ln_bwd_tokens", "op": "ln_bwd", "rows": 16384, "cols": 4096, "pad": 0,
         "addend": True},
        # one 3x3 128 -> 128 conv weight: latency of the whole iteration
        {"name": "ns_conv_128", "op": "ns", "shapes": "128x1152"},
        # odd wide, tall and nearly square matrices in one call
        {"name": "ns_ragged", "op": "ns", "shapes": "257x1531,1531x129,997x1001,3x36,640x1"},
        # one large square matrix: the matrix products' rate
        {"name": "ns_square_4096", "op": "ns", "shapes": "4096x4096"},
        # the time MLP's two weights
        {"name": "muon_time_mlp", "op": "muon", "shapes": "512x128,512x512", "nesterov": True},
        # every hidden weight of the motion U-Net
        {"name": "muon_unet", "op": "muon", "shapes": UNET, "nesterov": True},
        # four transformer blocks of width 1024
        {"name": "muon_blocks", "op": "muon", "shapes": BLOCKS, "nesterov": True},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["ln_fwd", "ln_bwd", "ns", "muon"])
    if op in ("ln_fwd", "ln_bwd"):
        cols = _log(rng, 1, 16384)
        rows = _log(rng, 1, max(1, min(3_000_000, (1 << 26) // cols)))
        case = {"op": op, "rows": rows, "cols": cols, "pad": rng.choice([0, 0, 1, 4, 12])}
        if op == "ln_bwd":
            case["addend"] = rng.random() < 0.5
        return case
    shapes = []
    for _ in range(rng.choice([1, 1, 2, 3, 6])):
        r = _log(rng, 1, 4096)
        c = _log(rng, 1, max(1, min(8192, (1 << 22) // r)))
        shapes.append("%dx%d" % (r, c))
    case = {"op": op, "shapes": ",".join(shapes)}
    if op == "muon":
        case["nesterov"] = rng.random() < 0.7
    return case


def _device():
    return torch.device("cuda", torch.cuda.current_device())


def _padded(gen, rows, cols, pad, scale=1.0):
    """rows x cols values inside a buffer of cols + pad columns."""
    buf = torch.randn(rows, cols + pad, generator=gen, device=_device())
    return buf.mul_(scale)[:, :cols]


def _update(gen, rows, cols):
    """A weight's gradient: a few strong directions in noise of the same energy."""
    rank = min(4, rows, cols)
    u = torch.randn(rows, rank, generator=gen, device=_device())
    v = torch.randn(rank, cols, generator=gen, device=_device())
    noise = torch.randn(rows, cols, generator=gen, device=_device())
    return (noise + (u @ v) / math.sqrt(rank)).mul_(0.01)


def _joined(parts):
    """One flat buffer with the parts' values, and the parts as views of it."""
    flat = torch.cat([t.reshape(-1) for t in parts])
    views = flat.split([t.numel() for t in parts])
    return flat, [v.view(t.shape) for v, t in zip(views, parts)]


def prepare(case, seed):
    gen = torch.Generator(device=_device()).manual_seed(seed)
    op = case["op"]
    if op in ("ln_fwd", "ln_bwd"):
        rows, cols, pad = case["rows"], case["cols"], case["pad"]
        x = _padded(gen, rows, cols, pad, 1.5).add_(0.3)
        s = {"op": op, "x": x,
             "gamma": torch.randn(cols, generator=gen, device=_device()).mul_(0.1).add_(1.0)}
        if op == "ln_fwd":
            s["beta"] = torch.randn(cols, generator=gen, device=_device()).mul_(0.1)
            return s
        s["dy"] = _padded(gen, rows, cols, pad)
        s["addend"] = _padded(gen, rows, cols, pad) if case["addend"] else None
        # the forward pass has left these behind
        s["mean"] = x.mean(1)
        s["rstd"] = (x.var(1, unbiased=False) + LN_EPS).rsqrt_()
        return s
    shapes = _shapes(case["shapes"])
    g = [_update(gen, r, c) for r, c in shapes]
    if op == "ns":
        return {"op": op, "x": g}
    # a model's weights and momenta lie one after the other in one buffer each
    flat_p, p = _joined([torch.randn(r, c, generator=gen, device=_device()).mul_(1 / math.sqrt(c))
                         for r, c in shapes])
    flat_m, m = _joined([_update(gen, r, c).mul_(5.0) for r, c in shapes])
    return {"op": op, "param": p, "grad": g, "momentum": m, "nesterov": case["nesterov"],
            "scale": [math.sqrt(max(1.0, r / c)) for r, c in shapes],
            "params": flat_p, "momenta": flat_m}


# ------------------------------------------------------------------ plain forms
def _ln_fwd(s):
    x = s["x"]
    mean = x.mean(1)
    d = x - mean[:, None]
    rstd = ((d * d).mean(1) + LN_EPS).rsqrt()
    return d * rstd[:, None] * s["gamma"] + s["beta"], mean, rstd


def _ln_bwd(s):
    xhat = (s["x"] - s["mean"][:, None]) * s["rstd"][:, None]
    dh = s["dy"] * s["gamma"]
    c1 = dh.mean(1, keepdim=True)
    c2 = (dh * xhat).mean(1, keepdim=True)
    dx = (dh - c1 - xhat * c2) * s["rstd"][:, None]
    if s["addend"] is not None:
        dx = dx + s["addend"]
    return dx, (s["dy"] * xhat).sum(0), s["dy"].sum(0)


def _orthogonalise(g):
    x = g.t() if g.shape[0] > g.shape[1] else g
    norm = x.double().square().sum().sqrt()  # a long sum: in 64 bits
    x = x * (1.0 / (norm + NS_EPS)).float()
    a, b, c = NS_COEFFS
    for _ in range(NS_STEPS):
        gram = x @ x.t()
        x = a * x + (b * gram + c * (gram @ gram)) @ x
    return x.t() if g.shape[0] > g.shape[1] else x


def _muon_one(p, g, m, nesterov, scale):
    m.mul_(MUON["momentum"]).add_(g)
    u = g + MUON["momentum"] * m if nesterov else m
    p.mul_(1 - MUON["lr"] * MUON["weight_decay"])
    p.sub_(MUON["lr"] * scale * _orthogonalise(u))


# ------------------------------------------------------------------ the library's calls
def _p(t):
    return ctypes.c_void_p(t.data_ptr()) if t is not None else None


def _context():
    from yumelayers_b200.session import Context
    ctx = Context.shared(torch.cuda.current_device())
    # torch's default stream has the handle 0; 1 names the same stream
    ctx.set_stream(torch.cuda.current_stream().cuda_stream or 1)
    return ctx.handle


def _own(s):
    from yumelayers_b200._lib import MuonTensor, NsMatrix, call
    h = _context()
    op = s["op"]
    if op == "ln_fwd":
        x = s["x"]
        rows, cols = x.shape
        y = torch.empty(rows, cols, device=x.device)
        mean, rstd = torch.empty(rows, device=x.device), torch.empty(rows, device=x.device)
        call("yl_layernorm_fwd", h, _p(x), x.stride(0), rows, cols, LN_EPS, _p(s["gamma"]),
             _p(s["beta"]), _p(y), cols, _p(mean), _p(rstd))
        return y, mean, rstd
    if op == "ln_bwd":
        x, dy, add = s["x"], s["dy"], s["addend"]
        rows, cols = x.shape
        dx = torch.empty(rows, cols, device=x.device)
        dg, db = torch.empty(cols, device=x.device), torch.empty(cols, device=x.device)
        call("yl_layernorm_bwd", h, _p(x), x.stride(0), _p(dy), dy.stride(0), rows, cols, LN_EPS,
             _p(s["gamma"]), _p(s["mean"]), _p(s["rstd"]), _p(add),
             add.stride(0) if add is not None else 0, _p(dx), cols, _p(dg), _p(db))
        return dx, dg, db
    if op == "ns":
        y = [torch.empty(x.shape, device=x.device) for x in s["x"]]
        table = (NsMatrix * len(y))(*[
            NsMatrix(x.data_ptr(), o.data_ptr(), x.shape[0], x.shape[1], x.shape[1], x.shape[1])
            for x, o in zip(s["x"], y)])
        call("yl_newton_schulz", h, table, len(y), NS_STEPS, None, NS_EPS)
        return y
    if "table" not in s:  # the weights stay where they are: a program lays this out once
        s["table"] = (MuonTensor * len(s["param"]))(*[
            MuonTensor(p.data_ptr(), g.data_ptr(), m.data_ptr(), p.shape[0], p.shape[1], k)
            for p, g, m, k in zip(s["param"], s["grad"], s["momentum"], s["scale"])])
    call("yl_muon_multi", h, s["table"], len(s["param"]), MUON["lr"], MUON["momentum"],
         int(s["nesterov"]), MUON["weight_decay"], NS_STEPS, None, NS_EPS, 1.0, 0.0, 0, None)
    return s["params"], s["momenta"]


def run(state):
    if own:
        return _own(state)
    op = state["op"]
    if op == "ln_fwd":
        return _ln_fwd(state)
    if op == "ln_bwd":
        return _ln_bwd(state)
    if op == "ns":
        return [_orthogonalise(x) for x in state["x"]]
    for p, g, m, k in zip(state["param"], state["grad"], state["momentum"], state["scale"]):
        _muon_one(p, g, m, state["nesterov"], k)
    return state["params"], state["momenta"]


# ------------------------------------------------------------------ work and exact values
def _ns_flops(r, c):
    """Per step, with m <= n: half of the symmetric m x m Gram matrix and of its
    square, and the m x m by m x n product."""
    m, n = min(r, c), max(r, c)
    return NS_STEPS * (m * (m + 1.0) * n + m * (m + 1.0) * m + 2.0 * m * m * n)


def work(case):
    op = case["op"]
    if op in ("ln_fwd", "ln_bwd"):
        rows, cols = case["rows"], case["cols"]
        n = rows * cols
        if op == "ln_fwd":
            return {"bytes": 4 * (2 * n + 2 * cols + 2 * rows), "flops": 8 * n}
        return {"bytes": 4 * ((4 if case["addend"] else 3) * n + 3 * cols + 2 * rows),
                "flops": 16 * n}
    shapes = _shapes(case["shapes"])
    n = sum(r * c for r, c in shapes)
    return {"bytes": (8 if op == "ns" else 20) * n, "flops": sum(_ns_flops(r, c) for r, c in shapes)}


def _polar_exact(g):
    """The iteration by its definition, in 64 bits: on the side of the shorter dimension."""
    z = g.double()
    z = z / (torch.sqrt(torch.sum(z * z)) + NS_EPS)
    a, b, c = (float(k) for k in NS_COEFFS)
    for _ in range(NS_STEPS):
        if z.shape[0] <= z.shape[1]:
            q = torch.mm(z, z.T)
            z = a * z + b * torch.mm(q, z) + c * torch.mm(q, torch.mm(q, z))
        else:
            q = torch.mm(z.T, z)
            z = a * z + b * torch.mm(z, q) + c * torch.mm(torch.mm(z, q), q)
    return z


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "ln_fwd":
        x = s["x"].double()
        var, mean = torch.var_mean(x, 1, correction=0)
        rstd = 1.0 / torch.sqrt(var + LN_EPS)
        y = (x - mean.unsqueeze(1)) * (rstd.unsqueeze(1) * s["gamma"].double())
        return y + s["beta"].double(), mean, rstd
    if op == "ln_bwd":
        x, dy = s["x"].double(), s["dy"].double()
        var, mean = torch.var_mean(x, 1, correction=0)
        inv = 1.0 / torch.sqrt(var + LN_EPS)
        h = (x - mean.unsqueeze(1)) * inv.unsqueeze(1)
        t = dy * s["gamma"].double()
        n = x.shape[1]
        dx = inv.unsqueeze(1) / n * (n * t - t.sum(1, keepdim=True)
                                     - h * torch.sum(t * h, 1, keepdim=True))
        if s["addend"] is not None:
            dx = dx + s["addend"].double()
        return dx, torch.sum(dy * h, 0), torch.sum(dy, 0)
    if op == "ns":
        return [_polar_exact(x) for x in s["x"]]
    params, momenta = [], []
    mu, lr = MUON["momentum"], MUON["lr"]
    for p, g, m, k in zip(s["param"], s["grad"], s["momentum"], s["scale"]):
        m2 = mu * m.double() + g.double()
        u = g.double() + mu * m2 if case["nesterov"] else m2
        decayed = p.double() * (1 - lr * MUON["weight_decay"])
        params.append((decayed - lr * k * _polar_exact(u)).reshape(-1))
        momenta.append(m2.reshape(-1))
    return torch.cat(params), torch.cat(momenta)
