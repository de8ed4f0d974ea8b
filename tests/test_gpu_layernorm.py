"""LayerNorm forward and backward on the GPU against the formulas in float64.

Tolerances (u = 2^-24, fp32's half step).  y: with h of order 1 a value carries
the roundings of x - mean (2 with the correction term), of 1/sqrt(var + eps)
(about 4: two divisions, the square root, the tree sums' log2(n) / sqrt(n)),
of two products and one sum: under 16 u of the output's root mean square, 1e-6.
dx has about twice as many (two row means more): 2e-6.  dgamma and dbeta sum
their rows in at most 64 fp32 additions before a wider or compensated step, of
random signs: 64 u = 4e-6 relative to the vector's norm, and 4e-6 is also what
statistics rounded to fp32 may move them by."""
import ctypes as C

import numpy as np
import pytest
import torch

from yumelayers_b200._lib import call

pytestmark = pytest.mark.gpu

TOL_Y, TOL_DX, TOL_SUM = 1e-6, 2e-6, 4e-6


def rel(a, b):
    a, b = np.asarray(a, np.float64), np.asarray(b, np.float64)
    return float(np.linalg.norm(a - b) / max(np.linalg.norm(b), 1e-30))


def stats64(x, eps):
    x = x.astype(np.float64)
    m = x.mean(-1)
    return m, 1.0 / np.sqrt(((x - m[:, None]) ** 2).mean(-1) + eps)


def fwd64(x, ga, be, eps):
    m, r = stats64(x, eps)
    return (x - m[:, None]) * r[:, None] * ga + be, m, r


def bwd64(x, dy, ga, eps, addend=None):
    m, r = stats64(x, eps)
    h = (x.astype(np.float64) - m[:, None]) * r[:, None]
    t = dy.astype(np.float64) * ga
    dx = r[:, None] * (t - t.mean(1, keepdims=True) - h * (t * h).mean(1, keepdims=True))
    if addend is not None:
        dx = dx + addend
    return dx, (dy * h).sum(0), dy.astype(np.float64).sum(0)


def p(t):
    return C.c_void_p(t.data_ptr()) if t is not None else None


@pytest.fixture
def h(ctx):
    """The shared context on torch's stream (as a caller with torch tensors sets it)."""
    ctx.set_stream(torch.cuda.current_stream().cuda_stream or 1)
    yield ctx.handle
    torch.cuda.synchronize()
    ctx.set_stream(None)


def rows_in(a, pad):
    """a as the first columns of a device buffer with `pad` more, filled with NaN."""
    buf = torch.full((a.shape[0], a.shape[1] + pad), float("nan"), device="cuda")
    buf[:, : a.shape[1]] = torch.from_numpy(a)
    return buf


SHAPES = [(1, 1), (3, 1), (1, 2), (5, 3), (2, 4), (33, 4), (1000, 5), (7, 31), (130, 32), (9, 33),
          (257, 64), (64, 96), (65, 127), (4099, 128), (31, 129), (100, 255), (77, 256), (3, 257),
          (515, 384), (32, 512), (50, 1000), (1, 1021), (20, 1024), (13, 2048), (6, 2049),
          (5, 4096), (3, 5000), (2, 8192), (4, 8195), (300, 13393), (90, 9000), (2, 16383), (2, 16384), (3, 20000), (1, 70001)]


@pytest.mark.parametrize("rows,cols", SHAPES)
@pytest.mark.parametrize("pad", [0, 3, 4])
def test_forward_backward(h, rows, cols, pad):
    rng = np.random.default_rng(rows * 131 + cols)
    f = lambda *s: rng.standard_normal(s).astype(np.float32)  # noqa: E731
    x, dy, add = f(rows, cols) * 1.5 + np.float32(0.3), f(rows, cols), f(rows, cols)
    ga, be = 1 + np.float32(0.1) * f(cols), np.float32(0.1) * f(cols)
    eps = 1e-5
    xd, dyd, ad = rows_in(x, pad), rows_in(dy, pad), rows_in(add, pad)
    gd, bd = torch.from_numpy(ga).cuda(), torch.from_numpy(be).cuda()
    ld = cols + pad
    y = torch.full((rows, ld), 7.0, device="cuda")
    mean, rstd = torch.empty(rows, device="cuda"), torch.empty(rows, device="cuda")
    call("yl_layernorm_fwd", h, p(xd), ld, rows, cols, eps, p(gd), p(bd), p(y), ld, p(mean),
         p(rstd))
    yr, mr, rr = fwd64(x, ga, be, eps)
    # one column: x - mean is 0 whatever rounding did, y is beta
    assert rel(y[:, :cols].cpu(), yr) < TOL_Y
    assert rel(rstd.cpu(), rr) < TOL_Y
    assert np.abs(mean.cpu().numpy() - mr).max() < 1e-6 * (np.abs(mr).max() + 1.5)
    assert torch.all(y[:, cols:] == 7.0)  # the padding stays as it was
    dxr, dgr, dbr = bwd64(x, dy, ga, eps, add)
    scale = np.linalg.norm(rr[:, None] * dy * ga) + np.linalg.norm(add)
    for given in (True, False):
        dx = torch.full((rows, ld), 7.0, device="cuda")
        dg, db = torch.empty(cols, device="cuda"), torch.empty(cols, device="cuda")
        call("yl_layernorm_bwd", h, p(xd), ld, p(dyd), ld, rows, cols, eps, p(gd),
             p(mean) if given else None, p(rstd) if given else None, p(ad), ld, p(dx), ld, p(dg),
             p(db))
        got = dx[:, :cols].double().cpu().numpy()
        assert np.linalg.norm(got - dxr) < TOL_DX * scale
        assert torch.all(dx[:, cols:] == 7.0)
        # sums of random signs: relative to the terms' norm, not to what cancels
        terms = np.sqrt((dy.astype(np.float64) ** 2).sum(0))
        assert np.linalg.norm(dg.cpu().numpy() - dgr) < TOL_SUM * np.linalg.norm(terms)
        assert np.linalg.norm(db.cpu().numpy() - dbr) < TOL_SUM * np.linalg.norm(terms)


def test_no_affine_partial_outputs_and_in_place(h):
    rng = np.random.default_rng(1)
    x, dy = (rng.standard_normal((37, 96)).astype(np.float32) for _ in range(2))
    xd, dyd = torch.from_numpy(x).cuda(), torch.from_numpy(dy).cuda()
    yr, _, _ = fwd64(x, 1.0, 0.0, 1e-6)
    dxr, dgr, dbr = bwd64(x, dy, 1.0, 1e-6)
    dx, dg, db = torch.empty_like(xd), torch.empty(96, device="cuda"), torch.empty(96, device="cuda")
    args = ("yl_layernorm_bwd", h, p(xd), 96, p(dyd), 96, 37, 96, 1e-6, None, None, None, None, 0)
    call(*args, p(dx), 96, None, None)
    assert rel(dx.cpu(), dxr) < TOL_DX
    call(*args, None, 0, p(dg), None)
    call(*args, None, 0, None, p(db))
    assert rel(dg.cpu(), dgr) < TOL_SUM and rel(db.cpu(), dbr) < TOL_SUM
    # dx added into the buffer that holds the addend
    acc = torch.ones_like(xd)
    call("yl_layernorm_bwd", h, p(xd), 96, p(dyd), 96, 37, 96, 1e-6, None, None, None, p(acc), 96,
         p(acc), 96, None, None)
    assert rel(acc.cpu(), dxr + 1.0) < TOL_DX
    call("yl_layernorm_fwd", h, p(xd), 96, 37, 96, 1e-6, None, None, p(xd), 96, None, None)
    assert rel(xd.cpu(), yr) < TOL_Y
    call("yl_layernorm_bwd", h, None, 96, None, 96, 0, 96, 1e-6, None, None, None, None, 0, None, 96,
         p(dg), p(db))
    assert not dg.any() and not db.any()


@pytest.mark.parametrize("cols", [48, 128, 1024, 6000])
def test_large_offset_and_constant_rows(h, cols):
    """A mean of 4096 standard deviations: the statistics come from differences
    with the mean, which are exact in fp32 there, so y keeps its accuracy.  With
    x = 4096 + d, the roundings left are those of the mean's correction term."""
    rng = np.random.default_rng(2)
    x = (4096 + rng.standard_normal((16, cols))).astype(np.float32)
    x[3] = 2.5  # constant: variance 0, y = beta
    xd, y = torch.from_numpy(x).cuda(), torch.empty(16, cols, device="cuda")
    call("yl_layernorm_fwd", h, p(xd), cols, 16, cols, 1e-5, None, None, p(y), cols, None, None)
    yr, _, _ = fwd64(x, 1.0, 0.0, 1e-5)
    assert rel(y.cpu(), yr) < TOL_Y
    assert not y[3].any()


def test_nan_and_inf_stay_in_their_rows(h):
    x = np.random.default_rng(3).standard_normal((40, 200)).astype(np.float32)
    bad = x.copy()
    bad[5, 7], bad[11, 0] = np.nan, np.inf
    outs = []
    for a in (x, bad):
        xd, y = torch.from_numpy(a).cuda(), torch.empty(40, 200, device="cuda")
        call("yl_layernorm_fwd", h, p(xd), 200, 40, 200, 1e-5, None, None, p(y), 200, None, None)
        outs.append(y.cpu().numpy())
    assert np.isnan(outs[1][[5, 11]]).all()
    keep = [r for r in range(40) if r not in (5, 11)]
    assert np.array_equal(outs[0][keep], outs[1][keep])


def test_gradients_against_differences(h):
    """dx, dgamma and dbeta against central differences of sum(y * dy) with step
    d = 2^-4 in fp32: the difference quotient carries y's rounding (16 u |dy|
    sqrt(n) / d) and a d^2 third-derivative term, both under 1e-2 of the gradient
    scale here."""
    rng = np.random.default_rng(4)
    rows, cols, d = 3, 24, 2.0 ** -4
    x, dy = (rng.standard_normal((rows, cols)).astype(np.float32) for _ in range(2))
    ga, be = (rng.standard_normal(cols).astype(np.float32) for _ in range(2))

    def f(x_, ga_, be_):
        t = [torch.from_numpy(np.ascontiguousarray(a, np.float32)).cuda() for a in (x_, ga_, be_)]
        y = torch.empty(rows, cols, device="cuda")
        call("yl_layernorm_fwd", h, p(t[0]), cols, rows, cols, 1e-5, p(t[1]), p(t[2]), p(y), cols,
             None, None)
        return float((y.double().cpu().numpy() * dy).sum())

    xd, dyd, gd = (torch.from_numpy(a).cuda() for a in (x, dy, ga))
    dx, dg, db = (torch.empty(s, device="cuda") for s in ((rows, cols), cols, cols))
    call("yl_layernorm_bwd", h, p(xd), cols, p(dyd), cols, rows, cols, 1e-5, p(gd), None, None, None,
         0, p(dx), cols, p(dg), p(db))
    for k in (0, 5, 23):
        for r in range(rows):
            e = np.zeros_like(x)
            e[r, k] = d
            num = (f(x + e, ga, be) - f(x - e, ga, be)) / (2 * d)
            assert abs(num - float(dx[r, k])) < 2e-2 * float(dx.abs().max())
        e = np.zeros_like(ga)
        e[k] = d
        assert abs((f(x, ga + e, be) - f(x, ga - e, be)) / (2 * d) - float(dg[k])) < 1e-3 * 10
        assert abs((f(x, ga, be + e) - f(x, ga, be - e)) / (2 * d) - float(db[k])) < 1e-3 * 10


def test_same_bits_twice_and_under_capture(h, ctx):
    """Equal inputs give equal bits; a captured backward pass replays them, also
    after a larger eager call has grown the context's workspace, and a second
    graph replayed beside it on another stream keeps its own."""
    rng = np.random.default_rng(5)

    def make(rows, cols):
        x, dy = (torch.from_numpy(rng.standard_normal((rows, cols)).astype(np.float32)).cuda()
                 for _ in range(2))
        return x, dy, torch.empty_like(x), torch.empty(cols, device="cuda"), torch.empty(
            cols, device="cuda")

    def step(s):
        x, dy, dx, dg, db = s
        rows, cols = x.shape
        call("yl_layernorm_bwd", h, p(x), cols, p(dy), cols, rows, cols, 1e-5, None, None, None,
             None, 0, p(dx), cols, p(dg), p(db))

    sets = [make(3000, 192), make(2500, 320)]
    want = []
    for s in sets:
        step(s)
        torch.cuda.synchronize()
        want.append([t.clone() for t in s[2:]])
        step(s)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(want[-1], s[2:]))
    graphs = []
    for s in sets:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            ctx.set_stream(torch.cuda.current_stream().cuda_stream)
            step(s)
        graphs.append(g)
    ctx.set_stream(torch.cuda.current_stream().cuda_stream or 1)
    big = make(200, 30000)
    step(big)
    for s in sets:
        for t in s[2:]:
            t.zero_()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in graphs]
    for _ in range(3):
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
    torch.cuda.synchronize()
    for s, w in zip(sets, want):
        assert all(torch.equal(a, b) for a, b in zip(w, s[2:]))


def test_calls_on_two_streams_share_the_workspace_in_order(ctx):
    rng = np.random.default_rng(6)
    x, dy = (torch.from_numpy(rng.standard_normal((20000, 256)).astype(np.float32)).cuda()
             for _ in range(2))
    outs = [(torch.empty(256, device="cuda"), torch.empty(256, device="cuda")) for _ in range(8)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for i, (dg, db) in enumerate(outs):
        ctx.set_stream(streams[i % 2].cuda_stream)
        call("yl_layernorm_bwd", ctx.handle, p(x), 256, p(dy), 256, 20000, 256, 1e-5, None, None,
             None, None, 0, None, 0, p(dg), p(db))
    torch.cuda.synchronize()
    ctx.set_stream(None)
    for dg, db in outs[1:]:
        assert torch.equal(dg, outs[0][0]) and torch.equal(db, outs[0][1])


def test_offsets_past_32_bits(h):
    """Rows 2^31 floats apart from the first ones (row stride 2^26, 48 rows: 12.9 GB)."""
    rows, cols, ld = 48, 100, 1 << 26
    buf = torch.empty(rows * ld, device="cuda")
    x = np.random.default_rng(7).standard_normal((rows, cols)).astype(np.float32)
    view = buf.view(rows, ld)
    view[:, :cols] = torch.from_numpy(x)
    y = torch.empty(rows, cols, device="cuda")
    call("yl_layernorm_fwd", h, p(buf), ld, rows, cols, 1e-5, None, None, p(y), cols, None, None)
    yr, _, _ = fwd64(x, 1.0, 0.0, 1e-5)
    assert rel(y.cpu(), yr) < TOL_Y
    dg, db = torch.empty(cols, device="cuda"), torch.empty(cols, device="cuda")
    call("yl_layernorm_bwd", h, p(buf), ld, p(buf), ld, rows, cols, 1e-5, None, None, None, None, 0,
         p(y), cols, p(dg), p(db))
    dxr, dgr, dbr = bwd64(x, x, 1.0, 1e-5)
    scale = np.linalg.norm(x)
    assert np.linalg.norm(y.cpu().numpy() - dxr) < TOL_DX * scale
    assert rel(dg.cpu(), dgr) < TOL_SUM and np.abs(db.cpu().numpy() - dbr).max() < TOL_SUM * scale
    del buf, view


def test_very_long_rows(h):
    """3 million columns, 3000 of them to a thread: the row's sums are in double."""
    rows, cols = 2, 3_000_001
    gen = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn(rows, cols, generator=gen, device="cuda") + 5.0
    dy = torch.randn(rows, cols, generator=gen, device="cuda")
    y, dx, dg, db = (torch.empty_like(x), torch.empty_like(x), torch.empty(cols, device="cuda"),
                     torch.empty(cols, device="cuda"))
    call("yl_layernorm_fwd", h, p(x), cols, rows, cols, 1e-5, None, None, p(y), cols, None, None)
    call("yl_layernorm_bwd", h, p(x), cols, p(dy), cols, rows, cols, 1e-5, None, None, None, None, 0,
         p(dx), cols, p(dg), p(db))
    xn, dn = x.cpu().numpy(), dy.cpu().numpy()
    yr, _, _ = fwd64(xn, 1.0, 0.0, 1e-5)
    dxr, dgr, dbr = bwd64(xn, dn, 1.0, 1e-5)
    assert rel(y.cpu(), yr) < TOL_Y and rel(dx.cpu(), dxr) < TOL_DX
    assert rel(dg.cpu(), dgr) < TOL_SUM and rel(db.cpu(), dbr) < TOL_SUM


def test_numpy_and_session_wrappers(ctx):
    from yumelayers_b200 import ops
    from yumelayers_b200.session import GPUTensor, GpuSession
    rng = np.random.default_rng(8)
    x, dy = (rng.standard_normal((6, 40)).astype(np.float32) for _ in range(2))
    ga, be = (rng.standard_normal(40).astype(np.float32) for _ in range(2))
    y, m, r = ops.layernorm_fwd(x.reshape(2, 3, 40), ga, be)
    yr, mr, rr = fwd64(x, ga, be, 1e-5)
    assert y.shape == (2, 3, 40) and m.shape == (2, 3)
    assert rel(y.reshape(6, 40), yr) < TOL_Y and rel(r.reshape(-1), rr) < TOL_Y
    dx, dg, db = ops.layernorm_bwd(x, dy, ga, mean=m, rstd=r)
    dxr, dgr, dbr = bwd64(x, dy, ga, 1e-5)
    assert rel(dx, dxr) < TOL_DX and rel(dg, dgr) < TOL_SUM and rel(db, dbr) < TOL_SUM
    s = GpuSession(ctx)
    t = lambda a, rows: GPUTensor(ctx, rows, data=a)  # noqa: E731
    xs, gs, bs = t(x, 6), t(ga, 1), t(be, 1)
    assert np.array_equal(s.layerNorm(xs, gs, bs).toArray().reshape(6, 40), y.reshape(6, 40))
    got = s.encodeLayerNormGrad(xs, t(dy, 6), gs)
    assert rel(got[0].toArray().reshape(6, 40), dxr) < TOL_DX
    assert rel(got[1].toArray(), dgr) < TOL_SUM and rel(got[2].toArray(), dbr) < TOL_SUM


@pytest.mark.parametrize("rows,pad", [(1, 0), (300, 3), (5000, 0)])
def test_rows_of_one_column_have_no_gradient(h, rows, pad):
    """One value is its own mean: y = beta, and dx is zero to the last bit."""
    g = torch.Generator(device="cuda").manual_seed(rows)
    x, dy, add = (torch.randn(rows, 1 + pad, generator=g, device="cuda") for _ in range(3))
    gamma, y = torch.full((1,), 1.7, device="cuda"), torch.empty(rows, 1, device="cuda")
    beta = torch.full((1,), -0.3, device="cuda")
    call("yl_layernorm_fwd", h, p(x), 1 + pad, rows, 1, 1e-5, p(gamma), p(beta), p(y), 1, None, None)
    assert torch.all(y == beta)
    dx, dg, db = torch.empty(rows, 1, device="cuda"), torch.empty(1, device="cuda"), torch.empty(1, device="cuda")
    for addend, want in ((None, torch.zeros_like(dx)), (add, add[:, :1])):
        call("yl_layernorm_bwd", h, p(x), 1 + pad, p(dy), 1 + pad, rows, 1, 1e-5, p(gamma), None,
             None, p(addend), 1 + pad, p(dx), 1, p(dg), p(db))
        assert torch.equal(dx, want)
        assert float(dg) == 0
        # 64 roundings of partial sums, of 64 values at most each, in fp32 behind one another
        exact = dy[:, 0].double()
        assert abs(float(db) - float(exact.sum())) <= 64 * 2 ** -24 * float(exact.abs().sum())
