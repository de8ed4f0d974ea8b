"""Newton-Schulz orthogonalisation and the Muon step on the GPU against their
definitions in float64.

Tolerances.  One product of the iteration carries a relative error of at most
e = 2^-20 of its operands' norms: 2^-22 for operands kept to 22 bits or more,
and the fp32 accumulation of up to 1200 terms.  A step has three products, so
its result is 3 e off; where all singular values grow alike (random matrices)
the five steps add up: 5 * 3 e = 1.5e-5, held to 2e-5.  Where small singular
values stand beside large ones, an error of the first step grows like the
smallest singular values do, by up to 3.4445^4 = 141 against the norm of the
result: 141 * 3 e = 4e-4, the bound for those cases.  A parameter moves by lr
times that."""
import ctypes as C

import numpy as np
import pytest
import torch

from yumelayers_b200._lib import MuonTensor, NsMatrix, YumeError, call

pytestmark = pytest.mark.gpu

TOL, TOL_SPREAD = 2e-5, 4e-4
QUINTIC = (3.4445, -4.7750, 2.0315)


def rel(a, b):
    a, b = np.asarray(a, np.float64), np.asarray(b, np.float64)
    return float(np.linalg.norm(a - b) / max(np.linalg.norm(b), 1e-30))


def ns64(x, steps=5, coeffs=None, eps=1e-7):
    x = np.asarray(x, np.float64)
    flip = x.shape[0] > x.shape[1]
    if flip:
        x = x.T
    x = x / (np.sqrt((x * x).sum()) + eps)
    for s in range(steps):
        a, b, c = coeffs[3 * s: 3 * s + 3] if coeffs else QUINTIC
        g = x @ x.T
        x = a * x + b * (g @ x) + c * (g @ (g @ x))
    return x.T if flip else x


@pytest.fixture
def h(ctx):
    ctx.set_stream(torch.cuda.current_stream().cuda_stream or 1)
    yield ctx.handle
    torch.cuda.synchronize()
    ctx.set_stream(None)


def normal(seed, r, c):
    return np.random.default_rng(seed).standard_normal((r, c)).astype(np.float32)


def run_ns(h, mats, steps=5, coeffs=None, eps=1e-7, pad=0):
    dev, out = [], []
    for x in mats:
        b = torch.full((x.shape[0], x.shape[1] + pad), float("nan"), device="cuda")
        b[:, : x.shape[1]] = torch.from_numpy(x)
        dev.append(b)
        out.append(torch.full_like(b, 9.0))
    table = (NsMatrix * len(mats))(*[
        NsMatrix(b.data_ptr(), o.data_ptr(), x.shape[0], x.shape[1], b.shape[1], b.shape[1])
        for b, o, x in zip(dev, out, mats)])
    q = (C.c_float * len(coeffs))(*coeffs) if coeffs else None
    call("yl_newton_schulz", h, table, len(mats), steps, q, eps)
    for o, x in zip(out, mats):
        assert torch.all(o[:, x.shape[1]:] == 9.0)
    return [o[:, : x.shape[1]].cpu().numpy() for o, x in zip(out, mats)]


SHAPES = [(1, 1), (1, 2), (2, 1), (3, 3), (1, 700), (700, 1), (4, 36), (3, 1152), (1152, 5),
          (15, 17), (63, 64), (64, 64), (64, 65), (65, 64), (100, 300), (127, 128), (128, 128),
          (128, 129), (128, 1152), (1152, 128), (129, 257), (257, 129), (128, 864), (192, 320),
          (256, 1000), (255, 511), (511, 255), (320, 320), (384, 1153), (2, 4096), (128, 2048),
          (2049, 120), (65, 2500), (4096, 128), (4033, 17), (64, 4097), (4200, 100), (128, 192),
          (257, 64), (70, 513), (3785, 2), (5, 6000), (6144, 60), (60, 6145), (64, 2000), (1000, 64)]


@pytest.mark.parametrize("r,c", SHAPES)
def test_one_matrix(h, r, c):
    x = normal(r * 7919 + c, r, c)
    got, = run_ns(h, [x], pad=(r + c) % 5)
    # a single row or column is a unit vector: nothing spreads; small ones may be nearly singular
    assert rel(got, ns64(x)) < (TOL if max(r, c) > 1.2 * min(r, c) or min(r, c) == 1 else TOL_SPREAD)


def check_on_device(h, shapes):
    """Normal matrices, two equal calls, against float64 on the device."""
    gen = torch.Generator(device="cuda").manual_seed(5)
    xs = [torch.randn(s, generator=gen, device="cuda") for s in shapes]
    ys, again = [torch.empty_like(x) for x in xs], [torch.empty_like(x) for x in xs]
    for out in (ys, again):
        table = (NsMatrix * len(xs))(*[
            NsMatrix(x.data_ptr(), y.data_ptr(), *x.shape, x.shape[1], x.shape[1])
            for x, y in zip(xs, out)])
        call("yl_newton_schulz", h, table, len(xs), 5, None, 1e-7)
    for x, y, y2 in zip(xs, ys, again):
        z = x.double() if x.shape[0] <= x.shape[1] else x.double().T
        z = z / (z.square().sum().sqrt() + 1e-7)
        for _ in range(5):
            g = z @ z.T
            z = QUINTIC[0] * z + QUINTIC[1] * (g @ z) + QUINTIC[2] * (g @ (g @ z))
        z = z if x.shape[0] <= x.shape[1] else z.T
        assert float((y.double() - z).norm() / z.norm()) < TOL
        assert torch.equal(y, y2)


@pytest.mark.parametrize("shapes", [[(4000, 3900)], [(900, 4097), (64, 700)] + [(1030, 1000)] * 14,
                                    [(2500, 2560), (2050, 2049)]])
def test_enough_tiles_for_pairs_of_blocks(h, shapes):
    """Sizes that run on 256 x 256 tiles."""
    check_on_device(h, shapes)


@pytest.mark.parametrize("shapes", [
    [(1500, 1200)], [(1200, 1501)], [(257, 20000)], [(20000, 200)], [(150, 700)] * 70])
def test_tiles_of_128_columns(h, shapes):
    """More tiles of a phase than SMs, in the caller's order; with shares of a long side."""
    check_on_device(h, shapes)


@pytest.mark.parametrize("shapes", [
    [(333, 2500)], [(2500, 333)], [(997, 700)], [(576, 700)], [(129, 1024), (300, 3000), (640, 900), (1024, 130)]])
def test_tiles_of_64_columns(h, shapes):
    """Fewer tiles than SMs, odd and even numbers of blocks; the last table has tiles of
    both widths."""
    check_on_device(h, shapes)


def test_singular_values_end_near_one(h):
    x = normal(0, 96, 400)
    s = np.linalg.svd(run_ns(h, [x])[0].astype(np.float64), compute_uv=False)
    assert s.min() > 0.6 and s.max() < 1.25


def test_many_matrices_in_one_call(h):
    """More than one launch's table.  The bits of a result may depend on the table
    (how the long side is shared out does), its accuracy does not."""
    rng = np.random.default_rng(1)
    mats = [normal(i, int(rng.integers(1, 200)), int(rng.integers(1, 200))) for i in range(150)]
    short = [m for m in mats if min(m.shape) <= 128]
    for table in (mats, short):
        together = run_ns(h, table)
        for got, again, x in zip(together, run_ns(h, table), table):
            assert np.array_equal(got, again)
            assert rel(got, ns64(x)) < TOL_SPREAD


@pytest.mark.parametrize("r,c", [(60, 200), (200, 60), (130, 140), (300, 280)])
@pytest.mark.parametrize("kind", ["decay", "rank3", "scaled_up", "scaled_down", "one_entry"])
def test_spectra_and_scales(h, r, c, kind):
    x = normal(r + c, r, c)
    if kind == "decay":
        u, s, v = np.linalg.svd(x, full_matrices=False)
        x = ((u * 10.0 ** (-6 * np.arange(s.size) / s.size)) @ v).astype(np.float32)
    elif kind == "rank3":
        x = normal(1, r, 3) @ normal(2, 3, c)
    elif kind == "scaled_up":
        x = x * np.float32(1e30)  # the squares pass fp32's range
    elif kind == "scaled_down":
        x = x * np.float32(1e-5)  # eps still small against the norm
    else:
        x = np.zeros_like(x)
        x[r // 2, c // 3] = -3.0
    assert rel(run_ns(h, [x])[0], ns64(x)) < TOL_SPREAD


def test_zero_nan_and_inf_matrices(h):
    good, zero, nan, inf = normal(3, 90, 130), np.zeros((70, 140), np.float32), normal(
        4, 140, 70), normal(5, 64, 64)
    nan[3, 5], inf[0, 0] = np.nan, np.inf
    for more in ([], [normal(6, 200, 300)]):  # alone on the chip, or beside a larger matrix
        got = run_ns(h, [nan, good, zero, inf] + more)
        clean = run_ns(h, [normal(4, 140, 70), good, zero, normal(5, 64, 64)] + more)
        assert np.array_equal(got[1], clean[1])
        assert not got[2].any()
        assert np.isnan(got[0]).all() and np.isnan(got[3]).all()


def test_steps_and_coefficients(h):
    x = normal(6, 100, 150)
    assert rel(run_ns(h, [x], steps=0)[0], ns64(x, 0)) < 1e-6
    cubic = (1.5, -0.5, 0.0) * 12
    got = run_ns(h, [x], steps=12, coeffs=cubic)[0]
    assert rel(got, ns64(x, 12, cubic)) < TOL_SPREAD
    mixed = (3.0, -3.2, 1.2, 2.0, -1.5, 0.5)
    assert rel(run_ns(h, [x], steps=2, coeffs=mixed)[0], ns64(x, 2, mixed)) < TOL


@pytest.mark.parametrize("r,c", [(40, 90), (90, 40), (128, 256), (300, 200)])
def test_in_place_and_column_slices(h, r, c):
    x = normal(8, r, c)
    want, = run_ns(h, [x])
    t = torch.from_numpy(x).cuda()
    table = (NsMatrix * 1)(NsMatrix(t.data_ptr(), t.data_ptr(), r, c, c, c))
    call("yl_newton_schulz", h, table, 1, 5, None, 1e-7)
    assert np.array_equal(t.cpu().numpy(), want)
    # two matrices side by side in one buffer, each written in place
    x2 = normal(9, r, c)
    apart = run_ns(h, [x, x2])
    both = torch.from_numpy(np.concatenate([x, x2], 1)).cuda()
    table = (NsMatrix * 2)(*[NsMatrix(both.data_ptr() + 4 * o, both.data_ptr() + 4 * o, r, c, 2 * c,
                                      2 * c) for o in (0, c)])
    call("yl_newton_schulz", h, table, 2, 5, None, 1e-7)
    assert np.array_equal(both[:, :c].cpu().numpy(), apart[0])
    assert np.array_equal(both[:, c:].cpu().numpy(), apart[1])


def muon64(p, g, m, lr, mu, nesterov, wd, scale):
    p, g, m = (np.asarray(a, np.float64) for a in (p, g, m))
    m2 = mu * m + g
    u = g + mu * m2 if nesterov else m2
    return p * (1 - lr * wd) - lr * scale * ns64(u), m2


@pytest.mark.parametrize("nesterov", [True, False])
@pytest.mark.parametrize("shapes", [[(5, 7)], [(128, 1152), (512, 128), (3, 1)],
                                    [(1, 1), (33, 200), (200, 33), (256, 300), (64, 64)]])
def test_muon_step(h, shapes, nesterov):
    from yumelayers_b200 import ops
    ps, gs, ms = ([normal(100 * k + i, *s) * np.float32(f) for i, s in enumerate(shapes)]
                  for k, f in enumerate((0.05, 0.01, 0.03)))
    for wd in (0.0, 0.1):
        p2, m2, _ = ops.muon_multi(ps, gs, ms, lr=0.02, momentum=0.9, nesterov=nesterov,
                                   weight_decay=wd)
        for i, s in enumerate(shapes):
            pr, mr = muon64(ps[i], gs[i], ms[i], 0.02, 0.9, nesterov, wd, ops.muon_scale(*s))
            assert rel(m2[i], mr) < 2e-7  # one product and one sum
            step = np.linalg.norm(pr - ps[i] * (1 - 0.02 * wd))
            # the step's error, and the parameter's own roundings
            assert np.linalg.norm(p2[i] - pr) < TOL_SPREAD * step + 1.5e-7 * np.linalg.norm(ps[i])


def test_muon_sanitize_clip_scale(h):
    from yumelayers_b200 import ops
    p, g, m = normal(1, 50, 80), normal(2, 50, 80), normal(3, 50, 80) * np.float32(0.01)
    g[0, 0], g[49, 79] = np.nan, -np.inf
    p2, m2, norm = ops.muon_multi([p], [g], [m], lr=0.02, grad_scale=0.25, clip_max_norm=2.0,
                                  sanitize=True)
    gc = np.where(np.isfinite(g), g * np.float64(0.25), 0.0)
    want = np.sqrt((gc * gc).sum())
    assert abs(norm - want) < 1e-6 * want and want > 2.0
    pr, mr = muon64(p, gc * (2.0 / want), m, 0.02, 0.95, True, 0.0, 1.0)
    assert rel(m2[0], mr) < 5e-7
    assert np.linalg.norm(p2[0] - pr) < TOL_SPREAD * np.linalg.norm(pr - p) + 1.5e-7 * np.linalg.norm(p)
    _, _, norm = ops.muon_multi([p], [p], [m], lr=0.02, grad_scale=2.0)  # norm without a clip
    assert abs(norm - 2 * np.linalg.norm(p.astype(np.float64))) < 1e-5 * norm
    # a norm below the limit leaves the gradient alone
    a = ops.muon_multi([p], [p], [m], lr=0.02, clip_max_norm=1e9)
    b = ops.muon_multi([p], [p], [m], lr=0.02)
    assert np.array_equal(a[0][0], b[0][0]) and np.array_equal(a[1][0], b[1][0])


def test_odd_alignment_inside_a_flat_buffer(h):
    shapes = [(3, 5), (129, 70), (7, 333), (64, 128)]
    n = sum(r * c for r, c in shapes)
    flat = [torch.from_numpy(normal(i, 1, n + 3).reshape(-1)).cuda() for i in range(3)]
    before = [t.cpu().numpy().copy() for t in flat]
    offs = np.cumsum([1] + [r * c for r, c in shapes])  # from float 1 on: 4-byte alignment only
    table = (MuonTensor * len(shapes))(*[
        MuonTensor(*[t.data_ptr() + 4 * int(o) for t in flat], r, c, 1.0)
        for o, (r, c) in zip(offs, shapes)])
    call("yl_muon_multi", h, table, len(shapes), 0.02, 0.95, 1, 0.0, 5, None, 1e-7, 1.0, 0.0, 0, None)
    after = [t.cpu().numpy() for t in flat]
    assert np.array_equal(after[1], before[1])
    for k in (0, 2):
        assert after[k][0] == before[k][0] and np.array_equal(after[k][offs[-1]:], before[k][offs[-1]:])
    for o, (r, c) in zip(offs, shapes):
        part = lambda a: a[o: o + r * c].reshape(r, c)  # noqa: E731
        pr, mr = muon64(*map(part, before), 0.02, 0.95, True, 0.0, 1.0)
        assert rel(part(after[2]), mr) < 2e-7
        assert np.linalg.norm(part(after[0]) - pr) < TOL_SPREAD * np.linalg.norm(
            pr - part(before[0])) + 1.5e-7 * np.linalg.norm(part(before[0]))


def test_same_bits_capture_and_two_graphs(h, ctx):
    def make(seed, *shapes):
        return [(torch.from_numpy(normal(seed + 3 * i, *s)).cuda(),
                 torch.empty(s, device="cuda")) for i, s in enumerate(shapes)]

    def step(s):
        table = (NsMatrix * len(s))(*[
            NsMatrix(x.data_ptr(), y.data_ptr(), *x.shape, x.shape[1], x.shape[1]) for x, y in s])
        call("yl_newton_schulz", h, table, len(s), 5, None, 1e-7)

    sets = [make(1, (128, 700), (300, 130)), make(50, (256, 256), (90, 33)),
            make(80, (128, 1152), (1000, 40))]
    want = []
    for s in sets:
        step(s)
        torch.cuda.synchronize()
        want.append([y.clone() for _, y in s])
        step(s)
        torch.cuda.synchronize()
        assert all(torch.equal(a, y) for a, (_, y) in zip(want[-1], s))
    graphs = []
    for s in sets:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            ctx.set_stream(torch.cuda.current_stream().cuda_stream)
            step(s)
        graphs.append(g)
    ctx.set_stream(torch.cuda.current_stream().cuda_stream or 1)
    step(make(99, (1500, 1400)))  # grows the context's workspace
    for s in sets:
        for _, y in s:
            y.zero_()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in graphs]
    for _ in range(4):
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
    torch.cuda.synchronize()
    for s, w in zip(sets, want):
        assert all(torch.equal(a, y) for a, (_, y) in zip(w, s))


def test_two_streams_in_turn(ctx):
    x = torch.from_numpy(normal(4, 500, 700)).cuda()
    outs = [torch.empty_like(x) for _ in range(6)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for i, y in enumerate(outs):
        ctx.set_stream(streams[i % 2].cuda_stream)
        table = (NsMatrix * 1)(NsMatrix(x.data_ptr(), y.data_ptr(), 500, 700, 700, 700))
        call("yl_newton_schulz", ctx.handle, table, 1, 5, None, 1e-7)
    torch.cuda.synchronize()
    ctx.set_stream(None)
    assert all(torch.equal(y, outs[0]) for y in outs)
    assert rel(outs[0].cpu(), ns64(x.cpu().numpy())) < TOL_SPREAD


def test_zero_and_tiny_matrices_without_eps(h):
    zero, tiny = np.zeros((30, 50), np.float32), normal(3, 40, 60) * np.float32(1e-38)
    tiny[0, :5] = 0.0
    for more in ([], [normal(4, 140, 150)]):
        got = run_ns(h, [zero, tiny] + more, eps=0.0)
        assert not got[0].any()
        assert rel(got[1], ns64(tiny, eps=0.0)) < TOL_SPREAD
    assert not run_ns(h, [zero], steps=0, eps=0.0)[0].any()
    inf = normal(5, 20, 30)
    inf[3, 3] = np.inf
    assert np.isnan(run_ns(h, [inf], steps=0)[0]).all()


def test_two_contexts_at_once():
    """Two contexts on two streams, each with more blocks than fit beside the other's."""
    from yumelayers_b200.session import Context
    a, b = Context(0), Context(0)
    sets = []
    for seed, shapes in ((1, [(700, 900), (128, 300)]), (20, [(128, 1152)] * 6)):
        xs = [torch.from_numpy(normal(seed + i, *s)).cuda() for i, s in enumerate(shapes)]
        sets.append((xs, [torch.empty_like(x) for x in xs]))
    tables = [(NsMatrix * len(xs))(*[
        NsMatrix(x.data_ptr(), y.data_ptr(), *x.shape, x.shape[1], x.shape[1])
        for x, y in zip(xs, ys)]) for xs, ys in sets]
    torch.cuda.synchronize()
    for _ in range(20):
        for c, t in ((a, tables[0]), (b, tables[1]), (b, tables[1])):
            call("yl_newton_schulz", c.handle, t, len(t), 5, None, 1e-7)
    torch.cuda.synchronize()
    for c in (a, b):
        c.check_device_errors()
        call("yl_ctx_destroy", c.handle)
    for xs, ys in sets:
        for x, y in zip(xs, ys):
            assert rel(y.cpu(), ns64(x.cpu().numpy())) < TOL_SPREAD


@pytest.mark.parametrize("shapes", [[(128, 1152)], [(300, 500), (64, 64)], [(1500, 1400)] * 8, [(2560, 2500)] * 2],
                         ids=["on chip", "single blocks", "many tiles", "pairs"])
def test_waits_that_run_out_return_a_status(ctx, shapes):
    """With a limit of 200 cycles the kernels' waits give up, every warp leaves, and the
    host reads a timeout; with the default again the same call is right."""
    xs = [torch.from_numpy(normal(7 + i, *s)).cuda() for i, s in enumerate(shapes)]
    ys = [torch.empty_like(x) for x in xs]
    table = (NsMatrix * len(xs))(*[
        NsMatrix(x.data_ptr(), y.data_ptr(), *x.shape, x.shape[1], x.shape[1])
        for x, y in zip(xs, ys)])
    torch.cuda.synchronize()
    ctx.set_wait_limit(200)
    try:
        call("yl_newton_schulz", ctx.handle, table, len(xs), 5, None, 1e-7)
        with pytest.raises(YumeError) as e:
            ctx.check_device_errors()
        assert e.value.status == 3  # YL_ERR_TIMEOUT
    finally:
        ctx.set_wait_limit(0)
    call("yl_newton_schulz", ctx.handle, table, len(xs), 5, None, 1e-7)
    ctx.check_device_errors()
    assert rel(ys[0].cpu(), ns64(xs[0].cpu().numpy())) < TOL_SPREAD


def test_many_small_weights_with_a_clip(h):
    """150 matrices: three tables, one norm over all of them."""
    from yumelayers_b200 import ops
    rng = np.random.default_rng(9)
    shapes = [(int(rng.integers(1, 60)), int(rng.integers(1, 90))) for _ in range(150)]
    ps, gs, ms = ([normal(1000 * k + i, *s) for i, s in enumerate(shapes)] for k in range(3))
    p2, m2, norm = ops.muon_multi(ps, gs, ms, lr=0.01, clip_max_norm=10.0)
    want = np.sqrt(sum((g.astype(np.float64) ** 2).sum() for g in gs))
    assert abs(norm - want) < 1e-6 * want
    for i in range(0, 150, 7):
        pr, mr = muon64(ps[i], gs[i] * (10.0 / want), ms[i], 0.01, 0.95, True, 0.0,
                        ops.muon_scale(*shapes[i]))
        assert rel(m2[i], mr) < 5e-7
        assert np.linalg.norm(p2[i] - pr) < TOL_SPREAD * np.linalg.norm(
            pr - ps[i]) + 1.5e-7 * np.linalg.norm(ps[i])


def test_refused_calls_leave_the_outputs_alone(h):
    x = torch.ones(4, 4, device="cuda")
    y = torch.full((4, 4), 5.0, device="cuda")
    table = (NsMatrix * 2)(NsMatrix(x.data_ptr(), y.data_ptr(), 4, 4, 4, 4),
                           NsMatrix(x.data_ptr(), None, 4, 4, 4, 4))
    with pytest.raises(YumeError):
        call("yl_newton_schulz", h, table, 2, 5, None, 1e-7)
    torch.cuda.synchronize()
    assert torch.all(y == 5.0)


def test_residual_mlp_trains_with_layernorm_muon_and_adam(ctx):
    """LayerNorm -> Linear -> SiLU -> Linear (+ residual), MSE; three steps with
    Muon on both weights and Adam on the vectors, against float64 throughout."""
    from yumelayers_b200 import ops
    rng = np.random.default_rng(11)
    n, d, hid, lr = 24, 48, 96, 0.02
    x, target = rng.standard_normal((n, d)), rng.standard_normal((n, d))
    W = {"w1": rng.standard_normal((hid, d)) / 7, "w2": rng.standard_normal((d, hid)) / 10}
    V = {"g": np.ones(d), "b": np.zeros(d), "b1": np.zeros(hid), "b2": np.zeros(d)}
    state = {k: np.zeros_like(v) for k, v in W.items()}
    adam = {k: (np.zeros_like(v), np.zeros_like(v)) for k, v in V.items()}
    f32 = lambda q: {k: v.astype(np.float32) for k, v in q.items()}  # noqa: E731
    Wg, Vg, Sg = f32(W), f32(V), f32(state)
    Ag = {k: [a.astype(np.float32) for a in v] for k, v in adam.items()}
    silu = lambda a: a / (1 + np.exp(-a))  # noqa: E731
    dsilu = lambda a: (1 + a * (1 - 1 / (1 + np.exp(-a)))) / (1 + np.exp(-a))  # noqa: E731
    x32 = x.astype(np.float32)
    x = x32.astype(np.float64)
    for t in (1, 2, 3):
        # float64
        m, r = x.mean(1, keepdims=True), 1 / np.sqrt(x.var(1, keepdims=True) + 1e-5)
        hh = (x - m) * r
        a0 = hh * V["g"] + V["b"]
        a1 = a0 @ W["w1"].T + V["b1"]
        a2 = silu(a1) @ W["w2"].T + V["b2"] + x
        d2 = 2 * (a2 - target) / a2.size
        G = {"w2": d2.T @ silu(a1)}
        d1 = (d2 @ W["w2"]) * dsilu(a1)
        G["w1"] = d1.T @ a0
        d0 = d1 @ W["w1"]
        Gv = {"g": (d0 * hh).sum(0), "b": d0.sum(0), "b1": d1.sum(0), "b2": d2.sum(0)}
        # the library's operators
        y0, mg, rg = ops.layernorm_fwd(x32, Vg["g"], Vg["b"])
        y1 = ops.linear_fwd(y0, Wg["w1"], Vg["b1"])
        s1 = silu(y1.astype(np.float64)).astype(np.float32)
        y2 = ops.linear_fwd(s1, Wg["w2"], Vg["b2"]) + x32
        e2 = (2 * (y2 - target) / y2.size).astype(np.float32)
        ds, dw2, db2 = ops.linear_bwd(s1, Wg["w2"], e2)
        e1 = (ds * dsilu(y1.astype(np.float64))).astype(np.float32)
        dy0, dw1, db1 = ops.linear_bwd(y0, Wg["w1"], e1)
        dx, dg, db = ops.layernorm_bwd(x32, dy0, Vg["g"], mean=mg, rstd=rg, addend=e2)
        dh = d0 * V["g"]
        dx_ref = r * (dh - dh.mean(1, keepdims=True) - hh * (dh * hh).mean(1, keepdims=True)) + d2
        assert rel(dx, dx_ref) < 1e-3 and rel(dw1, G["w1"]) < 1e-3 and rel(dg, Gv["g"]) < 1e-3
        # update
        for k in W:
            W[k], state[k] = muon64(W[k], G[k], state[k], lr, 0.95, True, 0.0,
                                    ops.muon_scale(*W[k].shape))
        names = list(V)
        for k in names:
            mm = 0.9 * adam[k][0] + 0.1 * Gv[k]
            vv = 0.999 * adam[k][1] + 0.001 * Gv[k] ** 2
            adam[k] = (mm, vv)
            V[k] = V[k] - 1e-3 * (mm / (1 - 0.9 ** t)) / (np.sqrt(vv / (1 - 0.999 ** t)) + 1e-8)
        ps, ms, _ = ops.muon_multi([Wg["w1"], Wg["w2"]], [dw1, dw2], [Sg["w1"], Sg["w2"]], lr=lr)
        Wg, Sg = dict(zip(("w1", "w2"), ps)), dict(zip(("w1", "w2"), ms))
        vs, m1, v1, _ = ops.adam_multi([Vg[k] for k in names], [dg, db, db1, db2],
                                       [Ag[k][0] for k in names], [Ag[k][1] for k in names],
                                       lr=1e-3, t=t)
        Vg = dict(zip(names, vs))
        Ag = {k: [a, b] for k, a, b in zip(names, m1, v1)}
        # each step's own error is 4e-4 of a step of norm lr * sqrt(rank); three of them, and
        # what earlier ones moved the gradients by
        for k in W:
            assert np.linalg.norm(Wg[k] - W[k]) < 2e-3 * lr * t * np.sqrt(min(W[k].shape)) * 2
