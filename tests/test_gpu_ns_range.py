"""Newton-Schulz and Muon on matrices that lie far below their scale: a norm far
under eps, where X0 = x / (|x| + eps) is small, and rows of different size.

Tolerance: as for single matrices of the other Newton-Schulz tests, 2e-5 of the
result's norm (five steps of three products, each 2^-20 off, are 1.5e-5); nine steps are
2.6e-5, held to 3.5e-5.  With X0 far below one a step is a X and loses less.  A
Muon parameter moves by lr times that and has its own two roundings."""
import ctypes as C

import numpy as np
import pytest
import torch

from yumelayers_b200._lib import MuonTensor, NsMatrix, YumeError, call

pytestmark = pytest.mark.gpu

TOL, TOL9 = 2e-5, 3.5e-5
QUINTIC = (3.4445, -4.7750, 2.0315)
# wide and tall, on the chip, in tiles of 64 and 128 columns; the last on pairs of blocks
SHAPES = [(96, 160), (160, 96), (64, 1000), (300, 200), (257, 1531), (1400, 1500)]
PAIRS = (2600, 2560)


@pytest.fixture
def h(ctx):
    ctx.set_stream(torch.cuda.current_stream().cuda_stream or 1)
    yield ctx.handle
    torch.cuda.synchronize()
    ctx.set_stream(None)


def normal(seed, r, c):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(r, c, generator=gen, device="cuda")


def ns64(x, steps=5, eps=1e-7, coeffs=None):
    z = x.double()
    z = z.T if z.shape[0] > z.shape[1] else z
    z = z / (z.square().sum().sqrt() + eps)
    for s in range(steps):
        a, b, c = coeffs[s] if coeffs else QUINTIC
        g = z @ z.T
        z = a * z + b * (g @ z) + c * (g @ (g @ z))
    return z.T if x.shape[0] > x.shape[1] else z


def run(h, xs, steps=5, eps=1e-7, coeffs=None):
    ys = [torch.empty_like(x) for x in xs]
    table = (NsMatrix * len(xs))(*[
        NsMatrix(x.data_ptr(), y.data_ptr(), *x.shape, x.shape[1], x.shape[1])
        for x, y in zip(xs, ys)])
    q = (C.c_float * (3 * steps))(*[v for s in coeffs for v in s]) if coeffs else None
    call("yl_newton_schulz", h, table, len(xs), steps, q, eps)
    return ys


def rel(y, z):
    return float((y.double() - z).norm() / z.norm())


@pytest.mark.parametrize("shape", SHAPES + [PAIRS])
@pytest.mark.parametrize("ratio", [0.3, 1e-3, 1e-5, 1e-7, 1e-9, 1e-15, 1e-28])
def test_norms_far_below_eps(h, shape, ratio):
    """|x| = ratio * eps."""
    x = normal(sum(shape), *shape)
    x *= ratio * 1e-7 / float(x.norm())
    y, = run(h, [x])
    assert rel(y, ns64(x)) < TOL


def test_norms_of_every_size_in_one_table(h):
    for shapes in ([(40, 70)] * 24, [(40, 70), (200, 300)] * 12):
        xs = [normal(i, *s) for i, s in enumerate(shapes)]
        for i, x in enumerate(xs):
            x *= 10.0 ** (2 - 1.5 * i) / float(x.norm())
        for y, x in zip(run(h, xs), xs):
            assert rel(y, ns64(x)) < TOL


@pytest.mark.parametrize("shape", [(96, 160), (300, 200)])
@pytest.mark.parametrize("eps", [1e-30, 1.0, 1e6, 1e30])
def test_any_eps(h, shape, eps):
    x = normal(3, *shape)
    y, = run(h, [x], eps=eps)
    z = ns64(x, eps=eps)
    assert rel(y, z) < TOL


@pytest.mark.parametrize("steps", [1, 2, 9])
@pytest.mark.parametrize("ratio", [1e-2, 1e-4, 1e-8])
def test_small_norms_over_other_numbers_of_steps(h, steps, ratio):
    """Nine steps carry 1e-4 of eps up to where the quintic bends."""
    for shape in ((96, 160), (257, 400)):
        x = normal(7, *shape)
        x *= ratio * 1e-7 / float(x.norm())
        y, = run(h, [x], steps=steps)
        assert rel(y, ns64(x, steps)) < TOL9


def test_small_norms_under_steps_that_shrink_and_grow(h):
    q = [(3.9, 0.0, 0.0), (0.25, 0.0, 0.0), (2.0, -1.5, 0.5), (0.01, 0.0, 0.0), (3.4445, -4.775, 2.0315)]
    for shape in ((96, 160), (257, 400)):
        for ratio in (1e3, 1e-3, 1e-9):
            x = normal(9, *shape)
            x *= ratio * 1e-7 / float(x.norm())
            y, = run(h, [x], steps=5, coeffs=q)
            assert rel(y, ns64(x, 5, coeffs=q)) < TOL


@pytest.mark.parametrize("shape", [(96, 160), (160, 96), (257, 400)])
@pytest.mark.parametrize("coeffs", [
    [(1e-9, 0.0, 0.0)], [(1e-9, 0.0, 0.0), (1.0, 0.0, 0.0)], [(1e-4, 0.0, 0.0)] * 4 + [(2.0, -1.0, 0.5)],
    [(0.0, 1e-6, 0.0), (3.0, 0.0, 0.0)], [(0.0, 0.0, 1e-3), (0.5, 0.0, 1.0), (2.0, 0.0, 0.0)],
    [(1e-12, 1e-12, -1e-12), (1e-12, 0.0, 0.0)], [(0.0, 0.0, 0.0), (1.0, 0.0, 0.0)]])
def test_steps_that_shrink(h, shape, coeffs):
    """Whatever the steps take off, the scales follow."""
    x = normal(13, *shape)
    y, = run(h, [x], steps=len(coeffs), coeffs=coeffs)
    z = ns64(x, len(coeffs), coeffs=[[float(np.float32(v)) for v in q] for q in coeffs])
    if not any(coeffs[0]):
        assert not y.any()
    else:
        assert rel(y, z) < TOL


@pytest.mark.parametrize("shape", [(96, 160), (160, 96), (300, 280), (512, 1024)])
@pytest.mark.parametrize("small", [1e-3, 1e-6, 1e-8, 1e-10])
@pytest.mark.parametrize("steps", [5, 9])
def test_rows_of_different_size(h, shape, small, steps):
    """Every other row (of the shorter side) by `small`: the largest number of default
    steps is the one at which fp32 products would still do no better."""
    x = normal(11, *shape)
    if shape[0] <= shape[1]:
        x[::2] *= small
    else:
        x[:, ::2] *= small
    y, = run(h, [x], steps=steps)
    assert rel(y, ns64(x, steps)) < TOL9


def test_a_muon_step_of_a_gradient_that_has_nearly_vanished(h):
    for shape in ((64, 128), (200, 300)):
        for size in (1e-9, 1e-13, 1e-20):
            p, g, m = normal(1, *shape) * 0.05, normal(2, *shape), normal(3, *shape)
            g, m = g * (size / float(g.norm())), m * (size / float(m.norm()))
            p0, m0 = p.double(), m.double()
            table = (MuonTensor * 1)(MuonTensor(p.data_ptr(), g.data_ptr(), m.data_ptr(), *shape, 1.0))
            call("yl_muon_multi", h, table, 1, 1.0, 0.95, 1, 0.0, 5, None, 1e-7, 1.0, 0.0, 0, None)
            torch.cuda.synchronize()
            m1 = 0.95 * m0 + g.double()
            step = ns64(g.double() + 0.95 * m1)
            assert float((p.double() - (p0 - step)).norm()) < (
                TOL * float(step.norm()) + 1.5e-7 * float(p0.norm()))


def test_the_trainer_refuses_steps_that_grow_too_far():
    from yumelayers_b200.trainer import Trainer, default_config
    tr = Trainer(default_config(batch=1, height=32, width=48))
    tr.set_muon(steps=9)
    with pytest.raises(YumeError) as e:
        tr.set_muon(steps=10)
    assert e.value.status == 8 and tr.muon["steps"] == 9
    tr.close()
