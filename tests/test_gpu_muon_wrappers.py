"""The array and session wrappers of Newton-Schulz and Muon, called as a user does:
against float64, and against each other (they reach the same entry points, so one
weight moves the same way, bit by bit, through either).  Tolerances as in the
Newton-Schulz tests: 2e-5 for wide and tall matrices; a parameter moves by lr scale
times that and has two roundings of its own."""
import numpy as np
import pytest

from test_gpu_muon import QUINTIC, TOL, muon64, normal, ns64, rel
from yumelayers_b200 import ops
from yumelayers_b200._lib import YumeError
from yumelayers_b200.session import GPUTensor, GpuSession

pytestmark = pytest.mark.gpu
SHAPES = [(40, 100), (100, 40), (300, 130), (1, 9), (9, 1)]


def test_newton_schulz_of_arrays(ctx):
    xs = [normal(i, *s) for i, s in enumerate(SHAPES)]
    for y, x in zip(ops.newton_schulz(xs), xs):
        assert y.shape == x.shape and rel(y, ns64(x)) < TOL
    coeffs = [(3.0, -3.2, 1.2), (2.0, -1.5, 0.5), QUINTIC]
    got = ops.newton_schulz(xs, steps=3, coeffs=coeffs, eps=1e-3)
    for y, x in zip(got, xs):
        assert rel(y, ns64(x, 3, [v for q in coeffs for v in q], 1e-3)) < TOL
    x = xs[0]
    assert rel(ops.newton_schulz([x], steps=0)[0], ns64(x, 0)) < 1e-6
    assert ops.newton_schulz([]) == []
    assert [y.shape for y in ops.newton_schulz([np.zeros((0, 3)), x, np.zeros((2, 0))])] == [
        (0, 3), x.shape, (2, 0)]
    with pytest.raises(ValueError, match="coefficients"):
        ops.newton_schulz([x], steps=2, coeffs=coeffs)


@pytest.mark.parametrize("shape", SHAPES)
def test_session_orthogonalize(ctx, shape):
    x = normal(7, *shape)
    s = GpuSession(ctx)
    t = GPUTensor(ctx, shape[0], data=x)
    y = s.orthogonalize(t)
    assert (y.rows, y.cols) == shape
    assert rel(y.toArray().reshape(shape), ns64(x)) < TOL
    assert np.array_equal(y.toArray().reshape(shape), ops.newton_schulz([x])[0])
    assert np.array_equal(t.toArray().reshape(shape), x)  # the argument stays
    assert rel(s.orthogonalize(t, steps=3, eps=1e-2).toArray().reshape(shape),
               ns64(x, 3, eps=1e-2)) < TOL


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("scale", [None, 0.5])
@pytest.mark.parametrize("nesterov", [True, False])
def test_session_muon_update(ctx, shape, scale, nesterov):
    """Without a scale both doors take sqrt(max(1, rows / cols))."""
    p, g, m = (normal(i, *shape) * np.float32(f) for i, f in enumerate((0.05, 0.01, 0.03)))
    s = GpuSession(ctx)
    pt, gt, mt = (GPUTensor(ctx, shape[0], data=a) for a in (p, g, m))
    kw = dict(nesterov=nesterov, weight_decay=0.1)
    s.muonUpdate(pt, gt, mt, 0.02, mu=0.9, scale=scale, **kw)
    p2, m2, _ = ops.muon_multi([p], [g], [m], 0.02, momentum=0.9,
                               scales=None if scale is None else [scale], **kw)
    assert np.array_equal(pt.toArray().reshape(shape), p2[0])
    assert np.array_equal(mt.toArray().reshape(shape), m2[0])
    assert np.array_equal(gt.toArray().reshape(shape), g)
    factor = max(1.0, shape[0] / shape[1]) ** 0.5 if scale is None else scale
    pr, mr = muon64(p, g, m, 0.02, 0.9, nesterov, 0.1, factor)
    assert rel(m2[0], mr) < 2e-7
    step = np.linalg.norm(pr - p * (1 - 0.02 * 0.1))
    assert np.linalg.norm(p2[0] - pr) < TOL * step + 1.5e-7 * np.linalg.norm(p)


def test_session_refuses_other_shapes(ctx):
    s = GpuSession(ctx)
    a, b = GPUTensor(ctx, 4, 6), GPUTensor(ctx, 6, 5)
    with pytest.raises(YumeError):
        s.muonUpdate(a, b, a, 0.1)
    with pytest.raises(YumeError):
        s.muonUpdate(a, GPUTensor(ctx, 4, 6), b, 0.1)
