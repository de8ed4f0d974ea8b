"""Argument checks of the LayerNorm, Newton-Schulz and Muon entry points: all
of them come before the first device call, so they run without a GPU on a
stand-in for the context."""
import ctypes as C

import numpy as np
import pytest

from yumelayers_b200 import ops
from yumelayers_b200._lib import MuonTensor, NsMatrix, YumeError, call

SHAPE, INVALID, UNSUPPORTED = 1, 7, 8
BASE = 0x7F0000000000  # stands for device memory; never dereferenced


@pytest.fixture
def ctx():
    return C.create_string_buffer(8192)


def refused(status, name, *args):
    with pytest.raises(YumeError) as e:
        call(name, *args)
    assert e.value.status == status, e.value


def fwd(ctx, x=BASE, ldx=64, rows=8, cols=64, eps=1e-5, y=BASE + (1 << 20), ldy=64):
    return ("yl_layernorm_fwd", ctx, x, ldx, rows, cols, eps, None, None, y, ldy, None, None)


def bwd(ctx, x=BASE, ldx=64, dy=BASE + (1 << 20), lddy=64, rows=8, cols=64, eps=1e-5, mean=None,
        rstd=None, add=None, ldadd=64, dx=BASE + (2 << 20), lddx=64):
    return ("yl_layernorm_bwd", ctx, x, ldx, dy, lddy, rows, cols, eps, None, mean, rstd, add,
            ldadd, dx, lddx, None, None)


@pytest.mark.parametrize("bad,status", [
    (dict(x=None), INVALID), (dict(y=None), INVALID), (dict(rows=-1), SHAPE), (dict(cols=0), SHAPE),
    (dict(cols=(1 << 29) + 1, ldx=1 << 30, ldy=1 << 30), SHAPE), (dict(ldx=63), SHAPE), (dict(ldy=63), SHAPE), (dict(eps=-1e-5), INVALID),
    (dict(eps=float("nan")), INVALID), (dict(y=BASE + 4), INVALID),
    (dict(y=BASE, ldy=65), INVALID), (dict(y=BASE + 8 * 64 * 4 - 4), INVALID),
    (dict(ldx=100, ldy=100, y=BASE + 63 * 4), INVALID), (dict(x=BASE + 2), INVALID),
])
def test_layernorm_fwd_refuses(ctx, bad, status):
    refused(status, *fwd(ctx, **bad))


@pytest.mark.parametrize("bad,status", [
    (dict(x=None), INVALID), (dict(dy=None), INVALID), (dict(rows=-1), SHAPE),
    (dict(cols=0), SHAPE), (dict(lddy=10), SHAPE), (dict(lddx=63), SHAPE),
    (dict(add=BASE + (3 << 20), ldadd=63), SHAPE), (dict(mean=BASE), INVALID),
    (dict(rstd=BASE), INVALID), (dict(dx=BASE), INVALID), (dict(dx=BASE + (1 << 20)), INVALID),
    (dict(add=BASE + (2 << 20), ldadd=65), INVALID), (dict(dy=BASE + (1 << 20) + 1), INVALID),
])
def test_layernorm_bwd_refuses(ctx, bad, status):
    refused(status, *bwd(ctx, **bad))


def test_layernorm_fwd_refuses_results_in_other_arguments(ctx):
    c, x, ldx, rows, cols, eps, _, _, y, ldy, _, _ = fwd(ctx)[1:]
    v = BASE + (4 << 20)
    for gamma, beta, mean, rstd in (
            (y + 4, None, None, None), (None, y + 400, None, None), (None, None, y, None),
            (None, None, None, x), (None, None, v, v), (None, None, v, v + 28), (v, None, v + 252, None),
            (None, v, None, v)):
        refused(INVALID, "yl_layernorm_fwd", c, x, ldx, rows, cols, eps, gamma, beta, y, ldy, mean,
                rstd)


def test_layernorm_bwd_refuses_results_in_other_arguments(ctx):
    v, x, dy, dx = BASE + (4 << 20), BASE, BASE + (1 << 20), BASE + (2 << 20)
    for gamma, mean, rstd, dg, db in (
            (v, None, None, v, None), (v, None, None, None, v + 252), (None, v, v + 64, v + 28, None),
            (None, v, v + 64, None, v + 64), (None, None, None, x + 512, None),
            (None, None, None, None, dy), (dx, None, None, None, None), (None, dx, v, None, None),
            (None, v, dx + 8, None, None)):
        refused(INVALID, "yl_layernorm_bwd", ctx, x, 64, dy, 64, 8, 64, 1e-5, gamma, mean, rstd,
                None, 64, dx, 64, dg, db)


def test_layernorm_bwd_refuses_overlapping_results(ctx):
    g = BASE + (4 << 20)
    for dg, db in ((g, g), (g, g + 4 * 63), (BASE + (2 << 20), None), (None, BASE + (2 << 20) + 400)):
        refused(INVALID, *bwd(ctx)[:-2], dg, db)


def test_long_tables_are_checked_quickly(ctx):
    mats = [(X + i * 4096, Y + i * 4096, 16, 64, 64, 64) for i in range(3000)]
    refused(INVALID, *ns(ctx, *mats, (X, Y + 2999 * 4096 + 64, 4, 4, 4, 4)))


def test_layernorm_without_rows_needs_no_data(ctx):
    call(*fwd(ctx, x=None, y=None, rows=0))


def ns(ctx, *mats, steps=5, coeffs=None, eps=1e-7, count=None):
    table = (NsMatrix * len(mats))(*[NsMatrix(*m) for m in mats]) if mats else None
    q = (C.c_float * len(coeffs))(*coeffs) if coeffs else None
    return ("yl_newton_schulz", ctx, table, len(mats) if count is None else count, steps, q, eps)


X, Y = BASE, BASE + (1 << 24)


@pytest.mark.parametrize("mats,kw,status", [
    ([(None, Y, 4, 4, 4, 4)], {}, INVALID), ([(X, None, 4, 4, 4, 4)], {}, INVALID),
    ([(X, Y, -1, 4, 4, 4)], {}, SHAPE), ([(X, Y, 4, 65537, 65537, 65537)], {}, SHAPE),
    ([(X, Y, 4, 4, 3, 4)], {}, SHAPE), ([(X, Y, 4, 4, 4, 3)], {}, SHAPE),
    ([(X + 2, Y, 4, 4, 4, 4)], {}, INVALID), ([(X, X + 16, 4, 4, 4, 4)], {}, INVALID),
    ([(X, X, 4, 4, 4, 5)], {}, INVALID),
    ([(X, Y, 4, 4, 4, 4), (X, Y, 4, 4, 4, 4)], {}, INVALID),
    ([(X, Y, 4, 4, 4, 4), (Y, Y + 4096, 4, 4, 4, 4)], {}, INVALID),
    ([(X, Y, 4, 4, 8, 8), (X + 12, Y + 12, 4, 4, 8, 8)], {}, INVALID),
    ([(X, Y, 4, 4, 4, 4)], dict(steps=-1), INVALID), ([(X, Y, 4, 4, 4, 4)], dict(steps=33), INVALID),
    ([(X, Y, 4, 4, 4, 4)], dict(eps=-1.0), INVALID),
    ([(X, Y, 4, 4, 4, 4)], dict(steps=1, coeffs=(5.0, 0.0, 0.0)), UNSUPPORTED),
    ([(X, Y, 4, 4, 4, 4)], dict(steps=2, coeffs=(2.0, 0.0, 0.0, 2.5, 0.0, 0.0)), UNSUPPORTED),
    ([(X, Y, 4, 4, 4, 4)], dict(steps=1, coeffs=(float("inf"), 0.0, 0.0)), INVALID),
    ([], dict(count=-1), INVALID), ([], dict(count=1), INVALID),
])
def test_newton_schulz_refuses(ctx, mats, kw, status):
    refused(status, *ns(ctx, *mats, **kw))


def test_newton_schulz_with_nothing_to_do(ctx):
    call(*ns(ctx))
    call(*ns(ctx, (None, None, 0, 7, 7, 7), (None, None, 3, 0, 0, 0)))


def muon(ctx, *mats, steps=5, eps=1e-7, norm=None):
    table = (MuonTensor * len(mats))(*[MuonTensor(*m) for m in mats])
    return ("yl_muon_multi", ctx, table, len(mats), 0.02, 0.95, 1, 0.0, steps, None, eps, 1.0, 0.0,
            0, norm)


P, G, M = BASE, BASE + (1 << 24), BASE + (2 << 24)


@pytest.mark.parametrize("mats,kw,status", [
    ([(None, G, M, 4, 4, 1.0)], {}, INVALID), ([(P, None, M, 4, 4, 1.0)], {}, INVALID),
    ([(P, G, None, 4, 4, 1.0)], {}, INVALID), ([(P, G, M, 4, -4, 1.0)], {}, SHAPE),
    ([(P, G, M + 1, 4, 4, 1.0)], {}, INVALID),
    ([(P, G, M, 4, 4, 1.0), (P, G + 64, M + 64, 4, 4, 1.0)], {}, INVALID),
    ([(P, G, M, 4, 4, 1.0), (P + 64, G + 64, M + 60, 4, 4, 1.0)], {}, INVALID),
    ([(P, G, G, 4, 4, 1.0)], {}, INVALID), ([(P, P + 32, M, 4, 4, 1.0)], {}, INVALID),
    ([(P, G, M, 4, 4, 1.0)], dict(steps=40), INVALID),
    ([(P, G, M, 4, 4, 1.0)], dict(eps=float("nan")), INVALID),
    ([(P, G, M, 4, 4, 1.0)], dict(norm=P + 60), INVALID),
    ([(P, G, M, 4, 4, 1.0)], dict(norm=G), INVALID),
    ([(P, G, M, 4, 4, 1.0)], dict(norm=M + 65), INVALID),
])
def test_muon_refuses(ctx, mats, kw, status):
    refused(status, *muon(ctx, *mats, **kw))


def test_null_context():
    refused(INVALID, *fwd(None))
    refused(INVALID, *bwd(None))
    refused(INVALID, *ns(None))
    refused(INVALID, *muon(None))


def test_ops_refuse_arguments_of_other_sizes():
    x = np.zeros((3, 8), np.float32)
    for bad in (dict(gamma=np.ones(7)), dict(beta=np.ones(9)), dict(gamma=np.ones((2, 8)))):
        with pytest.raises(ValueError, match="values, not 8"):
            ops.layernorm_fwd(x, **bad)
    for bad in (dict(gamma=np.ones(4)), dict(mean=np.ones(4), rstd=np.ones(3)),
                dict(mean=np.ones(3), rstd=np.ones(2)), dict(dy=x[:2]), dict(addend=x[:, :7])):
        with pytest.raises(ValueError):
            ops.layernorm_bwd(x, **{"dy": x, **bad})
    for empty in (np.zeros((3, 0)), np.float32(1)):
        with pytest.raises(ValueError, match="no columns"):
            ops.layernorm_fwd(empty)
    with pytest.raises(ValueError, match="two axes"):
        ops.newton_schulz([x, x[0]])
    with pytest.raises(ValueError, match="two axes"):
        ops.muon_multi([x[0]], [x[0]], [x[0]], 0.1)
    with pytest.raises(ValueError, match="shapes"):
        ops.muon_multi([x], [x.T], [x], 0.1)
    with pytest.raises(ValueError, match="scales"):
        ops.muon_multi([x], [x], [x], 0.1, scales=[1.0, 2.0])
