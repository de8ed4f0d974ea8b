"""LayerNorm of rows far from size one: what fp32's squares hold keeps its accuracy,
what they do not hold is NaN and never a value.

Scaling a row by a power of two scales its mean by it, its 1 / sqrt(var) by the
inverse, and leaves y alone where eps is next to nothing, so the bounds are those of
rows of size one: 1e-6 for y and the statistics, 2e-6 for dx, 4e-6 for the sums (the
roundings counted in the LayerNorm tests), relative to the float64 formulas."""
import numpy as np
import pytest
import torch

from test_gpu_layernorm import TOL_DX, TOL_SUM, TOL_Y, bwd64, fwd64, h, p, rel  # noqa: F401
from yumelayers_b200._lib import call

pytestmark = pytest.mark.gpu

# groups of lanes, blocks, wide rows, and rows past 16384 columns; 16-byte rows and others
COLS = [4, 7, 24, 100, 128, 333, 1000, 1021, 2048, 2050, 6000, 16384, 16001, 16388, 20001]
LONG = 16384  # rows of more columns are summed in double


def calls(h, x, dy, ga, be, eps):  # noqa: F811
    rows, cols = x.shape
    xd, dyd, gd, bd = (torch.from_numpy(a).cuda() for a in (x, dy, ga, be))
    y, mean, rstd = torch.empty_like(xd), torch.empty(rows, device="cuda"), torch.empty(rows, device="cuda")
    call("yl_layernorm_fwd", h, p(xd), cols, rows, cols, eps, p(gd), p(bd), p(y), cols, p(mean), p(rstd))
    back = []
    for given in (True, False):
        dx = torch.empty_like(xd)
        dg, db = torch.empty(cols, device="cuda"), torch.empty(cols, device="cuda")
        call("yl_layernorm_bwd", h, p(xd), cols, p(dyd), cols, rows, cols, eps, p(gd),
             p(mean) if given else None, p(rstd) if given else None, None, 0, p(dx), cols, p(dg), p(db))
        back.append((dx, dg, db))
    return [t.double().cpu().numpy() for t in (y, mean, rstd)], [
        [t.double().cpu().numpy() for t in b] for b in back]


def check(h, x, dy, ga, be, eps):  # noqa: F811
    (y, mean, rstd), back = calls(h, x, dy, ga, be, eps)
    yr, mr, rr = fwd64(x, ga, be, eps)
    for r in range(len(x)):
        assert rel(y[r], yr[r]) < TOL_Y, r
        assert abs(rstd[r] - rr[r]) < TOL_Y * rr[r], r
        assert abs(mean[r] - mr[r]) < 1e-6 * (abs(mr[r]) + np.abs(x[r]).mean(dtype=np.float64)), r
    dxr, dgr, dbr = bwd64(x, dy, ga, eps)
    terms = np.linalg.norm(np.sqrt((dy.astype(np.float64) ** 2).sum(0)))
    for dx, dg, db in back:
        for r in range(len(x)):
            assert np.linalg.norm(dx[r] - dxr[r]) < TOL_DX * rr[r] * np.linalg.norm(dy[r] * ga), r
        assert np.linalg.norm(dg - dgr) < TOL_SUM * terms
        assert np.linalg.norm(db - dbr) < TOL_SUM * terms


def rows_of(sizes, cols):
    rng = np.random.default_rng(cols)
    rows = 2 * len(sizes) + 1
    unit = lambda *s: np.clip(rng.standard_normal(s), -6, 6)  # noqa: E731
    x = (unit(rows, cols) + 0.4) * np.resize(np.asarray(sizes), rows)[:, None]
    return (x.astype(np.float32), unit(rows, cols).astype(np.float32),
            (1 + 0.1 * unit(cols)).astype(np.float32), (0.1 * unit(cols)).astype(np.float32))


@pytest.mark.parametrize("cols", COLS)
@pytest.mark.parametrize("sizes,eps", [((1.0, 1e5, 1e10, 1e15, 1e16), 1e-5),
                                       ((1.0, 1e-5, 1e-10, 1e-15), 0.0),
                                       ((1e10, 1.0, 1e-10, 1e-15, 1e-17), 1e-30)])
def test_rows_of_many_sizes(h, cols, sizes, eps):  # noqa: F811
    """Squares up to 37e32 times 20001 and down to 1e-34: all inside fp32's normal range."""
    check(h, *rows_of(sizes, cols), float(np.float32(eps)))


@pytest.mark.parametrize("cols", [c for c in COLS if c > LONG])
def test_long_rows_of_every_size(h, cols):  # noqa: F811
    check(h, *rows_of((1.0, 1e20, 1e25, 1e30, 2.0 ** 122), cols), float(np.float32(1e-5)))
    check(h, *rows_of((1.0, 1e-20, 1e-25, 1e-30), cols), 0.0)


@pytest.mark.parametrize("cols", COLS)
def test_rows_past_the_range_are_nan(h, cols):  # noqa: F811
    """Every other row is one of: squares past the range, a sum past the range, one large
    value among others, differences past the range, a NaN or an infinity beside large values,
    both infinities.  The rows between them are as without them, bit by bit."""
    x = np.random.default_rng(cols).standard_normal((15, cols)).astype(np.float32)
    one, zero = np.ones(cols, np.float32), np.zeros(cols, np.float32)
    clean, clean_back = calls(h, x, x, one, zero, 1e-5)
    bad = x.copy()
    bad[1] *= np.float32(1e25)
    bad[3] = 3e38
    bad[3, 0] = 1e38
    bad[5, cols // 2] = -1e25
    bad[7, :] = -3.4e38
    bad[7, 0] = 3.4e38
    bad[9] *= np.float32(1e30)
    bad[9, -1] = np.nan
    bad[11] *= np.float32(1e30)
    bad[11, cols // 2] = np.inf
    bad[13, 0], bad[13, -1] = np.inf, -np.inf
    got, back = calls(h, bad, x, one, zero, 1e-5)
    for a, b in zip(got, clean):
        assert np.array_equal(a[::2], b[::2])
    nan = [7, 9, 11, 13] if cols > LONG else [1, 3, 5, 7, 9, 11, 13]
    assert np.isnan(got[0][nan]).all() and np.isnan(got[2][nan]).all()
    if cols > LONG:
        yr, _, _ = fwd64(bad[1:6:2], one, zero, 1e-5)
        assert rel(got[0][1:6:2], yr) < TOL_Y
    for (dx, dg, _), (clean_dx, _, _) in zip(back, clean_back):
        assert np.isnan(dx[nan]).all() and np.array_equal(dx[::2], clean_dx[::2])
        assert np.isnan(dg).all()
