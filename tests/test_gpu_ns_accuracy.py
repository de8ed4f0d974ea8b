"""Newton-Schulz against fp32 torch products on the same inputs: the mean error over
eight seeds, relative to the result's norm, both measured against float64.

An fp32 product rounds each addition; the tensor core truncates, up to eight additions
to an accumulator, which takes 2^-22 off a product of dense matrices and nothing off one
whose sums have a single term.  Half of it is put back, so either kind keeps an error of
2^-23 = 1.2e-7 of a product, always the same way, where fp32's is 2^-24 times a few of
random sign: the results end about as far off.  1.6 times is the bound (without what is
put back 1.9, with all of it 2.9 and more).  Sides of up to 128 in tiles, beside longer
matrices, meet the iteration's least stable point with it (64 x 1000: 2.7; without 3.3):
3 times."""
import ctypes as C

import numpy as np
import pytest
import torch

from yumelayers_b200._lib import MuonTensor, NsMatrix, call

pytestmark = pytest.mark.gpu
QUINTIC = (3.4445, -4.7750, 2.0315)
SHORT = [(7, 1131), (20, 64), (33, 50), (63, 64), (64, 64), (64, 65), (64, 100), (64, 1000), (50, 700),
         (65, 64), (65, 100), (65, 1000), (66, 66), (100, 1000), (128, 128), (128, 1152), (100, 300),
         (1152, 128)]
LONG = [(129, 2000), (200, 3000), (256, 256), (256, 2304), (512, 512), (300, 700), (1000, 1000),
        (2304, 256)]
SEEDS = 8


@pytest.fixture
def h(ctx):
    ctx.set_stream(torch.cuda.current_stream().cuda_stream or 1)
    tf32 = torch.backends.cuda.matmul.allow_tf32
    torch.backends.cuda.matmul.allow_tf32 = False
    yield ctx.handle
    torch.cuda.synchronize()
    torch.backends.cuda.matmul.allow_tf32 = tf32
    call("yl_debug_cluster_limit", ctx.handle, -1)
    ctx.set_stream(None)


def matrix(kind, r, c, seed):
    gen = torch.Generator(device="cuda").manual_seed(100 + seed)
    if kind == "normal":
        return torch.randn(r, c, generator=gen, device="cuda")
    x, n = torch.zeros(r, c, device="cuda"), min(r, c)
    values = torch.rand(n, generator=gen, device="cuda") + 0.1
    if kind == "diagonal":
        x[range(n), range(n)] = values
    else:  # one entry
        x[seed * 7 % r, seed * 11 % c] = values[0]
    return x


def plain(x, dtype):
    z = x.to(dtype)
    z = z.T if z.shape[0] > z.shape[1] else z
    z = z * (1.0 / (x.double().square().sum().sqrt() + 1e-7)).to(dtype)
    for _ in range(5):
        g = z @ z.T
        z = QUINTIC[0] * z + (QUINTIC[1] * g + QUINTIC[2] * (g @ g)) @ z
    return z.T if x.shape[0] > x.shape[1] else z


def off(a, b):
    return float((a.double() - b).norm() / b.norm())


def orthogonalise(h, xs):
    ys = [torch.empty_like(x) for x in xs]
    table = (NsMatrix * len(xs))(*[
        NsMatrix(x.data_ptr(), y.data_ptr(), *x.shape, x.shape[1], x.shape[1])
        for x, y in zip(xs, ys)])
    call("yl_newton_schulz", h, table, len(xs), 5, None, C.c_float(1e-7))
    return ys


def ratio(h, kind, shape):
    ours, fp32 = [], []
    for seed in range(SEEDS):
        x = matrix(kind, *shape, seed)
        want = plain(x, torch.float64)
        ours.append(off(orthogonalise(h, [x])[0], want))
        fp32.append(off(plain(x, torch.float32), want))
    return float(np.mean(ours) / np.mean(fp32))


@pytest.mark.parametrize("kind", ["normal", "diagonal", "one"])
@pytest.mark.parametrize("shape", SHORT + LONG)
def test_mean_error_is_that_of_fp32_products(h, kind, shape):
    assert ratio(h, kind, shape) < 1.6


@pytest.mark.parametrize("kind", ["normal", "diagonal", "one"])
@pytest.mark.parametrize("shape", SHORT)
def test_short_sides_in_tiles(h, kind, shape):
    """As beside longer matrices: the form that keeps X on the chip is put aside."""
    call("yl_debug_cluster_limit", h, 0)
    assert ratio(h, kind, shape) < 3.0


# square and mixed tables; the forms they run in: on the chip, tiles of 64 and 128
# columns, pairs of blocks
TABLES = [[(64, 64), (100, 100), (128, 128), (17, 17)], [(300, 300)], [(700, 700), (129, 129)],
          [(1500, 1500)] * 2, [(1030, 1000)] * 14 + [(64, 700)], [(2560, 2500)] * 2, SHORT + LONG]


@pytest.mark.parametrize("shapes", TABLES, ids=lambda t: "%dx%d of %d" % (*t[0], len(t)))
def test_every_matrix_of_a_table(h, shapes):
    """Square matrices have small singular values, which magnify what a first step loses in
    every arithmetic: so against fp32 products of the same matrix, one by one.  Single
    errors scatter about their mean: twice the bound of the means."""
    xs = [matrix("normal", *s, k) for k, s in enumerate(shapes)]
    for x, y in zip(xs, orthogonalise(h, xs)):
        want = plain(x, torch.float64)
        bound = 1.6 if min(x.shape) > 128 or max(map(min, shapes)) <= 128 else 3.0
        assert off(y, want) < 2 * bound * off(plain(x, torch.float32), want)


@pytest.mark.parametrize("nesterov", [1, 0])
def test_muon_step_of_a_table(h, nesterov):
    """The parameters' own roundings are 1.5 of 2^-24 against their values; weights of zero
    leave the update alone to be seen."""
    shapes = SHORT + LONG
    zero = [torch.zeros(s, device="cuda") for s in shapes]
    g, m = ([matrix("normal", *s, k + o) for k, s in enumerate(shapes)] for o in (0, 50))
    m0 = [t.clone() for t in m]
    table = (MuonTensor * len(shapes))(*[
        MuonTensor(p.data_ptr(), a.data_ptr(), b.data_ptr(), *s, 1.0)
        for p, a, b, s in zip(zero, g, m, shapes)])
    call("yl_muon_multi", h, table, len(shapes), 1.0, 0.5, nesterov, 0.0, 5, None, 1e-7, 1.0, 0.0, 0, None)
    for p, a, b in zip(zero, g, m0):
        b = 0.5 * b + a  # exact products; one rounding of the sum, as in the kernel
        u = a + 0.5 * b if nesterov else b
        want = -plain(u, torch.float64)
        bound = 1.6 if min(p.shape) > 128 else 3.0
        assert off(p, want) < 2 * bound * off(-plain(u, torch.float32), want) + 2.0 ** -23
