"""Calls that the documentation allows and that are easy to forget: arrays without
rows or matrices, a context whose first call of all is captured into a graph, one
replayed while its context works on something larger."""
import ctypes as C

import numpy as np
import pytest
import torch

from yumelayers_b200 import ops
from yumelayers_b200._lib import NsMatrix, call
from yumelayers_b200.session import Context

pytestmark = pytest.mark.gpu


def test_arrays_without_rows(ctx):
    y, mean, rstd = ops.layernorm_fwd(np.zeros((0, 8), np.float32))
    assert y.shape == (0, 8) and mean.shape == (0,) and rstd.shape == (0,)
    x = np.zeros((2, 0, 8), np.float32)
    dx, dg, db = ops.layernorm_bwd(x, x, np.ones(8))
    assert dx.shape == x.shape and not dg.any() and not db.any()


def test_a_muon_step_of_no_matrices(ctx):
    assert ops.muon_multi([], [], [], 0.1) == ([], [], 0.0)
    p, m, norm = ops.muon_multi([np.zeros((0, 4))], [np.zeros((0, 4))], [np.zeros((0, 4))], 0.1,
                                clip_max_norm=1.0)
    assert p[0].shape == (0, 4) and m[0].shape == (0, 4) and norm == 0.0


@pytest.mark.parametrize("shapes", [[(128, 1152)], [(300, 500), (64, 64)], [(2560, 2500)] * 2],
                         ids=["on chip", "tiles", "pairs"])
def test_the_first_call_of_a_context_may_be_captured(ctx, shapes):
    gen = torch.Generator(device="cuda").manual_seed(1)
    xs = [torch.randn(s, generator=gen, device="cuda") for s in shapes]
    dy = torch.randn(xs[0].shape, generator=gen, device="cuda")
    rows, cols = xs[0].shape

    def run(c, ys, dx, dg):
        table = (NsMatrix * len(xs))(*[
            NsMatrix(x.data_ptr(), y.data_ptr(), *x.shape, x.shape[1], x.shape[1])
            for x, y in zip(xs, ys)])
        call("yl_newton_schulz", c.handle, table, len(xs), 5, None, 1e-7)
        p = lambda t: C.c_void_p(t.data_ptr())  # noqa: E731
        call("yl_layernorm_bwd", c.handle, p(xs[0]), cols, p(dy), cols, rows, cols, 1e-5, None, None,
             None, None, 0, p(dx), cols, p(dg), None)

    want = [torch.empty_like(x) for x in xs], torch.empty_like(dy), torch.empty(cols, device="cuda")
    got = [torch.empty_like(x) for x in xs], torch.empty_like(dy), torch.empty(cols, device="cuda")
    torch.cuda.synchronize()
    run(ctx, *want)
    torch.cuda.synchronize()
    fresh = Context(0)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        fresh.set_stream(torch.cuda.current_stream().cuda_stream)
        run(fresh, *got)
    fresh.set_stream(None)
    big = torch.randn(3000, 3000, device="cuda")
    out = torch.empty_like(big)
    torch.cuda.synchronize()
    for _ in range(3):
        graph.replay()
        table = (NsMatrix * 1)(NsMatrix(big.data_ptr(), out.data_ptr(), 3000, 3000, 3000, 3000))
        call("yl_newton_schulz", fresh.handle, table, 1, 1, None, 1e-7)
    torch.cuda.synchronize()
    fresh.check_device_errors()
    for a, b in zip([*want[0], *want[1:]], [*got[0], *got[1:]]):
        assert torch.equal(a, b)
    del graph
    torch.cuda.synchronize()
    call("yl_ctx_destroy", fresh.handle)
