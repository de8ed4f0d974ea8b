"""The on-chip form where clusters of 16 blocks find no room, as in a part of a device:
the same calls with smaller clusters, and in the kernel in memory where the matrix is
too long for them.  Tolerance: 2e-5, as in the Newton-Schulz tests."""
import pytest

from test_gpu_muon import TOL, h, normal, ns64, rel, run_ns  # noqa: F401
from yumelayers_b200._lib import YumeError, call

pytestmark = pytest.mark.gpu
SHAPES = [(128, 1152), (1152, 128), (64, 2000), (60, 6144), (3000, 40), (100, 3000), (33, 50), (5, 1)]


@pytest.mark.parametrize("limit", [-1, 16, 8, 4, 2, 1, 0])
def test_smaller_clusters(h, ctx, limit):  # noqa: F811
    xs = [normal(i, *s) for i, s in enumerate(SHAPES)]
    call("yl_debug_cluster_limit", ctx.handle, limit)
    try:
        for x in xs:
            assert rel(run_ns(h, [x])[0], ns64(x)) < TOL
        for got, x in zip(run_ns(h, xs), xs):
            assert rel(got, ns64(x)) < TOL
        ctx.check_device_errors()
    finally:
        call("yl_debug_cluster_limit", ctx.handle, -1)


def test_refused_limits(ctx):
    for limit in (-2, 3, 12, 17, 32):
        with pytest.raises(YumeError):
            call("yl_debug_cluster_limit", ctx.handle, limit)
    with pytest.raises(YumeError):
        call("yl_debug_cluster_limit", None, 8)
