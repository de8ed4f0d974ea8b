"""One context's workspace under a stream handle that is given out again: calls on
new streams behind destroyed ones with work left."""
import ctypes as C

import numpy as np
import pytest
import torch

from yumelayers_b200._lib import NsMatrix, call
from yumelayers_b200.session import Context

pytestmark = pytest.mark.gpu


@pytest.fixture
def own():
    c = Context(0)
    yield c
    torch.cuda.synchronize()
    call("yl_ctx_destroy", c.handle)


def matrices(seeds, r, c):
    xs = [torch.from_numpy(np.random.default_rng(s).standard_normal((r, c)).astype(np.float32)).cuda()
          for s in seeds]
    return xs, [torch.empty_like(x) for x in xs]


def orthogonalise(ctx, x, y):
    r, c = x.shape
    table = (NsMatrix * 1)(NsMatrix(x.data_ptr(), y.data_ptr(), r, c, c, c))
    call("yl_newton_schulz", ctx.handle, table, 1, 5, None, 1e-7)


def test_streams_destroyed_with_work_left(own):
    xs, ys = matrices(range(10, 18), 600, 900)
    want = []
    for x, y in zip(xs, ys):
        orthogonalise(own, x, y)
        torch.cuda.synchronize()
        want.append(y.clone())
        y.zero_()
    torch.cuda.synchronize()
    rt = torch.cuda.cudart()
    handles = set()
    for x, y in zip(xs, ys):
        s = C.c_void_p()
        assert int(rt.cudaStreamCreate(C.addressof(s))) == 0
        handles.add(s.value)
        own.set_stream(s.value)
        orthogonalise(own, x, y)
        own.set_stream(None)
        assert int(rt.cudaStreamDestroy(s.value)) == 0
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, ys)), handles
