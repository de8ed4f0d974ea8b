"""Which coefficients the Newton-Schulz entry points take: the checks come before
the first device call, so they run without a GPU.  A negative eps, which is looked
at behind them, ends every call there."""
import ctypes as C

import numpy as np
import pytest

from yumelayers_b200._lib import NsMatrix, YumeError, call

INVALID, UNSUPPORTED = 7, 8
BASE = 0x7F0000000000  # stands for device memory; never dereferenced


def refused(*coeffs):
    """Whether these steps are refused as letting singular values grow too far."""
    flat = [v for step in coeffs for v in step]
    table = (NsMatrix * 1)(NsMatrix(BASE, BASE + 4096, 4, 4, 4, 4))
    with pytest.raises(YumeError) as e:
        call("yl_newton_schulz", C.create_string_buffer(8192), table, 1, len(coeffs),
             (C.c_float * len(flat))(*flat), -1.0)
    assert e.value.status in (INVALID, UNSUPPORTED), e.value
    return e.value.status == UNSUPPORTED


def largest(coeffs, points=200001):
    """The largest |p(s)| of each step on a fine grid of [0, the largest so far]."""
    top, out = 1.0, []
    for a, b, c in coeffs:
        s = np.linspace(0.0, top, points)
        top = float(np.abs(s * (a + s * s * (b + s * s * c))).max())
        out.append(top)
    return out


TINY = [0.0, 1e-30, -1e-30, 1e-17, -1e-17, 1e-9, -1e-9]


@pytest.mark.parametrize("c", TINY)
def test_the_largest_value_between_the_ends(c):
    """p = a s + b s^3 has its largest value 2 a / 3 sqrt(a / (3 |b|)) inside, with any c
    next to nothing: 11.5 for (30, -30), 4.04 for (10.5, -10.5), 3.85 for (10, -10)."""
    assert refused((30.0, -30.0, c))
    assert refused((10.5, -10.5, c))
    assert not refused((10.0, -10.0, c))
    # the second step starts from that value: p(1.155) = 4.17 and 3.94
    assert refused((3.0, -3.0, c), (3.61, 0.0, c))
    assert not refused((3.0, -3.0, c), (3.41, 0.0, c))


def test_random_coefficients_against_a_grid():
    rng = np.random.default_rng(0)
    seen = {True: 0, False: 0}
    for _ in range(400):
        q = [tuple(np.float32(v) for v in rng.uniform(-6, 6, 3) * rng.choice([1.0, 1e-3, 0.0], 3))
             for _ in range(int(rng.integers(1, 3)))]
        top = max(largest([tuple(map(float, t)) for t in q]))
        if abs(top - 4.0) < 1e-3:
            continue
        seen[top > 4.0] += 1
        assert refused(*q) == (top > 4.0), (q, top)
    assert min(seen.values()) > 50, seen


def test_growth_of_small_values():
    """Small singular values may grow by 2^17 against the largest: |p(s)| <= g s with g the
    largest |a + b s^2 + c s^4|, so by the product of the g over the largest value at the
    end.  The default's g is 3.4445 and its values stay under 1.21: 9 steps 5.7e4, 10
    steps 1.9e5."""
    quintic = (3.4445, -4.7750, 2.0315)
    for steps in range(1, 33):
        assert refused(*[quintic] * steps) == (steps > 9), steps
    for steps in (1, 12, 29):  # 1.5^29 = 1.28e5, the largest value is 1
        assert not refused(*[(1.5, -0.5, 0.0)] * steps)
    assert refused(*[(1.5, -0.5, 0.0)] * 30)
    # growth that the next step takes back lets nothing grow against the largest value
    assert not refused(*[(3.9, 0.0, 0.0), (0.25, 0.0, 0.0)] * 16)
    assert not refused(*[(1.0, 0.0, 0.0)] * 32)
    # five is the most a step can do to an odd polynomial of degree five
    assert not any(refused(*[(5.0, -20.0, 16.0)] * n) for n in range(1, 8))


def test_no_growth_limit_below_seven_steps():
    rng = np.random.default_rng(1)
    for _ in range(100):
        q = []
        while len(q) < 7:
            step = rng.uniform(-5, 5, 3)
            step *= rng.uniform(0.3, 3.9) / largest(q + [tuple(step)], 2001)[-1]
            q.append(tuple(float(np.float32(v)) for v in step))
        assert not refused(*q), q


def test_the_default_coefficients_are_checked_too():
    table = (NsMatrix * 1)(NsMatrix(BASE, BASE + 4096, 4, 4, 4, 4))
    for steps, status in ((9, INVALID), (10, UNSUPPORTED), (32, UNSUPPORTED)):
        with pytest.raises(YumeError) as e:
            call("yl_newton_schulz", C.create_string_buffer(8192), table, 1, steps, None, -1.0)
        assert e.value.status == status
