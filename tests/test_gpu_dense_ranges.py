"""The dense product's epilogue over the range of its activation, and products that are not finite."""
import numpy as np
import pytest
import torch

import operator_cases as oc
from test_gpu_operators import _release_device_arrays, dev, ptr, run_product  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("variant", [0, 1, 2, 3, 4])
@pytest.mark.parametrize("lo,hi", [(-6, 6), (-1e-3, 1e-3), (0.5, 1.5), (-40, 40)])
def test_gelu_over_its_range(hip, variant, lo, hi):
    """A product without a contraction is its bias: GELU of a dense sweep.

    y = z (1 + erf(t)) / 2, t = z / sqrt 2.  The erf is off by 1.5e-7 (the polynomial's fp32 evaluation 9.1e-8, the hardware
    exponential one step of [1/2, 1), 6e-8), t by 2^-23 relative (t erf'(t) is at most 0.49), 1 + erf by 2^-24, the product by
    2^-24 of itself: together |z| (7.5e-8 + 2.9e-8 + 3e-8 + 6e-8)."""
    z = np.linspace(lo, hi, 1 << 17).astype(np.float32)
    n = z.size
    out, bias = dev(hip, np.full(n, np.nan, np.float32)), dev(hip, z)
    hip.check(hip.bh_gemm_epilogue_force(variant, 0))
    try:
        hip.check(hip.bh_gemm_epilogue(0, 0, 1, n, 0, None, 0, None, n, ptr(out), n, ptr(bias), oc.ACTS["gelu"], None, 0, None, 0))
    finally:
        hip.check(hip.bh_gemm_epilogue_force(-1, 0))
    z64 = z.astype(np.float64)
    want = 0.5 * z64 * torch.special.erfc(torch.from_numpy(-z64 * 0.5 ** 0.5)).numpy()
    assert (np.abs(out.numpy() - want) <= 1.95e-7 * np.abs(z64)).all()


@pytest.mark.parametrize("variant,splits", [(0, 1), (1, 1), (2, 1), (3, 1), (4, 1), (1, 3)])
@pytest.mark.parametrize("k", [7, 8, 9, 333])
def test_sums_that_are_not_finite(hip, rng, variant, splits, k):
    """Infinities and NaN at both ends of the contraction and of the eight that are read at a time, and sums that overflow."""
    a, b = rng.standard_normal((40, k)).astype(np.float32), rng.standard_normal((k, 36)).astype(np.float32)
    last = k - 1
    a[1, 0], a[2, last], a[3, k // 2] = np.inf, -np.inf, np.nan
    a[4, 0], a[4, last] = np.inf, np.inf                  # infinities of one sign, or of two that make NaN
    b[0, 7], b[last, 8] = np.nan, np.inf
    a[10], b[:, 20] = 3e38, 10.0                          # an infinity by overflow
    hip.check(hip.bh_gemm_epilogue_force(variant, splits))
    try:
        for ta, tb in ((0, 0), (1, 0), (0, 1), (1, 1)):
            y, _ = run_product(hip, a, b, ta, tb, "none", None, None, False, pad=1)
            with np.errstate(all="ignore"):
                want = np.zeros((40, 36), np.float32)
                for i in range(k):                        # in order, as fp32 arithmetic
                    want += a[:, i:i + 1] * b[i:i + 1]
            other = np.ones(40, bool)
            other[10] = False                             # its sums may overflow in one order and not in another
            assert np.array_equal(np.isnan(y[other]), np.isnan(want[other])) and np.array_equal(np.isinf(y[other]), np.isinf(want[other]))
            hit = np.isinf(want) & other[:, None]
            assert np.array_equal(y[hit], want[hit])
            assert np.isposinf(y[10, 20]) and not np.isfinite(y[10, 7])
    finally:
        hip.check(hip.bh_gemm_epilogue_force(-1, 0))


def test_a_diverged_matrix_takes_no_longer_than_a_few_others(hip, rng):
    """Every operand NaN: each of the 8 M sums is looked at again, which ends with its first terms."""
    import time
    m, n, k = 4096, 2048, 1024
    a, b, c = dev(hip, rng.standard_normal((m, k)).astype(np.float32)), dev(hip, rng.standard_normal((k, n)).astype(np.float32)), hip.empty((m, n))
    bad = dev(hip, np.full((m, k), np.nan, np.float32))

    def best(x):
        times = []
        for _ in range(5):
            hip.check(hip.bh_synchronize())
            start = time.perf_counter()
            hip.check(hip.bh_gemm_epilogue(0, 0, m, n, k, ptr(x), k, ptr(b), n, ptr(c), n, None, -1, None, 0, None, 0))
            hip.check(hip.bh_synchronize())
            times.append(time.perf_counter() - start)
        return min(times)
    usual = best(a)
    assert np.isfinite(c.numpy()).all()
    assert best(bad) < 15 * usual and np.isnan(c.numpy()).all()
