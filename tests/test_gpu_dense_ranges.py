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
