"""Relative-bias attention where operands are not finite or lie at the ends of fp32's range, in every form of the kernels."""
import numpy as np
import pytest

import operator_cases as oc
from test_gpu_operators import _release_device_arrays, attention_case, run_attention  # noqa: F401

pytestmark = pytest.mark.gpu

FORMS = [(0, 1), (0, 3), (1, 1), (1, 3)]          # (kernel for few rows, parts of the keys)


@pytest.fixture
def form(hip, request):
    rows, splits = request.param
    hip.check(hip.bh_relbias_attention_force_rows(rows))
    hip.check(hip.bh_relbias_attention_force_splits(splits))
    yield request.param
    hip.check(hip.bh_relbias_attention_force_rows(-1))
    hip.check(hip.bh_relbias_attention_force_splits(0))


@pytest.mark.parametrize("form", FORMS, indirect=True)
@pytest.mark.parametrize("d", [32, 80, 128])
def test_nan_is_not_hidden(hip, rng, form, d):
    """A query of NaN, a table entry of NaN that all of a row's keys meet, a sequence of NaN keys: their rows are NaN, the others are not."""
    for spoilt in ("query", "table", "keys"):
        q, k, v, table, d_out = attention_case(rng, 2, 2, 2, 9, 700, d, 8)
        bad = np.zeros(q.shape[:3], bool)
        if spoilt == "query":
            q[1, 0, 4, d // 2] = np.nan
            bad[1, 0, 4] = True
        elif spoilt == "table":
            table[:, 1] = np.nan
            bad[:, 1] = True
        else:
            k[0, 1] = np.nan
            bad[0, 1] = True
        got = run_attention(hip, q, k, v, table, None, 691, 8, 20, False, True, d ** -0.5, d_out)
        assert np.isnan(got["lse"][bad]).all() and np.isfinite(got["lse"][~bad]).all(), spoilt
        assert np.isnan(got["out"][bad]).all() and np.isfinite(got["out"][~bad]).all(), spoilt
        assert np.isnan(got["dq"][bad]).all() and np.isfinite(got["dq"][~bad]).all(), spoilt
