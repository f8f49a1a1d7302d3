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


@pytest.mark.parametrize("form", FORMS, indirect=True)
@pytest.mark.parametrize("operand", ["q", "k", "v", "d_out"])
@pytest.mark.parametrize("d", [32, 80, 128])
def test_values_past_the_largest_bf16(hip, rng, form, operand, d):
    """fp32 values next to its largest one in a column of an operand whose partner holds zeros there: the scores stay ordinary, the
    column of the gradient (or output) that sums the operand itself is large and finite."""
    big = rng.uniform(3.397e38, 3.402e38, 4).astype(np.float32) * np.array([1, -1, 1, -1], np.float32)
    if operand == "v":
        big[1:] = 1          # the weighted sum before its division by the sum of weights has to be in range too: one such value
    q, k, v, table, d_out = attention_case(rng, 1, 2, 1, 40, 300, d, 8)
    # The sums have to be in range before they are scaled: the four large values of q (or k) meet dS = p (dP - delta) in dk (dq).
    # dP is a sum of d products of normal numbers, so |dP - delta| stays below 8 sqrt(d) < 91 without this factor, and four
    # |dS| below 1 with it even where p is 1 / 6; p is at most about 0.2 here (scores of standard deviation 1 / 4 and the bias).
    d_out /= 64
    arrays, partner = {"q": q, "k": k, "v": v, "d_out": d_out}, {"q": "k", "k": "q", "v": "d_out", "d_out": "v"}
    c = d - 3
    arrays[partner[operand]][..., c] = 0
    arrays[operand][0, 0, [1, 9, 20, 33], c] = big
    args = (table, None, 260, 8, 20, False, True, d ** -0.5 / 4)
    got = run_attention(hip, q, k, v, *args, d_out)
    want, bound = oc.attention(q, k, v, *args, d_out)
    for n in got:
        assert np.isfinite(got[n]).all(), n
        assert (np.abs(got[n] - want[n]) <= bound[n] + 1e-37).all(), n


@pytest.mark.parametrize("form", FORMS, indirect=True)
def test_infinite_values_end_as_nan_where_they_are_seen(hip, rng, form):
    """An infinity behind a sequence is not read; one that a query sees makes the rows it enters not finite, and no others."""
    q, k, v, table, d_out = attention_case(rng, 2, 2, 2, 9, 700, 64, 8)
    v[0, 1, 3, 5] = np.inf
    v[1, :, 650:] = np.inf
    k[1, :, 650:] = -np.inf
    got = run_attention(hip, q, k, v, table, np.array([700, 650], np.int32), 691, 8, 20, False, True, 0.125)
    assert np.isnan(got["out"][0, 1, :, 5]).all()
    got["out"][0, 1, :, 5] = 0
    assert np.isfinite(got["out"]).all() and np.isfinite(got["lse"]).all()
