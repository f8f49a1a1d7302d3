"""Relative-bias attention of a padded batch whose queries are each sequence's last tokens: a decoder's step over a ragged cache."""
import ctypes as C

import numpy as np
import pytest

import operator_cases as oc
from test_gpu_operators import _release_device_arrays, attention_case, dev, ptr  # noqa: F401

pytestmark = pytest.mark.gpu

LENS = [300, 128, 1, 0, 33, 299, 500]


def run(hip, q, k, v, table, lens, offset, distance, both, causal, scale, at_end, d_out=None):
    strides = [(a.shape[1] * a.shape[2] * a.shape[3], a.shape[2] * a.shape[3], a.shape[3]) for a in (q, k)]
    plan = hip.relbias_attention(batch=q.shape[0], heads=q.shape[1], kv_heads=k.shape[1], sq=q.shape[2], sk=k.shape[2], d=q.shape[3],
                                 q_stride=strides[0], k_stride=strides[1], v_stride=strides[1], o_stride=strides[0], query_offset=offset,
                                 num_buckets=table.shape[0], max_distance=distance, bidirectional=int(both), causal=int(causal), scale=scale,
                                 queries_at_end=int(at_end))
    a = [dev(hip, x) for x in (q, k, v, table, None if lens is None else np.asarray(lens, np.int32))]
    out, lse = (dev(hip, np.full(s, np.nan, np.float32)) for s in (q.shape, q.shape[:3]))
    hip.check(hip.bh_relbias_attention_forward(plan, *map(ptr, a), ptr(out), ptr(lse)))
    got = {"out": out.numpy(), "lse": lse.numpy()}
    if d_out is not None:
        g = [dev(hip, np.full(x.shape, np.nan, np.float32)) for x in (q, k, v, table)]
        hip.check(hip.bh_relbias_attention_backward(plan, *map(ptr, a), ptr(out), ptr(lse), ptr(dev(hip, d_out)), *map(ptr, g), 0))
        got.update({n: x.numpy() for n, x in zip(("dq", "dk", "dv", "dtable"), g)})
    return got


def expected(q, k, v, table, lens, offset, distance, both, causal, scale, d_out):
    """sequence by sequence, each at its own position"""
    want, bound = None, None
    for b, n in enumerate(lens):
        n = min(max(n, 0), k.shape[2])
        one = [x[b:b + 1] for x in (q, k, v)]
        w, e = oc.attention(*one, table, np.array([n]), n - q.shape[2] + offset, table.shape[0], distance, both, causal, scale, d_out[b:b + 1])
        if want is None:
            want, bound = {x: [y] for x, y in w.items()}, {x: [y] for x, y in e.items()}
        else:
            for x in w:
                want[x].append(w[x])
                bound[x].append(e[x])
    join = lambda d: {x: sum(y) if x == "dtable" else np.concatenate(y) for x, y in d.items()}  # noqa: E731
    return join(want), join(bound)


@pytest.mark.parametrize("rows", [0, 1])
@pytest.mark.parametrize("splits", [0, 1, 3])
@pytest.mark.parametrize("sq,offset", [(1, 0), (5, 0), (40, 0), (130, 0), (7, 3), (7, -20)])
@pytest.mark.parametrize("causal", [True, False])
def test_last_tokens_of_a_padded_batch(hip, rng, rows, splits, sq, offset, causal):
    q, k, v, table, d_out = attention_case(rng, len(LENS), 4, 2, sq, 300, 48, 16)
    args = (LENS, offset, 60, not causal, causal, 48 ** -0.5)
    want, bound = expected(q, k, v, table, *args, d_out)
    for b, n in enumerate(LENS):                          # what lies behind a sequence is not read
        k[b, :, n:], v[b, :, n:] = np.nan, np.inf
    hip.check(hip.bh_relbias_attention_force_rows(rows))
    hip.check(hip.bh_relbias_attention_force_splits(splits))
    try:
        got = run(hip, q, k, v, table, *args, True, d_out)
    finally:
        hip.check(hip.bh_relbias_attention_force_rows(-1))
        hip.check(hip.bh_relbias_attention_force_splits(0))
    assert np.array_equal(np.isneginf(got["lse"]), np.isneginf(want["lse"]))
    for n in got:
        live = np.isfinite(want[n])
        assert (np.abs(got[n][live] - want[n][live]) <= bound[n][live] + 1e-37).all(), n


@pytest.mark.parametrize("sq", [1, 200])
def test_sequences_of_full_length_stand_where_the_offset_says(hip, rng, sq):
    q, k, v, table, d_out = attention_case(rng, 2, 2, 2, sq, 250, 64, 16)
    ends = run(hip, q, k, v, table, None, 0, 60, False, True, 0.125, True, d_out)
    told = run(hip, q, k, v, table, None, 250 - sq, 60, False, True, 0.125, False, d_out)
    for n in ends:
        assert np.array_equal(ends[n], told[n]), n


def test_on_the_tape(boat, rng):
    import boat_amd.capi as capi
    boat.boat_clear_error()
    lens = [50, 9, 33]
    q, k, v, table, _ = attention_case(rng, 3, 4, 2, 6, 50, 16, 8)
    ones = np.ones_like(q)
    want, bound = expected(q, k, v, table, lens, 0, 20, False, True, 0.25, ones)
    plan = capi.RelativeAttentionConfig(8, 20, False, True, 0, 0.25, True)
    swap = lambda a: np.ascontiguousarray(a.transpose(0, 2, 1, 3))  # noqa: E731
    made = [boat.tensor(a) for a in (swap(q), swap(k), swap(v), table, np.array(lens, np.int32))]
    eager = boat.boat_hip_relative_attention(C.byref(plan), *made, None)
    xs = [boat.boat_variable_create(t, True) for t in made[:4]]
    out = boat.boat_hip_var_relative_attention(C.byref(plan), *xs, made[4])
    assert np.array_equal(boat.numpy(eager), boat.numpy(boat.boat_variable_data(out)))
    assert (np.abs(swap(boat.numpy(eager)) - want["out"]) <= bound["out"]).all()
    boat.boat_variable_backward_full(out)
    for n, x in zip(("dq", "dk", "dv"), xs):
        assert (np.abs(swap(boat.numpy(boat.boat_variable_grad(x))) - want[n]) <= bound[n] + 1e-37).all(), n
    assert (np.abs(boat.numpy(boat.boat_variable_grad(xs[3])) - want["dtable"]) <= bound["dtable"] + 1e-37).all()
    for x in [out, *xs]:
        boat.boat_variable_free(x)
    for t in [eager, *made]:
        boat.boat_tensor_unref(t)
    assert not boat.boat_has_error()


@pytest.mark.parametrize("rows", [0, 1])
def test_keys_that_all_sequences_share(hip, rng, rows):
    """A stride of zero over the batch (one prompt for all) or over the key heads, read but never written."""
    q, k, v, table, _ = attention_case(rng, 3, 4, 2, 20, 150, 48, 16)
    for axis in (0, 1):
        one = [np.ascontiguousarray(np.take(x, [0], axis)) for x in (k, v)]
        ks = [one[0].shape[1] * 150 * 48, 150 * 48, 48]
        ks[axis] = 0
        plan = hip.relbias_attention(batch=3, heads=4, kv_heads=2, sq=20, sk=150, d=48, q_stride=(4 * 20 * 48, 20 * 48, 48), k_stride=ks, v_stride=ks,
                                     o_stride=(4 * 20 * 48, 20 * 48, 48), query_offset=130, num_buckets=16, max_distance=60, bidirectional=0, causal=1,
                                     scale=0.125)
        out, lse = dev(hip, np.full(q.shape, np.nan, np.float32)), dev(hip, np.full(q.shape[:3], np.nan, np.float32))
        hip.check(hip.bh_relbias_attention_force_rows(rows))
        try:
            hip.check(hip.bh_relbias_attention_forward(plan, ptr(dev(hip, q)), *(ptr(dev(hip, x)) for x in one), ptr(dev(hip, table)), None, ptr(out), ptr(lse)))
        finally:
            hip.check(hip.bh_relbias_attention_force_rows(-1))
        want, bound = oc.attention(q, *(np.repeat(x, k.shape[axis], axis) for x in one), table, None, 130, 16, 60, False, True, 0.125)
        assert (np.abs(out.numpy() - want["out"]) <= bound["out"]).all() and (np.abs(lse.numpy() - want["lse"]) <= bound["lse"]).all()
