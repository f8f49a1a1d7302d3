"""The fused training operators on the GPU against plain float64 forms: sizes at which tiles, segments and tails end, padded
leading dimensions, empty rows, infinities, work split over the contraction, calls in place, from two threads and twice."""
import ctypes as C
import threading

import numpy as np
import pytest

import operator_cases as oc
from oracle_lib import fp32_gemm_bound, rel_fro

pytestmark = pytest.mark.gpu

_KEEP = []


@pytest.fixture(autouse=True)
def _release_device_arrays():
    yield
    _KEEP.clear()


def dev(hip, a):
    """Uploaded and kept until the test ends."""
    if a is None:
        return None
    d = hip.to_device(np.ascontiguousarray(a))
    _KEEP.append(d)
    return d


def ptr(d, elements=0):
    return None if d is None else C.c_void_p(d.ptr + 4 * elements)


def padded(a, ld, fill=np.nan):
    """a [rows, cols] inside rows of ld floats."""
    p = np.full((a.shape[0], ld), fill, np.float32)
    p[:, :a.shape[1]] = a
    return p


# ------------------------------------------------------------------ product with epilogue

def run_product(hip, a, b, ta, tb, act, bias, residual, keep, pad=0, in_place=False):
    m, k = a.shape
    n = b.shape[1]
    sa, sb = (a.T if ta else a), (b.T if tb else b)
    lda, ldb, ldc = sa.shape[1] + pad, sb.shape[1] + pad, n + pad
    da, db = dev(hip, padded(sa, lda)), dev(hip, padded(sb, ldb))
    dr = None if residual is None else dev(hip, padded(residual, ldc, 7.0))
    dc = dr if in_place else dev(hip, np.full((m, ldc), 7.0, np.float32))
    ds = dev(hip, np.full((m, ldc), 7.0, np.float32)) if keep else None
    hip.check(hip.bh_gemm_epilogue(ta, tb, m, n, k, ptr(da), lda, ptr(db), ldb, ptr(dc), ldc, ptr(dev(hip, bias)), oc.ACTS[act],
                                   ptr(ds), ldc, ptr(dr), ldc), "bh_gemm_epilogue")
    c = dc.numpy()
    assert (c[:, n:] == 7.0).all()                   # what lies between the rows stays
    s = ds.numpy()[:, :n] if keep else None
    return c[:, :n], s


def check_product(hip, rng, m, n, k, ta, tb, act, with_bias, with_residual, keep, pad=0, in_place=False):
    a, b = rng.standard_normal((m, k)).astype(np.float32), rng.standard_normal((k, n)).astype(np.float32)
    bias = rng.standard_normal(n).astype(np.float32) if with_bias else None
    residual = rng.standard_normal((m, n)).astype(np.float32) if with_residual else None
    y, saved = run_product(hip, a, b, ta, tb, act, bias, residual, keep, pad, in_place)
    a64, b64 = a.astype(np.float64), b.astype(np.float64)
    z = a64 @ b64 + (bias if with_bias else 0)
    want = oc.act(act, z) + (residual if with_residual else 0)
    ez = oc.product_bound(a64, b64, 2 * oc.U * np.abs(z))
    # every activation's slope is at most 1.13; its own evaluation is a handful of roundings of values up to |z| + 1
    ey = 1.13 * ez + 16 * oc.U * (np.abs(z) + 1) + 2 * oc.U * np.abs(want)
    assert (np.abs(y - want) <= ey).all(), np.max(np.abs(y - want) / ey)
    if keep:
        held = z if act in ("none", "relu", "gelu") else oc.act(act, z)
        assert (np.abs(saved - held) <= ey).all()
    if k > 0 and act == "none" and not with_residual:
        assert rel_fro(y, want) <= fp32_gemm_bound(k)    # what narrower operands would fail


@pytest.mark.parametrize("variant", [0, 1, 2, 3, 4])
@pytest.mark.parametrize("ta,tb", [(0, 0), (0, 1), (1, 0), (1, 1)])
@pytest.mark.parametrize("m,n,k", [(1, 1, 1), (33, 31, 17), (129, 257, 100), (256, 128, 64), (300, 140, 523)])
def test_product_every_tile(hip, rng, variant, ta, tb, m, n, k):
    hip.check(hip.bh_gemm_epilogue_force(variant, 0))
    try:
        check_product(hip, rng, m, n, k, ta, tb, "none", False, False, False, pad=0)
        check_product(hip, rng, m, n, k, ta, tb, "gelu", True, True, True, pad=3)
    finally:
        hip.check(hip.bh_gemm_epilogue_force(-1, 0))


@pytest.mark.parametrize("act", list(oc.ACTS))
@pytest.mark.parametrize("variant", [0, 1, 2, 3, 4])
def test_product_activations(hip, rng, act, variant):
    hip.check(hip.bh_gemm_epilogue_force(variant, 0))
    try:
        check_product(hip, rng, 70, 132, 48, 0, 0, act, True, False, True, pad=4)
        check_product(hip, rng, 260, 256, 32, 0, 1, act, False, True, True)
    finally:
        hip.check(hip.bh_gemm_epilogue_force(-1, 0))


@pytest.mark.parametrize("variant,splits", [(0, 2), (0, 7), (1, 3), (2, 2), (2, 64), (3, 3), (4, 2)])
@pytest.mark.parametrize("ta,tb", [(0, 0), (0, 1), (1, 0), (1, 1)])
def test_product_split_contraction(hip, rng, variant, splits, ta, tb):
    hip.check(hip.bh_gemm_epilogue_force(variant, splits))
    try:
        check_product(hip, rng, 130, 67, 333, ta, tb, "none", True, False, False)
        check_product(hip, rng, 40, 130, 1000, ta, tb, "tanh", True, True, True, pad=1, in_place=True)
        check_product(hip, rng, 5, 3, 9, ta, tb, "relu", True, True, True)      # fewer steps than splits
    finally:
        hip.check(hip.bh_gemm_epilogue_force(-1, 0))


@pytest.mark.parametrize("m,n,k", [(1, 4096, 1024), (1, 5, 4000), (7, 1000, 784), (64, 128, 784), (500, 500, 500), (777, 513, 784), (2048, 1024, 256),
                                   (1000, 1, 300), (4100, 3, 50)])
def test_product_by_shape(hip, rng, m, n, k):
    check_product(hip, rng, m, n, k, 0, 0, "none", True, False, False)
    check_product(hip, rng, m, n, k, 1, 0, "gelu", True, True, True)
    check_product(hip, rng, m, n, k, 0, 1, "none", True, True, False, in_place=True)


def test_product_without_contraction_and_without_rows(hip, rng):
    check_product(hip, rng, 5, 6, 0, 0, 0, "sigmoid", True, True, True)
    d = dev(hip, np.full(8, 3.0, np.float32))
    hip.check(hip.bh_gemm_epilogue(0, 0, 0, 4, 4, None, 4, ptr(d), 4, ptr(d), 4, None, -1, None, 0, None, 0))
    assert (d.numpy() == 3.0).all()


@pytest.mark.parametrize("variant,splits", [(0, 0), (1, 0), (2, 0), (1, 3), (3, 0), (4, 2)])
def test_product_infinities_and_nan(hip, rng, variant, splits):
    """What is not finite comes out as fp32 arithmetic gives it; the other rows and columns are untouched by it."""
    hip.check(hip.bh_gemm_epilogue_force(variant, splits))
    try:
        a, b = rng.standard_normal((40, 70)).astype(np.float32), rng.standard_normal((70, 36)).astype(np.float32)
        a[3, 5] = np.inf
        a[7, 0] = np.nan
        b[69, 11] = -np.inf
        a[9, 9], b[9, 20] = 3.3999e38, 1e-3        # finite, but past the largest bf16
        b[:, 30] = 0
        for ta, tb in ((0, 0), (1, 0), (0, 1), (1, 1)):
            y, _ = run_product(hip, a, b, ta, tb, "none", None, None, False)
            with np.errstate(all="ignore"):
                # in fp32 a product past the largest float is an infinity before the others are added to it
                prod = a.astype(np.float64)[:, :, None] * b.astype(np.float64)[None]
                prod = np.where(np.abs(prod) > 3.4028235e38, np.sign(prod) * np.inf, prod)
                want = prod.sum(1)
            assert (np.isnan(y) == np.isnan(want)).all(), np.argwhere(np.isnan(y) != np.isnan(want))
            assert (y[np.isinf(want)] == want[np.isinf(want)]).all()
            ok = np.isfinite(want)
            assert (np.abs(y - want)[ok] <= 200 * oc.U * (np.abs(np.nan_to_num(a, posinf=0, neginf=0)).astype(np.float64)
                                                          @ np.abs(np.nan_to_num(b, posinf=0, neginf=0)) + 1e-30)[ok]).all()
    finally:
        hip.check(hip.bh_gemm_epilogue_force(-1, 0))


@pytest.mark.parametrize("scale_a,scale_b", [(1e-30, 1e30), (1e-36, 1e20), (1e18, 1e18), (1e-20, 1e-19)])
def test_product_over_the_exponent_range(hip, rng, scale_a, scale_b):
    a = (rng.standard_normal((33, 40)) * scale_a).astype(np.float32)
    b = (rng.standard_normal((40, 35)) * scale_b).astype(np.float32)
    y, _ = run_product(hip, a, b, 0, 0, "none", None, None, False)
    a64, b64 = a.astype(np.float64), b.astype(np.float64)
    # below 2^-110 a value's last part is a subnormal bf16, off by half of 2^-133 at most, against the other operand
    tail = 2.0 ** -133 * (np.abs(b64).sum(0)[None] + np.abs(a64).sum(1)[:, None]) + 2.0 ** -126
    assert (np.abs(y - a64 @ b64) <= oc.product_bound(a64, b64) + tail).all()


def test_product_twice_is_the_same_and_threads_do_not_mix(hip, rng):
    a, b = rng.standard_normal((300, 1000)).astype(np.float32), rng.standard_normal((1000, 200)).astype(np.float32)
    first = run_product(hip, a, b, 0, 0, "gelu", None, None, True)
    again = run_product(hip, a, b, 0, 0, "gelu", None, None, True)
    assert np.array_equal(first[0], again[0]) and np.array_equal(first[1], again[1])
    da, db = dev(hip, a), dev(hip, b)
    outs = [dev(hip, np.zeros((300, 200), np.float32)) for _ in range(8)]
    rcs = []

    def call(o):
        for _ in range(10):
            rcs.append(hip.bh_gemm_epilogue(0, 0, 300, 200, 1000, ptr(da), 1000, ptr(db), 200, ptr(o), 200, None, 3, None, 0, None, 0))
    threads = [threading.Thread(target=call, args=(o,)) for o in outs]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert rcs == [0] * 80
    for o in outs:
        assert np.array_equal(o.numpy(), first[0])


@pytest.mark.parametrize("act", list(oc.ACTS))
@pytest.mark.parametrize("m,k,n", [(1, 5, 3), (64, 784, 128), (333, 130, 65), (1000, 256, 300)])
def test_dense_backward(hip, rng, act, m, k, n):
    x, w = rng.standard_normal((m, k)).astype(np.float32), (rng.standard_normal((k, n)) / np.sqrt(k)).astype(np.float32)
    b, dy = rng.standard_normal(n).astype(np.float32), rng.standard_normal((m, n)).astype(np.float32)
    dx_, dw_, db_, ddy = dev(hip, x), dev(hip, w), dev(hip, b), dev(hip, dy)
    y, saved = hip.empty((m, n)), hip.empty((m, n))
    hip.check(hip.bh_gemm_epilogue(0, 0, m, n, k, ptr(dx_), k, ptr(dw_), n, ptr(y), n, ptr(db_), oc.ACTS[act], ptr(saved), n, None, 0))
    gx = dev(hip, np.full((m, k), np.nan, np.float32))
    gw, gb = dev(hip, np.full((k, n), np.nan, np.float32)), dev(hip, np.full(n, np.nan, np.float32))
    call = (oc.ACTS[act], ptr(dx_), ptr(dw_), ptr(saved), ptr(ddy), ptr(gx), ptr(gw), ptr(gb), m, k, n)
    hip.check(hip.bh_dense_act_backward(*call, 0))
    x64, w64 = x.astype(np.float64), w.astype(np.float64)
    z = x64 @ w64 + b
    dz = dy * oc.act_slope(act, z)
    # dz: the saved value's error (z's bound) times a second derivative of at most 1.2, and ten roundings; a ReLU's sign may
    # turn where z is as small as its bound
    ez = oc.product_bound(x64, w64, 2 * oc.U * np.abs(z))
    edz = np.abs(dy) * (1.2 * ez + 16 * oc.U) + (np.abs(dy) * (np.abs(z) <= ez) if act == "relu" else 0)
    ex = oc.product_bound(dz, w64.T) + edz @ np.abs(w64).T
    ew = oc.product_bound(x64.T, dz) + np.abs(x64).T @ edz
    eb = 2 * m * oc.U * np.abs(dz).sum(0) + edz.sum(0)
    first = [gx.numpy(), gw.numpy(), gb.numpy()]
    for got, want, bound in zip(first, (dz @ w64.T, x64.T @ dz, dz.sum(0)), (ex, ew, eb)):
        assert (np.abs(got - want) <= bound + 1e-30).all()
    hip.check(hip.bh_dense_act_backward(*call, 1))           # dx assigned, gw and gb added to
    assert np.array_equal(gx.numpy(), first[0])
    assert (np.abs(gw.numpy() - 2 * first[1].astype(np.float64)) <= 4 * oc.U * np.abs(first[1])).all()
    assert (np.abs(gb.numpy() - 2 * first[2].astype(np.float64)) <= 2 * eb + 4 * oc.U * np.abs(first[2])).all()
    for drop in (5, 6, 7):                                   # any of the three may be left out
        part = list(call)
        part[drop] = None
        hip.check(hip.bh_dense_act_backward(*part, 0))
    assert np.array_equal(gx.numpy(), first[0])


@pytest.mark.parametrize("variant,splits,pair", [(0, 1, 0), (1, 3, 0), (2, 1, 0), (3, 1, 0), (3, 2, 0), (4, 1, 0), (-1, 0, 1)])
@pytest.mark.parametrize("m,k,n", [(1, 1, 1), (40, 33, 70), (700, 100, 300), (270, 513, 65)])
def test_bias_gradient_with_and_without_the_weights(hip, rng, variant, splits, pair, m, k, n):
    x, w, dy = (rng.standard_normal(s).astype(np.float32) for s in ((m, k), (k, n), (m, n)))
    z = rng.standard_normal((m, n)).astype(np.float32)
    dx_, dw_, ddy, dz_ = (dev(hip, a) for a in (x, w, dy, z))
    slope = (dy * (z > 0)).astype(np.float64)
    hip.check(hip.bh_gemm_epilogue_force(variant, splits))
    hip.check(hip.bh_dense_act_backward_force(pair))
    try:
        for act, want in ((-1, dy.astype(np.float64)), (0, slope)):
            bound = 2 * m * oc.U * np.abs(want).sum(0)
            for weights in (True, False):
                gw, gb = dev(hip, np.full((k, n), np.nan, np.float32)), dev(hip, np.full(n, np.nan, np.float32))
                gx = dev(hip, np.full((m, k), np.nan, np.float32))
                call = (act, ptr(dx_), ptr(dw_), ptr(dz_), ptr(ddy), ptr(gx), ptr(gw) if weights else None, ptr(gb), m, k, n)
                hip.check(hip.bh_dense_act_backward(*call, 0))
                first = gb.numpy()
                assert (np.abs(first - want.sum(0)) <= bound).all()
                hip.check(hip.bh_dense_act_backward(*call, 1))
                assert (np.abs(gb.numpy() - 2 * first.astype(np.float64)) <= 2 * bound + 4 * oc.U * np.abs(first)).all()
                assert not weights or (np.abs(gw.numpy() - 2 * (x.T.astype(np.float64) @ want)) <=
                                       4 * oc.product_bound(x.T.astype(np.float64), want) + 1e-30).all()
    finally:
        hip.check(hip.bh_gemm_epilogue_force(-1, 0))
        hip.check(hip.bh_dense_act_backward_force(-1))


@pytest.mark.parametrize("pair", [0, 1])
@pytest.mark.parametrize("m,k,n", [(1, 1, 1), (1, 5, 3), (40, 33, 70), (333, 130, 65), (700, 260, 300)])
def test_dense_backward_in_one_launch_and_in_two(hip, rng, pair, m, k, n):
    """dx and dW of a linear layer; either may be left out, and the other keeps its bits."""
    x, w, dy = (rng.standard_normal(s).astype(np.float32) for s in ((m, k), (k, n), (m, n)))
    dx_, dw_, ddy = dev(hip, x), dev(hip, w), dev(hip, dy)
    hip.check(hip.bh_dense_act_backward_force(pair))
    try:
        gx, gw = dev(hip, np.full((m, k), np.nan, np.float32)), dev(hip, np.full((k, n), np.nan, np.float32))
        hip.check(hip.bh_dense_act_backward(-1, ptr(dx_), ptr(dw_), None, ptr(ddy), ptr(gx), ptr(gw), None, m, k, n, 0))
        alone = dev(hip, np.full((m, k), np.nan, np.float32)), dev(hip, np.full((k, n), np.nan, np.float32))
        hip.check(hip.bh_dense_act_backward(-1, None, ptr(dw_), None, ptr(ddy), ptr(alone[0]), None, None, m, k, n, 0))
        hip.check(hip.bh_dense_act_backward(-1, ptr(dx_), None, None, ptr(ddy), None, ptr(alone[1]), None, m, k, n, 0))
        assert np.array_equal(gx.numpy(), alone[0].numpy()) and np.array_equal(gw.numpy(), alone[1].numpy())
        hip.check(hip.bh_dense_act_backward(-1, ptr(dx_), ptr(dw_), None, ptr(ddy), ptr(gx), ptr(alone[1]), None, m, k, n, 1))
    finally:
        hip.check(hip.bh_dense_act_backward_force(-1))
    x64, w64, d64 = x.astype(np.float64), w.astype(np.float64), dy.astype(np.float64)
    bw = oc.product_bound(x64.T, d64)
    assert (np.abs(gx.numpy() - d64 @ w64.T) <= oc.product_bound(d64, w64.T)).all()
    assert (np.abs(gw.numpy() - x64.T @ d64) <= bw).all()
    assert (np.abs(alone[1].numpy() - 2 * (x64.T @ d64)) <= 2 * bw + 2 * oc.U * np.abs(2 * (x64.T @ d64))).all()


@pytest.mark.parametrize("act", ["sigmoid", "tanh", "gelu"])
def test_dense_backward_against_differences(hip, rng, act):
    m, k, n = 9, 20, 7
    x, w, b = rng.standard_normal((m, k)), rng.standard_normal((k, n)) / 4, rng.standard_normal(n)
    x, w, b = (t.astype(np.float32) for t in (x, w, b))
    dy = rng.standard_normal((m, n)).astype(np.float32)
    args = [dev(hip, t) for t in (x, w, b, dy)]
    y, saved, gx, gw, gb = hip.empty((m, n)), hip.empty((m, n)), hip.empty((m, k)), hip.empty((k, n)), hip.empty(n)
    hip.check(hip.bh_gemm_epilogue(0, 0, m, n, k, ptr(args[0]), k, ptr(args[1]), n, ptr(y), n, ptr(args[2]), oc.ACTS[act], ptr(saved), n, None, 0))
    hip.check(hip.bh_dense_act_backward(oc.ACTS[act], ptr(args[0]), ptr(args[1]), ptr(saved), ptr(args[3]), ptr(gx), ptr(gw), ptr(gb), m, k, n, 0))

    def loss(x, w, b):
        return float((oc.act(act, x.astype(np.float64) @ w + b) * dy).sum())
    eps = 1e-5
    for grad, at in ((gx.numpy(), 0), (gw.numpy(), 1), (gb.numpy(), 2)):
        d = rng.standard_normal(grad.shape)
        up, down = [x, w, b], [x, w, b]
        up[at], down[at] = up[at] + eps * d, down[at] - eps * d
        diff = (loss(*up) - loss(*down)) / (2 * eps)
        # differences: eps^2 of third derivatives (1e-10 times a few hundred) and 1e-16 / eps of rounding, times sum |terms|
        assert abs(float((grad * d).sum()) - diff) <= 1e-5 * float(np.abs(grad * d).sum() + 1)


def test_dense_backward_of_nothing(hip):
    gw, gb = dev(hip, np.full((3, 2), 5.0, np.float32)), dev(hip, np.full(2, 5.0, np.float32))
    hip.check(hip.bh_dense_act_backward(3, None, None, None, None, None, ptr(gw), ptr(gb), 0, 3, 2, 1))
    assert (gw.numpy() == 5.0).all() and (gb.numpy() == 5.0).all()
    hip.check(hip.bh_dense_act_backward(3, None, None, None, None, None, ptr(gw), ptr(gb), 0, 3, 2, 0))
    assert (gw.numpy() == 0).all() and (gb.numpy() == 0).all()


# ------------------------------------------------------------------ distillation

def distill_case(rng, rows, vocab, topk, labels=True):
    z = (2.5 * rng.standard_normal((rows, vocab))).astype(np.float32)
    teacher = (3 * rng.standard_normal((rows, topk))).astype(np.float32)
    index = rng.integers(0, vocab, (rows, topk)).astype(np.int32)            # repeats among them
    if topk:
        index[rng.random((rows, topk)) < 0.15] = -1
        index[rows // 2] = -1                                                # a row with nothing kept
        index[rows // 3, 0] = vocab + 3                                      # past the vocabulary: left out
        index[-1] = index[-1, 0]                                             # one entry many times over
        teacher[0, 0] = -np.inf
    lab = rng.integers(0, vocab, rows).astype(np.int32) if labels else None
    if labels:
        lab[0] = -1
        if topk and index[-1, 0] >= 0:
            lab[-1] = min(index[-1, 0], vocab - 1)                           # the label among the teacher's entries
    return z, teacher, index, lab


def run_distill(hip, z, teacher, index, labels, temperature, alpha, scale, pad=0, shift=0, in_place=False):
    rows, vocab = z.shape
    ld = vocab + pad
    flat = np.full(rows * ld + shift + 4, 9.0, np.float32)
    flat[shift:shift + rows * ld].reshape(rows, ld)[:, :vocab] = z
    dz_flat = np.full_like(flat, 9.0)
    dl = dev(hip, flat)
    dg = dl if in_place else dev(hip, dz_flat)
    row, stats, loss = hip.zeros(max(rows, 1)), hip.zeros(3 * max(rows, 1)), hip.zeros(1)
    head = (ptr(dl, shift), ld, ptr(dev(hip, teacher)), ptr(dev(hip, index)), ptr(dev(hip, labels)), rows, vocab, teacher.shape[1],
            temperature, alpha, scale)
    hip.check(hip.bh_distill_forward(*head, ptr(row), ptr(stats), ptr(loss)), "bh_distill_forward")
    forward = row.numpy()[:rows], float(loss.numpy()[0])
    seed = dev(hip, np.array([2.0], np.float32))
    if not in_place:
        hip.check(hip.bh_distill_backward(*head, ptr(stats), ptr(seed), ptr(dg, shift), ld), "bh_distill_backward")
        flat_back = dg.numpy()
    hip.check(hip.bh_distill_loss_grad(*head, ptr(row), ptr(loss), ptr(dg, shift), ld), "bh_distill_loss_grad")
    both = row.numpy()[:rows], float(loss.numpy()[0])
    out = dg.numpy()
    inner = out[shift:shift + rows * ld].reshape(rows, ld)
    assert (inner[:, vocab:] == 9.0).all() and (out[:shift] == 9.0).all() and (out[shift + rows * ld:] == 9.0).all()
    back = None if in_place else flat_back[shift:shift + rows * ld].reshape(rows, ld)[:, :vocab]
    return forward, both, inner[:, :vocab], back


def check_distill(hip, z, teacher, index, labels, temperature, alpha, pad=0, shift=0, in_place=False):
    scale = 1.0 / z.shape[0]
    want_row, want_loss, want_dz = oc.distill(z, teacher, index, labels, temperature, alpha, scale)
    tol_row, tol_dz = oc.distill_bounds(z, teacher, temperature, alpha, scale)
    (row, loss), (row2, loss2), dz, back = run_distill(hip, z, teacher, index, labels, temperature, alpha, scale, pad, shift, in_place)
    for r in (row, row2):
        assert (np.abs(r - want_row) <= tol_row + 4 * oc.U * np.abs(want_row)).all(), np.abs(r - want_row).max() / tol_row
    for l in (loss, loss2):
        assert abs(l - want_loss) <= tol_row + 4 * oc.U * abs(want_loss)
    assert (np.abs(dz - want_dz) <= tol_dz).all(), np.abs(dz - want_dz).max() / tol_dz
    if back is not None:
        assert (np.abs(back - 2 * want_dz) <= 2 * tol_dz).all()
        # a dense part that is relatively as good: far from the special places the gradient is a softmax value
        big = np.abs(want_dz) > 1e-12
        assert rel_fro(dz[big], want_dz[big]) <= 4e-6


@pytest.mark.parametrize("vocab", [1, 2, 3, 5, 64, 1000, 1024, 1025, 4096, 4099])
@pytest.mark.parametrize("rows,topk", [(1, 1), (5, 8), (300, 3)])
def test_distill_small_vocabularies(hip, rng, rows, topk, vocab):
    check_distill(hip, *distill_case(rng, rows, vocab, topk), 2.0, 0.6)


@pytest.mark.parametrize("rows,vocab,topk", [(257, 16385, 5), (256, 32771, 7), (256, 70003, 4), (3, 70003, 64), (1, 131072, 200), (37, 9001, 16),
                                             (2, 8192, 1)])
def test_distill_large_vocabularies(hip, rng, rows, vocab, topk):
    check_distill(hip, *distill_case(rng, rows, vocab, topk), 3.0, 0.8, pad=3 if rows < 100 else 0)


@pytest.mark.parametrize("rows,vocab", [(2, 900), (2, 1900), (3, 3000), (2, 6000), (2, 16000), (2, 30000), (129, 26000)])
def test_distill_most_kept_entries(hip, rng, rows, vocab):
    check_distill(hip, *distill_case(rng, rows, vocab, 4096), 2.0, 0.7)


@pytest.mark.parametrize("rows,vocab", [(1, 16387), (127, 16383), (127, 16384), (128, 16384), (70, 40003), (1, 12001)])
def test_distill_rows_in_segments_and_whole(hip, rng, rows, vocab):
    check_distill(hip, *distill_case(rng, rows, vocab, 11), 2.0, 0.7, pad=1 if rows < 100 else 0)


@pytest.mark.parametrize("temperature", [0.25, 1.0, 8.0])
@pytest.mark.parametrize("alpha", [0.0, 0.5, 1.0])
@pytest.mark.parametrize("labels", [True, False])
def test_distill_mixtures(hip, rng, temperature, alpha, labels):
    check_distill(hip, *distill_case(rng, 7, 777, 9, labels), temperature, alpha, pad=5, shift=1)


@pytest.mark.parametrize("rows,vocab", [(4, 1001), (3, 20001), (300, 2050), (256, 66000)])
def test_distill_gradient_in_place(hip, rng, rows, vocab):
    check_distill(hip, *distill_case(rng, rows, vocab, 12), 2.0, 0.5, in_place=True)


def test_distill_backward_in_place_over_segments(hip, rng):
    rows, vocab, topk = 3, 40001, 30
    z, teacher, index, labels = distill_case(rng, rows, vocab, topk)
    apart = run_distill(hip, z, teacher, index, labels, 2.0, 0.5, 1.0)
    dl, stats, loss = dev(hip, z), hip.zeros(3 * rows), hip.zeros(1)
    head = (ptr(dl), vocab, ptr(dev(hip, teacher)), ptr(dev(hip, index)), ptr(dev(hip, labels)), rows, vocab, topk, 2.0, 0.5, 1.0)
    hip.check(hip.bh_distill_forward(*head, None, ptr(stats), ptr(loss)))
    seed = dev(hip, np.array([2.0], np.float32))
    hip.check(hip.bh_distill_backward(*head, ptr(stats), ptr(seed), ptr(dl), vocab))
    assert np.array_equal(dl.numpy(), apart[3])


def test_distill_without_teacher_is_cross_entropy(hip, rng):
    z, _, _, labels = distill_case(rng, 20, 333, 1)
    check_distill(hip, z, np.zeros((20, 0), np.float32), np.zeros((20, 0), np.int32), labels, 1.0, 0.0)


@pytest.mark.parametrize("rows,vocab", [(4, 100), (2, 20000)])
def test_distill_masked_logits(hip, rng, rows, vocab):
    """A vocabulary entry masked with -inf or with the lowest float has no probability and no gradient."""
    z, teacher, index, labels = distill_case(rng, rows, vocab, 6)
    z[:, ::3] = -np.inf
    z[:, 1::3] = np.finfo(np.float32).min
    z[:, 2] = 1.0
    index = np.where(index >= 0, index - index % 3 + 2, index)
    index[index >= vocab] = 2
    labels = np.where(labels >= 0, 2, labels).astype(np.int32)
    scale = 1.0 / rows
    want_row, _, want_dz = oc.distill(z, teacher, index, labels, 2.0, 0.5, scale)
    (row, _), _, dz, _ = run_distill(hip, z, teacher, index.astype(np.int32), labels, 2.0, 0.5, scale)
    tol_row, tol_dz = oc.distill_bounds(np.where(z < -1e30, 0, z), teacher, 2.0, 0.5, scale)
    assert (np.abs(row - want_row) <= tol_row).all() and (np.abs(dz - want_dz) <= tol_dz).all()
    assert (dz[:, ::3] == 0).all() and (dz[:, 1::3] == 0).all()


def test_distill_no_rows(hip):
    loss = dev(hip, np.array([5.0], np.float32))
    hip.check(hip.bh_distill_forward(None, 10, None, None, None, 0, 10, 3, 1.0, 1.0, 1.0, None, None, ptr(loss)))
    assert loss.numpy()[0] == 0
    hip.check(hip.bh_distill_backward(None, 10, None, None, None, 0, 10, 3, 1.0, 1.0, 1.0, None, None, None, 10))


def test_distill_against_differences(hip, rng):
    rows, vocab, topk = 6, 40, 5
    z, teacher, index, labels = distill_case(rng, rows, vocab, topk)
    _, _, dz, _ = run_distill(hip, z, teacher, index, labels, 1.5, 0.4, 1.0)
    d = rng.standard_normal(z.shape)
    eps = 1e-5
    up = oc.distill(z + eps * d, teacher, index, labels, 1.5, 0.4, 1.0)[1]
    down = oc.distill(z - eps * d, teacher, index, labels, 1.5, 0.4, 1.0)[1]
    # eps^2 times third derivatives of order one, 1e-16 |loss| / eps of rounding, and the gradient's own bound
    assert abs(float((dz * d).sum()) - (up - down) / (2 * eps)) <= 1e-6 + oc.distill_bounds(z, teacher, 1.5, 0.4, 1.0)[1] * np.abs(d).sum()


def test_distill_twice_is_the_same(hip, rng):
    case = distill_case(rng, 5, 30000, 40)
    one, two = (run_distill(hip, *case, 2.0, 0.5, 0.2) for _ in range(2))
    assert np.array_equal(one[0][0], two[0][0]) and one[0][1] == two[0][1] and np.array_equal(one[2], two[2]) and np.array_equal(one[3], two[3])


# ------------------------------------------------------------------ attention with a relative position bias

def layout(a, order, pad=0, fill=np.nan):
    """a [batch, heads, rows, d] in memory in the given order of the three, each row followed by `pad` floats; the array and
    its (batch, head, row) strides in elements."""
    t = np.transpose(a, [*order, 3])
    p = np.full((*t.shape[:3], t.shape[3] + pad), fill, np.float32)
    p[..., :t.shape[3]] = t
    step = [p.shape[1] * p.shape[2] * p.shape[3], p.shape[2] * p.shape[3], p.shape[3]]
    strides = [0, 0, 0]
    for place, axis in enumerate(order):
        strides[axis] = step[place]
    return p, strides


def unlayout(p, order, d):
    back = [0, 0, 0]
    for place, axis in enumerate(order):
        back[axis] = place
    return np.transpose(p[..., :d], [*back, 3])


def run_attention(hip, q, k, v, table, lens, offset, buckets, distance, both, causal, scale, d_out=None, order=(0, 1, 2), pad=0, accumulate=None):
    d = q.shape[3]
    (pq, qs), (pk, ks), (pv, vs) = (layout(a, order, pad) for a in (q, k, v))
    po, os_ = layout(np.full(q.shape, np.nan), order, pad, 7.0)
    plan = hip.relbias_attention(batch=q.shape[0], heads=q.shape[1], kv_heads=k.shape[1], sq=q.shape[2], sk=k.shape[2], d=d, q_stride=qs,
                                 k_stride=ks, v_stride=vs, o_stride=os_, query_offset=offset, num_buckets=buckets, max_distance=distance,
                                 bidirectional=int(both), causal=int(causal), scale=scale)
    dq, dk, dv, dt, dl, do = (dev(hip, x) for x in (pq, pk, pv, table, lens, po))
    lse = dev(hip, np.full(q.shape[:3], np.nan, np.float32))
    hip.check(hip.bh_relbias_attention_forward(plan, ptr(dq), ptr(dk), ptr(dv), ptr(dt), ptr(dl), ptr(do), ptr(lse)), "forward")
    o = do.numpy()
    assert pad == 0 or (o[..., d:] == 7.0).all()
    got = {"out": unlayout(o, order, d), "lse": lse.numpy()}
    if d_out is not None:
        dd = dev(hip, layout(d_out, order, pad)[0])
        gq, gk, gv = (dev(hip, np.full_like(x, 7.0)) for x in (pq, pk, pv))
        gt = dev(hip, np.full(table.shape, np.nan, np.float32) if accumulate is None else accumulate)
        hip.check(hip.bh_relbias_attention_backward(plan, ptr(dq), ptr(dk), ptr(dv), ptr(dt), ptr(dl), ptr(do), ptr(lse), ptr(dd), ptr(gq), ptr(gk),
                                                    ptr(gv), ptr(gt), int(accumulate is not None)), "backward")
        for n, x in (("dq", gq), ("dk", gk), ("dv", gv)):
            x = x.numpy()
            assert pad == 0 or (x[..., d:] == 7.0).all()
            got[n] = unlayout(x, order, d)
        got["dtable"] = gt.numpy()
    return got


def attention_case(rng, batch, heads, kv_heads, sq, sk, d, buckets):
    f = lambda *s: rng.standard_normal(s).astype(np.float32)  # noqa: E731
    return f(batch, heads, sq, d), f(batch, kv_heads, sk, d), f(batch, kv_heads, sk, d), f(buckets, heads), f(batch, heads, sq, d)


def check_attention(hip, case, lens=None, offset=None, distance=20, both=False, causal=True, scale=None, train=True, order=(0, 1, 2), pad=0, poison=False):
    q, k, v, table, d_out = case
    offset = k.shape[2] - q.shape[2] if offset is None else offset
    scale = q.shape[3] ** -0.5 if scale is None else scale
    buckets = table.shape[0]
    lens = None if lens is None else np.asarray(lens, np.int32)
    want, bound = oc.attention(q, k, v, table, lens, offset, buckets, distance, both, causal, scale, d_out if train else None)
    if poison:       # what lies behind a sequence is not read
        for b, n in enumerate(lens):
            k[b, :, max(int(n), 0):] = np.nan
            v[b, :, max(int(n), 0):] = np.inf
    got = run_attention(hip, q, k, v, table, lens, offset, buckets, distance, both, causal, scale, d_out if train else None, order, pad)
    assert np.array_equal(np.isneginf(got["lse"]), np.isneginf(want["lse"]))
    for n in got:
        live = np.isfinite(want[n])
        off = np.abs(got[n][live] - want[n][live]) / (bound[n][live] + 1e-37)
        assert (off <= 1).all(), (n, off.max())
    return got


@pytest.mark.parametrize("rows", [0, 1])
@pytest.mark.parametrize("d", [1, 8, 32, 33, 64, 80, 96, 100, 128])
def test_attention_head_sizes(hip, rng, rows, d):
    hip.check(hip.bh_relbias_attention_force_rows(rows))
    try:
        check_attention(hip, attention_case(rng, 2, 4, 2, 37, 70, d, 8), train=rows == 0)
        check_attention(hip, attention_case(rng, 1, 2, 2, 130, 67, d, 12), both=True, causal=False, distance=40, train=rows == 0)
    finally:
        hip.check(hip.bh_relbias_attention_force_rows(-1))


@pytest.mark.parametrize("rows", [0, 1])
@pytest.mark.parametrize("sq,sk", [(1, 1), (1, 64), (1, 300), (2, 31), (31, 33), (32, 32), (33, 129), (64, 64), (65, 65), (128, 128), (129, 200), (200, 129),
                                   (5, 0), (40, 1)])
@pytest.mark.parametrize("causal", [True, False])
def test_attention_lengths(hip, rng, rows, sq, sk, causal):
    hip.check(hip.bh_relbias_attention_force_rows(rows))
    try:
        check_attention(hip, attention_case(rng, 2, 2, 1, sq, sk, 32, 16), causal=causal, both=not causal, distance=50, train=rows == 0)
    finally:
        hip.check(hip.bh_relbias_attention_force_rows(-1))


@pytest.mark.parametrize("rows", [0, 1])
def test_attention_padded_batches(hip, rng, rows):
    """Sequences of length zero, one, past a tile and beyond both ends; keys behind them hold NaN and infinities."""
    hip.check(hip.bh_relbias_attention_force_rows(rows))
    try:
        for causal in (True, False):
            got = check_attention(hip, attention_case(rng, 7, 2, 1, 45, 140, 40, 16), lens=[0, 1, 64, 65, 139, 500, -3], causal=causal, train=rows == 0,
                                  poison=True)
            assert (got["out"][0] == 0).all() and (got["out"][6] == 0).all()
            if rows == 0:
                assert (got["dk"][0] == 0).all() and (got["dv"][2, :, 64:] == 0).all() and (got["dq"][6] == 0).all()
    finally:
        hip.check(hip.bh_relbias_attention_force_rows(-1))


@pytest.mark.parametrize("rows", [0, 1])
@pytest.mark.parametrize("offset", [-60, -1, 0, 7, 300])
@pytest.mark.parametrize("causal", [True, False])
def test_attention_offsets_and_rows_that_see_nothing(hip, rng, rows, offset, causal):
    hip.check(hip.bh_relbias_attention_force_rows(rows))
    try:
        check_attention(hip, attention_case(rng, 1, 2, 2, 50, 90, 24, 32), offset=offset, causal=causal, both=True, distance=30, train=rows == 0)
    finally:
        hip.check(hip.bh_relbias_attention_force_rows(-1))


@pytest.mark.parametrize("order", [(0, 1, 2), (0, 2, 1), (2, 0, 1), (1, 0, 2)])
@pytest.mark.parametrize("pad,d", [(0, 64), (4, 64), (3, 64), (1, 17)])
def test_attention_layouts(hip, rng, order, pad, d):
    check_attention(hip, attention_case(rng, 3, 4, 2, 70, 90, d, 16), lens=[90, 33, 70], order=order, pad=pad)
    check_attention(hip, attention_case(rng, 2, 4, 4, 1, 90, d, 16), order=order, pad=pad, train=False)


@pytest.mark.parametrize("buckets,distance,both", [(2, 2, False), (4, 3, True), (32, 128, True), (32, 128, False), (256, 1000, False), (256, 70, True)])
def test_attention_buckets(hip, rng, buckets, distance, both):
    for rows in (0, 1):
        hip.check(hip.bh_relbias_attention_force_rows(rows))
        try:
            check_attention(hip, attention_case(rng, 1, 3, 3, 150, 330, 32, buckets), distance=distance, both=both, causal=False, train=rows == 0)
        finally:
            hip.check(hip.bh_relbias_attention_force_rows(-1))


def test_attention_masked_buckets(hip, rng):
    """-inf or the lowest float in the table masks its distances; a row with nothing else is empty."""
    for low in (-np.inf, np.finfo(np.float32).min):
        q, k, v, table, d_out = attention_case(rng, 1, 2, 2, 140, 140, 32, 8)
        table[2:, 0] = low                     # head 0 sees the two nearest keys
        table[:, 1] = low                      # head 1 nothing
        got = check_attention(hip, (q, k, v, table, d_out))
        assert (got["out"][0, 1] == 0).all() and np.isneginf(got["lse"][0, 1]).all()
        assert (got["dq"][0, 1] == 0).all() and (got["dk"][0, 1] == 0).all() and (got["dtable"][:, 1] == 0).all()


@pytest.mark.parametrize("sq,sk,rows", [(1, 5000, 1), (16, 3000, 1), (40, 2500, 0), (128, 1500, 0), (70, 4000, 1)])
def test_attention_over_long_histories(hip, rng, sq, sk, rows):
    hip.check(hip.bh_relbias_attention_force_rows(rows))
    try:
        check_attention(hip, attention_case(rng, 2, 2, 1, sq, sk, 64, 32), lens=[sk, sk // 3], distance=128, train=False)
    finally:
        hip.check(hip.bh_relbias_attention_force_rows(-1))


def test_attention_training_of_a_longer_sequence(hip, rng):
    check_attention(hip, attention_case(rng, 1, 2, 1, 600, 600, 64, 32), distance=128)
    check_attention(hip, attention_case(rng, 1, 1, 1, 500, 700, 128, 64), both=True, causal=False, distance=1024)


@pytest.mark.parametrize("splits", [1, 2, 3, 64])
@pytest.mark.parametrize("d", [24, 64, 96, 128])
def test_attention_backward_in_parts(hip, rng, splits, d):
    """The keys of dq and the queries of dk and dv cut into parts, some of them past a causal mask's or a sequence's end."""
    hip.check(hip.bh_relbias_attention_force_splits(splits))
    try:
        check_attention(hip, attention_case(rng, 2, 4, 2, 150, 230, d, 16), lens=[230, 41])
        check_attention(hip, attention_case(rng, 2, 2, 2, 40, 300, d, 16), lens=[0, 300], causal=False, both=True, order=(0, 2, 1), pad=3)
        check_attention(hip, attention_case(rng, 1, 2, 1, 300, 20, d, 16), offset=-100)
    finally:
        hip.check(hip.bh_relbias_attention_force_splits(0))


def test_attention_large_scores(hip, rng):
    q, k, v, table, d_out = attention_case(rng, 1, 2, 2, 70, 100, 64, 16)
    check_attention(hip, (q * 6, k * 6, v, table * 20, d_out), scale=0.3)
    check_attention(hip, (q, k, v, table, d_out), scale=-1.0)
    check_attention(hip, (q, k, v, table, d_out), scale=0.0)


def test_attention_table_gradient_accumulates_and_repeats(hip, rng):
    case = attention_case(rng, 2, 4, 2, 150, 150, 64, 16)
    args = (*case[:4], None, 0, 16, 40, False, True, 0.125, case[4])
    one, two = run_attention(hip, *args), run_attention(hip, *args)
    for n in one:
        assert np.array_equal(one[n], two[n])
    start = rng.standard_normal(case[3].shape).astype(np.float32)
    more = run_attention(hip, *args, accumulate=start)
    assert (np.abs(more["dtable"] - (start.astype(np.float64) + one["dtable"])) <= 2 * oc.U * (np.abs(start) + np.abs(one["dtable"]))).all()


def test_attention_against_differences(hip, rng):
    q, k, v, table, d_out = attention_case(rng, 1, 2, 1, 20, 24, 8, 8)
    args = (None, 4, 8, 12, False, True, 0.4)
    got = run_attention(hip, q, k, v, table, *args, d_out)

    def loss(*x):
        return float((oc.attention(*x, *args)[0]["out"] * d_out).sum())
    eps = 1e-5
    for at, n in enumerate(("dq", "dk", "dv", "dtable")):
        base = [x.astype(np.float64) for x in (q, k, v, table)]
        d = rng.standard_normal(base[at].shape)
        up, down = list(base), list(base)
        up[at], down[at] = base[at] + eps * d, base[at] - eps * d
        # third derivatives of order ten times eps^2, 1e-16 |loss| / eps, and fp32 gradients
        assert abs(float((got[n] * d).sum()) - (loss(*up) - loss(*down)) / (2 * eps)) <= 1e-5 * float(np.abs(got[n] * d).sum() + 1)


# ------------------------------------------------------------------ all of them

def test_capture_is_refused(hip):
    """Work memory comes from the library's cache, so a call on a capturing stream is refused before it queues anything."""
    rt = hip.lib        # the runtime the library is linked to: its symbols are found through the library
    graph = C.c_void_p()
    d = dev(hip, np.ones(64, np.float32))
    i = dev(hip, np.zeros(64, np.int32))
    plan = hip.relbias_attention(batch=1, heads=1, kv_heads=1, sq=2, sk=2, d=4, q_stride=(8, 8, 4), k_stride=(8, 8, 4), v_stride=(8, 8, 4),
                                 o_stride=(8, 8, 4), query_offset=0, num_buckets=4, max_distance=8, bidirectional=0, causal=0, scale=1.0)
    assert rt.hipStreamBeginCapture(C.c_void_p(hip.bh_stream()), 2) == 0
    try:
        rcs = [hip.bh_gemm_epilogue(0, 0, 4, 4, 4, ptr(d), 4, ptr(d), 4, ptr(d, 32), 4, None, -1, None, 0, None, 0),
               hip.bh_distill_forward(ptr(d), 8, ptr(d), ptr(i), None, 2, 8, 2, 1.0, 1.0, 1.0, None, None, ptr(d, 32)),
               hip.bh_relbias_attention_forward(plan, ptr(d), ptr(d), ptr(d), ptr(d), None, ptr(d, 32), ptr(d, 48))]
        text = hip.bh_last_error().decode()
    finally:
        assert rt.hipStreamEndCapture(C.c_void_p(hip.bh_stream()), C.byref(graph)) == 0
        if graph:
            rt.hipGraphDestroy(graph)
    assert rcs == [-1, -1, -1] and "captured" in text
    assert (d.numpy() == 1).all()


def test_attention_and_distillation_from_several_threads(hip, rng):
    """Work memory of one call is not another's: the same inputs give the same bits from every thread."""
    q, k, v, table, d_out = attention_case(rng, 2, 4, 2, 70, 300, 48, 16)
    strides = [(a.shape[1] * a.shape[2] * a.shape[3], a.shape[2] * a.shape[3], a.shape[3]) for a in (q, k, v, q)]
    plan = hip.relbias_attention(batch=2, heads=4, kv_heads=2, sq=70, sk=300, d=48, q_stride=strides[0], k_stride=strides[1], v_stride=strides[2],
                                 o_stride=strides[3], query_offset=230, num_buckets=16, max_distance=64, bidirectional=0, causal=1, scale=0.2)
    dq, dk, dv, dt, dd = (dev(hip, a) for a in (q, k, v, table, d_out))
    z, teacher, index, labels = distill_case(rng, 5, 20001, 7)
    dz, de, di, dy = (dev(hip, a) for a in (z, teacher, index, labels))
    rcs = []

    def outputs():
        return [dev(hip, np.full(s, np.nan, np.float32)) for s in (q.shape, (2, 4, 70), q.shape, k.shape, v.shape, table.shape, z.shape, (1,))]

    def call(o):
        for _ in range(5):
            rcs.append(hip.bh_relbias_attention_forward(plan, ptr(dq), ptr(dk), ptr(dv), ptr(dt), None, ptr(o[0]), ptr(o[1])))
            rcs.append(hip.bh_relbias_attention_backward(plan, ptr(dq), ptr(dk), ptr(dv), ptr(dt), None, ptr(o[0]), ptr(o[1]), ptr(dd), ptr(o[2]),
                                                         ptr(o[3]), ptr(o[4]), ptr(o[5]), 0))
            rcs.append(hip.bh_distill_loss_grad(ptr(dz), 20001, ptr(de), ptr(di), ptr(dy), 5, 20001, 7, 2.0, 0.5, 0.2, None, ptr(o[7]), ptr(o[6]), 20001))
    first = outputs()
    call(first)
    want = [x.numpy() for x in first]
    assert all(np.isfinite(x).all() for x in want)
    outs = [outputs() for _ in range(4)]
    threads = [threading.Thread(target=call, args=(o,)) for o in outs]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert rcs == [0] * 75
    for o in outs:
        for x, w in zip(o, want):
            assert np.array_equal(x.numpy(), w)


FAR = (1 << 30) + 64                                         # floats between rows or sequences: three of them pass 2^32 bytes


@pytest.fixture(scope="module")
def far(hip):
    """One buffer that rows and sequences lie far apart in; put() and get() move rows of it."""
    whole = hip.empty((3 * FAR,))

    class Far:
        @staticmethod
        def at(offset=0):
            return C.c_void_p(whole.ptr + 4 * offset)

        @staticmethod
        def put(offset, rows):
            for i, row in enumerate(rows):
                row = np.ascontiguousarray(row, dtype=np.float32)
                hip.check(hip.bh_memcpy_h2d(whole.ptr + 4 * (offset + i * FAR), row.ctypes.data, row.nbytes))

        @staticmethod
        def get(offset, shape):
            out = np.empty(shape, np.float32)
            for i in range(shape[0]):
                part = np.empty(shape[1:], np.float32)
                hip.check(hip.bh_memcpy_d2h(part.ctypes.data, whole.ptr + 4 * (offset + i * FAR), part.nbytes))
                out[i] = part
            return out
    yield Far


def test_product_rows_far_apart(hip, rng, far):
    a, b, r = (rng.standard_normal(s).astype(np.float32) for s in ((3, 100), (100, 70), (3, 70)))
    far.put(0, a)
    far.put(1000, r)
    hip.check(hip.bh_gemm_epilogue(0, 0, 3, 70, 100, far.at(0), FAR, ptr(dev(hip, b)), 70, far.at(2000), FAR, None, -1, far.at(3000), FAR,
                                   far.at(1000), FAR))
    z, bound = a.astype(np.float64) @ b, oc.product_bound(a.astype(np.float64), b.astype(np.float64))
    assert (np.abs(far.get(3000, (3, 70)) - z) <= bound).all()
    assert (np.abs(far.get(2000, (3, 70)) - z - r) <= bound + 2 * oc.U * np.abs(z + r)).all()


def test_distill_rows_far_apart(hip, rng, far):
    z, teacher, index, labels = distill_case(rng, 3, 1000, 6)
    want_row, want_loss, want_dz = oc.distill(z, teacher, index, labels, 2.0, 0.5, 1.0)
    tol_row, tol_dz = oc.distill_bounds(z, teacher, 2.0, 0.5, 1.0)
    far.put(0, z)
    loss = hip.zeros(1)
    hip.check(hip.bh_distill_loss_grad(far.at(0), FAR, ptr(dev(hip, teacher)), ptr(dev(hip, index)), ptr(dev(hip, labels)), 3, 1000, 6, 2.0, 0.5, 1.0,
                                       None, ptr(loss), far.at(5000), FAR))
    assert abs(loss.numpy()[0] - want_loss) <= 3 * tol_row + 4 * oc.U * abs(want_loss)
    assert (np.abs(far.get(5000, (3, 1000)) - want_dz) <= tol_dz).all()


@pytest.mark.parametrize("sq", [1, 40])
def test_attention_sequences_far_apart(hip, rng, far, sq):
    """a cache of keys and values whose sequences lie 2^30 floats apart"""
    q, k, v, table, d_out = attention_case(rng, 3, 2, 1, sq, 90, 32, 16)
    want, bound = oc.attention(q, k, v, table, None, 90 - sq, 16, 20, False, True, 0.2, d_out)
    places = {n: 100000 * i for i, n in enumerate(("q", "k", "v", "out", "d_out", "dq", "dk", "dv"))}
    for n, x in (("q", q), ("k", k), ("v", v), ("d_out", d_out)):
        far.put(places[n], x)
    at = {n: far.at(o) for n, o in places.items()}
    plan = hip.relbias_attention(batch=3, heads=2, kv_heads=1, sq=sq, sk=90, d=32, q_stride=(FAR, sq * 32, 32), k_stride=(FAR, 90 * 32, 32),
                                 v_stride=(FAR, 90 * 32, 32), o_stride=(FAR, sq * 32, 32), query_offset=90 - sq, num_buckets=16, max_distance=20,
                                 bidirectional=0, causal=1, scale=0.2)
    dt, lse, gt = dev(hip, table), hip.empty((3, 2, sq)), hip.empty(table.shape)
    hip.check(hip.bh_relbias_attention_forward(plan, at["q"], at["k"], at["v"], ptr(dt), None, at["out"], ptr(lse)))
    hip.check(hip.bh_relbias_attention_backward(plan, at["q"], at["k"], at["v"], ptr(dt), None, at["out"], ptr(lse), at["d_out"], at["dq"], at["dk"],
                                                at["dv"], ptr(gt), 0))
    got = {n: far.get(places[n], x.shape) for n, x in (("out", q), ("dq", q), ("dk", k), ("dv", v))}
    got["dtable"], got["lse"] = gt.numpy(), lse.numpy()
    for n in got:
        assert (np.abs(got[n] - want[n]) <= bound[n] + 1e-37).all(), n
