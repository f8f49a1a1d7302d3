"""Distillation where the logits lie far from zero: whole ranges of the vocabulary masked with large negative numbers, common
offsets of the student's or the teacher's logits, every form of the kernels (rows in registers, in LDS, streamed, in segments)."""
import math

import numpy as np
import pytest

import operator_cases as oc
from test_gpu_operators import _release_device_arrays, dev, distill_case, ptr, run_distill  # noqa: F401

pytestmark = pytest.mark.gpu

SHAPES = [(5, 700), (3, 1900), (4, 3000), (3, 6001), (5, 16000), (129, 26001), (130, 60003), (3, 40001)]


def bounds(z, teacher, temperature, alpha, scale, vocab):
    """(row loss, gradient) bounds from the spread of what is live.  An exponent (x - max)/T is off by 3 roundings of itself (the
    difference, log2 e / T, the product), its exponential by 2u, and by T times both where exp(x) is exp(x/T)^T; the sum of `vocab`
    positive terms by (vocab/256 + 80)u; a weight of the gradient is a product of such factors, a loss term holds two logarithms."""
    spread = max((r[np.isfinite(r)].max() - r[np.isfinite(r)].min() for r in z), default=0.0) / min(temperature, 1.0)
    spread_t = max((r[np.isfinite(r)].max() - r[np.isfinite(r)].min() if np.isfinite(r).any() else 0.0 for r in teacher), default=0.0) / temperature
    rel = oc.U * (3 * (spread + spread_t) + 2 * max(temperature, 1.0) + 2 * vocab / 256 + 180)
    logs = spread + spread_t + math.log(vocab + 1) + 10
    row = (alpha * temperature ** 2 + 1 - alpha) * (rel + 8 * oc.U * logs) * 2
    return row, scale * (alpha * temperature + 1 - alpha) * rel * 2


def check(hip, z, live, teacher, index, labels, temperature, alpha, in_place=False):
    """live [rows, vocab]: what is not masked; the masked logits' own probability is 0 in fp32 and below 1e-300 in truth"""
    rows, vocab = z.shape
    scale = 1.0 / rows
    want_row, want_loss, want_dz = oc.distill(z, teacher, index, labels, temperature, alpha, scale)
    tol_row, tol_dz = bounds(np.where(live, z.astype(np.float64), np.nan), teacher.astype(np.float64), temperature, alpha, scale, vocab)
    forward, both, dz, back = run_distill(hip, z, teacher, index, labels, temperature, alpha, scale, in_place=in_place)
    for row, loss in (forward, both):
        assert np.isfinite(row).all() and (np.abs(row - want_row) <= tol_row + 4 * oc.U * np.abs(want_row)).all()
        assert abs(loss - want_loss) <= tol_row + 4 * oc.U * np.abs(want_row).sum() * scale
    assert np.isfinite(dz).all() and (np.abs(dz - want_dz) <= tol_dz).all(), np.abs(dz - want_dz).max() / tol_dz
    assert (dz[~live] == 0).all()
    if back is not None:
        assert (np.abs(back - 2 * want_dz) <= 2 * tol_dz).all() and (back[~live] == 0).all()


def masked_case(rng, rows, vocab, topk, pattern, value, labels):
    z, teacher, index, lab = distill_case(rng, rows, vocab, topk, labels)
    live = np.zeros((rows, vocab), bool)
    if pattern == "few":                                         # some allowed words only
        for r in range(rows):
            live[r, rng.choice(vocab, 7, replace=False)] = True
    else:
        cut = vocab * 3 // 5
        live[:, cut if pattern == "leading" else 0:vocab if pattern == "leading" else vocab - cut] = True
    z[~live] = value
    allowed = [np.flatnonzero(m) for m in live]                  # teacher and labels name allowed words
    index = np.stack([np.where((i >= 0) & (i < vocab), a[i % len(a)], i) for i, a in zip(index, allowed)]).astype(np.int32)
    if labels:
        lab = np.array([a[i % len(a)] if i >= 0 else i for i, a in zip(lab, allowed)], np.int32)
    return z, live, teacher, index, lab


@pytest.mark.parametrize("rows,vocab", SHAPES)
@pytest.mark.parametrize("value", [-1e10, -1e20, -1e30, float(np.finfo(np.float32).min)])
@pytest.mark.parametrize("temperature", [1.0, 2.0, 2.5, 3.0, 4.0])
def test_masked_ranges(hip, rng, rows, vocab, value, temperature):
    patterns = ["few", "leading", "trailing"]
    for i, pattern in enumerate(patterns if rows < 100 else patterns[int(temperature) % 3:][:1]):
        check(hip, *masked_case(rng, rows, vocab, 6, pattern, value, i != 1), temperature, 0.6 if i < 2 else 1.0)


@pytest.mark.parametrize("rows,vocab", SHAPES)
@pytest.mark.parametrize("offset", [1e3, -1e3, 1e4, -1e4])
def test_common_offsets(hip, rng, rows, vocab, offset):
    for temperature, labels, of_teacher in ((1.0, True, False), (2.0, False, True), (2.5, True, True), (4.0, True, True)):
        z, teacher, index, lab = distill_case(rng, rows, vocab, 9, labels)
        z = (z + np.float32(offset)).astype(np.float32)
        if of_teacher:
            teacher = (teacher - np.float32(offset)).astype(np.float32)
        check(hip, z, np.ones(z.shape, bool), teacher, index, lab, temperature, 0.5, in_place=not labels)


@pytest.mark.parametrize("rows,vocab", [(5, 700), (129, 26001), (3, 40001)])
def test_rows_of_one_value(hip, rng, rows, vocab):
    """Every logit of the row the type's lowest or highest value, or a large mask: a uniform distribution."""
    for value in (float(np.finfo(np.float32).min), float(np.finfo(np.float32).max), -1e10, -1e30):
        _, teacher, index, lab = distill_case(rng, rows, vocab, 5)
        check(hip, np.full((rows, vocab), value, np.float32), np.ones((rows, vocab), bool), teacher, index, lab, 2.5, 0.5)


def test_teacher_of_far_values(hip, rng):
    """A teacher's list may hold its type's lowest value; below temperature 1 its quotient by the temperature would be infinite."""
    z, teacher, index, lab = distill_case(rng, 7, 500, 6)
    teacher[2, :] = np.finfo(np.float32).min
    teacher[4, 1:4] = np.finfo(np.float32).min
    want_row, _, want_dz = oc.distill(z, teacher, index, lab, 0.5, 0.7, 1.0)
    spread = np.where(teacher < -1e30, 0, teacher)
    tol_row, tol_dz = bounds(z, spread, 0.5, 0.7, 1.0, 500)
    (row, _), _, dz, _ = run_distill(hip, z, teacher, index, lab, 0.5, 0.7, 1.0)
    assert (np.abs(row - want_row) <= tol_row + 4 * oc.U * np.abs(want_row)).all() and (np.abs(dz - want_dz) <= tol_dz).all()


@pytest.mark.parametrize("rows,vocab", SHAPES)
def test_the_temperature_leaves_the_hard_part_alone(hip, rng, rows, vocab):
    """Without weight on the teacher the loss is a cross entropy at temperature 1, whatever the temperature: the same bits."""
    case = distill_case(rng, rows, vocab, 3)
    want = run_distill(hip, *case, 1.0, 0.0, 0.5)
    for temperature in (2.0, 2.5, 3.0, 4.0):
        got = run_distill(hip, *case, temperature, 0.0, 0.5)
        for (row, loss), (row1, loss1) in zip(got[:2], want[:2]):
            assert np.array_equal(row, row1) and loss == loss1
        assert np.array_equal(got[2], want[2]) and np.array_equal(got[3], want[3]), temperature


@pytest.mark.parametrize("rows,vocab", SHAPES)
def test_a_teacher_without_weight_is_not_looked_at(hip, rng, rows, vocab):
    """alpha = 0: masked student logits under the teacher's entries, or a teacher of NaN, leave the cross entropy as it is."""
    z, teacher, index, lab = distill_case(rng, rows, vocab, 6)
    for r in range(rows):
        for i in index[r]:
            if 0 <= i < vocab and i != lab[r]:
                z[r, i] = -np.inf
    none = np.zeros((rows, 0), np.float32), np.zeros((rows, 0), np.int32)
    want = run_distill(hip, z, *none, lab, 2.0, 0.0, 0.5)
    assert np.isfinite(want[0][0]).all() and np.isfinite(want[2]).all()
    for t in (teacher, np.full_like(teacher, np.nan), np.full_like(teacher, np.inf)):
        got = run_distill(hip, z, t, index, lab, 2.0, 0.0, 0.5)
        assert np.array_equal(got[0][0], want[0][0]) and got[0][1] == want[0][1] and np.array_equal(got[1][0], want[1][0])
        assert np.array_equal(got[2], want[2]) and np.array_equal(got[3], want[3])


@pytest.mark.parametrize("rows,vocab", SHAPES)
@pytest.mark.parametrize("temperature", [1.0, 2.5])
def test_rows_without_a_softmax(hip, rng, rows, vocab, temperature):
    """-inf all over a row, +inf or NaN in it: that row is NaN, the others are what they are without it."""
    z, teacher, index, lab = distill_case(rng, rows, vocab, 6)
    index[0], lab[0] = 0, 0                                      # the spoilt row has entries and a label
    want = run_distill(hip, z, teacher, index, lab, temperature, 0.5, 0.5)
    for spoil in ("empty", np.inf, np.nan):
        bad = z.copy()
        if spoil == "empty":
            bad[0] = -np.inf
        else:
            bad[0, vocab // 2] = spoil
        (row, loss), (row2, loss2), dz, back = run_distill(hip, bad, teacher, index, lab, temperature, 0.5, 0.5)
        assert np.isnan([row[0], row2[0], loss, loss2]).all() and np.isnan(dz[0]).all() and np.isnan(back[0]).all(), spoil
        assert np.array_equal(row[1:], want[0][0][1:]) and np.array_equal(row2[1:], want[1][0][1:])
        assert np.array_equal(dz[1:], want[2][1:]) and np.array_equal(back[1:], want[3][1:])


def test_more_rows_than_a_grids_second_dimension(hip, rng):
    rows, vocab = 66000, 33
    z, teacher, index, lab = distill_case(rng, rows, vocab, 3)
    want_row, want_loss, want_dz = oc.distill(z, teacher, index, lab, 2.0, 0.5, 1.0 / rows)
    tol_row, tol_dz = bounds(z, teacher, 2.0, 0.5, 1.0 / rows, vocab)
    (row, loss), (row2, _), dz, back = run_distill(hip, z, teacher, index, lab, 2.0, 0.5, 1.0 / rows)
    assert (np.abs(row - want_row) <= tol_row + 4 * oc.U * np.abs(want_row)).all() and np.array_equal(row, row2)
    assert abs(loss - want_loss) <= tol_row + 4 * oc.U * abs(want_loss)
    assert (np.abs(dz - want_dz) <= tol_dz).all() and (np.abs(back - 2 * want_dz) <= 2 * tol_dz).all()
