"""Plain float64 forms of the fused training operators and the rounding bounds their tests use.

u = 2^-24 is half a step of fp32 relative to the value, the most one rounding can be off."""
import math

import numpy as np

U = 2.0 ** -24
ACTS = {"none": -1, "relu": 0, "sigmoid": 1, "tanh": 2, "gelu": 3}

_erf = np.vectorize(math.erf, otypes=[np.float64])


def act(name, z):
    if name == "relu":
        return np.maximum(z, 0)
    if name == "sigmoid":
        return 1 / (1 + np.exp(-z))
    if name == "tanh":
        return np.tanh(z)
    if name == "gelu":
        return 0.5 * z * (1 + _erf(z / math.sqrt(2)))
    return z


def act_slope(name, z):
    if name == "relu":
        return (z > 0).astype(np.float64)
    if name == "sigmoid":
        y = 1 / (1 + np.exp(-z))
        return y * (1 - y)
    if name == "tanh":
        return 1 - np.tanh(z) ** 2
    if name == "gelu":
        return 0.5 * (1 + _erf(z / math.sqrt(2))) + z * np.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    return np.ones_like(z)


def product_bound(a, b, extra=0.0):
    """Most that sum_k a_ik b_kj may be off in fp32: k additions in any order, each rounding (or cutting, 2u) a partial sum
    that is at most sum |a||b|, and the products' own error of at most u."""
    k = a.shape[1]
    return (2 * k + 4) * U * (np.abs(a) @ np.abs(b)) + extra


def distill(z, teacher, index, labels, temperature, alpha, scale):
    """Row losses, loss and gradient from the definition, row by row."""
    rows, vocab = z.shape
    row, dz = np.zeros(rows), np.zeros((rows, vocab))
    z = z.astype(np.float64)
    for r in range(rows):
        with np.errstate(all="ignore"):
            def log_softmax(x):
                m = x.max()
                return x - m - np.log(np.exp(x - m).sum())
            keep = [j for j in range(index.shape[1]) if 0 <= index[r, j] < vocab]
            t = np.array([float(teacher[r, j]) for j in keep]) / temperature
            if len(keep) and t.max() > -np.inf:
                lp, lq = log_softmax(t), log_softmax(z[r] / temperature)
                p = np.exp(lp)
                dz[r] += scale * alpha * temperature * np.exp(lq)
                for j, pj, l in zip(keep, p, lp):
                    if pj > 0:
                        row[r] += alpha * temperature ** 2 * pj * (l - lq[index[r, j]])
                    dz[r, index[r, j]] -= scale * alpha * temperature * pj
            if labels is not None and 0 <= labels[r] < vocab:
                l1 = log_softmax(z[r])
                row[r] -= (1 - alpha) * l1[labels[r]]
                dz[r] += scale * (1 - alpha) * np.exp(l1)
                dz[r, labels[r]] -= scale * (1 - alpha)
    return row, scale * row.sum(), dz


def distill_bounds(z, teacher, temperature, alpha, scale):
    """(row loss, gradient) absolute bounds.  A softmax's exponent is off by 3 roundings of |z - max|/T, its exp by 2u, the sum
    of `vocab` positive terms in blocks of a thread by at most (vocab/256 + 80) u; a weight of the gradient is a product of
    such factors (6 more roundings); a loss term also holds the two logarithms (|log| <= range/T + log vocab + 1)."""
    rows, vocab = z.shape
    finite = np.where(np.isfinite(z), z, 0)
    spread = float((finite.max(1) - finite.min(1)).max()) / min(temperature, 1.0)
    tf = np.where(np.isfinite(teacher), teacher, 0) if teacher.size else np.zeros((1, 1))
    spread_t = float((tf.max(1) - tf.min(1)).max()) / temperature + float(np.abs(tf).max()) / temperature
    rel = U * (3 * (spread + spread_t) + 2 * vocab / 256 + 180)
    logs = spread + spread_t + math.log(vocab + 1) + 10
    row = (alpha * temperature ** 2 + 1 - alpha) * (rel + 8 * U * logs) * 2
    return row, scale * (alpha * temperature + 1 - alpha) * rel * 2
