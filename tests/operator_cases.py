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


# ------------------------------------------------------------------ attention with a relative position bias

def bucket(rel, buckets, distance, both):
    """The bucket of one relative position, the logarithm's borders decided in whole numbers."""
    first = 0
    if both:
        buckets //= 2
        first, n = (buckets if rel > 0 else 0), abs(rel)
    else:
        n = max(-rel, 0)
    e = buckets // 2
    if n < e:
        return first + n
    if n >= distance:
        return first + buckets - 1
    j = 0
    while j + 1 < buckets - e and n ** (buckets - e) * e ** (j + 1) >= distance ** (j + 1) * e ** (buckets - e):
        j += 1
    return first + e + j


def attention(q, k, v, table, lens, offset, buckets, distance, both, causal, scale, d_out=None):
    """[batch, heads, rows, d] arrays; returns out, lse and, with d_out, dq, dk, dv, dtable, each with a bound on its rounding error."""
    batch, heads, sq, d = q.shape
    kv_heads, sk = k.shape[1:3]
    group = heads // kv_heads
    rel = np.arange(sk)[None] - (np.arange(sq)[:, None] + offset)
    lut = {r: bucket(int(r), buckets, distance, both) for r in np.unique(rel)}
    idx = np.array([[lut[r] for r in row] for row in rel], dtype=np.int64).reshape(sq, sk)
    z = {n: np.zeros(a.shape) for n, a in (("out", q), ("dq", q), ("dk", k), ("dv", v), ("dtable", table))}
    e = {n: np.zeros(a.shape) for n, a in z.items()}
    z["lse"], e["lse"] = np.full((batch, heads, sq), -np.inf), np.zeros((batch, heads, sq))
    for b in range(batch):
        seen = np.broadcast_to(np.arange(sk)[None] < (sk if lens is None else min(max(int(lens[b]), 0), sk)), (sq, sk))
        if causal:
            seen = seen & (rel <= 0)
        some = seen.any(1)
        for h in range(heads):
            K = np.where(seen.any(0)[:, None], k[b, h // group], 0).astype(np.float64) if lens is not None else k[b, h // group].astype(np.float64)
            V = np.where(seen.any(0)[:, None], v[b, h // group], 0).astype(np.float64) if lens is not None else v[b, h // group].astype(np.float64)
            Q = q[b, h].astype(np.float64)
            bias = np.where(table[:, h] <= -1e30, -np.inf, table[:, h].astype(np.float64))[idx]
            x = np.where(seen, scale * (Q @ K.T) + bias, -np.inf)
            alive = some & (x.max(1, initial=-np.inf) > -np.inf)
            m = np.where(alive, x.max(1, initial=-np.inf), 0)
            p = np.exp(x - m[:, None])
            total = p.sum(1)
            p = p / np.where(alive, total, 1)[:, None]
            z["out"][b, h] = p @ V
            z["lse"][b, h] = np.where(alive, m + np.log(np.where(alive, total, 1)), -np.inf)
            # scores: the product's bound and four roundings; a probability twice that (numerator and sum) and the exponential's
            ex = abs(scale) * product_bound(Q, K.T) + 4 * U * (np.abs(np.where(seen & np.isfinite(x), x, 0)) + np.abs(m)[:, None])
            ex = np.where(seen, ex, 0).max(1, initial=0)[:, None]
            rel_p = 2 * ex + (2 * sk + 16) * U
            e["out"][b, h] = (rel_p + (2 * sk + 8) * U) * (p @ np.abs(V))
            e["lse"][b, h] = (ex + (2 * sk + 8) * U)[:, 0] + 4 * U * np.abs(np.where(alive, z["lse"][b, h], 0))
            if d_out is None:
                continue
            G = d_out[b, h].astype(np.float64)
            rel_p = rel_p + 8 * U * np.abs(np.where(alive, z["lse"][b, h], 0))[:, None]
            dp = G @ V.T
            delta = (p * dp).sum(1)[:, None]
            ds = p * (dp - delta)
            e_delta = (2 * d + 4) * U * (np.abs(G) * np.abs(z["out"][b, h])).sum(1)[:, None] + (np.abs(G) * e["out"][b, h]).sum(1)[:, None]
            e_ds = p * (rel_p * np.abs(dp - delta) + product_bound(G, V.T) + e_delta + 4 * U * (np.abs(dp) + np.abs(delta)))
            z["dq"][b, h] = scale * (ds @ K)
            e["dq"][b, h] = abs(scale) * (e_ds @ np.abs(K) + product_bound(ds, K)) * (1 + 4 * U)
            z["dk"][b, h // group] += scale * (ds.T @ Q)
            e["dk"][b, h // group] += abs(scale) * (e_ds.T @ np.abs(Q) + group * product_bound(ds.T, Q))
            z["dv"][b, h // group] += p.T @ G
            e["dv"][b, h // group] += (p * rel_p).T @ np.abs(G) + group * product_bound(p.T, G)
            for s in range(buckets):
                z["dtable"][s, h] += ds[idx == s].sum()
                e["dtable"][s, h] += e_ds[idx == s].sum() + 2 * (sk + 64) * U * np.abs(ds[idx == s]).sum()
    return z, e
