"""The training operators that are timed, as cases: a dense product with its epilogue, attention with a learned relative position
bias, and distillation from a teacher's top logits.  `run` computes a case in plain torch, or through the library where `own` is set."""
import math

import torch

own = False

ACTS = {"none": -1, "relu": 0, "sigmoid": 1, "tanh": 2, "gelu": 3}


# ---------------------------------------------------------------- cases
def _dense(name, m, k, n, act, residual, train):
    return {"name": name, "op": "dense", "m": m, "k": k, "n": n, "act": act, "residual": residual, "train": train}


def _attention(name, batch, heads, kv_heads, sq, sk, d, buckets, distance, both, causal, padded, rows_first, train):
    return {"name": name, "op": "attention", "batch": batch, "heads": heads, "kv_heads": kv_heads, "sq": sq, "sk": sk, "d": d,
            "buckets": buckets, "distance": distance, "both": both, "causal": causal, "padded": padded,
            "rows_first": rows_first, "train": train}


def _distill(name, rows, vocab, topk, temperature, alpha, labels, train):
    return {"name": name, "op": "distill", "rows": rows, "vocab": vocab, "topk": topk, "temperature": temperature, "alpha": alpha,
            "labels": labels, "train": train}


def listed():
    return [
        # the feed-forward product of the benchmark's block for one new token: the weights are read once, latency counts
        _dense("dense 1 token", 1, 1024, 4096, "gelu", False, False),
        # the benchmark MLP's first layer on an odd number of rows, with a residual: small and ragged
        _dense("dense ragged residual", 777, 784, 513, "relu", True, True),
        # the block's output projection with the residual stream added in the same store
        _dense("dense projection", 8192, 1024, 1024, "none", True, False),
        # the block's feed-forward first layer in training: pre-activation kept, then dX, dW, db
        _dense("dense feed-forward train", 8192, 1024, 4096, "gelu", False, True),
        # one decoder's new token over a long history, keys and values stored token by token
        _attention("attention 1 token", 4, 16, 16, 1, 8001, 64, 32, 128, False, True, True, True, False),
        # the block's attention forward over whole sequences, both directions
        _attention("attention encoder", 8, 16, 16, 1024, 1024, 64, 32, 128, True, False, False, False, False),
        # training a decoder: causal, half the buckets' range in use, the table's gradient with q, k, v
        _attention("attention decoder train", 8, 16, 16, 1024, 1024, 64, 32, 128, False, True, False, False, True),
        # padded batch of odd lengths, shared key heads, an unusual head size, queries and keys of different lengths
        _attention("attention ragged train", 3, 12, 4, 333, 517, 80, 48, 250, True, False, True, True, True),
        # a small student's step: few classes, a short list of teacher logits
        _distill("distill small", 96, 1000, 8, 2.0, 0.5, True, True),
        # validation pass over a mid-sized vocabulary: the loss only
        _distill("distill forward", 4096, 32000, 64, 1.0, 1.0, False, False),
        # few rows of a large vocabulary of odd length (the last micro-batch of a step)
        _distill("distill few rows train", 37, 128001, 50, 2.0, 0.9, True, True),
        # a full training batch over a large vocabulary: the largest tensor a step touches
        _distill("distill train", 8192, 50001, 100, 3.0, 0.7, True, True),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    op = rng.choice(["dense", "attention", "distill"])
    if op == "dense":
        train = rng.random() < 0.5
        k, n = _log(rng, 60, 4100), _log(rng, 60, 4100)
        most = 8192 * 1024 * 4096 * 3 // (k * n * (3 if train else 1))
        c = _dense("", _log(rng, 1, max(1, min(8192, most))), k, n, rng.choice(list(ACTS)), rng.random() < 0.5, train)
    elif op == "attention":
        train = rng.random() < 0.5
        group, kv_heads = rng.choice([1, 1, 2, 4]), rng.choice([1, 2, 3, 4, 8])
        heads, batch = group * kv_heads, rng.randint(1, 6)
        sk, d = _log(rng, 1, 8200), rng.choice([24, 32, 40, 64, 64, 80, 96, 128])
        most = 8 * 16 * 1024 * 1024 * 64 // (batch * heads * sk * max(64, d))
        sq = _log(rng, 1, max(1, min(1500, most)))
        both = rng.random() < 0.5
        c = _attention("", batch, heads, kv_heads, sq, sk, d, rng.choice([16, 32, 32, 64]),
                       rng.choice([64, 128, 128, 300, 1024]), both, not both, rng.random() < 0.5, rng.random() < 0.5, train)
    else:
        vocab = _log(rng, 200, 131000)
        c = _distill("", _log(rng, 1, min(8192, 8192 * 50001 // vocab)), vocab, _log(rng, 1, 128), rng.choice([1.0, 2.0, 4.0]),
                     rng.choice([1.0, 0.7, 0.5]), rng.random() < 0.6, rng.random() < 0.6)
        if c["alpha"] < 1.0:
            c["labels"] = True
    del c["name"]
    return c


# ---------------------------------------------------------------- inputs
def _normal(g, *shape, std=1.0):
    return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32) * std


def _heads(t, rows_first):
    """[batch, heads, rows, d] as the program stores it: contiguous, or token by token ([batch, rows, heads, d])."""
    return t.transpose(1, 2).contiguous().transpose(1, 2) if rows_first else t


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    s = {"case": case}
    if case["op"] == "dense":
        m, k, n = case["m"], case["k"], case["n"]
        s["x"], s["w"], s["bias"] = _normal(g, m, k), _normal(g, k, n, std=k ** -0.5), _normal(g, n, std=0.1)
        s["residual"] = _normal(g, m, n) if case["residual"] else None
        s["dy"] = _normal(g, m, n, std=1.0 / m) if case["train"] else None
    elif case["op"] == "attention":
        b, h, hk, sq, sk, d = (case[x] for x in ("batch", "heads", "kv_heads", "sq", "sk", "d"))
        first = case["rows_first"]
        s["q"] = _heads(_normal(g, b, h, sq, d), first)
        s["k"] = _heads(_normal(g, b, hk, sk, d), first)
        s["v"] = _heads(_normal(g, b, hk, sk, d), first)
        s["table"] = _normal(g, case["buckets"], h)
        # lengths of a padded batch: anything up to the whole, one sequence whole
        lens = torch.randint((sk + 1) // 2, sk + 1, (b,), generator=g, device="cuda", dtype=torch.int32)
        lens[0] = sk
        s["lens"] = lens if case["padded"] else None
        s["d_out"] = _heads(_normal(g, b, h, sq, d, std=1.0 / sq), first) if case["train"] else None
    else:
        rows, vocab, topk = case["rows"], case["vocab"], min(case["topk"], case["vocab"])
        z = _normal(g, rows, vocab, std=2.5)
        t = torch.randn(rows, vocab, generator=g, device="cuda").mul_(1.5).add_(z)   # a teacher that agrees in part
        top, idx = t.topk(topk, dim=1)
        del t
        idx = idx.to(torch.int32)
        # a teacher list may be shorter than the table: its tail is marked -1 (some rows), or empty (a padding position)
        kept = torch.randint(0, 8 * topk, (rows, 1), generator=g, device="cuda")
        idx = torch.where(torch.arange(topk, device="cuda")[None] < kept, idx, torch.full_like(idx, -1)).contiguous()
        labels = torch.randint(0, vocab, (rows,), generator=g, device="cuda", dtype=torch.int32)
        labels = torch.where(torch.rand(rows, generator=g, device="cuda") < 0.1, torch.full_like(labels, -1), labels)
        s["logits"], s["teacher"], s["index"] = z, top.contiguous(), idx
        s["labels"] = labels if case["labels"] else None
    return s


# ---------------------------------------------------------------- plain forms
def _act(act, z):
    if act == "relu":
        return torch.clamp(z, min=0)
    if act == "sigmoid":
        return 1 / (1 + torch.exp(-z))
    if act == "tanh":
        return torch.tanh(z)
    if act == "gelu":
        return 0.5 * z * (1 + torch.erf(z * math.sqrt(0.5)))
    return z


def _act_slope(act, z):
    if act == "relu":
        return (z > 0).to(z.dtype)
    if act == "sigmoid":
        y = 1 / (1 + torch.exp(-z))
        return y * (1 - y)
    if act == "tanh":
        y = torch.tanh(z)
        return 1 - y * y
    if act == "gelu":
        return 0.5 * (1 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) * (1 / math.sqrt(2 * math.pi))
    return torch.ones_like(z)


def _dense_plain(s):
    c, x, w = s["case"], s["x"], s["w"]
    z = x @ w + s["bias"]
    y = _act(c["act"], z)
    if s["residual"] is not None:
        y = y + s["residual"]
    if not c["train"]:
        return {"y": y}
    dz = s["dy"] * _act_slope(c["act"], z) if c["act"] != "none" else s["dy"]
    return {"y": y, "dx": dz @ w.t(), "gw": x.t() @ dz, "gb": dz.sum(0)}


def _buckets(rel, buckets, distance, both):
    """The bucket of each relative position (key - query): exact small distances, then logarithmic ones up to `distance`."""
    first = 0
    if both:
        buckets //= 2
        first = (rel > 0).long() * buckets
        n = rel.abs()
    else:
        n = (-rel).clamp(min=0)
    exact = buckets // 2
    step = torch.log(n.clamp(min=1).double() / exact) / math.log(distance / exact) * (buckets - exact)
    far = (exact + torch.floor(step + 1e-9).long()).clamp(max=buckets - 1)
    return first + torch.where(n < exact, n, far)


def _attention_plain(s):
    c, q, k, v = s["case"], s["q"], s["k"], s["v"]
    b, h, hk, sq, sk, d = (c[x] for x in ("batch", "heads", "kv_heads", "sq", "sk", "d"))
    group, scale = h // hk, d ** -0.5
    rel = torch.arange(sk, device=q.device)[None] - (torch.arange(sq, device=q.device)[:, None] + sk - sq)
    bucket = _buckets(rel, c["buckets"], c["distance"], c["both"])
    ke, ve = (k.repeat_interleave(group, 1), v.repeat_interleave(group, 1)) if group > 1 else (k, v)
    x = q @ ke.transpose(2, 3)
    x = x * scale + s["table"][bucket].permute(2, 0, 1)[None]
    shut = (rel > 0)[None, None] if c["causal"] else None
    if s["lens"] is not None:
        pad = (torch.arange(sk, device=q.device)[None] >= s["lens"][:, None])[:, None, None]
        shut = pad if shut is None else shut | pad
    if shut is not None:
        x = x.masked_fill(shut, -math.inf)
    top = x.amax(3, keepdim=True).clamp(min=-3.0e38)
    e = torch.exp(x - top)
    total = e.sum(3, keepdim=True)
    p = torch.where(total > 0, e / total, torch.zeros_like(e))
    out = p @ ve
    lse = (top + torch.log(total))[..., 0]
    if not c["train"]:
        return {"out": out, "lse": lse}
    do = s["d_out"]
    dv = (p.transpose(2, 3) @ do).reshape(b, hk, group, sk, d).sum(2)
    dp = do @ ve.transpose(2, 3)
    ds = p * (dp - (do * out).sum(3, keepdim=True))
    dq = (ds @ ke) * scale
    dk = ((ds.transpose(2, 3) @ q) * scale).reshape(b, hk, group, sk, d).sum(2)
    # the table's gradient: every relative position is a diagonal; rows reversed and shifted make it a column
    skew = torch.nn.functional.pad(ds.sum(0, dtype=torch.float64).flip(1), (0, sq)).reshape(h, -1)[:, :sq * (sk + sq - 1)]
    of_rel = skew.reshape(h, sq, sk + sq - 1).sum(1)
    rels = torch.arange(-(sk - 1), sq, device=q.device)
    member = _buckets(rels, c["buckets"], c["distance"], c["both"])[:, None] == torch.arange(c["buckets"], device=q.device)
    table = of_rel @ member.double()
    return {"out": out, "lse": lse, "dq": dq, "dk": dk, "dv": dv, "dtable": table.t().float().contiguous()}


def _distill_plain(s):
    c, z, idx = s["case"], s["logits"], s["index"]
    heat, alpha, scale = c["temperature"], c["alpha"], 1.0 / c["rows"]
    kept, at = idx >= 0, idx.clamp(min=0).long()
    some = kept.any(1, keepdim=True)
    t = torch.where(kept, s["teacher"] / heat, torch.full_like(s["teacher"], -math.inf))
    top = torch.where(some, t.amax(1, keepdim=True), torch.zeros_like(t[:, :1]))
    e = torch.exp(t - top)
    total = e.sum(1, keepdim=True)
    p = torch.where(some, e / total, torch.zeros_like(e))
    log_p = torch.where(kept, t - top - torch.log(total), torch.zeros_like(t))
    u = z / heat
    m = u.amax(1, keepdim=True)
    eu = torch.exp(u - m)
    su = eu.sum(1, keepdim=True)
    log_q = u.gather(1, at) - m - torch.log(su)
    row = alpha * heat * heat * torch.where(p > 0, p * (log_p - log_q), torch.zeros_like(p)).sum(1)
    hard = s["labels"] is not None and alpha < 1
    if hard:
        y = s["labels"].clamp(min=0).long()[:, None]
        mine = s["labels"][:, None] >= 0
        m1 = z.amax(1, keepdim=True)
        e1 = torch.exp(z - m1)
        s1 = e1.sum(1, keepdim=True)
        ce = torch.where(mine, m1 + torch.log(s1) - z.gather(1, y), torch.zeros_like(m1))
        row = row + (1 - alpha) * ce[:, 0]
    loss = (row.sum(dtype=torch.float64) * scale).float().reshape(1)
    if not c["train"]:
        return {"loss": loss, "row_loss": row}
    dz = eu / su * (alpha * heat * scale * some.float())
    dz.scatter_add_(1, at, -alpha * heat * scale * p)
    if hard:
        dz += e1 / s1 * ((1 - alpha) * scale * mine.float())
        dz.scatter_add_(1, y, -(1 - alpha) * scale * mine.float())
    return {"loss": loss, "row_loss": row, "dlogits": dz}


# ---------------------------------------------------------------- the library's calls
def _ptr(t):
    return None if t is None else t.data_ptr()


def _buffer(s, name, like=None, shape=None):
    """An output buffer that the program keeps from call to call."""
    if name not in s:
        s[name] = torch.empty_like(like) if like is not None else torch.empty(shape, device="cuda", dtype=torch.float32)
    return s[name]


def _dense_own(s):
    from boat_amd import hip
    c = s["case"]
    m, k, n, act = c["m"], c["k"], c["n"], ACTS[c["act"]]
    y = _buffer(s, "y", shape=(m, n))
    saved = _buffer(s, "saved", shape=(m, n)) if c["train"] and act >= 0 else None
    hip.check(hip.bh_gemm_epilogue(0, 0, m, n, k, _ptr(s["x"]), k, _ptr(s["w"]), n, _ptr(y), n, _ptr(s["bias"]), act, _ptr(saved), n,
                                   _ptr(s["residual"]), n), "bh_gemm_epilogue")
    if not c["train"]:
        return {"y": y}
    dx, gw, gb = _buffer(s, "dx", shape=(m, k)), _buffer(s, "gw", shape=(k, n)), _buffer(s, "gb", shape=(n,))
    hip.check(hip.bh_dense_act_backward(act, _ptr(s["x"]), _ptr(s["w"]), _ptr(saved), _ptr(s["dy"]), _ptr(dx), _ptr(gw), _ptr(gb), m, k, n, 0),
              "bh_dense_act_backward")
    return {"y": y, "dx": dx, "gw": gw, "gb": gb}


def _attention_own(s):
    from boat_amd import hip
    c, q, k, v = s["case"], s["q"], s["k"], s["v"]
    out = _buffer(s, "out", like=q)
    if "plan" not in s:
        s["plan"] = hip.relbias_attention(batch=c["batch"], heads=c["heads"], kv_heads=c["kv_heads"], sq=c["sq"], sk=c["sk"], d=c["d"],
                                          q_stride=q.stride()[:3], k_stride=k.stride()[:3], v_stride=v.stride()[:3], o_stride=out.stride()[:3],
                                          query_offset=c["sk"] - c["sq"], num_buckets=c["buckets"], max_distance=c["distance"],
                                          bidirectional=int(c["both"]), causal=int(c["causal"]), scale=c["d"] ** -0.5)
    lse = _buffer(s, "lse", shape=(c["batch"], c["heads"], c["sq"]))
    hip.check(hip.bh_relbias_attention_forward(s["plan"], _ptr(q), _ptr(k), _ptr(v), _ptr(s["table"]), _ptr(s["lens"]), _ptr(out), _ptr(lse)),
              "bh_relbias_attention_forward")
    if not c["train"]:
        return {"out": out, "lse": lse}
    dq, dk, dv, dt = _buffer(s, "dq", like=q), _buffer(s, "dk", like=k), _buffer(s, "dv", like=v), _buffer(s, "dt", like=s["table"])
    hip.check(hip.bh_relbias_attention_backward(s["plan"], _ptr(q), _ptr(k), _ptr(v), _ptr(s["table"]), _ptr(s["lens"]), _ptr(out), _ptr(lse),
                                                _ptr(s["d_out"]), _ptr(dq), _ptr(dk), _ptr(dv), _ptr(dt), 0), "bh_relbias_attention_backward")
    return {"out": out, "lse": lse, "dq": dq, "dk": dk, "dv": dv, "dtable": dt}


def _distill_own(s):
    from boat_amd import hip
    c, z = s["case"], s["logits"]
    rows, vocab, topk = c["rows"], c["vocab"], s["index"].shape[1]
    loss, row = _buffer(s, "loss", shape=(1,)), _buffer(s, "row", shape=(rows,))
    head = (_ptr(z), vocab, _ptr(s["teacher"]), _ptr(s["index"]), _ptr(s["labels"]), rows, vocab, topk, c["temperature"], c["alpha"], 1.0 / rows)
    if not c["train"]:
        hip.check(hip.bh_distill_forward(*head, _ptr(row), None, _ptr(loss)), "bh_distill_forward")
        return {"loss": loss, "row_loss": row}
    dz = _buffer(s, "dz", shape=(rows, vocab))
    hip.check(hip.bh_distill_loss_grad(*head, _ptr(row), _ptr(loss), _ptr(dz), vocab), "bh_distill_loss_grad")
    return {"loss": loss, "row_loss": row, "dlogits": dz}


def run(state):
    op = state["case"]["op"]
    if own:
        return {"dense": _dense_own, "attention": _attention_own, "distill": _distill_own}[op](state)
    return {"dense": _dense_plain, "attention": _attention_plain, "distill": _distill_plain}[op](state)


# ---------------------------------------------------------------- what a pass cannot do without
def work(case):
    if case["op"] == "dense":
        m, k, n = case["m"], case["k"], case["n"]
        words = m * k + k * n + n + m * n * (1 + int(case["residual"]))
        flops = 2 * m * n * k
        if case["train"]:
            words += m * n + m * k + k * n + n   # dy in; dx, gw, gb out
            flops *= 3
        return {"bytes": 4 * words, "flops": flops}
    if case["op"] == "attention":
        b, h, hk, sq, sk, d = (case[x] for x in ("batch", "heads", "kv_heads", "sq", "sk", "d"))
        off = sk - sq
        pairs = sum(min(sk, max(0, i + off + 1)) for i in range(sq)) if case["causal"] else sq * sk
        pairs = pairs * (0.75 if case["padded"] else 1)
        words = b * d * (2 * h * sq + 2 * hk * sk) + case["buckets"] * h + b * h * sq
        flops = 4 * b * h * pairs * d
        if case["train"]:
            words += b * d * (2 * h * sq + 2 * hk * sk) + case["buckets"] * h
            flops += 10 * b * h * pairs * d
        return {"bytes": 4 * words, "flops": flops}
    n, lists = case["rows"] * case["vocab"], case["rows"] * case["topk"] * 2
    return {"bytes": 4 * (n * (2 if case["train"] else 1) + lists + 2 * case["rows"]), "flops": 4 * n}


# ---------------------------------------------------------------- the definitions in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    return {"dense": _dense_exact, "attention": _attention_exact, "distill": _distill_exact}[case["op"]](case, s)


def _dense_exact(case, s):
    x, w = s["x"].double(), s["w"].double().requires_grad_(case["train"])
    bias = s["bias"].double().requires_grad_(case["train"])
    x.requires_grad_(case["train"])
    z = torch.addmm(bias, x, w)
    forms = {"none": lambda a: a, "relu": torch.relu, "sigmoid": torch.sigmoid, "tanh": torch.tanh, "gelu": torch.nn.functional.gelu}
    y = forms[case["act"]](z)
    if case["residual"]:
        y = y + s["residual"].double()
    if not case["train"]:
        return {"y": y}
    dx, gw, gb = torch.autograd.grad(y, (x, w, bias), s["dy"].double())
    return {"y": y.detach(), "dx": dx, "gw": gw, "gb": gb}


def _bucket_of(rel, buckets, distance, both):
    """One relative position's bucket in whole numbers: log(n/e)/log(D/e)*(b-e) >= j  <=>  n^(b-e) e^j >= D^j e^(b-e)."""
    first = 0
    if both:
        buckets //= 2
        first = buckets if rel > 0 else 0
        n = abs(rel)
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


def _attention_exact(case, s):
    b, h, hk, sq, sk, d = (case[x] for x in ("batch", "heads", "kv_heads", "sq", "sk", "d"))
    group, off = h // hk, sk - sq
    lut = torch.tensor([_bucket_of(r, case["buckets"], case["distance"], case["both"]) for r in range(-(sk - 1) - max(0, sq - sk), sk + sq)],
                       device="cuda")
    base = (sk - 1) + max(0, sq - sk)
    i, j = torch.arange(sq, device="cuda")[:, None], torch.arange(sk, device="cuda")[None]
    rel = j - i - off
    bucket = lut[rel + base]
    lens = [sk] * b if s["lens"] is None else [int(n) for n in s["lens"]]
    out, lse = torch.zeros(b, h, sq, d, dtype=torch.float64, device="cuda"), torch.zeros(b, h, sq, dtype=torch.float64, device="cuda")
    dq, dk, dv = torch.zeros_like(out), torch.zeros(b, hk, sk, d, dtype=torch.float64, device="cuda"), torch.zeros(b, hk, sk, d, dtype=torch.float64, device="cuda")
    dt = torch.zeros(case["buckets"], h, dtype=torch.float64, device="cuda")
    for n in range(b):
        live = j < lens[n]
        if case["causal"]:
            live = live & (rel <= 0)
        for a in range(h):
            q, k, v = s["q"][n, a].double(), s["k"][n, a // group].double(), s["v"][n, a // group].double()
            x = (q @ k.t()) / math.sqrt(d) + s["table"].double()[bucket, a]
            x = torch.where(live, x, torch.full_like(x, -math.inf))
            z = torch.logsumexp(x, 1)
            p = torch.where(live, torch.exp(x - torch.where(z > -math.inf, z, torch.zeros_like(z))[:, None]), torch.zeros_like(x))
            out[n, a], lse[n, a] = p @ v, z
            if case["train"]:
                g = s["d_out"][n, a].double()
                dp = g @ v.t()
                ds = p * (dp - (p * dp).sum(1, keepdim=True))
                dv[n, a // group] += p.t() @ g
                dq[n, a] = ds @ k / math.sqrt(d)
                dk[n, a // group] += ds.t() @ q / math.sqrt(d)
                dt[:, a] += torch.bincount(bucket.reshape(-1), weights=ds.reshape(-1), minlength=case["buckets"])
    r = {"out": out, "lse": lse}
    return {**r, "dq": dq, "dk": dk, "dv": dv, "dtable": dt} if case["train"] else r


def _distill_exact(case, s):
    rows, vocab, heat, alpha = case["rows"], case["vocab"], case["temperature"], case["alpha"]
    block = max(1, (1 << 27) // vocab)
    row = torch.zeros(rows, dtype=torch.float64, device="cuda")
    dz = torch.zeros(rows, vocab, dtype=torch.float64, device="cuda") if case["train"] else None
    for lo in range(0, rows, block):
        hi = min(rows, lo + block)
        z, idx = s["logits"][lo:hi].double(), s["index"][lo:hi].long()
        here = idx >= 0
        any_here = here.any(1)
        t = s["teacher"][lo:hi].double() / heat
        t = torch.where(here, t, torch.full_like(t, -1e300))
        lp = torch.log_softmax(t, 1)
        p = torch.where(here, lp.exp(), torch.zeros_like(lp))
        lq = torch.log_softmax(z / heat, 1)
        picked = lq.gather(1, torch.where(here, idx, torch.zeros_like(idx)))
        row[lo:hi] = alpha * heat ** 2 * torch.where(here & (p > 0), p * (lp - picked), torch.zeros_like(p)).sum(1)
        if case["train"]:
            g = lq.exp() * any_here[:, None]
            at = here.nonzero()
            g.index_put_((at[:, 0], idx[at[:, 0], at[:, 1]]), -p[at[:, 0], at[:, 1]], accumulate=True)
            dz[lo:hi] = g * (alpha * heat / rows)
        if s["labels"] is not None and alpha < 1:
            y = s["labels"][lo:hi].long()
            r = (y >= 0).nonzero()[:, 0]
            l1 = torch.log_softmax(z[r], 1)
            row[lo + r] -= (1 - alpha) * l1[torch.arange(len(r), device="cuda"), y[r]]
            if case["train"]:
                g = l1.exp()
                g[torch.arange(len(r), device="cuda"), y[r]] -= 1
                dz[lo + r] += g * ((1 - alpha) / rows)
    loss = (row.sum() / rows).reshape(1)
    return {"loss": loss, "row_loss": row, "dlogits": dz} if case["train"] else {"loss": loss, "row_loss": row}
