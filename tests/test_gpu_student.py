"""A student block as its user writes it, on the tape: dense layers with activation and residual, attention with a relative
position bias, distillation from a teacher's kept logits; values and every gradient against float64.

Tolerance: the same formulas are evaluated on the CPU in float32 as well.  The block's error against float64 is a sum of the
same roundings taken in another order, so four times what plain float32 loses in a quantity, and 2^-22 of its largest
value for quantities that plain float32 happens to hit, bounds it.  Where a true gradient is zero because a row has one key
(p = 1, so dP - delta = 0), or because a softmax does not see what all scores of a row share (the bias of the keys: the sum of
p (dP - delta) over a row is 0), what is left is the rounding of the two sums of d products dO . V, at most (2 d + 8) 2^-24 of the
sum of their magnitudes: the gradients behind it may be that times the magnitudes they sum."""
import ctypes as C

import numpy as np
import pytest
import torch

import operator_cases as oc

pytestmark = pytest.mark.gpu

ACTS = {-1: lambda z: z, 0: torch.relu, 1: torch.sigmoid, 2: torch.tanh, 3: torch.nn.functional.gelu}


def shape(*s):
    return (C.c_int64 * len(s))(*s), len(s)


class Block:
    """x -> act(x W1 + b1) = h -> q, k, v -> attention -> act(a Wo + bo) + h -> logits, distilled."""

    def __init__(self, rng, batch=3, seq=37, heads=4, kv_heads=2, d=16, vocab=101, kept=7, lens=(37, 20, 0), causal=False, acts=(3, 2)):
        self.__dict__.update({k: v for k, v in locals().items() if k not in ("self", "rng")})
        w, kvw = heads * d, kv_heads * d
        r = lambda *s: rng.standard_normal(s).astype(np.float32)
        sizes = {"in": (w, w), "q": (w, w), "k": (w, kvw), "v": (w, kvw), "o": (w, w), "head": (w, vocab)}
        self.weights = {n: (r(*s) / np.sqrt(np.float32(s[0]))) for n, s in sizes.items()}
        self.biases = {n: 0.1 * r(s[1]) for n, s in sizes.items()}
        self.x, self.table = r(batch * seq, w), r(8, heads)
        self.teacher, self.labels = 3 * r(batch * seq, kept), rng.integers(0, vocab, batch * seq).astype(np.int32)
        self.index = rng.integers(0, vocab, (batch * seq, kept)).astype(np.int32)
        self.labels[::5] = -1                               # rows without a label
        self.index[1::4, 0] = vocab                         # entries outside the vocabulary

    def plain(self, dtype):
        t = lambda a: torch.tensor(a, dtype=dtype, requires_grad=True)
        W, B = {n: t(a) for n, a in self.weights.items()}, {n: t(a) for n, a in self.biases.items()}
        x, table = t(self.x), t(self.table)
        dense = lambda n, a: a @ W[n] + B[n]
        h = ACTS[self.acts[0]](dense("in", x))
        cut = lambda a, n: a.reshape(self.batch, self.seq, n, self.d).transpose(1, 2)
        q, k, v = cut(dense("q", h), self.heads), cut(dense("k", h), self.kv_heads), cut(dense("v", h), self.kv_heads)
        group = self.heads // self.kv_heads
        k, v = k.repeat_interleave(group, 1), v.repeat_interleave(group, 1)
        rel = np.arange(self.seq)[None] - np.arange(self.seq)[:, None]
        idx = torch.tensor(np.vectorize(lambda r: oc.bucket(int(r), 8, 32, not self.causal))(rel))
        s = self.d ** -0.5 * (q @ k.transpose(2, 3)) + table[idx].permute(2, 0, 1)[None]
        off = torch.arange(self.seq)[None, :] >= torch.tensor(self.lens)[:, None]
        off = off[:, None, None, :] | (torch.tensor(rel > 0) & self.causal)[None, None]
        s = s.masked_fill(off, float("-inf"))
        dead = off.all(-1, keepdim=True)
        p = torch.softmax(s.masked_fill(dead, 0.0), -1).masked_fill(dead, 0.0)
        a = (p @ v).transpose(1, 2).reshape(x.shape)
        y = ACTS[self.acts[1]](dense("o", a)) + h
        z = dense("head", y)
        T, alpha, rows = 2.0, 0.75, x.shape[0]
        index = torch.tensor(self.index).long()
        ok = index < self.vocab
        pt = torch.softmax(torch.tensor(self.teacher, dtype=dtype).masked_fill(~ok, float("-inf")) / T, -1)
        logq = torch.log_softmax(z / T, -1).gather(1, index.clamp(max=self.vocab - 1))
        soft = torch.where(ok, pt * (torch.log(pt.clamp(min=1e-30)) - logq), torch.zeros((), dtype=dtype)).sum()
        label = torch.tensor(self.labels).long()
        hard = -torch.log_softmax(z, -1).gather(1, label.clamp(min=0)[:, None])[:, 0].masked_fill(label < 0, 0.0).sum()
        loss = (alpha * T * T * soft + (1 - alpha) * hard) / rows
        a.retain_grad()
        loss.backward()
        out = {"loss": loss, "logits": z, "x": x.grad, "table": table.grad}
        out.update({f"w_{n}": p.grad for n, p in W.items()})
        out.update({f"b_{n}": p.grad for n, p in B.items()})
        # what gradients of the scores alone sum, by magnitude
        mag = p * (cut(a.grad.abs(), self.heads) @ v.abs().transpose(2, 3))
        fold = lambda m: m.reshape(self.batch, -1, group, self.seq, self.d).sum(2)
        rows = lambda m: m.transpose(1, 2).reshape(x.shape[0], -1)
        mq, mk = rows(self.d ** -0.5 * mag @ k.abs()), rows(fold(self.d ** -0.5 * mag.transpose(2, 3) @ q.abs()))
        out["mass"] = torch.stack([mag.sum(), (h.abs().T @ mq).max(), mq.sum(0).max(), (h.abs().T @ mk).max(), mk.sum(0).max()])
        return {n: p.detach().double().numpy().reshape(-1) for n, p in out.items()}

    def layers(self, api):
        made = {}
        for n, w in self.weights.items():
            made[n] = api.boat_dense_layer_create(w.shape[0], w.shape[1], True)
            api.write(api.boat_dense_layer_get_weight(made[n]), w)
            api.write(api.boat_dense_layer_get_bias(made[n]), self.biases[n])
        return made

    def run(self, api, layers, x, table, keep_names=True):
        """forward and backward; variables of the middle are freed before the backward pass"""
        import boat_amd.capi as capi
        plan = capi.RelativeAttentionConfig(8, 32, not self.causal, self.causal, 0, self.d ** -0.5)
        consts = [api.tensor(a) for a in (np.array(self.lens, np.int32), self.teacher, self.index, self.labels)]
        dense = lambda n, a, act=-1, res=None: api.boat_hip_var_dense_act(a, layers[n], act, res)
        h = dense("in", x, self.acts[0])
        flat = [dense(n, h) for n in "qkv"]
        cut = [api.boat_hip_var_reshape(f, *shape(self.batch, self.seq, n, self.d)) for f, n in zip(flat, (self.heads, self.kv_heads, self.kv_heads))]
        a4 = api.boat_hip_var_relative_attention(C.byref(plan), *cut, table, consts[0])
        a = api.boat_hip_var_reshape(a4, *shape(self.batch * self.seq, self.heads * self.d))
        y = dense("o", a, self.acts[1], h)
        z = dense("head", y)
        loss = api.boat_hip_var_distillation_loss(z, *consts[1:], 2.0, 0.75)
        assert loss
        got = {"logits": api.numpy(api.boat_variable_data(z)), "loss": api.numpy(api.boat_variable_data(loss))}
        for t in consts:
            api.boat_tensor_unref(t)
        for v in [h, *flat, *cut, a4, a, y, z]:
            api.boat_variable_free(v)
        api.boat_variable_backward_full(loss)
        api.boat_variable_free(loss)
        return got


def gradients(api, layers, x, table):
    got = {"x": api.numpy(api.boat_variable_grad(x)), "table": api.numpy(api.boat_variable_grad(table))}
    for n, l in layers.items():
        got[f"w_{n}"] = api.numpy(api.boat_dense_layer_get_grad_weight(l))
        got[f"b_{n}"] = api.numpy(api.boat_dense_layer_get_grad_bias(l))
    return got


def compare(got, want, single, d, times=1):
    for n, value in got.items():
        scale = np.abs(want[n]).max()
        tol = 4 * np.abs(single[n] - want[n]).max() + 2.0 ** -22 * scale
        mass = dict(zip(("table", "w_q", "b_q", "w_k", "b_k"), want["mass"])).get(n, 0)
        if scale <= 2.0 ** -40 * mass:
            tol += (2 * d + 8) * 2.0 ** -24 * mass
        err = np.abs(value.reshape(-1).astype(np.float64) - times * want[n]).max()
        assert np.isfinite(value).all() and err <= times * tol, (n, err, tol, scale)


@pytest.mark.parametrize("change", [
    {}, dict(causal=True, acts=(0, 1)), dict(batch=1, seq=1, lens=(1,)), dict(heads=5, kv_heads=5, d=8, acts=(1, 3)),
    dict(batch=2, seq=130, heads=2, kv_heads=1, d=33, lens=(1, 130), acts=(2, -1), vocab=1003),
])
def test_block_trains_against_a_teacher(boat, rng, change):
    boat.boat_clear_error()                                 # other tests' refusals are not this one's
    block = Block(rng, **change)
    want, single = block.plain(torch.float64), block.plain(torch.float32)
    layers = block.layers(boat)
    tx, tt = boat.tensor(block.x), boat.tensor(block.table)
    x, table = boat.boat_variable_create(tx, True), boat.boat_variable_create(tt, True)
    compare(block.run(boat, layers, x, table), want, single, block.d)
    compare(gradients(boat, layers, x, table), want, single, block.d)
    block.run(boat, layers, x, table)                       # a second step without a zero_grad adds the same once more
    compare(gradients(boat, layers, x, table), want, single, block.d, times=2)
    for v in (x, table):
        boat.boat_variable_free(v)
    for t in (tx, tt):
        boat.boat_tensor_unref(t)
    for l in layers.values():
        boat.boat_dense_layer_free(l)
    assert not boat.boat_has_error()


def test_only_what_requires_a_gradient_gets_one(boat, rng):
    layer = boat.boat_dense_layer_create(6, 6, True)
    x, r = (boat.tensor(rng.standard_normal((4, 6)).astype(np.float32)) for _ in range(2))
    vx, vr = boat.boat_variable_create(x, False), boat.boat_variable_create(r, True)
    y = boat.boat_hip_var_dense_act(vx, layer, 3, vr)
    boat.boat_variable_backward_full(y)
    assert not boat.boat_variable_grad(vx)
    assert np.all(boat.numpy(boat.boat_variable_grad(vr)) == 1)
    # the layer learns even where its input needs no gradient, as long as the op was recorded
    assert np.abs(boat.numpy(boat.boat_dense_layer_get_grad_weight(layer))).max() > 0
    boat.boat_variable_free(y)
    alone = boat.boat_hip_var_dense_act(vx, layer, 3, None)
    assert not boat.boat_variable_requires_grad(alone)
    for v in (alone, vx, vr):
        boat.boat_variable_free(v)
    for t in (x, r):
        boat.boat_tensor_unref(t)
    boat.boat_dense_layer_free(layer)


def test_the_residual_may_be_the_input(boat, rng):
    """y = x + tanh(x W + b): both contributions reach x, and data reset before the backward pass does not change them"""
    w, xs = (rng.standard_normal((8, 8)) / 3).astype(np.float32), rng.standard_normal((5, 8)).astype(np.float32)
    layer = boat.boat_dense_layer_create(8, 8, False)
    boat.write(boat.boat_dense_layer_get_weight(layer), w)
    t, other = boat.tensor(xs), boat.tensor(np.zeros((5, 8), np.float32))
    x = boat.boat_variable_create(t, True)
    y = boat.boat_hip_var_dense_act(x, layer, 2, x)
    assert boat.boat_variable_reset_data(x, other)
    boat.boat_variable_backward_full(y)
    slope = 1 - np.tanh(xs.astype(np.float64) @ w) ** 2
    want = 1 + slope @ w.T.astype(np.float64)
    # eight products and their sums, the slope's rounding, and the final sum: 24 roundings of values at most |slope| . |w|^T + 1
    bound = 24 * 2.0 ** -24 * (1 + slope @ np.abs(w.T)) + 2 * 2.0 ** -24 * 8 * np.abs(xs).max() * np.abs(w).max() * np.abs(w).sum(1)
    assert np.all(np.abs(boat.numpy(boat.boat_variable_grad(x)) - want) <= bound)
    assert np.allclose(boat.numpy(boat.boat_dense_layer_get_grad_weight(layer)), xs.T.astype(np.float64) @ slope, rtol=0, atol=1e-4)
    for v in (y, x):
        boat.boat_variable_free(v)
    for s in (t, other):
        boat.boat_tensor_unref(s)
    boat.boat_dense_layer_free(layer)


def test_without_recording_nothing_is_kept(boat, rng):
    layer = boat.boat_dense_layer_create(6, 4, True)
    t = boat.tensor(rng.standard_normal((3, 6)).astype(np.float32))
    x = boat.boat_variable_create(t, True)
    context = boat.boat_autodiff_get_current_context()
    boat.boat_autodiff_context_disable_grad(context)
    y = boat.boat_hip_var_dense_act(x, layer, 3, None)
    boat.boat_autodiff_context_enable_grad(context)
    boat.boat_variable_backward_full(y)
    assert not boat.boat_variable_grad(x)
    for v in (y, x):
        boat.boat_variable_free(v)
    boat.boat_tensor_unref(t)
    boat.boat_dense_layer_free(layer)
