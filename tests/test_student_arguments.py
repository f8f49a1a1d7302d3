"""The Boat-level forms of the fused training operators refuse tensors that do not fit before they touch the device."""
import ctypes as C

import numpy as np
import pytest

capi = pytest.importorskip("boat_amd.capi")


@pytest.fixture(scope="module")
def api():
    return capi.default_api()


def f32(*shape):
    return np.zeros(shape, np.float32)


def i32(*shape):
    return np.zeros(shape, np.int32)


def refused(api, arrays, call, text):
    made = [a if a is None else api.tensor(a) for a in arrays]
    api.boat_clear_error()
    assert not call(*made)
    assert text in api.boat_get_last_error_message().decode()
    api.boat_clear_error()
    for t in made:
        if t:
            api.boat_tensor_unref(t)


@pytest.mark.parametrize("x,act,residual,text", [
    (f32(3, 5), 3, None, "input"), (f32(3, 2, 2), 3, None, "input"), (np.zeros((3, 4)), 3, None, "input"), (f32(0, 4), 3, None, "input"),
    (f32(3, 4), 4, None, "activation"), (f32(3, 4), -2, None, "activation"),
    (f32(3, 4), 3, f32(3, 5), "residual"), (f32(3, 4), 3, f32(2, 6), "residual"), (f32(3, 4), 3, f32(6), "residual"),
    (f32(3, 4), 3, np.zeros((3, 6)), "residual"),
])
def test_dense_act_refusals(api, x, act, residual, text):
    layer = api.boat_dense_layer_create(4, 6, True)
    refused(api, [x, residual], lambda a, r: api.boat_hip_dense_act(layer, a, act, r, None), text)

    def tracked(a, r):
        va = api.boat_variable_create(a, True)
        vr = api.boat_variable_create(r, True) if r else None
        out = api.boat_hip_var_dense_act(va, layer, act, vr)
        for v in (va, vr):
            if v:
                api.boat_variable_free(v)
        return out
    refused(api, [x, residual], tracked, text)
    api.boat_dense_layer_free(layer)


GOOD = dict(q=f32(2, 3, 4, 8), k=f32(2, 5, 2, 8), v=f32(2, 5, 2, 8), table=f32(8, 4), lengths=i32(2))


@pytest.mark.parametrize("change,config,text", [
    (dict(q=f32(2, 3, 32)), {}, "query"), (dict(k=f32(2, 5, 2, 9)), {}, "query"), (dict(v=f32(2, 6, 2, 8)), {}, "query"),
    (dict(k=f32(3, 5, 2, 8), v=f32(3, 5, 2, 8)), {}, "query"), (dict(k=f32(2, 0, 2, 8), v=f32(2, 0, 2, 8)), {}, "query"),
    (dict(q=np.zeros((2, 3, 4, 8))), {}, "query"), (dict(table=f32(4, 8)), {}, "table"), (dict(table=f32(8)), {}, "table"),
    (dict(lengths=i32(3)), {}, "lengths"), (dict(lengths=f32(2)), {}, "lengths"), ({}, dict(num_buckets=6), "table"),
] + [pytest.param(*c, marks=pytest.mark.gpu) for c in [      # refused by the kernels' entry point, behind the tensors' upload
    (dict(k=f32(2, 5, 3, 8), v=f32(2, 5, 3, 8)), {}, "multiple"), ({}, dict(max_distance=1), "distance"),
    ({}, dict(scale=float("nan")), "scale"), ({}, dict(query_offset=1 << 40), "2^28"),
    (dict(q=f32(2, 3, 4, 136), k=f32(2, 5, 2, 136), v=f32(2, 5, 2, 136)), {}, "head size"),
]])
def test_relative_attention_refusals(api, change, config, text):
    fields = dict(num_buckets=8, max_distance=16, bidirectional=True, causal=False, query_offset=0, scale=1.0)
    fields.update(config)
    plan = capi.RelativeAttentionConfig(**fields)
    arrays = dict(GOOD)
    arrays.update(change)
    refused(api, [arrays[n] for n in ("q", "k", "v", "table", "lengths")],
            lambda q, k, v, t, n: api.boat_hip_relative_attention(C.byref(plan), q, k, v, t, n, None), text)


@pytest.mark.parametrize("z,teacher,index,labels,t,alpha,text", [
    (f32(3), f32(3, 2), i32(3, 2), None, 1.0, 0.5, "logits"), (np.zeros((3, 9)), f32(3, 2), i32(3, 2), None, 1.0, 0.5, "logits"),
    (f32(3, 9), f32(4, 2), i32(4, 2), None, 1.0, 0.5, "teacher"), (f32(3, 9), f32(3, 2), f32(3, 2), None, 1.0, 0.5, "INT32"),
    (f32(3, 9), f32(3, 2), i32(3, 3), None, 1.0, 0.5, "INT32"), (f32(3, 9), f32(3, 2), i32(3, 2), i32(4), 1.0, 0.5, "labels"),
    pytest.param(f32(3, 9), f32(3, 2), i32(3, 2), None, 0.0, 0.5, "temperature", marks=pytest.mark.gpu),
    pytest.param(f32(3, 9), f32(3, 2), i32(3, 2), None, 1.0, 1.5, "alpha", marks=pytest.mark.gpu),
])
def test_distillation_refusals(api, z, teacher, index, labels, t, alpha, text):
    def call(*made):
        grad = C.c_void_p(1)
        out = api.boat_hip_distillation_loss(*made, t, alpha, C.byref(grad))
        assert not grad.value
        return out
    refused(api, [z, teacher, index, labels], call, text)
