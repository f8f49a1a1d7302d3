"""The fused training operators refuse what they cannot take before they touch the device: these calls run without a GPU."""
import ctypes as C

import pytest

hip = pytest.importorskip("boat_amd.hip")
ANY = C.c_void_p(64)      # a pointer that is never followed


def refused(rc, text):
    assert rc == -1
    assert text in hip.bh_last_error().decode()


def gemm(m=4, n=4, k=4, a=ANY, lda=4, b=ANY, ldb=4, c=ANY, ldc=4, bias=None, act=-1, saved=None, lds=4, residual=None, ldr=4, ta=0, tb=0):
    return hip.bh_gemm_epilogue(ta, tb, m, n, k, a, lda, b, ldb, c, ldc, bias, act, saved, lds, residual, ldr)


@pytest.mark.parametrize("change,text", [
    (dict(m=-1), "negative"), (dict(n=-1), "negative"), (dict(k=-1), "negative"),
    (dict(act=-2), "activation"), (dict(act=4), "activation"),
    (dict(a=None), "null"), (dict(b=None), "null"), (dict(c=None), "null"),
    (dict(lda=3), "leading"), (dict(ldb=3), "leading"), (dict(ldc=3), "leading"),
    (dict(saved=ANY, lds=3), "leading"), (dict(residual=ANY, ldr=3), "leading"),
    (dict(ta=1, m=5), "leading"), (dict(tb=1, k=5, lda=5), "leading"),
])
def test_product_refusals(change, text):
    refused(gemm(**change), text)


def test_empty_products_need_no_device():
    assert gemm(m=0, a=None, b=None, c=None) == 0
    assert gemm(n=0, a=None, b=None, c=None) == 0


@pytest.mark.parametrize("change,text", [
    (dict(m=-1), "negative"), (dict(act=7), "activation"), (dict(dy=None), "null"), (dict(w=None), "null"), (dict(x=None), "null"),
    (dict(act=3, saved=None), "null"),
])
def test_dense_backward_refusals(change, text):
    a = dict(act=-1, x=ANY, w=ANY, saved=ANY, dy=ANY, dx=ANY, gw=ANY, gb=ANY, m=4, k=4, n=4)
    a.update(change)
    refused(hip.bh_dense_act_backward(*a.values(), 0), text)


def distill_args(**change):
    a = dict(z=ANY, ld=100, teacher=ANY, index=ANY, labels=None, rows=3, vocab=100, topk=5, temperature=1.0, alpha=0.5, scale=1.0)
    a.update(change)
    return list(a.values())


@pytest.mark.parametrize("change,text", [
    (dict(rows=-1), "rows"), (dict(vocab=0, ld=0), "vocab"), (dict(topk=-1), "topk"), (dict(topk=4097), "topk"), (dict(ld=99), "leading"),
    (dict(vocab=1 << 31, ld=1 << 31), "vocabulary"), (dict(temperature=0.0), "temperature"), (dict(temperature=-1.0), "temperature"),
    (dict(temperature=float("nan")), "temperature"), (dict(temperature=float("inf")), "temperature"),
    (dict(alpha=-0.1), "alpha"), (dict(alpha=1.1), "alpha"), (dict(alpha=float("nan")), "alpha"),
    (dict(z=None), "null"), (dict(teacher=None), "null"), (dict(index=None), "null"),
])
def test_distillation_refusals(change, text):
    refused(hip.bh_distill_forward(*distill_args(**change), None, None, ANY), text)
    refused(hip.bh_distill_loss_grad(*distill_args(**change), None, None, ANY, 1 << 40), text)
    refused(hip.bh_distill_backward(*distill_args(**change), ANY, None, ANY, 1 << 40), text)


def test_a_residual_in_place_has_the_outputs_rows():
    refused(gemm(residual=ANY, ldr=5), "in place")


@pytest.mark.parametrize("temperature", [2e19, 1e-39, 3e38])
def test_distillation_refuses_temperatures_out_of_range(temperature):
    refused(hip.bh_distill_forward(*distill_args(temperature=temperature), None, None, ANY), "temperature")


def test_distillation_refuses_more_rows_than_a_launch_holds():
    refused(hip.bh_distill_forward(*distill_args(rows=(1 << 22) + 1), None, None, ANY), "too many rows")


def test_distillation_gradient_refusals():
    refused(hip.bh_distill_loss_grad(*distill_args(), None, None, ANY, 99), "leading")
    refused(hip.bh_distill_loss_grad(*distill_args(), None, None, None, 100), "null")
    refused(hip.bh_distill_loss_grad(*distill_args(), None, None, ANY, 101), "in place")
    refused(hip.bh_distill_backward(*distill_args(), None, None, C.c_void_p(128), 100), "null")
    refused(hip.bh_distill_backward(*distill_args(), ANY, None, ANY, 101), "in place")


# ------------------------------------------------------------------ attention with a relative position bias

@pytest.mark.parametrize("buckets,distance,both", [(32, 128, 1), (32, 128, 0), (2, 2, 0), (4, 5, 1), (3, 9, 0), (48, 250, 1), (64, 1024, 0), (256, 100000, 0),
                                                   (256, 129, 0), (16, 64, 1)])
def test_buckets_against_whole_numbers(buckets, distance, both):
    import operator_cases as oc
    for r in list(range(-300, 301)) + [-distance, distance, -distance - 1, distance - 1, 1 - distance, 10 ** 12, -10 ** 12]:
        assert hip.bh_relative_position_bucket(r, buckets, distance, both) == oc.bucket(r, buckets, distance, both), r


@pytest.mark.parametrize("buckets,distance,both", [(1, 10, 0), (0, 10, 0), (257, 1000, 0), (5, 100, 1), (2, 100, 1), (32, 16, 0), (32, 8, 1), (32, -1, 0)])
def test_bucket_refusals(buckets, distance, both):
    assert hip.bh_relative_position_bucket(3, buckets, distance, both) == -1
    assert "buckets" in hip.bh_last_error().decode()


def description(**change):
    a = dict(batch=2, heads=4, kv_heads=2, sq=3, sk=5, d=8, q_stride=(96, 24, 8), k_stride=(80, 40, 8), v_stride=(80, 40, 8), o_stride=(96, 24, 8),
             query_offset=2, num_buckets=8, max_distance=20, bidirectional=0, causal=1, scale=1.0)
    a.update(change)
    return hip.relbias_attention(**a)


@pytest.mark.parametrize("change,text", [
    (dict(batch=-1), "negative"), (dict(sq=-1), "negative"), (dict(sk=-1), "negative"), (dict(d=0), "head size"), (dict(d=129), "head size"),
    (dict(kv_heads=3), "multiple"), (dict(kv_heads=0), "multiple"), (dict(sk=1 << 29), "2^28"), (dict(query_offset=-(1 << 29)), "2^28"),
    (dict(q_stride=(96, -24, 8)), "negative stride"), (dict(num_buckets=1), "buckets"), (dict(max_distance=4), "buckets"),
    (dict(bidirectional=1, num_buckets=7), "buckets"), (dict(scale=float("nan")), "scale"), (dict(scale=float("inf")), "scale"),
    (dict(batch=1 << 20, heads=1 << 12, kv_heads=1), "heads"),
])
def test_attention_refusals(change, text):
    p = description(**change)
    refused(hip.bh_relbias_attention_forward(p, ANY, ANY, ANY, ANY, None, ANY, ANY), text)
    refused(hip.bh_relbias_attention_backward(p, ANY, ANY, ANY, ANY, None, ANY, ANY, ANY, ANY, ANY, ANY, ANY, 0), text)


def test_attention_pointer_and_overlap_refusals():
    p = description()
    for at in (0, 1, 2, 3, 5, 6):
        args = [ANY] * 7
        args[at] = None
        refused(hip.bh_relbias_attention_forward(p, *args), "null")
    for at in (0, 1, 2, 3, 5, 6, 7, 8, 9, 10, 11):
        args = [ANY] * 12
        args[at] = None
        refused(hip.bh_relbias_attention_backward(p, *args, 0), "null")
    refused(hip.bh_relbias_attention_forward(None, *[ANY] * 7), "null")
    refused(hip.bh_relbias_attention_forward(description(o_stride=(96, 24, 7)), *[ANY] * 7), "overlap")
    refused(hip.bh_relbias_attention_forward(description(o_stride=(0, 24, 8)), *[ANY] * 7), "overlap")
    # a key that several sequences share (a stride of zero) can be read, but its gradient has no place
    refused(hip.bh_relbias_attention_backward(description(k_stride=(0, 40, 8)), *[ANY] * 12, 0), "overlap")
    refused(hip.bh_relbias_attention_backward(description(sq=0), *[ANY] * 12, 0), "without queries")


def test_empty_attention_needs_no_device():
    for change in (dict(batch=0), dict(sq=0), dict(heads=0)):
        assert hip.bh_relbias_attention_forward(description(**change), *[None] * 7) == 0
    assert hip.bh_relbias_attention_backward(description(batch=0), *[None] * 12, 0) == 0
