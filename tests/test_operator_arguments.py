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


def test_distillation_gradient_refusals():
    refused(hip.bh_distill_loss_grad(*distill_args(), None, None, ANY, 99), "leading")
    refused(hip.bh_distill_loss_grad(*distill_args(), None, None, None, 100), "null")
    refused(hip.bh_distill_loss_grad(*distill_args(), None, None, ANY, 101), "in place")
    refused(hip.bh_distill_backward(*distill_args(), None, None, C.c_void_p(128), 100), "null")
    refused(hip.bh_distill_backward(*distill_args(), ANY, None, ANY, 101), "in place")
