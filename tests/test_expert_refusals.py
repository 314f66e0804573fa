"""Calls of the expert and adapter operators that are refused before any device work (CPU)."""
import ctypes

import pytest
import torch

from logos_amd import _lib, vedic

P = 4096  # a non-null address that no refused call reads


def grouped(**kw):
    d = dict(op=0, in_dtype=1, out_dtype=0, epilogue=0, groups=2, rows=8, M=16, N=16, K=16, offsets=P, row_index=None,
             a_rows=8, A=P, lda=16, B=P, ldb=16, stride_b=256, C=P, ldc=16, stride_c=256, bias=None, preact=None,
             ld_preact=0, beta=0.0, db=None, db_beta=0.0, stream=None)
    d.update(kw)
    return _lib.load().vedic_gemm_grouped(ctypes.byref(_lib.GroupedDesc(**d)))


@pytest.mark.parametrize("kw,status", [
    (dict(op=3), _lib.STATUS_BAD_LAYOUT),
    (dict(in_dtype=2), _lib.STATUS_BAD_DTYPE),
    (dict(in_dtype=0, out_dtype=1), _lib.STATUS_BAD_DTYPE),
    (dict(op=2, out_dtype=1), _lib.STATUS_BAD_DTYPE),
    (dict(groups=0), _lib.STATUS_BAD_DIM),
    (dict(rows=-1), _lib.STATUS_BAD_DIM),
    (dict(N=0), _lib.STATUS_BAD_DIM),
    (dict(K=0), _lib.STATUS_BAD_DIM),
    (dict(op=2, M=0), _lib.STATUS_BAD_DIM),
    (dict(row_index=P, a_rows=0), _lib.STATUS_BAD_DIM),
    (dict(epilogue=1), _lib.STATUS_BAD_EPILOGUE),                    # no bias
    (dict(op=1, epilogue=1, bias=P), _lib.STATUS_BAD_EPILOGUE),      # NT has none
    (dict(epilogue=4, preact=P, ld_preact=16), _lib.STATUS_BAD_EPILOGUE),
    (dict(op=1, epilogue=4), _lib.STATUS_BAD_EPILOGUE),              # no pre-activation
    (dict(preact=P, ld_preact=16), _lib.STATUS_BAD_EPILOGUE),        # nothing to do with it
    (dict(epilogue=5), _lib.STATUS_BAD_EPILOGUE),
    (dict(beta=1.0), _lib.STATUS_BAD_EPILOGUE),
    (dict(op=2, beta=float("nan")), _lib.STATUS_BAD_EPILOGUE),
    (dict(db=P), _lib.STATUS_BAD_EPILOGUE),
    (dict(offsets=None), _lib.STATUS_NULL_POINTER),
    (dict(A=None), _lib.STATUS_NULL_POINTER),
    (dict(C=None), _lib.STATUS_NULL_POINTER),
    (dict(op=2, rows=0, C=None), _lib.STATUS_NULL_POINTER),
    (dict(lda=15), _lib.STATUS_BAD_LD),
    (dict(ldb=15), _lib.STATUS_BAD_LD),
    (dict(ldc=15), _lib.STATUS_BAD_LD),
    (dict(epilogue=2, bias=P, preact=P, ld_preact=15), _lib.STATUS_BAD_LD),
    (dict(stride_b=-1), _lib.STATUS_BAD_LD),
    (dict(op=2, stride_c=255), _lib.STATUS_BAD_LD),                  # groups of dW that overlap
    (dict(groups=1025), _lib.STATUS_TOO_LARGE),
    (dict(lda=1 << 22), _lib.STATUS_TOO_LARGE),
    (dict(rows=1 << 30), _lib.STATUS_TOO_LARGE),
    (dict(rows=0), _lib.STATUS_OK),                                  # nothing to do
])
def test_grouped(kw, status):
    assert grouped(**kw) == status


def test_null_descriptor():
    assert _lib.load().vedic_gemm_grouped(None) == _lib.STATUS_NULL_POINTER


@pytest.mark.parametrize("args,status", [
    ((P, 8, -1, 8, 2, 1, P, P, P, P, P, None), _lib.STATUS_BAD_DIM),
    ((P, 8, 4, 8, 0, 1, P, P, P, P, P, None), _lib.STATUS_BAD_DIM),
    ((P, 8, 4, 8, 9, 1, P, P, P, P, P, None), _lib.STATUS_BAD_DIM),
    ((P, 2000, 4, 2000, 2, 1, P, P, P, P, P, None), _lib.STATUS_TOO_LARGE),
    ((P, 100, 4, 100, 65, 1, P, P, P, P, P, None), _lib.STATUS_TOO_LARGE),
    ((P, 8, 1 << 29, 8, 2, 1, P, P, P, P, P, None), _lib.STATUS_TOO_LARGE),
    ((P, 7, 4, 8, 2, 1, P, P, P, P, P, None), _lib.STATUS_BAD_LD),
    ((None, 8, 4, 8, 2, 1, P, P, P, P, P, None), _lib.STATUS_NULL_POINTER),
    ((P, 8, 4, 8, 2, 1, P, P, None, P, P, None), _lib.STATUS_NULL_POINTER),
])
def test_route(args, status):
    assert _lib.load().vedic_route_topk(*args) == status


@pytest.mark.parametrize("args,status", [
    ((P, 8, P, P, P, 4, 8, 9, 1, P, 8, None), _lib.STATUS_BAD_DIM),
    ((P, 8, P, P, P, 4, 8, 2, 1, P, 7, None), _lib.STATUS_BAD_LD),
    ((P, 8, P, P, None, 4, 8, 2, 1, P, 8, None), _lib.STATUS_NULL_POINTER),
    ((None, 8, None, None, None, 0, 8, 2, 1, None, 8, None), _lib.STATUS_OK),
])
def test_route_backward(args, status):
    assert _lib.load().vedic_route_topk_bwd(*args) == status


@pytest.mark.parametrize("args,status", [
    ((P, -1, 1, 4, P, P, P, None), _lib.STATUS_BAD_DIM),
    ((P, 4, 0, 4, P, P, P, None), _lib.STATUS_BAD_DIM),
    ((P, 4, 1, 0, P, P, P, None), _lib.STATUS_BAD_DIM),
    ((P, 4, 1, 1025, P, P, P, None), _lib.STATUS_TOO_LARGE),
    ((None, 4, 1, 4, P, P, P, None), _lib.STATUS_NULL_POINTER),
])
def test_group_rows(args, status):
    assert _lib.load().vedic_group_rows(*args) == status


@pytest.mark.parametrize("args,status", [
    ((P, 2, 8, 4, P, P, None, 0, P, 8, 2, 2, 8, None), _lib.STATUS_BAD_DTYPE),
    ((P, 0, 8, 4, P, P, None, 0, P, 8, 2, 0, 8, None), _lib.STATUS_BAD_DIM),
    ((P, 0, 7, 4, P, P, None, 0, P, 8, 2, 2, 8, None), _lib.STATUS_BAD_LD),
    ((P, 0, 8, 4, P, P, P, 7, P, 8, 2, 2, 8, None), _lib.STATUS_BAD_LD),
    ((P, 0, 8, 4, None, P, None, 0, P, 8, 2, 2, 8, None), _lib.STATUS_NULL_POINTER),
    ((P, 0, 8, 4, P, P, None, 0, P, 8, 0, 2, 8, None), _lib.STATUS_OK),
])
def test_combine(args, status):
    assert _lib.load().vedic_combine_rows(*args) == status


@pytest.mark.parametrize("args,status", [
    ((P, 8, P, 0, 8, 4, P, P, P, 2, 8, P, 2, 2, 8, None), _lib.STATUS_BAD_DTYPE),
    ((P, 8, P, 0, 8, 4, P, P, P, 1, 7, P, 2, 2, 8, None), _lib.STATUS_BAD_LD),
    ((P, 8, P, 0, 8, 4, P, None, P, 1, 8, P, 2, 2, 8, None), _lib.STATUS_NULL_POINTER),
])
def test_combine_backward(args, status):
    assert _lib.load().vedic_combine_rows_bwd(*args) == status


@pytest.mark.parametrize("args,status", [
    ((P, 2, 8, 4, P, P, 2, 4, P, P, 4, None, P, 8, 8, 8, None), _lib.STATUS_BAD_DTYPE),
    ((P, 1, 8, 4, P, P, 2, 0, P, P, 4, None, P, 8, 8, 8, None), _lib.STATUS_BAD_DIM),
    ((P, 1, 8, 4, P, P, 2, 129, P, P, 4, None, P, 8, 8, 8, None), _lib.STATUS_TOO_LARGE),
    ((P, 1, 7, 4, P, P, 2, 4, P, P, 4, None, P, 8, 8, 8, None), _lib.STATUS_BAD_LD),
    ((P, 1, 8, 4, None, P, 2, 4, P, P, 4, None, P, 8, 8, 8, None), _lib.STATUS_NULL_POINTER),
    ((None, 1, 8, 4, None, None, 2, 4, None, None, 0, None, None, 8, 8, 8, None), _lib.STATUS_OK),
])
def test_lora(args, status):
    assert _lib.load().vedic_lora_add(*args) == status


@pytest.mark.parametrize("kw,args,status", [
    (dict(op=1), (P, P, 2, 4, P, P, 4, None), _lib.STATUS_BAD_LAYOUT),
    (dict(in_dtype=2), (P, P, 2, 4, P, P, 4, None), _lib.STATUS_BAD_DTYPE),
    (dict(out_dtype=1), (P, P, 2, 4, P, P, 4, None), _lib.STATUS_BAD_DTYPE),
    (dict(epilogue=2, bias=P), (P, P, 2, 4, P, P, 4, None), _lib.STATUS_BAD_EPILOGUE),
    (dict(preact=P), (P, P, 2, 4, P, P, 4, None), _lib.STATUS_BAD_EPILOGUE),
    (dict(), (P, P, 2, 129, P, P, 4, None), _lib.STATUS_TOO_LARGE),
    (dict(), (None, P, 2, 4, P, P, 4, None), _lib.STATUS_NULL_POINTER),
    (dict(epilogue=1), (P, P, 2, 4, P, P, 0, None), _lib.STATUS_BAD_EPILOGUE),  # the product's own refusal: no bias
    (dict(epilogue=1), (P, P, 2, 4, P, P, 4, None), _lib.STATUS_BAD_EPILOGUE),
    (dict(B=None), (P, P, 2, 4, P, P, 4, None), _lib.STATUS_NULL_POINTER),
    (dict(ldb=7), (P, P, 2, 4, P, P, 4, None), _lib.STATUS_BAD_LD),
])
def test_gemm_lora(kw, args, status):
    d = dict(op=0, in_dtype=1, out_dtype=0, M=8, N=8, K=8, A=P, lda=8, B=P, ldb=8, C=P, ldc=8, alpha=1.0, beta=0.0,
             bias=None, epilogue=0, preact=None, ld_preact=0, stream=None)
    d.update(kw)
    assert _lib.load().vedic_gemm_lora(ctypes.byref(_lib.GemmDesc(**d)), *args) == status
    assert _lib.load().vedic_gemm_lora(None, *args) == _lib.STATUS_NULL_POINTER


@pytest.mark.parametrize("args,status", [
    ((P, 2, 8, 4, 8, P, 2, 0.0, P, None), _lib.STATUS_BAD_DTYPE),
    ((P, 1, 7, 4, 8, P, 2, 0.0, P, None), _lib.STATUS_BAD_LD),
    ((P, 1, 8, 4, 8, None, 2, 0.0, P, None), _lib.STATUS_NULL_POINTER),
    ((P, 1, 8, 4, 8, P, 1025, 0.0, P, None), _lib.STATUS_TOO_LARGE),
])
def test_bias_grad(args, status):
    assert _lib.load().vedic_bias_grad_grouped(*args) == status


def test_operands_on_the_cpu():
    x, i = torch.zeros(4, 8), torch.zeros(3, dtype=torch.int32)
    for call in (lambda: vedic.route_topk(x, 2), lambda: vedic.group_rows(i, 2),
                 lambda: vedic.gemm_grouped(vedic.OP_NN, x, torch.zeros(2, 8, 8), i),
                 lambda: vedic.combine_rows(x, torch.zeros(2, 2, dtype=torch.int32)),
                 lambda: vedic.gemm_lora(x, torch.zeros(8, 8), torch.zeros(2, 8, 4), torch.zeros(2, 4, 8), i, i)):
        with pytest.raises(ValueError):
            call()
