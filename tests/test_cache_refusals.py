"""Calls of the paged cache, attention over it and four-bit products that are refused before any device work (CPU)."""
import ctypes

import pytest
import torch

from logos_amd import _lib, vedic

P = 4096  # a non-null address that no refused call reads


def cache(**kw):
    d = dict(format=_lib.KV_F16, pages=4, page_size=16, heads=2, dh=64, k=P, v=P, stride_page=2048, stride_head=1024,
             stride_token=64, table=P, ld_table=2, table_cols=2, lens=P, q_start=P, batch=2, tokens=8)
    d.update(kw)
    return _lib.Kv(**d)


FOUR = dict(format=_lib.KV_I4, stride_page=1280, stride_head=640, stride_token=40)
CACHE = [
    (dict(format=2), _lib.STATUS_BAD_DTYPE),
    (dict(pages=0), _lib.STATUS_BAD_DIM),
    (dict(page_size=0), _lib.STATUS_BAD_DIM),
    (dict(heads=0), _lib.STATUS_BAD_DIM),
    (dict(dh=0), _lib.STATUS_BAD_DIM),
    (dict(dh=60), _lib.STATUS_BAD_DIM),
    (dict(dh=264), _lib.STATUS_BAD_DIM),
    (dict(FOUR, dh=72), _lib.STATUS_BAD_DIM),
    (dict(table_cols=0), _lib.STATUS_BAD_DIM),
    (dict(batch=-1), _lib.STATUS_BAD_DIM),
    (dict(tokens=-1), _lib.STATUS_BAD_DIM),
    (dict(q_start=None), _lib.STATUS_BAD_DIM),                # 8 rows of 2 sequences
    (dict(page_size=1 << 30), _lib.STATUS_TOO_LARGE),
    (dict(batch=1 << 20), _lib.STATUS_TOO_LARGE),
    (dict(tokens=1 << 29), _lib.STATUS_TOO_LARGE),
    (dict(k=None), _lib.STATUS_NULL_POINTER),
    (dict(v=None), _lib.STATUS_NULL_POINTER),
    (dict(table=None), _lib.STATUS_NULL_POINTER),
    (dict(lens=None), _lib.STATUS_NULL_POINTER),
    (dict(k=P + 8), _lib.STATUS_BAD_LD),
    (dict(FOUR, v=P + 2), _lib.STATUS_BAD_LD),
    (dict(stride_token=56), _lib.STATUS_BAD_LD),
    (dict(stride_token=68), _lib.STATUS_BAD_LD),
    (dict(FOUR, stride_token=42), _lib.STATUS_BAD_LD),
    (dict(stride_head=0), _lib.STATUS_BAD_LD),
    (dict(stride_page=-64), _lib.STATUS_BAD_LD),
    (dict(ld_table=1), _lib.STATUS_BAD_LD),
]


def append(kv, **kw):
    d = dict(dtype=1, q=P, q_token=256, q_head=64, q_heads=4, q_out=2 * P, q_out_token=256, q_out_head=64, k=P, k_token=128,
             k_head=64, v=P, v_token=128, v_head=64, rope=P, rope_rows=32, rope_dims=64, interleaved=0, stream=None)
    d.update(kw)
    return _lib.load().vedic_kv_append(None if kv is None else ctypes.byref(kv), *d.values())


def attend(kv, **kw):
    d = dict(q=P, q_token=256, q_head=64, q_heads=4, out=2 * P, out_token=256, out_head=64, lse=None, scale=1.0, causal=1,
             window=0, stride=0, stream=None)
    d.update(kw)
    return _lib.load().vedic_paged_attention(None if kv is None else ctypes.byref(kv), *d.values())


def read(kv, k=P, v=P):
    return _lib.load().vedic_kv_read(None if kv is None else ctypes.byref(kv), k, v, None)


@pytest.mark.parametrize("call", [append, attend, read])
@pytest.mark.parametrize("kw,status", CACHE)
def test_cache(call, kw, status):
    assert call(cache(**kw)) == status


@pytest.mark.parametrize("call", [append, attend, read])
def test_nothing_to_do(call):
    assert call(None) == _lib.STATUS_NULL_POINTER
    assert call(cache(tokens=0)) == _lib.STATUS_OK
    assert call(cache(batch=0, k=None, table=None)) == _lib.STATUS_OK


@pytest.mark.parametrize("kw,status", [
    (dict(dtype=2), _lib.STATUS_BAD_DTYPE),
    (dict(q_heads=-1), _lib.STATUS_BAD_DIM),
    (dict(rope_dims=-2), _lib.STATUS_BAD_DIM),
    (dict(rope_dims=3), _lib.STATUS_BAD_DIM),
    (dict(rope_dims=66), _lib.STATUS_BAD_DIM),
    (dict(rope_rows=0), _lib.STATUS_BAD_DIM),
    (dict(q_heads=1 << 16), _lib.STATUS_TOO_LARGE),
    (dict(k=None), _lib.STATUS_NULL_POINTER),
    (dict(v=None), _lib.STATUS_NULL_POINTER),
    (dict(q=None), _lib.STATUS_NULL_POINTER),
    (dict(q_out=None), _lib.STATUS_NULL_POINTER),
    (dict(rope=None), _lib.STATUS_NULL_POINTER),
    (dict(q_out=P), _lib.STATUS_BAD_LD),                      # q itself
    (dict(q_out=2 * P + 8), _lib.STATUS_BAD_LD),
    (dict(q_out_token=56), _lib.STATUS_BAD_LD),               # tokens that overlap
    (dict(q_out_head=0), _lib.STATUS_BAD_LD),
    (dict(q_out_head=68), _lib.STATUS_BAD_LD),
    (dict(k_token=-1), _lib.STATUS_BAD_LD),
    (dict(v_head=-1), _lib.STATUS_BAD_LD),
    (dict(q_token=-1), _lib.STATUS_BAD_LD),
])
def test_append(kw, status):
    assert append(cache(), **kw) == status


@pytest.mark.parametrize("kw,status", [
    (dict(q_heads=0), _lib.STATUS_BAD_DIM),
    (dict(q_heads=3), _lib.STATUS_BAD_DIM),                   # not a multiple of the cache's two
    (dict(window=-1), _lib.STATUS_BAD_DIM),
    (dict(stride=-1, window=4), _lib.STATUS_BAD_DIM),
    (dict(stride=4), _lib.STATUS_BAD_DIM),                    # a stride without a window
    (dict(window=4, causal=0), _lib.STATUS_BAD_DIM),
    (dict(q_heads=1 << 16), _lib.STATUS_TOO_LARGE),
    (dict(q=None), _lib.STATUS_NULL_POINTER),
    (dict(out=None), _lib.STATUS_NULL_POINTER),
    (dict(out=P), _lib.STATUS_BAD_LD),                        # q itself
    (dict(q=P + 2), _lib.STATUS_BAD_LD),
    (dict(out=2 * P + 8), _lib.STATUS_BAD_LD),
    (dict(q_token=260), _lib.STATUS_BAD_LD),
    (dict(q_head=-64), _lib.STATUS_BAD_LD),
    (dict(out_token=56), _lib.STATUS_BAD_LD),
    (dict(out_head=0), _lib.STATUS_BAD_LD),
])
def test_attention(kw, status):
    assert attend(cache(), **kw) == status


def test_attention_of_more_workgroups_than_a_launch_takes():
    assert attend(cache(tokens=1 << 20, batch=(1 << 20) - 1, heads=32, stride_page=32768), q_heads=32) == _lib.STATUS_TOO_LARGE


def test_read():
    assert read(cache(), None, None) == _lib.STATUS_OK
    assert read(cache(), P + 8, P) == _lib.STATUS_BAD_LD
    assert read(cache(tokens=1 << 24)) == _lib.STATUS_TOO_LARGE


def weight(**kw):
    d = dict(codes=P, scales=P, K=64, N=32, group=64)
    d.update(kw)
    return _lib.W4Desc(**d)


def gemm(w, **kw):
    d = dict(X=P, x_dtype=1, ldx=64, M=4, C=P, c_dtype=0, ldc=32, bias=None, epilogue=0, stream=None)
    d.update(kw)
    return _lib.load().vedic_gemm_w4(None if w is None else ctypes.byref(w), *d.values())


def unpack(w, W=P, ldw=32):
    return _lib.load().vedic_w4_unpack(None if w is None else ctypes.byref(w), W, ldw, None)


@pytest.mark.parametrize("call", [gemm, unpack])
@pytest.mark.parametrize("kw,status", [
    (dict(K=0), _lib.STATUS_BAD_DIM),
    (dict(N=0), _lib.STATUS_BAD_DIM),
    (dict(group=16), _lib.STATUS_BAD_DIM),
    (dict(group=0), _lib.STATUS_BAD_DIM),
    (dict(K=1 << 22), _lib.STATUS_TOO_LARGE),
    (dict(N=1 << 22), _lib.STATUS_TOO_LARGE),
    (dict(codes=None), _lib.STATUS_NULL_POINTER),
    (dict(scales=None), _lib.STATUS_NULL_POINTER),
    (dict(codes=P + 4), _lib.STATUS_BAD_LD),
    (dict(scales=P + 2), _lib.STATUS_BAD_LD),
    (None, _lib.STATUS_NULL_POINTER),
])
def test_weight(call, kw, status):
    assert call(None if kw is None else weight(**kw)) == status


def test_unpack():
    assert unpack(weight(), None) == _lib.STATUS_NULL_POINTER
    assert unpack(weight(), P, 31) == _lib.STATUS_BAD_LD


@pytest.mark.parametrize("kw,status", [
    (dict(M=-1), _lib.STATUS_BAD_DIM),
    (dict(x_dtype=2), _lib.STATUS_BAD_DTYPE),
    (dict(c_dtype=2), _lib.STATUS_BAD_DTYPE),
    (dict(epilogue=1), _lib.STATUS_BAD_EPILOGUE),             # no bias
    (dict(epilogue=3, bias=P), _lib.STATUS_BAD_EPILOGUE),
    (dict(epilogue=4, bias=P), _lib.STATUS_BAD_EPILOGUE),
    (dict(epilogue=99), _lib.STATUS_BAD_EPILOGUE),
    (dict(epilogue=vedic.EPI_RESIDUAL, c_dtype=1), _lib.STATUS_BAD_EPILOGUE),
    (dict(ldx=1 << 22), _lib.STATUS_TOO_LARGE),
    (dict(ldc=1 << 22), _lib.STATUS_TOO_LARGE),
    (dict(M=1 << 30), _lib.STATUS_TOO_LARGE),
    (dict(X=None), _lib.STATUS_NULL_POINTER),
    (dict(C=None), _lib.STATUS_NULL_POINTER),
    (dict(ldx=63), _lib.STATUS_BAD_LD),
    (dict(ldc=31), _lib.STATUS_BAD_LD),
    (dict(M=0, X=None, C=None), _lib.STATUS_OK),
])
def test_gemm(kw, status):
    assert gemm(weight(), **kw) == status


@pytest.mark.parametrize("args,status", [
    ((P, 2, 32, 64, 32, 64, P, P, None), _lib.STATUS_BAD_DTYPE),
    ((P, 0, 32, 0, 32, 64, P, P, None), _lib.STATUS_BAD_DIM),
    ((P, 0, 32, 64, 32, 48, P, P, None), _lib.STATUS_BAD_DIM),
    ((None, 0, 32, 64, 32, 64, P, P, None), _lib.STATUS_NULL_POINTER),
    ((P, 0, 32, 64, 32, 64, None, P, None), _lib.STATUS_NULL_POINTER),
    ((P, 0, 31, 64, 32, 64, P, P, None), _lib.STATUS_BAD_LD),
])
def test_quantize(args, status):
    assert _lib.load().vedic_w4_quantize(*args) == status


def test_tensors_that_are_not_on_a_gpu():
    k, v = vedic.kv_cache(4, 16, 2, 64, device="cpu")
    table, lens = torch.zeros((3, 2), dtype=torch.int32), torch.ones(3, dtype=torch.int32)
    x = torch.zeros((3, 2, 64), dtype=torch.float16)
    w = vedic.W4(torch.zeros((8, 8), dtype=torch.int32), torch.zeros((8, 1, 2), dtype=torch.float16), 64, 64)
    for call in (lambda: vedic.kv_append(None, x, x, k, v, table, lens), lambda: vedic.kv_read(k, v, table, lens),
                 lambda: vedic.paged_attention(x, k, v, table, lens), lambda: vedic.gemm_w4(x[:, 0], w),
                 lambda: vedic.w4_quantize(x[:, 0]), lambda: vedic.w4_unpack(w)):
        with pytest.raises(ValueError):
            call()


@pytest.mark.parametrize("dh,four_bit", [(0, False), (60, False), (264, False), (40, True), (288, True)])
def test_cache_sizes(dh, four_bit):
    with pytest.raises(ValueError):
        vedic.kv_cache(4, 16, 2, dh, four_bit, device="cpu")
