"""Python mirror of the LOGOS Vedic GEMM API over the gfx950 C ABI.

Names and argument meaning follow the reference:
  vedic_gemm(A, B)                 include/VedicGEMM.hpp:25-54 / cuda_vedic_gemm
  vedic_gemm_bias(A, W, bias)      include/VedicGEMM.hpp:56-65 / cuda_vedic_gemm_bias
  gemm_fp16_fp32out(A, B, ...)     cuda_gemm_fp16_fp32out (cuda/VedicGEMM.cu:1150)
  gemm_fp16_fp16out(A, B, ...)     cuda_gemm_fp16_fp16out (cuda/VedicGEMM.cu:1182)
  gemm_nt(dY, W) / gemm_tn(X, dY)  the NT/TN backward products (include/Backprop.hpp:48-63,
                                   cuda/train_gpu.cu:210-545)
  gemm_bias_gelu(X, W, b)          FeedForward::forward's first half (include/FeedForward.hpp:112-114)
  gemm_nt_gelu_bwd(dY, W, H)       ffn_da + gelu_bwd + bias_grad (cuda/train_gpu.cu:263-345), fused
  bias_grad(dY)                    bias_grad_kernel (cuda/train_gpu.cu:263-273), deterministic
  add_bias / gelu_ / cast_*        add_bias_kernel, cuda_gelu, cuda_cast_fp32_to_fp16 ...
  verify(A, B, C)                  cuda_vedic_verify (cuda/VedicGEMM.cu:765-814)
  flash_attention_fwd(Q, K, V)     cuda_flash_attention_fwd (cuda/VedicGEMM.cu:1065-1104)

New here, with no counterpart in the reference: products whose rows choose their weights.
  route_topk / route_topk_bwd      a router's choice, weights and plan, and its backward
  gemm_grouped(op, A, B, offsets)  the experts' products, forward and backward (bias_grad_grouped, group_rows)
  combine_rows / combine_rows_bwd  the experts' rows in token order, and the backward
  gemm_lora / lora_add             low-rank adapters of many requests beside a shared projection
and decoding with a paged cache of keys and values (binary16 or four bits) and four-bit weights:
  kv_cache / kv_append / kv_read   a cache, new tokens into it with their positions' rotation, and rows of it back
  paged_attention(q, k, v, ...)    attention of new tokens over it: one token a sequence, prompts, pieces of prompts
  gemm_w4(X, W4)                   products with four-bit weights (w4_quantize, w4_unpack)

Operands are torch tensors resident on the GPU (torch is used for device
memory and streams only); every call runs on torch's current stream.  Shape
errors raise ValueError (the reference's std::invalid_argument), device
errors RuntimeError (its std::runtime_error).
"""
from __future__ import annotations

import ctypes
from dataclasses import dataclass
from typing import NamedTuple

import torch

from . import _lib
from ._lib import (DT_F16, DT_F32, EPI_BIAS, EPI_BIAS_GELU, EPI_BIAS_RESIDUAL, EPI_GELU, EPI_GELU_BWD, EPI_NONE,
                   EPI_RESIDUAL, OP_NN, OP_NT, OP_TN)

__all__ = [
    "OP_NN", "OP_NT", "OP_TN", "EPI_NONE", "EPI_BIAS", "EPI_BIAS_GELU", "EPI_GELU", "EPI_GELU_BWD",
    "EPI_RESIDUAL", "EPI_BIAS_RESIDUAL", "gemm_bias_residual", "layernorm", "layernorm_fp16",
    "gemm", "vedic_gemm", "vedic_gemm_bias", "gemm_fp16_fp32out", "gemm_fp16_fp16out",
    "gemm_bias_gelu", "amp_gemm", "gemm_nt", "gemm_tn", "gemm_nt_gelu_bwd", "bias_grad", "gemm_scatter", "gemm_gather", "cast_stack_fp16",
    "cast_pack_fp16", "add_bias", "gelu_",
    "cast_fp32_to_fp16",
    "cast_fp16_to_fp32", "verify", "gemm_checked", "VerifyResult", "uses_vendor_blas", "backend_name",
    "flash_attention_fwd", "flash_attention_fwd_heads", "flash_attention_bwd", "flash_attention_bwd_heads",
    "Routing", "route_topk", "route_topk_bwd", "group_rows", "gemm_grouped", "bias_grad_grouped", "combine_rows",
    "combine_rows_bwd", "lora_add", "gemm_lora",
    "kv_cache", "kv_append", "kv_read", "paged_attention", "W4", "w4_quantize", "w4_unpack", "gemm_w4",
]

_DT = {torch.float32: DT_F32, torch.float16: DT_F16}


def _check(status: int) -> None:
    if status == _lib.STATUS_OK:
        return
    msg = _lib.status_string(status)
    if status in (_lib.STATUS_BAD_DIM, _lib.STATUS_BAD_LD, _lib.STATUS_BAD_LAYOUT,
                  _lib.STATUS_BAD_EPILOGUE, _lib.STATUS_BAD_DTYPE, _lib.STATUS_NULL_POINTER,
                  _lib.STATUS_TOO_LARGE, _lib.STATUS_UNSUPPORTED):
        raise ValueError(f"VedicGEMM: {msg}")
    code = _lib.load().vedic_last_hip_error()
    raise RuntimeError(f"VedicGEMM: {msg} (hipError {code})")


# torch's raw handle of a device's current stream: the stream object that
# torch.cuda.current_stream() builds for it costs 2.7 us per call, more than
# half of what a decode product takes on the GPU.
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def _stream() -> int:
    if _raw_stream is None:
        return torch.cuda.current_stream().cuda_stream
    return _raw_stream(torch.cuda.current_device())


def _mat(t: torch.Tensor, name: str) -> tuple[int, int, int]:
    """(rows, cols, leading dimension) of a row-major 2-D GPU matrix."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if not t.is_cuda:
        raise ValueError(f"{name} must be on the GPU")
    shape = t.shape
    if len(shape) == 1:
        return _mat(t.view(1, -1), name)
    if len(shape) != 2:
        raise ValueError(f"{name} must be 2-D, got shape {tuple(shape)}")
    r, c = shape
    rs, cs = t.stride()
    if c > 1 and cs != 1:
        raise ValueError(f"{name} must be row-major with unit column stride")
    return r, c, max(rs if r > 1 else c, c)


def gemm(op: int, A: torch.Tensor, B: torch.Tensor, C: torch.Tensor | None = None, *,
         alpha: float = 1.0, beta: float = 0.0, bias: torch.Tensor | None = None,
         epilogue: int = EPI_NONE, preact: torch.Tensor | None = None,
         out_dtype: torch.dtype = torch.float32, colsum: torch.Tensor | None = None,
         colsum_beta: float = 0.0) -> torch.Tensor:
    """General GEMM: C = epi(alpha * op(A) op(B) + beta * C + bias) (see include/logos_vedic.h).

    epilogue=EPI_GELU_BWD multiplies by gelu_tanh'(preact) (preact is then an
    input).  colsum (N float32 values) receives colsum_beta * colsum + the
    column sums of the final C."""
    amp = A.dtype == torch.float32 and B.dtype == torch.float16  # A converted to binary16 in the GEMM
    if (A.dtype != B.dtype or A.dtype not in _DT) and not amp:
        raise ValueError(f"A and B must share dtype float16 or float32, or be float32 A with float16 B "
                         f"(got {A.dtype}, {B.dtype})")
    if amp and op != OP_NN:
        raise ValueError("a float32 A with a float16 B is an NN product")
    ar, ac, lda = _mat(A, "A")
    br, bc, ldb = _mat(B, "B")
    if op == OP_NN:
        M, K, N, Kb = ar, ac, bc, br
    elif op == OP_NT:
        M, K, N, Kb = ar, ac, br, bc
    elif op == OP_TN:
        M, K, N, Kb = ac, ar, bc, br
    else:
        raise ValueError(f"unknown op {op}")
    if Kb != K:
        raise ValueError(f"VedicGEMM: inner dimensions differ (A gives K={K}, B gives K={Kb})")
    if epilogue in (EPI_RESIDUAL, EPI_BIAS_RESIDUAL):
        if C is None or C.dtype != torch.float32:
            raise ValueError("the residual epilogues add to an existing float32 C (the residual stream)")
        if beta != 0.0:
            raise ValueError("the residual epilogues take beta = 0 (C is the residual)")
    if C is None:
        if beta != 0.0:
            raise ValueError("beta != 0 needs an existing C")
        C = torch.empty((M, N), dtype=out_dtype, device=A.device)
    cr, cc, ldc = _mat(C, "C")
    if (cr, cc) != (M, N):
        raise ValueError(f"C must be {M}x{N}, got {cr}x{cc}")
    if C.dtype not in _DT:
        raise ValueError("C must be float32 or float16")
    if bias is not None:
        if bias.dtype != torch.float32 or bias.numel() != N or not bias.is_cuda:
            raise ValueError(f"bias must be {N} float32 values on the GPU")
        bias = bias.contiguous()
    ldp = 0
    if preact is not None:
        pr, pc, ldp = _mat(preact, "preact")
        if (pr, pc) != (M, N) or preact.dtype != torch.float32:
            raise ValueError(f"preact must be float32 {M}x{N}")
    if colsum is not None:
        if colsum.dtype != torch.float32 or colsum.numel() != N or not colsum.is_cuda or not colsum.is_contiguous():
            raise ValueError(f"colsum must be {N} contiguous float32 values on the GPU")
    # (in the order of _lib.GemmDesc's fields)
    d = _lib.GemmDesc(
        op, _lib.DT_F32_F16 if amp else _DT[A.dtype], _DT[C.dtype], M, N, K, A.data_ptr(), lda, B.data_ptr(), ldb,
        C.data_ptr(), ldc, alpha, beta, bias.data_ptr() if bias is not None else None, epilogue,
        preact.data_ptr() if preact is not None else None, ldp, _stream(),
        colsum.data_ptr() if colsum is not None else None, colsum_beta)
    _check(_lib.load().vedic_gemm(ctypes.byref(d)))
    return C


def gemm_bias_residual(X: torch.Tensor, W: torch.Tensor, bias: torch.Tensor | None, residual: torch.Tensor,
                       out_pre: torch.Tensor | None = None) -> torch.Tensor:
    """residual += X . W (+ bias), in place, with the product (and bias)
    rounded before the residual is added: the reference's FFN-down
    amp_gemm_bias into a temporary followed by residual_add_kernel
    (cuda/ModelGPU.cu:1044-1048), and its W_proj projection, saved and then
    added (:1005-1012), with out_pre receiving the product.  X and W float32,
    or float16, or float32 X with a float16 shadow W (AMP)."""
    epi = EPI_BIAS_RESIDUAL if bias is not None else EPI_RESIDUAL
    return gemm(OP_NN, X, W, residual, bias=bias, epilogue=epi, preact=out_pre)


def vedic_gemm(A: torch.Tensor, B: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
    """C = A . B in fp32 (vedic_gemm / cuda_vedic_gemm)."""
    if A.dtype != torch.float32:
        raise ValueError("vedic_gemm takes float32 operands")
    return gemm(OP_NN, A, B, out)


def vedic_gemm_bias(A: torch.Tensor, W: torch.Tensor, bias: torch.Tensor,
                    out: torch.Tensor | None = None) -> torch.Tensor:
    """C = A . W + bias[j] in fp32 (vedic_gemm_bias / cuda_vedic_gemm_bias)."""
    if A.dtype != torch.float32:
        raise ValueError("vedic_gemm_bias takes float32 operands")
    return gemm(OP_NN, A, W, out, bias=bias, epilogue=EPI_BIAS)


def gemm_fp16_fp32out(A: torch.Tensor, B: torch.Tensor, C: torch.Tensor | None = None,
                      alpha: float = 1.0, beta: float = 0.0) -> torch.Tensor:
    """fp32 C = alpha A.B + beta C with fp16 A, B (cuda_gemm_fp16_fp32out)."""
    if A.dtype != torch.float16:
        raise ValueError("gemm_fp16_fp32out takes float16 operands")
    return gemm(OP_NN, A, B, C, alpha=alpha, beta=beta)


def gemm_fp16_fp16out(A: torch.Tensor, B: torch.Tensor, C: torch.Tensor | None = None,
                      alpha: float = 1.0, beta: float = 0.0) -> torch.Tensor:
    """fp16 C = alpha A.B + beta C, fp32 accumulation (cuda_gemm_fp16_fp16out)."""
    if A.dtype != torch.float16:
        raise ValueError("gemm_fp16_fp16out takes float16 operands")
    return gemm(OP_NN, A, B, C, alpha=alpha, beta=beta, out_dtype=torch.float16)


def gemm_bias_gelu(X: torch.Tensor, W: torch.Tensor, bias: torch.Tensor,
                   out: torch.Tensor | None = None, preact: torch.Tensor | None = None) -> torch.Tensor:
    """H = gelu_tanh(X . W + bias), fp32 output; preact receives X . W + bias."""
    return gemm(OP_NN, X, W, out, bias=bias, epilogue=EPI_BIAS_GELU, preact=preact)


def amp_gemm(A: torch.Tensor, W16: torch.Tensor | None, W32: torch.Tensor | None = None,
             out: torch.Tensor | None = None, bias: torch.Tensor | None = None, gelu: bool = False,
             preact: torch.Tensor | None = None) -> torch.Tensor:
    """The reference's amp_gemm / amp_gemm_bias (cuda/ModelGPU.cu:819-859) from a
    float32 activation A: C = binary16(A) . W16 (+ bias, then GELU if asked),
    with A clamped and rounded to binary16 inside the GEMM or, for wide and long
    products (see vedic_amp_gemm in logos_vedic.h), by a pass before it; fp32
    accumulation and output.  W16 None: the fp32 product with W32, the
    reference's fallback for a parameter without a binary16 shadow."""
    if A.dtype != torch.float32:
        raise ValueError("amp_gemm takes a float32 activation")
    W = W16 if W16 is not None else W32
    if W is None:
        raise ValueError("amp_gemm needs W16 or W32")
    if W16 is not None and W16.dtype != torch.float16:
        raise ValueError("W16 must be float16")
    if W16 is None and W32.dtype != torch.float32:
        raise ValueError("W32 must be float32")
    if gelu and bias is None:
        raise ValueError("the fused GELU form takes a bias")
    epi = EPI_BIAS_GELU if gelu else EPI_BIAS if bias is not None else EPI_NONE
    return gemm(OP_NN, A, W, out, bias=bias, epilogue=epi, preact=preact)


def gemm_nt(dY: torch.Tensor, W: torch.Tensor, out: torch.Tensor | None = None,
            beta: float = 0.0) -> torch.Tensor:
    """dX = dY . W^T (+ beta dX); W stored [N x K]."""
    return gemm(OP_NT, dY, W, out, beta=beta)


def gemm_tn(X: torch.Tensor, dY: torch.Tensor, out: torch.Tensor | None = None,
            beta: float = 0.0) -> torch.Tensor:
    """dW = X^T . dY (+ beta dW); X stored [K x M], dY [K x N]."""
    return gemm(OP_TN, X, dY, out, beta=beta)


def gemm_nt_gelu_bwd(dY: torch.Tensor, W: torch.Tensor, H: torch.Tensor, out: torch.Tensor | None = None,
                     db: torch.Tensor | None = None) -> torch.Tensor:
    """dH = (dY . W^T) * gelu_tanh'(H), W stored [N x K], H the cached
    pre-activation [M x N]; db (if given) += column sums of dH (the bias
    gradient).  One fused launch for ffn_da + gelu_bwd + bias_grad."""
    return gemm(OP_NT, dY, W, out, epilogue=EPI_GELU_BWD, preact=H, colsum=db,
                colsum_beta=1.0)


def bias_grad(dY: torch.Tensor, db: torch.Tensor | None = None, beta: float = 0.0) -> torch.Tensor:
    """db = beta * db + column sums of dY (bias_grad_kernel), summed in a fixed order."""
    M, N, ld = _mat(dY, "dY")
    if ld != N or dY.dtype != torch.float32:
        raise ValueError("dY must be a contiguous float32 matrix")
    if db is None:
        if beta != 0.0:
            raise ValueError("beta != 0 needs an existing db")
        db = torch.empty(N, dtype=torch.float32, device=dY.device)
    if db.numel() != N or db.dtype != torch.float32 or not db.is_contiguous():
        raise ValueError(f"db must be {N} contiguous float32 values")
    _check(_lib.load().vedic_bias_grad(dY.data_ptr(), db.data_ptr(), M, N, beta, _stream()))
    return db


def gemm_scatter(X: torch.Tensor, W: torch.Tensor, heads: list[torch.Tensor],
                 bias: torch.Tensor | None = None) -> list[torch.Tensor]:
    """heads[h] = (X . W + bias)[:, h*hc:(h+1)*hc] for equal-width heads (hc a
    multiple of 32): the packed Q/K/V projection written straight into the
    per-head buffers."""
    if X.dtype != W.dtype or X.dtype not in _DT:
        raise ValueError("X and W must share dtype float16 or float32")
    M, K, lda = _mat(X, "X")
    Kb, N, ldb = _mat(W, "W")
    if Kb != K:
        raise ValueError(f"VedicGEMM: inner dimensions differ ({K} vs {Kb})")
    if not heads:
        raise ValueError("no heads")
    hc = heads[0].shape[-1]
    for t in heads:
        if tuple(t.shape) != (M, hc) or t.dtype != torch.float32 or not t.is_contiguous() or not t.is_cuda:
            raise ValueError(f"every head must be a contiguous float32 [{M} x {hc}] GPU matrix")
    if bias is not None and (bias.dtype != torch.float32 or bias.numel() != N):
        raise ValueError(f"bias must be {N} float32 values")
    bias = bias.contiguous() if bias is not None else None
    d = _lib.GemmDesc(
        op=OP_NN, in_dtype=_DT[X.dtype], out_dtype=DT_F32, M=M, N=N, K=K,
        A=X.data_ptr(), lda=lda, B=W.data_ptr(), ldb=ldb, C=None, ldc=N,
        alpha=1.0, beta=0.0, bias=bias.data_ptr() if bias is not None else None,
        epilogue=EPI_BIAS if bias is not None else EPI_NONE, preact=None, ld_preact=0, stream=_stream(),
        colsum=None, colsum_beta=0.0,
    )
    ptrs = (ctypes.c_void_p * len(heads))(*[t.data_ptr() for t in heads])
    _check(_lib.load().vedic_gemm_scatter(ctypes.byref(d), ptrs, len(heads), hc))
    return heads


def cast_pack_fp16(srcs: list[torch.Tensor], out: torch.Tensor | None = None) -> torch.Tensor:
    """binary16 copy of fp32 [rows x cols] matrices packed side by side
    (out[:, i*cols:(i+1)*cols] = srcs[i]), with the reference cast's clamp."""
    if not srcs:
        raise ValueError("no sources")
    rows, cols = srcs[0].shape
    for t in srcs:
        if tuple(t.shape) != (rows, cols) or t.dtype != torch.float32 or not t.is_contiguous() or not t.is_cuda:
            raise ValueError(f"every source must be a contiguous float32 [{rows} x {cols}] GPU matrix")
    if out is None:
        out = torch.empty((rows, len(srcs) * cols), dtype=torch.float16, device=srcs[0].device)
    r, c, ld = _mat(out, "out")
    if r != rows or c != len(srcs) * cols or out.dtype != torch.float16:
        raise ValueError("out must be float16 [rows x nsrc*cols]")
    ptrs = (ctypes.c_void_p * len(srcs))(*[t.data_ptr() for t in srcs])
    _check(_lib.load().vedic_cast_pack_f16(ptrs, len(srcs), rows, cols, out.data_ptr(), ld, _stream()))
    return out


def cast_stack_fp16(srcs: list[torch.Tensor], out: torch.Tensor | None = None) -> torch.Tensor:
    """binary16 copy of fp32 [rows x cols] matrices stacked by rows
    (out[i*rows:(i+1)*rows] = srcs[i]), with the reference cast's clamp: a
    layer's per-head W_O blocks as the B operand of gemm_gather."""
    if not srcs:
        raise ValueError("no sources")
    rows, cols = srcs[0].shape
    for t in srcs:
        if tuple(t.shape) != (rows, cols) or t.dtype != torch.float32 or not t.is_contiguous() or not t.is_cuda:
            raise ValueError(f"every source must be a contiguous float32 [{rows} x {cols}] GPU matrix")
    if out is None:
        out = torch.empty((len(srcs) * rows, cols), dtype=torch.float16, device=srcs[0].device)
    r, c, ld = _mat(out, "out")
    if r != len(srcs) * rows or c != cols or out.dtype != torch.float16:
        raise ValueError("out must be float16 [nsrc*rows x cols]")
    ptrs = (ctypes.c_void_p * len(srcs))(*[t.data_ptr() for t in srcs])
    _check(_lib.load().vedic_cast_stack_f16(ptrs, len(srcs), rows, cols, out.data_ptr(), ld, _stream()))
    return out


def gemm_gather(heads: list[torch.Tensor], W: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
    """C = sum over h, in head order, of heads[h] . W[h*hc:(h+1)*hc] onto a
    zeroed C (each head's product from zero in fp32): the reference's
    per-head amp_gemm(head_out, W_O[h]) + residual_add_kernel loop
    (cuda/ModelGPU.cu:976-986) in one launch, bit for bit.  heads: equal
    [M x hc] float16 or float32 GPU matrices (float32: rounded to binary16 as
    they are read, the AMP path); W: float16 [nheads*hc x N] (cast_stack_fp16);
    out: float32 [M x N]."""
    if not heads:
        raise ValueError("no heads")
    dt = heads[0].dtype
    if dt not in (torch.float16, torch.float32):
        raise ValueError("heads must be float16 or float32")
    M, hc, lda = _mat(heads[0], "heads[0]")
    for t in heads:
        if tuple(t.shape) != (M, hc) or t.dtype != dt or t.stride() != heads[0].stride() or not t.is_cuda:
            raise ValueError(f"every head must be a {dt} [{M} x {hc}] GPU matrix with the same strides")
    K, N, ldb = _mat(W, "W")
    if W.dtype != torch.float16:
        raise ValueError("W must be float16")
    if K != len(heads) * hc:
        raise ValueError(f"VedicGEMM: W has {K} rows, the heads {len(heads)} x {hc} columns")
    if out is None:
        out = torch.empty((M, N), dtype=torch.float32, device=W.device)
    Mo, No, ldc = _mat(out, "out")
    if (Mo, No) != (M, N) or out.dtype != torch.float32:
        raise ValueError(f"out must be float32 [{M} x {N}]")
    d = _lib.GemmDesc(
        op=OP_NN, in_dtype=DT_F16 if dt == torch.float16 else _lib.DT_F32_F16, out_dtype=DT_F32, M=M, N=N, K=K,
        A=None, lda=lda, B=W.data_ptr(), ldb=ldb, C=out.data_ptr(), ldc=ldc,
        alpha=1.0, beta=0.0, bias=None, epilogue=EPI_NONE, preact=None, ld_preact=0, stream=_stream(),
        colsum=None, colsum_beta=0.0,
    )
    ptrs = (ctypes.c_void_p * len(heads))(*[t.data_ptr() for t in heads])
    _check(_lib.load().vedic_gemm_gather(ctypes.byref(d), ptrs, len(heads), hc))
    return out


def add_bias(C: torch.Tensor, bias: torch.Tensor) -> torch.Tensor:
    """C[i][j] += bias[j] in place (add_bias_kernel)."""
    M, N, ld = _mat(C, "C")
    if ld != N or C.dtype != torch.float32:
        raise ValueError("C must be a contiguous float32 matrix")
    if bias.numel() != N or bias.dtype != torch.float32:
        raise ValueError("bias size mismatch")
    _check(_lib.load().vedic_add_bias(C.data_ptr(), bias.contiguous().data_ptr(), M, N, _stream()))
    return C


def _ln_args(X, gamma, beta, dtype):
    if not X.is_cuda or X.dtype != dtype or X.dim() != 2 or not X.is_contiguous():
        raise ValueError(f"X must be a contiguous 2-D {dtype} GPU tensor")
    seq, d = X.shape
    for name, t in (("gamma", gamma), ("beta", beta)):
        if not t.is_cuda or t.dtype != torch.float32 or t.numel() != d or not t.is_contiguous():
            raise ValueError(f"{name} must be {d} contiguous float32 values on the GPU")
    return seq, d


def layernorm(X: torch.Tensor, gamma: torch.Tensor, beta: torch.Tensor, out: torch.Tensor | None = None,
              out16: torch.Tensor | None = None, eps: float = 1e-5, fp32: bool = True,
              fp16: bool = False) -> tuple[torch.Tensor | None, torch.Tensor | None]:
    """Row layer normalisation (cuda_layernorm): returns (Y fp32, Y16 binary16),
    each written when asked for (fp32 / fp16, or out / out16 given); Y16 holds
    the bits cast_fp32_to_fp16(Y) would give, written in the same pass."""
    seq, d = _ln_args(X, gamma, beta, torch.float32)
    if out is None and fp32:
        out = torch.empty_like(X)
    if out16 is None and fp16:
        out16 = torch.empty(X.shape, dtype=torch.float16, device=X.device)
    if out is None and out16 is None:
        raise ValueError("ask for at least one output")
    for t, dt in ((out, torch.float32), (out16, torch.float16)):
        if t is not None and (t.shape != X.shape or t.dtype != dt or not t.is_contiguous()):
            raise ValueError(f"outputs must be contiguous {seq}x{d} tensors")
    _check(_lib.load().vedic_layernorm(X.data_ptr(), gamma.data_ptr(), beta.data_ptr(),
                                       out.data_ptr() if out is not None else None,
                                       out16.data_ptr() if out16 is not None else None, seq, d, eps, _stream()))
    return out, out16


def layernorm_fp16(X16: torch.Tensor, gamma: torch.Tensor, beta: torch.Tensor, out16: torch.Tensor | None = None,
                   eps: float = 1e-5) -> torch.Tensor:
    """cuda_layernorm_fp16: binary16 rows in and out, fp32 statistics."""
    seq, d = _ln_args(X16, gamma, beta, torch.float16)
    if out16 is None:
        out16 = torch.empty_like(X16)
    if out16.shape != X16.shape or out16.dtype != torch.float16 or not out16.is_contiguous():
        raise ValueError(f"out16 must be a contiguous float16 {seq}x{d} tensor")
    _check(_lib.load().vedic_layernorm_f16(X16.data_ptr(), gamma.data_ptr(), beta.data_ptr(), out16.data_ptr(), seq,
                                           d, eps, _stream()))
    return out16


def gelu_(x: torch.Tensor) -> torch.Tensor:
    """In-place tanh-GELU (cuda_gelu)."""
    if not x.is_cuda or x.dtype != torch.float32 or not x.is_contiguous():
        raise ValueError("gelu_ takes a contiguous float32 GPU tensor")
    _check(_lib.load().vedic_gelu(x.data_ptr(), x.numel(), _stream()))
    return x


def cast_fp32_to_fp16(x: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
    """fp16 copy with the reference's +-65504 clamp (cuda_cast_fp32_to_fp16)."""
    if not x.is_cuda or x.dtype != torch.float32 or not x.is_contiguous():
        raise ValueError("cast_fp32_to_fp16 takes a contiguous float32 GPU tensor")
    if out is None:
        out = torch.empty(x.shape, dtype=torch.float16, device=x.device)
    if out.numel() != x.numel() or out.dtype != torch.float16 or not out.is_contiguous():
        raise ValueError("out must be a contiguous float16 tensor of the same size")
    _check(_lib.load().vedic_cast_f32_to_f16(x.data_ptr(), out.data_ptr(), x.numel(), _stream()))
    return out


def cast_fp16_to_fp32(x: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
    """fp32 copy of an fp16 tensor (cuda_cast_fp16_to_fp32)."""
    if not x.is_cuda or x.dtype != torch.float16 or not x.is_contiguous():
        raise ValueError("cast_fp16_to_fp32 takes a contiguous float16 GPU tensor")
    if out is None:
        out = torch.empty(x.shape, dtype=torch.float32, device=x.device)
    _check(_lib.load().vedic_cast_f16_to_f32(x.data_ptr(), out.data_ptr(), x.numel(), _stream()))
    return out


@dataclass
class VerifyResult:
    """Mirror of VedicVerifyResult (cuda/VedicGEMM.cuh:162-167)."""

    checksum_C: float
    checksum_vedic: float
    relative_error: float
    passed: bool


def verify(A: torch.Tensor, B: torch.Tensor, C: torch.Tensor, tolerance: float = 0.01) -> VerifyResult:
    """Gunitasamuchayah check: sum(C) against colsum(A) . rowsum(B)."""
    M, K, lda = _mat(A, "A")
    Kb, N, ldb = _mat(B, "B")
    Mc, Nc, ldc = _mat(C, "C")
    if Kb != K or (Mc, Nc) != (M, N) or lda != K or ldb != N or ldc != N:
        raise ValueError("verify takes contiguous A[MxK], B[KxN], C[MxN]")
    r = _lib.VerifyResult()
    _check(_lib.load().vedic_verify(A.data_ptr(), B.data_ptr(), C.data_ptr(), M, K, N, tolerance,
                                    ctypes.byref(r), _stream()))
    return VerifyResult(r.checksum_C, r.checksum_vedic, r.relative_error, bool(r.pass_))


def gemm_checked(op: int, A: torch.Tensor, B: torch.Tensor, C: torch.Tensor | None = None, *,
                 alpha: float = 1.0, bias: torch.Tensor | None = None,
                 tolerance: float = 0.01) -> tuple[torch.Tensor, VerifyResult]:
    """C = alpha op(A) op(B) (+ bias) with the Gunitasamuchayah check computed on
    the way: sum(C) from the GEMM's own column sums (C is not read again)
    against colsum(op(A)) . rowsum(op(B)).  Synchronous, like verify()."""
    if A.dtype != B.dtype or A.dtype not in _DT:
        raise ValueError("A and B must share dtype float16 or float32")
    ar, ac, lda = _mat(A, "A")
    br, bc, ldb = _mat(B, "B")
    M, K, N, Kb = {OP_NN: (ar, ac, bc, br), OP_NT: (ar, ac, br, bc), OP_TN: (ac, ar, bc, br)}[op]
    if Kb != K:
        raise ValueError(f"VedicGEMM: inner dimensions differ (A gives K={K}, B gives K={Kb})")
    if C is None:
        C = torch.empty((M, N), dtype=torch.float32, device=A.device)
    cr, cc, ldc = _mat(C, "C")
    if (cr, cc) != (M, N) or C.dtype != torch.float32:
        raise ValueError(f"C must be float32 {M}x{N}")
    if bias is not None and (bias.dtype != torch.float32 or bias.numel() != N):
        raise ValueError(f"bias must be {N} float32 values")
    bias = bias.contiguous() if bias is not None else None
    d = _lib.GemmDesc(
        op=op, in_dtype=_DT[A.dtype], out_dtype=DT_F32, M=M, N=N, K=K,
        A=A.data_ptr(), lda=lda, B=B.data_ptr(), ldb=ldb, C=C.data_ptr(), ldc=ldc,
        alpha=alpha, beta=0.0, bias=bias.data_ptr() if bias is not None else None,
        epilogue=EPI_BIAS if bias is not None else EPI_NONE, preact=None, ld_preact=0, stream=_stream(),
        colsum=None, colsum_beta=0.0,
    )
    r = _lib.VerifyResult()
    _check(_lib.load().vedic_gemm_checked(ctypes.byref(d), tolerance, ctypes.byref(r)))
    return C, VerifyResult(r.checksum_C, r.checksum_vedic, r.relative_error, bool(r.pass_))


def uses_vendor_blas() -> bool:
    """Always False (cuda_vedic_gemm_uses_cublas's counterpart)."""
    return bool(_lib.load().vedic_uses_vendor_blas())


def backend_name() -> str:
    return _lib.load().vedic_backend_name().decode()


def _head(t: torch.Tensor, name: str, seq: int | None = None, dh: int | None = None) -> tuple[int, int]:
    if not isinstance(t, torch.Tensor) or not t.is_cuda or t.dtype != torch.float32 or t.dim() != 2 \
            or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous float32 [seq x dh] GPU matrix")
    s, d = t.shape
    if (seq is not None and s != seq) or (dh is not None and d != dh):
        raise ValueError(f"{name} has shape {tuple(t.shape)}, expected [{seq} x {dh}]")
    return s, d


def flash_attention_fwd(Q: torch.Tensor, K: torch.Tensor, V: torch.Tensor, out: torch.Tensor | None = None,
                        scale: float | None = None, causal: bool = True, shunyam: bool = False, window: int = 0,
                        stride: int = 1, attn: torch.Tensor | None = None,
                        lse: torch.Tensor | None = None) -> torch.Tensor:
    """out = softmax(scale Q K^T + mask) V for one head, fp32 [seq x dh] (dh 1
    to 128): cuda_flash_attention_fwd (cuda/VedicGEMM.cu:1065-1104).  scale
    defaults to 1/sqrt(dh), the caller's value (cuda/ModelGPU.cu:963).  The
    mask drops keys after the query (causal) and, with shunyam and seq >
    window, keys outside [query - window, query] that are not multiples of
    stride.  attn (optional contiguous float32 [seq x seq] GPU tensor)
    receives the reference's probability copy, with the reference's values:
    allowed entries expf(s - m_t) / l (m_t the running maximum after the
    16-key tile holding the key: the reference's FA_TILE,
    cuda/VedicGEMM.cu:898), masked entries their previous content / l.
    lse (optional float32 [seq] GPU tensor, not together with attn) receives
    each row's log-sum-exp ln(sum over allowed keys of e^(scale q.k)), for
    flash_attention_bwd."""
    seq, dh = _head(Q, "Q")
    _head(K, "K", seq, dh)
    _head(V, "V", seq, dh)
    if out is None:
        out = torch.empty_like(Q)
    _head(out, "out", seq, dh)
    if scale is None:
        scale = 1.0 / float(dh) ** 0.5
    flags = (float(scale), int(causal), int(shunyam), int(window), int(stride), _stream())
    if lse is not None:
        if attn is not None:
            raise ValueError("attn and lse are separate calls")
        _vec(lse, "lse", seq)
        _check(_lib.load().vedic_flash_attention_fwd_lse(Q.data_ptr(), K.data_ptr(), V.data_ptr(), out.data_ptr(),
                                                         lse.data_ptr(), seq, dh, *flags))
        return out
    if attn is not None:
        if not isinstance(attn, torch.Tensor) or not attn.is_cuda or attn.dtype != torch.float32 \
                or tuple(attn.shape) != (seq, seq) or not attn.is_contiguous():
            raise ValueError(f"attn must be a contiguous float32 [{seq} x {seq}] GPU matrix")
    ap = None if attn is None else attn.data_ptr()
    _check(_lib.load().vedic_flash_attention_fwd(Q.data_ptr(), K.data_ptr(), V.data_ptr(), out.data_ptr(), ap, seq,
                                                 dh, *flags))
    return out


def _vec(t: torch.Tensor, name: str, n: int) -> None:
    if not isinstance(t, torch.Tensor) or not t.is_cuda or t.dtype != torch.float32 or t.numel() != n \
            or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous float32 GPU tensor of {n} values")


def flash_attention_fwd_heads(Qs: list[torch.Tensor], Ks: list[torch.Tensor], Vs: list[torch.Tensor],
                              outs: list[torch.Tensor] | None = None, scale: float | None = None,
                              causal: bool = True, shunyam: bool = False, window: int = 0,
                              stride: int = 1, lses: list[torch.Tensor] | None = None) -> list[torch.Tensor]:
    """flash_attention_fwd for several heads (all [seq x dh]) in one launch;
    lses: optional per-head log-sum-exp outputs."""
    n = len(Qs)
    if n == 0 or len(Ks) != n or len(Vs) != n:
        raise ValueError("Qs, Ks and Vs must be non-empty lists of the same length")
    seq, dh = _head(Qs[0], "Q[0]")
    for i in range(n):
        _head(Qs[i], f"Q[{i}]", seq, dh)
        _head(Ks[i], f"K[{i}]", seq, dh)
        _head(Vs[i], f"V[{i}]", seq, dh)
    if outs is None:
        outs = [torch.empty_like(q) for q in Qs]
    if len(outs) != n:
        raise ValueError("outs must have one tensor per head")
    for i in range(n):
        _head(outs[i], f"out[{i}]", seq, dh)
    if scale is None:
        scale = 1.0 / float(dh) ** 0.5
    if lses is not None:
        if len(lses) != n:
            raise ValueError("lses must have one tensor per head")
        for i in range(n):
            _vec(lses[i], f"lse[{i}]", seq)
    arr = lambda ts: (ctypes.c_void_p * n)(*[t.data_ptr() for t in ts])
    _check(_lib.load().vedic_flash_attention_fwd_heads(arr(Qs), arr(Ks), arr(Vs), arr(outs),
                                                       None if lses is None else arr(lses), n, seq, dh,
                                                       float(scale), int(causal), int(shunyam), int(window),
                                                       int(stride), _stream()))
    return outs


def flash_attention_bwd(Q, K, V, O, dO, lse, dQ=None, dK=None, dV=None, scale: float | None = None,
                        causal: bool = True, shunyam: bool = False, window: int = 0, stride: int = 1):
    """(dQ, dK, dV) of flash_attention_fwd for one head from Q, K, V, its
    output O, the output gradient dO and the forward's lse; same mask
    arguments as the forward.  Replaces the backward of cuda/train_gpu.cu:672-740."""
    return tuple(t[0] for t in flash_attention_bwd_heads([Q], [K], [V], [O], [dO], [lse],
                                                          None if dQ is None else [dQ], None if dK is None else [dK],
                                                          None if dV is None else [dV], scale, causal, shunyam,
                                                          window, stride))


def flash_attention_bwd_heads(Qs, Ks, Vs, Os, dOs, lses, dQs=None, dKs=None, dVs=None, scale: float | None = None,
                              causal: bool = True, shunyam: bool = False, window: int = 0, stride: int = 1):
    """flash_attention_bwd for 1..32 heads in one launch; returns (dQs, dKs, dVs)."""
    n = len(Qs)
    if n == 0 or any(len(x) != n for x in (Ks, Vs, Os, dOs, lses)):
        raise ValueError("Qs, Ks, Vs, Os, dOs and lses must be non-empty lists of the same length")
    seq, dh = _head(Qs[0], "Q[0]")
    for i in range(n):
        for t, name in ((Qs[i], "Q"), (Ks[i], "K"), (Vs[i], "V"), (Os[i], "O"), (dOs[i], "dO")):
            _head(t, f"{name}[{i}]", seq, dh)
        _vec(lses[i], f"lse[{i}]", seq)
    out = []
    for given in (dQs, dKs, dVs):
        ts = [torch.empty_like(q) for q in Qs] if given is None else given
        if len(ts) != n:
            raise ValueError("gradient lists must have one tensor per head")
        for i in range(n):
            _head(ts[i], f"gradient[{i}]", seq, dh)
        out.append(ts)
    if scale is None:
        scale = 1.0 / float(dh) ** 0.5
    arr = lambda ts: (ctypes.c_void_p * n)(*[t.data_ptr() for t in ts])
    _check(_lib.load().vedic_flash_attention_bwd_heads(arr(Qs), arr(Ks), arr(Vs), arr(Os), arr(dOs), arr(lses),
                                                       arr(out[0]), arr(out[1]), arr(out[2]), n, seq, dh,
                                                       float(scale), int(causal), int(shunyam), int(window),
                                                       int(stride), _stream()))
    return tuple(out)


# ---------------------------------------------------------------- rows that choose their weights


def _on_current(t: torch.Tensor, name: str, dtype, dev: int) -> int:
    """t's address, checked to be on the current device (whose stream the call runs on) and of `dtype`."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if not t.is_cuda or t.get_device() != dev:
        raise ValueError(f"{name} must be on the current GPU (cuda:{dev})")
    if t.dtype != dtype:
        raise ValueError(f"{name} must be {dtype}, got {t.dtype}")
    return t.data_ptr()


_current_device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device


def _device(t: torch.Tensor) -> int:
    """The current device, for operands like t (which has to be on a GPU)."""
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise ValueError("the operands must be on the current GPU")
    return _current_device()


def _ints(t: torch.Tensor, name: str, shape: tuple, dev: int) -> int:
    p = _on_current(t, name, torch.int32, dev)
    if tuple(t.shape) != shape or not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous int32 of shape {shape}, got {tuple(t.shape)}")
    return p


def _floats(t: torch.Tensor, name: str, shape: tuple, dev: int) -> int:
    p = _on_current(t, name, torch.float32, dev)
    if tuple(t.shape) != shape or not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous float32 of shape {shape}, got {tuple(t.shape)}")
    return p


def _rows2d(t: torch.Tensor, name: str, dtype, dev: int) -> tuple[int, int, int, int]:
    """(address, rows, cols, leading dimension) of a row-major matrix of `dtype` on the current device."""
    p = _on_current(t, name, dtype, dev)
    if t.dim() != 2:
        raise ValueError(f"{name} must be 2-D, got shape {tuple(t.shape)}")
    r, c = t.shape
    rs, cs = t.stride()
    if r > 0 and c > 1 and cs != 1:
        raise ValueError(f"{name} must be row-major with unit column stride")
    if r > 1 and rs < c:
        raise ValueError(f"{name}'s rows overlap (row stride {rs}, {c} columns)")
    return p, r, c, rs if r > 1 else c


class Routing(NamedTuple):
    """What route_topk returns (int32 but for the float32 weights)."""

    ids: torch.Tensor      # [T, k] experts in descending order of the logits; -1: none
    weights: torch.Tensor  # [T, k]
    offsets: torch.Tensor  # [E + 1] first sorted place of each expert
    rows: torch.Tensor     # [T * k] token of each place
    slots: torch.Tensor    # [T, k] place of each pair


def route_topk(logits: torch.Tensor, k: int, renorm: bool = True) -> Routing:
    """A router's choice: the k largest of each token's float32 logits [T, E] (a tie to the lower expert, -infinity
    never), their softmax weights -- among the chosen (renorm) or within all E -- and the plan that gemm_grouped and
    combine_rows read: the pairs sorted by expert.  See vedic_route_topk in logos_vedic.h."""
    dev = _device(logits)
    p, T, E, ld = _rows2d(logits, "logits", torch.float32, dev)
    if not 0 < k <= E:
        raise ValueError(f"k must be 1 .. {E}, got {k}")
    # (new_empty and empty_like take a third less time than empty with a device)
    weights = logits.new_empty((T, k))
    ids = logits.new_empty((T, k), dtype=torch.int32)
    slots = torch.empty_like(ids)
    offsets, rows = ids.new_empty(E + 1), ids.new_empty(T * k)
    _check(_lib.load().vedic_route_topk(p, ld, T, E, k, renorm, ids.data_ptr(), weights.data_ptr(), offsets.data_ptr(),
                                        rows.data_ptr(), slots.data_ptr(), _stream()))
    return Routing(ids, weights, offsets, rows, slots)


def route_topk_bwd(logits: torch.Tensor, ids: torch.Tensor, weights: torch.Tensor, dweights: torch.Tensor,
                   renorm: bool = True, out: torch.Tensor | None = None) -> torch.Tensor:
    """The gradient of route_topk's weights with respect to the logits, float32 [T, E]; renorm as in the forward."""
    dev = _device(logits)
    p, T, E, ld = _rows2d(logits, "logits", torch.float32, dev)
    if ids.dim() != 2 or ids.shape[0] != T or not 0 < ids.shape[1] <= E:
        raise ValueError(f"ids must be [{T}, k] with k <= {E}, got {tuple(ids.shape)}")
    shape = tuple(ids.shape)
    pi, pw, pg = _ints(ids, "ids", shape, dev), _floats(weights, "weights", shape, dev), \
        _floats(dweights, "dweights", shape, dev)
    if out is None:
        out = logits.new_empty((T, E))
        po, ldo = out.data_ptr(), E
    else:
        po, To, Eo, ldo = _rows2d(out, "out", torch.float32, dev)
        if (To, Eo) != (T, E):
            raise ValueError(f"out must be {T}x{E}")
    _check(_lib.load().vedic_route_topk_bwd(p, ld, pi, pw, pg, T, E, shape[1], renorm, po, ldo, _stream()))
    return out


def group_rows(ids: torch.Tensor, groups: int, per_row: int = 1) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """(offsets, rows, slots) of the plan that sorts the int32 `ids` by group, stable: rows[place] = entry // per_row.
    An id outside 0 .. groups - 1 belongs to no group (slot -1); its row comes
    behind offsets[groups]."""
    dev = _device(ids)
    p = _ints(ids, "ids", tuple(ids.shape), dev)
    n, d = ids.numel(), ids.device
    offsets = torch.empty(max(groups, 0) + 1, dtype=torch.int32, device=d)
    rows = torch.empty(n, dtype=torch.int32, device=d)
    slots = torch.empty(ids.shape, dtype=torch.int32, device=d)
    _check(_lib.load().vedic_group_rows(p, n, per_row, groups, offsets.data_ptr(), rows.data_ptr(), slots.data_ptr(),
                                        _stream()))
    return offsets, rows, slots


def _offsets(t: torch.Tensor, groups: int, dev: int) -> int:
    return _ints(t, "offsets", (groups + 1,), dev)


def gemm_grouped(op: int, A: torch.Tensor, B: torch.Tensor, offsets: torch.Tensor, C: torch.Tensor | None = None, *,
                 rows: torch.Tensor | None = None, bias: torch.Tensor | None = None, epilogue: int = EPI_NONE,
                 preact: torch.Tensor | None = None, beta: float = 0.0, db: torch.Tensor | None = None,
                 db_beta: float = 0.0, out_dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """Products grouped by expert (vedic_gemm_grouped in logos_vedic.h): rows offsets[g] .. offsets[g + 1] - 1 take
    group g's weight.

      OP_NN  C[i] = epi(A[i] . B[g])       B [G, K, N]; epilogue NONE, BIAS or BIAS_GELU (bias [G, N], preact an output)
      OP_NT  C[i] = epi(A[i] . B[g]^T)     B [G, N, K]; epilogue NONE or GELU_BWD (preact an input)
      OP_TN  C[g] = beta C[g] + A_g^T . B_g  A [R, M], B [R, N], C [G, M, N]; db [G, N] = db_beta db + column sums of B

    rows (int32 [R]): A[i] is row rows[i] of A.  A and B float16 or float32; C and preact float32, or float16
    (out_dtype) with float16 operands and OP_NN / OP_NT.  Rows of C behind offsets[G] are left as they are."""
    dev = _device(A)
    dt = A.dtype
    if dt not in _DT:
        raise ValueError(f"A must be float16 or float32, got {dt}")
    if op not in (OP_NN, OP_NT, OP_TN):
        raise ValueError(f"unknown op {op}")
    if epilogue not in ((EPI_NONE, EPI_BIAS, EPI_BIAS_GELU), (EPI_NONE, EPI_GELU_BWD), (EPI_NONE,))[op]:
        raise ValueError("VedicGEMM: epilogue not offered with this op (NN: NONE, BIAS, BIAS_GELU; NT: NONE, GELU_BWD; "
                         "TN: NONE)")
    pa, a_rows, a_cols, lda = _rows2d(A, "A", dt, dev)
    G = offsets.numel() - 1
    if G < 1:
        raise ValueError("offsets must hold groups + 1 values")
    poff = _offsets(offsets, G, dev)
    R = a_rows
    pr = None
    if rows is not None:
        R = rows.numel()
        pr = _ints(rows, "rows", (R,), dev)
    d = A.device
    stride_b = stride_c = 0
    M = K = 0
    if op == OP_TN:
        pb, b_rows, N, ldb = _rows2d(B, "B", dt, dev)
        M = a_cols
        if b_rows != R:
            raise ValueError(f"VedicGEMM: A gives {R} rows, B {b_rows}")
        if C is None:
            if beta != 0.0:
                raise ValueError("beta != 0 needs an existing C")
            C = torch.empty((G, M, N), dtype=torch.float32, device=d)
        pc = _on_current(C, "C", torch.float32, dev)
        if tuple(C.shape) != (G, M, N) or (N > 1 and C.stride(2) != 1) or (M > 1 and C.stride(1) < N):
            raise ValueError(f"C must be float32 [{G}, {M}, {N}] with row-major matrices")
        ldc, stride_c = (C.stride(1) if M > 1 else N), C.stride(0)
    else:
        pb = _on_current(B, "B", dt, dev)
        if B.dim() != 3 or B.shape[0] != G:
            raise ValueError(f"B must be [{G}, {'K, N' if op == OP_NN else 'N, K'}], got {tuple(B.shape)}")
        br, bc = B.shape[1], B.shape[2]
        K, N = (br, bc) if op == OP_NN else (bc, br)
        if (bc > 1 and B.stride(2) != 1) or (br > 1 and B.stride(1) < bc):
            raise ValueError("B must hold row-major matrices")
        ldb, stride_b = (B.stride(1) if br > 1 else bc), B.stride(0)
        if K != a_cols:
            raise ValueError(f"VedicGEMM: inner dimensions differ (A gives K={a_cols}, B gives K={K})")
        if beta != 0.0 or db is not None:
            raise ValueError("beta and db belong to OP_TN")
        if C is None:
            C = torch.empty((R, N), dtype=out_dtype, device=d)
        if C.dtype not in _DT or (C.dtype == torch.float16 and dt != torch.float16):
            raise ValueError("C must be float32, or float16 with float16 operands")
        pc, cr, cc, ldc = _rows2d(C, "C", C.dtype, dev)
        if (cr, cc) != (R, N):
            raise ValueError(f"C must be {R}x{N}, got {cr}x{cc}")
    pbias = pp = pdb = None
    if epilogue in (EPI_BIAS, EPI_BIAS_GELU):
        if bias is None:
            raise ValueError("this epilogue takes a bias")
        pbias = _floats(bias, "bias", (G, N), dev)
    elif bias is not None:
        raise ValueError("a bias goes with EPI_BIAS or EPI_BIAS_GELU")
    ldp = 0
    if preact is not None:
        pp, prow, pcol, ldp = _rows2d(preact, "preact", C.dtype, dev)
        if (prow, pcol) != (R, N):
            raise ValueError(f"preact must be {R}x{N}")
    if db is not None:
        pdb = _floats(db, "db", (G, N), dev)
    desc = _lib.GroupedDesc(op, _DT[dt], _DT[C.dtype], epilogue, G, R, M, N, K, poff, pr, a_rows, pa, lda, pb, ldb, stride_b,
                            pc, ldc, stride_c, pbias, pp, ldp, beta, pdb, db_beta, _stream())
    _check(_lib.load().vedic_gemm_grouped(ctypes.byref(desc)))
    return C


def bias_grad_grouped(dY: torch.Tensor, offsets: torch.Tensor, db: torch.Tensor | None = None,
                      beta: float = 0.0) -> torch.Tensor:
    """db[g] = beta db[g] + the column sums of group g's rows of dY (float16 or float32 [R, N]), in a fixed order."""
    dev = _device(dY)
    if dY.dtype not in _DT:
        raise ValueError(f"dY must be float16 or float32, got {dY.dtype}")
    p, R, N, ld = _rows2d(dY, "dY", dY.dtype, dev)
    G = offsets.numel() - 1
    po = _offsets(offsets, G, dev)
    if db is None:
        if beta != 0.0:
            raise ValueError("beta != 0 needs an existing db")
        db = torch.empty((G, N), dtype=torch.float32, device=dY.device)
    pd = _floats(db, "db", (G, N), dev)
    _check(_lib.load().vedic_bias_grad_grouped(p, _DT[dY.dtype], ld, R, N, po, G, beta, pd, _stream()))
    return db


def combine_rows(Y: torch.Tensor, slots: torch.Tensor, weights: torch.Tensor | None = None,
                 residual: torch.Tensor | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """out[t] = residual[t] + sum over j of weights[t, j] Y[slots[t, j]], float32 [T, D]: the experts' rows back in token
    order (weights None: ones, the backward of reading rows through a list; residual may be out)."""
    dev = _device(Y)
    if Y.dtype not in _DT:
        raise ValueError(f"Y must be float16 or float32, got {Y.dtype}")
    p, R, D, ldy = _rows2d(Y, "Y", Y.dtype, dev)
    if slots.dim() != 2:
        raise ValueError("slots must be [T, k]")
    T, k = slots.shape
    ps = _ints(slots, "slots", (T, k), dev)
    pw = None if weights is None else _floats(weights, "weights", (T, k), dev)
    pres, ldr = None, 0
    if residual is not None:
        pres, rr, rc, ldr = _rows2d(residual, "residual", torch.float32, dev)
        if (rr, rc) != (T, D):
            raise ValueError(f"residual must be {T}x{D}")
    if out is None:
        out = slots.new_empty((T, D), dtype=torch.float32)
        po, ldo = out.data_ptr(), D
    else:
        po, To, Do, ldo = _rows2d(out, "out", torch.float32, dev)
        if (To, Do) != (T, D):
            raise ValueError(f"out must be {T}x{D}")
    _check(_lib.load().vedic_combine_rows(p, _DT[Y.dtype], ldy, R, ps, pw, pres, ldr, po, ldo, T, k, D, _stream()))
    return out


def combine_rows_bwd(dout: torch.Tensor, Y: torch.Tensor, slots: torch.Tensor, weights: torch.Tensor,
                     dY: torch.Tensor | None = None, out_dtype: torch.dtype = torch.float32
                     ) -> tuple[torch.Tensor, torch.Tensor]:
    """(dY, dweights) of combine_rows: dY[slots[t, j]] = weights[t, j] dout[t] in out_dtype (float32 or float16),
    dweights[t, j] = <dout[t], Y[slots[t, j]]>.  Every slot at most once; rows that no slot names are left as they are
    (undefined in a dY allocated here)."""
    dev = _device(Y)
    if Y.dtype not in _DT:
        raise ValueError(f"Y must be float16 or float32, got {Y.dtype}")
    p, R, D, ldy = _rows2d(Y, "Y", Y.dtype, dev)
    if slots.dim() != 2:
        raise ValueError("slots must be [T, k]")
    T, k = slots.shape
    ps = _ints(slots, "slots", (T, k), dev)
    pw = _floats(weights, "weights", (T, k), dev)
    pg, gr, gc, ldg = _rows2d(dout, "dout", torch.float32, dev)
    if (gr, gc) != (T, D):
        raise ValueError(f"dout must be {T}x{D}")
    if dY is None:
        dY = Y.new_empty((R, D), dtype=out_dtype)
    if dY.dtype not in _DT:
        raise ValueError("dY must be float16 or float32")
    po, orr, oc, ldo = _rows2d(dY, "dY", dY.dtype, dev)
    if (orr, oc) != (R, D):
        raise ValueError(f"dY must be {R}x{D}")
    dw = torch.empty_like(weights)
    _check(_lib.load().vedic_combine_rows_bwd(pg, ldg, p, _DT[Y.dtype], ldy, R, ps, pw, po, _DT[dY.dtype], ldo,
                                              dw.data_ptr(), T, k, D, _stream()))
    return dY, dw


def lora_add(C: torch.Tensor, X: torch.Tensor, A: torch.Tensor, B: torch.Tensor, offsets: torch.Tensor,
             rows: torch.Tensor, scales: torch.Tensor | None = None) -> torch.Tensor:
    """C[i] += scales[g] (X[i] . A[g]) . B[g], in place, for the rows i = rows[offsets[g] .. offsets[g + 1] - 1] of each
    adapter g (a plan of group_rows).  X [M, K], A [G, K, r], B [G, r, N] all float16 or all float32, C float32 [M, N];
    r <= 128.  A row is listed at most once; others keep their content."""
    dev = _device(X)
    px, M, K, ldx, pa, pb, N, G, r, n, po, pr, psc = _lora_args(X, A, B, offsets, rows, scales, dev)
    pc, Mc, Nc, ldc = _rows2d(C, "C", torch.float32, dev)
    if (Mc, Nc) != (M, N):
        raise ValueError(f"C must be {M}x{N}, got {Mc}x{Nc}")
    _check(_lib.load().vedic_lora_add(px, _DT[X.dtype], ldx, M, pa, pb, G, r, po, pr, n, psc, pc, ldc, K, N, _stream()))
    return C


def _lora_args(X, A, B, offsets, rows, scales, dev):
    dt = X.dtype
    if dt not in _DT:
        raise ValueError(f"X must be float16 or float32, got {dt}")
    px, M, K, ldx = _rows2d(X, "X", dt, dev)
    pa, pb = _on_current(A, "A", dt, dev), _on_current(B, "B", dt, dev)
    if A.dim() != 3 or not A.is_contiguous() or A.shape[1] != K:
        raise ValueError(f"A must be contiguous [G, {K}, r], got {tuple(A.shape)}")
    G, _, r = A.shape
    if B.dim() != 3 or B.shape[0] != G or B.shape[1] != r or not B.is_contiguous():
        raise ValueError(f"B must be contiguous [{G}, {r}, N], got {tuple(B.shape)}")
    n = rows.numel()
    psc = None if scales is None else _floats(scales, "scales", (G,), dev)
    return px, M, K, ldx, pa, pb, B.shape[2], G, r, n, _offsets(offsets, G, dev), _ints(rows, "rows", (n,), dev), psc


def gemm_lora(X: torch.Tensor, W: torch.Tensor, A: torch.Tensor, B: torch.Tensor, offsets: torch.Tensor,
              rows: torch.Tensor, bias: torch.Tensor | None = None, scales: torch.Tensor | None = None,
              out: torch.Tensor | None = None) -> torch.Tensor:
    """Y = X . W (+ bias), float32, with every listed row's adapter added (lora_add): one shared projection for the
    requests of a batch, each with low-rank weights of its own."""
    dev = _device(X)
    px, M, K, ldx, pa, pb, N, G, r, n, po, pr, psc = _lora_args(X, A, B, offsets, rows, scales, dev)
    pw, Kw, Nw, ldw = _rows2d(W, "W", X.dtype, dev)
    if (Kw, Nw) != (K, N):
        raise ValueError(f"VedicGEMM: W must be {K}x{N}, got {Kw}x{Nw}")
    if out is None:
        out = X.new_empty((M, N), dtype=torch.float32)
    pc, Mc, Nc, ldc = _rows2d(out, "out", torch.float32, dev)
    if (Mc, Nc) != (M, N):
        raise ValueError(f"out must be {M}x{N}")
    pbias = None if bias is None else _floats(bias, "bias", (N,), dev)
    dt = _DT[X.dtype]
    d = _lib.GemmDesc(OP_NN, dt, DT_F32, M, N, K, px, ldx, pw, ldw, pc, ldc, 1.0, 0.0, pbias,
                      EPI_NONE if bias is None else EPI_BIAS, None, 0, _stream(), None, 0.0)
    _check(_lib.load().vedic_gemm_lora(ctypes.byref(d), pa, pb, G, r, po, pr, n, psc))
    return out


# ---------------------------------------------------------------- a paged cache, weights in four bits


def kv_cache(pages: int, page_size: int, heads: int, dh: int, four_bit: bool = False,
             device=None) -> tuple[torch.Tensor, torch.Tensor]:
    """Zeroed (k, v) of a cache, [pages, heads, page_size, row]: rows of dh float16 values, or of 5 dh / 8 bytes (uint8)
    with four_bit (vedic_kv_format_t in logos_vedic.h).  Any tensors of that shape and element type will do whose last
    dimension is contiguous, and whose other strides are whole rows apart."""
    if dh <= 0 or dh % (32 if four_bit else 8) != 0 or dh > 256:
        raise ValueError(f"dh must be a multiple of {32 if four_bit else 8} up to 256, got {dh}")
    shape = (pages, heads, page_size, dh * 5 // 8 if four_bit else dh)
    dt = torch.uint8 if four_bit else torch.float16
    device = torch.device("cuda") if device is None else device
    return torch.zeros(shape, dtype=dt, device=device), torch.zeros(shape, dtype=dt, device=device)


def _kv(k, v, table, lens, q_start, tokens, dev) -> _lib.Kv:
    """The cache and the sequences of a call, checked."""
    dt = k.dtype
    if dt not in (torch.float16, torch.uint8):
        raise ValueError(f"a cache is float16 or uint8 (four bits), got {dt}")
    pk, pv = _on_current(k, "the cache's k", dt, dev), _on_current(v, "the cache's v", dt, dev)
    shape, strides = k.shape, k.stride()
    if len(shape) != 4 or v.shape != shape or v.stride() != strides:
        raise ValueError(f"a cache's k and v are [pages, heads, page_size, row] with equal strides, got {tuple(shape)} and "
                         f"{tuple(v.shape)}")
    pages, heads, ps, row = shape
    sp, sh, st, one = strides
    if one != 1 and row > 1:
        raise ValueError("a cache's rows must be contiguous")
    i4 = dt is torch.uint8
    if i4 and row % 5 != 0:
        raise ValueError(f"a four-bit row has 5 dh / 8 bytes, got {row}")
    pt, pl, pq = _on_current(table, "table", torch.int32, dev), _on_current(lens, "lens", torch.int32, dev), None
    if table.dim() != 2:
        raise ValueError("table must be [sequences, pages]")
    B, W = table.shape
    tb, tw = table.stride()
    if tw != 1 and W > 1:
        raise ValueError("table's rows must be contiguous")
    if lens.dim() != 1 or lens.shape[0] != B or not lens.is_contiguous():
        raise ValueError(f"lens must be contiguous int32 of shape ({B},), got {tuple(lens.shape)}")
    if q_start is not None:
        pq = _ints(q_start, "q_start", (B + 1,), dev)
    elif tokens != B:
        raise ValueError(f"{tokens} rows for {B} sequences: q_start tells which are whose")
    # (a dimension of one has any stride)
    return _lib.Kv(i4, pages, ps, heads, row * 8 // 5 if i4 else row, pk, pv, sp if pages > 1 else max(sp, row),
                   sh if heads > 1 else max(sh, row), st if ps > 1 else max(st, row), pt, tb if B > 1 else W, W, pl, pq, B, tokens)


def _heads3d(t: torch.Tensor, name: str, dtype, dev: int) -> tuple[int, int, int, int, int, int]:
    """(address, tokens, heads, dh, token stride, head stride) of [tokens, heads, dh] with contiguous rows."""
    p = _on_current(t, name, dtype, dev)
    if t.dim() != 3:
        raise ValueError(f"{name} must be [tokens, heads, dh], got shape {tuple(t.shape)}")
    n, h, d = t.shape
    st, sh, one = t.stride()
    if d > 1 and one != 1:
        raise ValueError(f"{name}'s rows must be contiguous")
    return p, n, h, d, st, sh


def kv_append(q: torch.Tensor | None, k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
              table: torch.Tensor, lens: torch.Tensor, q_start: torch.Tensor | None = None,
              rope: torch.Tensor | None = None, interleaved: bool = False,
              out: torch.Tensor | None = None) -> torch.Tensor | None:
    """New tokens' keys and values into the cache; returns q turned by the tokens' positions, float16 (None without q).

    q [tokens, q_heads, dh], k and v [tokens, heads, dh], all float32 or all float16 (views of one packed projection do).
    table int32 [sequences, pages]; lens int32 [sequences]: tokens of each, these included; q_start int32
    [sequences + 1]: rows q_start[b] .. q_start[b + 1] - 1 are sequence b's (None: one row each).  rope float32
    [positions, dims]: dims / 2 cosines, then the sines, of each position's angles; pairs (i, i + dims / 2), or
    (2i, 2i + 1) with interleaved; the values behind dims are not turned.  See vedic_kv_append in logos_vedic.h."""
    dev = _device(k)
    dt = k.dtype
    if dt not in _DT:
        raise ValueError(f"k must be float16 or float32, got {dt}")
    pk, T, H, D, kt, kh = _heads3d(k, "k", dt, dev)
    pv, Tv, Hv, Dv, vt, vh = _heads3d(v, "v", dt, dev)
    kv = _kv(k_cache, v_cache, table, lens, q_start, T, dev)
    if (Tv, Hv, Dv) != (T, H, D) or (H, D) != (kv.heads, kv.dh):
        raise ValueError(f"k and v must be [tokens, {kv.heads}, {kv.dh}], got {tuple(k.shape)} and {tuple(v.shape)}")
    pq = po = None
    Hq = qt = qh = ot = oh = 0
    if q is not None:
        pq, Tq, Hq, Dq, qt, qh = _heads3d(q, "q", dt, dev)
        if (Tq, Dq) != (T, D):
            raise ValueError(f"q must be [{T}, q_heads, {D}], got {tuple(q.shape)}")
        if out is None:
            out = q.new_empty((T, Hq, D), dtype=torch.float16)
            po, ot, oh = out.data_ptr(), Hq * D, D
        else:
            po, To, Ho, Do, ot, oh = _heads3d(out, "out", torch.float16, dev)
            if (To, Ho, Do) != (T, Hq, D):
                raise ValueError(f"out must be {T}x{Hq}x{D}")
    pr, rows, dims = None, 0, 0
    if rope is not None:
        pr = _on_current(rope, "rope", torch.float32, dev)
        if rope.dim() != 2 or not rope.is_contiguous() or rope.shape[1] > D or rope.shape[1] % 2 != 0:
            raise ValueError(f"rope must be contiguous float32 [positions, dims], dims even and at most {D}")
        rows, dims = rope.shape
    _check(_lib.load().vedic_kv_append(ctypes.byref(kv), _DT[dt], pq, qt, qh, Hq, po, ot, oh, pk, kt, kh, pv, vt, vh, pr, rows,
                                       dims, interleaved, _stream()))
    return out if q is not None else None


def kv_read(k_cache: torch.Tensor, v_cache: torch.Tensor, table: torch.Tensor, lens: torch.Tensor,
            q_start: torch.Tensor | None = None, tokens: int | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """The rows that kv_append's arguments name, from the cache: (k, v) float16 [tokens, heads, dh].  q_start the running
    sums of lens gives whole sequences (tokens: q_start's last value, which is on the GPU).  Rows of no sequence are undefined."""
    dev = _device(k_cache)
    if tokens is None:
        if q_start is not None:
            raise ValueError("tokens (the last value of q_start) is needed with q_start")
        tokens = table.shape[0]
    kv = _kv(k_cache, v_cache, table, lens, q_start, tokens, dev)
    k = torch.empty((tokens, kv.heads, kv.dh), dtype=torch.float16, device=k_cache.device)
    v = torch.empty_like(k)
    _check(_lib.load().vedic_kv_read(ctypes.byref(kv), k.data_ptr(), v.data_ptr(), _stream()))
    return k, v


def paged_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, table: torch.Tensor,
                    lens: torch.Tensor, q_start: torch.Tensor | None = None, scale: float | None = None,
                    causal: bool = True, window: int = 0, stride: int = 0, out: torch.Tensor | None = None,
                    lse: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of new tokens over a paged cache that holds them (kv_append): q float16 [tokens, q_heads, dh], head j with
    key head j // (q_heads // heads); float16 out.  A row sees the keys up to its own position (causal; else its
    sequence's all), with window > 0 those from `window` before it on, and further back, with stride > 0, those at multiples of
    stride.  scale defaults to 1/sqrt(dh).  lse (float32 [tokens, q_heads]) receives each row's log-sum-exp.  table, lens
    and q_start as for kv_append.  See vedic_paged_attention in logos_vedic.h."""
    dev = _device(q)
    pq, T, Hq, D, qt, qh = _heads3d(q, "q", torch.float16, dev)
    kv = _kv(k_cache, v_cache, table, lens, q_start, T, dev)
    if D != kv.dh or Hq % kv.heads != 0:
        raise ValueError(f"q must be [tokens, a multiple of {kv.heads}, {kv.dh}], got {tuple(q.shape)}")
    if out is None:
        out = q.new_empty((T, Hq, D))
        po, ot, oh = out.data_ptr(), Hq * D, D
    else:
        po, To, Ho, Do, ot, oh = _heads3d(out, "out", torch.float16, dev)
        if (To, Ho, Do) != (T, Hq, D):
            raise ValueError(f"out must be {T}x{Hq}x{D}")
    pl = None if lse is None else _floats(lse, "lse", (T, Hq), dev)
    if scale is None:
        scale = 1.0 / float(D) ** 0.5
    _check(_lib.load().vedic_paged_attention(ctypes.byref(kv), pq, qt, qh, Hq, po, ot, oh, pl, scale, causal, window, stride,
                                             _stream()))
    return out


class W4(NamedTuple):
    """A weight [K, N] in four bits (vedic_w4_t in logos_vedic.h)."""

    codes: torch.Tensor   # int32 [N, ceil(K / 32) * 4]: words of eight codes along K
    scales: torch.Tensor  # float16 [N, ceil(K / group), 2]: pairs (s, m)
    K: int
    group: int


def _w4(w: W4, dev: int) -> _lib.W4Desc:
    pc = _on_current(w.codes, "codes", torch.int32, dev)
    ps = _on_current(w.scales, "scales", torch.float16, dev)
    K, group = w.K, w.group
    if group not in (32, 64, 128) or K <= 0:
        raise ValueError(f"group must be 32, 64 or 128 and K positive, got {group} and {K}")
    N = w.codes.shape[0]
    if tuple(w.codes.shape) != (N, -(-K // 32) * 4) or tuple(w.scales.shape) != (N, -(-K // group), 2) or \
            not w.codes.is_contiguous() or not w.scales.is_contiguous():
        raise ValueError(f"codes must be contiguous [N, {-(-K // 32) * 4}] and scales [N, {-(-K // group)}, 2], got "
                         f"{tuple(w.codes.shape)} and {tuple(w.scales.shape)}")
    return _lib.W4Desc(pc, ps, K, N, group)


def w4_quantize(W: torch.Tensor, group: int = 64) -> W4:
    """W (float16 or float32 [K, N]) in four bits, a scale and a minimum per `group` (32, 64, 128) values along K."""
    dev = _device(W)
    if W.dtype not in _DT:
        raise ValueError(f"W must be float16 or float32, got {W.dtype}")
    p, K, N, ld = _rows2d(W, "W", W.dtype, dev)
    if group not in (32, 64, 128):
        raise ValueError(f"group must be 32, 64 or 128, got {group}")
    w = W4(torch.empty((N, -(-K // 32) * 4), dtype=torch.int32, device=W.device),
           torch.empty((N, -(-K // group), 2), dtype=torch.float16, device=W.device), K, group)
    _check(_lib.load().vedic_w4_quantize(p, _DT[W.dtype], ld, K, N, group, w.codes.data_ptr(), w.scales.data_ptr(), _stream()))
    return w


def w4_unpack(w: W4, out: torch.Tensor | None = None) -> torch.Tensor:
    """The values a four-bit weight stands for, float16 [K, N]."""
    dev = _device(w.codes)
    d = _w4(w, dev)
    if out is None:
        out = torch.empty((d.K, d.N), dtype=torch.float16, device=w.codes.device)
    p, r, c, ld = _rows2d(out, "out", torch.float16, dev)
    if (r, c) != (d.K, d.N):
        raise ValueError(f"out must be {d.K}x{d.N}")
    _check(_lib.load().vedic_w4_unpack(ctypes.byref(d), p, ld, _stream()))
    return out


def gemm_w4(X: torch.Tensor, w: W4, bias: torch.Tensor | None = None, epilogue: int | None = None,
            out: torch.Tensor | None = None, out_dtype: torch.dtype = torch.float32) -> torch.Tensor:
    """C = epi(X . W) with a four-bit weight: X float16 [M, K], or float32 (clamped and rounded to float16 as it is read);
    fp32 sums; C float32 or float16.  epilogue EPI_NONE, EPI_BIAS, EPI_BIAS_GELU, or EPI_RESIDUAL, EPI_BIAS_RESIDUAL, which
    add to a float32 `out`; by default EPI_BIAS with a bias, EPI_NONE without.  See vedic_gemm_w4 in logos_vedic.h."""
    dev = _device(X)
    if X.dtype not in _DT:
        raise ValueError(f"X must be float16 or float32, got {X.dtype}")
    px, M, K, ldx = _rows2d(X, "X", X.dtype, dev)
    d = _w4(w, dev)
    if K != d.K:
        raise ValueError(f"VedicGEMM: inner dimensions differ (X gives K={K}, W gives K={d.K})")
    if epilogue is None:
        epilogue = EPI_NONE if bias is None else EPI_BIAS
    if out is None:
        if epilogue in (EPI_RESIDUAL, EPI_BIAS_RESIDUAL):
            raise ValueError("the residual epilogues add to an existing float32 out")
        out = X.new_empty((M, d.N), dtype=out_dtype)
    if out.dtype not in _DT:
        raise ValueError("out must be float32 or float16")
    pc, Mc, Nc, ldc = _rows2d(out, "out", out.dtype, dev)
    if (Mc, Nc) != (M, d.N):
        raise ValueError(f"out must be {M}x{d.N}, got {Mc}x{Nc}")
    wants = epilogue in (EPI_BIAS, EPI_BIAS_GELU, EPI_BIAS_RESIDUAL)
    if wants != (bias is not None):
        raise ValueError("a bias goes with EPI_BIAS, EPI_BIAS_GELU and EPI_BIAS_RESIDUAL")
    pb = None if bias is None else _floats(bias, "bias", (d.N,), dev)
    _check(_lib.load().vedic_gemm_w4(ctypes.byref(d), px, _DT[X.dtype], ldx, M, pc, _DT[out.dtype], ldc, pb, epilogue, _stream()))
    return out
