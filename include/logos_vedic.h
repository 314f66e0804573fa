/*
 * logos_vedic.h -- C ABI of the MI355X-native (gfx950) LOGOS Vedic GEMM.
 *
 * Drop-in boundary for the GEMM hot path of LOGOS
 * (reference: cuda/VedicGEMM.cuh, cuda/MixedPrecision.cuh).  Plain pointers
 * and sizes only; device pointers are HIP device memory; `stream` is a
 * hipStream_t (NULL = the null stream).  Every call is asynchronous on its
 * stream unless stated otherwise, and returns a vedic_status_t.
 *
 * Layout: all matrices are row-major with an explicit leading dimension in
 * elements.  Sizes are int (the reference uses int everywhere); element
 * offsets are computed in 64 bits.
 *
 * Semantics of one GEMM (every entry point below is a special case of
 * vedic_gemm):
 *     acc   = op(A) . op(B)                      (fp32 accumulation)
 *     t     = alpha * acc + beta * C_old         (C_old not read if beta == 0)
 *     t     = t + bias[j]                        (if the epilogue has a bias)
 *     pre   = t                                  (stored if preact != NULL)
 *     C     = gelu_tanh(t) or t                  (per the epilogue)
 *     C     = t * gelu_tanh'(P)                  (VEDIC_EPI_GELU_BWD, P read from preact)
 *     C     = C_old + t                          (VEDIC_EPI_*RESIDUAL, beta = 0; t after the bias)
 *     colsum[j] = colsum_beta * colsum[j] + sum_i C[i][j]   (if colsum != NULL)
 * where gelu_tanh(x) = 0.5 x (1 + tanh(0.7978845608 (x + 0.044715 x^3)))
 * (include/FeedForward.hpp:11-13).  For alpha = 1, beta = 0 the bias is added
 * after the full dot product, as vedic_gemm_bias does
 * (include/VedicGEMM.hpp:56-65).
 *
 * Memory: the caller allocates every output.  A product whose output has too
 * few tiles to fill the GPU and whose contraction is long (fp16: fewer than
 * 128 tiles of 128 x 128 and K >= 2048; fp32: fewer than 256 and K >= 256) runs
 * split over K and takes an fp32 workspace of S * M * N * 4 bytes (S <= 8;
 * S <= 16 for fp32 products with N <= 64).  Workspaces (this, column partials, the AMP cast
 * buffer, attention partials and padded copies) come from a block of device
 * memory kept per (device, stream):
 * grown with hipMallocAsync on `stream` when a call needs more than it holds,
 * reused by every later call on that stream (their work runs in stream
 * order), and held until the process ends or vedic_workspace_release(stream).
 * Host threads may share a stream: a call holds the block from its first
 * request until its last kernel is enqueued.  Results never depend on timing:
 * slices are added in a fixed order.
 *
 * Stream capture: nothing is allocated during one.  The first captured call
 * that needs temporaries takes over the block that an earlier call left on the
 * stream (run the largest call once before the capture, and let it finish
 * before the graph is launched); the graph keeps it until
 * vedic_workspace_release(stream), to be called after the graph's last launch.
 * Without one, products and attention run unsplit and AMP products convert in
 * the kernel where they can, and a call that cannot do without memory returns
 * VEDIC_STATUS_HIP_ERROR (hipErrorStreamCaptureUnsupported) and records
 * nothing.  vedic_gemm_noalloc never needs the block.
 *
 * Errors follow the reference's conventions: shape errors are
 * VEDIC_STATUS_BAD_DIM (the reference throws std::invalid_argument,
 * include/VedicGEMM.hpp:27-30), device errors VEDIC_STATUS_HIP_ERROR (the
 * reference throws std::runtime_error from CUDA_CHECK, cuda/VedicGEMM.cuh:111-133).
 * The C++ header VedicGEMM_hip.hpp rethrows them as those exceptions.
 */
#ifndef LOGOS_VEDIC_H
#define LOGOS_VEDIC_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

typedef enum {
    VEDIC_STATUS_OK = 0,
    VEDIC_STATUS_BAD_DIM = 1,      /* non-positive or inconsistent M/N/K */
    VEDIC_STATUS_BAD_LAYOUT = 2,   /* unknown op */
    VEDIC_STATUS_NULL_POINTER = 3, /* required pointer is NULL */
    VEDIC_STATUS_BAD_LD = 4,       /* leading dimension smaller than the row */
    VEDIC_STATUS_BAD_EPILOGUE = 5, /* unknown epilogue / bias missing */
    VEDIC_STATUS_BAD_DTYPE = 6,    /* unsupported dtype combination */
    VEDIC_STATUS_HIP_ERROR = 7,    /* HIP runtime or launch error */
    VEDIC_STATUS_TOO_LARGE = 8,    /* size beyond a documented limit */
    VEDIC_STATUS_UNSUPPORTED = 9   /* a case this build does not provide (documented per call) */
} vedic_status_t;

typedef enum {
    VEDIC_OP_NN = 0, /* C[MxN] = A[MxK] . B[KxN]                       */
    VEDIC_OP_NT = 1, /* C[MxN] = A[MxK] . B^T,  B stored [NxK]          */
    VEDIC_OP_TN = 2  /* C[MxN] = A^T . B,       A stored [KxM], B [KxN] */
} vedic_op_t;

typedef enum {
    VEDIC_EPI_NONE = 0,
    VEDIC_EPI_BIAS = 1,      /* + bias[j]                 */
    VEDIC_EPI_BIAS_GELU = 2, /* gelu_tanh(t + bias[j])    */
    VEDIC_EPI_GELU = 3,      /* gelu_tanh(t)              */
    VEDIC_EPI_GELU_BWD = 4,  /* t * gelu_tanh'(P[i][j]), P = the cached
                                pre-activation, read through `preact` */
    VEDIC_EPI_RESIDUAL = 5,  /* C_old + t: C holds the residual stream on entry
                                (beta must be 0; fp32 C; `preact`, if set,
                                receives t) -- the reference's projection
                                followed by residual_add_kernel,
                                cuda/ModelGPU.cu:57-60, 1005-1012 */
    VEDIC_EPI_BIAS_RESIDUAL = 6 /* C_old + (t + bias[j]): the reference's
                                FFN-down amp_gemm_bias into a temporary, then
                                residual_add_kernel (cuda/ModelGPU.cu:1044-1048) */
} vedic_epilogue_t;

typedef enum {
    VEDIC_DT_F32 = 0,     /* IEEE binary32 */
    VEDIC_DT_F16 = 1,     /* IEEE binary16 */
    VEDIC_DT_F32_F16 = 2  /* in_dtype only, op NN only: A binary32, B binary16;
                             A is clamped to +-65504 and rounded to binary16
                             (round to nearest even, as vedic_cast_f32_to_f16)
                             inside the GEMM -- the AMP product of an fp32
                             activation with a binary16 shadow weight */
} vedic_dtype_t;

/* Full descriptor of one GEMM.  A and B share in_dtype (but see
 * VEDIC_DT_F32_F16); C is out_dtype (F16 output only with F16 or F32_F16
 * inputs); bias and preact are always fp32.
 * Zero-initialise it (`= {0}`) so that fields a caller does not use are off. */
typedef struct {
    int op;        /* vedic_op_t */
    int in_dtype;  /* vedic_dtype_t of A and B */
    int out_dtype; /* vedic_dtype_t of C */
    int M, N, K;
    const void* A;
    int64_t lda;
    const void* B;
    int64_t ldb;
    void* C;
    int64_t ldc;
    float alpha;
    float beta;
    const float* bias; /* [N], required for *_BIAS* epilogues */
    int epilogue;      /* vedic_epilogue_t */
    float* preact;     /* optional [M x ld_preact] pre-activation output;
                          the pre-activation input of VEDIC_EPI_GELU_BWD */
    int64_t ld_preact;
    void* stream;      /* hipStream_t */
    /* Optional column sums of the final C (fp32 C only):
     *     colsum[j] = colsum_beta * colsum[j] + sum_i C[i][j]
     * -- the bias gradient of a layer whose output gradient C is.  Added in a
     * fixed order (no atomics), so the result does not depend on timing. */
    float* colsum;
    float colsum_beta;
} vedic_gemm_desc_t;

/* The general entry point.  New: the reference has no single descriptor
 * call; every function below forwards to it. */
int vedic_gemm(const vedic_gemm_desc_t* desc);

/* vedic_gemm that allocates nothing, for callers that cannot call hipMalloc
 * (code under HIP graph capture, tight serving loops, harnesses that forbid
 * allocation).  No counterpart in the reference.  Same semantics, kernels and
 * results as vedic_gemm; the temporary memory vedic_gemm takes from the
 * stream's workspace block (split-K partial slabs, column partials, the AMP
 * cast buffer) comes instead from a fixed per-GPU region of
 * vedic_noalloc_scratch_bytes() bytes (32 MiB) compiled into the library and
 * held until the process ends.  A call that needs more returns
 * VEDIC_STATUS_TOO_LARGE before launching anything that writes C.  Every call
 * on one GPU shares that region, so calls whose kernels can be in flight at
 * the same time race: calls from two host threads, and also calls made one
 * after another by one thread on two different streams (the second call's
 * kernels may start before the first call's have finished).  Order such
 * calls on the GPU: issue them on one stream, or make the second stream wait
 * for an event recorded after the first call. */
int vedic_gemm_noalloc(const vedic_gemm_desc_t* desc);

/* Size of the region vedic_gemm_noalloc draws from (per GPU). */
size_t vedic_noalloc_scratch_bytes(void);

/* Frees the workspace block kept for `stream` on the current device, and the
 * attention work-queue counter kept with it (in stream order, after the work
 * queued on them); the next call on the stream allocates new ones.  Call it
 * before destroying a stream the library has used: blocks are keyed by the
 * stream handle, and a stream created later with the same handle would
 * otherwise inherit the block while work of the destroyed stream may still be
 * using it.  hipStreamPerThread names a different stream in every host
 * thread; its blocks are kept per thread, and a thread that used it releases
 * its own (pass hipStreamPerThread) before it exits.  New: the reference
 * allocates per call and keeps nothing. */
int vedic_workspace_release(void* stream);

/* ---- reference-compatible entry points ------------------------------- */

/* C[MxN] = A[MxK] . B[KxN], fp32.
 * Replaces cuda_vedic_gemm (cuda/VedicGEMM.cuh:182, cuda/VedicGEMM.cu:645-673). */
int vedic_gemm_f32(const float* A, const float* B, float* C, int M, int K, int N, void* stream);

/* C = A . W + bias[j], fp32.
 * Replaces cuda_vedic_gemm_bias (cuda/VedicGEMM.cuh:184, cuda/VedicGEMM.cu:675-690). */
int vedic_gemm_bias_f32(const float* A, const float* W, const float* bias, float* C, int M, int K,
                        int N, void* stream);

/* C[MxN] fp32 = alpha * A[MxK] . B[KxN] + beta * C, fp16 inputs, fp32 accumulate.
 * Replaces cuda_gemm_fp16_fp32out (cuda/VedicGEMM.cuh:251, cuda/VedicGEMM.cu:1150-1178,
 * cuda/MixedPrecision.cuh:301-330).  A, B point to binary16 data. */
int vedic_gemm_f16_f32out(const void* A, int M, int K, const void* B, int N, float* C, float alpha,
                          float beta, void* stream);

/* Same with a binary16 C (fp32 accumulate, rounded once at the store).
 * Replaces cuda_gemm_fp16_fp16out (cuda/VedicGEMM.cuh:252, cuda/VedicGEMM.cu:1182-1197). */
int vedic_gemm_f16_f16out(const void* A, int M, int K, const void* B, int N, void* C, float alpha,
                          float beta, void* stream);

/* Fused FFN-up: H = gelu_tanh(X . W + bias), fp16 X/W, fp32 accumulate and
 * output; preact (nullable) receives X . W + bias.
 * Replaces the amp_gemm_bias + D2D copy + cuda_gelu sequence
 * (cuda/ModelGPU.cu:1023-1028, cuda/VedicGEMM.cu:96-102,202-208,707-711). */
int vedic_gemm_bias_gelu_f16(const void* X, const void* W, const float* bias, float* H,
                             float* preact, int M, int K, int N, void* stream);

/* fp32 form of the same fused epilogue (FeedForward::forward,
 * include/FeedForward.hpp:112-114). */
int vedic_gemm_bias_gelu_f32(const float* X, const float* W, const float* bias, float* H,
                             float* preact, int M, int K, int N, void* stream);

/* AMP products from an fp32 activation, the reference's amp_gemm /
 * amp_gemm_bias lambdas (cuda/ModelGPU.cu:819-859):
 *     C[MxN] = binary16(A)[MxK] . W16[KxN]            (+ bias[j])
 * with binary16(A) the clamp-and-round of cast_fp32_to_fp16_kernel
 * (cuda/MixedPrecision.cuh:149-161), applied inside the GEMM as A is staged
 * (no cast pass and no per-call buffer, where the reference allocates and
 * casts the activation on every call, cuda/ModelGPU.cu:825-827); fp32
 * accumulation and output.  When W16 is NULL the call is the fp32 product
 * with W32, as the reference falls back to cuda_vedic_gemm(_bias) for a
 * parameter without a shadow.  A and C contiguous.  For N > 1024, for
 * N > 512 with K >= 2048 and M > 32, or an A whose base is not 16-byte aligned
 * or whose K is not a multiple of 8, the call casts A into an M x K binary16
 * workspace (the stream's workspace block) and runs the fp16 GEMM on it: each
 * output tile reads and converts its own rows of the fp32 A, ceil(N / 128)
 * times per element, which loses to one cast pass for wide products.  Results
 * are the same bits either way. */
int vedic_amp_gemm(const float* A, int M, int K, const void* W16, const float* W32, int N, float* C,
                   void* stream);
int vedic_amp_gemm_bias(const float* A, int M, int K, const void* W16, const float* W32, int N,
                        const float* bias, float* C, void* stream);

/* The fused FFN-up from the fp32 activation: H = gelu_tanh(binary16(X) . W16
 * + bias), preact (nullable) receives the pre-activation.  Replaces
 * amp_gemm_bias + D2D copy + cuda_gelu (cuda/ModelGPU.cu:1023-1028) with one
 * launch; W16 NULL gives the fp32 form with W32 (vedic_gemm_bias_gelu_f32). */
int vedic_amp_gemm_bias_gelu(const float* X, int M, int K, const void* W16, const float* W32, int N,
                             const float* bias, float* H, float* preact, void* stream);

/* NT backward: dX[MxN] = dY[MxK] . W^T + beta * dX, W stored [NxK].
 * Replaces lmhead_grad_dx / ffn_da / ffn_dx / attn_dConcat / attn_dHeadOut
 * (cuda/train_gpu.cu:221-230,323-332,358-367,536-545,514-523; beta = 0) and
 * attn_dX_from_QKV (:492-501; beta = 1). */
int vedic_gemm_nt_f32(const float* dY, const float* W, float* dX, int M, int N, int K, float beta,
                      void* stream);
int vedic_gemm_nt_f16(const void* dY, const void* W, float* dX, int M, int N, int K, float beta,
                      void* stream);

/* TN backward: dW[MxN] = X^T . dY + beta * dW, X stored [KxM], dY [KxN].
 * Replaces lmhead_grad_dw / ffn_w2_grad / ffn_w1_grad / attn_dWproj /
 * attn_dWO / attn_dWQKV (cuda/train_gpu.cu:210-219,312-321,347-356,525-534,
 * 503-512,481-490), which atomicAdd into zeroed, micro-batch-accumulated
 * buffers: beta = 1 reproduces that accumulation deterministically. */
int vedic_gemm_tn_f32(const float* X, const float* dY, float* dW, int M, int N, int K, float beta,
                      void* stream);
int vedic_gemm_tn_f16(const void* X, const void* dY, float* dW, int M, int N, int K, float beta,
                      void* stream);

/* The GEMM of `desc` with the columns of C scattered to separate matrices:
 * columns [h * head_cols, (h + 1) * head_cols) of C go to heads[h], a
 * row-major [M x head_cols] fp32 matrix (desc->C and ldc are not used).
 * head_cols a multiple of 32, nheads * head_cols = N, nheads <= 64;
 * epilogue NONE or BIAS, alpha = 1, beta = 0, no colsum or preact; A and B
 * aligned as for the 16-byte-load path (VEDIC_STATUS_BAD_LD otherwise).
 * New: one packed Q/K/V projection (see vedic_cast_pack_f16) that still
 * fills the per-head hc.Q / hc.K / hc.V buffers the reference's attention
 * reads (cuda/ModelGPU.cu:894-906, 48 amp_gemm calls per layer). */
int vedic_gemm_scatter(const vedic_gemm_desc_t* desc, float* const* heads, int nheads, int head_cols);

/* fp16 convenience form: heads <- X[MxK] . W[KxN], X and W binary16. */
int vedic_gemm_f16_scatter(const void* X, int M, int K, const void* W, int N, float* const* heads, int nheads,
                           int head_cols, void* stream);

/* The mirror of vedic_gemm_scatter on the A side, for the attention-output
 * projection: A is gathered from separate matrices and the contraction is
 * accumulated head by head,
 *     C[MxN] = sum over h in 0..nheads-1, in that order, of
 *              heads[h][M x head_cols] . B[h head_cols .. (h+1) head_cols)[KxN],
 * each head's product taken from zero in fp32 and added to the running sum
 * (round to nearest), starting from a zeroed C: bit for bit the result of
 * zeroing C and calling vedic_gemm once per head with beta = 1.  Replaces the
 * reference's per-head loop amp_gemm(hc.head_out, W_O[h]) + residual_add_kernel
 * into `concat` (cuda/ModelGPU.cu:976-986; residual_add_kernel :57-60), 16
 * launches of K = 64 and 16 passes over the 32 MB concat per layer, with one
 * launch over the row-stacked W_O (vedic_cast_stack_f16).
 * desc: op NN; in_dtype VEDIC_DT_F16 (binary16 heads) or VEDIC_DT_F32_F16
 * (fp32 heads, the reference's head_out, rounded to binary16 as they are
 * read, as the AMP entry points do); B binary16 [K x N], K = nheads *
 * head_cols; out_dtype F32; epilogue NONE, alpha 1, beta 0, no colsum or
 * preact (VEDIC_STATUS_BAD_EPILOGUE otherwise); desc->A unused; desc->lda is
 * the heads' leading dimension (>= head_cols).  nheads <= 64.
 * One launch when head_cols is a multiple of 64, N > 64, M > 32 and every
 * head, B and the leading dimensions are aligned as for the 16-byte-load path
 * (then each per-head product is one MFMA chain per output, which the launch
 * repeats); otherwise the per-head calls themselves (same result).  With fp32 heads and N > 1024
 * the heads are first cast into an M x K binary16 block of the stream's
 * workspace. */
int vedic_gemm_gather(const vedic_gemm_desc_t* desc, const void* const* heads, int nheads, int head_cols);

/* FFN backward through the activation, fused:
 *     dH[MxN] = (dY[MxK] . W^T) * gelu_tanh'(H),   W stored [NxK],
 *     db[j]  += sum_i dH[i][j]                     (db nullable),
 * with H the cached pre-activation [MxN] (the `preact` output of
 * vedic_gemm_bias_gelu_*).  Replaces ffn_da + gelu_bwd + bias_grad
 * (cuda/train_gpu.cu:323-332, 334-345, 263-273, launched at :590-597 and
 * :617-618): one pass over dH instead of three, and no atomics. */
int vedic_gemm_nt_gelu_bwd_f16(const void* dY, const void* W, const float* H, float* dH, float* db, int M,
                               int N, int K, void* stream);
int vedic_gemm_nt_gelu_bwd_f32(const float* dY, const float* W, const float* H, float* dH, float* db, int M,
                               int N, int K, void* stream);

/* db[j] = beta * db[j] + sum_i dY[i][j] over an MxN fp32 matrix, summed in a
 * fixed order.  Replaces bias_grad_kernel (cuda/train_gpu.cu:263-273), which
 * atomicAdds into db (beta = 1). */
int vedic_bias_grad(const float* dY, float* db, int M, int N, float beta, void* stream);

/* ---- elementwise helpers on the path ---------------------------------- */

/* C[i][j] += bias[j] over an MxN matrix.
 * Replaces add_bias_kernel (cuda/VedicGEMM.cuh:191, cuda/VedicGEMM.cu:96-102). */
int vedic_add_bias(float* C, const float* bias, int M, int N, void* stream);

/* Row layer normalisation: Y[i][j] = gamma[j] (X[i][j] - mean_i) /
 * sqrt(var_i + eps) + beta[j], the mean and the biased variance of row i's d
 * values accumulated in fp32 (in a fixed order).  Replaces cuda_layernorm
 * (cuda/VedicGEMM.cuh:186, cuda/VedicGEMM.cu:157-193,699-705).  Y (fp32) and
 * Y16 (binary16) are each optional, at least one: Y16 receives Y clamped to
 * +-65504 and rounded to nearest even -- the bits vedic_cast_f32_to_f16(Y)
 * would give -- in the same pass, so an fp16 GEMM takes the normalised
 * activation without the per-call cast of the reference's amp_gemm
 * (cuda/ModelGPU.cu:825-827).  New: the reference writes fp32 only.
 * The summation order is fixed for a given d and operand alignment (rows with
 * d a multiple of 4 up to 4096 and 16-byte aligned X, gamma, beta, Y and
 * 8-byte aligned Y16 are reduced one wave per row, others one workgroup per
 * row), so repeated calls give the same bits; the same rows at another
 * alignment may differ in the last bits. */
int vedic_layernorm(const float* X, const float* gamma, const float* beta, float* Y, void* Y16, int seq, int d,
                    float eps, void* stream);

/* The same on binary16 rows, binary16 out (fp32 statistics; the output
 * clamped to +-65504 before rounding).  Replaces cuda_layernorm_fp16
 * (cuda/VedicGEMM.cuh:253, cuda/MixedPrecision.cuh:458-511).  One wave per
 * row when d is a multiple of 4 up to 4096 and X16 and Y16 are 8-byte
 * aligned (gamma and beta 16-byte), one workgroup per row otherwise; as
 * above, the bits are repeatable for a given alignment. */
int vedic_layernorm_f16(const void* X16, const float* gamma, const float* beta, void* Y16, int seq, int d, float eps,
                        void* stream);

/* In-place tanh-GELU over n floats.
 * Replaces cuda_gelu (cuda/VedicGEMM.cuh:187, cuda/VedicGEMM.cu:707-711). */
int vedic_gelu(float* x, int64_t n, void* stream);

/* dst = binary16(clamp(src, -65504, 65504)), round to nearest even.
 * Replaces cuda_cast_fp32_to_fp16 (cuda/MixedPrecision.cuh:149-161,177-190). */
int vedic_cast_f32_to_f16(const float* src, void* dst, int64_t n, void* stream);

/* nsrc fp32 [rows x cols] matrices cast to binary16 (the clamp and rounding
 * above) and packed side by side: dst[r][i * cols + c] = src[i][r][c], dst
 * row-major with leading dimension ld_dst >= nsrc * cols; nsrc <= 64.  The
 * shadow-weight cast of cuda/train_gpu.cu:1542-1547, with the per-head
 * W_Q / W_K / W_V of a layer packed into one [D x 3 H DH] matrix for
 * vedic_gemm_f16_scatter. */
int vedic_cast_pack_f16(const float* const* src, int nsrc, int rows, int cols, void* dst, int64_t ld_dst,
                        void* stream);

/* The same cast with the matrices stacked by rows: dst[i * rows + r][c] =
 * src[i][r][c], dst row-major with leading dimension ld_dst >= cols; nsrc <=
 * 64.  The shadow-weight cast of cuda/train_gpu.cu:1542-1547 applied to a
 * layer's per-head W_O[h] [DH x D] blocks, stacked into the [H DH x D] B
 * operand of vedic_gemm_gather. */
int vedic_cast_stack_f16(const float* const* src, int nsrc, int rows, int cols, void* dst, int64_t ld_dst,
                         void* stream);

/* dst = float(src).  Replaces cuda_cast_fp16_to_fp32 (cuda/MixedPrecision.cuh:164-172,192-196). */
int vedic_cast_f16_to_f32(const void* src, float* dst, int64_t n, void* stream);

/* Gunitasamuchayah check of C = A . B (fp32, NN): sum(C) against
 * colsum(A) . rowsum(B).  Synchronous (it returns host values).
 * Replaces cuda_vedic_verify (cuda/VedicGEMM.cuh:193, cuda/VedicGEMM.cu:765-814). */
typedef struct {
    float checksum_C;
    float checksum_vedic;
    float relative_error;
    int pass;
} vedic_verify_result_t;

int vedic_verify(const float* A, const float* B, const float* C, int M, int K, int N,
                 float tolerance, vedic_verify_result_t* out, void* stream);

/* The GEMM `desc` with the same check computed on the way (algorithm-based
 * fault tolerance): sum(C) from column sums the GEMM's epilogue accumulates,
 * so C is not read again, against colsum(op(A)) . rowsum(op(B)) (times alpha,
 * plus M * sum(bias) with VEDIC_EPI_BIAS) from one pass over A and B, in
 * double.  Any op and input dtype; fp32 C; epilogue NONE or BIAS; beta = 0;
 * desc->colsum must be NULL.  Synchronous, like vedic_verify.  The result
 * doubles land in a 64-byte pinned host slot allocated on a host thread's
 * first call and kept for the process (one per thread).  New: the
 * reference verifies with a separate pass over C at checkpoints
 * (cuda/train_gpu.cu:1695-1719). */
int vedic_gemm_checked(const vedic_gemm_desc_t* desc, float tolerance, vedic_verify_result_t* out);

/* ---- attention ------------------------------------------------------------ */

/* Fused attention forward of one head, fp32:
 *   out[seq x dh] = softmax(scale * Q K^T + mask) V,   Q, K, V [seq x dh] row-major
 * mask: key > query when `causal`; when `shunyam` and seq > window, also every
 * key outside [query - window, query] that is not a multiple of `stride`.
 * Masked scores are left out of the sums; a row whose sum is <= 1e-9 is 0.
 * Replaces cuda_flash_attention_fwd (cuda/VedicGEMM.cuh:236, cuda/VedicGEMM.cu:1065-1104;
 * kernel :898-1063), called per head at cuda/ModelGPU.cu:959-968.
 * attn (NULL, or [seq x seq]): the reference's optional probability copy,
 * with the reference's values (its flash kernel walks the keys in tiles of 16,
 * FA_TILE at cuda/VedicGEMM.cu:898, with a running row maximum): an allowed
 * key k gets expf(s_k - m_t) / l,
 * m_t the running maximum after the tile holding k and l the row sum; a
 * masked key keeps its previous content times 1 / l (the reference's final
 * pass scales the whole row; 0 for a row with l <= 1e-9).  Computed by a
 * second kernel after the output, two passes over the keys.
 * Limits: 1 <= dh <= 128 (BAD_DIM otherwise, where the reference throws);
 * stride >= 1 when the sparse mask applies; seq * (dh <= 64 ? 64 : 128) <
 * 2^29.  The kernels run
 * at dh 64 and 128 on 16-byte-aligned matrices; any other dh, or an
 * unaligned matrix, is copied into zero-padded [seq x 64] or [seq x 128]
 * matrices first and the output copied back (the zero columns add exact
 * zeros to every sum).  A call on a single head splits long key ranges over
 * several workgroups; partial results and padded copies live in the
 * stream's workspace block (see vedic_gemm). */
int vedic_flash_attention_fwd(const float* Q, const float* K, const float* V, float* out, float* attn, int seq,
                              int dh, float scale, int causal, int shunyam, int window, int stride, void* stream);

/* vedic_flash_attention_fwd that also writes lse[seq]: for each query row,
 * ln of its softmax denominator, ln(sum over allowed keys of e^(scale q.k))
 * (+inf for a row with no allowed key) -- what the backward below needs.
 * New: the reference keeps no such statistic and recomputes the whole
 * probability matrix for its backward (cuda/train_gpu.cu:672-700). */
int vedic_flash_attention_fwd_lse(const float* Q, const float* K, const float* V, float* out, float* lse, int seq,
                                  int dh, float scale, int causal, int shunyam, int window, int stride,
                                  void* stream);

/* The same for nheads (1..64) heads in one launch: Q[h], K[h], V[h], out[h]
 * per head, every head [seq x dh]; lse may be NULL, or an array of per-head
 * lse outputs (entries may be NULL).  New: the reference calls the one-head
 * kernel once per head (cuda/ModelGPU.cu:888-968). */
int vedic_flash_attention_fwd_heads(const float* const* Q, const float* const* K, const float* const* V,
                                    float* const* out, float* const* lse, int nheads, int seq, int dh, float scale,
                                    int causal, int shunyam, int window, int stride, void* stream);

/* Fused attention backward of one head, fp32: from Q, K, V, the forward's
 * output O and lse (vedic_flash_attention_fwd_lse, same mask arguments) and
 * the output gradient dO, writes
 *   dV = P^T dO,  dQ = scale dS K,  dK = scale dS^T Q,
 *   P = exp(scale Q K^T + mask - lse),  dS = P * (dO V^T - rowsum(dO * O)).
 * Replaces the per-head backward of cuda/train_gpu.cu:672-740 (score
 * recompute, causal mask, softmax, attn_dV_kernel, attn_dAttnProbs_kernel,
 * softmax_bwd_kernel, attn_dQ_kernel, attn_dK_kernel: :422-479) without its
 * two seq x seq buffers.  That code recomputes the probabilities with the
 * causal mask only; with shunyam set this function differentiates the
 * forward as computed (sparse mask included).  dQ, dK, dV are overwritten.
 * Limits and padding as for the forward; takes a workspace of 8 * seq bytes
 * per head, plus the padded copies when dh is not 64 or 128 or a matrix is
 * not 16-byte aligned (the stream's workspace block, see vedic_gemm). */
int vedic_flash_attention_bwd(const float* Q, const float* K, const float* V, const float* O, const float* dO,
                              const float* lse, float* dQ, float* dK, float* dV, int seq, int dh, float scale,
                              int causal, int shunyam, int window, int stride, void* stream);

/* The same for nheads (1..32) heads in one launch (per-head pointer arrays). */
int vedic_flash_attention_bwd_heads(const float* const* Q, const float* const* K, const float* const* V,
                                    const float* const* O, const float* const* dO, const float* const* lse,
                                    float* const* dQ, float* const* dK, float* const* dV, int nheads, int seq,
                                    int dh, float scale, int causal, int shunyam, int window, int stride,
                                    void* stream);

/* ---- rows that choose their weights: routed experts, adapters ------------- */

/* New: the reference has one feed-forward layer per block (include/FeedForward.hpp)
 * and no adapters.  One plan serves them all: `rows` lists rows sorted by group
 * (an expert, an adapter), offsets[g] .. offsets[g + 1] - 1 are group g's places in
 * it.  Plans stay on the GPU: no call reads one on the host or waits for it.  What
 * a plan holds is clamped where it is read (an offset to 0 .. n, a row or slot
 * outside its matrix counts as none), so a bad plan gives wrong values but no
 * access outside the arrays.  Limits: 1024 groups; counts below 2^30 (places of a grouped
 * product 2^27, of adapters 2^23); leading dimensions of grouped products and adapters
 * below 2^22; and fewer than 2^24 tiles, counted as (places / 128 + groups) x (N / 128) for
 * grouped products on the general kernels (TN: groups x (M / 128) x (N / 128)) and for
 * adapters that are F32 or not 16-byte aligned, as (places / 16 + groups) x (N / 256) for
 * the other adapters, each quotient rounded up.  VEDIC_STATUS_TOO_LARGE past them. */

/* The router: for each of T tokens the k largest of its E logits, a tie to the
 * lower index, and their weights exp(x_j - max) / sum, the sum over the chosen
 * ones (renorm != 0) or over all E (renorm == 0); then the T k pairs sorted by
 * expert and, within one, by token.
 *   ids, weights [T x k]   in descending order of the logits
 *   offsets [E + 1]        the first sorted place of each expert, and the end
 *   rows [T k]             the token of each place
 *   slots [T x k]          the place of each pair
 * A logit of -infinity is never chosen: a token with fewer than k others gets id
 * -1, weight 0 and slot -1 in the rest, whose tokens fill the places behind
 * offsets[E].  NaN counts as larger than every number (and makes its token's weights NaN).
 * k <= 64.  More than 64 tokens or 1024 pairs take a few KB of the stream's
 * workspace block. */
int vedic_route_topk(const float* logits, int64_t ld_logits, int T, int E, int k, int renorm, int* ids, float* weights,
                     int* offsets, int* rows, int* slots, void* stream);

/* Its backward: dlogits [T x E] from the choice, its weights and their gradient.
 *   renorm: w_j (dw_j - sum w dw) at the chosen logits, 0 elsewhere;
 *   else:   p_e (dw_e - sum w dw), p the softmax over all, dw_e = 0 if not chosen.
 * The choice itself has no gradient. */
int vedic_route_topk_bwd(const float* logits, int64_t ld_logits, const int* ids, const float* weights,
                         const float* dweights, int T, int E, int k, int renorm, float* dlogits, int64_t ld_dlogits,
                         void* stream);

/* The plan alone: n entries of ids sorted by group, stable.  rows[place] = entry /
 * per_row (1 for one group per row, k for [rows x k] ids), slots (may be NULL) the
 * place of each entry; an id outside 0 .. groups - 1 belongs to no group (slot -1) and
 * its row is among those behind offsets[groups]. */
int vedic_group_rows(const int* ids, int n, int per_row, int groups, int* offsets, int* rows, int* slots, void* stream);

/* Products grouped by expert.  For the places i of group g:
 *   NN  C[i] = epi(A[i] . B_g)      A [rows x K], B_g [K x N], C [rows x N]
 *   NT  C[i] = epi(A[i] . B_g^T)    A [rows x K], B_g [N x K]
 *   TN  C_g = beta C_g + sum over i of A[i]^T B[i]   A [rows x M], B [rows x N], C_g [M x N]
 * with A[i] read at row row_index[i] of A's a_rows rows where a list is given (any
 * row any number of times).  Rows of C behind offsets[groups] keep their content; a
 * group without rows gives C_g = beta C_g.
 * Types: F32 in and out; F16 in, fp32 accumulation, F32 or (NN, NT) F16 out,
 * rounded to nearest even once.  preact has C's type.
 * Epilogues: NN NONE, BIAS, BIAS_GELU (bias [groups x N]; preact, if set, receives
 * the value before the GELU); NT NONE, GELU_BWD (times gelu_tanh'(preact)); TN
 * NONE, and db_g = db_beta db_g + the column sums of group g's rows of B if db is set.
 * The order of every sum is fixed.  Binary16 operands with 16-byte-aligned bases,
 * leading dimensions and strides that are multiples of 8 and contiguous extents that
 * are multiples of 8 run on the fast kernels as they are; others are copied into padded
 * rows in the stream's workspace block first, up to 256 MiB of them, or run on general
 * kernels.  Also in that block: the listed rows of fp32 TN products and of an A of 2 GiB
 * or more, and the slabs of products with few tiles and a long contraction, which several
 * workgroups then share (at most 16 MiB; epilogues NONE and BIAS).  A captured call whose
 * stream has no such block, or one too small, does without the padded copies and the
 * slabs (results may then differ in rounding), and is refused where it needs the listed
 * rows. */
typedef struct {
    int op, in_dtype, out_dtype, epilogue;
    int groups;
    int rows;    /* places: rows of C (NN, NT) or of B (TN) */
    int M, N, K; /* M: TN only; K: NN and NT only */
    const int* offsets;   /* [groups + 1] */
    const int* row_index; /* NULL, or [rows] */
    int a_rows;           /* rows of A, with row_index */
    const void* A;
    int64_t lda;
    const void* B;
    int64_t ldb;
    int64_t stride_b; /* elements from B_g to B_(g+1) (NN, NT) */
    void* C;
    int64_t ldc;
    int64_t stride_c; /* elements from C_g to C_(g+1) (TN) */
    const float* bias;
    void* preact;
    int64_t ld_preact;
    float beta; /* TN only */
    float* db;  /* TN only: [groups x N] */
    float db_beta;
    void* stream;
} vedic_grouped_desc_t;

int vedic_gemm_grouped(const vedic_grouped_desc_t* desc);

/* db_g = beta db_g + the column sums of group g's rows of dY (F32 or F16). */
int vedic_bias_grad_grouped(const void* dY, int dtype, int64_t ld, int R, int N, const int* offsets, int groups, float beta,
                            float* db, void* stream);

/* Sorted rows back in token order:
 *   out[t] = residual[t] + sum over j of weights[t, j] Y[slots[t, j]]
 * (residual NULL: none, it may be out; weights NULL: ones, which is the backward of
 * reading rows through a list).  Y F32 or F16 [R x D]; a slot outside adds nothing.
 * Added in ascending j in fp32. */
int vedic_combine_rows(const void* Y, int y_dtype, int64_t ldy, int R, const int* slots, const float* weights,
                       const float* residual, int64_t ld_residual, float* out, int64_t ld_out, int T, int k, int D,
                       void* stream);

/* Its backward: dY[slots[t, j]] = weights[t, j] dout[t] (F32 or F16, rounded to
 * nearest even), dweights[t, j] = <dout[t], Y[slots[t, j]]> (0 without a slot).  No
 * two pairs may share a slot (those of a plan never do); rows of dY that no slot
 * names keep their content. */
int vedic_combine_rows_bwd(const float* dout, int64_t ld_dout, const void* Y, int y_dtype, int64_t ldy, int R,
                           const int* slots, const float* weights, void* dY, int dy_dtype, int64_t ld_dy, float* dweights,
                           int T, int k, int D, void* stream);

/* Low-rank adapters of many requests beside a shared projection: for the places p
 * of adapter g, i = rows[p]:  C[i] += scales[g] (X[i] . A_g) . B_g, A_g [K x r],
 * B_g [r x N] contiguous, one after another; X, A, B all F32 or all F16, C fp32
 * [M x N], scales NULL: ones.  The product with A_g is summed in fp32 and
 * keeps its values (the kernel for 16-byte-aligned F16 operands holds them as three
 * binary16 parts: to 2^-24 of a value from the row's largest down to 2^-28 of it, to 2^-22
 * down to 2^-40, to 2^-51 of the largest below).  A row may be listed
 * once (two adapters on one row would add to it at the same time); rows not listed
 * keep their content.  r <= 128.  Takes about 6 n r bytes of the stream's workspace block
 * (r rounded up to 32, 64 or 128), and n K values where X is 2 GiB or more and is F32 or
 * not 16-byte aligned. */
int vedic_lora_add(const void* X, int dtype, int64_t ldx, int M, const void* A, const void* B, int groups, int r,
                   const int* offsets, const int* rows, int n, const float* scales, float* C, int64_t ldc, int K, int N,
                   void* stream);

/* The shared projection with them: base's product, then vedic_lora_add of base->A
 * onto base->C.  base: op NN, F32 or F16 in, F32 out, epilogue NONE or BIAS, no preact
 * or colsum.  Operands that are not 16-byte aligned run on the grouped kernels (one
 * group), whose sums may round differently from vedic_gemm's.  A refused call has
 * written nothing. */
int vedic_gemm_lora(const vedic_gemm_desc_t* base, const void* A, const void* B, int groups, int r, const int* offsets,
                    const int* rows, int n, const float* scales);

/* ---- decoding: a paged cache of keys and values, weights in four bits ------ */

/* New: the reference keeps no keys and values (every generated token is a whole forward,
 * cuda/train_gpu.cu:2045) and multiplies binary16 or fp32 weights only.
 *
 * Four bits.  A 32-bit word holds eight consecutive values, value 2i in bits 4i .. 4i + 3 and
 * value 2i + 1 in bits 16 + 4i .. 19 + 4i; code n of a group with the binary16 pair (s, m)
 * stands for binary16(s n + m), rounded once.  Groups are quantised from their binary16
 * values as m = the least, s = binary16((largest - least) / 15), n = (x - m) / s to the
 * nearest (even) of 0 .. 15, 0 where s is 0; a group with an infinity or NaN stands for NaN. */
typedef enum {
    VEDIC_KV_F16 = 0, /* a row: dh binary16 values (dh a multiple of 8)                       */
    VEDIC_KV_I4 = 1   /* a row: dh / 8 words, then dh / 32 pairs (s, m), one per 32 values:
                         5 dh / 8 bytes (dh a multiple of 32)                                 */
} vedic_kv_format_t;

/* A cache and the sequences of one call.  Row `offset` of page p, key head h starts at
 * p stride_page + h stride_head + offset stride_token (binary16 values with F16, bytes with
 * I4) of k and of v.  Position t of sequence b lies in page table[b ld_table + t / page_size],
 * row t % page_size.  lens[b] counts sequence b's tokens, the call's new ones included; its
 * new ones are the last n_b, the call's rows q_start[b] .. q_start[b + 1] - 1 (q_start NULL: row
 * b alone, tokens = batch).  Rows before q_start[0] or from q_start[batch] on belong to no
 * sequence.  The lists stay on the GPU and are clamped where they are read (lengths to what
 * table_cols pages hold, rows to 0 .. tokens, a page outside the cache is page 0 when read
 * and is not written), so that bad ones give wrong values but no access outside the arrays.
 * Limits: dh <= 256; 2^30 positions; fewer than 2^30 query rows (tokens x heads), 2^20
 * sequences and 2^24 workgroups a launch (VEDIC_STATUS_TOO_LARGE past them).
 * Alignment: rows, q and outputs of 16 bytes, I4 rows of 4 (VEDIC_STATUS_BAD_LD). */
typedef struct {
    int format; /* vedic_kv_format_t */
    int pages, page_size, heads, dh;
    void* k;
    void* v;
    int64_t stride_page, stride_head, stride_token;
    const int* table;
    int64_t ld_table;
    int table_cols;
    const int* lens;
    const int* q_start;
    int batch, tokens;
} vedic_kv_t;

/* New tokens into the cache: k and v [tokens x heads x dh], F32 or F16 at any strides (in values),
 * k turned by its position, both rounded to binary16 (nearest even) and stored in the cache's
 * format; and, with q_heads > 0, q [tokens x q_heads x dh] turned and rounded into q_out (which
 * overlaps none of q, k and v).  Rotation (rope_dims > 0, even): pairs (x_i, x_(i + rope_dims / 2)) of a row, or
 * (x_2i, x_(2i + 1)) with interleaved, by the angle of row `position` (the last one past the
 * end) of rope [rope_rows x rope_dims]: rope_dims / 2 cosines, then the sines, fp32:
 *     (a, b) -> (a cos - b sin, b cos + a sin),  each product and sum rounded to fp32.
 * No two rows may have one place in the cache.  A row of no sequence, or before its
 * sequence's first position, writes nothing, q_out included. */
int vedic_kv_append(const vedic_kv_t* kv, int dtype, const void* q, int64_t q_token, int64_t q_head, int q_heads,
                    void* q_out, int64_t q_out_token, int64_t q_out_head, const void* k, int64_t k_token,
                    int64_t k_head, const void* v, int64_t v_token, int64_t v_head, const float* rope, int rope_rows,
                    int rope_dims, int interleaved, void* stream);

/* The same tokens' rows back from the cache: k and v [tokens x heads x dh] binary16, contiguous,
 * either NULL (q_start the running sums of lens: whole sequences).  Rows of no sequence are
 * left as they are. */
int vedic_kv_read(const vedic_kv_t* kv, void* k, void* v, void* stream);

/* Attention of the new rows over the cache: q [tokens x q_heads x dh] binary16, head j of q with key
 * head j / (q_heads / heads).  The row at position p = lens[b] - n_b + i sees keys
 * t <= p (causal; else all lens[b]) and, with window > 0 (causal only), of those t >= p - window and,
 * with stride > 0, also t a multiple of stride -- the masks of vedic_flash_attention_fwd:
 *     out = sum over t of e^(scale q.k_t - M) v_t / sum of the same without v_t,
 * 0 for a row that sees no key, NaN for one that sees only keys of score -infinity.  lse (NULL, or
 * [tokens x q_heads]): ln of sum e^(scale q.k_t), +inf and NaN for such rows.  out (which does not overlap q)
 * binary16, rounded once; scores and sums fp32.  The weights that multiply v_t are binary16 relative to the row's
 * largest: of two parts (22 bits) for the sequences that share out their keys over a binary16 cache (below), else of
 * one.  What a masked key or a page's unused row holds, NaN included, does not reach the output.  Rows of no sequence
 * are left as they are.
 * Sequences of up to 64 rows (n_b x q_heads / heads) share out their keys evenly over the GPU,
 * others -- and, with q_start and heads up to 192, all those of a call with 64 rows and more a
 * sequence on average -- take 128 rows a workgroup and share keys where that leaves CUs idle; parts are added in
 * a fixed order, 512 x CUs x (dh + 2) fp32 of the stream's workspace block at
 * most.  A captured call without such a block does not split (results may then differ in
 * rounding), and of more than 2^14 sequences it is refused (VEDIC_STATUS_HIP_ERROR).  Calls of more than 128 sequences
 * sum up their work in one more launch. */
int vedic_paged_attention(const vedic_kv_t* kv, const void* q, int64_t q_token, int64_t q_head, int q_heads, void* out,
                          int64_t out_token, int64_t out_head, float* lse, float scale, int causal, int window,
                          int stride, void* stream);

/* A weight W [K x N] in four bits: column n's ceil(K / 32) * 4 words (values past K are not used, but
 * their codes are there) at codes + n * that, and its ceil(K / group) pairs (s, m); group 32, 64 or
 * 128 consecutive values of K.  codes 16-byte, scales 4-byte aligned. */
typedef struct {
    const void* codes;
    const void* scales;
    int K, N, group;
} vedic_w4_t;

/* W (F32 or F16, row-major; F32 values rounded to binary16 with the clamp of vedic_cast_f32_to_f16,
 * infinities and NaN kept) into that form. */
int vedic_w4_quantize(const void* W, int dtype, int64_t ldw, int K, int N, int group, void* codes, void* scales,
                      void* stream);

/* The values it stands for, binary16 [K x N]. */
int vedic_w4_unpack(const vedic_w4_t* w, void* W16, int64_t ldw, void* stream);

/* C[M x N] = epi(X[M x K] . W): X F16, or F32 clamped and rounded to binary16 as it is read; products of
 * binary16 values summed in fp32; C F32 or F16.  Epilogues NONE, BIAS, BIAS_GELU, and (F32 C)
 * RESIDUAL, BIAS_RESIDUAL.  Rows are taken 64 at a time (up to 96 or 128 of them, or where that is
 * a workgroup a CU), in tiles, or by the binary16 tiles from W expanded into the stream's workspace
 * block, in slabs of columns of up to 64 MiB (large products, and a long K of few tiles).  The tiles take an X that is
 * F32, or whose rows are not whole 16 bytes, from a binary16 copy in that block.  A captured call
 * without such a block goes 64 rows at a time (results may then differ in rounding). */
int vedic_gemm_w4(const vedic_w4_t* w, const void* X, int x_dtype, int64_t ldx, int M, void* C, int c_dtype, int64_t ldc,
                  const float* bias, int epilogue, void* stream);

/* ---- test hooks --------------------------------------------------------- */

/* Off by default.  When on, every GEMM with column sums allocates its
 * per-32-row-block partial-sum workspace with a guard band of 8 block rows
 * past its end, filled with a marker; after the GEMM the call checks the band
 * (synchronously) and adds the number of overwritten words to a
 * process-wide counter.  New: no counterpart in the reference; for the
 * regression tests of the workspace bound on partial last tiles. */
void vedic_debug_set_workspace_guard(int on);

/* Overwritten guard words seen since the process started. */
long vedic_debug_workspace_guard_hits(void);

/* ---- backend queries --------------------------------------------------- */

/* Always 0: no vendor BLAS is linked.
 * Replaces cuda_vedic_gemm_uses_cublas (cuda/VedicGEMM.cuh:183, cuda/VedicGEMM.cu:637-643). */
int vedic_uses_vendor_blas(void);

/* "hip-native-gfx950" -- for logs, as the reference logs its GEMM backend
 * (cuda/train_gpu.cu:1920). */
const char* vedic_backend_name(void);

/* Human-readable text for a vedic_status_t. */
const char* vedic_status_string(int status);

/* The last HIP error code seen by this library on the calling thread
 * (0 if none), for VEDIC_STATUS_HIP_ERROR diagnostics. */
int vedic_last_hip_error(void);

#ifdef __cplusplus
}
#endif

#endif /* LOGOS_VEDIC_H */
