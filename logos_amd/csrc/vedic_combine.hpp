// vedic_combine.hpp -- launch interface of vedic_combine.hip.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace vedic {

struct CombineArgs {
    const void* Y;  // [R x ldy]
    int64_t ldy;
    int R;
    const int* slots;      // [T x k]; outside 0 .. R - 1: no row
    const float* weights;  // [T x k], or null: ones
    const float* residual; // or null
    int64_t ldr;
    float* out;
    int64_t ldo;
    int T, k, D;
};

struct CombineBwdArgs {
    const float* dout;
    int64_t ldg;
    const void* Y;
    int64_t ldy;
    int R;
    const int* slots;
    const float* weights;
    void* dY;
    int64_t ldo;
    float* dweights;
    int T, k, D;
};

hipError_t launch_combine(CombineArgs a, bool f16, hipStream_t s);
hipError_t launch_combine_bwd(const CombineBwdArgs& a, bool f16, bool out16, hipStream_t s);
// dst[i] = src[rows[i]], `cols` values of es bytes (2 or 4); n > 0.
hipError_t launch_gather_rows(const void* src, int64_t ld, int nsrc, const int* rows, int n, int cols, int es, void* dst,
                              int64_t ldd, hipStream_t s);
// C_g = beta C_g + the sum of S slabs [groups][M x N], in order.
hipError_t launch_slab_sum(const float* ws, int S, int groups, int M, int N, float* C, int64_t ldc, int64_t stride_c, float beta,
                           hipStream_t s);
// C (binary16 with out16) = the sum of S slabs [R x N], in order, plus the group's bias (or
// none) in the rows 0 .. offsets[groups] - 1 (null offsets: one group of all rows).
hipError_t launch_slab_rows(const float* ws, int S, int R, int N, const int* offsets, int groups, const float* bias, void* C,
                            int64_t ldc, bool out16, hipStream_t s);
// dst [n x roundup(cols, 8)] binary16 = n rows of `cols` values of src (matrices of `per`
// rows, `stride` apart; or its rows rows[i], nsrc of them there), padded with zeros; n > 0.
hipError_t launch_pad_rows(const void* src, int64_t ld, int per, int64_t stride, int nsrc, const int* rows, int64_t n, int cols,
                           void* dst, hipStream_t s);
// db[e] = beta db[e] + column sums of the group's rows of X.
hipError_t launch_group_colsum(const void* X, bool f16, int64_t ld, int R, int N, const int* offsets, int groups, float beta,
                               float* db, hipStream_t s);

}  // namespace vedic
