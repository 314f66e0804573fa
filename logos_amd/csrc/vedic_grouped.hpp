// vedic_grouped.hpp -- what the grouped products share: their arguments, the
// map from a work item to a group and a tile, and the epilogue.
//
// A grouped product has R rows sorted by group (expert): rows offsets[e] ..
// offsets[e + 1] - 1 belong to group e and take weight B_e.
//   NN  C[i] = epi(A[i] . B_e)      B_e [K x N]
//   NT  C[i] = epi(A[i] . B_e^T)    B_e [N x K]
//   TN  C_e  = beta C_e + A_e^T . B_e over the group's rows (B the gradient rows)
// with A[i] row rows[i] of A where a row list is given.  The group sizes are
// known to the GPU only, so nothing of the grid depends on them: every workgroup
// reads the offsets, counts each group's tiles and finds its own.
//
// Offsets are data: each is clamped to 0 .. R and a group that would end before
// it starts is empty, a row index outside A reads as zeros, so no content of
// either list makes an access out of range.
#pragma once

#include "vedic_common.hpp"
#include "vedic_epilogue.hpp"

namespace vedic {

constexpr int kMaxGroups = 1024;

enum GroupedKind : int {
    GK_LINEAR = 0,    // C = acc (+ b)
    GK_GELU = 1,      // C = gelu(acc (+ b)), P = acc (+ b) if P
    GK_GELU_BWD = 2,  // C = acc * gelu'(P)
    GK_BETA = 3,      // C = acc + beta C
};

struct GroupedArgs {
    const void* A;
    const void* B;
    void* C;
    const float* bias;  // [groups x N]
    void* P;            // of C's type
    const int* offsets;
    const int* rows;    // null: A's own order
    int64_t lda, ldb, ldc, ldp, stride_b, stride_c;
    int groups;
    int R;       // rows of C (NN / NT), of B (TN): offsets are clamped to it
    int a_rows;  // rows of A
    int M, N, K; // NN / NT: N and K; TN: M and N
    float beta;
    int tiles_m, tiles_n;
};

// Tiles before each group, and the clamped offsets, in LDS.
struct GroupIndex {
    int off[kMaxGroups + 1];
    int pre[kMaxGroups + 1];  // row tiles of the groups before e; pre[groups]: all
};

// Fills `ix` (NT threads; ends with a barrier).  BM: rows per tile.
template <int NT>
__device__ __forceinline__ void group_index(const GroupedArgs& a, GroupIndex& ix, int bm) {
    const int tid = threadIdx.x;
    for (int e = tid; e <= a.groups; e += NT) ix.off[e] = min(max(a.offsets[e], 0), a.R);
    __syncthreads();
    if (tid < 64) {
        int carry = 0;
        for (int e0 = 0; e0 < a.groups; e0 += 64) {
            const int e = e0 + tid;
            const int n = e < a.groups ? max(0, ix.off[e + 1] - ix.off[e]) : 0;
            int t = (n + bm - 1) / bm;
#pragma unroll
            for (int d = 1; d < 64; d <<= 1) {
                const int u = __shfl_up(t, d);
                if (tid >= d) t += u;
            }
            if (e < a.groups) ix.pre[e + 1] = carry + t;
            carry += __shfl(t, 63);
        }
        if (tid == 0) ix.pre[0] = 0;
    }
    __syncthreads();
}

// The group that holds row tile t (0 <= t < pre[groups]): the number of groups
// that end at or before it.  Uniform across the wave.
__device__ __forceinline__ int group_of(const GroupIndex& ix, int groups, int t, int lane) {
    int e = 0;
    for (int e0 = 0; e0 < groups; e0 += 64)
        e += __popcll(__ballot(e0 + lane < groups && ix.pre[min(e0 + lane, groups - 1) + 1] <= t));
    return __builtin_amdgcn_readfirstlane(e);
}

// gelu_tanh'(x) = s + 2 c x s (1 - s) (1 + 3 * 0.044715 x^2), s = 1 / (1 + e), e =
// exp(-2 c (x + 0.044715 x^3)), with 1 - s taken as e s: subtracted, its rounding
// error of a unit or two of s is multiplied by up to 2 c x (1 + 3 * 0.044715 x^2), 35
// at x = 5 (gelu_tanh_grad); so it stays below 16 units of 2^-24.  Past +-30, where the
// derivative is 1 or 0 to every bit, x counts as +-30 (its powers would overflow; a
// NaN stays one), and e is held to a finite number, where s rounds to zero.
__device__ __forceinline__ float gelu_grad_fine(float x) {
    constexpr float c = 0.7978845608f;
    constexpr float k0 = -2.0f * c * 1.4426950408889634f;
    constexpr float k1 = -2.0f * c * 0.044715f * 1.4426950408889634f;
    constexpr float k3 = 3.0f * 0.044715f;
    x = x > 30.0f ? 30.0f : x < -30.0f ? -30.0f : x;
    const float x2 = x * x;
    const float e = fminf(__builtin_amdgcn_exp2f(x * __builtin_fmaf(k1, x2, k0)), 3.0e38f);
    const float s = __builtin_amdgcn_rcpf(1.0f + e);
    const float t = x * s * (e * s);
    return __builtin_fmaf(2.0f * c * t, __builtin_fmaf(k3, x2, 1.0f), s);
}

template <typename OT>
__device__ __forceinline__ float ld_out(__amdgpu_buffer_rsrc_t rs, uint32_t voff, uint32_t soff) {
    if constexpr (sizeof(OT) == 2) return ld_f16(rs, voff, soff);
    else return ld_f32(rs, voff, soff);
}
template <typename OT>
__device__ __forceinline__ void st_out(float v, __amdgpu_buffer_rsrc_t rs, uint32_t voff, uint32_t soff) {
    if constexpr (sizeof(OT) == 2) st_f16(v, rs, voff, soff);
    else st_f32(v, rs, voff, soff);
}

// Writes a (32 MI) x (32 NI) wave tile.  C and P point at the tile's first row
// (column 0); `nrow` rows and N columns exist past (that row, column 0); bias
// is the group's, or null.
template <int KIND, typename OT, bool CHECK, int MI, int NI>
__device__ __forceinline__ void grouped_epilogue(void* C, int64_t ldc, void* P, int64_t ldp, const float* bias,
                                                 float beta, const float16_t (&acc)[MI][NI], int nrow, int N, int col0,
                                                 int lane) {
    const int l32 = lane & 31, h = lane >> 5;
    constexpr int ES = sizeof(OT);
    const __amdgpu_buffer_rsrc_t rc = buffer_rsrc(C);
    const __amdgpu_buffer_rsrc_t rp = buffer_rsrc(P);
    const uint32_t ldcb = (uint32_t)(ldc * ES), ldpb = (uint32_t)(ldp * ES);
    const bool wp = KIND == GK_GELU && P != nullptr;
#pragma unroll
    for (int j = 0; j < NI; ++j) {
        const int col = col0 + 32 * j + l32;
        const bool col_ok = !CHECK || col < N;
        const float bj = (KIND == GK_LINEAR || KIND == GK_GELU) && bias != nullptr && col_ok ? bias[col] : 0.0f;
#pragma unroll
        for (int i = 0; i < MI; ++i) {
            float old[16];
            uint32_t oc[16], op[16];
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const int u = 32 * i + 8 * (e >> 2) + (e & 3);
                const bool ok = !CHECK || (col_ok && u + 4 * h < nrow);
                oc[e] = ok ? (uint32_t)(4 * h) * ldcb + (uint32_t)(col * ES) : kOob;
                op[e] = ok ? (uint32_t)(4 * h) * ldpb + (uint32_t)(col * ES) : kOob;
                if constexpr (KIND == GK_GELU_BWD) old[e] = ld_out<OT>(rp, op[e], (uint32_t)u * ldpb);
                if constexpr (KIND == GK_BETA) old[e] = ld_out<OT>(rc, oc[e], (uint32_t)u * ldcb);
            }
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const int u = 32 * i + 8 * (e >> 2) + (e & 3);
                float v = acc[i][j][e];
                if constexpr (KIND == GK_LINEAR) {
                    v += bj;
                } else if constexpr (KIND == GK_GELU) {
                    v += bj;
                    if (wp) st_out<OT>(v, rp, op[e], (uint32_t)u * ldpb);
                    v = gelu_tanh(v);
                } else if constexpr (KIND == GK_GELU_BWD) {
                    v *= gelu_grad_fine(old[e]);
                } else {
                    v = __builtin_fmaf(beta, old[e], v);
                }
                st_out<OT>(v, rc, oc[e], (uint32_t)u * ldcb);
            }
            __builtin_amdgcn_sched_barrier(0);  // one block's offsets at a time
        }
    }
}

}  // namespace vedic
