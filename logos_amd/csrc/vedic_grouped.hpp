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

#include <type_traits>

#include "vedic_common.hpp"
#include "vedic_epilogue.hpp"

namespace vedic {

constexpr int kMaxGroups = 1024;

// Workgroups of 256 threads that a launch can have: 2^32 threads and more are cut
// without an error.
constexpr int64_t kMaxBlocks = int64_t(1) << 24;

// Row tiles of `bm` that R rows in `groups` groups can have at most.
inline int64_t grouped_row_tiles_max(int R, int groups, int bm) { return R / bm + (groups < R ? groups : R); }

// Whether the general kernels (a workgroup per tile; 128 x 128 where there are many) and
// the binary16 few-row kernel (16 x 64, NT 16 x 32) can launch a product.
inline bool grouped_any_fits(int op, int groups, int R, int M, int N) {
    const int64_t rows = op == 2 ? (int64_t)groups * ((M + 127) / 128) : grouped_row_tiles_max(R, groups, 128);
    return rows * ((N + 127) / 128) < kMaxBlocks;
}
inline bool grouped_skinny_fits(int op, int groups, int R, int N) {
    const int bn = op == 1 ? 32 : 64;
    return grouped_row_tiles_max(R, groups, 16) * ((N + bn - 1) / bn) < kMaxBlocks;
}

enum GroupedKind : int {
    GK_LINEAR = 0,    // C = acc (+ b)
    GK_GELU = 1,      // C = gelu(acc (+ b))
    GK_GELU_P = 2,    // P = acc (+ b), C = gelu(P)
    GK_GELU_BWD = 3,  // C = acc * gelu'(P)
    GK_BETA = 4,      // C = acc + beta C
    GK_ADD = 5,       // C[out_rows[i]] += scales[group] acc[i]   (fp32 adapters)
};

// Whether a kind reads P or the old C; the others add a bias.
constexpr bool grouped_reads(int kind) { return kind == GK_GELU_BWD || kind == GK_BETA; }

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
    // Binary16 kernels: the columns that A (TN) and B (NN, TN) have, which a padded copy
    // has more of than M and N, and the steps of K that are A's padding alone (NN).
    int Mp, Np, kpad;
    float beta;
    const int* out_rows;  // GK_ADD: [R] rows of C, out_limit of them there
    int out_limit;
    const float* scales;  // GK_ADD: [groups], or null
    float* db;  // TN: [groups x N] column sums of B, or null
    float db_beta;
    // The contraction split over workgroups: slice s goes to C + s split_c (C then a
    // workspace of [ksplit][groups][M x N], NN and NT [ksplit][R x N]) and db + s groups
    // N.  1: no split.
    int ksplit;
    int64_t split_c;
    int tiles_m, tiles_n;
    int most;   // work items that a plan in order can have at most
    bool wide;  // grouped_wide_rows
};

// (no offsets: one group of all rows)
__device__ __forceinline__ int group_start(const GroupedArgs& a, int e) {
    if (a.offsets == nullptr) return e > 0 ? a.R : 0;
    return min(max(a.offsets[e], 0), a.R);
}
__device__ __forceinline__ int group_count(const GroupedArgs& a, int e) {
    return max(0, group_start(a, e + 1) - group_start(a, e));
}

// NN, NT: row tiles before each group, in LDS; pre[groups]: all of them.  TN: the
// groups in descending order of their rows (group_order).
struct GroupIndex {
    int pre[kMaxGroups + 1];
};

// Fills `ix` (ends with a barrier).  bm: rows per tile.  The first wave scans the
// groups 64 at a time; the offsets of the first 256 are loaded at once.
__device__ __forceinline__ void group_index(const GroupedArgs& a, GroupIndex& ix, int bm) {
    const int tid = threadIdx.x;
    if (tid < 64) {
        int carry = 0;
        for (int e0 = 0; e0 < a.groups; e0 += 256) {
            int n[4];
#pragma unroll
            for (int v = 0; v < 4; ++v) {
                const int e = e0 + 64 * v + tid;
                n[v] = e < a.groups ? (group_count(a, e) + bm - 1) / bm : 0;
            }
#pragma unroll
            for (int v = 0; v < 4; ++v) {
                const int e = e0 + 64 * v + tid;
                if (e0 + 64 * v >= a.groups) break;
                int t = n[v];
#pragma unroll
                for (int d = 1; d < 64; d <<= 1) {
                    const int u = __shfl_up(t, d);
                    if (tid >= d) t += u;
                }
                if (e < a.groups) ix.pre[e + 1] = carry + t;
                carry += __shfl(t, 63);
            }
        }
        if (tid == 0) ix.pre[0] = 0;
    }
    __syncthreads();
}

// Fills `ix` with the groups in descending order of their rows, the lower index
// first among equals (NT threads; ends with a barrier).  Past kOrderGroups, where
// counting a group's betters takes longer than the tiles' unequal lengths cost,
// their own order.
constexpr int kOrderGroups = 256;
template <int NT>
__device__ __forceinline__ void group_order(const GroupedArgs& a, GroupIndex& ix, int* count) {
    const int tid = threadIdx.x;
    if (a.groups > kOrderGroups) {
        for (int e = tid; e < a.groups; e += NT) ix.pre[e] = e;
        __syncthreads();
        return;
    }
    if (tid < a.groups) count[tid] = group_count(a, tid);
    __syncthreads();
    if (tid < a.groups) {
        const int n = count[tid];
        int rank = 0;
        for (int e = 0; e < a.groups; ++e) rank += count[e] > n || (count[e] == n && e < tid);
        ix.pre[rank] = tid;
    }
    __syncthreads();
}

// The group that holds row tile t (0 <= t < pre[groups]): the number of groups
// that end at or before it.  Uniform across the wave.
__device__ __forceinline__ int group_of(const GroupIndex& ix, int groups, int t, int lane) {
    int e = 0;
    for (int e0 = 0; e0 < groups; e0 += 64)
        e += __popcll(__ballot(e0 + lane < groups && ix.pre[min(e0 + lane, groups - 1) + 1] <= t));
    // (a bad plan's tiles can exceed what the grid was made for: never past the last group)
    return __builtin_amdgcn_readfirstlane(min(e, groups - 1));
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
typedef _Float16 half4_t __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2_t __attribute__((ext_vector_type(2)));
// Four values as loaded, and their values.
template <typename OT>
using raw4_t = std::conditional_t<sizeof(OT) == 2, u32x2_t, u32x4_t>;
template <typename OT>
__device__ __forceinline__ raw4_t<OT> ld_raw4(__amdgpu_buffer_rsrc_t rs, uint32_t voff, uint32_t soff) {
    if constexpr (sizeof(OT) == 2)
        return __builtin_bit_cast(u32x2_t, __builtin_amdgcn_raw_buffer_load_b64(rs, (int)voff, (int)soff, 0));
    else
        return __builtin_bit_cast(u32x4_t, __builtin_amdgcn_raw_buffer_load_b128(rs, (int)voff, (int)soff, 0));
}
template <typename OT>
__device__ __forceinline__ float4_t value4(const raw4_t<OT>& r) {
    if constexpr (sizeof(OT) == 2) return __builtin_convertvector(__builtin_bit_cast(half4_t, r), float4_t);
    else return __builtin_bit_cast(float4_t, r);
}
template <typename OT>
__device__ __forceinline__ void st_out4(float4_t v, __amdgpu_buffer_rsrc_t rs, uint32_t voff, uint32_t soff) {
    if constexpr (sizeof(OT) == 2) {
        __builtin_amdgcn_raw_buffer_store_b64(__builtin_bit_cast(u32x2_t, __builtin_convertvector(v, half4_t)), rs, (int)voff,
                                              (int)soff, 0);
    } else {
        __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4_t, v), rs, (int)voff, (int)soff, 0);
        asm volatile("s_nop 3" ::"v"(v));  // (store16_hold)
    }
}

// The value of lane l ^ X of the same four, X = 1 or 2.
template <int X>
__device__ __forceinline__ float quad_swap(float v) {
    constexpr int ctrl = X == 1 ? 0xB1 : 0x4E;  // quad_perm 1 0 3 2, 2 3 0 1
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), ctrl, 0xF, 0xF, true));
}

// Four rows of one column per lane -> one row's four columns: lane q of every four
// holds v[r] = (row r, column q) and gets (row q, columns 0 .. 3).
__device__ __forceinline__ float4_t quad_transpose(float v0, float v1, float v2, float v3, int lane) {
    const bool odd = lane & 1, up = lane & 2;
    const float s0 = quad_swap<1>(odd ? v0 : v1), s1 = quad_swap<1>(odd ? v2 : v3);
    // (row 0 or 1, columns 0 1 or 2 3) and (row 2 or 3, the same columns)
    const float a0 = odd ? s0 : v0, a1 = odd ? v1 : s0, b0 = odd ? s1 : v2, b1 = odd ? v3 : s1;
    const float t0 = quad_swap<2>(up ? a0 : b0), t1 = quad_swap<2>(up ? a1 : b1);
    return float4_t{up ? t0 : a0, up ? t1 : a1, up ? b0 : t0, up ? b1 : t1};
}

// Writes a (32 MI) x (32 NI) wave tile.  C and P point at the tile's first row
// (column 0); `nrow` rows and N columns exist past (that row, column 0); bias
// points at the bias of the wave's first column in LDS (zeros where there is none).
//
// Kinds that only write store as the MFMA leaves the values, a column per lane.
// Kinds that read P or the old C (VEC: their rows allow 16-byte accesses, 8-byte ones
// for binary16, and N is a multiple of 4) let four neighbouring lanes, which hold four
// rows of four columns, exchange them first: a lane then has four columns of one row
// and a 32 x 32 block takes 4 loads and stores instead of 16 (8192 x 2 rows of 1024 into
// 4096 binary16 columns times gelu' 275 -> 261 us; stores alone are not bound by their
// number, the exchange cost the GELU products 195 -> 206).
template <int KIND, typename OT, bool CHECK, bool VEC, int MI, int NI>
__device__ __forceinline__ void grouped_epilogue(void* C, int64_t ldc, void* P, int64_t ldp, const float* bias, float beta,
                                                 const float16_t (&acc)[MI][NI], int nrow, int N, int col0, int lane) {
    constexpr int ES = sizeof(OT);
    constexpr bool RD = grouped_reads(KIND);
    const int h = lane >> 5;
    const __amdgpu_buffer_rsrc_t rc = buffer_rsrc(C);
    const __amdgpu_buffer_rsrc_t rp = buffer_rsrc(P);
    const uint32_t ldcb = (uint32_t)(ldc * ES), ldpb = (uint32_t)(ldp * ES);
    if constexpr (!RD || !VEC) {
#pragma unroll
        for (int j = 0; j < NI; ++j) {
            const int col = col0 + 32 * j + (lane & 31);
            float bj = 0.0f;
            if constexpr (!RD) bj = bias[32 * j + (lane & 31)];
#pragma unroll
            for (int i = 0; i < MI; ++i) {
                auto off = [&](int e, uint32_t ldb) -> uint32_t {
                    const bool ok = !CHECK || (col < N && 32 * i + 8 * (e >> 2) + (e & 3) + 4 * h < nrow);
                    return ok ? (uint32_t)(4 * h) * ldb + (uint32_t)(col * ES) : kOob;
                };
                float old[16];
                if constexpr (RD) {
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                        const uint32_t u = 32 * i + 8 * (e >> 2) + (e & 3);
                        old[e] = KIND == GK_GELU_BWD ? ld_out<OT>(rp, off(e, ldpb), u * ldpb)
                                                     : ld_out<OT>(rc, off(e, ldcb), u * ldcb);
                    }
                }
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const uint32_t u = 32 * i + 8 * (e >> 2) + (e & 3);
                    float v = acc[i][j][e];
                    if constexpr (!RD) v += bj;
                    if constexpr (KIND == GK_GELU_P) st_out<OT>(v, rp, off(e, ldpb), u * ldpb);
                    if constexpr (KIND == GK_GELU || KIND == GK_GELU_P) {
                        v = gelu_tanh(v);
                    } else if constexpr (KIND == GK_GELU_BWD) {
                        v *= gelu_grad_fine(old[e]);
                    } else if constexpr (KIND == GK_BETA) {
                        v = __builtin_fmaf(beta, old[e], v);
                    }
                    st_out<OT>(v, rc, off(e, ldcb), u * ldcb);
                }
                __builtin_amdgcn_sched_barrier(0);  // one block's offsets at a time
            }
        }
    } else {
        const int q = lane & 3, c4 = lane & 28;  // this lane's row of four, first of its four columns
        const __amdgpu_buffer_rsrc_t rr = KIND == GK_GELU_BWD ? rp : rc;
        const uint32_t ldrb = KIND == GK_GELU_BWD ? ldpb : ldcb;
        // row 32 i + 8 g + 4 h + q of block (i, j)
        auto off = [&](int i, int j, int g, uint32_t ldb) -> uint32_t {
            const int col = col0 + 32 * j + c4;
            const bool ok = !CHECK || (col < N && 32 * i + 8 * g + 4 * h + q < nrow);
            return ok ? (uint32_t)(4 * h + q) * ldb + (uint32_t)(col * ES) : kOob;
        };
        raw4_t<OT> cur[4], nxt[4];
        auto fetch = [&](int bk, raw4_t<OT> (&d)[4]) {
            const int j = bk / MI, i = bk % MI;
#pragma unroll
            for (int g = 0; g < 4; ++g) d[g] = ld_raw4<OT>(rr, off(i, j, g, ldrb), (uint32_t)(32 * i + 8 * g) * ldrb);
        };
        fetch(0, cur);
#pragma unroll
        for (int bk = 0; bk < MI * NI; ++bk) {
            const int j = bk / MI, i = bk % MI;
            if (bk + 1 < MI * NI) fetch(bk + 1, nxt);
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                float4_t v = quad_transpose(acc[i][j][4 * g], acc[i][j][4 * g + 1], acc[i][j][4 * g + 2], acc[i][j][4 * g + 3],
                                            lane);
                const float4_t old = value4<OT>(cur[g]);
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    v[e] = KIND == GK_GELU_BWD ? v[e] * gelu_grad_fine(old[e]) : __builtin_fmaf(beta, old[e], v[e]);
                st_out4<OT>(v, rc, off(i, j, g, ldcb), (uint32_t)(32 * i + 8 * g) * ldcb);
            }
#pragma unroll
            for (int g = 0; g < 4; ++g) cur[g] = nxt[g];
            __builtin_amdgcn_sched_barrier(0);  // one block's offsets at a time
        }
    }
}

// GK_ADD: adds a (32 MI) x (32 NI) wave tile, times `scale`, to the rows of C that
// `rows` lists (nrow of them; a row outside 0 .. limit - 1 takes nothing).
template <int MI, int NI>
__device__ __forceinline__ void grouped_add(float* C, int64_t ldc, const int* rows, int limit, float scale,
                                            const float16_t (&acc)[MI][NI], int nrow, int N, int col0, int lane) {
#pragma unroll
    for (int i = 0; i < MI; ++i) {
        // (the rows, then all old values of 32 rows, before the first store: a store would
        // hold back every later load: 898 rows of rank 64 onto 2496 columns 32.9 us, so 19.0)
        int row[16];
        float old[16][NI];
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            const int u = 32 * i + 8 * (e >> 2) + 4 * (lane >> 5) + (e & 3);
            row[e] = u < nrow ? rows[u] : -1;
        }
#pragma unroll
        for (int e = 0; e < 16; ++e)
#pragma unroll
            for (int j = 0; j < NI; ++j) {
                const int col = col0 + 32 * j + (lane & 31);
                old[e][j] = (unsigned)row[e] < (unsigned)limit && col < N ? C[(int64_t)row[e] * ldc + col] : 0.0f;
            }
#pragma unroll
        for (int e = 0; e < 16; ++e)
#pragma unroll
            for (int j = 0; j < NI; ++j) {
                const int col = col0 + 32 * j + (lane & 31);
                if ((unsigned)row[e] < (unsigned)limit && col < N)
                    C[(int64_t)row[e] * ldc + col] = __builtin_fmaf(scale, acc[i][j][e], old[e][j]);
            }
    }
}

// Whether C and P allow the epilogue's wide accesses (strides in elements; every
// group's first row too, as `stride` has it).
inline bool grouped_wide_rows(const GroupedArgs& a, int es) {
    auto ok = [&](const void* p, int64_t ld) {
        return p == nullptr || (reinterpret_cast<uintptr_t>(p) % (4 * es) == 0 && ld % 4 == 0);
    };
    return a.N % 4 == 0 && ok(a.C, a.ldc) && ok(a.P, a.ldp) && a.stride_c % 4 == 0;
}

}  // namespace vedic
