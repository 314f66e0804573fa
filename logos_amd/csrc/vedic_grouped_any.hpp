// vedic_grouped_any.hpp -- the grouped products for binary32 operands and for
// binary16 ones that the 16-byte kernels cannot load, any alignment.
//
// Every value is split into bf16 parts as it goes to LDS (vedic_split.hpp), six
// v_mfma_f32_32x32x16_bf16 per 32 x 32 x 16 block, the arithmetic of the
// ungrouped fp32 product (vedic_gemm_f32s.hpp), whose LDS layout this shares.
// (A binary16 value has two parts; the third is zero.)  The matrix pipe and the split's
// VALU work bound it, at small sizes each stage's latency: 2006 rows in 7 groups, 1999 into
// 1001, take 77 us (104 TFLOP/s; the ungrouped library product of this card does 153).
// One 128 x 128 tile, or 64 x 64 where those would leave CUs idle, per workgroup; per stage of 16
// contraction steps the values of stage k + 2 are in registers on their way,
// those of stage k + 1 are split into one LDS buffer while stage k's fragments
// are read from the other.
#pragma once

#include "vedic_gemm_f32s.hpp"
#include "vedic_grouped.hpp"

namespace vedic {

template <typename T>
__device__ __forceinline__ float ld_value(__amdgpu_buffer_rsrc_t rs, uint32_t off, uint32_t soff) {
    return ld_out<T>(rs, off, soff);
}

// One operand's staging (SideSplit with a value type and a row list): R rows of
// the tile, NT threads.  Contraction contiguous (KC): fp32, eight steps of one row per
// thread by two 16-byte loads, which need no more than the values' own 4-byte
// alignment (whole fours of steps: the caller adds the last three or fewer); binary16 in pairs of steps,
// value by value, as it may lie at any 2 bytes.  Otherwise eight values down one
// column, coalesced across the lanes.
template <typename T, bool KC, int R, int NT>
struct SideAny {
    static constexpr int ES = sizeof(T);
    static constexpr bool PAIRS = KC && ES == 2;
    static constexpr int UNITS = PAIRS ? R * 8 : R * 2;
    static constexpr int U = UNITS / NT;
    static constexpr int PER = PAIRS ? 2 : 8;
    static_assert(UNITS % NT == 0, "units divide among the threads");
    uint32_t off[U];
    int k0[U];
    typedef float Values[U][PER];

    __device__ __forceinline__ static int row_of(int tid, int i) {
        const int u = i * NT + tid;
        return PAIRS ? u >> 3 : KC ? u >> 1 : u % R;
    }
    // list (KC): the tile's rows of the operand, `limit` of them there (a row
    // outside is read as zeros); null: consecutive rows.
    __device__ __forceinline__ void init(int tid, int64_t ld, int left, const int* list, int limit) {
#pragma unroll
        for (int i = 0; i < U; ++i) {
            const int u = i * NT + tid, row = row_of(tid, i);
            k0[i] = PAIRS ? 2 * (u & 7) : KC ? 8 * (u & 1) : 8 * __builtin_amdgcn_readfirstlane(u / R);
            bool ok = row < left;
            if constexpr (KC) {
                int64_t r = row;
                if (list != nullptr) {
                    const int x = ok ? list[row] : 0;
                    ok = ok && (unsigned)x < (unsigned)limit;
                    r = x;
                }
                off[i] = ok ? (uint32_t)(r * ld * ES + k0[i] * ES) : kOob;
            } else {
                off[i] = ok ? (uint32_t)(row * ES) : kOob;
            }
        }
    }
    // `steps` of the stage's 16 steps exist (maybe none); the others load as zeros.
    __device__ __forceinline__ void load(Values& v, const T* base, int64_t ld, int steps) const {
#pragma unroll
        for (int i = 0; i < U; ++i) {
            // (a stage past the range touches no memory: no records)
            const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(
                const_cast<T*>(KC || steps <= k0[i] ? base : base + (int64_t)k0[i] * ld), 0,
                steps > (KC ? 0 : k0[i]) ? 0x7FFFFFFF : 0, 0x00020000);
            if constexpr (KC && !PAIRS) {
#pragma unroll
                for (int q = 0; q < 8; q += 4) {
                    const uint32_t o = k0[i] + q < steps ? off[i] : kOob;
                    const float4_t w = __builtin_bit_cast(
                        float4_t, __builtin_amdgcn_raw_buffer_load_b128(rs, (int)(o == kOob ? kOob : o + q * ES), 0, 0));
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[i][q + e] = w[e];
                }
            } else if constexpr (KC) {
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const uint32_t o = k0[i] + e < steps ? off[i] : kOob;
                    v[i][e] = ld_value<T>(rs, o == kOob ? kOob : o + ES * e, 0);
                }
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    v[i][e] = ld_value<T>(rs, k0[i] + e < steps ? off[i] : kOob, (uint32_t)e * (uint32_t)ld * ES);
            }
        }
    }
    __device__ __forceinline__ void commit(const Values& v, char* lds, int tid) const {
#pragma unroll
        for (int i = 0; i < U; ++i) {
            const int row = row_of(tid, i);
            char* dst = lds + row * kSplitRowBytes + split_half(row, k0[i] >> 3);
            if constexpr (PAIRS) {
                const SplitPair s = split_pair(v[i][0] * kSplitScale, v[i][1] * kSplitScale);
#pragma unroll
                for (int p = 0; p < 3; ++p) *reinterpret_cast<uint32_t*>(dst + 32 * p + (k0[i] & 7) * 2) = s.p[p];
            } else {
                float w[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) w[e] = v[i][e] * kSplitScale;
                const SplitFrag f = split8(w);
#pragma unroll
                for (int p = 0; p < 3; ++p) *reinterpret_cast<bf16x8_t*>(dst + 32 * p) = f.p[p];
            }
        }
    }
};

// acc += a wave's block over steps kb .. K - 1 on v_mfma_f32_32x32x2_f32 from the
// operands themselves: for blocks whose split sums are not finite, for one or two
// steps, and for the steps behind the last four.  pa, pb: this lane's row and column
// (lane half h takes step kb + 2 q + h), ka, kb_ the distance of two steps' elements; a
// row that is not there has oka = false and counts as zeros.
template <typename T, typename TB, int MI, int NI>
__device__ __forceinline__ void any_block_slow(const T* const (&pa)[MI], const bool (&oka)[MI], int64_t ka,
                                               const TB* const (&pb)[NI], int64_t kb_, int kb, int K, int h,
                                               float16_t (&acc)[MI][NI]) {
#pragma unroll 1
    for (int k = kb + h; k < K + h; k += 2) {
        const bool in = k < K;
        const int64_t q = in ? k : K - 1;
        float x[MI], y[NI];
#pragma unroll
        for (int i = 0; i < MI; ++i) x[i] = in && oka[i] ? (float)pa[i][q * ka] : 0.0f;
#pragma unroll
        for (int j = 0; j < NI; ++j) y[j] = in ? (float)pb[j][q * kb_] : 0.0f;
#pragma unroll
        for (int i = 0; i < MI; ++i)
#pragma unroll
            for (int j = 0; j < NI; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x2f32(x[i], y[j], acc[i][j], 0, 0, 0);
    }
}

// One BM x BN tile per workgroup.  NN / NT: work item w is column tile w mod
// tiles_n of row tile w / tiles_n (row tiles counted through the groups).  TN: w
// is tile w mod (tiles_m tiles_n) of group w / (tiles_m tiles_n).
//
// WGK > 1: that many groups of WGM x WGN waves, each with LDS buffers of its own and
// a part of the contraction (whole stages); the others leave their sums in LDS for the
// first, which adds them in order and runs the epilogue.
// a.ksplit > 1: the grid's second dimension counts slices of the
// contraction (TN: of each group's), each into its own slab (vedic_grouped.hpp).
// T, TB, OT: the types of A, B and C.
template <int OP, typename T, typename TB, typename OT, int BM, int BN, int WGM, int WGN, int WGK, int KIND>
__global__ void __launch_bounds__(WGM* WGN * WGK * 64) grouped_any_kernel(GroupedArgs a) {
    constexpr int NT = WGM * WGN * 64, WM = BM / WGM, WN = BN / WGN, MI = WM / 32, NI = WN / 32;
    constexpr bool A_KC = OP != 2, B_KC = OP == 1;
    constexpr int BYTES = (BM + BN) * kSplitRowBytes;
    // VALU instructions placed after each MFMA: the split's 7 per element
    constexpr int VPM = (7 * (BM + BN) * kSplitK / NT + kSplitProducts * MI * NI - 1) / (kSplitProducts * MI * NI);
    __shared__ __attribute__((aligned(1024))) char all0[WGK * BYTES];
    __shared__ __attribute__((aligned(1024))) char all1[WGK * BYTES];
    __shared__ __attribute__((aligned(16))) float sbias[BN];
    const int tid = threadIdx.x % NT;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
    const int wk = WGK > 1 ? __builtin_amdgcn_readfirstlane(threadIdx.x / NT) : 0;
    char* const buf0 = all0 + wk * BYTES;
    char* const buf1 = all1 + wk * BYTES;
    const int wm = wave / WGN, wn = wave % WGN;

    int e, m0, n0, K, left, start, count;  // left: rows of C from m0 on
    if constexpr (OP == 2) {
        const int tiles = a.tiles_m * a.tiles_n;
        e = blockIdx.x / tiles;
        const int t = blockIdx.x - e * tiles;
        m0 = t % a.tiles_m * BM;
        n0 = t / a.tiles_m * BN;
        start = group_start(a, e);
        count = group_count(a, e);
        K = count;
        left = a.M - m0;
    } else {
        GroupIndex& ix = *reinterpret_cast<GroupIndex*>(all0);
        static_assert(BN <= NT && sizeof(GroupIndex) <= BYTES, "the index fits a stage buffer");
        group_index(a, ix, BM);
        const int t = blockIdx.x / a.tiles_n;
        if (t >= ix.pre[a.groups]) return;
        e = group_of(ix, a.groups, t, lane);
        start = group_start(a, e);
        count = group_count(a, e);
        m0 = (t - __builtin_amdgcn_readfirstlane(ix.pre[e])) * BM;
        n0 = (blockIdx.x - t * a.tiles_n) * BN;
        K = a.K;
        left = count - m0;
        __syncthreads();  // the index's LDS becomes a stage buffer
    }
    // (read after the barriers of the stages or the one before the epilogue)
    if (wk == 0 && tid < BN) sbias[tid] = a.bias != nullptr && n0 + tid < a.N ? a.bias[(int64_t)e * a.N + n0 + tid] : 0.0f;
    const T* A = static_cast<const T*>(a.A);
    const int* list = nullptr;
    if constexpr (OP == 2) {
        A += (int64_t)start * a.lda + m0;
    } else if (a.rows != nullptr) {
        list = a.rows + start + m0;
    } else {
        A += (int64_t)(start + m0) * a.lda;
    }
    const TB* B = static_cast<const TB*>(a.B);
    if constexpr (OP == 2) B += (int64_t)start * a.ldb + n0;
    else B += (int64_t)e * a.stride_b + (B_KC ? (int64_t)n0 * a.ldb : n0);
    const int64_t ka = A_KC ? 1 : a.lda, kb = B_KC ? 1 : a.ldb;

    using SA = SideAny<T, A_KC, BM, NT>;
    using SB = SideAny<TB, B_KC, BN, NT>;
    SA sa;
    SB sb;
    sa.init(tid, a.lda, left, list, a.a_rows);
    sb.init(tid, a.ldb, a.N - n0, nullptr, 0);
    typename SA::Values va;
    typename SB::Values vb;
    const bool few = K < kSplitMinK;
    // (fp32 rows are loaded four steps at a time: the last K mod 4 come at the end)
    const int Kq = OP != 2 && sizeof(T) == 4 ? K & ~3 : K;
    const int nk_all = few ? 0 : (Kq + kSplitK - 1) / kSplitK;
    const int slices = gridDim.y, slice = blockIdx.y;
    const int nk = (nk_all + WGK * slices - 1) / (WGK * slices);  // stages of a wave group
    const int kt0 = (slice * WGK + wk) * nk;                      // the first of this one's
    const int Ka = min(Kq, slice * WGK * nk * kSplitK), Kz = slice + 1 < slices ? min(Kq, Ka + WGK * nk * kSplitK) : K;
    auto load = [&](int kt) {
        const bool in = kt < nk && kt0 + kt < nk_all;
        const int64_t k = in ? (int64_t)(kt0 + kt) * kSplitK : 0;
        const int steps = in ? min(kSplitK, Kq - (kt0 + kt) * kSplitK) : 0;
        sa.load(va, A + k * ka, a.lda, steps);
        sb.load(vb, B + k * kb, a.ldb, steps);
    };
    auto commit = [&](char* buf) {
        sa.commit(va, buf, tid);
        sb.commit(vb, buf + BM * kSplitRowBytes, tid);
    };
    float16_t acc[MI][NI];
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int j = 0; j < NI; ++j) acc[i][j] = float16_t{};
    auto stage = [&](const char* cur, char* nxt, int kt) {
        SplitFrag fa[MI], fb[NI];
#pragma unroll
        for (int j = 0; j < NI; ++j) fb[j] = read_split(cur + BM * kSplitRowBytes, wn * WN + 32 * j, lane);
#pragma unroll
        for (int i = 0; i < MI; ++i) fa[i] = read_split(cur, wm * WM + 32 * i, lane);
        commit(nxt);
        load(kt + 2);
#pragma unroll
        for (int q = 0; q < kSplitProducts; ++q)
#pragma unroll
            for (int i = 0; i < MI; ++i)
#pragma unroll
                for (int j = 0; j < NI; ++j)
                    acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fa[i].p[kSplitA[q]], fb[j].p[kSplitB[q]],
                                                                        acc[i][j], 0, 0, 0);
        // the fragment reads, then a few VALU instructions of the split (and an LDS
        // write once there is one) after every MFMA
        __builtin_amdgcn_sched_group_barrier(0x100, 3 * (MI + NI), 0);
#pragma unroll
        for (int x = 0; x < kSplitProducts * MI * NI; ++x) {
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
            __builtin_amdgcn_sched_group_barrier(0x002, VPM, 0);
            __builtin_amdgcn_sched_group_barrier(0x200, 1, 0);
        }
        __builtin_amdgcn_sched_barrier(0);
        stage_barrier();  // (not a fence: stage kt + 2's loads stay in flight)
    };
    if (nk > 0) {
        load(0);
        commit(buf0);
        load(1);
        stage_barrier();
        for (int kt = 0; kt < nk; kt += 2) {  // (a stage past the last is zeros)
            stage(buf0, buf1, kt);
            stage(buf1, buf0, kt + 1);
        }
    }
    if constexpr (WGK > 1) {
        // partial (group, i) of a wave: 32 x WN sums
        constexpr int PIECE = WGM * WGN * 32 * WN * 4, PER = WGK * BYTES / PIECE;
        static_assert((WGK - 1) * MI <= 2 * PER, "the partial sums fit the buffers");
        auto piece = [&](int p) {
            return reinterpret_cast<float4_t*>((p < PER ? all0 : all1) + (p % PER) * PIECE + wave * (32 * WN * 4));
        };
        __syncthreads();
        if (wk > 0) {
#pragma unroll
            for (int i = 0; i < MI; ++i)
#pragma unroll
                for (int j = 0; j < NI; ++j)
#pragma unroll
                    for (int q = 0; q < 4; ++q)
                        piece((wk - 1) * MI + i)[(j * 4 + q) * 64 + lane] =
                            float4_t{acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]};
        }
        __syncthreads();
        if (wk > 0) return;
#pragma unroll
        for (int g = 0; g < WGK - 1; ++g)
#pragma unroll
            for (int i = 0; i < MI; ++i)
#pragma unroll
                for (int j = 0; j < NI; ++j)
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        const float4_t v = piece(g * MI + i)[(j * 4 + q) * 64 + lane];
#pragma unroll
                        for (int e2 = 0; e2 < 4; ++e2) acc[i][j][4 * q + e2] += v[e2];
                    }
    }
    float probe = 0.0f;
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int j = 0; j < NI; ++j) {
            acc[i][j] *= kSplitUnscale2;
            probe = nonfinite_probe(acc[i][j], probe);
        }
    const bool again = few || __any(probe != 0.0f);
    if (again || Kq < Kz) {
        const T* pa[MI];
        const TB* pb[NI];
        bool oka[MI];
#pragma unroll
        for (int i = 0; i < MI; ++i) {
            int r = min(wm * WM + 32 * i + (lane & 31), left - 1);
            oka[i] = true;
            if (left <= 0) r = 0, oka[i] = false;
            if (list != nullptr && oka[i]) {
                r = list[r];
                oka[i] = (unsigned)r < (unsigned)a.a_rows;
                if (!oka[i]) r = 0;
            }
            pa[i] = A_KC ? A + (int64_t)r * a.lda : A + r;
        }
#pragma unroll
        for (int j = 0; j < NI; ++j) {
            const int n = min(wn * WN + 32 * j + (lane & 31), a.N - n0 - 1);
            pb[j] = B_KC ? B + (int64_t)n * a.ldb : B + n;
        }
        if (again) {
#pragma unroll
            for (int i = 0; i < MI; ++i)
#pragma unroll
                for (int j = 0; j < NI; ++j) acc[i][j] = float16_t{};
        }
        any_block_slow<T, TB, MI, NI>(pa, oka, ka, pb, kb, again ? Ka : Kq, Kz, lane >> 5, acc);
    }
    if constexpr (KIND == GK_ADD) {
        grouped_add<MI, NI>(static_cast<float*>(a.C), a.ldc, a.out_rows + start + m0 + wm * WM, a.out_limit,
                            a.scales ? a.scales[e] : 1.0f, acc, left - wm * WM, a.N, n0 + wn * WN, lane);
        return;
    }
    const int row0 = m0 + wm * WM;
    const int64_t crow = OP == 2 ? row0 : start + row0;
    OT* C = static_cast<OT*>(a.C) + slice * a.split_c + (OP == 2 ? (int64_t)e * a.stride_c : 0) + crow * a.ldc;
    OT* P = a.P != nullptr ? static_cast<OT*>(a.P) + crow * a.ldp : nullptr;
    if constexpr (WGK == 1) __syncthreads();  // the bias (the sums' barriers have shown it otherwise)
    if (grouped_reads(KIND) && a.wide)
        grouped_epilogue<KIND, OT, true, true, MI, NI>(C, a.ldc, P, a.ldp, sbias + wn * WN, a.beta, acc, left - wm * WM, a.N,
                                                       n0 + wn * WN, lane);
    else
        grouped_epilogue<KIND, OT, true, false, MI, NI>(C, a.ldc, P, a.ldp, sbias + wn * WN, a.beta, acc, left - wm * WM, a.N,
                                                        n0 + wn * WN, lane);
}

struct CfgAMid {  // 128 x 128, four waves of 64 x 64
    static constexpr int BM = 128, BN = 128, WGM = 2, WGN = 2;
};
struct CfgASmall {  // 64 x 64, two waves of 32 x 64
    static constexpr int BM = 64, BN = 64, WGM = 2, WGN = 1;
};
constexpr int kAnyGroups = 3;  // wave groups of a workgroup where few tiles share the CUs

// Row tiles that R rows in `groups` groups about have.
inline double grouped_row_tiles(int R, int groups, int bm) {
    return (double)R / bm + 0.5 * (groups < R ? groups : R);
}

template <int OP, typename T, typename TB, typename OT, class Cfg, int WGK, int KIND>
static hipError_t launch_any(GroupedArgs a, hipStream_t s) {
    a.tiles_n = (a.N + Cfg::BN - 1) / Cfg::BN;
    a.tiles_m = OP == 2 ? (a.M + Cfg::BM - 1) / Cfg::BM : 0;
    a.wide = grouped_wide_rows(a, sizeof(OT));
    const int64_t work = OP == 2 ? (int64_t)a.groups * a.tiles_m * a.tiles_n
                                 : grouped_row_tiles_max(a.R, a.groups, Cfg::BM) * a.tiles_n;
    if (work * (Cfg::WGM * Cfg::WGN * WGK * 64) >= int64_t(1) << 32) return hipErrorInvalidValue;  // (grouped_any_fits)
    if (work == 0) return hipSuccess;
    hipLaunchKernelGGL((grouped_any_kernel<OP, T, TB, OT, Cfg::BM, Cfg::BN, Cfg::WGM, Cfg::WGN, WGK, KIND>),
                       dim3((unsigned)work, a.ksplit > 1 ? a.ksplit : 1), dim3(Cfg::WGM * Cfg::WGN * WGK * 64), 0, s, a);
    return hipGetLastError();
}

// 64 x 64 tiles where 128 x 128 ones would leave half the CUs without one (and slices of the
// contraction do not fill them).  Three wave
// groups where a CU gets no more than one 128 x 128 tile, and with the small ones, for
// contractions long enough to share (us, one group / three: 2006 rows in 7 groups of
// 2000 into 1000, 156 tiles, NN 103 / 79, NT 101 / 74; the same TN, 896 tiles of 286 steps,
// 63 / 73; 16 rows of 1024 into 4096 in 8 groups 55 / 45; 300 rows of 512 into 777 24 / 17).
template <int OP, typename T, typename TB, typename OT, int KIND>
static hipError_t launch_any_tiles(const GroupedArgs& a, hipStream_t s) {
    auto tiles = [&](int b) {
        return (OP == 2 ? (double)a.groups * ((a.M + b - 1) / b) : grouped_row_tiles(a.R, a.groups, b)) * ((a.N + b - 1) / b);
    };
    const int cus = device_cu_count();
    const bool split = (OP == 2 ? a.R / a.groups : a.K) >= 256;
    if (tiles(128) * 2 > cus || (a.ksplit > 1 && tiles(64) * 2 > cus)) {
        if (split && tiles(128) <= cus) return launch_any<OP, T, TB, OT, CfgAMid, kAnyGroups, KIND>(a, s);
        return launch_any<OP, T, TB, OT, CfgAMid, 1, KIND>(a, s);
    }
    if (split) return launch_any<OP, T, TB, OT, CfgASmall, kAnyGroups, KIND>(a, s);
    return launch_any<OP, T, TB, OT, CfgASmall, 1, KIND>(a, s);
}

template <int OP, int KIND>
static hipError_t launch_any_kind(const GroupedArgs& a, bool f16, bool f16out, hipStream_t s) {
    if constexpr (OP != 2)
        if (f16out) return launch_any_tiles<OP, _Float16, _Float16, _Float16, KIND>(a, s);
    return f16 ? launch_any_tiles<OP, _Float16, _Float16, float, KIND>(a, s) : launch_any_tiles<OP, float, float, float, KIND>(a, s);
}

#define VEDIC_ANY_KERNELS(OP, T, TB, OT, KIND)                                                               \
    template __global__ void grouped_any_kernel<OP, T, TB, OT, 128, 128, 2, 2, 1, KIND>(GroupedArgs);          \
    template __global__ void grouped_any_kernel<OP, T, TB, OT, 128, 128, 2, 2, kAnyGroups, KIND>(GroupedArgs); \
    template __global__ void grouped_any_kernel<OP, T, TB, OT, 64, 64, 2, 1, 1, KIND>(GroupedArgs);            \
    template __global__ void grouped_any_kernel<OP, T, TB, OT, 64, 64, 2, 1, kAnyGroups, KIND>(GroupedArgs)

}  // namespace vedic
