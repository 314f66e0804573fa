// vedic_grouped_f16.hpp -- the grouped products on binary16 operands that 16-byte
// loads can take: the tiles, LDS layouts and stage pipeline of
// vedic_gemm_f16.hpp with every work item's operands taken from its group.
//
// Persistent tiles: at most one workgroup per CU (NN / NT tiles counted through
// the groups from the offsets, so the loop's end is known on the GPU only).  A
// group's tiles are consecutive and run down eight rows before moving right, and
// the renumbering of workgroups gives an XCD consecutive ones: its L2 sees one
// expert's weights at a time.
//
// Rows of A through a list go into the per-lane offsets that the direct loads use
// anyway (NN, NT) or are picked per stage (TN), so that the gathered copy of the
// activations is never written (TN of 16384 listed rows, 1024 x 4096 in eight groups:
// 165 us with a copy, 154 without).  The bias gradient of TN is summed from the stages
// in LDS (221 us with a pass of its own, 147).
//
// What bounds it: 16384 rows of 1024 into 4096 in eight even groups run at the rate of
// the ungrouped product (0.96 PFLOP/s; a 256 x 256 tile per CU and 64 steps 1.65 us);
// the bursts of stores at the end of each round (64 MiB per binary16 output) and the
// GELU's two transcendental operations per value come on top, not overlapped with the
// next tile's MFMAs (two 128 x 256 workgroups per CU to overlap them: 197 -> 254 us).
#pragma once

#include "vedic_gemm_f16.hpp"
#include "vedic_grouped.hpp"

namespace vedic {

// Side<true, ...> with rows from a list.  The list's entries of a tile are read a
// tile ahead (next), their latency under the current tile's contraction.
template <int R, int BK, int NW>
struct SideRows {
    using S = Side<true, R, BK, NW>;
    static constexpr int BYTES = S::BYTES, NLD = S::NLD;
    S s;
    int row[NLD];  // of the tile to come: row of A (of the tile without a list), -1: none
    __device__ __forceinline__ void next(int wave, int lane, int left, const int* list) {
#pragma unroll
        for (int i = 0; i < NLD; ++i) {
            int r, c;
            S::geom(wave, lane, i, r, c);
            row[i] = r >= left ? -1 : list != nullptr ? list[r] : r;
        }
    }
    __device__ __forceinline__ void init(int wave, int lane, int64_t ld, int limit) {
#pragma unroll
        for (int i = 0; i < NLD; ++i) {
            int r, c;
            S::geom(wave, lane, i, r, c);
            s.off[i] = (unsigned)row[i] < (unsigned)limit ? (uint32_t)((int64_t)row[i] * ld * 2 + c * 16) : kOob;
            s.kend[i] = 8 * c + 8;
        }
    }
    __device__ __forceinline__ void load(const _Float16* tile, char* lds, int wave, int lane, int krem) const {
        s.load(tile, lds, wave, lane, krem);
    }
};

// Side<false, ...> of A in TN with the contraction's rows from a list (LIST).  A
// wave's rows of a stage are neighbours in the list: they are read one stage ahead
// into scalar registers, and a lane picks its own of each access's RPI.
template <int R, int BK, int NW, bool LIST>
struct SideListed {
    using S = Side<false, R, BK, NW>;
    static constexpr int BYTES = S::BYTES, NLD = S::NLD, RPI = 64 / S::CPR;
    static_assert(RPI == 2 || RPI == 4, "rows of 256 or 128 columns");
    typedef const __attribute__((address_space(4))) int* list_t;  // (scalar loads)
    S s;
    int row[LIST ? NLD : 1][RPI];  // of the next stage
    list_t list;
    int last, at, limit;  // the list's last entry, this wave's first of the next stage, A's rows
    uint32_t pitch;       // bytes

    __device__ __forceinline__ void fetch() {
#pragma unroll
        for (int i = 0; i < NLD; ++i)
#pragma unroll
            for (int q = 0; q < RPI; ++q) row[i][q] = list[min(at + i * RPI + q, last)];
        at += BK;
    }
    __device__ __forceinline__ void init(int wave, int lane, int64_t ld, int m0, int M, const int* rows, int start, int R_,
                                         int a_rows) {
        s.init(wave, lane, LIST ? 0 : ld, m0, M);
        if constexpr (LIST) {
            list = (list_t)(uintptr_t)rows;
            at = start + wave * NLD * RPI;
            last = R_ - 1;
            limit = a_rows;
            pitch = (uint32_t)(ld * 2);
            fetch();
        }
    }
    // `tile`: A's first row (with a list) or the stage's, at column m0.
    __device__ __forceinline__ void load(const _Float16* tile, char* lds, int wave, int lane, int krem) {
        if constexpr (!LIST) {
            s.load(tile, lds, wave, lane, krem);
        } else {
            const __amdgpu_buffer_rsrc_t rs = buffer_rsrc(tile);
#pragma unroll
            for (int i = 0; i < NLD; ++i) {
                // (values, not places: a choice among places would put the array in memory)
                const int r0 = row[i][0], r1 = row[i][1], r2 = row[i][RPI - 2], r3 = row[i][RPI - 1];
                const int lo = (RPI == 4 ? lane & 16 : lane & 32) ? r1 : r0, hi = lane & 16 ? r3 : r2;
                const int r = RPI == 4 && (lane & 32) ? hi : lo;
                const bool ok = s.kend[i] <= krem && (unsigned)r < (unsigned)limit;
                // (s.off: the lane's columns, or kOob past M)
                __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (lds_void_t*)(lds + (wave * NLD + i) * 1024), 16,
                                                         ok && s.off[i] != kOob ? (uint32_t)r * pitch + s.off[i] : kOob, 0, 0, 0);
            }
            fetch();
        }
    }
};

// Column sums of B's stages, BN columns, BK rows, for the bias gradient: wave w adds
// rows w BK / NW ..., 4 columns a lane (64 / (BN / 4) rows at a time), in fp32.  The
// tiles of the first M rows do this beside their MFMAs: B is not read again.
template <int BN, int BK, int NW>
struct StageSums {
    static constexpr int LR = BN / 4, RPI = 64 / LR, NR = BK / NW / RPI;  // lanes a row, rows an access, accesses
    float4_t sum = {0.0f, 0.0f, 0.0f, 0.0f};
    __device__ __forceinline__ void add(const char* b, int wave, int lane) {
        const int slot = (lane % LR) >> 1;
#pragma unroll
        for (int i = 0; i < NR; ++i) {
            const int k = wave * (BK / NW) + i * RPI + lane / LR;
            const half4_t v = *reinterpret_cast<const half4_t*>(b + k * (2 * BN) + ((slot ^ swz_mc<BN>(k)) << 4) + 8 * (lane & 1));
            sum += __builtin_convertvector(v, float4_t);
        }
    }
    // db[0 .. BN) of the tile through `sh` (NW RPI BN floats), all threads.
    __device__ __forceinline__ void finish(float* sh, float* db, int n, float beta, int wave, int lane) const {
        *reinterpret_cast<float4_t*>(sh + (wave * RPI + lane / LR) * BN + 4 * (lane % LR)) = sum;
        __syncthreads();
        const int c = threadIdx.x;
        if (c < BN && c < n) {
            float t = sh[c];
            for (int q = 1; q < NW * RPI; ++q) t += sh[q * BN + c];
            db[c] = beta == 0.0f ? t : __builtin_fmaf(beta, db[c], t);
        }
        __syncthreads();
    }
};

// One work item: a tile of one group.
struct GroupedItem {
    int e, start, m0, n0, left, K, nk, slice, k0;  // k0: NN and NT, the slice's first step
};

// Work item w counts tiles of PM x PN; with SM x SN > 1 a tile is cut into that
// many parts of BM x BN and w counts the parts.
template <int OP, int BM, int BN, int BK, int SM, int SN, bool SPLIT>
__device__ __forceinline__ GroupedItem grouped_item(const GroupedArgs& a, const GroupIndex& ix, int w, int lane) {
    constexpr int PM = BM * SM, PN = BN * SN;
    GroupedItem it;
    const int part = w % (SM * SN);
    w /= SM * SN;
    if constexpr (OP == 2) {
        const int tiles = a.tiles_m * a.tiles_n;
        it.slice = __builtin_amdgcn_readfirstlane(w / (a.groups * tiles));
        w -= it.slice * a.groups * tiles;
        const int place = w / tiles, t = w - place * tiles;
        it.e = __builtin_amdgcn_readfirstlane(ix.pre[place]);
        it.m0 = t % a.tiles_m * PM;
        it.n0 = t / a.tiles_m * PN;
        const int count = group_count(a, it.e), len = ((count + a.ksplit - 1) / a.ksplit + BK - 1) / BK * BK;
        it.K = max(0, min(len, count - it.slice * len));
        it.left = a.M;
    } else {
        it.slice = it.k0 = 0;
        it.K = a.K;
        if constexpr (SPLIT) {
            if (a.ksplit > 1) {
                const int len = ((a.K + a.ksplit - 1) / a.ksplit + BK - 1) / BK * BK;
                const int each = __builtin_amdgcn_readfirstlane(ix.pre[a.groups]) * a.tiles_n;
                it.slice = __builtin_amdgcn_readfirstlane(w / each);
                w -= it.slice * each;
                it.k0 = min(a.K, it.slice * len);
                it.K = min(len, a.K - it.k0);
            }
        }
        it.e = group_of(ix, a.groups, w / a.tiles_n, lane);
        const int p0 = __builtin_amdgcn_readfirstlane(ix.pre[it.e]);
        const int mt = __builtin_amdgcn_readfirstlane(ix.pre[it.e + 1]) - p0;
        constexpr int GM = 8;
        const int q = w - p0 * a.tiles_n, g = q / (GM * a.tiles_n), first = g * GM;
        const int rows = min(GM, mt - first), in = q - g * GM * a.tiles_n;
        it.m0 = (first + in % rows) * PM;
        it.n0 = in / rows * PN;
        it.left = group_count(a, it.e);
    }
    it.m0 += part % SM * BM;
    it.n0 += part / SM * BN;
    // (uniform, said so that the loads' resources stay in scalar registers)
    it.e = __builtin_amdgcn_readfirstlane(it.e);
    it.start = __builtin_amdgcn_readfirstlane(group_start(a, it.e));
    if constexpr (OP == 2) {
        if (a.ksplit > 1) {
            // (an empty slice may start past the group's end: nothing is read there)
            const int count = group_count(a, it.e);
            it.start += min(count, it.slice * (((count + a.ksplit - 1) / a.ksplit + BK - 1) / BK * BK));
            it.start = __builtin_amdgcn_readfirstlane(it.start);
        }
    }
    it.m0 = __builtin_amdgcn_readfirstlane(it.m0);
    it.n0 = __builtin_amdgcn_readfirstlane(it.n0);
    it.left = __builtin_amdgcn_readfirstlane(it.left) - it.m0;
    it.K = __builtin_amdgcn_readfirstlane(it.K);
    it.nk = (it.K + BK - 1) / BK;
    return it;
}

// The loads of the next stage into (la) and (lb), and the operands moved on (past
// the range nothing is read: the stage has no steps left).
#define VEDIC_G_ISSUE(la, lb)                       \
    do {                                            \
        sa.load(Ab, (la), wave, lane, krem);        \
        sb.load(Bb, (lb), wave, lane, krem - kpad); \
        Ab += A_KC ? (int64_t)BK : astep;           \
        Bb += B_KC ? (int64_t)BK : BK * a.ldb;      \
        krem -= BK;                                 \
    } while (0)
// A pointer said to be uniform: its halves in scalar registers.
__device__ __forceinline__ const _Float16* uniform(const _Float16* p) {
    const uint64_t v = reinterpret_cast<uint64_t>(p);
    const uint32_t lo = __builtin_amdgcn_readfirstlane((int)(uint32_t)v), hi = __builtin_amdgcn_readfirstlane((int)(v >> 32));
    return reinterpret_cast<const _Float16*>((uint64_t)hi << 32 | lo);
}

// What work item `nx` reads besides its operands: the row list, the bias.
#define VEDIC_G_NEXT()                                                                                         \
    do {                                                                                                       \
        if constexpr (OP != 2) sa.next(wave, lane, nx.left, a.rows ? a.rows + nx.start + nx.m0 : nullptr);     \
        if constexpr (kBias)                                                                                   \
            bnext = a.bias != nullptr && (int)threadIdx.x < BN && nx.n0 + (int)threadIdx.x < a.N               \
                        ? a.bias[(int64_t)nx.e * a.N + nx.n0 + threadIdx.x]                                    \
                        : 0.0f;                                                                                \
    } while (0)
// The operands of work item `it` and the loads of its first stages.
#define VEDIC_G_START()                                                                                        \
    do {                                                                                                       \
        Ab = static_cast<const _Float16*>(a.A);                                                                \
        Bb = static_cast<const _Float16*>(a.B);                                                                \
        if constexpr (OP == 2) {                                                                               \
            Ab += (LIST ? 0 : (int64_t)it.start * a.lda) + it.m0;                                              \
            Bb += (int64_t)it.start * a.ldb + it.n0;                                                           \
            sa.init(wave, lane, a.lda, it.m0, a.Mp, a.rows, it.start, a.R, a.a_rows);                          \
        } else {                                                                                               \
            Bb += (int64_t)it.e * a.stride_b + (B_KC ? (int64_t)it.n0 * a.ldb : it.n0);                        \
            if (!a.rows) Ab += (int64_t)(it.start + it.m0) * a.lda;                                            \
            if constexpr (SPLIT) {                                                                             \
                Ab += it.k0;                                                                                   \
                Bb += B_KC ? (int64_t)it.k0 : it.k0 * a.ldb;                                                   \
                kpad = OP == 0 && it.k0 + it.K == a.K ? a.kpad : 0;                                            \
            }                                                                                                  \
            sa.init(wave, lane, a.lda, a.rows ? a.a_rows : BM);                                                \
        }                                                                                                      \
        sb.init(wave, lane, a.ldb, it.n0, B_KC ? a.N : a.Np);                                                  \
        if (kBias && (int)threadIdx.x < BN) sbias[par][threadIdx.x] = bnext;                                   \
        Ab = uniform(Ab);                                                                                      \
        Bb = uniform(Bb);                                                                                      \
        krem = it.K;                                                                                           \
        VEDIC_G_ISSUE(As[0], Bs[0]);                                                                           \
        if constexpr (ST > 2) VEDIC_G_ISSUE(As[1], Bs[1]);                                                     \
    } while (0)

// Work items w, w + step, ... below nwork (LOOP false: w alone) on tiles of BM x BN,
// or parts of that size (grouped_item).
template <int OP, int BM, int BN, int BK, int ST, int WGM, int WGN, int SM, int SN, bool LOOP, bool LIST, int KIND, typename OT>
__device__ __forceinline__ void grouped_tiles(const GroupedArgs& a, const GroupIndex& ix, char* t0, char* t1, char* t2,
                                              float* sb0, float* sb1, int first, int nwork, int step) {
    constexpr int NW = WGM * WGN, WM = BM / WGM, WN = BN / WGN, MI = WM / 32, NI = WN / 32;
    constexpr bool A_KC = OP != 2, B_KC = OP == 1;
    using SA = std::conditional_t<A_KC, SideRows<BM, BK, NW>, SideListed<BM, BK, NW, LIST>>;
    using SB = Side<B_KC, BN, BK, NW>;
    constexpr int L = SA::NLD + SB::NLD;
    static_assert(ST >= 2 && ST <= 3, "2 or 3 LDS stages");
    constexpr bool kInterleave = BM * BN >= 256 * 256;
    constexpr bool SPLIT = OP != 2 && ST == 3;  // (the small kernel's tiles)
    constexpr bool kBias = !grouped_reads(KIND);
    char* const As[3] = {t0, t1, t2};
    char* const Bs[3] = {t0 + SA::BYTES, t1 + SA::BYTES, t2 + SA::BYTES};
    float* const sbias[2] = {sb0, sb1};
    int par = 0;  // which of them holds the current tile's bias

    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int lane = threadIdx.x & 63;
    const int wm = wave / WGN, wn = wave % WGN;
    GroupedItem it = grouped_item<OP, BM, BN, BK, SM, SN, SPLIT>(a, ix, first, lane), nx = it;
    if (SM * SN > 1 && (it.left <= 0 || it.n0 >= a.N)) return;  // a part past the tile's edge
    SA sa;
    SB sb;
    const _Float16* Ab;
    const _Float16* Bb;
    float bnext = 0.0f;
    int krem;  // contraction steps not yet loaded
    int kpad = OP == 0 ? a.kpad : 0;
    const int64_t astep = LIST ? 0 : BK * a.lda;  // (TN)
    VEDIC_G_NEXT();
    VEDIC_G_START();
    int round = 0;
    while (true) {
        // (TN: the groups descend, so every other round runs backwards: a workgroup's
        // long tiles meet short ones)
        ++round;
        const int wn_ = OP == 2 && LOOP && (round & 1) ? first + round * step + (step - 1 - 2 * (first % step)) : first + round * step;
        const bool more = LOOP && wn_ < nwork;
        if (more) {
            nx = grouped_item<OP, BM, BN, BK, SM, SN, SPLIT>(a, ix, wn_, lane);
            VEDIC_G_NEXT();
        }
        float16_t acc[MI][NI];
#pragma unroll
        for (int i = 0; i < MI; ++i)
#pragma unroll
            for (int j = 0; j < NI; ++j) acc[i][j] = float16_t{};
        const int nk = it.nk;
        const bool sums = OP == 2 && a.db != nullptr && it.m0 == 0;
        StageSums<BN, BK, NW> ss;
        for (int k0 = 0; k0 < nk; k0 += ST) {
#pragma unroll
            for (int s = 0; s < ST; ++s) {
                const int kt = k0 + s;
                wait_vmcnt<(ST - 2) * L>();  // stage kt has landed
                stage_barrier();
                const int sl = (s + ST - 1) % ST;
                if constexpr (kInterleave) {
                    if (kt < nk) {
                        VEDIC_G_ISSUE(As[sl], Bs[sl]);
                        mfma_stage<A_KC, B_KC, BM, BN, BK, MI, NI, L, 1>(As[s], Bs[s], wm * WM, wn * WN, lane, acc);
                    } else {
                        VEDIC_G_ISSUE(As[sl], Bs[sl]);
                    }
                } else {
                    VEDIC_G_ISSUE(As[sl], Bs[sl]);
                    if (kt < nk) mfma_stage<A_KC, B_KC, BM, BN, BK, MI, NI>(As[s], Bs[s], wm * WM, wn * WN, lane, acc);
                }
                if constexpr (OP == 2) {
                    if (sums && kt < nk) ss.add(Bs[s], wave, lane);
                }
            }
        }
        if constexpr (OP == 2) {
            if (sums) {
                wait_vmcnt<0>();  // (zero loads past the range may still write the buffers)
                __syncthreads();
                ss.finish(reinterpret_cast<float*>(t0), a.db + ((int64_t)it.slice * a.groups + it.e) * a.N + it.n0, a.N - it.n0, a.db_beta, wave, lane);
            }
        }
        const GroupedItem done = it;
        const float* const bias = sbias[par] + (kBias ? wn * WN : 0);
        if (more) {
            wait_vmcnt<0>();  // (zero loads past the range may still write the buffers)
            __syncthreads();  // every wave is done reading them
            it = nx;
            par ^= 1;
            VEDIC_G_START();
        }
        const int row0 = done.m0 + wm * WM, col0 = done.n0 + wn * WN, left = done.left - wm * WM;
        const int64_t crow = OP == 2 ? row0 : done.start + row0;
        OT* const C = static_cast<OT*>(a.C) + (OP == 2 ? done.slice * a.split_c + (int64_t)done.e * a.stride_c : SPLIT ? done.slice * a.split_c : 0) +
                      crow * a.ldc;
        OT* const P = a.P != nullptr ? static_cast<OT*>(a.P) + crow * a.ldp : nullptr;
        if (nk == 0) __syncthreads();  // (no stage's barrier has shown the bias)
        if (grouped_reads(KIND) && !a.wide)
            grouped_epilogue<KIND, OT, true, false, MI, NI>(C, a.ldc, P, a.ldp, bias, a.beta, acc, left, a.N, col0, lane);
        else if (left >= WM && col0 + WN <= a.N)
            grouped_epilogue<KIND, OT, false, true, MI, NI>(C, a.ldc, P, a.ldp, bias, a.beta, acc, left, a.N, col0, lane);
        else
            grouped_epilogue<KIND, OT, true, true, MI, NI>(C, a.ldc, P, a.ldp, bias, a.beta, acc, left, a.N, col0, lane);
        if (!more) break;
    }
    wait_vmcnt<0>();  // the trailing zero loads still write LDS
}

// 256 x 256 tiles, eight waves of 128 x 64, while there is one for every workgroup;
// the tiles of the last, partial round in halves or quarters, if there is then still
// at most one for every workgroup: a round of whole tiles would leave the others idle
// for as long as a full one takes.  (16384 rows in eight groups of 655 to 3384: 1024
// into 4096 with GELU 207 -> 188 us, 4096 into 1024 187 -> 148.)
//
// TN: the groups in descending order of their rows, every other round backwards, so
// that a workgroup with a long tile gets a short one next (the same rows, 1024 x 4096
// per group 196 -> 151 us; even groups 140).
//
// LIST: TN through a row list (NN and NT read theirs at run time).
template <int OP, int KIND, typename OT, bool LIST>
__global__ void __launch_bounds__(512) grouped_f16_large_kernel(GroupedArgs a) {
    __shared__ __attribute__((aligned(1024))) char t0[65536];
    __shared__ __attribute__((aligned(1024))) char t1[65536];
    __shared__ GroupIndex ix;
    __shared__ __attribute__((aligned(16))) float sb0[256];
    __shared__ __attribute__((aligned(16))) float sb1[256];
    if constexpr (OP != 2) group_index(a, ix, 256);
    else group_order<512>(a, ix, reinterpret_cast<int*>(t0));
    const int nwork = OP == 2 ? a.groups * a.tiles_m * a.tiles_n * a.ksplit
                              : min((int64_t)__builtin_amdgcn_readfirstlane(ix.pre[a.groups]) * a.tiles_n, (int64_t)a.most);
    const int G = gridDim.x, b = blockIdx.x;
    const int w = (G & 7) == 0 ? (b & 7) * (G >> 3) + (b >> 3) : b;
    const int rest = nwork % G, whole = rest * 2 <= G ? nwork - rest : nwork;
    if (w < whole)
        grouped_tiles<OP, 256, 256, 64, 2, 2, 4, 1, 1, true, LIST, KIND, OT>(a, ix, t0, t1, nullptr, sb0, sb1, w, whole, G);
    if (whole == nwork) return;
    __syncthreads();
    if (rest * 4 <= G) {
        if (w < rest * 4)
            grouped_tiles<OP, 128, 128, 128, 2, 2, 4, 2, 2, false, LIST, KIND, OT>(a, ix, t0, t1, nullptr, sb0, sb1,
                                                                                   whole * 4 + w, 0, 0);
    } else if (w < rest * 2) {
        grouped_tiles<OP, 256, 128, 64, 2, 4, 2, 1, 2, false, LIST, KIND, OT>(a, ix, t0, t1, nullptr, sb0, sb1, whole * 2 + w,
                                                                              0, 0);
    }
}

// 128 x 128 tiles, four waves of 64 x 64, three stages (NN, NT).
template <int OP, int KIND, typename OT>
__global__ void __launch_bounds__(256) grouped_f16_small_kernel(GroupedArgs a) {
    __shared__ __attribute__((aligned(1024))) char t0[32768];
    __shared__ __attribute__((aligned(1024))) char t1[32768];
    __shared__ __attribute__((aligned(1024))) char t2[32768];
    __shared__ GroupIndex ix;
    __shared__ __attribute__((aligned(16))) float sb0[128];
    __shared__ __attribute__((aligned(16))) float sb1[128];
    group_index(a, ix, 128);
    const int nwork = min((int64_t)__builtin_amdgcn_readfirstlane(ix.pre[a.groups]) * a.tiles_n * a.ksplit, (int64_t)a.most);
    const int G = gridDim.x, b = blockIdx.x;
    const int w = (G & 7) == 0 ? (b & 7) * (G >> 3) + (b >> 3) : b;
    if (w < nwork)
        grouped_tiles<OP, 128, 128, 64, 3, 2, 2, 1, 1, true, false, KIND, OT>(a, ix, t0, t1, t2, sb0, sb1, w, nwork, G);
}

#undef VEDIC_G_START
#undef VEDIC_G_NEXT
#undef VEDIC_G_ISSUE

int device_cu_count();

// Workgroups for tiles of b x b: one per CU, or one per tile if there are fewer
// (parts: a tile may become that many).
inline hipError_t grouped_grid(int op, GroupedArgs& a, int b, int parts, int es_out, int& grid) {
    a.tiles_n = (a.N + b - 1) / b;
    a.tiles_m = op == 2 ? (a.M + b - 1) / b : 0;
    a.wide = grouped_wide_rows(a, es_out);
    if (a.ksplit < 1) a.ksplit = 1;
    const int64_t most = op == 2 ? (int64_t)a.groups * a.tiles_m * a.tiles_n * a.ksplit
                                 : (int64_t)(a.R / b + (a.groups < a.R ? a.groups : a.R)) * a.tiles_n;
    if (most * parts * (op == 2 ? 1 : a.ksplit) > 0x7FFFFFFF) return hipErrorInvalidValue;  // (the caller has refused such sizes)
    a.most = (int)(op == 2 ? most : most * a.ksplit);
    const int cus = device_cu_count();
    grid = (int64_t)a.most * parts < cus ? a.most * parts : cus;
    return hipSuccess;
}

// NN and NT run on 128 x 128 tiles where those are expected to fit one round (a group
// ends half way through a tile on average): us on the large kernel / the small one,
// 1024 into 4096 in 8 groups, 8 rows 22.6 / 16.6, 512 rows (256 tiles) 23.2 / 19.2, 1024
// rows 25.5 / 30.2, 4096 rows 52.4 / 64.7; 4096 rows of 512 into 512 in 16 groups (160
// tiles) 13.7 / 13.0; 4096 into 1024 in 8 groups, 2048 rows (160 tiles) 39.3 / 37.7, 4096
// rows (288) 66.8 / 72.8.  TN has few rows in no tile: 1024 x 4096 in 8 groups, 64 rows
// 29.6 / 38.4, 1024 rows 35.2 / 43.2; 16384 rows in 32 groups of 256 x 1024 24.5 / 23.4.
inline bool grouped_small_tiles(const GroupedArgs& a, int cus) {
    const int used = a.groups < a.R ? a.groups : a.R;
    return ((double)a.R / 128 + 0.5 * used) * ((a.N + 127) / 128) <= cus;
}

template <int OP, int KIND, typename OT, bool LIST = false>
static hipError_t launch_grouped_tiles(GroupedArgs a, hipStream_t s) {
    int grid = 0;
    if constexpr (OP == 2) {
        if constexpr (!LIST)
            if (a.rows) return launch_grouped_tiles<OP, KIND, OT, true>(a, s);
    } else {
        if (grouped_small_tiles(a, device_cu_count())) {
            const hipError_t e = grouped_grid(OP, a, 128, 1, sizeof(OT), grid);
            if (e != hipSuccess || grid == 0) return e;
            hipLaunchKernelGGL((grouped_f16_small_kernel<OP, KIND, OT>), dim3(grid), dim3(256), 0, s, a);
            return hipGetLastError();
        }
    }
    const hipError_t e = grouped_grid(OP, a, 256, 4, sizeof(OT), grid);
    if (e != hipSuccess || grid == 0) return e;
    hipLaunchKernelGGL((grouped_f16_large_kernel<OP, KIND, OT, LIST>), dim3(grid), dim3(512), 0, s, a);
    return hipGetLastError();
}

#define VEDIC_GROUPED_INSTANTIATE(OP, KIND, OT)                                    \
    template __global__ void grouped_f16_large_kernel<OP, KIND, OT, false>(GroupedArgs); \
    template __global__ void grouped_f16_small_kernel<OP, KIND, OT>(GroupedArgs)
#define VEDIC_GROUPED_INSTANTIATE_TN(KIND)                                            \
    template __global__ void grouped_f16_large_kernel<2, KIND, float, false>(GroupedArgs); \
    template __global__ void grouped_f16_large_kernel<2, KIND, float, true>(GroupedArgs)

}  // namespace vedic
