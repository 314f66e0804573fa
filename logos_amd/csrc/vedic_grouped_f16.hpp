// vedic_grouped_f16.hpp -- the grouped products on binary16 operands that 16-byte
// loads can take: the tiles, LDS layouts and stage pipeline of
// vedic_gemm_f16.hpp with every work item's operands taken from its group.
//
// Persistent tiles: at most one workgroup per CU (NN / NT tiles counted through
// the groups from the offsets, so the loop's end is known on the GPU only).  A
// group's tiles are consecutive and run down GROUP_M rows before moving right, and
// the renumbering of workgroups gives an XCD consecutive ones: its L2 sees one
// expert's weights at a time.
//
// Rows of A through a list: the list is read as a tile starts, into the per-lane
// offsets that the direct loads use anyway, so the gathered copy of the
// activations is never written.
#pragma once

#include "vedic_gemm_f16.hpp"
#include "vedic_grouped.hpp"

namespace vedic {

// Side<true, ...> with rows from a list (null: consecutive rows).
template <int R, int BK, int NW>
struct SideRows {
    using S = Side<true, R, BK, NW>;
    static constexpr int BYTES = S::BYTES, NLD = S::NLD;
    S s;
    __device__ __forceinline__ void init(int wave, int lane, int64_t ld, int left, const int* list, int limit) {
#pragma unroll
        for (int i = 0; i < NLD; ++i) {
            int row, c;
            S::geom(wave, lane, i, row, c);
            bool ok = row < left;
            int64_t r = row;
            if (list != nullptr) {
                const int x = ok ? list[row] : 0;
                ok = ok && (unsigned)x < (unsigned)limit;
                r = x;
            }
            s.off[i] = ok ? (uint32_t)(r * ld * 2 + c * 16) : kOob;
            s.kend[i] = 8 * c + 8;
        }
    }
    __device__ __forceinline__ void load(const _Float16* tile, char* lds, int wave, int lane, int krem) const {
        s.load(tile, lds, wave, lane, krem);
    }
};

// One work item: a tile of one group.
struct GroupedItem {
    int e, start, m0, n0, left, K, nk;
};

template <int OP, int BM, int BN, int BK>
__device__ __forceinline__ GroupedItem grouped_item(const GroupedArgs& a, const GroupIndex& ix, int w, int lane) {
    GroupedItem it;
    if constexpr (OP == 2) {
        const int tiles = a.tiles_m * a.tiles_n;
        it.e = w / tiles;
        const int t = w - it.e * tiles;
        it.m0 = t % a.tiles_m * BM;
        it.n0 = t / a.tiles_m * BN;
        it.start = __builtin_amdgcn_readfirstlane(ix.off[it.e]);
        it.K = max(0, __builtin_amdgcn_readfirstlane(ix.off[it.e + 1]) - it.start);
        it.left = a.M - it.m0;
    } else {
        it.e = group_of(ix, a.groups, w / a.tiles_n, lane);
        it.start = __builtin_amdgcn_readfirstlane(ix.off[it.e]);
        const int p0 = __builtin_amdgcn_readfirstlane(ix.pre[it.e]);
        const int mt = __builtin_amdgcn_readfirstlane(ix.pre[it.e + 1]) - p0;
        const int count = __builtin_amdgcn_readfirstlane(ix.off[it.e + 1]) - it.start;
        constexpr int GM = 8;
        const int q = w - p0 * a.tiles_n, g = q / (GM * a.tiles_n), first = g * GM;
        const int rows = min(GM, mt - first), in = q - g * GM * a.tiles_n;
        it.m0 = (first + in % rows) * BM;
        it.n0 = in / rows * BN;
        it.left = count - it.m0;
        it.K = a.K;
    }
    it.nk = (it.K + BK - 1) / BK;
    return it;
}

#define VEDIC_G_ISSUE(kt, la, lb)                                                                              \
    do {                                                                                                       \
        const int k_ = (kt) * BK;                                                                              \
        const int64_t kk_ = k_ < it.K ? k_ : 0;                                                                \
        sa.load(A_KC ? Ab + kk_ : Ab + kk_ * a.lda, (la), wave, lane, it.K - k_);                              \
        sb.load(B_KC ? Bb + kk_ : Bb + kk_ * a.ldb, (lb), wave, lane, it.K - k_);                              \
    } while (0)
// The operands of work item `it` and the loads of its first stages.
#define VEDIC_G_START()                                                                                        \
    do {                                                                                                       \
        Ab = static_cast<const _Float16*>(a.A);                                                                \
        Bb = static_cast<const _Float16*>(a.B);                                                                \
        if constexpr (OP == 2) {                                                                               \
            Ab += (int64_t)it.start * a.lda + it.m0;                                                           \
            Bb += (int64_t)it.start * a.ldb + it.n0;                                                           \
            sa.init(wave, lane, a.lda, it.m0, a.M);                                                            \
        } else {                                                                                               \
            Bb += (int64_t)it.e * a.stride_b + (B_KC ? (int64_t)it.n0 * a.ldb : it.n0);                        \
            const int* list_ = a.rows ? a.rows + it.start + it.m0 : nullptr;                                   \
            if (!list_) Ab += (int64_t)(it.start + it.m0) * a.lda;                                             \
            sa.init(wave, lane, a.lda, it.left, list_, a.a_rows);                                              \
        }                                                                                                      \
        sb.init(wave, lane, a.ldb, it.n0, a.N);                                                                \
        VEDIC_G_ISSUE(0, As[0], Bs[0]);                                                                        \
        if constexpr (ST > 2) VEDIC_G_ISSUE(1, As[1], Bs[1]);                                                  \
    } while (0)

template <int OP, int BM, int BN, int BK, int ST, int WGM, int WGN, int KIND, typename OT>
__global__ void __launch_bounds__(WGM* WGN * 64) grouped_f16_kernel(GroupedArgs a) {
    constexpr int NW = WGM * WGN, WM = BM / WGM, WN = BN / WGN, MI = WM / 32, NI = WN / 32;
    constexpr bool A_KC = OP != 2, B_KC = OP == 1;
    using SA = std::conditional_t<A_KC, SideRows<BM, BK, NW>, Side<false, BM, BK, NW>>;
    using SB = Side<B_KC, BN, BK, NW>;
    constexpr int L = SA::NLD + SB::NLD;
    static_assert(ST >= 2 && ST <= 3, "2 or 3 LDS stages");
    constexpr bool kInterleave = BM * BN >= 256 * 256;
    constexpr int SBYTES = SA::BYTES + SB::BYTES;
    __shared__ __attribute__((aligned(1024))) char t0[SBYTES];
    __shared__ __attribute__((aligned(1024))) char t1[SBYTES];
    __shared__ __attribute__((aligned(1024))) char t2[ST > 2 ? SBYTES : 16];
    __shared__ GroupIndex ix;
    char* const As[3] = {t0, t1, t2};
    char* const Bs[3] = {t0 + SA::BYTES, t1 + SA::BYTES, t2 + SA::BYTES};

    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int lane = threadIdx.x & 63;
    const int wm = wave / WGN, wn = wave % WGN;
    group_index<NW * 64>(a, ix, BM);
    const int nwork = OP == 2 ? a.groups * a.tiles_m * a.tiles_n
                              : __builtin_amdgcn_readfirstlane(ix.pre[a.groups]) * a.tiles_n;
    const int G = gridDim.x, b = blockIdx.x;
    int w = (G & 7) == 0 ? (b & 7) * (G >> 3) + (b >> 3) : b;
    if (w >= nwork) return;
    GroupedItem it = grouped_item<OP, BM, BN, BK>(a, ix, w, lane);
    SA sa;
    SB sb;
    const _Float16* Ab;
    const _Float16* Bb;
    VEDIC_G_START();
    while (true) {
        float16_t acc[MI][NI];
#pragma unroll
        for (int i = 0; i < MI; ++i)
#pragma unroll
            for (int j = 0; j < NI; ++j) acc[i][j] = float16_t{};
        const int nk = it.nk;
        for (int k0 = 0; k0 < nk; k0 += ST) {
#pragma unroll
            for (int s = 0; s < ST; ++s) {
                const int kt = k0 + s;
                wait_vmcnt<(ST - 2) * L>();  // stage kt has landed
                stage_barrier();
                const int sl = (s + ST - 1) % ST;
                if constexpr (kInterleave) {
                    if (kt < nk) {
                        VEDIC_G_ISSUE(kt + ST - 1, As[sl], Bs[sl]);
                        mfma_stage<A_KC, B_KC, BM, BN, BK, MI, NI, L, 1>(As[s], Bs[s], wm * WM, wn * WN, lane, acc);
                    } else {
                        VEDIC_G_ISSUE(kt + ST - 1, As[sl], Bs[sl]);
                    }
                } else {
                    VEDIC_G_ISSUE(kt + ST - 1, As[sl], Bs[sl]);
                    if (kt < nk) mfma_stage<A_KC, B_KC, BM, BN, BK, MI, NI>(As[s], Bs[s], wm * WM, wn * WN, lane, acc);
                }
            }
        }
        const GroupedItem done = it;
        w += G;
        const bool more = w < nwork;
        if (more) {
            wait_vmcnt<0>();  // (zero loads past the range may still write the buffers)
            __syncthreads();  // every wave is done reading them
            it = grouped_item<OP, BM, BN, BK>(a, ix, w, lane);
            VEDIC_G_START();
        }
        const int row0 = done.m0 + wm * WM, col0 = done.n0 + wn * WN, left = done.left - wm * WM;
        const int64_t crow = OP == 2 ? row0 : done.start + row0;
        OT* const C = static_cast<OT*>(a.C) + (OP == 2 ? (int64_t)done.e * a.stride_c : 0) + crow * a.ldc;
        OT* const P = a.P != nullptr ? static_cast<OT*>(a.P) + crow * a.ldp : nullptr;
        const float* const bias = a.bias != nullptr ? a.bias + (int64_t)done.e * a.N : nullptr;
        if (left >= WM && col0 + WN <= a.N)
            grouped_epilogue<KIND, OT, false, MI, NI>(C, a.ldc, P, a.ldp, bias, a.beta, acc, left, a.N, col0, lane);
        else
            grouped_epilogue<KIND, OT, true, MI, NI>(C, a.ldc, P, a.ldp, bias, a.beta, acc, left, a.N, col0, lane);
        if (!more) break;
    }
    wait_vmcnt<0>();  // the trailing zero loads still write LDS
}

#undef VEDIC_G_START
#undef VEDIC_G_ISSUE

struct CfgGLarge {  // 256 x 256, eight waves of 128 x 64
    static constexpr int BM = 256, BN = 256, BK = 64, ST = 2, WGM = 2, WGN = 4;
};
struct CfgGSmall {  // 128 x 128, four waves of 64 x 64
    static constexpr int BM = 128, BN = 128, BK = 64, ST = 3, WGM = 2, WGN = 2;
};

int device_cu_count();

template <int OP, class Cfg, int KIND, typename OT>
static hipError_t launch_grouped(GroupedArgs a, hipStream_t s) {
    a.tiles_n = (a.N + Cfg::BN - 1) / Cfg::BN;
    a.tiles_m = OP == 2 ? (a.M + Cfg::BM - 1) / Cfg::BM : 0;
    const int64_t most = OP == 2 ? (int64_t)a.groups * a.tiles_m * a.tiles_n
                                 : (int64_t)(a.R / Cfg::BM + (a.groups < a.R ? a.groups : a.R)) * a.tiles_n;
    if (most > 0x7FFFFFFF) return hipErrorInvalidValue;  // (the caller has refused such sizes)
    if (most == 0) return hipSuccess;
    const int cus = device_cu_count();
    const int grid = most < cus ? (int)most : cus;
    hipLaunchKernelGGL((grouped_f16_kernel<OP, Cfg::BM, Cfg::BN, Cfg::BK, Cfg::ST, Cfg::WGM, Cfg::WGN, KIND, OT>), dim3(grid),
                       dim3(Cfg::WGM * Cfg::WGN * 64), 0, s, a);
    return hipGetLastError();
}

// Rounds of tiles times the work of one, over the tiles' relative rate.
inline bool grouped_large_tiles(int op, const GroupedArgs& a, int cus) {
    const int used = a.groups < a.R ? a.groups : a.R;
    auto cost = [&](int b, double rate) {
        const double rows = op == 2 ? (double)a.groups * ((a.M + b - 1) / b) : (double)a.R / b + 0.5 * used;
        const double tiles = rows * ((a.N + b - 1) / b);
        const double rounds = tiles / cus < 1.0 ? 1.0 : tiles / cus;
        return rounds * b * b / rate;
    };
    return cost(256, 1.0) < cost(128, 0.75);
}

template <int OP, int KIND, typename OT>
static hipError_t launch_grouped_tiles(const GroupedArgs& a, hipStream_t s) {
    if (grouped_large_tiles(OP, a, device_cu_count())) return launch_grouped<OP, CfgGLarge, KIND, OT>(a, s);
    return launch_grouped<OP, CfgGSmall, KIND, OT>(a, s);
}

#define VEDIC_GROUPED_KERNEL(OP, Cfg, KIND, OT) \
    template __global__ void grouped_f16_kernel<OP, Cfg::BM, Cfg::BN, Cfg::BK, Cfg::ST, Cfg::WGM, Cfg::WGN, KIND, OT>(GroupedArgs)
#define VEDIC_GROUPED_INSTANTIATE(OP, KIND, OT)     \
    VEDIC_GROUPED_KERNEL(OP, CfgGLarge, KIND, OT);  \
    VEDIC_GROUPED_KERNEL(OP, CfgGSmall, KIND, OT)

}  // namespace vedic
