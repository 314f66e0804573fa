// vedic_route.hip -- the router of an expert layer: the k largest of each
// token's E logits, their softmax weights, and the tokens sorted by expert; and
// the logits' gradient.
//
// Choice.  16 lanes per token, four tokens a wave (64 lanes, one token, past 256
// experts or 16 choices), lane l of a token holding logits EPL l .. EPL l + EPL - 1
// as unsigned keys in the order of the values.  A pick is the largest key of the
// token's lanes (one v_max_u32 with DPP per halving), the lowest lane that has it and
// that lane's lowest place: the lowest expert among equals, without comparing
// indexes.  The weights are exp(x_j - x_max) over their sum, in fp32.  Instructions
// bound it: 8192 tokens of 128 experts, 8 chosen, take 6.3 us (66 with a wave per token)
// and their placement 7.9; the 5.2 MB they read and write would take 1.1.
//
// Sorting is a stable counting sort by expert in two launches: the choice leaves
// each workgroup's counts per expert, and the placement adds the counts of the
// workgroups before its own.  A pair's rank among its wave's pairs of one expert
// is a popcount of the lanes that match it in every bit of the index, so no
// atomic decides an order.
#include "vedic_common.hpp"
#include "vedic_route.hpp"

namespace vedic {

namespace {

// v_max_u32 with DPP (identity 0).
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t dpp_max(uint32_t v) {
    const uint32_t o = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xF, true);
    return v > o ? v : o;
}
// Largest value of the lane's 16 lanes, in every lane of them: rotations by 8, 4, 2, 1.
__device__ __forceinline__ uint32_t row_max(uint32_t v) {
    v = dpp_max<0x128, 0xF>(v);
    v = dpp_max<0x124, 0xF>(v);
    v = dpp_max<0x122, 0xF>(v);
    return dpp_max<0x121, 0xF>(v);
}
// Largest value of the wave, in every lane.
__device__ __forceinline__ uint32_t wave_max(uint32_t v) {
    v = row_max(v);
    v = dpp_max<0x142, 0xA>(v);  // row_bcast 15, 31: the last lane has all
    v = dpp_max<0x143, 0xC>(v);
    return (uint32_t)__builtin_amdgcn_readlane((int)v, 63);
}
template <int LPT>
__device__ __forceinline__ uint32_t token_max(uint32_t v) {
    if constexpr (LPT == 16) return row_max(v);
    else return wave_max(v);
}
template <int LPT>
__device__ __forceinline__ float token_sum(float v) {
#pragma unroll
    for (int d = LPT / 2; d > 0; d >>= 1) v += __shfl_xor(v, d);
    return v;
}
__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) v += __shfl_xor(v, d);
    return v;
}

// Keys in the order of the values: 0 for -infinity (never chosen), NaN above
// everything, -0 and +0 alike.
__device__ __forceinline__ uint32_t key_of(float x) {
    if (x != x) return 0xFFFFFFFFu;
    if (x == -__builtin_inff()) return 0u;
    const uint32_t u = __builtin_bit_cast(uint32_t, x + 0.0f);
    return u >> 31 ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t key) {  // of a chosen one
    return __builtin_bit_cast(float, key >> 31 ? key == 0xFFFFFFFFu ? key : key & 0x7FFFFFFFu : ~key);
}

// One token by LPT lanes, `l` of them this one: lane j < k gets the j-th choice (id -1
// and weight 0 where fewer than k logits are above -infinity).  All lanes of a wave
// take k picks; x may be null for lanes without a token.
template <int LPT, int EPL>
__device__ __forceinline__ void choose(const float* x, int E, int k, bool renorm, bool wide, int l, int& id, float& w) {
    uint32_t key[EPL];
    if (EPL >= 4 && wide) {
#pragma unroll
        for (int i = 0; i < EPL; i += 4) {
            const int e = l * EPL + i;
            const bool in = x != nullptr && e < E;
            float4_t v = {0.0f, 0.0f, 0.0f, 0.0f};
            if (in) v = *reinterpret_cast<const float4_t*>(x + e);
#pragma unroll
            for (int q = 0; q < 4 && q < EPL; ++q) key[i + q] = in ? key_of(v[q]) : 0u;
        }
    } else {
#pragma unroll
        for (int i = 0; i < EPL; ++i) {
            const int e = l * EPL + i;
            key[i] = x != nullptr && e < E ? key_of(x[e]) : 0u;
        }
    }
    uint32_t top = 0;  // this lane's largest
#pragma unroll
    for (int i = 0; i < EPL; ++i) top = top > key[i] ? top : key[i];
    uint32_t first = 0, mine = 0;
    float total = 0.0f;
    id = -1;
    for (int j = 0; j < k; ++j) {
        const uint32_t m = token_max<LPT>(top);
        if (j == 0) {
            first = m;
            if (!renorm) {
                // the softmax over all experts: summed before the keys are spent
                const float x0 = value_of(m);
#pragma unroll
                for (int i = 0; i < EPL; ++i)
                    if (key[i] != 0) total += expf(value_of(key[i]) - x0);
            }
        }
        // the lowest of the token's lanes that holds it (none left: m is 0, and every
        // lane's top is)
        const unsigned long long hold = __ballot(top == m);
        const int shift = LPT == 16 ? (threadIdx.x & 48) : 0;
        const unsigned long long mask = LPT == 16 ? (hold >> shift) & 0xFFFFull : hold;
        const int from = __ffsll(mask) - 1;
        const bool winner = l == from && m != 0;
        int place = 0;
#pragma unroll
        for (int i = EPL - 1; i >= 0; --i) place = key[i] == m ? i : place;
        // (expert + 1 of the winner in every lane of the token; 0: none)
        const uint32_t e = token_max<LPT>(winner ? (uint32_t)(l * EPL + place + 1) : 0u);
        if (l == j) {
            id = (int)e - 1;
            mine = m;
        }
        if (EPL == 1) {
            top = winner ? 0u : top;
        } else {
            uint32_t t = 0;
#pragma unroll
            for (int i = 0; i < EPL; ++i) {
                key[i] = winner && i == place ? 0u : key[i];
                t = t > key[i] ? t : key[i];
            }
            top = t;
        }
    }
    const float ex = id >= 0 ? expf(value_of(mine) - value_of(first)) : 0.0f;
    total = token_sum<LPT>(renorm ? ex : total);
    w = id >= 0 ? ex / total : 0.0f;
}

// Distance of two workgroups' counts: groups + 1 of them, whole 16-byte accesses.
__host__ __device__ inline int count_pitch(int groups) { return (groups + 4) / 4 * 4; }

constexpr int kChooseThreads = 512;
constexpr int kPlaceThreads = 1024, kPlaceWaves = kPlaceThreads / 64;

// Where pairs go.  base[bin]: the next free position of each bin (bin `groups`:
// the pairs that belong to none).
struct PlaceLds {
    int base[kMaxGroups + 1];
    int before[kMaxGroups + 1];  // counts of earlier workgroups, then of this one's waves
    int wave[kPlaceWaves][kMaxGroups + 1];
    int carry[kPlaceWaves];
};

__device__ __forceinline__ int bin_of(int id, int groups) { return (unsigned)id < (unsigned)groups ? id : groups; }

// This wave's counts of one round of pairs into l.wave[wave] (zero before), and
// the rank of this lane's pair among the wave's pairs of its bin.
__device__ __forceinline__ int wave_rank(PlaceLds& l, int wave, int lane, int bin, bool there, int bits) {
    unsigned long long same = __ballot(there);
    for (int b = 0; b < bits; ++b) {
        const unsigned long long set = __ballot((bin >> b) & 1);
        same &= (bin >> b) & 1 ? set : ~set;
    }
    const unsigned long long below = same & ((1ull << lane) - 1);
    if (there && below == 0) l.wave[wave][bin] = __popcll(same);
    return __popcll(below);
}

// Exclusive scan of l.base[0 .. n) in place by the whole workgroup.
__device__ __forceinline__ void scan_base(PlaceLds& l, int n) {
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
    // (n <= 1025: two entries a thread at most)
    const int i0 = 2 * tid, v0 = i0 < n ? l.base[i0] : 0, v1 = i0 + 1 < n ? l.base[i0 + 1] : 0;
    int s = v0 + v1;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int u = __shfl_up(s, d);
        if (lane >= d) s += u;
    }
    if (lane == 63) l.carry[wave] = s;
    __syncthreads();
    int c = 0;
    for (int q = 0; q < wave; ++q) c += l.carry[q];
    const int ex = c + s - v0 - v1;
    if (i0 < n) l.base[i0] = ex;
    if (i0 + 1 < n) l.base[i0 + 1] = ex + v0;
    __syncthreads();
}

// Positions of the pairs [p0, p1) of `ids`, rounds of 1024.  Only the first
// round's counts are known where `single` (its base is made of them).
template <bool SINGLE>
__device__ __forceinline__ void place(PlaceLds& l, const int* ids, int p0, int p1, int per_row, int groups, int bits,
                                      int* offsets, int* rows, int* slots) {
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, bins = groups + 1;
    for (int q = p0; q < p1 || (SINGLE && q == p0); q += kPlaceThreads) {
        for (int i = tid; i < kPlaceWaves * bins; i += kPlaceThreads) l.wave[i / bins][i % bins] = 0;
        __syncthreads();
        const int p = q + tid;
        const bool there = p < p1;
        const int id = there ? ids[p] : -1, bin = bin_of(id, groups);
        int at = wave_rank(l, wave, lane, bin, there, bits);
        __syncthreads();
        if constexpr (SINGLE) {
            for (int b = tid; b < bins; b += kPlaceThreads) {
                int n = 0;
                for (int v = 0; v < kPlaceWaves; ++v) n += l.wave[v][b];
                l.base[b] = n;
            }
            __syncthreads();
            scan_base(l, bins);
            for (int b = tid; b < bins; b += kPlaceThreads) offsets[b] = l.base[b];
        }
        if (there) {
            for (int v = 0; v < wave; ++v) at += l.wave[v][bin];
            at += l.base[bin];
            rows[at] = p / per_row;
            if (slots) slots[p] = bin < groups ? at : -1;
        }
        if (q + kPlaceThreads < p1) {
            __syncthreads();
            for (int b = tid; b < bins; b += kPlaceThreads) {
                int n = 0;
                for (int v = 0; v < kPlaceWaves; ++v) n += l.wave[v][b];
                l.base[b] += n;
            }
            __syncthreads();
        }
    }
}

// Tokens [t0, t1) of this workgroup: choices, weights, and the counts per expert
// in cnt (LDS).
template <int LPT, int EPL>
__device__ __forceinline__ void choose_tokens(const RouteArgs& a, int t0, int t1, int nwaves, int* cnt) {
    constexpr int TPW = 64 / LPT;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l = threadIdx.x & (LPT - 1);
    for (int tw = t0 + wave * TPW; tw < t1; tw += nwaves * TPW) {
        const int t = tw + (threadIdx.x & 63) / LPT;
        int id;
        float w;
        choose<LPT, EPL>(t < t1 ? a.logits + (int64_t)t * a.ld : nullptr, a.E, a.k, a.renorm, a.wide, l, id, w);
        if (t < t1 && l < a.k) {
            a.ids[(int64_t)t * a.k + l] = id;
            a.weights[(int64_t)t * a.k + l] = w;
            if (cnt) atomicAdd(&cnt[bin_of(id, a.E)], 1);  // (an integer count: any order)
        }
    }
}

template <int LPT, int EPL>
__global__ void __launch_bounds__(kChooseThreads) route_choose_kernel(RouteArgs a) {
    __shared__ int cnt[kMaxGroups + 1];
    for (int e = threadIdx.x; e <= a.E; e += kChooseThreads) cnt[e] = 0;
    __syncthreads();
    const int t0 = blockIdx.x * a.tokens;
    choose_tokens<LPT, EPL>(a, t0, min(a.T, t0 + a.tokens), kChooseThreads / 64, cnt);
    __syncthreads();
    for (int e = threadIdx.x; e <= a.E; e += kChooseThreads) a.counts[(int64_t)blockIdx.x * count_pitch(a.E) + e] = cnt[e];
}

// Few tokens: choice and placement by one workgroup.
template <int LPT, int EPL>
__global__ void __launch_bounds__(kPlaceThreads) route_small_kernel(RouteArgs a) {
    __shared__ PlaceLds l;
    choose_tokens<LPT, EPL>(a, 0, a.T, kPlaceWaves, nullptr);
    __threadfence_block();
    __syncthreads();
    place<true>(l, a.ids, 0, a.T * a.k, a.k, a.E, a.bits, a.offsets, a.rows, a.slots);
}

// Counts per group of each chunk of ids.
__global__ void __launch_bounds__(256) group_count_kernel(const int* ids, int n, int groups, int chunk, int* counts) {
    __shared__ int cnt[kMaxGroups + 1];
    for (int e = threadIdx.x; e <= groups; e += 256) cnt[e] = 0;
    __syncthreads();
    const int64_t p0 = (int64_t)blockIdx.x * chunk;
    const int64_t p1 = min((int64_t)n, p0 + chunk);
    for (int64_t p = p0 + threadIdx.x; p < p1; p += 256) atomicAdd(&cnt[bin_of(ids[p], groups)], 1);
    __syncthreads();
    for (int e = threadIdx.x; e <= groups; e += 256) counts[(int64_t)blockIdx.x * count_pitch(groups) + e] = cnt[e];
}

// Placement of chunk blockIdx.x; counts [nrow][count_pitch], `per` rows a chunk.
// Thread t sums four bins of every (1024 / quads)-th row of counts, in registers; the
// rest is added in LDS (integers: any order).
__global__ void __launch_bounds__(kPlaceThreads) group_place_kernel(const int* ids, int n, int per_row, int groups, int bits,
                                                                     int chunk, const int* counts, int nrow, int per,
                                                                     int* offsets, int* rows, int* slots) {
    __shared__ PlaceLds l;
    const int tid = threadIdx.x, bins = groups + 1, me = blockIdx.x;
    typedef int int4_t __attribute__((ext_vector_type(4)));
    const int quads = count_pitch(groups) / 4, lanes = kPlaceThreads / quads, q = tid % quads, r0 = tid / quads;
    int4_t all = {0, 0, 0, 0}, mine = {0, 0, 0, 0};
    if (r0 < lanes) {
#pragma unroll 8
        for (int r = r0; r < nrow; r += lanes) {
            const int4_t v = reinterpret_cast<const int4_t*>(counts)[(int64_t)r * quads + q];
            all += v;
            if (r < me * per) mine += v;
        }
    }
    for (int b = tid; b < bins; b += kPlaceThreads) l.base[b] = l.before[b] = 0;
    __syncthreads();
    if (r0 < lanes) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (4 * q + e < bins) {
                if (all[e]) atomicAdd(&l.base[4 * q + e], all[e]);
                if (mine[e]) atomicAdd(&l.before[4 * q + e], mine[e]);
            }
    }
    __syncthreads();
    scan_base(l, bins);
    if (me == 0)
        for (int b = tid; b < bins; b += kPlaceThreads) offsets[b] = l.base[b];
    for (int b = tid; b < bins; b += kPlaceThreads) l.base[b] += l.before[b];
    __syncthreads();
    const int64_t p0 = (int64_t)me * chunk;
    place<false>(l, ids, (int)p0, (int)min((int64_t)n, p0 + chunk), per_row, groups, bits, offsets, rows, slots);
}

__global__ void __launch_bounds__(kPlaceThreads) group_small_kernel(const int* ids, int n, int per_row, int groups, int bits,
                                                                     int* offsets, int* rows, int* slots) {
    __shared__ PlaceLds l;
    place<true>(l, ids, 0, n, per_row, groups, bits, offsets, rows, slots);
}

// dlogits of one token by one wave.
__global__ void __launch_bounds__(256) route_bwd_kernel(const float* logits, int64_t ld, const int* ids, const float* weights,
                                                         const float* dweights, int T, int E, int k, int renorm, float* out,
                                                         int64_t ldo) {
    const int t = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    if (t >= T) return;
    int id = -1;
    float w = 0.0f, dw = 0.0f;
    if (lane < k) {
        id = ids[(int64_t)t * k + lane];
        if (id >= 0) {  // (a place without an expert has no weight to differentiate)
            w = weights[(int64_t)t * k + lane];
            dw = dweights[(int64_t)t * k + lane];
        }
    }
    const float inner = wave_sum(w * dw);
    const float* x = logits + (int64_t)t * ld;
    float* o = out + (int64_t)t * ldo;
    float x0 = 0.0f, total = 1.0f;
    if (!renorm) {
        uint32_t m = 0;
        for (int e = lane; e < E; e += 64) {
            const uint32_t q = key_of(x[e]);
            m = m > q ? m : q;
        }
        m = wave_max(m);
        x0 = value_of(m);
        float s = 0.0f;
        if (m != 0)
            for (int e = lane; e < E; e += 64) s += expf(x[e] - x0);
        total = m != 0 ? wave_sum(s) : 0.0f;
    }
    for (int e0 = 0; e0 < E; e0 += 64) {
        const int e = e0 + lane;
        float g = 0.0f, p = 0.0f;
        bool chosen = false;
        for (int j = 0; j < k; ++j) {
            const bool hit = __builtin_amdgcn_readlane(id, j) == e;
            const float wj = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, w), j));
            const float dj = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, dw), j));
            if (hit) {
                g = dj;
                p = wj;
                chosen = true;
            }
        }
        if (e < E) {
            if (renorm) o[e] = chosen ? p * (g - inner) : 0.0f;
            else o[e] = total == 0.0f ? 0.0f : expf(x[e] - x0) / total * (g - inner);
        }
    }
}

int bits_for(int bins) {
    int b = 0;
    while ((1 << b) < bins) ++b;
    return b;
}

// Entries per workgroup of the placement: 1024, or the multiple of it that keeps the
// workgroups, which read each others' counts, to about 128.
int64_t place_chunk(int64_t n) { return 1024 * ((n + 128 * 1024 - 1) / (128 * 1024)); }

// Tokens per workgroup of the choice: 32 a pass (8 with a wave per token), at most
// 512 workgroups, and whole rows of counts per chunk of the placement.
struct RoutePlan {
    int tokens, per;  // tokens a workgroup, workgroups a chunk
    int64_t blocks, chunks;
    bool wide;  // a wave per token
};
RoutePlan route_plan(int64_t T, int E, int k) {
    RoutePlan p;
    p.wide = E > 256 || k > 16;
    const int pass = kChooseThreads / (p.wide ? 64 : 16);
    const int64_t t = T > 512 ? (T + 511) / 512 : 1;
    p.tokens = (int)((t + pass - 1) / pass * pass);
    const int64_t want = place_chunk(T * k) / k;  // tokens a chunk
    p.per = (int)(want > p.tokens ? want / p.tokens : 1);
    p.blocks = (T + p.tokens - 1) / p.tokens;
    p.chunks = (p.blocks + p.per - 1) / p.per;
    return p;
}

template <int LPT, int EPL>
hipError_t launch_route(const RouteArgs& a, bool small, int64_t blocks, hipStream_t s) {
    if (small) hipLaunchKernelGGL((route_small_kernel<LPT, EPL>), dim3(1), dim3(kPlaceThreads), 0, s, a);
    else hipLaunchKernelGGL((route_choose_kernel<LPT, EPL>), dim3((unsigned)blocks), dim3(kChooseThreads), 0, s, a);
    return hipGetLastError();
}

}  // namespace

// Tokens that one workgroup takes alone.
constexpr int kRouteSmall = 64;

static bool route_small(int64_t T, int k) { return T <= kRouteSmall && T * k <= kPlaceThreads; }

size_t route_count_bytes(int64_t T, int E, int k) {
    if (route_small(T, k)) return 0;
    return sizeof(int) * (size_t)route_plan(T, E, k).blocks * count_pitch(E);
}

hipError_t launch_route_topk(RouteArgs a, hipStream_t s) {
    const bool small = route_small(a.T, a.k);
    const RoutePlan p = route_plan(a.T, a.E, a.k);
    a.bits = bits_for(a.E + 1);
    a.wide = a.E % 4 == 0 && a.ld % 4 == 0 && (reinterpret_cast<uintptr_t>(a.logits) & 15) == 0;
    a.tokens = p.tokens;
    hipError_t e;
    if (p.wide)
        e = a.E <= 64    ? launch_route<64, 1>(a, small, p.blocks, s)
            : a.E <= 256 ? launch_route<64, 4>(a, small, p.blocks, s)
                         : launch_route<64, 16>(a, small, p.blocks, s);
    else
        e = a.E <= 16    ? launch_route<16, 1>(a, small, p.blocks, s)
            : a.E <= 32  ? launch_route<16, 2>(a, small, p.blocks, s)
            : a.E <= 64  ? launch_route<16, 4>(a, small, p.blocks, s)
            : a.E <= 128 ? launch_route<16, 8>(a, small, p.blocks, s)
                         : launch_route<16, 16>(a, small, p.blocks, s);
    if (e != hipSuccess || small) return e;
    hipLaunchKernelGGL(group_place_kernel, dim3((unsigned)p.chunks), dim3(kPlaceThreads), 0, s, a.ids, a.T * a.k, a.k, a.E,
                       a.bits, p.tokens * p.per * a.k, a.counts, (int)p.blocks, p.per, a.offsets, a.rows, a.slots);
    return hipGetLastError();
}

size_t group_count_bytes(int64_t n, int groups) {
    if (n <= kPlaceThreads) return 0;
    const int64_t c = place_chunk(n);
    return sizeof(int) * (size_t)((n + c - 1) / c) * count_pitch(groups);
}

hipError_t launch_group_rows(const int* ids, int n, int per_row, int groups, int* counts, int* offsets, int* rows, int* slots,
                             hipStream_t s) {
    const int bits = bits_for(groups + 1);
    if (n <= kPlaceThreads) {
        hipLaunchKernelGGL(group_small_kernel, dim3(1), dim3(kPlaceThreads), 0, s, ids, n, per_row, groups, bits, offsets,
                           rows, slots);
        return hipGetLastError();
    }
    const int64_t chunk = place_chunk(n), blocks = (n + chunk - 1) / chunk;
    hipLaunchKernelGGL(group_count_kernel, dim3((unsigned)blocks), dim3(256), 0, s, ids, n, groups, (int)chunk, counts);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL(group_place_kernel, dim3((unsigned)blocks), dim3(kPlaceThreads), 0, s, ids, n, per_row, groups, bits,
                       (int)chunk, counts, (int)blocks, 1, offsets, rows, slots);
    return hipGetLastError();
}

hipError_t launch_route_topk_bwd(const float* logits, int64_t ld, const int* ids, const float* weights, const float* dweights,
                                 int T, int E, int k, int renorm, float* out, int64_t ldo, hipStream_t s) {
    // (in launches of fewer than 2^32 threads)
    constexpr int kTokens = (1 << 26) - 4;
    for (int64_t t = 0; t < T; t += kTokens) {
        const int n = (int)(T - t < kTokens ? T - t : kTokens);
        hipLaunchKernelGGL(route_bwd_kernel, dim3((n + 3) / 4), dim3(256), 0, s, logits + t * ld, ld, ids + t * k,
                           weights + t * k, dweights + t * k, n, E, k, renorm, out + t * ldo, ldo);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

}  // namespace vedic
