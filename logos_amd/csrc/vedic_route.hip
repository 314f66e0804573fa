// vedic_route.hip -- the router of an expert layer: the k largest of each
// token's E logits, their softmax weights, and the tokens sorted by expert; and
// the logits' gradient.
//
// Choice.  One wave per token, lane l holding logits EPL l .. EPL l + EPL - 1 as
// unsigned keys in the order of the values.  A pick is the largest key of the
// wave (six DPP steps), the lowest lane that has it and that lane's lowest place:
// the lowest expert among equals, without comparing indexes.  The weights are
// exp(x_j - x_max) over their sum, in fp32.
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

// Largest value of the wave, in every lane (v_max_u32 with DPP; identity 0).
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t dpp_max(uint32_t v) {
    const uint32_t o = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xF, true);
    return v > o ? v : o;
}
__device__ __forceinline__ uint32_t wave_max(uint32_t v) {
    v = dpp_max<0x111, 0xF>(v);  // row_shr 1, 2, 4, 8
    v = dpp_max<0x112, 0xF>(v);
    v = dpp_max<0x114, 0xF>(v);
    v = dpp_max<0x118, 0xF>(v);
    v = dpp_max<0x142, 0xA>(v);  // row_bcast 15, 31: the last lane has all
    v = dpp_max<0x143, 0xC>(v);
    return (uint32_t)__builtin_amdgcn_readlane((int)v, 63);
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

// One token by one wave: lane j < k gets the j-th choice (id -1 and weight 0 where
// fewer than k logits are above -infinity).
template <int EPL>
__device__ __forceinline__ void choose(const float* x, int E, int k, bool renorm, int lane, int& id, float& w) {
    uint32_t key[EPL];
#pragma unroll
    for (int i = 0; i < EPL; ++i) {
        const int e = lane * EPL + i;
        key[i] = e < E ? key_of(x[e]) : 0u;
    }
    uint32_t top = 0;  // this lane's largest
#pragma unroll
    for (int i = 0; i < EPL; ++i) top = top > key[i] ? top : key[i];
    uint32_t first = 0;
    float total = 0.0f, mine = 0.0f;
    id = -1;
    for (int j = 0; j < k; ++j) {
        const uint32_t m = wave_max(top);
        if (j == 0) {
            first = m;
            if (!renorm && m != 0) {
                // the softmax over all experts: summed before the keys are spent
                const float x0 = value_of(m);
#pragma unroll
                for (int i = 0; i < EPL; ++i)
                    if (key[i] != 0) total += expf(value_of(key[i]) - x0);
            }
        }
        if (m == 0) break;
        const int from = __ffsll((unsigned long long)__ballot(top == m)) - 1;
        int place = 0;
#pragma unroll
        for (int i = EPL - 1; i >= 0; --i) place = key[i] == m ? i : place;
        const int e = __builtin_amdgcn_readlane(place, from) + from * EPL;
        if (lane == j) {
            id = e;
            mine = value_of(m);
        }
        if (lane == from) {
            top = 0;
#pragma unroll
            for (int i = 0; i < EPL; ++i) {
                if (i == place) key[i] = 0;
                top = top > key[i] ? top : key[i];
            }
        }
    }
    const float ex = id >= 0 ? expf(mine - value_of(first)) : 0.0f;
    total = wave_sum(renorm ? ex : total);
    w = id >= 0 ? ex / total : 0.0f;
}

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
            rows[at] = bin < groups ? p / per_row : -1;
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
template <int EPL>
__device__ __forceinline__ void choose_tokens(const RouteArgs& a, int t0, int t1, int nwaves, int* cnt) {
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    for (int t = t0 + wave; t < t1; t += nwaves) {
        int id;
        float w;
        choose<EPL>(a.logits + (int64_t)t * a.ld, a.E, a.k, a.renorm, lane, id, w);
        if (lane < a.k) {
            a.ids[(int64_t)t * a.k + lane] = id;
            a.weights[(int64_t)t * a.k + lane] = w;
            if (cnt) atomicAdd(&cnt[bin_of(id, a.E)], 1);  // (an integer count: any order)
        }
    }
}

template <int EPL>
__global__ void __launch_bounds__(256) route_choose_kernel(RouteArgs a) {
    __shared__ int cnt[kMaxGroups + 1];
    for (int e = threadIdx.x; e <= a.E; e += 256) cnt[e] = 0;
    __syncthreads();
    const int t0 = blockIdx.x * a.chunk;
    choose_tokens<EPL>(a, t0, min(a.T, t0 + a.chunk), 4, cnt);
    __syncthreads();
    for (int e = threadIdx.x; e <= a.E; e += 256) a.counts[(int64_t)blockIdx.x * (a.E + 1) + e] = cnt[e];
}

// Few tokens: choice and placement by one workgroup.
template <int EPL>
__global__ void __launch_bounds__(kPlaceThreads) route_small_kernel(RouteArgs a) {
    __shared__ PlaceLds l;
    choose_tokens<EPL>(a, 0, a.T, kPlaceWaves, nullptr);
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
    for (int e = threadIdx.x; e <= groups; e += 256) counts[(int64_t)blockIdx.x * (groups + 1) + e] = cnt[e];
}

// Placement of chunk blockIdx.x; counts [gridDim.x][groups + 1].
__global__ void __launch_bounds__(kPlaceThreads) group_place_kernel(const int* ids, int n, int per_row, int groups, int bits,
                                                                     int chunk, const int* counts, int* offsets, int* rows,
                                                                     int* slots) {
    __shared__ PlaceLds l;
    const int tid = threadIdx.x, bins = groups + 1;
    for (int b = tid; b < bins; b += kPlaceThreads) l.base[b] = l.before[b] = 0;
    __syncthreads();
    const int nb = gridDim.x, me = blockIdx.x;
    const int64_t cells = (int64_t)nb * bins;
    for (int64_t i = tid; i < cells; i += kPlaceThreads) {
        const int c = counts[i], b = (int)(i % bins);
        if (c != 0) {
            atomicAdd(&l.base[b], c);
            if (i / bins < me) atomicAdd(&l.before[b], c);
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

// Pairs per workgroup of the placement: whole tokens, 1024 or the multiple of it
// that keeps the workgroups, whose counts each of them reads, to about 128.
int chunk_tokens(int64_t T, int k) {
    const int64_t pairs = T * k;
    const int64_t per = 1024 * ((pairs + 128 * 1024 - 1) / (128 * 1024));
    const int64_t t = per / k;
    return (int)(t < 1 ? 1 : t);
}

template <int EPL>
hipError_t launch_route(const RouteArgs& a, bool small, int blocks, hipStream_t s) {
    if (small) hipLaunchKernelGGL((route_small_kernel<EPL>), dim3(1), dim3(kPlaceThreads), 0, s, a);
    else hipLaunchKernelGGL((route_choose_kernel<EPL>), dim3(blocks), dim3(256), 0, s, a);
    return hipGetLastError();
}

}  // namespace

// Tokens that one workgroup takes alone.
constexpr int kRouteSmall = 64;

static bool route_small(int64_t T, int k) { return T <= kRouteSmall && T * k <= kPlaceThreads; }

size_t route_count_bytes(int64_t T, int E, int k) {
    if (route_small(T, k)) return 0;
    const int64_t c = chunk_tokens(T, k);
    return sizeof(int) * (size_t)((T + c - 1) / c) * (E + 1);
}

hipError_t launch_route_topk(RouteArgs a, hipStream_t s) {
    const bool small = route_small(a.T, a.k);
    a.bits = bits_for(a.E + 1);
    a.chunk = chunk_tokens(a.T, a.k);
    const int blocks = (a.T + a.chunk - 1) / a.chunk;
    hipError_t e = a.E <= 64    ? launch_route<1>(a, small, blocks, s)
                   : a.E <= 128 ? launch_route<2>(a, small, blocks, s)
                   : a.E <= 256 ? launch_route<4>(a, small, blocks, s)
                   : a.E <= 512 ? launch_route<8>(a, small, blocks, s)
                                : launch_route<16>(a, small, blocks, s);
    if (e != hipSuccess || small) return e;
    hipLaunchKernelGGL(group_place_kernel, dim3(blocks), dim3(kPlaceThreads), 0, s, a.ids, a.T * a.k, a.k, a.E, a.bits,
                       a.chunk * a.k, a.counts, a.offsets, a.rows, a.slots);
    return hipGetLastError();
}

size_t group_count_bytes(int64_t n, int groups) {
    if (n <= kPlaceThreads) return 0;
    const int64_t c = chunk_tokens(n, 1);
    return sizeof(int) * (size_t)((n + c - 1) / c) * (groups + 1);
}

hipError_t launch_group_rows(const int* ids, int n, int per_row, int groups, int* counts, int* offsets, int* rows, int* slots,
                             hipStream_t s) {
    const int bits = bits_for(groups + 1);
    if (n <= kPlaceThreads) {
        hipLaunchKernelGGL(group_small_kernel, dim3(1), dim3(kPlaceThreads), 0, s, ids, n, per_row, groups, bits, offsets,
                           rows, slots);
        return hipGetLastError();
    }
    const int chunk = chunk_tokens(n, 1), blocks = (n + chunk - 1) / chunk;
    hipLaunchKernelGGL(group_count_kernel, dim3(blocks), dim3(256), 0, s, ids, n, groups, chunk, counts);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL(group_place_kernel, dim3(blocks), dim3(kPlaceThreads), 0, s, ids, n, per_row, groups, bits, chunk,
                       counts, offsets, rows, slots);
    return hipGetLastError();
}

hipError_t launch_route_topk_bwd(const float* logits, int64_t ld, const int* ids, const float* weights, const float* dweights,
                                 int T, int E, int k, int renorm, float* out, int64_t ldo, hipStream_t s) {
    hipLaunchKernelGGL(route_bwd_kernel, dim3((T + 3) / 4), dim3(256), 0, s, logits, ld, ids, weights, dweights, T, E, k,
                       renorm, out, ldo);
    return hipGetLastError();
}

}  // namespace vedic
