// vedic_paged_many.hpp -- attention of many new rows a sequence (a prompt, or the next piece
// of one) over its paged cache.
//
//   S^T = K Q^T (32 tokens x 32 rows per v_mfma_f32_32x32x16_f16), weights 2^(x - m + 14) with a
//   running maximum and sum in fp32, O^T += V^T P^T.
//
// A workgroup has a tile of 128 rows (four waves of 32) and a range of keys (vedic_paged.hpp).
// Blocks of 64 keys (32 with heads past 128) go through two buffers of LDS, one barrier a block: while a block is
// multiplied, the next one's rows are on their way into registers (from the pages, 16 bytes a
// thread and load; four bits are expanded on their way to LDS) and the places of the one
// after that are looked up.  K's rows lie 2 DP + 16 bytes apart (ds_read_b128 of eight rows meets
// every bank once), V's 2 DP + 32 (the same for the transposing ds_read_b64_tr_b16).  The scores'
// layout, a row of Q per lane, is what the second product takes: the weights stay in
// registers.  A wave leaves out blocks none of its rows sees, and looks at masks only where
// some key of a block is hidden from one of them.
#pragma once

#include "vedic_paged.hpp"

namespace vedic {

namespace {

typedef short many_short4_t __attribute__((ext_vector_type(4)));
typedef _Float16 many_half4_t __attribute__((ext_vector_type(4)));

// Keys of a block: with heads past 128 the next block's rows would take 64 registers more.
constexpr int many_keys(int dp) { return dp <= 128 ? 64 : 32; }
constexpr int kManyUnit = 256;   // parts are whole multiples of it

// The pieces of a block (64 rows of K, then of V) that a thread carries from the pages to LDS.
template <int DP, bool I4>
struct BlockShare {
    static constexpr int KEYS = many_keys(DP), KP = 2 * DP + 16, VP = 2 * DP + 32;
    static constexpr int PER = I4 ? DP / 32 : DP / 8;  // pieces of a row
    static constexpr int ALL = 2 * KEYS * PER, N = (ALL + 255) / 256;
    u32x4_t v[N];
    uint32_t sm[I4 ? N : 1];
    const char* from[N];  // the piece in the row at offset 0 (heads narrower than DP: the last one again past the end)
    const char* pair[I4 ? N : 1];
    __device__ __forceinline__ static bool of_v(int x) { return index(x) >= KEYS * PER; }
    __device__ __forceinline__ static int row(int x) { return index(x) % (KEYS * PER) / PER; }
    __device__ __forceinline__ static int piece(int x) { return index(x) % PER; }
    __device__ __forceinline__ BlockShare(const char* kb, const char* vb, int D) {
#pragma unroll
        for (int x = 0; x < N; ++x) {
            const char* base = of_v(x) ? vb : kb;
            if constexpr (I4) {
                const int at = min(piece(x), D / 32 - 1);
                from[x] = base + 16 * at;
                pair[x] = base + D / 2 + 4 * at;
            } else {
                from[x] = base + 16 * min(piece(x), D / 8 - 1);
            }
        }
    }
    __device__ __forceinline__ void load(const int64_t* off) {
#pragma unroll
        for (int x = 0; x < N; ++x) {
            const int64_t o = off[row(x)];
            if constexpr (I4) {
                v[x] = __builtin_bit_cast(u32x4_t, *reinterpret_cast<const u32x4_a4_t*>(from[x] + o));
                sm[x] = *reinterpret_cast<const uint32_t*>(pair[x] + o);
            } else {
                v[x] = *reinterpret_cast<const u32x4_t*>(from[x] + o);
            }
        }
    }
    // To LDS, V's rows from `left` on as zeros (what lies there is nobody's).
    __device__ __forceinline__ void store(char* k, char* vl, int left) {
        if (left < KEYS) {
#pragma unroll
            for (int x = 0; x < N; ++x)
                if (of_v(x) && row(x) >= left) {
                    if constexpr (I4) sm[x] = 0u;
                    else v[x] = u32x4_t{0, 0, 0, 0};
                }
        }
#pragma unroll
        for (int x = 0; x < N; ++x) {
            char* to = (of_v(x) ? vl + row(x) * VP : k + row(x) * KP) + piece(x) * (I4 ? 64 : 16);
            if constexpr (I4) {
                half2_t s, m;
                four_bit_pair(sm[x], s, m);
#pragma unroll
                for (int i = 0; i < 4; ++i) *reinterpret_cast<half8_t*>(to + 16 * i) = four_bit_values(v[x][i], s, m);
            } else {
                *reinterpret_cast<u32x4_t*>(to) = v[x];
            }
        }
    }

private:
    // (the last threads have a piece fewer where they do not come out even: they take the last once more)
    __device__ __forceinline__ static int index(int x) {
        const int u = threadIdx.x + 256 * x;
        return ALL % 256 == 0 ? u : min(u, ALL - 1);
    }
};

// Keys among the places from t on (the first of a block), to the end of their list.
__device__ __forceinline__ int keys_left(const PagedItem& it, int t) { return (t < it.near ? min(it.hi, it.far) : it.hi) - t; }

template <int DP, bool I4>
__global__ void __launch_bounds__(256, DP <= 64 ? 3 : DP <= 128 ? 2 : 1) paged_many_kernel(PagedArgs a) {
    typedef BlockShare<DP, I4> Share;
    constexpr int KEYS = Share::KEYS, U = KEYS / 32, KK = DP / 16, DT = DP / 32;
    constexpr int KP = Share::KP, VP = Share::VP, BUF = KEYS * (KP + VP);
    __shared__ __attribute__((aligned(16))) char lds[2 * BUF];
    __shared__ int64_t off[2][KEYS];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    PagedItem it;
    if (!find_item<kManyRows, true, kManyUnit, false>(a, blockIdx.x, lane, it)) return;
    const KvView& c = a.c;
    const int r = lane & 31, h = lane >> 5;

    const int base = it.tile * kManyRows + 32 * wave;  // the wave's first row
    const int rho = base + r, i = rho / a.G;
    const bool mine = i < it.n;
    const int pos = mine ? it.len - it.n + i : -1;
    const int64_t tok = it.first + (mine ? i : 0);
    const int head = it.h * a.G + (mine ? rho - i * a.G : 0);
    half8_t qf[KK];
    {
        const _Float16* q = a.q + tok * a.q_token + (int64_t)head * a.q_head;
#pragma unroll
        for (int kk = 0; kk < KK; ++kk) {
            const int d = 16 * kk + 8 * h;
            qf[kk] = half8_t{};
            if (d < c.D) qf[kk] = *reinterpret_cast<const half8_t*>(q + d) * (_Float16)a.sign;
        }
    }
    const int khi = !mine ? 0 : a.causal ? pos + 1 : it.len;
    const int klo = a.window > 0 ? pos - a.window : INT32_MIN;
    // of the wave's rows: all see the keys [klo_all, khi_all), none those outside [klo_some, khi_some)
    const bool any = base < (int64_t)it.n * a.G;
    const int p0 = it.len - it.n + base / a.G, p1 = it.len - it.n + min(it.n - 1, (base + 31) / a.G);
    const int khi_all = a.causal ? p0 + 1 : it.len, khi_some = !any ? 0 : a.causal ? p1 + 1 : it.len;
    const int klo_all = a.window > 0 ? p1 - a.window : INT32_MIN;
    const int klo_some = a.window > 0 && a.stride == 0 ? p0 - a.window : INT32_MIN;

    const char* kb = c.k + (int64_t)it.h * c.head;
    const char* vb = c.v + (int64_t)it.h * c.head;
    auto place = [&](int t) {  // the offset of the key at place t + tid (tid < KEYS)
        return c.row_offset(it.b, key_at(a, it, min(t + tid, it.hi - 1)));
    };

    float m = kNoScore, l = 0.0f;
    float16_t acc[DT];
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[d][e] = 0.0f;

    Share share(kb, vb, c.D);
    if (it.lo < it.hi) {
        if (tid < KEYS) {
            off[0][tid] = place(it.lo);
            off[1][tid] = place(it.lo + KEYS);
        }
        __syncthreads();
        share.load(off[0]);
        share.store(lds, lds + KEYS * KP, keys_left(it, it.lo));
        __syncthreads();
    }
    int buf = 0;
    for (int t = it.lo; t < it.hi; t += KEYS, buf ^= 1) {
        const bool more = t + KEYS < it.hi;
        int64_t next = 0;
        if (more) {
            share.load(off[buf ^ 1]);
            if (tid < KEYS) next = place(t + 2 * KEYS);
        }
        const char* kl = lds + buf * BUF;
        const char* vl = kl + KEYS * KP;
        const bool isnear = t >= it.near;
        const int key0 = it.base + t - it.near, left = keys_left(it, t);
        if (any && (!isnear || (key0 < khi_some && key0 + KEYS > klo_some))) {
            float16_t s[U];
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int e = 0; e < 16; ++e) s[u][e] = 0.0f;
            // (FRAGS of K's operands are on their way before the first product that takes one)
            constexpr int FRAGS = DP <= 64 ? KK : 4;
#pragma unroll
            for (int k0 = 0; k0 < KK; k0 += FRAGS) {
                half8_t kf[U][FRAGS];
#pragma unroll
                for (int kk = 0; kk < FRAGS; ++kk)
#pragma unroll
                    for (int u = 0; u < U; ++u)
                        kf[u][kk] = *reinterpret_cast<const half8_t*>(kl + (32 * u + r) * KP + 32 * (k0 + kk) + 16 * h);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int kk = 0; kk < FRAGS; ++kk)
#pragma unroll
                    for (int u = 0; u < U; ++u)
                        s[u] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf[u][kk], qf[k0 + kk], s[u], 0, 0, 0);
            }
            if (left < KEYS || (isnear && (key0 + KEYS > khi_all || key0 < klo_all))) {
                // places [0, upto) and, of a window's block, from `from` on or on the stride
                const int upto = min(isnear ? khi - key0 : mine ? KEYS : 0, left) - 4 * h;
                if (isnear && a.window > 0) {
                    const int from = klo - key0 - 4 * h;
                    const uint64_t bits = a.stride > 0 ? stride_bits(key0, a.stride) >> (4 * h) : 0u;
#pragma unroll
                    for (int u = 0; u < U; ++u) {
                        const uint32_t half = (uint32_t)(bits >> (32 * u));
#pragma unroll
                        for (int e = 0; e < 16; ++e) {
                            const int at = 32 * u + 8 * (e >> 2) + (e & 3);
                            s[u][e] = at < upto && (at >= from || (half >> (at & 31) & 1)) ? s[u][e] : kNoScore;
                        }
                    }
                } else {
#pragma unroll
                    for (int u = 0; u < U; ++u)
#pragma unroll
                        for (int e = 0; e < 16; ++e) {
                            const int at = 32 * u + 8 * (e >> 2) + (e & 3);
                            s[u][e] = at < upto ? s[u][e] : kNoScore;
                        }
                }
            }
            float mx = s[0][0];
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int e = 0; e < 16; ++e) mx = __builtin_fmaxf(mx, s[u][e]);
            mx = __builtin_fmaxf(mx, __shfl_xor(mx, 32)) * a.scale;
            if (__any(mx > m)) {
                const float mn = __builtin_fmaxf(m, mx), f = mn == kNoScore ? 1.0f : exp2_fast(m - mn);
                l *= f;
#pragma unroll
                for (int d = 0; d < DT; ++d) acc[d] *= f;
                m = mn;
            }
            const float bias = kWeightBits - (m == kNoScore ? 0.0f : m);
            half8_t p[2 * U];
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const float w = exp2_fast(__builtin_fmaf(s[u][e], a.scale, bias));
                    l += w;
                    p[2 * u + (e >> 3)][e & 7] = (_Float16)w;
                }
#pragma unroll
            for (int d = 0; d < DT; ++d)
#pragma unroll
                for (int q = 0; q < 2 * U; ++q) {
                    union {
                        many_short4_t q[2];
                        half8_t h;
                    } x;
#pragma unroll
                    for (int b = 0; b < 2; ++b)
                        x.q[b] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                            (__attribute__((address_space(3))) many_short4_t*)(vl + (16 * q + 8 * b + 4 * h + ((lane & 15) >> 2)) * VP +
                                                                               2 * (32 * d + 16 * ((lane >> 4) & 1) + 4 * (lane & 3))));
                    acc[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(x.h, p[q], acc[d], 0, 0, 0);
                }
        }
        if (more) {
            char* to = lds + (buf ^ 1) * BUF;
            share.store(to, to + KEYS * KP, keys_left(it, t + KEYS));
            if (tid < KEYS) off[buf][tid] = next;
        }
        __syncthreads();
    }

    l += __shfl_xor(l, 32);
    bool fine = l < __builtin_inff();
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int e = 0; e < 16; ++e) fine = fine && __builtin_fabsf(acc[d][e]) < __builtin_inff();
    const int64_t s0 = (int64_t)it.slot * kManyRows + 32 * wave;
    if (mine) {
        const float inv = l > 0.0f ? 1.0f / l : 0.0f;
        if (it.parts == 1) {
            _Float16* out = a.out + tok * a.o_token + (int64_t)head * a.o_head;
#pragma unroll
            for (int d = 0; d < DT; ++d)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int at = 32 * d + 8 * e + 4 * h;
                    const many_half4_t v = {(_Float16)(acc[d][4 * e] * inv), (_Float16)(acc[d][4 * e + 1] * inv),
                                            (_Float16)(acc[d][4 * e + 2] * inv), (_Float16)(acc[d][4 * e + 3] * inv)};
                    if (at < c.D) *reinterpret_cast<many_half4_t*>(out + at) = v;
                }
            if (a.lse && h == 0) a.lse[tok * a.Hq + head] = lse_of(m, l);
        } else {
            float* po = a.part_o + (s0 + r) * c.D;
#pragma unroll
            for (int d = 0; d < DT; ++d)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int at = 32 * d + 8 * e + 4 * h;
                    const float4_t v = {acc[d][4 * e], acc[d][4 * e + 1], acc[d][4 * e + 2], acc[d][4 * e + 3]};
                    if (at < c.D) *reinterpret_cast<float4_t*>(po + at) = v;
                }
            if (h == 0) {
                a.part_ml[2 * (s0 + r)] = m;
                a.part_ml[2 * (s0 + r) + 1] = l;
            }
        }
    }
    // rows with an infinite or undefined value once more, key by key (slow_row)
    uint64_t bad = __ballot(mine && !fine);
    bad = (bad | bad >> 32) & 0xFFFFFFFFu;
    while (bad) {
        const int w = __builtin_ctzll(bad);
        bad &= bad - 1;
        const int brho = base + w, bi = brho / a.G, bh = it.h * a.G + brho - bi * a.G;
        const int64_t bt = it.first + bi;
        float ov[DP / 64], bm, bl;
        slow_row<DP, I4>(a, it, it.len - it.n + bi, a.q + bt * a.q_token + (int64_t)bh * a.q_head, lane, ov,
                         bm, bl);
        const float bin = bl > 0.0f || bl != bl ? 1.0f / bl : 0.0f;
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // (the stores above come first)
#pragma unroll
        for (int j = 0; j < DP / 64; ++j) {
            const int d = lane + 64 * j;
            if (d >= c.D) continue;
            if (it.parts == 1) a.out[bt * a.o_token + (int64_t)bh * a.o_head + d] = (_Float16)(ov[j] * bin);
            else a.part_o[(s0 + w) * c.D + d] = ov[j];
        }
        if (lane == 0) {
            if (it.parts == 1) {
                if (a.lse) a.lse[bt * a.Hq + bh] = lse_of(bm, bl);
            } else {
                a.part_ml[2 * (s0 + w)] = bm;
                a.part_ml[2 * (s0 + w) + 1] = bl;
            }
        }
    }
}

}  // namespace

template <bool I4>
hipError_t paged_many(const PagedArgs& a, hipStream_t s) {
    const int64_t tiles = ((int64_t)a.c.T * a.G / kManyRows + (a.c.B < a.c.T ? a.c.B : a.c.T)) * a.c.H;
    // (a sequence has two parts only where it is longer than the average of `target`)
    const dim3 grid((unsigned)(tiles + a.target));
    if (a.c.D <= 64) paged_many_kernel<64, I4><<<grid, 256, 0, s>>>(a);
    else if (a.c.D <= 128) paged_many_kernel<128, I4><<<grid, 256, 0, s>>>(a);
    else if (a.c.D <= 192) paged_many_kernel<192, I4><<<grid, 256, 0, s>>>(a);
    else paged_many_kernel<256, I4><<<grid, 256, 0, s>>>(a);
    hipError_t e = hipGetLastError();
    if (e == hipSuccess && a.target > 0) {
        paged_join_kernel<kManyRows, true, kManyUnit><<<dim3((unsigned)(tiles < a.target ? tiles : a.target), kManyRows / 4), 256, 0, s>>>(a);
        e = hipGetLastError();
    }
    return e;
}

}  // namespace vedic
