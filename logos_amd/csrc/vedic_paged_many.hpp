// vedic_paged_many.hpp -- attention of many new rows a sequence (a prompt, or the next piece
// of one) over its paged cache.
//
//   S^T = K Q^T (32 tokens x 32 rows per v_mfma_f32_32x32x16_f16), weights 2^(x - m + 14) with a
//   running maximum and sum in fp32, O^T += V^T P^T.
//
// A workgroup has a tile of 128 rows (four waves of 32) and a range of keys (vedic_paged.hpp).
// Blocks of 64 keys (32 with heads past 128) go through two buffers of LDS, one barrier a block: while
// a block is multiplied, the next one's rows are on their way into registers (from the pages, 16 bytes a
// thread and load; four bits are expanded on their way to LDS) and the places of the one
// after that are looked up.  K's rows lie 2 DP + 16 bytes apart (ds_read_b128 of eight rows meets
// every bank once), V's 2 DP + 32 (the same for the transposing ds_read_b64_tr_b16).  The scores'
// layout, a row of Q per lane, is what the second product takes: the weights stay in
// registers.  Masks are looked at only where some key of a block is hidden from a row of the wave.
//
// Bound by the vector and the matrix instructions of a wave, which take turns more than they overlap: of a prompt of 8192 in 16
// heads of 64 (198 us in a row of calls, 690 TFLOP/s of what its mask leaves; 195 to 209 by box) the vector pipes are busy 63 %
// and the matrix pipes 32 %, the LDS 33 %.  A block of 64 keys takes a wave 16 matrix instructions and about 220 vector ones,
// 144 of them the weights' (maximum, fma, exponential, sum, half a conversion each), the others rescaling, masks and the next
// block's way to LDS.  Three waves a SIMD hide some of one kind behind the other (two: 237 us).
#pragma once

#include "vedic_paged.hpp"

namespace vedic {

namespace {

typedef short many_short4_t __attribute__((ext_vector_type(4)));

// Keys of a block: with heads past 128 the next block's rows would take 64 registers more.
constexpr int many_keys(int dp) { return dp <= 128 ? 64 : 32; }

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
    // To LDS, V's rows from `left` on as zeros (what lies there is nobody's), and pieces past the end of a head narrower than DP
    // (Q has zeros there, but what the last piece holds may be infinite).
    __device__ __forceinline__ void store(char* k, char* vl, int left, int D) {
        if (left < KEYS || D < DP) {
#pragma unroll
            for (int x = 0; x < N; ++x)
                if ((of_v(x) && row(x) >= left) || piece(x) * (I4 ? 32 : 8) >= D) {
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

template <int DP, bool I4, bool PLAN>
__global__ void __launch_bounds__(256, DP <= 64 ? 3 : DP <= 128 ? 2 : 1) paged_many_kernel(PagedArgs a) {
    typedef BlockShare<DP, I4> Share;
    constexpr int KEYS = Share::KEYS, U = KEYS / 32, KK = DP / 16, DT = DP / 32;
    constexpr int KP = Share::KP, VP = Share::VP;
    __shared__ __attribute__((aligned(16))) char kbuf[2][KEYS * KP];
    __shared__ __attribute__((aligned(16))) char vbuf[2][KEYS * VP];
    __shared__ int64_t off[2][KEYS];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    PagedItem it;
    if (!find_item<kManyRows, true, kManyUnit, false, PLAN>(a, blockIdx.x, lane, it)) return;
    const KvView& c = a.c;
    const int r = lane & 31, h = lane >> 5;

    const int base = it.tile * kManyRows + 32 * wave;  // the wave's first row
    const int rho = base + r, i = a.by_group(rho);
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
    // of the wave's rows: all see the keys [klo_all, khi_all)
    const int p0 = it.len - it.n + a.by_group(base), p1 = it.len - it.n + min(it.n - 1, a.by_group(base + 31));
    const int khi_all = base + 32 > (int64_t)it.n * a.G ? 0 : a.causal ? p0 + 1 : it.len;
    const int klo_all = a.window > 0 ? p1 - a.window : INT32_MIN;

    const char* kb = c.k + (int64_t)it.h * c.head;
    const char* vb = c.v + (int64_t)it.h * c.head;
    // Where the key at place t + tid (tid < KEYS) lies: its page, looked up now, and its row's offset once that is there.
    const int* table = c.table + it.b * c.ldt;
    auto find = [&](int t, int& page, int& inside) {
        const int key = key_at(a, it, min(t + tid, it.hi - 1)), tp = c.page_of(key);
        page = table[tp];
        inside = key - tp * c.ps;
    };
    auto offset = [&](int page, int inside) {
        return ((unsigned)page < (unsigned)c.pages ? page : 0) * c.page + inside * c.token;
    };

    float m = kNoScore, l = 0.0f;
    float16_t acc[DT];
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[d][e] = 0.0f;
    Share share(kb, vb, c.D);

    const int kat = r * KP + 16 * h, vat = (4 * h + ((lane & 15) >> 2)) * VP + 2 * (16 * ((lane >> 4) & 1) + 4 * (lane & 3));
    if (it.lo < it.hi) {
        if (tid < KEYS) {
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                int page, inside;
                find(it.lo + x * KEYS, page, inside);
                off[x][tid] = offset(page, inside);
            }
        }
        __syncthreads();
        share.load(off[0]);
        share.store(kbuf[0], vbuf[0], keys_left(it, it.lo), c.D);
        __syncthreads();
    }
    int buf = 0;
    for (int t = it.lo; t < it.hi; t += KEYS, buf ^= 1) {
        const bool more = t + KEYS < it.hi;
        int page = 0, inside = 0;
        if (more) {
            if (tid < KEYS) find(t + 2 * KEYS, page, inside);  // (first: the rows that follow need not be there for its answer)
            share.load(off[buf ^ 1]);
        }
        float16_t s[U];
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int e = 0; e < 16; ++e) s[u][e] = 0.0f;
        // (FRAGS of K's operands are on their way before the first product that takes one)
        constexpr int FRAGS = 4;
#pragma unroll
        for (int k0 = 0; k0 < KK; k0 += FRAGS) {
            half8_t kf[U][FRAGS];
#pragma unroll
            for (int kk = 0; kk < FRAGS; ++kk)
#pragma unroll
                for (int u = 0; u < U; ++u)
                    kf[u][kk] = *reinterpret_cast<const half8_t*>(kbuf[buf] + kat + 32 * u * KP + 32 * (k0 + kk));
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int kk = 0; kk < FRAGS; ++kk)
#pragma unroll
                for (int u = 0; u < U; ++u)
                    s[u] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf[u][kk], qf[k0 + kk], s[u], 0, 0, 0);
        }
        const bool isnear = t >= it.near;
        const int key0 = it.base + t - it.near, left = keys_left(it, t);
        if (left < KEYS || (isnear ? key0 + KEYS > khi_all || key0 < klo_all : khi_all == 0)) {
            const int upto = min(isnear ? khi - key0 : mine ? KEYS : 0, left) - 4 * h;
            const bool window = isnear && a.window > 0;
            const uint64_t strided = window && a.stride > 0 ? stride_bits(key0, a.stride) >> (4 * h) : 0;
            const uint64_t bits = place_bits(window ? klo - key0 - 4 * h : 0, upto, strided);
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const uint32_t bit = 1u << (8 * (e >> 2) + (e & 3));
                    s[u][e] = (uint32_t)(bits >> (32 * u)) & bit ? s[u][e] : kNoScore;
                }
        }
        float mx = s[0][0];
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int e = 0; e < 16; ++e) mx = __builtin_fmaxf(mx, s[u][e]);
        mx = both_halves_max(mx);
        if (__any(mx > m)) {
            const float mn = __builtin_fmaxf(m, mx), f = mn == kNoScore ? 1.0f : exp2_fast((m - mn) * a.scale);
            l *= f;
#pragma unroll
            for (int d = 0; d < DT; ++d) acc[d] *= f;
            m = mn;
        }
        const float mu = m == kNoScore ? 0.0f : m;
        float bias = __builtin_fmaf(-mu, a.scale, kWeightBits);
        // (c m's rounding is in all of a block's weights, but not the same in the next block's, and below 2^-14 of them up to
        // here; past it differences of scores, as everywhere else)
        if (__any(__builtin_fabsf(bias) > 0x1p10f)) {
            bias = kWeightBits;
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int e = 0; e < 16; ++e) s[u][e] -= mu;
        }
        // (In 11 bits, which is off about as much as the output's own rounding.  A second part would cost 27 to 37 %: a prompt of
        // 8192 in 16 heads of 64 195 / 266 us, three pieces of 500 rows over four bits 187 / 237.)
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
        for (int q = 0; q < 2 * U; ++q)
#pragma unroll
            for (int d = 0; d < DT; ++d) {
                union {
                    many_short4_t q[2];
                    half8_t h;
                } x;
#pragma unroll
                for (int b = 0; b < 2; ++b)
                    x.q[b] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                        (__attribute__((address_space(3))) many_short4_t*)(vbuf[buf] + vat + (16 * q + 8 * b) * VP + 64 * d));
                acc[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(x.h, p[q], acc[d], 0, 0, 0);
            }
        if (more) {
            share.store(kbuf[buf ^ 1], vbuf[buf ^ 1], keys_left(it, t + KEYS), c.D);
            if (tid < KEYS) off[buf][tid] = offset(page, inside);
        }
        __syncthreads();
    }
    finish_rows<DP, I4>(a, it, base, (int64_t)it.slot * kManyRows + 32 * wave, acc, m, l, lane);
}

}  // namespace

template <bool I4, bool PLAN>
hipError_t paged_many_by(const PagedArgs& a, hipStream_t s) {
    const int64_t tiles = ((int64_t)a.c.T * a.G / kManyRows + (a.c.B < a.c.T ? a.c.B : a.c.T)) * a.c.H;
    const dim3 grid((unsigned)(tiles + a.target)), join((unsigned)(tiles < a.target ? tiles : a.target), 4);
    if (a.c.D <= 64) paged_many_kernel<64, I4, PLAN><<<grid, 256, 0, s>>>(a);
    else if (a.c.D <= 128) paged_many_kernel<128, I4, PLAN><<<grid, 256, 0, s>>>(a);
    else if (a.c.D <= 192) paged_many_kernel<192, I4, PLAN><<<grid, 256, 0, s>>>(a);
    else paged_many_kernel<256, I4, PLAN><<<grid, 256, 0, s>>>(a);
    hipError_t e = hipGetLastError();
    if (e == hipSuccess && a.target > 0) {
        paged_join_kernel<kManyRows, true, kManyUnit, false, PLAN><<<join, 256, 0, s>>>(a, kManyRows / 4);
        e = hipGetLastError();
    }
    return e;
}

template <bool I4>
hipError_t paged_many(const PagedArgs& a, hipStream_t s) {
    return a.plan ? paged_many_by<I4, true>(a, s) : paged_many_by<I4, false>(a, s);
}

}  // namespace vedic
