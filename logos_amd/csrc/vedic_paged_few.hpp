// vedic_paged_few.hpp -- attention of a few new rows a sequence over its paged cache: one
// decoded token, or up to some rows of a key head's group of query heads.
//
//   S^T = K Q^T (16 tokens x 16 rows per v_mfma_f32_16x16x32_f16), weights 2^(x - m + 14) with a
//   running maximum and sum in fp32, O^T += V^T P^T.
//
// A workgroup has a tile of 16 rows and a range of keys (vedic_paged.hpp); its four waves
// take 32 keys each in turn, on their own: a wave reads K into the registers that the MFMA
// takes, V through a piece of LDS of its own (written as rows, read by the transposing
// ds_read_b64_tr_b16), and no barrier is met until the four partial results are added.  The
// scores come out with a row of Q per lane and tokens 4 g + i, 16 + 4 g + i in lane group g, which is
// the order in which the second product then contracts: the weights stay in registers.
// K and V of the next 32 keys are loaded as soon as their registers are free; a wave has 16 KB
// under way (binary16, heads of 128), a CU eight to twelve waves.  Reading the cache bounds it (32 sequences of up to
// 16384 tokens, 8 key heads of 128: 203 us, 5.5 TB/s), in four bits expanding it as well (64 sequences: 184 us, 4.0 TB/s, the
// vector pipes busy 63 % of it), and for one sequence what an item looks up one after another: lists, table, rows (4099 tokens
// in 16 heads of 64: 8.7 us).
//
// Four bits: lane group g takes values g DP/4 .. + DP/4 - 1 of a token's row, whole words; K is
// expanded in registers as the MFMA takes it, V as it goes to LDS.
#pragma once

#include "vedic_paged.hpp"

namespace vedic {

namespace {

typedef short paged_short4_t __attribute__((ext_vector_type(4)));
typedef _Float16 half4_t __attribute__((ext_vector_type(4)));

// A lane's share of one token's row, DP / 4 values in KK pieces of eight; `first` is where its
// pieces begin (a place fixed for the lane).  Heads narrower than DP: pieces past the end hold
// others once more, which of V are columns of the output that nobody reads; K's are taken as
// zeros (Q's alone would not do: what they hold may be infinite).
template <int DP, bool I4>
struct RowShare;
template <int DP>
struct RowShare<DP, false> {
    static constexpr int KK = DP / 32;
    u32x4_t v[KK];
    // Piece kk: the row's values 32 kk + 8 g .. + 7.
    struct Place {
        int at[KK];  // bytes
        __device__ __forceinline__ Place(int D, int g) {
#pragma unroll
            for (int kk = 0; kk < KK; ++kk) at[kk] = 2 * min(32 * kk + 8 * g, D - 8);
        }
        __device__ __forceinline__ bool own(int kk, int D, int g) const { return 32 * kk + 8 * g < D; }
        __device__ __forceinline__ int value(int kk, int g) const { return 32 * kk + 8 * g; }
    };
    __device__ __forceinline__ void load(const char* row, const Place& p, int) {
#pragma unroll
        for (int kk = 0; kk < KK; ++kk) v[kk] = *reinterpret_cast<const u32x4_t*>(row + p.at[kk]);
    }
    __device__ __forceinline__ half8_t frag(int kk, const Place&) const { return __builtin_bit_cast(half8_t, v[kk]); }
    // (the last two pieces are the only ones that may lie past the end: D > DP - 64)
    __device__ __forceinline__ half8_t key(int kk, const Place& p, int D, int g) const {
        return kk >= KK - 2 && !p.own(kk, D, g) ? half8_t{} : frag(kk, p);
    }
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int kk = 0; kk < KK; ++kk) v[kk] = u32x4_t{0, 0, 0, 0};
    }
};
template <int DP>
struct RowShare<DP, true> {
    static constexpr int KK = DP / 32, NS = (KK + 3) / 4;
    uint32_t w[KK];
    uint32_t sm[NS];
    // Piece kk: word `first` + kk of the row, first = g KK or so far down that KK words are left.
    struct Place {
        int first, pairs[NS];  // word; byte offsets of its groups' pairs
        __device__ __forceinline__ Place(int D, int g) {
            first = min(g * KK, D / 8 - KK);
#pragma unroll
            for (int i = 0; i < NS; ++i) pairs[i] = D / 2 + 4 * min(first / 4 + i, D / 32 - 1);
        }
        __device__ __forceinline__ bool own(int kk, int, int g) const { return first + kk >= g * KK; }
        __device__ __forceinline__ int value(int kk, int) const { return 8 * (first + kk); }
    };
    __device__ __forceinline__ void load(const char* row, const Place& q, int) {
        const uint32_t* p = reinterpret_cast<const uint32_t*>(row) + q.first;
        if constexpr (KK % 4 == 0) {
#pragma unroll
            for (int i = 0; i < KK / 4; ++i) {
                const u32x4_a4_t x = *reinterpret_cast<const u32x4_a4_t*>(p + 4 * i);
#pragma unroll
                for (int j = 0; j < 4; ++j) w[4 * i + j] = x[j];
            }
        } else {
            typedef uint32_t u32x2_a4_t __attribute__((ext_vector_type(2), aligned(4)));
#pragma unroll
            for (int i = 0; i < KK / 2; ++i) {
                const u32x2_a4_t x = *reinterpret_cast<const u32x2_a4_t*>(p + 2 * i);
                w[2 * i] = x[0];
                w[2 * i + 1] = x[1];
            }
        }
#pragma unroll
        for (int i = 0; i < NS; ++i) sm[i] = *reinterpret_cast<const uint32_t*>(row + q.pairs[i]);
    }
    __device__ __forceinline__ uint32_t pair(int kk, const Place& q) const {
        if constexpr (NS > 1) return (q.first + kk) / 4 > q.first / 4 ? sm[1] : sm[0];  // (DP / 4 values: two groups at most)
        return sm[0];
    }
    __device__ __forceinline__ half8_t values(int kk, uint32_t x) const {
        half2_t s, m;
        four_bit_pair(x, s, m);
        return four_bit_values(w[kk], s, m);
    }
    __device__ __forceinline__ half8_t frag(int kk, const Place& q) const { return values(kk, pair(kk, q)); }
    // (at most the first four pieces are another lane group's: D >= DP - 32)
    __device__ __forceinline__ half8_t key(int kk, const Place& q, int D, int g) const {
        return values(kk, kk < 4 && !q.own(kk, D, g) ? 0u : pair(kk, q));
    }
    __device__ __forceinline__ void clear() {  // (a pair of zeros: the value 0 whatever the code)
#pragma unroll
        for (int i = 0; i < NS; ++i) sm[i] = 0u;
    }
};

// NARROW: heads of fewer than DP values.  (Looked at here instead, K's zeros cost full heads over four bits 2 to 5 %.)
template <int DP, bool I4, bool NARROW, bool PLAN>
__global__ void __launch_bounds__(256, I4 || DP <= 192 ? 2 : 1) paged_few_kernel(PagedArgs a) {
    typedef RowShare<DP, I4> Share;
    constexpr int KK = DP / 32, DT = DP / 16, PITCH = 2 * DP + 32, OP = DP + 4;
    static_assert(16 * OP * 4 <= 32 * PITCH, "a wave's partial result fits its piece of LDS");
    __shared__ __attribute__((aligned(16))) char lds[4 * 32 * PITCH];
    __shared__ float ml[4][16][2];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    PagedItem it;
    if (!find_item<kFewRows, false, kFewUnit, false, PLAN>(a, blockIdx.x, lane, it)) return;
    const KvView& c = a.c;
    const int r = lane & 15, g = lane >> 4;
    char* vb = lds + wave * (32 * PITCH);

    // this lane's row of Q
    const int rho = it.tile * kFewRows + r, i = a.by_group(rho);
    const bool mine = i < it.n;
    const int pos = mine ? it.len - it.n + i : -1;
    const typename Share::Place where(c.D, g);
    half8_t qf[KK];
    {
        const _Float16* q = a.q + (int64_t)(it.first + (mine ? i : 0)) * a.q_token +
                            (int64_t)(it.h * a.G + (mine ? rho - i * a.G : 0)) * a.q_head;
#pragma unroll
        for (int kk = 0; kk < KK; ++kk) {
            qf[kk] = half8_t{};
            if (where.own(kk, c.D, g)) qf[kk] = *reinterpret_cast<const half8_t*>(q + where.value(kk, g)) * (_Float16)a.sign;
        }
    }
    // keys [klo, khi) of this row, and of all rows of the tile
    const int khi = !mine ? 0 : a.causal ? pos + 1 : it.len;
    const int klo = a.window > 0 ? pos - a.window : INT32_MIN;
    const int i0 = a.by_group(it.tile * kFewRows), i1 = min(it.n - 1, a.by_group(it.tile * kFewRows + kFewRows - 1));
    const int khi_all = a.causal ? it.len - it.n + i0 + 1 : it.len;
    const int klo_all = a.window > 0 ? it.len - it.n + i1 - a.window : INT32_MIN;

    const char* kb = c.k + (int64_t)it.h * c.head;
    const char* vbase = c.v + (int64_t)it.h * c.head;
    const int* table = c.table + it.b * c.ldt;
    // The page and the row in it of each of the lane's two tokens of the 32 places at t.  Where pages are
    // whole sixteens, the sixteen near keys of a tile lie in one: one lookup, and the lane's own row
    // apart from it (rows behind the sequence's end are some row of its page).
    const bool whole = c.ps % 16 == 0;
    const int64_t mine_off = r * c.token;
    auto place = [&](int t, int (&page)[2], int (&inside)[2]) {
        if (whole && t >= it.near) {
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const int key = it.base + min(t + 16 * u, (it.hi - 1) & ~15) - it.near, tp = c.page_of(key);
                page[u] = table[tp];
                inside[u] = key - tp * c.ps;
            }
        } else {
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const int key = key_at(a, it, min(t + 16 * u + r, it.hi - 1)), tp = c.page_of(key);
                page[u] = table[tp];
                inside[u] = key - tp * c.ps;
            }
        }
    };
    auto offset = [&](int t, int (&page)[2], int (&inside)[2], int64_t (&off)[2]) {
        if (whole && t >= it.near) {
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const int p = __builtin_amdgcn_readfirstlane(page[u]), i = __builtin_amdgcn_readfirstlane(inside[u]);
                off[u] = ((unsigned)p < (unsigned)c.pages ? p : 0) * c.page + i * c.token + mine_off;
            }
        } else {
#pragma unroll
            for (int u = 0; u < 2; ++u)
                off[u] = ((unsigned)page[u] < (unsigned)c.pages ? page[u] : 0) * c.page + inside[u] * c.token;
        }
    };

    float m = kNoScore, l = 0.0f;
    float4_t acc[DT];
#pragma unroll
    for (int d = 0; d < DT; ++d) acc[d] = float4_t{0.0f, 0.0f, 0.0f, 0.0f};

    int t = it.lo + 32 * wave;
    Share k[2], v[2];
    int64_t off[2];
    int page[2], inside[2];
    if (t < it.hi) {
        place(t, page, inside);
        offset(t, page, inside, off);
#pragma unroll
        for (int u = 0; u < 2; ++u) k[u].load(kb + off[u], where, g);
#pragma unroll
        for (int u = 0; u < 2; ++u) v[u].load(vbase + off[u], where, g);
        if (t + kFewUnit < it.hi) place(t + kFewUnit, page, inside);
    }
    for (; t < it.hi; t += kFewUnit) {
        const bool more = t + kFewUnit < it.hi;
        float4_t s[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            s[u] = float4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int kk = 0; kk < KK; ++kk)
                s[u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(NARROW ? k[u].key(kk, where, c.D, g) : k[u].frag(kk, where), qf[kk], s[u], 0,
                                                              0, 0);
        }
        if (more) {
            offset(t + kFewUnit, page, inside, off);
#pragma unroll
            for (int u = 0; u < 2; ++u) k[u].load(kb + off[u], where, g);
        }
        // V of this block to LDS; rows past the range as zeros (what lies there is nobody's)
        const bool isnear = t >= it.near;
        const int left = min(it.hi, isnear ? it.hi : it.far) - t;  // places that are keys
        if (left < 32) {
#pragma unroll
            for (int u = 0; u < 2; ++u)
                if (16 * u + r >= left) v[u].clear();
        }
        asm volatile("" ::: "memory");
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int kk = 0; kk < KK; ++kk)
                *reinterpret_cast<half8_t*>(vb + (16 * u + r) * PITCH + 2 * where.value(kk, g)) = v[u].frag(kk, where);
        asm volatile("" ::: "memory");
        if (more) {
#pragma unroll
            for (int u = 0; u < 2; ++u) v[u].load(vbase + off[u], where, g);
            if (t + 2 * kFewUnit < it.hi) place(t + 2 * kFewUnit, page, inside);
        }
        // weights
        const int key0 = it.base + t - it.near;
        if (left < 32 || (isnear && (key0 + 32 > khi_all || key0 < klo_all))) {
            const int upto = min(isnear ? khi - key0 : mine ? 32 : 0, left) - 4 * g;
            const bool window = isnear && a.window > 0;
            const uint64_t more = window && a.stride > 0 ? stride_bits(key0, a.stride) >> (4 * g) : 0;
            const uint32_t bits = (uint32_t)place_bits(window ? klo - key0 - 4 * g : 0, upto, more);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const uint32_t bit = 1u << (16 * (e >> 2) + (e & 3));
                s[e >> 2][e & 3] = bits & bit ? s[e >> 2][e & 3] : kNoScore;
            }
        }
        float mx = kNoScore;
#pragma unroll
        for (int e = 0; e < 8; ++e) mx = __builtin_fmaxf(mx, s[e >> 2][e & 3]);
        mx = __builtin_fmaxf(mx, __shfl_xor(mx, 16));
        mx = __builtin_fmaxf(mx, __shfl_xor(mx, 32));
        if (__any(mx > m)) {
            const float mn = __builtin_fmaxf(m, mx), f = mn == kNoScore ? 1.0f : exp2_fast((m - mn) * a.scale);
            m = mn;
            l *= f;
#pragma unroll
            for (int d = 0; d < DT; ++d) acc[d] *= f;
        }
        const float mu = m == kNoScore ? 0.0f : m;
        // Over binary16 a weight is multiplied in two parts, 22 bits of it, which reading the cache hides (32 sequences 207 us with
        // one part and with two).  Over four bits in one: a step of the cache's codes is 1/15 of its group's range, and the second
        // part would take 10 % (64 sequences 181 / 198 us, or 197 in the registers of one part).
        constexpr int PARTS = I4 ? 1 : 2;
        half8_t p[PARTS];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float w = exp2_fast(__builtin_fmaf(s[e >> 2][e & 3] - mu, a.scale, kWeightBits));
            l += w;
            p[0][e] = (_Float16)w;
            if constexpr (PARTS == 2) p[1][e] = (_Float16)(w - (float)p[0][e]);
        }
#pragma unroll
        for (int d = 0; d < DT; ++d) {
            union {
                paged_short4_t q[2];
                half8_t h;
            } u;
#pragma unroll
            for (int b = 0; b < 2; ++b)
                u.q[b] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                    (__attribute__((address_space(3))) paged_short4_t*)(vb + (16 * b + 4 * g + (r >> 2)) * PITCH +
                                                                        2 * (16 * d + 4 * (r & 3))));
#pragma unroll
            for (int x = 0; x < PARTS; ++x) acc[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(u.h, p[x], acc[d], 0, 0, 0);
        }
        asm volatile("" ::: "memory");
    }

    // the four waves' results
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);
    if (g == 0) {
        ml[wave][r][0] = m;
        ml[wave][r][1] = l;
    }
    float* po = reinterpret_cast<float*>(vb);
#pragma unroll
    for (int d = 0; d < DT; ++d) *reinterpret_cast<float4_t*>(po + r * OP + 16 * d + 4 * g) = acc[d];
    __syncthreads();
    const int row = threadIdx.x >> 4, col = 4 * (threadIdx.x & 15);
    const int rrho = it.tile * kFewRows + row, ri = a.by_group(rrho);
    float M = kNoScore, L = 0.0f, fw[4];
#pragma unroll
    for (int w = 0; w < 4; ++w) M = __builtin_fmaxf(M, ml[w][row][0]);
    const float mu = M == kNoScore ? 0.0f : M;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        fw[w] = exp2_fast((ml[w][row][0] - mu) * a.scale);
        L += ml[w][row][1] * fw[w];
    }
    float4_t o[DP / 64];
    bool fine = true;
#pragma unroll
    for (int j = 0; j < DP / 64; ++j) {
        o[j] = float4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int w = 0; w < 4; ++w)
            o[j] += *reinterpret_cast<const float4_t*>(lds + w * (32 * PITCH) + 4 * (row * OP + col + 64 * j)) * fw[w];
#pragma unroll
        for (int q = 0; q < 4; ++q) fine = fine && (col + 64 * j >= c.D || __builtin_fabsf(o[j][q]) < __builtin_inff());
    }
    fine |= L != L;
    const bool here = ri < it.n;
    const int head = it.h * a.G + rrho - ri * a.G, rpos = it.len - it.n + ri;
    const int64_t tok = it.first + ri;
    const float inv = inverse_of(a, rpos, it.len, L);
    if (here) {
        if (it.parts == 1) {
            _Float16* out = a.out + tok * a.o_token + (int64_t)head * a.o_head + col;
#pragma unroll
            for (int j = 0; j < DP / 64; ++j)
                if (col + 64 * j < c.D) {
                    const half4_t h = {(_Float16)(o[j][0] * inv), (_Float16)(o[j][1] * inv), (_Float16)(o[j][2] * inv),
                                       (_Float16)(o[j][3] * inv)};
                    *reinterpret_cast<half4_t*>(out + 64 * j) = h;
                }
            if (a.lse && col == 0) a.lse[tok * a.Hq + head] = lse_of(a, rpos, it.len, M, L);
        } else {
            const int64_t s0 = (int64_t)it.slot * kFewRows + row;
#pragma unroll
            for (int j = 0; j < DP / 64; ++j)
                if (col + 64 * j < c.D) *reinterpret_cast<float4_t*>(a.part_o + s0 * c.D + col + 64 * j) = o[j];
            if (col == 0) {
                a.part_ml[2 * s0] = M;
                a.part_ml[2 * s0 + 1] = L;
            }
        }
    }
    // rows with an infinite or undefined value once more, key by key (slow_row)
    if (!__syncthreads_or(here && !fine)) return;
    const uint64_t bad = __ballot(here && !fine);
    for (int w = 0; w < 4; ++w) {
        if (((bad >> (16 * w)) & 0xFFFF) == 0) continue;  // row 4 wave + w
        const int brho = it.tile * kFewRows + 4 * wave + w, bi = a.by_group(brho), bh = it.h * a.G + brho - bi * a.G;
        const int bpos = it.len - it.n + bi;
        const int64_t bt = it.first + bi;
        float ov[DP / 64], bm, bl;
        slow_row<DP, I4>(a, it, bpos, a.q + bt * a.q_token + (int64_t)bh * a.q_head, lane, ov,
                         bm, bl);
        const float bin = inverse_of(a, bpos, it.len, bl);
        const int64_t s0 = (int64_t)it.slot * kFewRows + 4 * wave + w;
#pragma unroll
        for (int j = 0; j < DP / 64; ++j) {
            const int d = lane + 64 * j;
            if (d >= c.D) continue;
            if (it.parts == 1) a.out[bt * a.o_token + (int64_t)bh * a.o_head + d] = (_Float16)(ov[j] * bin);
            else a.part_o[s0 * c.D + d] = ov[j];
        }
        if (lane == 0) {
            if (it.parts == 1) {
                if (a.lse) a.lse[bt * a.Hq + bh] = lse_of(a, bpos, it.len, bm, bl);
            } else {
                a.part_ml[2 * s0] = bm;
                a.part_ml[2 * s0 + 1] = bl;
            }
        }
    }
}

}  // namespace

template <int DP, bool I4, bool PLAN>
void paged_few_of(const PagedArgs& a, const dim3& grid, hipStream_t s) {
    if (a.c.D < DP) paged_few_kernel<DP, I4, true, PLAN><<<grid, 256, 0, s>>>(a);
    else paged_few_kernel<DP, I4, false, PLAN><<<grid, 256, 0, s>>>(a);
}

template <bool I4, bool PLAN>
hipError_t paged_few_by(const PagedArgs& a, hipStream_t s) {
    const int64_t tiles = ((int64_t)a.c.T * a.G / kFewRows + (a.c.B < a.c.T ? a.c.B : a.c.T)) * a.c.H;
    const dim3 grid((unsigned)(tiles + a.target));
    if (a.c.D <= 64) paged_few_of<64, I4, PLAN>(a, grid, s);
    else if (a.c.D <= 128) paged_few_of<128, I4, PLAN>(a, grid, s);
    else if (a.c.D <= 192) paged_few_of<192, I4, PLAN>(a, grid, s);
    else paged_few_of<256, I4, PLAN>(a, grid, s);
    hipError_t e = hipGetLastError();
    if (e == hipSuccess && a.target > 0) {
        const int rows = a.c.q_start == nullptr && a.G < kFewRows ? a.G : kFewRows;
        const unsigned units = (unsigned)(tiles < a.target ? tiles : a.target);
        // A workgroup a row of few tiles (one sequence of 16000 tokens, 8 heads of 128: 12.3 us by a wave a row, 5.4), a wave
        // a row of many.
        if ((int64_t)units * rows <= 2 * a.target) paged_join_kernel<kFewRows, false, kFewUnit, true, PLAN><<<dim3(units, rows), 256, 0, s>>>(a, 1);
        else paged_join_kernel<kFewRows, false, kFewUnit, false, PLAN><<<dim3(units, (rows + 3) / 4), 256, 0, s>>>(a, 4);
        e = hipGetLastError();
    }
    return e;
}

template <bool I4>
hipError_t paged_few(const PagedArgs& a, hipStream_t s) {
    return a.plan ? paged_few_by<I4, true>(a, s) : paged_few_by<I4, false>(a, s);
}

}  // namespace vedic
