// vedic_paged.hpp -- what the attention kernels over a paged cache share: how the work is
// dealt out, which keys a row sees, a row computed without matrix instructions, and the
// join of split items.
//
// A work item is a tile of ROWS rows of one sequence and one key head, and a range of its
// keys.  Row rho of a sequence is new token rho / G, head rho % G of the G query heads that
// share the key head, so that a key is read once for all of them.  Lengths are known on the
// GPU only: every workgroup adds up the keys of all tiles, takes 1 / target of them (rounded
// up) as the length of a part, and finds its own item by a scan over the sequences; the
// host's grid is as large as the items can be.  So a batch of one long and many short
// sequences is dealt out evenly, whatever the table's width.  Of many sequences the sums are made
// beforehand, by 64 sequences (vedic_paged_plan.hip).
//
// Parts hold their sums relative to their own largest score m: O = sum of 2^(c (q.k - m) + 14) v and l
// the same without v, c the scale times log2(e); the join multiplies by 2^(c (m - M)) in the order of
// the parts.  The 2^14 keeps weights normal binary16 numbers down to 2^-28 of the largest.  (Differences of scores, not of
// c times them: c m is rounded, by more than a weight's range from 2^29 on.)
#pragma once

#include "vedic_cache.hpp"

namespace vedic {

constexpr float kWeightBits = 14.0f;
constexpr float kNoScore = -__builtin_inff();

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

// The larger of a lane's value and that of the lane 32 from it.
__device__ __forceinline__ float both_halves_max(float x) {
    const uint32_t b = __builtin_bit_cast(uint32_t, x);
    const auto r = __builtin_amdgcn_permlane32_swap(b, b, false, false);
    return __builtin_fmaxf(__builtin_bit_cast(float, (uint32_t)r[0]), __builtin_bit_cast(float, (uint32_t)r[1]));
}

struct PagedItem {
    int b, tile, h;       // sequence, tile of its rows, key head
    int first, n, len;    // its new rows and its tokens
    int base, far, near;  // the tile's keys (tile_keys)
    int lo, hi;           // places of this part
    int part, parts;
    int slot;             // of the partial result (parts > 1)
};

constexpr int kPlaces = 64;  // a block of keys lies in one of the two lists

// The keys that rows i0 .. i1 of a sequence see, as a list: places 0 .. far - 1 are the multiples of
// the stride before `base` (every row's window begins at or after it), places near .. hi - 1
// the keys base, base + 1, .., of which a row may see some; near is far in whole blocks.
__device__ __forceinline__ int tile_keys(const PagedArgs& a, int len, int n, int i0, int i1, int& base, int& far, int& near) {
    const int end = a.causal ? max(0, len - n + i1 + 1) : len;
    base = a.window > 0 ? max(0, len - n + i0 - a.window) & ~(kPlaces - 1) : 0;
    far = a.stride > 0 ? (base + a.stride - 1) / a.stride : 0;
    near = (far + kPlaces - 1) & ~(kPlaces - 1);
    return near + max(0, end - base);
}
// The key at a place (far ones past the end: the last).
__device__ __forceinline__ int key_at(const PagedArgs& a, const PagedItem& it, int place) {
    return place < it.near ? min(place, it.far - 1) * a.stride : it.base + place - it.near;
}

// A sequence's new rows and tokens, its tiles, and the longest list of keys among them (the last one's, or near it).
struct SequenceWork {
    int first, n, len, tiles, span;
};
template <int ROWS, bool MANY>
__device__ __forceinline__ SequenceWork sequence_work(const PagedArgs& a, int b) {
    SequenceWork w{0, 0, 0, 0, 0};
    if (b >= a.c.B) return w;
    a.c.rows_of(b, w.first, w.n);
    w.len = a.c.len_of(b);
    const int rows = w.n * a.G;  // (below 2^30)
    if (w.n == 0 || (rows > a.few_most) != MANY) return w;
    w.tiles = (rows + ROWS - 1) / ROWS;
    int base, far, near;
    w.span = tile_keys(a, w.len, w.n, a.by_group((w.tiles - 1) * ROWS), w.n - 1, base, far, near);
    return w;
}

// Sums over the lanes up to each (DPP: shifts within rows of 16, then the rows' last lanes).
template <int CTRL, int ROWS_OF>
__device__ __forceinline__ int dpp_or_0(int v) { return __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS_OF, 0xF, true); }
__device__ __forceinline__ int lane_sums(int v) {
    v += dpp_or_0<0x111, 0xF>(v);
    v += dpp_or_0<0x112, 0xF>(v);
    v += dpp_or_0<0x114, 0xF>(v);
    v += dpp_or_0<0x118, 0xF>(v);
    v += dpp_or_0<0x142, 0xA>(v);
    return v + dpp_or_0<0x143, 0xC>(v);
}
template <int CTRL, int ROWS_OF>
__device__ __forceinline__ float dpp_or_0(float v) {
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, ROWS_OF, 0xF, true));
}
__device__ __forceinline__ float wave_total(float v) {
    v += dpp_or_0<0x111, 0xF>(v);
    v += dpp_or_0<0x112, 0xF>(v);
    v += dpp_or_0<0x114, 0xF>(v);
    v += dpp_or_0<0x118, 0xF>(v);
    v += dpp_or_0<0x142, 0xA>(v);
    v += dpp_or_0<0x143, 0xC>(v);
    return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), 63));
}

// a / b for a below 2^24, b > 0.
__device__ __forceinline__ int small_quotient(int a, int b) {
    int q = (int)((float)a * __builtin_amdgcn_rcpf((float)b));
    if ((int64_t)q * b > a) --q;
    if ((int64_t)(q + 1) * b <= a) ++q;
    return q;
}

// Keys of a part, from `total`, the sum of all tiles' keys: whole UNITs, and no more parts than there are slots for (rounded up
// by more than the sums' and products' roundings).
template <int UNIT>
__device__ __forceinline__ int part_keys(const PagedArgs& a, float total) {
    const float each = total * (float)a.c.H / (float)a.target * 1.0001f + 1.0f;
    return each < 1e9f ? ((int)each + UNIT - 1) / UNIT * UNIT : INT32_MAX;
}
// A sequence's parts a tile, tiles, items, and those of its tiles and items that are split (sums of a list that is not ascending
// stay in range too).
struct SequenceUnits {
    int parts, tiles, items, split_tiles, split_items;
    __device__ __forceinline__ SequenceUnits(const PagedArgs& a, const SequenceWork& w, int chunk) {
        parts = w.span > chunk ? (int)(((int64_t)w.span + chunk - 1) / chunk) : 1;
        tiles = (int)min((int64_t)w.tiles * a.c.H, int64_t(1) << 24);
        items = (int)min((int64_t)tiles * parts, int64_t(1) << 24);
        split_tiles = parts > 1 ? tiles : 0;
        split_items = parts > 1 ? items : 0;
    }
};

// The item (JOIN: the split tile) number id; false if there is none.  A part has at least UNIT keys, in whole UNITs.  PLAN: the
// sums are there.  (Looked at here instead, other registers cost the kernels of few sequences 2 %.)
template <int ROWS, bool MANY, int UNIT, bool JOIN, bool PLAN>
__device__ __forceinline__ bool find_item(const PagedArgs& a, int id, int lane, PagedItem& it) {
    int chunk = INT32_MAX, b0 = 0, end = a.c.B;
    int before = 0, slots = 0;  // items (JOIN: tiles) and split items of the sequences before
    SequenceWork w;
    if constexpr (PLAN) {
        const int blocks = (a.c.B + 63) >> 6;
        const int* items = a.plan + 1 + (JOIN ? blocks : 0);
        const int block = __builtin_amdgcn_readfirstlane(last_at_most(items, blocks, id, lane));
        chunk = __builtin_amdgcn_readfirstlane(a.plan[0]);
        before = __builtin_amdgcn_readfirstlane(items[block]);
        slots = __builtin_amdgcn_readfirstlane(a.plan[1 + 2 * blocks + block]);
        b0 = 64 * block;
        end = b0 + 64;
        w = sequence_work<ROWS, MANY>(a, b0 + lane);
    } else {
        w = sequence_work<ROWS, MANY>(a, lane);
        if (a.target > 0) {
            float total = (float)w.tiles * (float)w.span;
            for (int b = 64; b < a.c.B; b += 64) {
                const SequenceWork x = sequence_work<ROWS, MANY>(a, b + lane);
                total += (float)x.tiles * (float)x.span;
            }
            chunk = __builtin_amdgcn_readfirstlane(part_keys<UNIT>(a, wave_total(total)));
        }
    }
    for (const int first = b0; b0 < end; b0 += 64) {
        if (b0 > first) w = sequence_work<ROWS, MANY>(a, b0 + lane);
        const SequenceUnits u(a, w, chunk);
        const int parts = u.parts, units = JOIN ? u.split_tiles : u.items, split = u.split_items;
        const int incl = lane_sums(units), sincl = lane_sums(split);
        const uint64_t past = __ballot(id - before < incl);
        if (past) {
            const int who = __builtin_ctzll(past);
            it.b = b0 + who;
            const int at = id - before - (__builtin_amdgcn_readlane(incl, who) - __builtin_amdgcn_readlane(units, who));
            it.parts = __builtin_amdgcn_readlane(parts, who);
            const int unit = JOIN || it.parts == 1 ? at : __builtin_amdgcn_readfirstlane(small_quotient(at, it.parts));
            it.part = JOIN ? 0 : at - unit * it.parts;
            const int s0 = slots + __builtin_amdgcn_readlane(sincl, who) - __builtin_amdgcn_readlane(split, who);
            it.slot = s0 + unit * it.parts + it.part;
            // (a prompt's last rows, which see the most keys, begin first, over all heads)
            const int tile = a.by_heads(unit);
            it.h = unit - tile * a.c.H;
            it.tile = __builtin_amdgcn_readlane(w.tiles, who) - 1 - tile;
            it.first = __builtin_amdgcn_readlane(w.first, who);
            it.n = __builtin_amdgcn_readlane(w.n, who);
            it.len = __builtin_amdgcn_readlane(w.len, who);
            const int i0 = a.by_group(it.tile * ROWS), i1 = min(it.n - 1, a.by_group(it.tile * ROWS + ROWS - 1));
            const int end = tile_keys(a, it.len, it.n, i0, i1, it.base, it.far, it.near);
            it.lo = 0;
            it.hi = end;
            if (it.parts > 1) {
                const int sp = __builtin_amdgcn_readlane(w.span, who);
                const int each = ((sp + it.parts - 1) / it.parts + UNIT - 1) / UNIT * UNIT;
                const int64_t p0 = (int64_t)it.part * each;
                it.lo = (int)min(p0, (int64_t)end);
                if (it.part < it.parts - 1) it.hi = (int)min(p0 + each, (int64_t)end);
            }
            return JOIN || it.parts == 1 || it.slot < a.slots;  // (at most 2 target of them: vedic_capi.hip)
        }
        before += __builtin_amdgcn_readlane(incl, 63);
        slots = min(slots + __builtin_amdgcn_readlane(sincl, 63), 1 << 29);
    }
    return false;
}

// Bits j < 64: key + j is a multiple of the stride.
__device__ __forceinline__ uint64_t stride_bits(int key, int stride) {
    uint64_t bits = 0;
    const int past = key % stride;
    for (int j = past ? stride - past : 0; j < 64; j += stride) bits |= uint64_t(1) << j;
    return bits;
}

// Bits [from, upto) and those of `more` below upto.
__device__ __forceinline__ uint64_t place_bits(int from, int upto, uint64_t more) {
    const uint64_t below = upto <= 0 ? 0 : upto >= 64 ? ~uint64_t(0) : (uint64_t(1) << upto) - 1;
    const uint64_t above = from <= 0 ? ~uint64_t(0) : from >= 64 ? 0 : ~uint64_t(0) << from;
    return below & (above | more);
}

// Whether the row at position pos sees key t < len.
__device__ __forceinline__ bool sees(const PagedArgs& a, int pos, int t) {
    if (a.causal && t > pos) return false;
    return a.window == 0 || t >= pos - a.window || (a.stride > 0 && t % a.stride == 0);
}

// The value d of a cache row.
template <bool I4>
__device__ __forceinline__ float cache_value(const char* row, int D, int d) {
    if constexpr (!I4) return (float)reinterpret_cast<const _Float16*>(row)[d];
    half2_t s, m;
    four_bit_pair(reinterpret_cast<const uint32_t*>(row + D / 2)[d >> 5], s, m);
    const half8_t v = four_bit_values(reinterpret_cast<const uint32_t*>(row)[d >> 3], s, m);
    float r = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) r = (d & 7) == i ? (float)v[i] : r;
    return r;
}

// One row's part by one wave, key by key (KEYS on their way at a time): what a key outside the row's mask
// holds never enters a sum.  For rows whose weights are fine and whose outputs came out infinite or NaN: in a product of
// tiles the zero weight of an unseen key times an infinity is NaN.  (A row with a score that is NaN or +infinity has a
// sum of weights that is NaN, and is NaN.)  o: values lane, lane + 64, ..
template <int DP, bool I4>
__device__ __forceinline__ void slow_row(const PagedArgs& a, const PagedItem& it, int pos, const _Float16* q, int lane,
                                      float (&o)[DP / 64], float& m, float& l) {
    constexpr int N = DP / 64, KEYS = I4 ? 2 : 8;  // (more of four bits cost the kernels that hold this a wave a SIMD)
    float qv[N];
#pragma unroll
    for (int j = 0; j < N; ++j) {
        const int d = lane + 64 * j;
        qv[j] = d < a.c.D ? (float)q[d] : 0.0f;
        o[j] = 0.0f;
    }
    m = kNoScore;
    l = 0.0f;
    for (int p0 = it.lo; p0 < it.hi; p0 += KEYS) {
        bool seen[KEYS];
        float x[KEYS], v[KEYS][N], mn = m;
#pragma unroll
        for (int e = 0; e < KEYS; ++e) {
            const int place = min(p0 + e, it.hi - 1), t = key_at(a, it, place);
            seen[e] = p0 + e < it.hi && !(place >= it.far && place < it.near) && sees(a, pos, t);
            const int64_t at = a.c.row_offset(it.b, t) + (int64_t)it.h * a.c.head;
            x[e] = 0.0f;
#pragma unroll
            for (int j = 0; j < N; ++j) {
                const int d = min(lane + 64 * j, a.c.D - 1);
                x[e] += lane + 64 * j < a.c.D ? qv[j] * cache_value<I4>(a.c.k + at, a.c.D, d) : 0.0f;
                v[e][j] = cache_value<I4>(a.c.v + at, a.c.D, d);
            }
        }
#pragma unroll
        for (int e = 0; e < KEYS; ++e) {
#pragma unroll
            for (int d = 32; d > 0; d >>= 1) x[e] += __shfl_xor(x[e], d);
            x[e] = seen[e] ? x[e] * a.sign : kNoScore;
            mn = __builtin_fmaxf(mn, x[e]);
        }
        const float mu = mn == kNoScore ? 0.0f : mn, f = exp2_fast((m - mu) * a.scale);
        m = mn;
        l *= f;
#pragma unroll
        for (int j = 0; j < N; ++j) o[j] *= f;
#pragma unroll
        for (int e = 0; e < KEYS; ++e) {
            const float p = exp2_fast(__builtin_fmaf(x[e] - mu, a.scale, kWeightBits));
            l += p;
#pragma unroll
            for (int j = 0; j < N; ++j) o[j] += seen[e] ? p * v[e][j] : 0.0f;
        }
    }
}

typedef _Float16 paged_half4_t __attribute__((ext_vector_type(4)));

// A row's 1 / l and log-sum-exp from its largest score m and its sum l.  A sum of 0: the row at position pos sees no key (0 and
// +infinity), or only keys whose scores are -infinity (nothing over nothing: NaN).
__device__ __forceinline__ float empty_row(const PagedArgs& a, int pos, int len, float unseen) {
    return (a.causal ? pos >= 0 : len > 0) ? __builtin_nanf("") : unseen;
}
__device__ __forceinline__ float inverse_of(const PagedArgs& a, int pos, int len, float l) {
    return l > 0.0f || l != l ? 1.0f / l : empty_row(a, pos, len, 0.0f);
}
__device__ __forceinline__ float lse_of(const PagedArgs& a, int pos, int len, float m, float l) {
    return l > 0.0f || l != l ? (__builtin_fmaf(m, a.scale, -kWeightBits) + __builtin_log2f(l)) * 0.6931471805599453f
                              : empty_row(a, pos, len, __builtin_inff());
}

namespace {

// The sums of 32 rows from `base` on, O^T in 32 x 32 blocks (lane l: row base + l mod 32; element 4 e + f of block
// d: value 32 d + 8 e + 4 (l / 32) + f), to the output or to the partial results from row s0 on.
template <int DP, bool I4>
__device__ __forceinline__ void finish_rows(const PagedArgs& a, const PagedItem& it, int base, int64_t s0,
                                            const float16_t (&acc)[DP / 32], float m, float l, int lane) {
    constexpr int DT = DP / 32;
    const int r = lane & 31, h = lane >> 5, rho = base + r, i = a.by_group(rho);
    const bool mine = i < it.n;
    const int64_t tok = it.first + i;
    const int head = it.h * a.G + rho - i * a.G, pos = it.len - it.n + i;
    l += __shfl_xor(l, 32);
    bool fine = true;
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int e = 0; e < 16; ++e) fine = fine && __builtin_fabsf(acc[d][e]) < __builtin_inff();
    fine |= l != l;
    if (mine) {
        const float inv = inverse_of(a, pos, it.len, l);
        if (it.parts == 1) {
            _Float16* out = a.out + tok * a.o_token + (int64_t)head * a.o_head;
#pragma unroll
            for (int d = 0; d < DT; ++d)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int at = 32 * d + 8 * e + 4 * h;
                    const paged_half4_t v = {(_Float16)(acc[d][4 * e] * inv), (_Float16)(acc[d][4 * e + 1] * inv),
                                            (_Float16)(acc[d][4 * e + 2] * inv), (_Float16)(acc[d][4 * e + 3] * inv)};
                    if (at < a.c.D) *reinterpret_cast<paged_half4_t*>(out + at) = v;
                }
            if (a.lse && h == 0) a.lse[tok * a.Hq + head] = lse_of(a, pos, it.len, m, l);
        } else {
            float* po = a.part_o + (s0 + r) * a.c.D;
#pragma unroll
            for (int d = 0; d < DT; ++d)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int at = 32 * d + 8 * e + 4 * h;
                    const float4_t v = {acc[d][4 * e], acc[d][4 * e + 1], acc[d][4 * e + 2], acc[d][4 * e + 3]};
                    if (at < a.c.D) *reinterpret_cast<float4_t*>(po + at) = v;
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
        const int brho = base + w, bi = a.by_group(brho), bh = it.h * a.G + brho - bi * a.G;
        const int bpos = it.len - it.n + bi;
        const int64_t bt = it.first + bi;
        float ov[DP / 64], bm, bl;
        slow_row<DP, I4>(a, it, bpos, a.q + bt * a.q_token + (int64_t)bh * a.q_head, lane, ov,
                         bm, bl);
        const float bin = inverse_of(a, bpos, it.len, bl);
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // (the stores above come first)
#pragma unroll
        for (int j = 0; j < DP / 64; ++j) {
            const int d = lane + 64 * j;
            if (d >= a.c.D) continue;
            if (it.parts == 1) a.out[bt * a.o_token + (int64_t)bh * a.o_head + d] = (_Float16)(ov[j] * bin);
            else a.part_o[(s0 + w) * a.c.D + d] = ov[j];
        }
        if (lane == 0) {
            if (it.parts == 1) {
                if (a.lse) a.lse[bt * a.Hq + bh] = lse_of(a, bpos, it.len, bm, bl);
            } else {
                a.part_ml[2 * (s0 + w)] = bm;
                a.part_ml[2 * (s0 + w) + 1] = bl;
            }
        }
    }
}

// Sums o, l relative to a maximum m, and others' o2, l2, m2, as one.
__device__ __forceinline__ void join_sums(float scale, float4_t& o, float& m, float& l, float4_t o2, float m2, float l2) {
    const float top = __builtin_fmaxf(m, m2), mu = top == kNoScore ? 0.0f : top;
    const float f = exp2_fast((m - mu) * scale), f2 = exp2_fast((m2 - mu) * scale);
    m = top;
    l = l * f + l2 * f2;
    o = o * f + o2 * f2;
}

// The parts of a tile joined.  A lane has four columns of a row's share of the parts: D / 4 lanes a share, a wave's
// shares of one row (`per` rows a workgroup, a wave each in turn), or with WHOLE a workgroup's.
template <int ROWS, bool MANY, int UNIT, bool WHOLE, bool PLAN>
__global__ void __launch_bounds__(256) paged_join_kernel(PagedArgs a, int per) {
    __shared__ float4_t wave_o[WHOLE ? 4 : 1][64];
    __shared__ float wave_ml[WHOLE ? 4 : 1][2];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    PagedItem it;
    if (!find_item<ROWS, MANY, UNIT, true, PLAN>(a, blockIdx.x, lane, it)) return;
    if ((int64_t)it.slot + it.parts > a.slots) return;
    const int D = a.c.D, cols = D / 4;
    const int lanes = D <= 64 ? 16 : D <= 128 ? 32 : 64;  // of a share
    const int shares = (WHOLE ? 4 : 1) * (64 / lanes), share = (WHOLE ? wave * (64 / lanes) : 0) + lane / lanes, c = lane % lanes;
    for (int r = blockIdx.y * per + (WHOLE ? 0 : wave); r < (int)(blockIdx.y + 1) * per; r += WHOLE ? 1 : 4) {
        const int rho = it.tile * ROWS + r, i = a.by_group(rho);
        if (i >= it.n) return;
        const int64_t s0 = (int64_t)it.slot * ROWS + r;
        float4_t o = {0.0f, 0.0f, 0.0f, 0.0f};
        float M = kNoScore, l = 0.0f;
        // (a running maximum: all loads of a round are on their way together)
        for (int p0 = share; p0 < it.parts; p0 += 8 * shares) {
            float mp[8], lp[8];
            float4_t v[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int64_t s = s0 + (int64_t)min(p0 + j * shares, it.parts - 1) * ROWS;
                mp[j] = a.part_ml[2 * s];
                lp[j] = a.part_ml[2 * s + 1];
                v[j] = *reinterpret_cast<const float4_t*>(a.part_o + s * D + 4 * min(c, cols - 1));
            }
            float top = M;
#pragma unroll
            for (int j = 0; j < 8; ++j) top = __builtin_fmaxf(top, mp[j]);
            const float mu = top == kNoScore ? 0.0f : top, g = exp2_fast((M - mu) * a.scale);
            M = top;
            l *= g;
            o *= g;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float f = exp2_fast((mp[j] - mu) * a.scale);
                if (p0 + j * shares < it.parts && !(lp[j] == 0.0f)) {  // (a part without keys has nothing to add)
                    l += lp[j] * f;
                    o += v[j] * f;
                }
            }
        }
        for (int d = lanes; d < 64; d <<= 1) {
            const float4_t oo = {__shfl_xor(o[0], d), __shfl_xor(o[1], d), __shfl_xor(o[2], d), __shfl_xor(o[3], d)};
            join_sums(a.scale, o, M, l, oo, __shfl_xor(M, d), __shfl_xor(l, d));
        }
        if constexpr (WHOLE) {
            wave_o[wave][lane] = o;
            wave_ml[wave][0] = M;
            wave_ml[wave][1] = l;
            __syncthreads();
            if (wave > 0) return;  // (per is 1)
#pragma unroll
            for (int x = 1; x < 4; ++x) join_sums(a.scale, o, M, l, wave_o[x][lane], wave_ml[x][0], wave_ml[x][1]);
        }
        const int head = it.h * a.G + rho - i * a.G, pos = it.len - it.n + i;
        const int64_t t = it.first + i;
        if (lane < lanes && c < cols) {
            const float inv = inverse_of(a, pos, it.len, l);
            const paged_half4_t v = {(_Float16)(o[0] * inv), (_Float16)(o[1] * inv), (_Float16)(o[2] * inv), (_Float16)(o[3] * inv)};
            *reinterpret_cast<paged_half4_t*>(a.out + t * a.o_token + (int64_t)head * a.o_head + 4 * c) = v;
        }
        if (a.lse && lane == 0) a.lse[t * a.Hq + head] = lse_of(a, pos, it.len, M, l);
    }
}

}  // namespace

}  // namespace vedic
