// vedic_cache.hpp -- a paged cache of keys and values, as the kernels that write it
// (vedic_cache.hip) and read it (vedic_paged.hpp) see it, and the four-bit format that
// the cache and the weights of vedic_w4.hip and vedic_w4_tile.hip share.
#pragma once

#include "vedic_common.hpp"

namespace vedic {

typedef _Float16 half2_t __attribute__((ext_vector_type(2)));
typedef uint32_t u32x2_t __attribute__((ext_vector_type(2)));
// 16 bytes at a 4-byte-aligned address (gfx950 loads and stores them as one access).
typedef uint32_t u32x4_a4_t __attribute__((ext_vector_type(4), aligned(4)));

// Positions stay below this.
constexpr int kMaxTokens = 1 << 30;

// Quotients of numbers below 2^30: n / d = n * magic >> shift.
struct Divider {
    uint32_t magic;
    int shift;
    __device__ __forceinline__ int operator()(int n) const { return (int)((uint64_t)(uint32_t)n * magic >> shift); }
};
inline Divider divider(int d) {
    int l = 0;
    while ((int64_t(1) << l) < d) ++l;
    return Divider{(uint32_t)((uint64_t(1) << (30 + l)) / d + 1), 30 + l};
}

struct KvView {
    char* k;
    char* v;
    int64_t page, head, token;  // strides in bytes
    int pages, ps, H, D;
    const int* table;  // [B x ldt]
    int64_t ldt;
    int tcols;
    const int* lens;     // [B]
    const int* q_start;  // [B + 1], or null: row b is sequence b's only new one
    int B, T;
    Divider by_page;  // of positions by ps

    __device__ __forceinline__ int page_of(int pos) const { return by_page(pos); }
    // Tokens of sequence b, as many as its pages can hold at most.
    __device__ __forceinline__ int len_of(int b) const {
        const int64_t cap = (int64_t)tcols * ps;
        const int most = cap < kMaxTokens ? (int)cap : kMaxTokens - 1;
        return max(0, min(lens[b], most));
    }
    // First new row and count of new rows of sequence b (clamped to 0 .. T).
    __device__ __forceinline__ void rows_of(int b, int& first, int& n) const {
        if (q_start == nullptr) {
            first = b;
            n = b < T ? 1 : 0;
            return;
        }
        first = max(0, min(q_start[b], T));
        n = max(0, min(q_start[b + 1], T) - first);
    }
    // Byte offset of the row of position pos < len (head 0); a page that is none counts as page 0.
    __device__ __forceinline__ int64_t row_offset(int b, int pos) const {
        const int t = page_of(pos);
        int p = table[b * ldt + t];
        if ((unsigned)p >= (unsigned)pages) p = 0;
        return p * page + (pos - t * ps) * token;
    }
};

// The last of n ascending values that is at most id (the first one is).
__device__ __forceinline__ int last_at_most(const int* v, int n, int id, int lane) {
    int lo = 0;
    for (int span = n; span > 1;) {
        const int step = (span + 63) >> 6, at = lane * step;
        const uint64_t ok = __ballot(at < span && v[lo + min(at, span - 1)] <= id);
        const int past = (63 - __builtin_clzll(ok | 1)) * step;
        lo += past;
        span = min(step, span - past);
    }
    return lo;
}

// Four-bit words: 32 bits hold eight consecutive values, value 2 i in bits 4 i .. 4 i + 3 and
// value 2 i + 1 in bits 16 + 4 i ..; code n of a group with the binary16 pair (s, m) stands
// for binary16(s n + m), one rounding.  n | 0x6400 is the binary16 1024 + n, and a nibble at
// bits 4 .. 7 under 0x5400 is 64 + n, so that a pair of values takes one and-or, one exact
// subtraction and one fused multiply-add.
// (A VOP3 instruction takes no 32-bit literal here and one scalar register: the masks are kept in scalar
// registers and the bases in vector registers, or each and-or would be two instructions.)
struct FourBits {
    uint32_t low, mid;     // 0x000F000F, 0x00F000F0 (scalar)
    uint32_t k1024, k64;   // 0x6400, 0x5400 twice (vector)
    __device__ __forceinline__ FourBits() : low(0x000F000Fu), mid(0x00F000F0u), k1024(0x64006400u), k64(0x54005400u) {
        asm volatile("" : "+s"(low), "+s"(mid), "+v"(k1024), "+v"(k64));
    }
    __device__ __forceinline__ half8_t operator()(uint32_t w, half2_t s, half2_t m) const {
        const half2_t m1024 = {(_Float16)1024.0f, (_Float16)1024.0f}, m64 = {(_Float16)64.0f, (_Float16)64.0f};
        const uint32_t w8 = w >> 8;
        const half2_t n0 = __builtin_bit_cast(half2_t, (w & low) | k1024) - m1024;
        const half2_t n1 = __builtin_bit_cast(half2_t, (w & mid) | k64) - m64;
        const half2_t n2 = __builtin_bit_cast(half2_t, (w8 & low) | k1024) - m1024;
        const half2_t n3 = __builtin_bit_cast(half2_t, (w8 & mid) | k64) - m64;
        union {
            half2_t p[4];
            half8_t h;
        } u;
        u.p[0] = __builtin_elementwise_fma(s, n0, m);
        u.p[1] = __builtin_elementwise_fma(s, n1, m);
        u.p[2] = __builtin_elementwise_fma(s, n2, m);
        u.p[3] = __builtin_elementwise_fma(s, n3, m);
        return u.h;
    }
};
__device__ __forceinline__ half8_t four_bit_values(uint32_t w, half2_t s, half2_t m) { return FourBits()(w, s, m); }
__device__ __forceinline__ void four_bit_pair(uint32_t sm, half2_t& s, half2_t& m) {
    const half2_t p = __builtin_bit_cast(half2_t, sm);
    s = half2_t{p[0], p[0]};
    m = half2_t{p[1], p[1]};
}

// store16_hold of eight binary16 values.
__device__ __forceinline__ void store_half8(void* p, half8_t h) {
    store16_hold(static_cast<float*>(p), __builtin_bit_cast(float4_t, h));
}

// A value that no multiply-add is formed across (the library is compiled with
// -ffp-contract=fast, which fuses a product into the sum that takes it).
__device__ __forceinline__ float rounded(float x) {
    asm volatile("" : "+v"(x));
    return x;
}

// The pair (s, m) of a group whose least and largest binary16 values are lo and hi.
__device__ __forceinline__ uint32_t four_bit_scale(float lo, float hi, bool bad) {
    if (bad) return 0x7E007E00u;  // NaN, NaN
    const half2_t sm = {(_Float16)((hi - lo) / 15.0f), (_Float16)lo};
    return __builtin_bit_cast(uint32_t, sm);
}
// The word of eight values: round((x - lo) / s).  A product with 1 / s is off the quotient by less than 2^-18 at quotients
// up to 16 (two roundings of 2^-24 and the division's own); only where that could decide the rounding is it divided.
__device__ __forceinline__ uint32_t four_bit_word(const float (&x)[8], float s, float lo) {
    if (!(s > 0.0f)) return 0u;
    const float inv = 1.0f / s;
    float n[8];
    bool near = false;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float q = (x[i] - lo) * inv;
        n[i] = __builtin_rintf(q);
        near |= __builtin_fabsf(q - n[i]) > 0.5f - 0x1p-17f;
    }
    if (near) {
#pragma unroll
        for (int i = 0; i < 8; ++i) n[i] = __builtin_rintf((x[i] - lo) / s);
    }
    uint32_t w = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) w |= (uint32_t)__builtin_fminf(__builtin_fmaxf(n[i], 0.0f), 15.0f) << (4 * (i >> 1) + 16 * (i & 1));
    return w;
}

struct KvAppendArgs {
    KvView c;
    bool i4, f32;  // cache format, type of q, k, v
    const void* q;
    const void* k;
    const void* v;
    int64_t q_token, q_head, k_token, k_head, v_token, v_head, o_token, o_head;  // strides in values
    _Float16* q_out;
    int Hq;
    const float* rope;  // [rope_rows x rot]: cosines, then sines
    int rope_rows, rot;
    bool inter;
};
hipError_t launch_kv_append(const KvAppendArgs& a, hipStream_t s);
// k, v: [T x H x D] binary16, either may be null.
hipError_t launch_kv_read(const KvView& c, bool i4, _Float16* k, _Float16* v, hipStream_t s);

// Attention of the new rows over the cache.
struct PagedArgs {
    KvView c;
    const _Float16* q;
    _Float16* out;
    float* lse;  // [T x Hq] or null
    int64_t q_token, q_head, o_token, o_head;  // strides in values
    int Hq, G;
    Divider by_group, by_heads;  // of rows by G, of units by the key heads
    float scale;  // |scale| log2(e), > 0
    float sign;   // of the scale: q is multiplied by it
    int causal, window, stride;
    // set by the rules in vedic_capi.hip: `target` workgroups' worth of keys per item
    // (0: items are not split), and the partial results of split items
    int64_t target;
    // null, or of many sequences the keys of a part, and for each 64 of them the items, split tiles and split
    // items of those before (launch_paged_plan)
    const int* plan;
    int few_most;  // sequences of at most so many rows (new rows x G) are the few-row kernel's
    int slots;
    float* part_o;   // [slots x rows x D]
    float* part_ml;  // [slots x rows x 2]: largest score, sum
};
// Rows of a tile, and what parts of a tile's keys are whole multiples of.
constexpr int kFewRows = 16, kManyRows = 128;
constexpr int kFewUnit = 128, kManyUnit = 256;
// Ints of a plan, and the plan of one kind of rows.
inline int64_t paged_plan_ints(int sequences) { return 1 + 3 * (((int64_t)sequences + 63) / 64); }
hipError_t launch_paged_plan(const PagedArgs& a, bool many, int* plan, hipStream_t s);
hipError_t launch_paged_few_f16(const PagedArgs& a, hipStream_t s);
hipError_t launch_paged_few_i4(const PagedArgs& a, hipStream_t s);
hipError_t launch_paged_many_f16(const PagedArgs& a, hipStream_t s);
hipError_t launch_paged_many_i4(const PagedArgs& a, hipStream_t s);

}  // namespace vedic
