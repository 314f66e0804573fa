// vedic_cache.hip -- new tokens' keys and values into a paged cache, turned by their
// positions on the way, and rows of the cache back as binary16.
//
// Rotation of a row x at position p, angle index i < rot / 2, (a, b) = (x_i, x_(i + rot/2)) or
// (x_2i, x_(2i+1)):   (a, b) -> (a cos - b sin, b cos + a sin),
// the cosines and sines of p from a table of fp32 values (their angles need more bits than
// fp32 has at far positions).  Each product and the sum are rounded to fp32, the result
// once more to binary16.  Rows of four bits: 32 values share (s, m) = (binary16((hi - lo) / 15), lo)
// of their binary16 values, code = round((x - m) / s).
//
// A thread takes eight consecutive values of a row: it reads them, their partners (a neighbouring
// thread's own: cached) and the angles, and writes 16 bytes, or a word; the four threads of a group of 32
// exchange its least and largest value by DPP.  Memory bounds it, and what comes before the angles can
// be asked for: a workgroup has one token, so that many are at it (8192 tokens of 48 heads of 64 from fp32, cold
// caches: 36 us, 4.3 TB/s; with four tokens a workgroup 46); the sequence of a token is the one whose rows it lies among
// (a ballot, after a search by 64ths among more than 64: 4096 tokens of as many sequences, 16 heads of 64, 50 us by a walk, 19 so).
#include "vedic_cache.hpp"

namespace vedic {

namespace {

constexpr int kThreads = 256;

typedef float float8_t __attribute__((ext_vector_type(8)));

// The sequence of new row t and its position (-1: none).  A lane looks at a sequence's rows and length at once: all
// comes from one round of loads.
__device__ __forceinline__ void find_row(const KvView& c, int t, int lane, int& seq, int& pos) {
    seq = 0;
    pos = -1;
    if (c.q_start == nullptr) {
        seq = t;
        pos = __builtin_amdgcn_readfirstlane(c.len_of(t)) - 1;
        return;
    }
    // (of many sequences the last that begins at the row or before it: empty ones begin where the next one does)
    const int b0 = c.B > 64 ? last_at_most(c.q_start, c.B, t, lane) : 0, b = min(b0 + lane, c.B - 1);
    int first, n;
    c.rows_of(b, first, n);
    const int at = c.len_of(b) - n - first;  // the row's position less t
    const uint64_t who = __ballot(b0 + lane < c.B && t >= first && t < first + n);
    if (who == 0) return;
    seq = b0 + __builtin_ctzll(who);
    pos = t + __builtin_amdgcn_readlane(at, __builtin_ctzll(who));
}

template <bool F32>
__device__ __forceinline__ void load8(const void* base, int64_t at, bool vec, float (&x)[8]) {
    if constexpr (F32) {
        const float* p = static_cast<const float*>(base) + at;
        if (vec) {
            const float4_t a = reinterpret_cast<const float4_t*>(p)[0], b = reinterpret_cast<const float4_t*>(p)[1];
#pragma unroll
            for (int i = 0; i < 4; ++i) x[i] = a[i], x[4 + i] = b[i];
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = p[i];
        }
    } else {
        const _Float16* p = static_cast<const _Float16*>(base) + at;
        if (vec) {
            const half8_t a = *reinterpret_cast<const half8_t*>(p);
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = (float)a[i];
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = (float)p[i];
        }
    }
}
template <bool F32>
__device__ __forceinline__ float load1(const void* base, int64_t at) {
    if constexpr (F32) return static_cast<const float*>(base)[at];
    else return (float)static_cast<const _Float16*>(base)[at];
}

// x: the eight values e0 .. e0 + 7 of the row at `row`, turned by the angles of table row `cs`.
// VEC: the partners (half the rotated width away) and the angles are whole 16-byte pieces.
template <bool F32, bool VEC>
__device__ __forceinline__ void rotate8(const KvAppendArgs& a, const void* src, int64_t row, int e0, const float* cs,
                                        float (&x)[8]) {
    const int half = a.rot >> 1;
    float c[8], s[8], o[8];
    if (a.inter) {
        float cc[4], ss[4];
        if constexpr (VEC) {  // (the rotated values are whole sixteens)
            const float4_t c4 = *reinterpret_cast<const float4_t*>(cs + (e0 >> 1)), s4 = *reinterpret_cast<const float4_t*>(cs + half + (e0 >> 1));
#pragma unroll
            for (int i = 0; i < 4; ++i) cc[i] = c4[i], ss[i] = s4[i];
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int j = (e0 >> 1) + i;
                cc[i] = j < half ? cs[j] : 1.0f;
                ss[i] = j < half ? cs[half + j] : 0.0f;
            }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            c[2 * i] = c[2 * i + 1] = cc[i];
            s[2 * i] = -ss[i];
            s[2 * i + 1] = ss[i];
            o[2 * i] = x[2 * i + 1];
            o[2 * i + 1] = x[2 * i];
        }
    } else if constexpr (VEC) {
        const bool second = e0 >= half;
        const int j = second ? e0 - half : e0;
        load8<F32>(src, row + (second ? j : e0 + half), true, o);
        const float4_t c0 = *reinterpret_cast<const float4_t*>(cs + j), c1 = *reinterpret_cast<const float4_t*>(cs + j + 4);
        const float4_t s0 = *reinterpret_cast<const float4_t*>(cs + half + j),
                       s1 = *reinterpret_cast<const float4_t*>(cs + half + j + 4);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            c[i] = i < 4 ? c0[i & 3] : c1[i & 3];
            const float ss = i < 4 ? s0[i & 3] : s1[i & 3];
            s[i] = second ? ss : -ss;
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int e = e0 + i;
            const bool in = e < a.rot, second = e >= half;
            const int j = second ? e - half : e;
            o[i] = in ? load1<F32>(src, row + (second ? j : e + half)) : 0.0f;
            c[i] = in ? cs[j] : 1.0f;
            const float ss = in ? cs[half + j] : 0.0f;
            s[i] = second ? ss : -ss;
        }
    }
    // (a cos + b (-sin) is a cos - b sin: the negation is exact)
#pragma unroll
    for (int i = 0; i < 8; ++i)
        if (e0 + i < a.rot) x[i] = rounded(x[i] * c[i]) + rounded(o[i] * s[i]);
}

template <int CTRL>
__device__ __forceinline__ float quad_swap(float v) {
    return __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), CTRL, 0xF, 0xF, true));
}

// Eight values of a cache row, as binary16 or four bits; all four threads of a group of 32 call it together.
__device__ __forceinline__ void store_row(char* row, bool i4, int D, int e0, const float (&x)[8], bool write) {
    half8_t h;
#pragma unroll
    for (int i = 0; i < 8; ++i) h[i] = (_Float16)x[i];
    if (!i4) {
        if (write) store_half8(row + 2 * e0, h);
        return;
    }
    float y[8], lo = __builtin_inff(), hi = -__builtin_inff();
    bool bad = false;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        y[i] = (float)h[i];
        bad |= !(__builtin_fabsf(y[i]) < __builtin_inff());
        lo = __builtin_fminf(lo, y[i]);
        hi = __builtin_fmaxf(hi, y[i]);
    }
    lo = bad ? -__builtin_inff() : lo;  // (one in the group is enough: the pair is NaN)
    lo = __builtin_fminf(lo, quad_swap<0xB1>(lo));  // lanes 1 0 3 2
    hi = __builtin_fmaxf(hi, quad_swap<0xB1>(hi));
    lo = __builtin_fminf(lo, quad_swap<0x4E>(lo));  // lanes 2 3 0 1
    hi = __builtin_fmaxf(hi, quad_swap<0x4E>(hi));
    const uint32_t sm = four_bit_scale(lo, hi, lo == -__builtin_inff());
    const float s = (float)__builtin_bit_cast(half2_t, sm)[0];
    if (!write) return;
    *reinterpret_cast<uint32_t*>(row + e0 / 2) = four_bit_word(y, s, lo);
    if ((e0 & 31) == 0) *reinterpret_cast<uint32_t*>(row + D / 2 + e0 / 8) = sm;
}

// A workgroup per token and 256 of its (Hq + 2 H) D / 8 eights.
template <bool F32>
__global__ void __launch_bounds__(kThreads) kv_append_kernel(KvAppendArgs a, int items, bool vec_in, bool vec_rot) {
    const KvView& c = a.c;
    const int t = blockIdx.x, item = blockIdx.y * kThreads + threadIdx.x;
    const int eights = c.D >> 3;
    const bool mine = item < items;
    const int head = mine ? item / eights : 0, e0 = mine ? 8 * (item - head * eights) : 0;
    const int kind = head < a.Hq ? 0 : head < a.Hq + c.H ? 1 : 2;
    const int hk = kind == 0 ? head : kind == 1 ? head - a.Hq : head - a.Hq - c.H;
    const void* src = kind == 0 ? a.q : kind == 1 ? a.k : a.v;
    const int64_t row = hk * (kind == 0 ? a.q_head : kind == 1 ? a.k_head : a.v_head) +
                        t * (kind == 0 ? a.q_token : kind == 1 ? a.k_token : a.v_token);
    float x[8];
    load8<F32>(src, row + e0, vec_in, x);
    int seq, pos;
    find_row(c, t, threadIdx.x & 63, seq, pos);
    if (pos < 0) return;
    const int tp = c.page_of(pos);
    const int page = c.table[seq * c.ldt + tp];
    if (kind < 2 && e0 < a.rot) {
        const float* cs = a.rope + (int64_t)min(pos, a.rope_rows - 1) * a.rot;
        if (vec_rot) rotate8<F32, true>(a, src, row, e0, cs, x);
        else rotate8<F32, false>(a, src, row, e0, cs, x);
    }
    if (kind == 0) {
        if (!mine) return;
        half8_t h;
#pragma unroll
        for (int j = 0; j < 8; ++j) h[j] = (_Float16)x[j];
        store_half8(a.q_out + t * a.o_token + hk * a.o_head + e0, h);
    } else {
        char* to = (kind == 1 ? c.k : c.v) + (int64_t)page * c.page + (int64_t)hk * c.head + (int64_t)(pos - tp * c.ps) * c.token;
        store_row(to, a.i4, c.D, e0, x, mine && (unsigned)page < (unsigned)c.pages);
    }
}

// One thread per eight values of K and of V.
__global__ void __launch_bounds__(kThreads) kv_read_kernel(KvView c, bool i4, _Float16* k, _Float16* v, int items) {
    const int t = blockIdx.x, item = blockIdx.y * kThreads + threadIdx.x;
    int seq, pos;
    find_row(c, t, threadIdx.x & 63, seq, pos);
    if (pos < 0 || item >= items) return;
    const int eights = c.D >> 3, head = item / eights, e0 = 8 * (item - head * eights);
    const int64_t at = c.row_offset(seq, pos) + (int64_t)head * c.head;
    const int64_t to = ((int64_t)t * c.H + head) * c.D + e0;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        _Float16* out = j ? v : k;
        if (!out) continue;
        const char* row = (j ? c.v : c.k) + at;
        half8_t h;
        if (i4) {
            half2_t s, m;
            four_bit_pair(*reinterpret_cast<const uint32_t*>(row + c.D / 2 + (e0 >> 5) * 4), s, m);
            h = four_bit_values(*reinterpret_cast<const uint32_t*>(row + e0 / 2), s, m);
        } else {
            h = *reinterpret_cast<const half8_t*>(row + 2 * e0);
        }
        store_half8(out + to, h);
    }
}

bool aligned(const void* p, int64_t a, int64_t b, int64_t bytes) {
    return (((uintptr_t)p | (uintptr_t)a | (uintptr_t)b) & (bytes - 1)) == 0;
}

}  // namespace

hipError_t launch_kv_append(const KvAppendArgs& a, hipStream_t s) {
    const KvView& c = a.c;
    const int es = a.f32 ? 4 : 2;
    bool vec = aligned(a.k, a.k_token * es, a.k_head * es, 16) && aligned(a.v, a.v_token * es, a.v_head * es, 16);
    if (a.Hq > 0) vec = vec && aligned(a.q, a.q_token * es, a.q_head * es, 16);
    const bool vrot = vec && a.rot % 16 == 0 && aligned(a.rope, 0, 0, 16);
    const int items = (a.Hq + 2 * c.H) * (c.D / 8);
    const unsigned y = (unsigned)((items + kThreads - 1) / kThreads);
    const dim3 grid((unsigned)c.T, y);
    if (a.f32) kv_append_kernel<true><<<grid, kThreads, 0, s>>>(a, items, vec, vrot);
    else kv_append_kernel<false><<<grid, kThreads, 0, s>>>(a, items, vec, vrot);
    return hipGetLastError();
}

hipError_t launch_kv_read(const KvView& c, bool i4, _Float16* k, _Float16* v, hipStream_t s) {
    const int items = c.H * (c.D / 8);
    kv_read_kernel<<<dim3((unsigned)c.T, (unsigned)((items + kThreads - 1) / kThreads)), kThreads, 0, s>>>(c, i4, k, v,
                                                                                                           items);
    return hipGetLastError();
}

}  // namespace vedic
