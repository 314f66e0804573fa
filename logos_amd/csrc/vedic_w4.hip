// vedic_w4.hip -- Y[M x N] = epi(X[M x K] . W[K x N]) with W held in four bits, for few rows;
// the same weights expanded to binary16 for the tiled kernels; and weights put into that form.
//
// Few rows (decoding): the product reads N K / 2 bytes and is bound by them.  A lane of
// v_mfma_f32_16x16x32_f16 takes eight values of one column of W: it loads 16 bytes of its column, 32
// consecutive codes of one group with one pair (s, m), expands a word at a time (13
// instructions for eight values) and multiplies; lane group g has the codes 128 i + 32 g .. + 31, and
// takes the same values of its row of X, straight from the cache.  The waves of a workgroup take
// 128 values of K in turn and add up their 16 x 16 blocks through LDS in a fixed order, so no
// second launch and no workspace are needed.  Column blocks a wave: one for a row or two
// (many workgroups), more with more rows, so that the rows of X are not read more often than
// the codes.
//
// More rows: the expanded weight (N K 2 bytes written and read once more) and the binary16
// tiles, in slabs of columns.
#include "vedic_w4.hpp"

namespace vedic {

namespace {

template <bool X32>
__device__ __forceinline__ half8_t load_x(const void* X, int64_t row, int k, int K, bool vec) {
    half8_t h = {};
    if constexpr (X32) {
        const float* p = static_cast<const float*>(X) + row + k;
        if (vec) {
            if (k < K) {
                const float4_t a = reinterpret_cast<const float4_t*>(p)[0], b = reinterpret_cast<const float4_t*>(p)[1];
#pragma unroll
                for (int i = 0; i < 4; ++i) h[i] = to_half_clamped(a[i]), h[4 + i] = to_half_clamped(b[i]);
            }
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (k + i < K) h[i] = to_half_clamped(p[i]);
        }
    } else {
        const _Float16* p = static_cast<const _Float16*>(X) + row + k;
        if (vec) {
            if (k < K) h = *reinterpret_cast<const half8_t*>(p);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (k + i < K) h[i] = p[i];
        }
    }
    return h;
}

// MT x NT blocks of 16 x 16, WAVES waves that share K, SH: log2(group / 32).
template <int MT, int NT, int WAVES, bool X32>
__global__ void __launch_bounds__(64 * WAVES) w4_few_kernel(W4Args a, int shift, bool vec) {
    constexpr int U = NT * MT >= 4 ? 2 : 4;  // steps whose loads are in flight together
    __shared__ __attribute__((aligned(16))) float part[WAVES * MT * NT * 256];
    const W4View& w = a.w;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int r = lane & 15, g = lane >> 4;
    const int n0 = blockIdx.x * (16 * NT), m0 = blockIdx.y * kW4FewRows;
    const int M = min(a.M - m0, 16 * MT), K = w.K;
    const uint32_t* codes[NT];
    const uint32_t* sm[NT];
#pragma unroll
    for (int j = 0; j < NT; ++j) {
        const int64_t n = min(n0 + 16 * j + r, w.N - 1);
        codes[j] = w.codes + n * w.words + 4 * g;
        sm[j] = w.sm + n * w.G;
    }
    int64_t row[MT];
#pragma unroll
    for (int i = 0; i < MT; ++i) row[i] = (int64_t)(m0 + min(16 * i + r, M - 1)) * a.ldx;

    float4_t acc[MT][NT];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) acc[i][j] = float4_t{0.0f, 0.0f, 0.0f, 0.0f};

    const int steps = (K + 127) / 128, chunks = w.words / 4;
    for (int s0 = wave; s0 < steps; s0 += WAVES * U) {
        u32x4_t c[U][NT];
        uint32_t p[U][NT];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int step = s0 + u * WAVES, chunk = 4 * step + g;
            const bool in = chunk < chunks;
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                // (a pair of zeros: the value 0 whatever the codes)
                c[u][j] = u32x4_t{0, 0, 0, 0};
                p[u][j] = 0;
                if (in) {
                    c[u][j] = *reinterpret_cast<const u32x4_t*>(codes[j] + 16 * step);
                    p[u][j] = sm[j][chunk >> shift];
                }
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int step = s0 + u * WAVES;
            if (step >= steps) break;
            half8_t x[MT][4];
#pragma unroll
            for (int i = 0; i < MT; ++i)
#pragma unroll
                for (int q = 0; q < 4; ++q) x[i][q] = load_x<X32>(a.X, row[i], 128 * step + 32 * g + 8 * q, K, vec);
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                half2_t s, m;
                four_bit_pair(p[u][j], s, m);
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const half8_t b = four_bit_values(c[u][j][q], s, m);
#pragma unroll
                    for (int i = 0; i < MT; ++i)
                        acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(x[i][q], b, acc[i][j], 0, 0, 0);
                }
            }
        }
    }
    // part[wave][block][row][column]
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) part[((wave * MT + i) * NT + j) * 256 + (4 * g + e) * 16 + r] = acc[i][j][e];
    __syncthreads();
    for (int at = tid; at < MT * NT * 256; at += 64 * WAVES) {
        const int i = at / (NT * 256), rr = (at / (NT * 16)) % 16, cc = at % (NT * 16);
        const int j = cc / 16, m = 16 * i + rr, n = n0 + cc;
        if (m >= M || n >= w.N) continue;
        const int from = (i * NT + j) * 256 + rr * 16 + cc % 16;
        float v = 0.0f;
#pragma unroll
        for (int q = 0; q < WAVES; ++q) v += part[q * MT * NT * 256 + from];
        if (a.bias) v += a.bias[n];
        if (a.gelu) v = gelu_tanh(v);
        const int64_t to = (int64_t)(m0 + m) * a.ldc + n;
        if (a.c16) static_cast<_Float16*>(a.C)[to] = (_Float16)v;
        else if (a.residual) static_cast<float*>(a.C)[to] += v;
        else static_cast<float*>(a.C)[to] = v;
    }
}

// A thread per 32 codes.
__global__ void __launch_bounds__(256) w4_expand_kernel(W4View w, int n0, int64_t pieces, half8_t* out, int shift) {
    const int chunks = w.words / 4;
    for (int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x; at < pieces; at += (int64_t)gridDim.x * 256) {
        const int n = (int)(at / chunks), c = (int)(at - (int64_t)n * chunks);
        const u32x4_t x = *reinterpret_cast<const u32x4_t*>(w.codes + (int64_t)(n0 + n) * w.words + 4 * c);
        half2_t s, m;
        four_bit_pair(w.sm[(int64_t)(n0 + n) * w.G + (c >> shift)], s, m);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            half8_t v = four_bit_values(x[i], s, m);
            const int k = 32 * c + 8 * i;
            if (k + 8 > w.K) {
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (k + j >= w.K) v[j] = (_Float16)0.0f;
            }
            store_half8(out + at * 4 + i, v);
        }
    }
}

template <bool X32>
__global__ void __launch_bounds__(256) w4_rows_kernel(const void* X, int64_t ldx, int64_t M, int K, half8_t* out, int eights,
                                                      bool vec) {
    for (int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x; at < M * eights; at += (int64_t)gridDim.x * 256) {
        const int64_t m = at / eights;
        store_half8(out + at, load_x<X32>(X, m * ldx, 8 * (int)(at - m * eights), K, vec));
    }
}

// A thread per column and group; W's rows are read along the columns.
template <bool F32>
__global__ void __launch_bounds__(256) w4_quantize_kernel(const void* W, int64_t ldw, W4View w, uint32_t* codes, uint32_t* sm) {
    const int n = blockIdx.x * 64 + (threadIdx.x & 63);
    if (n >= w.N) return;
    auto value = [&](int k) {
        const int64_t at = (int64_t)k * ldw + n;
        if constexpr (!F32) return (float)static_cast<const _Float16*>(W)[at];
        // (finite values clamp; an infinity or NaN stays one, for the whole group)
        const float x = static_cast<const float*>(W)[at];
        return __builtin_fabsf(x) < __builtin_inff() ? (float)to_half_clamped(x) : x;
    };
    for (int g = blockIdx.y * 4 + (threadIdx.x >> 6); g < w.G; g += gridDim.y * 4) {
        const int k0 = g * w.group, k1 = min(w.K, k0 + w.group);
        float lo = __builtin_inff(), hi = -__builtin_inff();
        bool bad = false;
        for (int k = k0; k < k1; ++k) {
            const float x = value(k);
            bad |= !(__builtin_fabsf(x) < __builtin_inff());
            lo = __builtin_fminf(lo, x);
            hi = __builtin_fmaxf(hi, x);
        }
        const uint32_t pair = four_bit_scale(lo, hi, bad);
        const float s = (float)__builtin_bit_cast(half2_t, pair)[0];
        sm[(int64_t)n * w.G + g] = pair;
        for (int k = k0; k < min(k0 + w.group, 8 * w.words); k += 8) {
            float x[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = k + i < k1 ? value(k + i) : lo;
            codes[(int64_t)n * w.words + k / 8] = four_bit_word(x, s, lo);
        }
    }
}

__global__ void __launch_bounds__(256) w4_unpack_kernel(W4View w, _Float16* out, int64_t ld, int shift) {
    const int n = blockIdx.x * 64 + (threadIdx.x & 63);
    if (n >= w.N) return;
    for (int c = blockIdx.y * 4 + (threadIdx.x >> 6); c < (w.K + 7) / 8; c += gridDim.y * 4) {
        half2_t s, m;
        four_bit_pair(w.sm[(int64_t)n * w.G + (c >> (shift + 2))], s, m);
        const half8_t v = four_bit_values(w.codes[(int64_t)n * w.words + c], s, m);
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (8 * c + i < w.K) out[(int64_t)(8 * c + i) * ld + n] = v[i];
    }
}

int group_shift(int group) { return group == 32 ? 0 : group == 64 ? 1 : 2; }

template <int MT, int NT, int WAVES>
void few(const W4Args& a, hipStream_t s, bool vec) {
    const dim3 grid((unsigned)((a.w.N + 16 * NT - 1) / (16 * NT)), (unsigned)((a.M + kW4FewRows - 1) / kW4FewRows));
    if (a.x32) w4_few_kernel<MT, NT, WAVES, true><<<grid, 64 * WAVES, 0, s>>>(a, group_shift(a.w.group), vec);
    else w4_few_kernel<MT, NT, WAVES, false><<<grid, 64 * WAVES, 0, s>>>(a, group_shift(a.w.group), vec);
}

}  // namespace

hipError_t launch_w4_few(const W4Args& a, int cus, hipStream_t s) {
    const int es = a.x32 ? 4 : 2;
    const bool vec = a.w.K % 8 == 0 && (((uintptr_t)a.X | (uintptr_t)(a.ldx * es)) & 15) == 0;
    if (a.M <= 16) few<1, 1, 8>(a, s, vec);
    else if (a.M <= 32) few<2, 2, 8>(a, s, vec);
    else few<4, 2, 8>(a, s, vec);
    return hipGetLastError();
}

hipError_t launch_w4_expand(const W4View& w, int n0, int n, _Float16* out, hipStream_t s) {
    const int64_t pieces = (int64_t)n * (w.words / 4);
    w4_expand_kernel<<<row_blocks((pieces + 255) / 256), 256, 0, s>>>(w, n0, pieces, reinterpret_cast<half8_t*>(out),
                                                                      group_shift(w.group));
    return hipGetLastError();
}

hipError_t launch_w4_rows(const void* X, bool x32, int64_t ldx, int M, int K, _Float16* out, int64_t ld, hipStream_t s) {
    const int eights = (int)(ld / 8);
    const bool vec = K % 8 == 0 && (((uintptr_t)X | (uintptr_t)(ldx * (x32 ? 4 : 2))) & 15) == 0;
    const unsigned blocks = row_blocks(((int64_t)M * eights + 255) / 256);
    if (x32) w4_rows_kernel<true><<<blocks, 256, 0, s>>>(X, ldx, M, K, reinterpret_cast<half8_t*>(out), eights, vec);
    else w4_rows_kernel<false><<<blocks, 256, 0, s>>>(X, ldx, M, K, reinterpret_cast<half8_t*>(out), eights, vec);
    return hipGetLastError();
}

hipError_t launch_w4_quantize(const void* W, bool f32, int64_t ldw, const W4View& w, uint32_t* codes, uint32_t* sm,
                              hipStream_t s) {
    const dim3 grid((unsigned)((w.N + 63) / 64), (unsigned)((w.G + 3) / 4 < 4096 ? (w.G + 3) / 4 : 4096));
    if (f32) w4_quantize_kernel<true><<<grid, 256, 0, s>>>(W, ldw, w, codes, sm);
    else w4_quantize_kernel<false><<<grid, 256, 0, s>>>(W, ldw, w, codes, sm);
    return hipGetLastError();
}

hipError_t launch_w4_unpack(const W4View& w, _Float16* out, int64_t ld, hipStream_t s) {
    const int words = (w.K + 7) / 8;
    const dim3 grid((unsigned)((w.N + 63) / 64), (unsigned)((words + 3) / 4 < 4096 ? (words + 3) / 4 : 4096));
    w4_unpack_kernel<<<grid, 256, 0, s>>>(w, out, ld, group_shift(w.group));
    return hipGetLastError();
}

}  // namespace vedic
