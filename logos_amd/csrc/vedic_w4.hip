// vedic_w4.hip -- Y[M x N] = epi(X[M x K] . W[K x N]) with W held in four bits, for few rows;
// the same weights expanded to binary16 for the tiled kernels; and weights put into that form.
//
// Few rows (decoding): the product reads N K / 2 bytes and is bound by them.  A lane of
// v_mfma_f32_16x16x32_f16 takes eight values of one column of W: it loads 16 bytes of its column, 32
// consecutive codes of one group with one pair (s, m), expands a word at a time (13
// instructions for eight values) and multiplies; lane group g has the codes 128 i + 32 g .. + 31, and
// takes the same values of its row of X, straight from the cache.  The waves of a workgroup share
// K and add up their 16 x 16 blocks through LDS in a fixed order, so no
// second launch and no workspace are needed.  Column blocks a wave: one for a row or two
// (many workgroups), more with more rows, so that the rows of X are not read more often than
// the codes.
//
// (16 rows of 4096 into 16384: 14 us, 2.4 TB/s of codes; the expanding of one SIMD's share alone takes 4.)
//
// The expanded weight (N K 2 bytes written and read once more) is for products that the binary16 tiles do faster
// than those of vedic_w4_tile.hip, in slabs of columns.
#include "vedic_w4.hpp"

namespace vedic {

namespace {

// Eight values of a row of X from k on, zeros from K on (16 bytes at any alignment are one load).
template <bool X32>
__device__ __forceinline__ half8_t load_x(const void* X, int64_t row, int k, int K) {
    half8_t h = {};
    if constexpr (X32) {
        typedef float4_t float4_any_t __attribute__((aligned(4)));
        const float* p = static_cast<const float*>(X) + row + k;
        if (k + 8 <= K) {
            const float4_t a = reinterpret_cast<const float4_any_t*>(p)[0], b = reinterpret_cast<const float4_any_t*>(p)[1];
#pragma unroll
            for (int i = 0; i < 4; ++i) h[i] = to_half_clamped(a[i]), h[4 + i] = to_half_clamped(b[i]);
        } else if (K & 7) {
            for (int i = 0; i < 8; ++i)
                if (k + i < K) h[i] = to_half_clamped(p[i]);
        }
    } else {
        typedef half8_t half8_any_t __attribute__((aligned(2)));
        const _Float16* p = static_cast<const _Float16*>(X) + row + k;
        if (k + 8 <= K) {
            h = *reinterpret_cast<const half8_any_t*>(p);
        } else if (K & 7) {
            for (int i = 0; i < 8; ++i)
                if (k + i < K) h[i] = p[i];
        }
    }
    return h;
}

// Eight values of X as they come (16 bytes at any alignment are one load), and as binary16.
template <bool X32>
struct XRaw {
    u32x4_t v[X32 ? 2 : 1];
    __device__ __forceinline__ void load(const void* X, int64_t at) {
        if constexpr (X32) {
            typedef u32x4_t any_t __attribute__((aligned(4)));
            const any_t* p = reinterpret_cast<const any_t*>(static_cast<const float*>(X) + at);
            v[0] = p[0];
            v[1] = p[1];
        } else {
            typedef u32x4_t any_t __attribute__((aligned(2)));
            v[0] = *reinterpret_cast<const any_t*>(static_cast<const _Float16*>(X) + at);
        }
    }
    __device__ __forceinline__ half8_t value() const {
        if constexpr (!X32) return __builtin_bit_cast(half8_t, v[0]);
        half8_t h;
        const float4_t a = __builtin_bit_cast(float4_t, v[0]), b = __builtin_bit_cast(float4_t, v[X32 ? 1 : 0]);
#pragma unroll
        for (int i = 0; i < 4; ++i) h[i] = to_half_clamped(a[i]), h[4 + i] = to_half_clamped(b[i]);
        return h;
    }
};

// MT x NT blocks of 16 x 16, WAVES waves that share K; shift: log2(group / 32).
template <int MT, int NT, int WAVES, bool X32>
__global__ void __launch_bounds__(64 * WAVES) w4_few_kernel(W4Args a, int shift) {
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

    // A wave's steps of 128 values lie together; the first waves have one more where they do not come out even, and the
    // last one what is left of K.
    const int steps = K / 128, each = steps / WAVES, rest = steps % WAVES;
    const int first = wave * each + min(wave, rest), n = each + (wave < rest ? 1 : 0);
    const FourBits expand;
    struct Step {
        u32x4_t c[NT];
        uint32_t p[NT];
        XRaw<X32> x[MT][4];
    };
    auto load = [&](Step& b, int step) {
#pragma unroll
        for (int j = 0; j < NT; ++j) {
            b.c[j] = *reinterpret_cast<const u32x4_t*>(codes[j] + 16 * step);
            b.p[j] = sm[j][(4 * step + g) >> shift];
        }
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int q = 0; q < 4; ++q) b.x[i][q].load(a.X, row[i] + 128 * step + 32 * g + 8 * q);
    };
    auto multiply = [&](const Step& b) {
        half8_t x[MT][4];
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int q = 0; q < 4; ++q) x[i][q] = b.x[i][q].value();
#pragma unroll
        for (int j = 0; j < NT; ++j) {
            half2_t s, m;
            four_bit_pair(b.p[j], s, m);
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const half8_t w = expand(b.c[j][q], s, m);
#pragma unroll
                for (int i = 0; i < MT; ++i)
                    acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(x[i][q], w, acc[i][j], 0, 0, 0);
            }
        }
    };
    // The next step is under way while one is multiplied (its loads without conditions, so that how many are under way
    // is known where the first one's are waited for).
    Step b0, b1;
    if (n > 0) {
        load(b0, first);
        int t = 0;
        for (; t + 2 < n; t += 2) {
            load(b1, first + t + 1);
            multiply(b0);
            load(b0, first + t + 2);
            multiply(b1);
        }
        if (t + 1 < n) {
            load(b1, first + t + 1);
            multiply(b0);
            multiply(b1);
        } else {
            multiply(b0);
        }
    }
    if (wave == WAVES - 1 && 128 * steps < K) {
        const int chunk = 4 * steps + g;
        Step b;
#pragma unroll
        for (int j = 0; j < NT; ++j) {
            // (a pair of zeros: the value 0 whatever the codes)
            b.c[j] = u32x4_t{0, 0, 0, 0};
            b.p[j] = 0;
            if (32 * chunk < K) {
                b.c[j] = *reinterpret_cast<const u32x4_t*>(codes[j] + 16 * steps);
                b.p[j] = sm[j][chunk >> shift];
            }
        }
        for (int q = 0; q < 4; ++q) {
            half8_t x[MT];
#pragma unroll
            for (int i = 0; i < MT; ++i) x[i] = load_x<X32>(a.X, row[i], 32 * chunk + 8 * q, K);
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                half2_t s, m;
                four_bit_pair(b.p[j], s, m);
                half8_t w = expand(q == 0 ? b.c[j][0] : q == 1 ? b.c[j][1] : q == 2 ? b.c[j][2] : b.c[j][3], s, m);
                // (codes from K on may be any: an infinity times the row's zero would count)
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (32 * chunk + 8 * q + e >= K) w[e] = (_Float16)0.0f;
#pragma unroll
                for (int i = 0; i < MT; ++i)
                    acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(x[i], w, acc[i][j], 0, 0, 0);
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

// A thread per word.
__global__ void __launch_bounds__(256) w4_expand_kernel(W4View w, int n0, int64_t words, half8_t* out, int shift) {
    for (int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x; at < words; at += (int64_t)gridDim.x * 256) {
        const int n = (int)(at / w.words), c = (int)(at - (int64_t)n * w.words);
        half2_t s, m;
        four_bit_pair(w.sm[(int64_t)(n0 + n) * w.G + (min(c, (w.K - 1) >> 3) >> (shift + 2))], s, m);
        half8_t v = four_bit_values(w.codes[(int64_t)(n0 + n) * w.words + c], s, m);
        if (8 * c + 8 > w.K) {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (8 * c + j >= w.K) v[j] = (_Float16)0.0f;
        }
        store_half8(out + at, v);
    }
}

template <bool X32>
__global__ void __launch_bounds__(256) w4_rows_kernel(const void* X, int64_t ldx, int64_t M, int K, half8_t* out, int eights) {
    for (int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x; at < M * eights; at += (int64_t)gridDim.x * 256) {
        const int64_t m = at / eights;
        store_half8(out + at, load_x<X32>(X, m * ldx, 8 * (int)(at - m * eights), K));
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
void few(const W4Args& a, hipStream_t s) {
    const dim3 grid((unsigned)((a.w.N + 16 * NT - 1) / (16 * NT)), (unsigned)((a.M + kW4FewRows - 1) / kW4FewRows));
    // (fp32 rows take twice the registers: four waves where 16 rows of binary16 do with half of a SIMD's)
    constexpr int W32 = MT >= 2 ? 4 : WAVES;
    if (a.x32) w4_few_kernel<MT, NT, W32, true><<<grid, 64 * W32, 0, s>>>(a, group_shift(a.w.group));
    else w4_few_kernel<MT, NT, WAVES, false><<<grid, 64 * WAVES, 0, s>>>(a, group_shift(a.w.group));
}

}  // namespace

hipError_t launch_w4_few(const W4Args& all, int cus, hipStream_t s) {
    // (a launch's second dimension ends at 2^16: only a captured call without a workspace block comes here with so many rows)
    constexpr int kMostRows = kW4FewRows * ((1 << 16) - 1);
    if (all.M > kMostRows) {
        W4Args part = all;
        for (int m = 0; m < all.M; m += part.M) {
            part.X = static_cast<const char*>(all.X) + m * all.ldx * (all.x32 ? 4 : 2);
            part.C = static_cast<char*>(all.C) + m * all.ldc * (all.c16 ? 2 : 4);
            part.M = all.M - m < kMostRows ? all.M - m : kMostRows;
            const hipError_t e = launch_w4_few(part, cus, s);
            if (e != hipSuccess) return e;
        }
        return hipSuccess;
    }
    const W4Args& a = all;
    // Column blocks a wave: as many as leave a workgroup for every CU, so that X is not read more often than that
    // needs (us with 1 / 2 / 4: 16 rows of 1024 into 4096 3.9 / 4.2 / 5.4, of 2048 into 8192 8.7 / 6.9 / 8.9, of 4096
    // into 16384 25.5 / 18.5 / 15.8; 64 rows of 1024 into 4096 7.0 / 7.7 / 11.2, of 4096 into 16384 74 / 46 / 32).
    const int64_t blocks = (a.w.N + 15) / 16;
    const int nt = blocks >= 4 * cus ? 4 : blocks >= 2 * cus ? 2 : 1;
    if (a.M <= 16) {
        if (nt == 1) few<1, 1, 8>(a, s);
        else if (nt == 2) few<1, 2, 8>(a, s);
        else few<1, 4, 8>(a, s);
    } else if (a.M <= 32) {
        if (nt == 1) few<2, 1, 8>(a, s);
        else if (nt == 2) few<2, 2, 8>(a, s);
        else few<2, 4, 8>(a, s);
    } else {
        if (nt == 1) few<4, 1, 8>(a, s);
        else if (nt == 2) few<4, 2, 4>(a, s);
        else few<4, 4, 4>(a, s);
    }
    return hipGetLastError();
}

hipError_t launch_w4_expand(const W4View& w, int n0, int n, _Float16* out, hipStream_t s) {
    const int64_t words = (int64_t)n * w.words;
    w4_expand_kernel<<<row_blocks((words + 255) / 256), 256, 0, s>>>(w, n0, words, reinterpret_cast<half8_t*>(out),
                                                                     group_shift(w.group));
    return hipGetLastError();
}

hipError_t launch_w4_rows(const void* X, bool x32, int64_t ldx, int M, int K, _Float16* out, int64_t ld, hipStream_t s) {
    const int eights = (int)(ld / 8);
    const unsigned blocks = row_blocks(((int64_t)M * eights + 255) / 256);
    if (x32) w4_rows_kernel<true><<<blocks, 256, 0, s>>>(X, ldx, M, K, reinterpret_cast<half8_t*>(out), eights);
    else w4_rows_kernel<false><<<blocks, 256, 0, s>>>(X, ldx, M, K, reinterpret_cast<half8_t*>(out), eights);
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
