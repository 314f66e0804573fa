// vedic_combine.hip -- rows sorted by expert back in token order, the backward of
// that, gathered and padded copies of rows, sums of slabs, and column sums by group.
//
// All are bound by memory: each value is read and written once, 16 bytes a lane
// where the rows allow it, sums in fp32 in a fixed order.  (8192 tokens of 2 rows of 1024
// fp32 values with a residual: 134 MB in 21.0 us; backward, 4099 tokens of 4 rows of 1000,
// binary16 gradients: 115 MB in 21.2 us.)
#include "vedic_combine.hpp"
#include "vedic_common.hpp"
#include "vedic_grouped.hpp"

namespace vedic {

namespace {

template <typename T>
__device__ __forceinline__ float4_t load4(const T* p) {
    if constexpr (sizeof(T) == 4) {
        return *reinterpret_cast<const float4_t*>(p);
    } else {
        typedef _Float16 half4_t __attribute__((ext_vector_type(4)));
        return __builtin_convertvector(*reinterpret_cast<const half4_t*>(p), float4_t);
    }
}
template <typename T>
__device__ __forceinline__ void store4(T* p, float4_t v) {
    if constexpr (sizeof(T) == 4) {
        store16_hold(p, v);
    } else {
        typedef _Float16 half4_t __attribute__((ext_vector_type(4)));
        *reinterpret_cast<half4_t*>(p) = __builtin_convertvector(v, half4_t);
    }
}

// The four columns of a lane in a strip of 256: neighbours with VEC, 64 apart
// without.
template <bool VEC>
__device__ __forceinline__ int column(int c0, int lane, int i) {
    return VEC ? c0 + 4 * lane + i : c0 + 64 * i + lane;
}
template <typename T, bool VEC>
__device__ __forceinline__ float4_t load_strip(const T* row, int c0, int lane, int D) {
    float4_t v = {0.0f, 0.0f, 0.0f, 0.0f};
    if constexpr (VEC) {
        if (c0 + 4 * lane < D) v = load4<T>(row + c0 + 4 * lane);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (column<false>(c0, lane, i) < D) v[i] = (float)row[column<false>(c0, lane, i)];
    }
    return v;
}
template <typename T, bool VEC>
__device__ __forceinline__ void store_strip(T* row, int c0, int lane, int D, float4_t v) {
    if constexpr (VEC) {
        if (c0 + 4 * lane < D) store4<T>(row + c0 + 4 * lane, v);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (column<false>(c0, lane, i) < D) row[column<false>(c0, lane, i)] = (T)v[i];
    }
}

// out[t] = residual[t] + sum over j, ascending, of w[t, j] Y[slot[t, j]]: one wave
// per 256 columns of a token, its k rows' loads in flight together (eight at a
// time).
template <typename T, bool VEC>
__global__ void __launch_bounds__(256) combine_kernel(CombineArgs a, int strips) {
    const int lane = threadIdx.x & 63;
    const int64_t item = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t t = item / strips;
    const int c0 = (int)(item - t * strips) * 256;
    if (t >= a.T) return;
    const T* Y = static_cast<const T*>(a.Y);
    float4_t sum = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int j0 = 0; j0 < a.k; j0 += 8) {
        float4_t y[8];
        float w[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            y[j] = float4_t{0.0f, 0.0f, 0.0f, 0.0f};
            w[j] = 0.0f;
            if (j0 + j < a.k) {
                const int s = __builtin_amdgcn_readfirstlane(a.slots[t * a.k + j0 + j]);
                if ((unsigned)s < (unsigned)a.R) {
                    y[j] = load_strip<T, VEC>(Y + (int64_t)s * a.ldy, c0, lane, a.D);
                    w[j] = a.weights ? a.weights[t * a.k + j0 + j] : 1.0f;
                }
            }
        }
#pragma unroll
        for (int j = 0; j < 8; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) sum[e] = __builtin_fmaf(w[j], y[j][e], sum[e]);
    }
    if (a.residual) sum += load_strip<float, VEC>(a.residual + t * a.ldr, c0, lane, a.D);
    store_strip<float, VEC>(a.out + t * a.ldo, c0, lane, a.D, sum);
}

// One pair (t, j) by one wave: dY[slot] = w dout[t], dw = <dout[t], Y[slot]>.  The
// k waves of a token are neighbours, so that dout's row comes from the caches for
// all but one.
template <typename T, typename DT, bool VEC>
__global__ void __launch_bounds__(256) combine_bwd_kernel(CombineBwdArgs a) {
    const int lane = threadIdx.x & 63;
    for (int64_t p = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); p < (int64_t)a.T * a.k;
         p += (int64_t)gridDim.x * 4) {
        const int64_t t = p / a.k;
        const int s = __builtin_amdgcn_readfirstlane(a.slots[p]);
        float dot = 0.0f;
        if ((unsigned)s < (unsigned)a.R) {
            const float w = a.weights[p];
            const float* g = a.dout + t * a.ldg;
            const T* y = static_cast<const T*>(a.Y) + (int64_t)s * a.ldy;
            DT* o = static_cast<DT*>(a.dY) + (int64_t)s * a.ldo;
            float4_t part = {0.0f, 0.0f, 0.0f, 0.0f};
            for (int c0 = 0; c0 < a.D; c0 += 512) {
                float4_t gv[2], yv[2];
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    gv[h] = load_strip<float, VEC>(g, c0 + 256 * h, lane, a.D);
                    yv[h] = load_strip<T, VEC>(y, c0 + 256 * h, lane, a.D);
                }
#pragma unroll
                for (int h = 0; h < 2; ++h) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) part[e] = __builtin_fmaf(gv[h][e], yv[h][e], part[e]);
                    store_strip<DT, VEC>(o, c0 + 256 * h, lane, a.D, gv[h] * w);
                }
            }
            dot = (part[0] + part[1]) + (part[2] + part[3]);
#pragma unroll
            for (int d = 32; d > 0; d >>= 1) dot += __shfl_xor(dot, d);
        }
        if (lane == 0) a.dweights[p] = dot;
    }
}

// dst[i] = src[rows[i]] (zeros for an index outside), `words` 2-byte words each:
// element-wise, for any alignment.
__global__ void __launch_bounds__(256) gather_rows_kernel(const uint16_t* src, int64_t ld, int nsrc, const int* rows, int n,
                                                           int words, uint16_t* dst, int64_t ldd) {
    for (int64_t i = blockIdx.x; i < n; i += gridDim.x) {
        const int r = rows[i];
        const bool ok = (unsigned)r < (unsigned)nsrc;
        const uint16_t* s = src + (int64_t)(ok ? r : 0) * ld;
        uint16_t* d = dst + i * ldd;
        for (int c = threadIdx.x; c < words; c += 256) d[c] = ok ? s[c] : (uint16_t)0;
    }
}

// The same by 16-byte chunks.
__global__ void __launch_bounds__(256) gather_rows16_kernel(const u32x4_t* src, int64_t ld, int nsrc, const int* rows, int n,
                                                             int chunks, u32x4_t* dst, int64_t ldd) {
    const int64_t total = (int64_t)n * chunks;
    for (int64_t q = (int64_t)blockIdx.x * 256 + threadIdx.x; q < total; q += (int64_t)gridDim.x * 256) {
        const int64_t i = q / chunks;
        const int c = (int)(q - i * chunks);
        const int r = rows[i];
        u32x4_t v = {0u, 0u, 0u, 0u};
        if ((unsigned)r < (unsigned)nsrc) v = src[(int64_t)r * ld + c];
        dst[i * ldd + c] = v;
    }
}

// dst[i][0 .. 8 octs) = binary16 src row i, zeros past `cols`: of matrices of `per` rows,
// `stride` apart, or, where a list is given, row rows[i] of the nsrc rows (zeros outside).
// 16-byte stores; loads of any alignment.
__global__ void __launch_bounds__(256) pad_rows_kernel(const _Float16* src, int64_t ld, int per, int64_t stride, int nsrc,
                                                        const int* rows, int64_t n, int cols, int octs, half8_t* dst) {
    for (int64_t q = (int64_t)blockIdx.x * 256 + threadIdx.x; q < n * octs; q += (int64_t)gridDim.x * 256) {
        const int64_t i = q / octs;
        const int c = (int)(q - i * octs) * 8;
        int64_t at;  // the row's first value
        bool ok = true;
        if (rows != nullptr) {  // (an entry is the row itself: `per` counts rows without a list)
            const int r = rows[i];
            ok = (unsigned)r < (unsigned)nsrc;
            at = ok ? (int64_t)r * ld : 0;
        } else {
            const int64_t m = i / per;
            at = m * stride + (i - m * per) * ld;
        }
        const _Float16* s = src + at + c;
        half8_t v;
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = ok && c + e < cols ? s[e] : (_Float16)0.0f;
        dst[q] = v;
    }
}

// db[e][j] = beta db[e][j] + sum of X[i][j] over the group's rows.  One workgroup
// per group and strip of columns, phase p of PH adding rows p, p + PH, ... in
// order and the phases then in order.  VEC: 64 columns by 16-byte loads; else one
// column a lane.
template <typename T, bool VEC>
__global__ void __launch_bounds__(256) group_colsum_kernel(const T* X, int64_t ld, int R, int N, const int* offsets, float beta,
                                                            float* db) {
    constexpr int V = VEC ? 16 / sizeof(T) : 1;  // columns a thread
    constexpr int CT = 64 / V, PH = 256 / CT;    // threads across a strip, row phases
    __shared__ float sh[PH][65];
    const int e = blockIdx.y, c = threadIdx.x % CT, ph = threadIdx.x / CT;
    const int j = blockIdx.x * 64 + c * V;
    const int i0 = min(max(offsets[e], 0), R), i1 = max(i0, min(max(offsets[e + 1], 0), R));
    float sum[V];
#pragma unroll
    for (int v = 0; v < V; ++v) sum[v] = 0.0f;
    if (j < N) {
#pragma unroll 8
        for (int i = i0 + ph; i < i1; i += PH) {
            if constexpr (VEC) {
                const u32x4_t w = *reinterpret_cast<const u32x4_t*>(X + (int64_t)i * ld + j);
                if constexpr (sizeof(T) == 2) {
#pragma unroll
                    for (int v = 0; v < V; ++v) sum[v] += (float)__builtin_bit_cast(half8_t, w)[v];
                } else {
#pragma unroll
                    for (int v = 0; v < V; ++v) sum[v] += __builtin_bit_cast(float4_t, w)[v];
                }
            } else {
                sum[0] += (float)X[(int64_t)i * ld + j];
            }
        }
    }
#pragma unroll
    for (int v = 0; v < V; ++v) sh[ph][c * V + v] = sum[v];
    __syncthreads();
    if (threadIdx.x < 64) {
        const int col = blockIdx.x * 64 + threadIdx.x;
        float t = sh[0][threadIdx.x];
        for (int q = 1; q < PH; ++q) t += sh[q][threadIdx.x];
        if (col < N) {
            float* o = db + (int64_t)e * N + col;
            *o = beta == 0.0f ? t : __builtin_fmaf(beta, *o, t);
        }
    }
}

// C_g = beta C_g + the sum of S slabs [groups][M x N], in order.
__global__ void __launch_bounds__(256) slab_sum_kernel(const float* ws, int S, int64_t slab, int M, int N, float* C, int64_t ldc,
                                                        int64_t stride_c, float beta) {
    for (int64_t q = (int64_t)blockIdx.x * 256 + threadIdx.x; q < slab; q += (int64_t)gridDim.x * 256) {
        float t = ws[q];
        for (int s = 1; s < S; ++s) t += ws[s * slab + q];
        const int64_t row = q / N;
        const int n = (int)(q - row * N);
        const int64_t g = row / M;
        float* c = C + g * stride_c + (row - g * M) * ldc + n;
        *c = beta == 0.0f ? t : __builtin_fmaf(beta, *c, t);
    }
}

// C = the sum of S slabs [R x N], in order, plus the group's bias, in the groups' rows.
// One row per workgroup row (blockIdx.y), found among the groups by bisection.
template <typename OT>
__global__ void __launch_bounds__(256) slab_rows_kernel(const float* ws, int S, int R, int N, const int* offsets, int groups,
                                                        const float* bias, OT* C, int64_t ldc) {
    const int n = blockIdx.x * 256 + threadIdx.x;
    if (n >= N) return;
    for (int r = blockIdx.y; r < R; r += gridDim.y) {
        int e = 0;
        if (offsets != nullptr) {
            // (the last group that starts at or before r: the groups before it end there)
            int lo = 0, hi = groups;
            while (lo < hi) {
                const int mid = (lo + hi + 1) >> 1;
                if (offsets[mid] <= r) lo = mid;
                else hi = mid - 1;
            }
            e = lo;
            if (e >= groups || offsets[0] > r) continue;
        }
        const float* w = ws + (int64_t)r * N + n;
        float t = w[0];
        for (int s = 1; s < S; ++s) t += w[(int64_t)s * R * N];
        if (bias != nullptr) t += bias[(int64_t)e * N + n];
        C[r * ldc + n] = (OT)t;
    }
}

bool rows_ok(const void* p, int64_t ld, int es, int chunk) {
    return p == nullptr || ((reinterpret_cast<uintptr_t>(p) % chunk) == 0 && (ld * es) % chunk == 0);
}

}  // namespace

hipError_t launch_combine(CombineArgs a, bool f16, hipStream_t s) {
    const int strips = (a.D + 255) / 256;
    // (rows padded to whole chunks would be read past D: D itself has to be a multiple)
    const bool vec = a.D % 4 == 0 && rows_ok(a.Y, a.ldy, f16 ? 2 : 4, f16 ? 8 : 16) && rows_ok(a.out, a.ldo, 4, 16) &&
                     rows_ok(a.residual, a.ldr, 4, 16);
    // (in launches of fewer than 2^32 threads; a loop in the kernel costs 1 % of 21 us)
    const int tokens = ((1 << 26) - 4) / strips;
    for (int64_t left = a.T; left > 0; left -= tokens) {
        a.T = (int)(left < tokens ? left : tokens);
        const dim3 g((unsigned)(((int64_t)a.T * strips + 3) / 4)), b(256);
        if (f16) {
            if (vec) hipLaunchKernelGGL((combine_kernel<_Float16, true>), g, b, 0, s, a, strips);
            else hipLaunchKernelGGL((combine_kernel<_Float16, false>), g, b, 0, s, a, strips);
        } else {
            if (vec) hipLaunchKernelGGL((combine_kernel<float, true>), g, b, 0, s, a, strips);
            else hipLaunchKernelGGL((combine_kernel<float, false>), g, b, 0, s, a, strips);
        }
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
        a.slots += (int64_t)a.T * a.k;
        if (a.weights) a.weights += (int64_t)a.T * a.k;
        if (a.residual) a.residual += a.T * a.ldr;
        a.out += a.T * a.ldo;
    }
    return hipSuccess;
}

template <typename T, typename DT>
static hipError_t launch_combine_bwd_t(const CombineBwdArgs& a, hipStream_t s) {
    const dim3 g(row_blocks(((int64_t)a.T * a.k + 3) / 4)), b(256);
    const bool vec = a.D % 4 == 0 && rows_ok(a.dout, a.ldg, 4, 16) && rows_ok(a.Y, a.ldy, sizeof(T), 4 * sizeof(T)) &&
                     rows_ok(a.dY, a.ldo, sizeof(DT), 4 * sizeof(DT));
    if (vec) hipLaunchKernelGGL((combine_bwd_kernel<T, DT, true>), g, b, 0, s, a);
    else hipLaunchKernelGGL((combine_bwd_kernel<T, DT, false>), g, b, 0, s, a);
    return hipGetLastError();
}

hipError_t launch_combine_bwd(const CombineBwdArgs& a, bool f16, bool out16, hipStream_t s) {
    if (f16) return out16 ? launch_combine_bwd_t<_Float16, _Float16>(a, s) : launch_combine_bwd_t<_Float16, float>(a, s);
    return out16 ? launch_combine_bwd_t<float, _Float16>(a, s) : launch_combine_bwd_t<float, float>(a, s);
}

hipError_t launch_gather_rows(const void* src, int64_t ld, int nsrc, const int* rows, int n, int cols, int es, void* dst,
                              int64_t ldd, hipStream_t s) {
    if (rows_ok(src, ld, es, 16) && rows_ok(dst, ldd, es, 16) && (int64_t)cols * es % 16 == 0) {
        const int chunks = cols * es / 16;
        int64_t blocks = ((int64_t)n * chunks + 255) / 256;
        if (blocks > 65536) blocks = 65536;
        hipLaunchKernelGGL(gather_rows16_kernel, dim3((unsigned)blocks), dim3(256), 0, s, static_cast<const u32x4_t*>(src),
                           ld * es / 16, nsrc, rows, n, chunks, static_cast<u32x4_t*>(dst), ldd * es / 16);
    } else {
        hipLaunchKernelGGL(gather_rows_kernel, dim3(row_blocks(n)), dim3(256), 0, s, static_cast<const uint16_t*>(src),
                           ld * (es / 2), nsrc, rows, n, cols * (es / 2), static_cast<uint16_t*>(dst), ldd * (es / 2));
    }
    return hipGetLastError();
}

hipError_t launch_slab_sum(const float* ws, int S, int groups, int M, int N, float* C, int64_t ldc, int64_t stride_c, float beta,
                           hipStream_t s) {
    const int64_t slab = (int64_t)groups * M * N;
    int64_t blocks = (slab + 255) / 256;
    if (blocks > 65536) blocks = 65536;
    hipLaunchKernelGGL(slab_sum_kernel, dim3((unsigned)blocks), dim3(256), 0, s, ws, S, slab, M, N, C, ldc, stride_c, beta);
    return hipGetLastError();
}

hipError_t launch_slab_rows(const float* ws, int S, int R, int N, const int* offsets, int groups, const float* bias, void* C,
                            int64_t ldc, bool out16, hipStream_t s) {
    const dim3 g((unsigned)((N + 255) / 256), (unsigned)(R < 32768 ? R : 32768)), b(256);
    if (out16)
        hipLaunchKernelGGL(slab_rows_kernel<_Float16>, g, b, 0, s, ws, S, R, N, offsets, groups, bias, static_cast<_Float16*>(C), ldc);
    else
        hipLaunchKernelGGL(slab_rows_kernel<float>, g, b, 0, s, ws, S, R, N, offsets, groups, bias, static_cast<float*>(C), ldc);
    return hipGetLastError();
}

hipError_t launch_pad_rows(const void* src, int64_t ld, int per, int64_t stride, int nsrc, const int* rows, int64_t n, int cols,
                           void* dst, hipStream_t s) {
    const int octs = (cols + 7) / 8;
    int64_t blocks = (n * octs + 255) / 256;
    if (blocks > 65536) blocks = 65536;
    hipLaunchKernelGGL(pad_rows_kernel, dim3((unsigned)blocks), dim3(256), 0, s, static_cast<const _Float16*>(src), ld, per,
                       stride, nsrc, rows, n, cols, octs, static_cast<half8_t*>(dst));
    return hipGetLastError();
}

hipError_t launch_group_colsum(const void* X, bool f16, int64_t ld, int R, int N, const int* offsets, int groups, float beta,
                               float* db, hipStream_t s) {
    const dim3 g((unsigned)((N + 63) / 64), (unsigned)groups), b(256);
    const int es = f16 ? 2 : 4;
    const bool vec = rows_ok(X, ld, es, 16) && N * es % 16 == 0;
    if (f16) {
        const _Float16* x = static_cast<const _Float16*>(X);
        if (vec) hipLaunchKernelGGL((group_colsum_kernel<_Float16, true>), g, b, 0, s, x, ld, R, N, offsets, beta, db);
        else hipLaunchKernelGGL((group_colsum_kernel<_Float16, false>), g, b, 0, s, x, ld, R, N, offsets, beta, db);
    } else {
        const float* x = static_cast<const float*>(X);
        if (vec) hipLaunchKernelGGL((group_colsum_kernel<float, true>), g, b, 0, s, x, ld, R, N, offsets, beta, db);
        else hipLaunchKernelGGL((group_colsum_kernel<float, false>), g, b, 0, s, x, ld, R, N, offsets, beta, db);
    }
    return hipGetLastError();
}

}  // namespace vedic
