// vedic_lora.hip -- low-rank adapters of many requests in one batch: for the rows
// i of adapter g (list position p, rows[p] = i),
//   C[i] += scale[g] (X[i] . A_g) . B_g,   A_g [K x r], B_g [r x N].
// Two launches, H = X A_g into a workspace in fp32 (never rounded), then C.
#include "vedic_common.hpp"
#include "vedic_grouped.hpp"
#include "vedic_lora.hpp"

namespace vedic {

namespace {

constexpr int kLoraRows = 8;  // rows per workgroup of one adapter

// H[p][0 .. r) of a tile of eight list positions: thread t takes rank t % RT of
// the steps k = t / RT, t / RT + ST, ...
template <typename T>
__global__ void __launch_bounds__(256) lora_shrink_kernel(LoraArgs a) {
    __shared__ GroupIndex ix;
    __shared__ float part[256][kLoraRows + 1];
    GroupedArgs q{};
    q.offsets = a.offsets;
    q.groups = a.groups;
    q.R = a.n;
    group_index<256>(q, ix, kLoraRows);
    const int lane = threadIdx.x & 63, t = blockIdx.x;
    if (t >= ix.pre[a.groups]) return;
    const int g = group_of(ix, a.groups, t, lane);
    const int p0 = ix.off[g] + (t - ix.pre[g]) * kLoraRows;
    const int np = min(kLoraRows, ix.off[g + 1] - p0);
    const T* A = static_cast<const T*>(a.A) + (int64_t)g * a.K * a.r;
    const T* X = static_cast<const T*>(a.X);
    const T* x[kLoraRows];
    bool ok[kLoraRows];
#pragma unroll
    for (int i = 0; i < kLoraRows; ++i) {
        const int row = i < np ? a.rows[p0 + i] : -1;
        ok[i] = (unsigned)row < (unsigned)a.M;
        x[i] = X + (int64_t)(ok[i] ? row : 0) * a.ldx;
    }
    int rt = 1;
    while (rt < a.r) rt <<= 1;  // ranks across the threads, a power of two
    const int c = threadIdx.x % rt, kp = threadIdx.x / rt, ks = 256 / rt;
    float acc[kLoraRows] = {};
    if (c < a.r)
        for (int k = kp; k < a.K; k += ks) {
            const float w = (float)A[(int64_t)k * a.r + c];
#pragma unroll
            for (int i = 0; i < kLoraRows; ++i) acc[i] = __builtin_fmaf(ok[i] ? (float)x[i][k] : 0.0f, w, acc[i]);
        }
#pragma unroll
    for (int i = 0; i < kLoraRows; ++i) part[threadIdx.x][i] = acc[i];
    __syncthreads();
    for (int o = threadIdx.x; o < a.r * kLoraRows; o += 256) {
        const int cc = o % a.r, i = o / a.r;
        if (i < np) {
            float s = 0.0f;
            for (int v = 0; v < ks; ++v) s += part[v * rt + cc][i];
            a.H[(int64_t)(p0 + i) * a.r + cc] = s;
        }
    }
}

// C += scale H B_g: a tile of eight rows by 256 columns, one column a thread.
template <typename T>
__global__ void __launch_bounds__(256) lora_expand_kernel(LoraArgs a) {
    __shared__ GroupIndex ix;
    __shared__ float h[kLoraRows][kLoraMaxRank];
    GroupedArgs q{};
    q.offsets = a.offsets;
    q.groups = a.groups;
    q.R = a.n;
    group_index<256>(q, ix, kLoraRows);
    const int strips = (a.N + 255) / 256;
    const int lane = threadIdx.x & 63, t = blockIdx.x / strips;
    if (t >= ix.pre[a.groups]) return;
    const int g = group_of(ix, a.groups, t, lane);
    const int p0 = ix.off[g] + (t - ix.pre[g]) * kLoraRows;
    const int np = min(kLoraRows, ix.off[g + 1] - p0);
    for (int o = threadIdx.x; o < kLoraRows * a.r; o += 256) {
        const int i = o / a.r;
        h[i][o % a.r] = i < np ? a.H[(int64_t)(p0 + i) * a.r + o % a.r] : 0.0f;
    }
    __syncthreads();
    const int col = (blockIdx.x - t * strips) * 256 + threadIdx.x;
    if (col >= a.N) return;
    const T* B = static_cast<const T*>(a.B) + (int64_t)g * a.r * a.N + col;
    float acc[kLoraRows] = {};
    for (int k = 0; k < a.r; ++k) {
        const float w = (float)B[(int64_t)k * a.N];
#pragma unroll
        for (int i = 0; i < kLoraRows; ++i) acc[i] = __builtin_fmaf(h[i][k], w, acc[i]);
    }
    const float sc = a.scales ? a.scales[g] : 1.0f;
    for (int i = 0; i < np; ++i) {
        const int row = a.rows[p0 + i];
        if ((unsigned)row < (unsigned)a.M) {
            float* c = a.C + (int64_t)row * a.ldc + col;
            *c = __builtin_fmaf(sc, acc[i], *c);
        }
    }
}

template <typename T>
hipError_t launch(const LoraArgs& a, hipStream_t s) {
    const int64_t tiles = a.n / kLoraRows + (a.groups < a.n ? a.groups : a.n);
    hipLaunchKernelGGL((lora_shrink_kernel<T>), dim3((unsigned)tiles), dim3(256), 0, s, a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL((lora_expand_kernel<T>), dim3((unsigned)(tiles * ((a.N + 255) / 256))), dim3(256), 0, s, a);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_lora(const LoraArgs& a, bool f16, hipStream_t s) {
    return f16 ? launch<_Float16>(a, s) : launch<float>(a, s);
}

}  // namespace vedic
