// vedic_grouped_skinny.hip -- the grouped binary16 products NN and NT for few rows per
// group (decoding): each chosen expert's weight is read for a handful of rows, so HBM
// bounds it, as it bounds the ungrouped decode product (vedic_gemm_skinny.hip): eight
// rows on five of eight experts, 1024 into 4096 with GELU, read 42 MB in 12.9 us (3.3 TB/s;
// a large copy reaches 5.0), start and end of the launch included.
//
// One workgroup per 64 (NN) or 32 (NT) columns and 16 rows of a group, so that a
// weight's 128-byte lines are read whole; its four waves take a quarter of K each
// through three LDS stages of their own (60 to 72 KiB a workgroup: two share a CU, and
// one's search for its group and first loads run under the other's), and the four sums
// are added through LDS in wave order.
#include "vedic_gemm_f16.hpp"
#include "vedic_grouped.hpp"

namespace vedic {

// Columns and contraction steps of a stage; LDS bytes of its A and B.
template <int OP>
struct Skinny {
    static constexpr int ROWS = 16, ST = 3, BN = OP == 1 ? 32 : 64, BK = OP == 1 ? 64 : 32, NB = BN / 32;
    static constexpr int ABYTES = ROWS * BK * 2, BBYTES = BN * BK * 2, STAGE = ABYTES + BBYTES;
    static constexpr int NA = ABYTES / 1024, L = NA + 4;  // load instructions per stage and wave
    static_assert(BBYTES == 4096, "four loads of B");
};

// MFMA operand of a stage's B.  NN: k rows of 64 bytes, eight of them per block of 32
// columns and KiB, by transposing reads.
template <int OP>
__device__ __forceinline__ half8_t skinny_frag_b(const char* lb, int kk, int blk, int lane) {
    if constexpr (OP == 1) {
        return read_frag<true, 32, Skinny<OP>::BK>(lb, 0, kk, lane);
    } else {
        const int g = lane >> 4, s = lane & 15, n = 16 * (g & 1) + 4 * (s & 3);
        union {
            short4_t q[2];
            half8_t h;
        } u;
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            const int k = 16 * kk + 8 * (g >> 1) + 4 * x + (s >> 2);
            u.q[x] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                (lds_short4_t*)(lb + (k >> 3) * 1024 + blk * 512 + (k & 7) * 64 + 2 * n));
        }
        return u.h;
    }
}

// N load instructions of a wave into 1 KiB each; off: the lanes' byte offsets, kend:
// the stage needs that many steps for a lane's chunk to be there.
template <int N>
__device__ __forceinline__ void skinny_load(const _Float16* base, const uint32_t (&off)[N], const int (&kend)[N], int krem,
                                            char* lds) {
    const __amdgpu_buffer_rsrc_t rs = buffer_rsrc(base);
#pragma unroll
    for (int i = 0; i < N; ++i)
        __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (lds_void_t*)(lds + i * 1024), 16, kend[i] <= krem ? off[i] : kOob, 0, 0, 0);
}

template <int OP, int KIND, typename OT>
__global__ void __launch_bounds__(256) grouped_f16_skinny_kernel(GroupedArgs a) {
    using S = Skinny<OP>;
    constexpr bool B_KC = OP == 1;
    constexpr int kRows = S::ROWS, kST = S::ST, kBK = S::BK, kABytes = S::ABYTES, kStage = S::STAGE, L = S::L, BN = S::BN,
                  NB = S::NB, NA = S::NA, CPR = kBK / 8;
    __shared__ __attribute__((aligned(1024))) char s0[4 * kStage];
    __shared__ __attribute__((aligned(1024))) char s1[4 * kStage];
    __shared__ __attribute__((aligned(1024))) char s2[4 * kStage];
    __shared__ GroupIndex ix;
    __shared__ __attribute__((aligned(16))) float sbias[BN];
    char* const Ss[kST] = {s0, s1, s2};
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    group_index(a, ix, kRows);
    const int b = blockIdx.x;  // (dealt to all XCDs: the tiles that exist come first)
    const int t = b / a.tiles_n;
    if (t >= ix.pre[a.groups]) return;
    const int e = group_of(ix, a.groups, t, lane);
    const int start = __builtin_amdgcn_readfirstlane(group_start(a, e));
    const int m0 = (t - __builtin_amdgcn_readfirstlane(ix.pre[e])) * kRows;
    const int left = min(kRows, __builtin_amdgcn_readfirstlane(group_count(a, e)) - m0);
    const int n0 = (b - t * a.tiles_n) * BN;
    if (threadIdx.x < BN)
        sbias[threadIdx.x] =
            a.bias != nullptr && n0 + (int)threadIdx.x < a.N ? a.bias[(int64_t)e * a.N + n0 + threadIdx.x] : 0.0f;

    const _Float16* A = static_cast<const _Float16*>(a.A);
    if (!a.rows) A += (int64_t)(start + m0) * a.lda;
    const _Float16* B = static_cast<const _Float16*>(a.B) + (int64_t)e * a.stride_b + (B_KC ? (int64_t)n0 * a.ldb : n0);
    uint32_t aoff[NA], boff[4];
    int ak[NA], bk[4];
#pragma unroll
    for (int i = 0; i < NA; ++i) {
        const int q = i * 64 + lane, row = q / CPR, c = (q % CPR) ^ swz_kc<CPR>(row);
        int r = row < left ? (a.rows ? a.rows[start + m0 + row] : row) : -1;
        if ((unsigned)r >= (unsigned)(a.rows ? a.a_rows : kRows)) r = -1;
        aoff[i] = r >= 0 ? (uint32_t)((int64_t)r * a.lda * 2 + c * 16) : kOob;
        ak[i] = 8 * c + 8;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (B_KC) {  // 32 rows of 128 bytes
            const int row = 8 * i + (lane >> 3), c = (lane & 7) ^ swz_kc<8>(row);
            boff[i] = n0 + row < a.N ? (uint32_t)((int64_t)row * a.ldb * 2 + c * 16) : kOob;
            bk[i] = 8 * c + 8;
        } else {  // eight k rows of two blocks of 32 columns (64 bytes) an instruction
            const int k = 8 * i + ((lane & 31) >> 2), col = 32 * (lane >> 5) + 8 * (lane & 3);
            boff[i] = n0 + col + 8 <= a.Np ? (uint32_t)((int64_t)k * a.ldb * 2 + col * 2) : kOob;
            bk[i] = k + 1;
        }
    }
    const int kq = (a.K + 4 * kBK - 1) / (4 * kBK) * kBK;
    const int kb = min(a.K, wave * kq), ke = min(a.K, kb + kq);
    auto issue = [&](int k, char* buf) {
        const int krem = ke - k;
        const int64_t kk = krem > 0 ? k : 0;
        skinny_load<NA>(A + kk, aoff, ak, krem, buf + wave * kStage);
        skinny_load<4>(B_KC ? B + kk : B + kk * a.ldb, boff, bk, min(krem, a.K - (B_KC ? 0 : a.kpad) - k), buf + wave * kStage + kABytes);
    };
    float16_t acc[1][NB] = {};
    // (rows 16 .. 31 of the MFMA's A read other LDS: they feed rows that are not stored)
    auto consume = [&](const char* buf) {
        const char* la = buf + wave * kStage;
#pragma unroll
        for (int kk = 0; kk < kBK / 16; ++kk) {
            const half8_t fa = read_frag<true, 32, kBK>(la, 0, kk, lane);
#pragma unroll
            for (int j = 0; j < NB; ++j)
                acc[0][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(fa, skinny_frag_b<OP>(la + kABytes, kk, j, lane), acc[0][j], 0, 0, 0);
        }
    };
    // Rounds of kST stages, the same shape for every wave; stages past the range load
    // zeros without touching memory.
    const int rounds = (kq + kST * kBK - 1) / (kST * kBK);
#pragma unroll
    for (int s = 0; s < kST; ++s) issue(kb + s * kBK, Ss[s]);
    for (int r = 0; r < rounds; ++r) {
#pragma unroll
        for (int s = 0; s < kST; ++s) {
            wait_vmcnt<(kST - 1) * L>();
            consume(Ss[s]);
            wait_lgkmcnt0();  // the stage's reads are done
            issue(kb + ((r + 1) * kST + s) * kBK, Ss[s]);
        }
    }
    wait_vmcnt<0>();  // the trailing zero loads still write LDS
    __syncthreads();
    float4_t* red = reinterpret_cast<float4_t*>(s0);
    static_assert(4 * NB * 2048 <= 4 * kStage, "the sums fit a stage object");
    auto part = [&](int w, int j, int q) { return red + ((w * NB + j) * 2 + q) * 64 + lane; };
#pragma unroll
    for (int j = 0; j < NB; ++j)
#pragma unroll
        for (int q = 0; q < 2; ++q)  // (rows 0 .. 15)
            *part(wave, j, q) = float4_t{acc[0][j][4 * q], acc[0][j][4 * q + 1], acc[0][j][4 * q + 2], acc[0][j][4 * q + 3]};
    __syncthreads();
    if (wave != 0) return;
#pragma unroll
    for (int j = 0; j < NB; ++j)
#pragma unroll
        for (int q = 0; q < 2; ++q) {  // (rows 0 .. 15)
            float4_t v = *part(0, j, q);
#pragma unroll
            for (int w = 1; w < 4; ++w) v += *part(w, j, q);
#pragma unroll
            for (int x = 0; x < 4; ++x) acc[0][j][4 * q + x] = v[x];
        }
    OT* const C = static_cast<OT*>(a.C) + (int64_t)(start + m0) * a.ldc;
    OT* const P = a.P != nullptr ? static_cast<OT*>(a.P) + (int64_t)(start + m0) * a.ldp : nullptr;
    grouped_epilogue<KIND, OT, true, false, 1, NB>(C, a.ldc, P, a.ldp, sbias, 0.0f, acc, left, a.N, n0, lane);
}

namespace {

template <int OP, int KIND, typename OT>
hipError_t launch(GroupedArgs a, hipStream_t s) {
    a.tiles_n = (a.N + Skinny<OP>::BN - 1) / Skinny<OP>::BN;
    const int64_t work = (int64_t)(a.R / Skinny<OP>::ROWS + (a.groups < a.R ? a.groups : a.R)) * a.tiles_n;
    hipLaunchKernelGGL((grouped_f16_skinny_kernel<OP, KIND, OT>), dim3((unsigned)work), dim3(256), 0, s, a);
    return hipGetLastError();
}

template <int OP, int KIND>
hipError_t launch_out(const GroupedArgs& a, bool f16out, hipStream_t s) {
    return f16out ? launch<OP, KIND, _Float16>(a, s) : launch<OP, KIND, float>(a, s);
}

}  // namespace

#define VEDIC_GROUPED_SKINNY(OP, KIND)                                               \
    template __global__ void grouped_f16_skinny_kernel<OP, KIND, float>(GroupedArgs); \
    template __global__ void grouped_f16_skinny_kernel<OP, KIND, _Float16>(GroupedArgs)
VEDIC_GROUPED_SKINNY(0, GK_LINEAR);
VEDIC_GROUPED_SKINNY(0, GK_GELU);
VEDIC_GROUPED_SKINNY(0, GK_GELU_P);
VEDIC_GROUPED_SKINNY(1, GK_LINEAR);
VEDIC_GROUPED_SKINNY(1, GK_GELU_BWD);

// Operands as for the kernels of vedic_grouped_f16.hpp; op NN (0) or NT (1).
hipError_t launch_grouped_f16_skinny(int op, const GroupedArgs& a, int kind, bool f16out, hipStream_t s) {
    if (op == 1) return kind == GK_GELU_BWD ? launch_out<1, GK_GELU_BWD>(a, f16out, s) : launch_out<1, GK_LINEAR>(a, f16out, s);
    return kind == GK_GELU     ? launch_out<0, GK_GELU>(a, f16out, s)
           : kind == GK_GELU_P ? launch_out<0, GK_GELU_P>(a, f16out, s)
                               : launch_out<0, GK_LINEAR>(a, f16out, s);
}

}  // namespace vedic
