// vedic_lora.hip -- low-rank adapters of many requests in one batch: for the rows
// i of adapter g (list position p, rows[p] = i),
//   C[i] += scale[g] (X[i] . A_g) . B_g,   A_g [K x r], B_g [r x N].
// Two launches, H = X A_g into a workspace (fp32, or the same as three binary16
// values), then C.  fp32 operands, and rows that 16-byte loads cannot take, run as two
// grouped products (vedic_grouped_any.hpp).
//
// 4096 rows, 1024 into 4096, 12 adapters of rank 64 (all but a twelfth of the rows): 8.2 us
// for H, bound by the latency of its few workgroups, and 28.2 us for C, bound by reading and
// writing it (125 MB, 4.4 TB/s); 16 rows of rank 16 4.8 and 5.2 us, two launches' latency.
#include "vedic_combine.hpp"
#include "vedic_common.hpp"
#include "vedic_gemm_f16.hpp"
#include "vedic_grouped.hpp"
#include "vedic_lora.hpp"

namespace vedic {

hipError_t launch_grouped_any_nn(const GroupedArgs& a, int kind, bool f16, bool f16out, hipStream_t s);

namespace {

// ------------------------------------------------ binary16, 16-byte rows

typedef short lora_short4_t __attribute__((ext_vector_type(4)));

// MFMA operand of 16 columns n0 .. n0 + 15 (lane l: column l mod 16) and the 32
// steps k0 .. k0 + 31 (lane l: 8 (l / 16) .. + 7) of an LDS matrix [k][pitch bytes],
// by two transposing reads; XOR16: the 16-byte slots of row k are XORed by 4 (k mod 4).
template <bool XOR16>
__device__ __forceinline__ half8_t read_tr16(const char* lds, int pitch, int k0, int n0, int lane) {
    const int g = lane >> 4, s = lane & 15;
    union {
        lora_short4_t q[2];
        half8_t h;
    } u;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
        const int k = k0 + 8 * g + 4 * t + (s >> 2), n = n0 + 4 * (s & 3);
        const int off = XOR16 ? k * pitch + (((n >> 3) ^ (4 * (k & 3))) << 4) + 2 * (n & 7) : k * pitch + 2 * n;
        u.q[t] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
            (__attribute__((address_space(3))) lora_short4_t*)(lds + off));
    }
    return u.h;
}

// H = X A_g of 16 places by one workgroup, eight waves each taking an eighth of K
// through two LDS stages of its own (A_g's rows k .. k + KC - 1 are one piece of
// memory; a wave reads what it loaded itself, so no barrier until the sum).  X's
// rows go straight into the MFMA's operand registers.
//
// H's fp32 values are kept as three binary16 ones each: row p is scaled by 2^-x so that
// its largest finite value lies in [2^14, 2^15), and h = hi + 2^-12 mid + 2^-24 lo, each
// part the binary16 nearest to 2^12 times what the last left behind (a remainder of at
// most 2^3: no overflow).  hi and mid are zero rather than subnormal: the MFMA aligns a
// product by its operands' exponents as they stand, so that a subnormal's product beside
// another keeps only the bits from 2^-38 of the other operand on.  What is lost is at most
// 2^-24 of h down to 2^-14, 2^-28 of the largest, 2^-22 (mid and lo alone) down to 2^-26,
// 2^-40 of it, and 2^-37, 2^-51 of the largest, below.
// (Two parts without the 2^12 lose bits from 2^-18 of the largest on; the fp32
// MFMA on H itself takes longer: 4096 rows, 1024 into 4096, projection included, two parts
// / three / three staged by the expansion / fp32 MFMA, rank 64 89 / 93 / 88 / 98 us, rank
// 128 113 / 119 / 109 / 147.)
// factor[p] = scale 2^x then multiplies the product's fp32 sums.
template <int RP, int KC>
__global__ void __launch_bounds__(512) lora_shrink_f16_kernel(LoraArgs a) {
    constexpr int NB = RP / 16, SB = KC * RP * 2, NI = (SB + 1023) / 1024, STAGE = NI * 1024;
    constexpr int RS = RP < 32 ? 32 : RP;  // columns of a part
    static_assert(8 * 16 * RP * 4 <= 8 * 2 * STAGE, "the partial sums fit the stages");
    __shared__ __attribute__((aligned(1024))) char s0[8 * STAGE];
    __shared__ __attribute__((aligned(1024))) char s1[8 * STAGE];
    __shared__ GroupIndex ix;
    GroupedArgs q{};
    q.offsets = a.offsets;
    q.groups = a.groups;
    q.R = a.n;
    group_index(q, ix, 16);
    const int tid = threadIdx.x, lane = tid & 63, t = blockIdx.x;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    if (t >= ix.pre[a.groups]) return;
    const int g = group_of(ix, a.groups, t, lane);
    const int b0 = (t - __builtin_amdgcn_readfirstlane(ix.pre[g])) * 16, p0 = group_start(q, g) + b0;
    const int np = min(16, group_count(q, g) - b0);
    // this lane's row of X and the wave's range of K, whole stages
    const int row = (lane & 15) < np ? a.rows[p0 + (lane & 15)] : -1;
    const bool ok = (unsigned)row < (unsigned)a.M;
    const half8_t* x =
        reinterpret_cast<const half8_t*>(static_cast<const _Float16*>(a.X) + (int64_t)(ok ? row : 0) * a.ldx);
    const int kw = (a.K + 8 * KC - 1) / (8 * KC) * KC;
    const int kb = min(a.K, wave * kw), ke = min(a.K, kb + kw);
    const char* A = static_cast<const char*>(a.A) + ((int64_t)g * a.K) * a.r * 2;
    const int rb = a.r * 2;
    auto issue = [&](int k, char* dst) {
        const __amdgpu_buffer_rsrc_t rs = buffer_rsrc(A + (int64_t)(k < ke ? k : 0) * rb);
        const int left = k < ke ? min(KC, ke - k) * rb : 0;
#pragma unroll
        for (int i = 0; i < NI; ++i) {
            const int off = i * 1024 + lane * 16;
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (lds_void_t*)(dst + wave * STAGE + i * 1024), 16,
                                                     off + 16 <= left ? (uint32_t)off : kOob, 0, 0, 0);
        }
        asm volatile("" ::: "memory");
    };
    // (loads without a condition, so that every stage has the same number in flight:
    // past the range the row's start, whose product with A_g's zeros is masked to zero)
    half8_t xf[2][KC / 32];
    auto fetch = [&](int k, half8_t (&f)[KC / 32]) {
#pragma unroll
        for (int c = 0; c < KC / 32; ++c) {
            const int kk = k + 32 * c + 8 * (lane >> 4);
            f[c] = x[kk < ke ? kk >> 3 : 0];
        }
        asm volatile("" ::: "memory");
    };
    float4_t acc[NB];
#pragma unroll
    for (int b = 0; b < NB; ++b) acc[b] = float4_t{0.0f, 0.0f, 0.0f, 0.0f};
    auto multiply = [&](const char* src, int k, half8_t (&f)[KC / 32]) {
#pragma unroll
        for (int c = 0; c < KC / 32; ++c) {
            if (!ok || k + 32 * c + 8 * (lane >> 4) >= ke) f[c] = half8_t{};
#pragma unroll
            for (int b = 0; b < NB; ++b)
                acc[b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(
                    f[c], read_tr16<false>(src + wave * STAGE, rb, 32 * c, 16 * b, lane), acc[b], 0, 0, 0);
        }
    };
    issue(kb, s0);
    fetch(kb, xf[0]);
    for (int k = kb; k < ke; k += 2 * KC) {
        issue(k + KC, s1);
        fetch(k + KC, xf[1]);
        wait_vmcnt<NI + KC / 32>();
        multiply(s0, k, xf[0]);
        wait_lgkmcnt0();
        issue(k + 2 * KC, s0);
        fetch(k + 2 * KC, xf[0]);
        wait_vmcnt<NI + KC / 32>();
        multiply(s1, k + KC, xf[1]);
        wait_lgkmcnt0();
    }
    wait_vmcnt<0>();
    __syncthreads();
    // sum of the eight partials in wave order: part[wave][row][column]
    float* part0 = reinterpret_cast<float*>(s0);
    float* part1 = reinterpret_cast<float*>(s1);
    constexpr int PW = 16 * RP;  // floats a wave
    auto part = [&](int w) { return w < 4 ? part0 + w * PW : part1 + (w - 4) * PW; };
    static_assert(4 * PW * 4 <= 8 * STAGE, "four waves' partials in each stage object");
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int e = 0; e < 4; ++e) part(wave)[(4 * (lane >> 4) + e) * RP + 16 * b + (lane & 15)] = acc[b][e];
    __syncthreads();
    // 32 threads a row, columns c, c + 32, ...
    const int i = tid >> 5, c0 = tid & 31;
    constexpr int NC = (RS + 31) / 32;
    float h[NC], top = 0.0f;
#pragma unroll
    for (int v = 0; v < NC; ++v) {
        const int c = c0 + 32 * v;
        h[v] = 0.0f;
        if (c < a.r && c < RP)
            for (int w = 0; w < 8; ++w) h[v] += part(w)[i * RP + c];
        if (fabsf(h[v]) < __builtin_inff()) top = fmaxf(top, fabsf(h[v]));
    }
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor(top, d, 32));
    if (i < np) {
        int ex = 0;  // (a row without finite values other than zero keeps its scale)
        if (top > 0.0f) {
            (void)frexpf(top, &ex);  // top = m 2^ex, m in [0.5, 1)
            ex -= 15;
        }
        const float down = ldexpf(1.0f, ex < -126 ? 126 : ex > 126 ? -126 : -ex);
        _Float16* o = a.Hs + (int64_t)(p0 + i) * (3 * RS);
#pragma unroll
        for (int v = 0; v < NC; ++v) {
            const int c = c0 + 32 * v;
            const float s = h[v] * down;
            auto normal = [](float x) { return (_Float16)(fabsf(x) < 0x1p-14f ? 0.0f : x); };
            const _Float16 hi = normal(s);
            const float r1 = fabsf(s) < __builtin_inff() ? (s - (float)hi) * 4096.0f : 0.0f;
            const _Float16 mid = normal(r1);
            o[c] = hi;
            o[RS + c] = mid;
            o[2 * RS + c] = (_Float16)((r1 - (float)mid) * 4096.0f);
        }
        if (c0 == 0) a.factor[p0 + i] = (a.scales ? a.scales[g] : 1.0f) / down;
    }
}

// C[rows[p]] += factor[p] (hi + 2^-12 mid + 2^-24 lo) B_g: 16 places by 256 columns, a wave
// 64 of them.  B_g's columns are staged in LDS once for the three parts, whose products
// have accumulators of their own; they are taken transposed, so that a lane holds four
// neighbouring columns of one row.  Past rank 32 the 16 rows of H are staged too, once for
// the four waves (4096 rows, 1024 into 4096, projection included, each wave its own / staged:
// rank 32 79.6 / 82.5 us, 64 93 / 88.8, 128 119 / 110).
template <int RS>
__global__ void __launch_bounds__(256) lora_expand_f16_kernel(LoraArgs a) {
    constexpr bool STAGED = RS > 32;
    constexpr int HB = 16 * 3 * RS * 2, CPP = RS / 8;  // bytes of the 16 rows, 16-byte chunks of a part
    __shared__ __attribute__((aligned(1024))) char sb[RS * 512];
    __shared__ __attribute__((aligned(1024))) char sh[STAGED ? HB : 16];
    GroupIndex& ix = *reinterpret_cast<GroupIndex*>(sb);
    static_assert(sizeof(GroupIndex) <= RS * 512, "the index fits B's buffer");
    GroupedArgs q{};
    q.offsets = a.offsets;
    q.groups = a.groups;
    q.R = a.n;
    group_index(q, ix, 16);
    const int strips = (a.N + 255) / 256;
    const int tid = threadIdx.x, lane = tid & 63, t = blockIdx.x / strips;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    if (t >= ix.pre[a.groups]) return;
    const int g = group_of(ix, a.groups, t, lane);
    const int b0 = (t - __builtin_amdgcn_readfirstlane(ix.pre[g])) * 16, p0 = group_start(q, g) + b0;
    const int np = min(16, group_count(q, g) - b0);
    const int n0 = (blockIdx.x - t * strips) * 256;
    __syncthreads();  // the index's LDS takes B
    const _Float16* B = static_cast<const _Float16*>(a.B) + (int64_t)g * a.r * a.N + n0;
    const __amdgpu_buffer_rsrc_t rs = buffer_rsrc(B);
#pragma unroll
    for (int i = 0; i < RS / 8; ++i) {  // an instruction: two rows of 32 slots
        const int k = 8 * i + 2 * wave + (lane >> 5), slot = (lane & 31) ^ (4 * (k & 3));
        const bool in = k < a.r && n0 + 8 * slot < a.N;
        __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (lds_void_t*)(sb + (8 * i + 2 * wave) * 512), 16,
                                                 in ? (uint32_t)(k * a.N * 2 + slot * 16) : kOob, 0, 0, 0);
    }
    const int p = lane & 15;
    const _Float16* H = a.Hs + (int64_t)p0 * (3 * RS);
    half8_t part[3][RS / 32];
    // (staged: a part's chunks of row p are XORed by p, so that the rows' reads spread over
    // the banks)
    auto chunk = [](int p, int c) { return c ^ (p & 7); };
    if constexpr (STAGED) {
        const __amdgpu_buffer_rsrc_t rh = buffer_rsrc(H);
#pragma unroll
        for (int i = 0; i < (HB / 1024 + 3) / 4; ++i) {
            const int at = 4 * i + wave, u = at * 64 + lane, pr = u / (3 * CPP), c = u % (3 * CPP), q3 = c / CPP;
            if (at < HB / 1024)
                __builtin_amdgcn_raw_ptr_buffer_load_lds(
                    rh, (lds_void_t*)(sh + at * 1024), 16,
                    pr < np ? (uint32_t)((pr * 3 * CPP + q3 * CPP + chunk(pr, c % CPP)) * 16) : kOob, 0, 0, 0);
        }
    } else {
        const _Float16* h = H + (p < np ? p : 0) * (3 * RS) + 8 * (lane >> 4);
#pragma unroll
        for (int q3 = 0; q3 < 3; ++q3)
#pragma unroll
            for (int c = 0; c < RS / 32; ++c) part[q3][c] = *reinterpret_cast<const half8_t*>(h + q3 * RS + 32 * c);
    }
    const float f = a.factor[p0 + (p < np ? p : 0)];
    const int row = p < np ? a.rows[p0 + p] : -1;
    const bool ok = (unsigned)row < (unsigned)a.M;
    float* crow = a.C + (int64_t)(ok ? row : 0) * a.ldc + n0 + 64 * wave + 4 * (lane >> 4);
    float4_t old[4];
#pragma unroll
    for (int b = 0; b < 4; ++b) {
        old[b] = float4_t{0.0f, 0.0f, 0.0f, 0.0f};
        if (ok && n0 + 64 * wave + 16 * b + 4 * (lane >> 4) < a.N) old[b] = *reinterpret_cast<const float4_t*>(crow + 16 * b);
    }
    wait_vmcnt<0>();
    __syncthreads();
    if constexpr (STAGED) {
#pragma unroll
        for (int q3 = 0; q3 < 3; ++q3)
#pragma unroll
            for (int c = 0; c < RS / 32; ++c)
                part[q3][c] = *reinterpret_cast<const half8_t*>(sh + ((p * 3 + q3) * CPP + chunk(p, 4 * c + (lane >> 4))) * 16);
    }
    float4_t acc[3][4];
#pragma unroll
    for (int q3 = 0; q3 < 3; ++q3)
#pragma unroll
        for (int b = 0; b < 4; ++b) acc[q3][b] = float4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int c = 0; c < RS / 32; ++c)
#pragma unroll
        for (int b = 0; b < 4; ++b) {
            const half8_t w = read_tr16<true>(sb, 512, 32 * c, 64 * wave + 16 * b, lane);
#pragma unroll
            for (int q3 = 0; q3 < 3; ++q3)
                acc[q3][b] = __builtin_amdgcn_mfma_f32_16x16x32_f16(w, part[q3][c], acc[q3][b], 0, 0, 0);
        }
#pragma unroll
    for (int b = 0; b < 4; ++b)
        if (ok && n0 + 64 * wave + 16 * b + 4 * (lane >> 4) < a.N) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float low = __builtin_fmaf(0x1p-12f, acc[2][b][e], acc[1][b][e]);
                old[b][e] = __builtin_fmaf(f, __builtin_fmaf(0x1p-12f, low, acc[0][b][e]), old[b][e]);
            }
            store16_hold(crow + 16 * b, old[b]);
        }
}

// Any types and alignment: two grouped products, the second adding to the listed rows
// of C.  (`copy`: the listed rows, where X is past the products' 32-bit offsets; `slabs`:
// H's slices with a.ksplit > 1, as the grouped products share a long contraction: us, one
// slice / as many as fit, projection included, one row of 768 into 256, rank 4
// 32.4 / 27.6; 898 rows of 896 into 2496, rank 64 98.3 / 90.6.)
bool copies_rows(const LoraArgs& a, bool f16) { return (int64_t)a.M * a.ldx * (f16 ? 2 : 4) >= (int64_t(1) << 31); }

hipError_t launch_any(const LoraArgs& a, bool f16, float* slabs, void* copy, hipStream_t s) {
    GroupedArgs q{};
    q.A = a.X;
    q.lda = a.ldx;
    q.rows = a.rows;
    q.a_rows = a.M;
    if (copies_rows(a, f16)) {
        const hipError_t e = launch_gather_rows(a.X, a.ldx, a.M, a.rows, a.n, a.K, f16 ? 2 : 4, copy, a.K, s);
        if (e != hipSuccess) return e;
        q.A = copy;
        q.lda = a.K;
        q.rows = nullptr;
    }
    q.B = a.A;
    q.ldb = a.r;
    q.stride_b = (int64_t)a.K * a.r;
    q.C = a.ksplit > 1 ? slabs : a.H;
    q.ldc = a.r;
    q.ksplit = a.ksplit;
    q.split_c = (int64_t)a.n * a.r;
    q.offsets = a.offsets;
    q.groups = a.groups;
    q.R = a.n;
    q.N = a.r;
    q.K = a.K;
    hipError_t e = launch_grouped_any_nn(q, GK_LINEAR, f16, false, s);
    if (e == hipSuccess && a.ksplit > 1)
        e = launch_slab_rows(slabs, a.ksplit, a.n, a.r, a.offsets, a.groups, nullptr, a.H, a.r, false, s);
    if (e != hipSuccess) return e;
    q.ksplit = 1;
    q.A = a.H;
    q.lda = a.r;
    q.rows = nullptr;
    q.B = a.B;
    q.ldb = a.N;
    q.stride_b = (int64_t)a.r * a.N;
    q.C = a.C;
    q.ldc = a.ldc;
    q.N = a.N;
    q.K = a.r;
    q.out_rows = a.rows;
    q.out_limit = a.M;
    q.scales = a.scales;
    return launch_grouped_any_nn(q, GK_ADD, f16, false, s);
}

template <int RP, int KC>
hipError_t launch_f16(const LoraArgs& a, hipStream_t s) {
    const int64_t tiles = grouped_row_tiles_max(a.n, a.groups, 16);
    hipLaunchKernelGGL((lora_shrink_f16_kernel<RP, KC>), dim3((unsigned)tiles), dim3(512), 0, s, a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL((lora_expand_f16_kernel<(RP < 32 ? 32 : RP)>), dim3((unsigned)(tiles * ((a.N + 255) / 256))), dim3(256),
                       0, s, a);
    return hipGetLastError();
}

bool al16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// Whether the matrix-core kernels take the call: whole 16-byte loads of every operand.
bool vec16(const LoraArgs& a) {
    return al16(a.X) && al16(a.A) && al16(a.B) && al16(a.C) && a.ldx % 8 == 0 && a.K % 8 == 0 && a.N % 8 == 0 && a.r % 4 == 0 &&
           a.ldc % 4 == 0;
}

}  // namespace

// Columns of a part of H.
static size_t part_columns(int r) { return r <= 32 ? 32 : r <= 64 ? 64 : 128; }

static size_t rounded(size_t bytes) { return (bytes + 255) / 256 * 256; }

bool lora_fits(const LoraArgs& a, bool f16) {
    if (!f16 || !vec16(a)) return grouped_any_fits(0, a.groups, a.n, 0, a.N);
    return grouped_row_tiles_max(a.n, a.groups, 16) * ((a.N + 255) / 256) < kMaxBlocks;
}

size_t lora_bytes(const LoraArgs& a, bool f16) {
    if (f16 && vec16(a)) return (size_t)a.n * (part_columns(a.r) * 6 + 4);  // three parts, and the factors
    const size_t h = (size_t)a.n * a.r * 4;
    return rounded(h) + (a.ksplit > 1 ? rounded(a.ksplit * h) : 0) + (copies_rows(a, f16) ? (size_t)a.n * a.K * (f16 ? 2 : 4) : 0);
}

hipError_t launch_lora(LoraArgs a, bool f16, void* work, hipStream_t s) {
    a.H = static_cast<float*>(work);
    if (!f16 || !vec16(a)) {
        const size_t h = (size_t)a.n * a.r * 4;
        char* const slabs = static_cast<char*>(work) + rounded(h);
        return launch_any(a, f16, reinterpret_cast<float*>(slabs), slabs + (a.ksplit > 1 ? rounded(a.ksplit * h) : 0), s);
    }
    a.Hs = static_cast<_Float16*>(work);
    a.factor = reinterpret_cast<float*>(a.Hs + (size_t)a.n * 3 * part_columns(a.r));
    if (a.r <= 16) return launch_f16<16, 64>(a, s);
    if (a.r <= 32) return launch_f16<32, 64>(a, s);
    if (a.r <= 64) return launch_f16<64, 64>(a, s);
    return launch_f16<128, 32>(a, s);
}

}  // namespace vedic
