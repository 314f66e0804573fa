// vedic_w4_tile.hip -- Y[M x N] = epi(X[M x K] . W[K x N]) with W held in four bits, in tiles for many rows.
//
// A workgroup's four waves take a tile of BM x 128, BM / 2 x 64 each, in steps of 64 values of K.  X's rows go straight
// to LDS, ST - 1 steps ahead (16-byte pieces, their places swapped by row so that a fragment's read meets every bank
// once), the codes and their pairs too, two steps at a time: a column's codes lie K / 2 bytes from the next one's, and the rate
// at which cache lines are touched bounds what loads them straight to registers (both wave rows, 16 bytes a line; 2048
// rows of 4096 into 16384: 371 us with BM = 128, 308 so).  In v_mfma_f32_32x32x16_f16 a lane has eight values of one column,
// which is one word, and the order of K is free as long as both sides agree: lanes 0 .. 31 multiply the step's words 0 .. 3,
// lanes 32 .. 63 its words 4 .. 7, read as one 16-byte piece and expanded a word a product (13 instructions,
// beside BM / 64 matrix instructions).
//
// Bound by a wave's own issue where tiles are few (a step of 128 rows 0.48 us, its matrix instructions alone 0.26: they
// and the expanding take turns more than they overlap); with every CU at it 600 to 950 TFLOP/s by K (2048 rows of 4096 into
// 16384 290 us, 8192 of 2048 into 1024 47), and what surrounds the steps: 7 us a launch with its first loads, GELU and stores.
//
// The sums pass through LDS by 32 rows, so that a lane has eight consecutive columns for the bias, GELU and stores of
// 16 bytes.
#include "vedic_gemm_f16.hpp"
#include "vedic_w4.hpp"

namespace vedic {

namespace {

constexpr int kBN = 128;
[[maybe_unused]] constexpr int kBK = 64;

// ST: X's places in LDS (3, or more where a CU has one workgroup only).
template <int BM, int ST>
__global__ void __launch_bounds__(256) w4_tile_kernel(W4Args a, int shift, int tm, int tn) {
#ifdef __HIP_DEVICE_COMPILE__  // (the host's pass drops the launch stub of a body that makes buffer resources in lambdas)
    constexpr int MI = BM / 64, AHEAD = ST / 2, RING = AHEAD + 1;
    using SideX = Side<true, BM, kBK, 4>;
    using SideC = Side<true, kBN, 32, 4>;  // 16 words a column, 128 values of K
    constexpr int STAGE = SideX::BYTES, PAIRS = kBN * 4 * 4, OUT = 4 * 32 * 68 * 4;
    __shared__ __attribute__((aligned(16))) char lds[ST * STAGE + RING * (SideC::BYTES + PAIRS)];
    static_assert(sizeof(lds) >= OUT && sizeof(lds) <= 160 * 1024, "LDS");
    char* lds_codes = lds + ST * STAGE;
    char* lds_pairs = lds_codes + RING * SideC::BYTES;
    const W4View& w = a.w;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r = lane & 31, h = lane >> 5;

    // Tiles of neighbouring workgroups of one L2 (every eighth) go two rows by as many columns as there are.
    const int tiles = tm * tn, x = blockIdx.x & 7, each = tiles >> 3, rest = tiles & 7;
    const int t = x * each + min(x, rest) + (blockIdx.x >> 3);
    const int pair = t / (2 * tn), in = t - pair * 2 * tn;
    const bool two = 2 * pair + 1 < tm;
    const int m0 = (2 * pair + (two ? in & 1 : 0)) * BM, n0 = (two ? in >> 1 : in) * kBN;
    const int K = w.K, steps = (K + kBK - 1) / kBK;

    SideX sx;
    sx.init(wave, lane, a.ldx, m0, a.M);
    const _Float16* tile = static_cast<const _Float16*>(a.X) + (int64_t)m0 * a.ldx;
    // X's rows of step s; TAIL: any K (X has zeros from K to the next multiple of eight), else steps that lie in K or
    // behind it as a whole (a resource without records then: zeros), which takes no vector instruction.
    auto load_x = [&](auto tail, int s, int place) {
        char* to = lds + place;
        const _Float16* from = tile + (int64_t)s * kBK;
        if constexpr (tail) {
            sx.load(from, to, wave, lane, (K + 7) / 8 * 8 - s * kBK);
        } else {
            const __amdgpu_buffer_rsrc_t rs =
                __builtin_amdgcn_make_buffer_rsrc(const_cast<_Float16*>(from), 0, s < steps ? 0x7FFFFFFF : 0, 0x00020000);
#pragma unroll
            for (int i = 0; i < SideX::NLD; ++i)
                __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (lds_void_t*)(to + (wave * SideX::NLD + i) * 1024), 16, sx.off[i], 0, 0, 0);
        }
    };
    // Codes of steps 2 d and 2 d + 1, and four pairs a column, one per 32 values (a larger group's more than once).
    SideC sc;
    sc.init(wave, lane, 2 * (int64_t)w.words, n0, w.N);
    const _Float16* codes = reinterpret_cast<const _Float16*>(w.codes + (int64_t)n0 * w.words);
    const __amdgpu_buffer_rsrc_t rp = buffer_rsrc(w.sm + (int64_t)n0 * w.G);
    uint32_t pair_at[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int col = (wave * 2 + i) * 16 + (lane >> 2);
        pair_at[i] = n0 + col < w.N ? (uint32_t)col * w.G * 4u : kOob;
    }
    auto load_codes = [&](int d, int place) {
        sc.load(codes + (int64_t)d * 32, lds_codes + place * SideC::BYTES, wave, lane, 2 * w.words - 32 * d);
        const int chunk = 4 * d + (lane & 3);
#pragma unroll
        for (int i = 0; i < 2; ++i)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rp, (lds_void_t*)(lds_pairs + place * PAIRS + (wave * 2 + i) * 256), 4,
                                                     32 * chunk < K ? pair_at[i] + 4u * (chunk >> shift) : kOob, 0, 0, 0);
    };
    constexpr int CODES = SideC::NLD + 2;  // loads
    struct Codes {
        u32x4_t c[2];
        uint32_t p[2];
    };
    // (column 64 (wave mod 2) + 32 j + r, piece 2 odd + h of its four: of two steps)
    const int code_col = 64 * (wave & 1) + r;
    const int code_at[2] = {code_col * 64 + ((h ^ swz_kc<4>(code_col)) << 4), code_col * 64 + (((2 + h) ^ swz_kc<4>(code_col)) << 4)};
    auto read_codes = [&](auto odd, int place, Codes& b) {
        const char* pc = lds_codes + place * SideC::BYTES + code_at[odd];
        const char* pp = lds_pairs + place * PAIRS + code_col * 16 + 4 * h;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            b.c[j] = *reinterpret_cast<const u32x4_t*>(pc + 32 * 64 * j);
            b.p[j] = *reinterpret_cast<const uint32_t*>(pp + 32 * 16 * j + 8 * odd);
        }
    };
    const FourBits expand;
    // Word q of a step; TAIL: zeros from K on.
    auto values = [&](auto tail, const Codes& b, int s, int q, half8_t (&v)[2]) {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            half2_t sc, m;
            four_bit_pair(b.p[j], sc, m);
            v[j] = expand(b.c[j][q], sc, m);
            if constexpr (tail) {
                const int left = K - s * kBK - 32 * h - 8 * q;
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (e >= left) v[j][e] = (_Float16)0.0f;
            }
        }
    };
    const int xr = BM / 2 * (wave >> 1);
    int row_at[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) row_at[q] = (xr + r) * 128 + (((4 * h + q) ^ swz_kc<8>(r)) << 4);
    auto rows = [&](int place, int q, half8_t (&v)[MI]) {
        const char* p = lds + place + row_at[q];
#pragma unroll
        for (int i = 0; i < MI; ++i) v[i] = *reinterpret_cast<const half8_t*>(p + 32 * 128 * i);
    };

    float16_t acc[MI][2];
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.0f;

    constexpr std::integral_constant<bool, true> yes{};
    constexpr std::integral_constant<bool, false> no{};
    half8_t xv[2][MI], wv[2][2];
    // The products of fragments q, beside what was written before them in their block: each matrix instruction followed by
    // its share of that (a wave issues in order).
    auto multiply = [&](auto loads, int q) {
#pragma unroll
        for (int i = 0; i < MI; ++i)
#pragma unroll
            for (int j = 0; j < 2; ++j)
                acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(xv[q & 1][i], wv[q & 1][j], acc[i][j], 0, 0, 0);
#pragma unroll
        for (int i = 0; i < 2 * MI; ++i) {
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);                  // matrix
            __builtin_amdgcn_sched_group_barrier(0x100, loads ? 2 : 1, 0);      // LDS read
            __builtin_amdgcn_sched_group_barrier(0x002, 28 / (2 * MI), 0);      // vector
            if constexpr (loads) __builtin_amdgcn_sched_group_barrier(0x010, MI == 2 ? 2 : 1, 0);  // loads
        }
        __builtin_amdgcn_sched_barrier(0);
    };
    // A step: the fragments of its next products are read and expanded beside the present ones; half way, the next
    // step's rows and codes have arrived (wait, barrier) and the places of the step before this one are free.  Issued
    // after those rows, and perhaps under way: the loads of ST - 3 steps, NLD of rows each, and of codes in the even ones.
    // (x0, x1, x2: bytes to X's places of the step before, of this and of the next one; d0, d1, d2: the codes' places, by two steps;
    // counted along, since the remainder by 3 or 5 would take vector instructions for every address)
    int x0 = (ST - 1) * STAGE, x1 = 0, x2 = STAGE, d0 = RING - 1, d1 = 0, d2 = 1;
    auto step = [&](auto tail, auto odd, int s, Codes& now, Codes& next) {
        rows(x1, 1, xv[1]);
        values(tail, now, s, 1, wv[1]);
        if constexpr (!odd) load_codes((s >> 1) + AHEAD, d0);
        multiply(no, 0);
        rows(x1, 2, xv[0]);
        values(tail, now, s, 2, wv[0]);
        multiply(no, 1);
        asm volatile("" ::: "memory");
        wait_vmcnt<(ST - 3) * SideX::NLD + (ST - 2 + !odd) / 2 * CODES>();
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        rows(x1, 3, xv[1]);
        if constexpr (odd) read_codes(no, d2, next);
        else read_codes(yes, d1, next);
        values(tail, now, s, 3, wv[1]);
        load_x(tail, s + ST - 1, x0);
        multiply(yes, 2);
        rows(x2, 0, xv[0]);
        values(tail, next, s + 1, 0, wv[0]);
        multiply(no, 3);
        x0 = x1;
        x1 = x2;
        x2 = x2 == (ST - 1) * STAGE ? 0 : x2 + STAGE;
        if constexpr (odd) {
            d0 = d1;
            d1 = d2;
            d2 = d2 == RING - 1 ? 0 : d2 + 1;
        }
    };
    // The loads in the steps' order, as if ST - 1 steps had been before.
    if constexpr (ST % 2 == 0) load_codes(0, 0);
#pragma unroll
    for (int i = 0; i < ST - 1; ++i) {
        constexpr int FIRST = ST - 1;
        if ((FIRST - i) % 2 == 0) load_codes((i - FIRST) / 2 + AHEAD, (i - FIRST) / 2 + AHEAD);
        load_x(yes, i, i * STAGE);
        asm volatile("" ::: "memory");
    }
    wait_vmcnt<(ST - 2) * SideX::NLD + (ST - 2) / 2 * CODES>();
    stage_barrier();
    Codes c0, c1;
    rows(0, 0, xv[0]);
    read_codes(no, 0, c0);
    values(yes, c0, 0, 0, wv[0]);
    // Steps without masks: all of a K of whole steps (but an odd last one), else those whose loads lie within K.
    const int plain = (K % kBK == 0 ? steps : max(K / kBK - ST + 1, 0)) & ~1;
    for (int s = 0; s < plain; s += 2) {
        step(no, no, s, c0, c1);
        step(no, yes, s + 1, c1, c0);
    }
    for (int s = plain; s < steps; s += 2) {
        step(yes, no, s, c0, c1);
        step(yes, yes, s + 1, c1, c0);
    }
    wait_vmcnt<0>();
    __syncthreads();

    // A wave's 32 x 64 block in rows of 68 sums, then a lane's eight columns of row 8 it + lane / 8.
    float* out = reinterpret_cast<float*>(lds) + wave * 32 * 68;
    const int n = n0 + 64 * (wave & 1) + 8 * (lane & 7);
    float bias[8];
#pragma unroll
    for (int c = 0; c < 8; ++c) bias[c] = a.bias && n + c < w.N ? a.bias[n + c] : 0.0f;
    const bool whole = n + 8 <= w.N && a.ldc % 8 == 0 && ((uintptr_t)a.C & 15) == 0;
#pragma unroll
    for (int i = 0; i < MI; ++i) {
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e) out[(8 * (e >> 2) + 4 * h + (e & 3)) * 68 + 32 * j + r] = acc[i][j][e];
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int it = 0; it < 4; ++it) {
            const int row = 8 * it + (lane >> 3), m = m0 + xr + 32 * i + row;
            const float4_t* from = reinterpret_cast<const float4_t*>(out + row * 68 + 8 * (lane & 7));
            float4_t v[2] = {from[0], from[1]};
            if (m >= a.M || n >= w.N) continue;
#pragma unroll
            for (int c = 0; c < 8; ++c) {
                float y = v[c >> 2][c & 3] + bias[c];
                v[c >> 2][c & 3] = a.gelu ? gelu_tanh(y) : y;
            }
            const int64_t to = (int64_t)m * a.ldc + n;
            if (whole) {
                if (a.c16) {
                    half8_t o;
#pragma unroll
                    for (int c = 0; c < 8; ++c) o[c] = (_Float16)v[c >> 2][c & 3];
                    store_half8(static_cast<_Float16*>(a.C) + to, o);
                } else {
                    float* p = static_cast<float*>(a.C) + to;
                    if (a.residual) {
                        v[0] += reinterpret_cast<const float4_t*>(p)[0];
                        v[1] += reinterpret_cast<const float4_t*>(p)[1];
                    }
                    store16_hold(p, v[0]);
                    store16_hold(p + 4, v[1]);
                }
                continue;
            }
#pragma unroll
            for (int c = 0; c < 8; ++c) {
                if (n + c >= w.N) break;
                const float y = v[c >> 2][c & 3];
                if (a.c16) static_cast<_Float16*>(a.C)[to + c] = (_Float16)y;
                else static_cast<float*>(a.C)[to + c] = a.residual ? static_cast<float*>(a.C)[to + c] + y : y;
            }
        }
        __builtin_amdgcn_wave_barrier();
    }
#endif
}

}  // namespace

hipError_t launch_w4_tile(const W4Args& a, int cus, hipStream_t s) {
    const int tn = (a.w.N + kBN - 1) / kBN, low = (a.M + 127) / 128, tall = (a.M + 255) / 256;
    const int shift = a.w.group == 32 ? 0 : a.w.group == 64 ? 1 : 2;
    // 256 rows (twice the products an expanded value) where a tile for every CU and a K of some length are there, else
    // 128: two workgroups a CU, or one with its loads further ahead (us of 256 / two of 128 / one: 8192 rows of 4096 into
    // 1024 84 / 88, 1024 of 4096 into 16384 151 / 159, 2048 of 1024 into 4096 29.0 / 29.6 / 35.4, 8192 103 / 95 / 119, 4096 of
    // 512 into 4096 37.3 / 33.4 / 42.9).
    if ((int64_t)tall * tn >= cus && a.w.K >= 2048) w4_tile_kernel<256, 4><<<(unsigned)(tall * tn), 256, 0, s>>>(a, shift, tall, tn);
    else if ((int64_t)low * tn > cus) w4_tile_kernel<128, 3><<<(unsigned)(low * tn), 256, 0, s>>>(a, shift, low, tn);
    else w4_tile_kernel<128, 5><<<(unsigned)(low * tn), 256, 0, s>>>(a, shift, low, tn);
    return hipGetLastError();
}

}  // namespace vedic
