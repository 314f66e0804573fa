// vedic_w4.hpp -- weights held in four bits: launch interface of vedic_w4.hip.
#pragma once

#include "vedic_cache.hpp"

namespace vedic {

// Column n of the weight: `words` words of eight codes (K rounded up to a multiple of 32; four-bit words
// of vedic_cache.hpp), and G = ceil(K / group) pairs (s, m).
struct W4View {
    const uint32_t* codes;  // [N x words]
    const uint32_t* sm;     // [N x G] pairs
    int K, N, group;
    int words, G;
};

struct W4Args {
    W4View w;
    const void* X;
    int64_t ldx;
    int M;
    bool x32;   // X fp32 (clamped and rounded to binary16 as it is read), else binary16
    void* C;
    int64_t ldc;
    bool c16;
    const float* bias;  // or null
    bool gelu, residual;
};
constexpr int kW4FewRows = 64;  // rows of a workgroup of the few-row kernel
hipError_t launch_w4_few(const W4Args& a, int cus, hipStream_t s);
// Many rows: X binary16 in whole 16 bytes (K and ldx multiples of 8, aligned).
hipError_t launch_w4_tile(const W4Args& a, int cus, hipStream_t s);
// Binary16 rows n0 .. n0 + n - 1 of the transposed weight, [n x 8 words], zeros from K on.
hipError_t launch_w4_expand(const W4View& w, int n0, int n, _Float16* out, hipStream_t s);
// X as binary16 [M x ld], zeros from K on.
hipError_t launch_w4_rows(const void* X, bool x32, int64_t ldx, int M, int K, _Float16* out, int64_t ld, hipStream_t s);
hipError_t launch_w4_quantize(const void* W, bool f32, int64_t ldw, const W4View& w, uint32_t* codes, uint32_t* sm,
                              hipStream_t s);
hipError_t launch_w4_unpack(const W4View& w, _Float16* out, int64_t ld, hipStream_t s);

}  // namespace vedic
