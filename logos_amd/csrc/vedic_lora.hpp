// vedic_lora.hpp -- launch interface of the adapters (vedic_lora.hip).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace vedic {

constexpr int kLoraMaxRank = 128;

struct LoraArgs {
    const void* X;  // [M x ldx]
    int64_t ldx;
    const void* A;  // [groups][K x r]
    const void* B;  // [groups][r x N]
    const int* offsets;
    const int* rows;  // n positions, sorted by adapter
    int n, groups;
    const float* scales;  // [groups], or null: ones
    float* C;             // [M x ldc]
    int64_t ldc;
    int M, K, N, r;
    int ksplit;  // slices of K in H's product, where that is a grouped product
    // set by the launch
    float* H;       // [n x r]
    _Float16* Hs;   // [n][hi, mid, lo]
    float* factor;  // [n]
};

// Whether a launch can have the call's tiles.
bool lora_fits(const LoraArgs& a, bool f16);
// Workspace of a call, and the call (work: that many bytes, 256-byte aligned).
size_t lora_bytes(const LoraArgs& a, bool f16);
hipError_t launch_lora(LoraArgs a, bool f16, void* work, hipStream_t s);

}  // namespace vedic
