// vedic_route.hpp -- launch interface of the router (vedic_route.hip).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "vedic_grouped.hpp"

namespace vedic {

constexpr int kMaxTopK = 64;

struct RouteArgs {
    const float* logits;  // [T x ld]
    int64_t ld;
    int T, E, k;
    int renorm;
    int* ids;        // [T x k]
    float* weights;  // [T x k]
    int* offsets;    // [E + 1]
    int* rows;       // [T k]
    int* slots;      // [T x k]
    int* counts;     // route_count_bytes() of workspace
    int bits, tokens;  // set by the launch
    bool wide;         // 16-byte loads of the logits
};

size_t route_count_bytes(int64_t T, int E, int k);
hipError_t launch_route_topk(RouteArgs a, hipStream_t s);
size_t group_count_bytes(int64_t n, int groups);
hipError_t launch_group_rows(const int* ids, int n, int per_row, int groups, int* counts, int* offsets, int* rows, int* slots,
                             hipStream_t s);
hipError_t launch_route_topk_bwd(const float* logits, int64_t ld, const int* ids, const float* weights, const float* dweights,
                                 int T, int E, int k, int renorm, float* out, int64_t ldo, hipStream_t s);

}  // namespace vedic
