// vedic_paged_plan.hip -- where the items of each 64 sequences begin (vedic_paged.hpp), for calls of so many that every
// workgroup's own walk over all lengths would take longest: with it, the work of a call grows with the square of its sequences.
//
// One workgroup: sums over blocks of 64 sequences, a wave a block, then the sums before each block, a wave an array.
#include "vedic_paged.hpp"

namespace vedic {

namespace {

constexpr int kWaves = 16;

template <int ROWS, bool MANY, int UNIT>
__global__ void __launch_bounds__(64 * kWaves) paged_plan_kernel(PagedArgs a, int* plan) {
    __shared__ float part[kWaves];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int blocks = (a.c.B + 63) >> 6;
    int chunk = INT32_MAX;
    if (a.target > 0) {
        float total = 0.0f;
        for (int b = wave; b < blocks; b += kWaves) {
            const SequenceWork w = sequence_work<ROWS, MANY>(a, 64 * b + lane);
            total += (float)w.tiles * (float)w.span;
        }
        total = wave_total(total);
        if (lane == 0) part[wave] = total;
        __syncthreads();
        total = 0.0f;
#pragma unroll
        for (int i = 0; i < kWaves; ++i) total += part[i];
        chunk = part_keys<UNIT>(a, total);
    }
    if (threadIdx.x == 0) plan[0] = chunk;
    for (int b = wave; b < blocks; b += kWaves) {
        const SequenceUnits u(a, sequence_work<ROWS, MANY>(a, 64 * b + lane), chunk);
        const int sums[3] = {lane_sums(u.items), lane_sums(u.split_tiles), lane_sums(u.split_items)};
#pragma unroll
        for (int i = 0; i < 3; ++i)
            if (lane == 63) plan[1 + i * blocks + b] = min(sums[i], 1 << 24);  // (all of a call are fewer)
    }
    __syncthreads();
    if (wave >= 3) return;
    int* sums = plan + 1 + wave * blocks;
    int before = 0;
    for (int b = 0; b < blocks; b += 64) {
        const int v = b + lane < blocks ? sums[b + lane] : 0, incl = lane_sums(v);
        if (b + lane < blocks) sums[b + lane] = before + incl - v;
        before = min(before + __builtin_amdgcn_readlane(incl, 63), 1 << 29);
    }
}

}  // namespace

hipError_t launch_paged_plan(const PagedArgs& a, bool many, int* plan, hipStream_t s) {
    if (many) paged_plan_kernel<kManyRows, true, kManyUnit><<<1, 64 * kWaves, 0, s>>>(a, plan);
    else paged_plan_kernel<kFewRows, false, kFewUnit><<<1, 64 * kWaves, 0, s>>>(a, plan);
    return hipGetLastError();
}

}  // namespace vedic
