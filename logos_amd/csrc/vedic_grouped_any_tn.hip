// vedic_grouped_any_tn.hip -- the any-alignment grouped products, op TN.
#include "vedic_grouped_any.hpp"

namespace vedic {

template __global__ void grouped_any_kernel<2, float, float, false, 128, 128, 2, 2, GK_LINEAR>(GroupedArgs);
template __global__ void grouped_any_kernel<2, float, float, false, 64, 64, 2, 1, GK_LINEAR>(GroupedArgs);
template __global__ void grouped_any_kernel<2, _Float16, float, false, 128, 128, 2, 2, GK_LINEAR>(GroupedArgs);
template __global__ void grouped_any_kernel<2, _Float16, float, false, 64, 64, 2, 1, GK_LINEAR>(GroupedArgs);
template __global__ void grouped_any_kernel<2, float, float, false, 128, 128, 2, 2, GK_BETA>(GroupedArgs);
template __global__ void grouped_any_kernel<2, float, float, false, 64, 64, 2, 1, GK_BETA>(GroupedArgs);
template __global__ void grouped_any_kernel<2, _Float16, float, false, 128, 128, 2, 2, GK_BETA>(GroupedArgs);
template __global__ void grouped_any_kernel<2, _Float16, float, false, 64, 64, 2, 1, GK_BETA>(GroupedArgs);

hipError_t launch_grouped_any_tn(const GroupedArgs& a, int kind, bool f16, bool f16out, bool vec, hipStream_t s) {
    if (kind == GK_BETA) return launch_any_kind<2, GK_BETA>(a, f16, f16out, vec, s);
    return launch_any_kind<2, GK_LINEAR>(a, f16, f16out, vec, s);
}

}  // namespace vedic
