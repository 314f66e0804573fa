// vedic_grouped_any_nt.hip -- the any-alignment grouped products, op NT.
#include "vedic_grouped_any.hpp"

namespace vedic {

template __global__ void grouped_any_kernel<1, float, float, false, 128, 128, 2, 2, GK_LINEAR>(GroupedArgs);
template __global__ void grouped_any_kernel<1, float, float, false, 64, 64, 2, 1, GK_LINEAR>(GroupedArgs);
template __global__ void grouped_any_kernel<1, _Float16, float, false, 128, 128, 2, 2, GK_LINEAR>(GroupedArgs);
template __global__ void grouped_any_kernel<1, _Float16, float, false, 64, 64, 2, 1, GK_LINEAR>(GroupedArgs);
template __global__ void grouped_any_kernel<1, float, float, true, 128, 128, 2, 2, GK_LINEAR>(GroupedArgs);
template __global__ void grouped_any_kernel<1, float, float, true, 64, 64, 2, 1, GK_LINEAR>(GroupedArgs);
template __global__ void grouped_any_kernel<1, _Float16, _Float16, false, 128, 128, 2, 2, GK_LINEAR>(GroupedArgs);
template __global__ void grouped_any_kernel<1, _Float16, _Float16, false, 64, 64, 2, 1, GK_LINEAR>(GroupedArgs);
template __global__ void grouped_any_kernel<1, float, float, false, 128, 128, 2, 2, GK_GELU_BWD>(GroupedArgs);
template __global__ void grouped_any_kernel<1, float, float, false, 64, 64, 2, 1, GK_GELU_BWD>(GroupedArgs);
template __global__ void grouped_any_kernel<1, _Float16, float, false, 128, 128, 2, 2, GK_GELU_BWD>(GroupedArgs);
template __global__ void grouped_any_kernel<1, _Float16, float, false, 64, 64, 2, 1, GK_GELU_BWD>(GroupedArgs);
template __global__ void grouped_any_kernel<1, float, float, true, 128, 128, 2, 2, GK_GELU_BWD>(GroupedArgs);
template __global__ void grouped_any_kernel<1, float, float, true, 64, 64, 2, 1, GK_GELU_BWD>(GroupedArgs);
template __global__ void grouped_any_kernel<1, _Float16, _Float16, false, 128, 128, 2, 2, GK_GELU_BWD>(GroupedArgs);
template __global__ void grouped_any_kernel<1, _Float16, _Float16, false, 64, 64, 2, 1, GK_GELU_BWD>(GroupedArgs);

hipError_t launch_grouped_any_nt(const GroupedArgs& a, int kind, bool f16, bool f16out, bool vec, hipStream_t s) {
    if (kind == GK_GELU_BWD) return launch_any_kind<1, GK_GELU_BWD>(a, f16, f16out, vec, s);
    return launch_any_kind<1, GK_LINEAR>(a, f16, f16out, vec, s);
}

}  // namespace vedic
