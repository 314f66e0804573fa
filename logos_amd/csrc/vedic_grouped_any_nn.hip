// vedic_grouped_any_nn.hip -- the any-alignment grouped products, op NN.
#include "vedic_grouped_any.hpp"

namespace vedic {

template __global__ void grouped_any_kernel<0, float, float, false, 128, 128, 2, 2, GK_LINEAR>(GroupedArgs);
template __global__ void grouped_any_kernel<0, float, float, false, 64, 64, 2, 1, GK_LINEAR>(GroupedArgs);
template __global__ void grouped_any_kernel<0, _Float16, float, false, 128, 128, 2, 2, GK_LINEAR>(GroupedArgs);
template __global__ void grouped_any_kernel<0, _Float16, float, false, 64, 64, 2, 1, GK_LINEAR>(GroupedArgs);
template __global__ void grouped_any_kernel<0, float, float, true, 128, 128, 2, 2, GK_LINEAR>(GroupedArgs);
template __global__ void grouped_any_kernel<0, float, float, true, 64, 64, 2, 1, GK_LINEAR>(GroupedArgs);
template __global__ void grouped_any_kernel<0, _Float16, _Float16, false, 128, 128, 2, 2, GK_LINEAR>(GroupedArgs);
template __global__ void grouped_any_kernel<0, _Float16, _Float16, false, 64, 64, 2, 1, GK_LINEAR>(GroupedArgs);
template __global__ void grouped_any_kernel<0, float, float, false, 128, 128, 2, 2, GK_GELU>(GroupedArgs);
template __global__ void grouped_any_kernel<0, float, float, false, 64, 64, 2, 1, GK_GELU>(GroupedArgs);
template __global__ void grouped_any_kernel<0, _Float16, float, false, 128, 128, 2, 2, GK_GELU>(GroupedArgs);
template __global__ void grouped_any_kernel<0, _Float16, float, false, 64, 64, 2, 1, GK_GELU>(GroupedArgs);
template __global__ void grouped_any_kernel<0, float, float, true, 128, 128, 2, 2, GK_GELU>(GroupedArgs);
template __global__ void grouped_any_kernel<0, float, float, true, 64, 64, 2, 1, GK_GELU>(GroupedArgs);
template __global__ void grouped_any_kernel<0, _Float16, _Float16, false, 128, 128, 2, 2, GK_GELU>(GroupedArgs);
template __global__ void grouped_any_kernel<0, _Float16, _Float16, false, 64, 64, 2, 1, GK_GELU>(GroupedArgs);
template __global__ void grouped_any_kernel<0, float, float, false, 128, 128, 2, 2, GK_GELU_P>(GroupedArgs);
template __global__ void grouped_any_kernel<0, float, float, false, 64, 64, 2, 1, GK_GELU_P>(GroupedArgs);
template __global__ void grouped_any_kernel<0, _Float16, float, false, 128, 128, 2, 2, GK_GELU_P>(GroupedArgs);
template __global__ void grouped_any_kernel<0, _Float16, float, false, 64, 64, 2, 1, GK_GELU_P>(GroupedArgs);
template __global__ void grouped_any_kernel<0, float, float, true, 128, 128, 2, 2, GK_GELU_P>(GroupedArgs);
template __global__ void grouped_any_kernel<0, float, float, true, 64, 64, 2, 1, GK_GELU_P>(GroupedArgs);
template __global__ void grouped_any_kernel<0, _Float16, _Float16, false, 128, 128, 2, 2, GK_GELU_P>(GroupedArgs);
template __global__ void grouped_any_kernel<0, _Float16, _Float16, false, 64, 64, 2, 1, GK_GELU_P>(GroupedArgs);

hipError_t launch_grouped_any_nn(const GroupedArgs& a, int kind, bool f16, bool f16out, bool vec, hipStream_t s) {
    if (kind == GK_GELU) return launch_any_kind<0, GK_GELU>(a, f16, f16out, vec, s);
    if (kind == GK_GELU_P) return launch_any_kind<0, GK_GELU_P>(a, f16, f16out, vec, s);
    return launch_any_kind<0, GK_LINEAR>(a, f16, f16out, vec, s);
}

}  // namespace vedic
