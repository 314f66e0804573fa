// vedic_grouped_f16_nn.hip -- the grouped binary16 products, op NN.
#include "vedic_grouped_f16.hpp"

namespace vedic {

VEDIC_GROUPED_INSTANTIATE(0, GK_LINEAR, float);
VEDIC_GROUPED_INSTANTIATE(0, GK_LINEAR, _Float16);
VEDIC_GROUPED_INSTANTIATE(0, GK_GELU, float);
VEDIC_GROUPED_INSTANTIATE(0, GK_GELU, _Float16);
VEDIC_GROUPED_INSTANTIATE(0, GK_GELU_P, float);
VEDIC_GROUPED_INSTANTIATE(0, GK_GELU_P, _Float16);

hipError_t launch_grouped_f16_nn(const GroupedArgs& a, int kind, bool f16out, hipStream_t s) {
    if (kind == GK_GELU) return f16out ? launch_grouped_tiles<0, GK_GELU, _Float16>(a, s) : launch_grouped_tiles<0, GK_GELU, float>(a, s);
    if (kind == GK_GELU_P) return f16out ? launch_grouped_tiles<0, GK_GELU_P, _Float16>(a, s) : launch_grouped_tiles<0, GK_GELU_P, float>(a, s);
    return f16out ? launch_grouped_tiles<0, GK_LINEAR, _Float16>(a, s) : launch_grouped_tiles<0, GK_LINEAR, float>(a, s);
}

}  // namespace vedic
