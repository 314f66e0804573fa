// vedic_grouped_f16_nt.hip -- the grouped binary16 products, op NT.
#include "vedic_grouped_f16.hpp"

namespace vedic {

VEDIC_GROUPED_INSTANTIATE(1, GK_LINEAR, float);
VEDIC_GROUPED_INSTANTIATE(1, GK_LINEAR, _Float16);
VEDIC_GROUPED_INSTANTIATE(1, GK_GELU_BWD, float);
VEDIC_GROUPED_INSTANTIATE(1, GK_GELU_BWD, _Float16);

hipError_t launch_grouped_f16_nt(const GroupedArgs& a, int kind, bool f16out, hipStream_t s) {
    if (kind == GK_GELU_BWD) return f16out ? launch_grouped_tiles<1, GK_GELU_BWD, _Float16>(a, s) : launch_grouped_tiles<1, GK_GELU_BWD, float>(a, s);
    return f16out ? launch_grouped_tiles<1, GK_LINEAR, _Float16>(a, s) : launch_grouped_tiles<1, GK_LINEAR, float>(a, s);
}

}  // namespace vedic
