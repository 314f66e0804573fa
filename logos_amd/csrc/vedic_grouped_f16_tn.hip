// vedic_grouped_f16_tn.hip -- the grouped binary16 products, op TN.
#include "vedic_grouped_f16.hpp"

namespace vedic {

VEDIC_GROUPED_INSTANTIATE_TN(GK_LINEAR);
VEDIC_GROUPED_INSTANTIATE_TN(GK_BETA);

hipError_t launch_grouped_f16_tn(const GroupedArgs& a, int kind, bool /*f16out*/, hipStream_t s) {
    if (kind == GK_BETA) return launch_grouped_tiles<2, GK_BETA, float>(a, s);
    return launch_grouped_tiles<2, GK_LINEAR, float>(a, s);
}

}  // namespace vedic
