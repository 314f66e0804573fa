// vedic_grouped_any_tn.hip -- the any-alignment grouped products, op TN.
#include "vedic_grouped_any.hpp"

namespace vedic {

VEDIC_ANY_KERNELS(2, float, float, float, GK_LINEAR);
VEDIC_ANY_KERNELS(2, _Float16, _Float16, float, GK_LINEAR);
VEDIC_ANY_KERNELS(2, float, float, float, GK_BETA);
VEDIC_ANY_KERNELS(2, _Float16, _Float16, float, GK_BETA);

hipError_t launch_grouped_any_tn(const GroupedArgs& a, int kind, bool f16, bool f16out, hipStream_t s) {
    if (kind == GK_BETA) return launch_any_kind<2, GK_BETA>(a, f16, f16out, s);
    return launch_any_kind<2, GK_LINEAR>(a, f16, f16out, s);
}

}  // namespace vedic
