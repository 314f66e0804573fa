// vedic_grouped_any_nt.hip -- the any-alignment grouped products, op NT.
#include "vedic_grouped_any.hpp"

namespace vedic {

VEDIC_ANY_KERNELS(1, float, float, float, GK_LINEAR);
VEDIC_ANY_KERNELS(1, _Float16, _Float16, float, GK_LINEAR);
VEDIC_ANY_KERNELS(1, _Float16, _Float16, _Float16, GK_LINEAR);
VEDIC_ANY_KERNELS(1, float, float, float, GK_GELU_BWD);
VEDIC_ANY_KERNELS(1, _Float16, _Float16, float, GK_GELU_BWD);
VEDIC_ANY_KERNELS(1, _Float16, _Float16, _Float16, GK_GELU_BWD);

hipError_t launch_grouped_any_nt(const GroupedArgs& a, int kind, bool f16, bool f16out, hipStream_t s) {
    if (kind == GK_GELU_BWD) return launch_any_kind<1, GK_GELU_BWD>(a, f16, f16out, s);
    return launch_any_kind<1, GK_LINEAR>(a, f16, f16out, s);
}

}  // namespace vedic
