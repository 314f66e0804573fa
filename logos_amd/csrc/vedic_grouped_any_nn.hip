// vedic_grouped_any_nn.hip -- the any-alignment grouped products, op NN.
#include "vedic_grouped_any.hpp"

namespace vedic {

VEDIC_ANY_KERNELS(0, float, float, float, GK_LINEAR);
VEDIC_ANY_KERNELS(0, _Float16, _Float16, float, GK_LINEAR);
VEDIC_ANY_KERNELS(0, _Float16, _Float16, _Float16, GK_LINEAR);
VEDIC_ANY_KERNELS(0, float, float, float, GK_GELU);
VEDIC_ANY_KERNELS(0, _Float16, _Float16, float, GK_GELU);
VEDIC_ANY_KERNELS(0, _Float16, _Float16, _Float16, GK_GELU);
VEDIC_ANY_KERNELS(0, float, float, float, GK_GELU_P);
VEDIC_ANY_KERNELS(0, _Float16, _Float16, float, GK_GELU_P);
VEDIC_ANY_KERNELS(0, _Float16, _Float16, _Float16, GK_GELU_P);
VEDIC_ANY_KERNELS(0, float, float, float, GK_ADD);
VEDIC_ANY_KERNELS(0, float, _Float16, float, GK_ADD);

hipError_t launch_grouped_any_nn(const GroupedArgs& a, int kind, bool f16, bool f16out, hipStream_t s) {
    if (kind == GK_GELU) return launch_any_kind<0, GK_GELU>(a, f16, f16out, s);
    if (kind == GK_GELU_P) return launch_any_kind<0, GK_GELU_P>(a, f16, f16out, s);
    // (the adapters' second product: fp32 A; f16: a binary16 B)
    if (kind == GK_ADD)
        return f16 ? launch_any_tiles<0, float, _Float16, float, GK_ADD>(a, s)
                   : launch_any_tiles<0, float, float, float, GK_ADD>(a, s);
    return launch_any_kind<0, GK_LINEAR>(a, f16, f16out, s);
}

}  // namespace vedic
