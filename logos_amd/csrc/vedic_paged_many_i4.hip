// vedic_paged_many_i4.hip -- paged_many_kernel over a four-bit cache.
#include "vedic_paged_many.hpp"

namespace vedic {

hipError_t launch_paged_many_i4(const PagedArgs& a, hipStream_t s) { return paged_many<true>(a, s); }

}  // namespace vedic
