// vedic_paged_few_i4.hip -- paged_few_kernel over a four-bit cache.
#include "vedic_paged_few.hpp"

namespace vedic {

hipError_t launch_paged_few_i4(const PagedArgs& a, hipStream_t s) { return paged_few<true>(a, s); }

}  // namespace vedic
