// vedic_paged_few_f16.hip -- paged_few_kernel over a binary16 cache.
#include "vedic_paged_few.hpp"

namespace vedic {

hipError_t launch_paged_few_f16(const PagedArgs& a, hipStream_t s) { return paged_few<false>(a, s); }

}  // namespace vedic
