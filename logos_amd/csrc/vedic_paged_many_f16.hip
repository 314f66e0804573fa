// vedic_paged_many_f16.hip -- paged_many_kernel over a binary16 cache.
#include "vedic_paged_many.hpp"

namespace vedic {

hipError_t launch_paged_many_f16(const PagedArgs& a, hipStream_t s) { return paged_many<false>(a, s); }

}  // namespace vedic
