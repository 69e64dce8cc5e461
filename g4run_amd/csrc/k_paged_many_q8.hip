// k_paged_many_q8.hip -- k_paged_many (paged_many.h) over Q8_0 pages
#include "paged_many.h"

namespace g4 {

hipError_t pa_many_q8(const PagedAttn &a, const PagedPlan &pl, hipStream_t s) { return pa_many<Q8_0>(a, pl, s); }

}  // namespace g4
