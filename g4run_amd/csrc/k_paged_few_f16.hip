// k_paged_few_f16.hip -- k_paged_few (paged_few.h) over F16 pages
#include "paged_few.h"

namespace g4 {

hipError_t pa_few_f16(const PagedAttn &a, const PagedPlan &pl, hipStream_t s) { return pa_few<F16>(a, pl, s); }

}  // namespace g4
