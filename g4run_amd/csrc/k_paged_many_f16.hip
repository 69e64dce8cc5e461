// k_paged_many_f16.hip -- k_paged_many (paged_many.h) over F16 pages
#include "paged_many.h"

namespace g4 {

hipError_t pa_many_f16(const PagedAttn &a, const PagedPlan &pl, hipStream_t s) { return pa_many<F16>(a, pl, s); }

}  // namespace g4
