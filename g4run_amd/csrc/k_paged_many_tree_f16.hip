// k_paged_many_tree_f16.hip -- k_paged_many (paged_many.h) over trees of new tokens and F16 pages
#include "paged_many.h"

namespace g4 {

hipError_t pa_many_tree_f16(const PagedAttn &a, const PagedPlan &pl, hipStream_t s) { return pa_many<F16, true>(a, pl, s); }

}  // namespace g4
