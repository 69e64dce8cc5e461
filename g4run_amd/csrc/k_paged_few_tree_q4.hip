// k_paged_few_tree_q4.hip -- k_paged_few (paged_few.h) over trees of new tokens and Q4_0 pages
#include "paged_few.h"

namespace g4 {

hipError_t pa_few_tree_q4(const PagedAttn &a, const PagedPlan &pl, hipStream_t s) { return pa_few<Q4_0, true>(a, pl, s); }

}  // namespace g4
