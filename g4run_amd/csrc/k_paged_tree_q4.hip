// k_paged_tree_q4.hip -- k_paged_tree (paged_tree.h) over Q4_0 pages
#include "paged_tree.h"

namespace g4 {

hipError_t pa_tree_q4(const PagedAttn &a, const PagedPlan &pl, bool wide, hipStream_t s) { return pa_tree<Q4_0>(a, pl, wide, s); }

}  // namespace g4
