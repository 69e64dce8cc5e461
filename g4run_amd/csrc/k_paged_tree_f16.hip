// k_paged_tree_f16.hip -- k_paged_tree (paged_tree.h) over F16 pages
#include "paged_tree.h"

namespace g4 {

hipError_t pa_tree_f16(const PagedAttn &a, const PagedPlan &pl, bool wide, hipStream_t s) { return pa_tree<F16>(a, pl, wide, s); }

}  // namespace g4
