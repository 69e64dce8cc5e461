// k_paged_q4.hip -- attention over the paged KV cache, Q4_0 pages (paged_attn.h)
#include "paged_attn.h"

namespace g4 {

hipError_t pa_launch_q4(const PagedAttn &a, const PagedPlan &pl, int v, unsigned blocks, hipStream_t s) {
    return pa_launch<Q4_0>(a, pl, v, blocks, s);
}

}  // namespace g4
