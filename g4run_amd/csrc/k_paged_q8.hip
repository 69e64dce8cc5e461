// k_paged_q8.hip -- attention over the paged KV cache, Q8_0 pages (paged_attn.h)
#include "paged_attn.h"

namespace g4 {

hipError_t pa_launch_q8(const PagedAttn &a, const PagedPlan &pl, int v, unsigned blocks, hipStream_t s) {
    return pa_launch<Q8_0>(a, pl, v, blocks, s);
}

}  // namespace g4
