// k_paged_f16.hip -- attention over the paged KV cache, F16 pages (paged_attn.h)
#include "paged_attn.h"

namespace g4 {

hipError_t pa_launch_f16(const PagedAttn &a, const PagedPlan &pl, int v, unsigned blocks, hipStream_t s) {
    return pa_launch<F16>(a, pl, v, blocks, s);
}

}  // namespace g4
