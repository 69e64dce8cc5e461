// k_paged.hip -- the paged KV cache's attention call: its launches (split as
// paged_split.h lays out) and the join of the partial results.
#include "paged_split.h"

namespace g4 {

namespace {

// One (token, head) row: out = sum of exp2(m_k - M) O_k / sum of exp2(m_k - M) l_k
// over the row's partial results in a fixed order.  SPLIT: a workgroup per row, or
// per row and 64 elements where those are few (36 rows of 512 from 250 pieces: 36 us,
// 9.6 so; 256 rows of 256 from a few: 5.0 us, 5.5 so), its groups of threads every
// so-many-th result; else a group of hd / 4 threads per row (many rows of few: a
// workgroup's one active group left the chip empty, 9000 rows of 256 took 18 us, now
// 11.4).  Bound by the latency of reads that depend on each other, so: what the
// kernels noted of the row and nothing else, four results' maxima and sums at once
// under a running maximum.
template <bool SPLIT>
__global__ __launch_bounds__(256) void k_paged_join(PagedAttn a, PagedPlan pl) {
    __shared__ float2 ml_of[SPLIT ? 16 : 1];                 // groups: of 16 threads at least
    __shared__ pa_v4f part[SPLIT ? 256 : 1];
    const int hd = a.p.hd, hd4 = hd / 4 / (SPLIT ? gridDim.y : 1), groups = 256 / hd4, gi = threadIdx.x / hd4, e4 = 4 * (threadIdx.x % hd4 + (SPLIT ? hd4 * blockIdx.y : 0));
    const int all = a.b.n_tok * a.n_head, mine = SPLIT ? (int)blockIdx.x : (int)blockIdx.x * groups + gi, row = min(mine, all - 1);   // up to 2^24
    const int tok = row / a.n_head, head = row - tok * a.n_head;
    const uint2 own = pl.own[row], pre = a.b.n_prefix > 0 ? pl.pre[row] : make_uint2(0, 0);
    const int n_pre = pre.x >> 2, n_own = own.x >> 2, total = n_pre + n_own;
    if (mine >= all || n_own == 0) return;
    pa_v4f s = {0.0f, 0.0f, 0.0f, 0.0f};
    float m = -__builtin_inff(), l = 0.0f;
    auto add = [&](float2 x, pa_v4f v, float mn) {
        const float f = x.x == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(x.x - mn);
        l += x.y == x.y ? f * x.y : x.y;                     // a bad page's NaN stays
        s += v * f;
    };
    constexpr int N = 4;
    const int step = SPLIT ? groups : 1;
    for (int k = SPLIT ? gi : 0; k < total; k += N * step) {
        float2 x[N];
        pa_v4f v[N];
#pragma unroll
        for (int j = 0; j < N; j++) {
            const PaPart part = pa_part(a, pl, row, pre, own, min(k + j * step, total - 1));
            x[j] = *part.ml;
            v[j] = *(const pa_v4f *)(part.o + e4);
        }
        float mn = m;
#pragma unroll
        for (int j = 0; j < N; j++) mn = fmaxf(mn, x[j].x);
        const float f = m == -__builtin_inff() ? 1.0f : __builtin_amdgcn_exp2f(m - mn);
        l *= f;
        s *= f;
        m = mn;
#pragma unroll
        for (int j = 0; j < N; j++)
            if (k + j * step < total) add(x[j], v[j], mn);
    }
    if constexpr (SPLIT) {
        part[threadIdx.x] = s;
        if (threadIdx.x % hd4 == 0) ml_of[gi] = make_float2(m, l);
        __syncthreads();
        if (gi) return;
        for (int k = 0; k < groups; k++) m = fmaxf(m, ml_of[k].x);
        s = pa_v4f{0.0f, 0.0f, 0.0f, 0.0f};
        l = 0.0f;
        for (int k = 0; k < groups; k++) add(ml_of[k], part[k * hd4 + threadIdx.x], m);
    }
    const bool none = own.x & 2;
    pa_store4(a.out + (size_t)tok * a.os + (size_t)head * hd + e4, none ? pa_v4f{0.0f, 0.0f, 0.0f, 0.0f} : s * (1.0f / l));
}

}  // namespace

size_t paged_attn_workspace(const PagedPool &p, const PagedBatch &b, int n_head) {
    return b.n_tok == 0 || b.n_seq == 0 ? 0 : paged_layout(p, b, n_head / p.n_kv, 0).total;
}

hipError_t launch_paged_attn(PagedAttn a, hipStream_t s) {
    const PagedPool &p = a.p;
    const PagedBatch &b = a.b;
    if (b.n_tok == 0 || b.n_seq == 0) return hipSuccess;
    a.window = paged_window(b, a.window);
    const PagedLayout y = paged_layout(p, b, a.grp, a.window);
    const PagedPlan pl = paged_places(y, a.ws);
    if (pl.many.rows)
        if (hipError_t e = p.type == F16 ? pa_many_f16(a, pl, s) : p.type == Q8_0 ? pa_many_q8(a, pl, s) : pa_many_q4(a, pl, s)) return e;
    if (pl.few.rows)
        if (hipError_t e = p.type == F16 ? pa_few_f16(a, pl, s) : p.type == Q8_0 ? pa_few_q8(a, pl, s) : pa_few_q4(a, pl, s)) return e;
    if (y.join) {
        const int64_t rows = (int64_t)b.n_tok * a.n_head;
        if (rows <= 2048) hipLaunchKernelGGL(k_paged_join<true>, dim3((unsigned)rows, rows * (p.hd / 64) <= 512 ? p.hd / 64 : 1), dim3(256), 0, s, a, pl);
        else hipLaunchKernelGGL(k_paged_join<false>, dim3(pa_ceil_div(rows, 256 / (p.hd / 4))), dim3(256), 0, s, a, pl);
        return hipGetLastError();
    }
    return hipSuccess;
}

}  // namespace g4
