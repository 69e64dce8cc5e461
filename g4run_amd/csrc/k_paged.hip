// k_paged.hip -- the paged KV cache's attention call: how it is split over the two
// kernels (paged_attn.h), its workspace, and the join of the partial results.
#include <algorithm>

#include "paged_attn.h"

namespace g4 {

namespace {

int ceil_div(int64_t a, int64_t b) { return (int)((a + b - 1) / b); }

struct Layout {
    PagedPlan pl;
    bool join;
    size_t fo, fml, mo, mml, own, pre, wo, wml, total;
};
// window 0 gives the most workspace
Layout layout(const PagedPool &p, const PagedBatch &b, int grp, int window) {
    Layout y;
    PagedPlan &pl = y.pl;
    PagedList &few = pl.few, &many = pl.many;
    const int64_t rows = (int64_t)b.n_tok * grp;             // of one KV head
    pl.grp_inv = 65536 / grp + 1;
    many.toks = 1;
    many.toks_inv = 0;
    // Sequences of at most few.rows rows are the few-row kernel's: 8 (one matrix
    // instruction per operand) where no sequence can have more, else 16.
    // None where sequences have 64 tokens on average: the other kernel then takes the
    // short ones among them too, and a launch is saved (four prompts: 82 -> 77 us).
    few.rows = grp > 16 || (b.q_off && b.n_tok >= 64 * (int64_t)b.n_seq) ? 0 : (b.q_off ? rows : grp) <= 8 ? 8 : 16;
    if (b.n_prefix && few.rows == 8 && rows > 8 && rows <= 16) few.rows = 16;
    few.toks = few.rows / grp;
    const bool few_pre = b.n_prefix && few.rows && rows <= few.rows;
    const bool many_own = b.q_off ? b.n_tok > few.toks : !few.rows;
    const bool many_pre = b.n_prefix && !few_pre;
    few.pre_tiles = few_pre ? 1 : 0;
    // positions a tile attends at most: its first token's window rounded down to
    // 32, and its later tokens
    auto span = [&](int tokens) { return window ? std::min<int64_t>(b.max_len, (int64_t)window + 32 + tokens) : (int64_t)b.max_len; };
    const int64_t fspan = span(16);
    // A step is what a workgroup takes at once (of heads of 512 its four waves share
    // 32 positions; with steps of 128, 16 windows of 1024 took 23.3 us, now 21.7); up to 256 positions stay
    // one step, so that no join is launched for them.  A sequence's tile counts as
    // `lead` steps more, for its queries, first loads and results: 64 sequences of
    // 2000 of 4096 positions, 8 KV heads of 128, 8 bits, take 75 us with a lead of 1, 73
    // with 2, 93 without; a lead of 2 is slower where steps are few (the shares' last
    // step rounded up).  None where every step has its workgroup.
    int64_t steps;
    for (few.shift = b.max_len <= 256 && !b.n_prefix ? 8 : p.hd == 512 ? 5 : p.hd == 256 ? 6 : 7;; few.shift++) {       // counted in 32 bits on the device
        few.unit = 1 << few.shift;
        few.pre_steps = few_pre ? ceil_div(b.n_prefix, few.unit) : 0;
        steps = ((int64_t)b.n_seq * std::max(1, ceil_div(fspan, few.unit)) + few.pre_steps) * p.n_kv;
        if (steps < (1 << 27)) break;
    }
    few.wgs = (int)std::min<int64_t>(256 * pa_few_per_cu(p.type, p.hd, few.rows <= 8), steps);
    few.lead = steps > few.wgs ? 1 : 0;
    y.join = b.n_prefix || (few.rows && fspan > few.unit);
    // Many rows: tiles of whole tokens, up to 128 rows (64 of heads of 512), evenly
    // filled; as many workgroups as fit on the device at once.  Steps of 32 positions,
    // each its workgroup where they are few (24 rows of 256 over 76 positions: 22 us,
    // with shares of 2 at least 29.6), a lead of 5 (four prompts of 509 behind 3800, 4
    // KV heads of 256: 91 us with 2, 83 with 4, 80 with 6; the same order for heads of 64).
    many.rows = 0;
    many.pre_tiles = many.lead = 0;
    if (many_own || many_pre) {
        const int most = paged_most_group(p.hd) / grp, toks = b.q_off || many_pre ? b.n_tok : 1;
        many.toks = ceil_div(toks, ceil_div(toks, most));
        many.toks_inv = many.toks == 1 ? 0 : (uint32_t)(0x100000000ull / many.toks + 1);
        many.rows = many.toks * grp;
        many.pre_tiles = many_pre ? ceil_div(b.n_tok, many.toks) : 0;
        const int64_t own = !many_own ? 0 : b.q_off ? ceil_div(b.n_tok, many.toks) + std::min(b.n_seq, b.n_tok / (few.toks + 1)) : b.n_seq;
        const int64_t mspan = span(many.toks);
        for (many.shift = 5;; many.shift++) {
            many.unit = 1 << many.shift;
            many.pre_steps = many_pre ? ceil_div(b.n_prefix, many.unit) : 0;
            steps = (own * std::max(1, ceil_div(mspan, many.unit)) + (int64_t)many.pre_tiles * many.pre_steps) * p.n_kv;
            if (steps < (1 << 27)) break;
        }
        many.wgs = (int)std::min<int64_t>(p.hd >= 128 ? 256 : 512, steps);
        many.lead = steps > many.wgs ? 5 : 0;
        y.join |= mspan > many.unit;
    }
    const size_t all = y.join ? (size_t)b.n_tok * p.n_kv * grp : 0, whole = b.n_prefix ? all : 0;
    const size_t f = y.join && few.rows ? (size_t)few.wgs * 2 * few.rows : 0, m = y.join && many.rows ? (size_t)many.wgs * 2 * many.rows : 0;
    size_t at = 0;
    auto take = [&](size_t bytes) { const size_t here = at; at += (bytes + 255) & ~(size_t)255; return here; };
    y.fo = take(f * p.hd * 4);
    y.fml = take(f * sizeof(float2));
    y.mo = take(m * p.hd * 4);
    y.mml = take(m * sizeof(float2));
    y.own = take(all * sizeof(uint2));
    y.pre = take(whole * sizeof(uint2));
    y.wo = take(whole * p.hd * 4);
    y.wml = take(whole * sizeof(float2));
    y.total = at;
    return y;
}

// One (token, head) row: out = sum of exp2(m_k - M) O_k / sum of exp2(m_k - M) l_k
// over the row's partial results in a fixed order.  SPLIT: a workgroup per row, or
// per row and 64 elements where those are few (36 rows of 512 from 250 pieces: 36 us,
// 9.6 so; 256 rows of 256 from a few: 5.0 us, 5.5 so), its groups of threads every
// so-many-th result; else a group of hd / 4 threads per row (many rows of few: a
// workgroup's one active group left the chip empty, 9000 rows of 256 took 18 us, now
// 11.4).  Bound by the latency of reads that depend on each other, so: the row's
// sequence by one load of the whole wave, four results' maxima and sums at once
// under a running maximum.
template <bool SPLIT>
__global__ __launch_bounds__(256) void k_paged_join(PagedAttn a, PagedPlan pl) {
    __shared__ float2 ml_of[SPLIT ? 16 : 1];                 // groups: of 16 threads at least
    __shared__ pa_v4f part[SPLIT ? 256 : 1];
    const int hd = a.p.hd, hd4 = hd / 4 / (SPLIT ? gridDim.y : 1), groups = 256 / hd4, gi = threadIdx.x / hd4, e4 = 4 * (threadIdx.x % hd4 + (SPLIT ? hd4 * blockIdx.y : 0));
    const int all = a.b.n_tok * a.n_head, mine = SPLIT ? (int)blockIdx.x : (int)blockIdx.x * groups + gi, row = min(mine, all - 1);   // up to 2^24
    const int tok = row / a.n_head, head = row - tok * a.n_head;
    const uint2 own = pl.own[row], pre = a.b.n_prefix > 0 ? pl.pre[row] : make_uint2(0, 0);      // of a row without a sequence: not used
    int seq = 0;
    if constexpr (SPLIT) seq = paged_find(a.b, tok);
    else {
        const int t1 = __builtin_amdgcn_readlane(tok, 63);   // a wave's rows lie in up to 4 tokens
        for (int t = pa_uniform(tok); t <= t1; t++) {
            const int s = paged_find(a.b, t);
            if (t == tok) seq = s;
        }
    }
    if (mine >= all || seq >= a.b.n_seq) return;             // behind the last row or sequence
    const PagedSeq sq = paged_seq(a.p, a.b, seq);
    const int i = tok - sq.t0;
    if (i < 0 || i >= sq.nq) return;
    const int n_pre = pre.x >> 1, n_own = own.x >> 1, total = n_pre + n_own;
    if (n_own == 0) return;                                  // written out
    // partial result k: the prefix's pieces, then the own ones
    auto at = [&](int k, const float *&o, const float2 *&ml) {
        const uint2 d = k < n_pre ? pre : own;
        if (k >= n_pre) k -= n_pre;
        if (d.y == ~0u) {
            o = pl.wo + (size_t)row * hd;
            ml = pl.wml + row;
            return;
        }
        const bool many = d.x & 1;
        const int w = (int)(d.y >> 9) + k, wgs = many ? pl.many.wgs : pl.few.wgs, rows = many ? pl.many.rows : pl.few.rows;
        const size_t s = (size_t)(2 * min(w, wgs - 1) + (k == 0 ? d.y >> 8 & 1 : 0)) * rows + (d.y & 255);
        o = (many ? pl.many.o : pl.few.o) + s * hd;
        ml = (many ? pl.many.ml : pl.few.ml) + s;
    };
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
            const float *o;
            const float2 *ml;
            at(min(k + j * step, total - 1), o, ml);
            x[j] = *ml;
            v[j] = *(const pa_v4f *)(o + e4);
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
    const bool none = !sq.bad && sq.len - sq.nq + i < 0;
    pa_store4(a.out + (size_t)tok * a.os + (size_t)head * hd + e4, none ? pa_v4f{0.0f, 0.0f, 0.0f, 0.0f} : s * (1.0f / l));
}

}  // namespace

size_t paged_attn_workspace(const PagedPool &p, const PagedBatch &b, int n_head) { return layout(p, b, n_head / p.n_kv, 0).total; }

hipError_t launch_paged_attn(const PagedAttn &a, hipStream_t s) {
    const PagedPool &p = a.p;
    const PagedBatch &b = a.b;
    if (b.n_tok == 0 || b.n_seq == 0) return hipSuccess;
    Layout y = layout(p, b, a.grp, a.window);
    PagedPlan &pl = y.pl;
    pl.few.o = (float *)(a.ws + y.fo);
    pl.few.ml = (float2 *)(a.ws + y.fml);
    pl.many.o = (float *)(a.ws + y.mo);
    pl.many.ml = (float2 *)(a.ws + y.mml);
    pl.own = y.join ? (uint2 *)(a.ws + y.own) : nullptr;
    pl.pre = (uint2 *)(a.ws + y.pre);
    pl.wo = (float *)(a.ws + y.wo);
    pl.wml = (float2 *)(a.ws + y.wml);
    if (pl.many.rows)
        if (hipError_t e = p.type == F16 ? pa_many_f16(a, pl, s) : p.type == Q8_0 ? pa_many_q8(a, pl, s) : pa_many_q4(a, pl, s)) return e;
    if (pl.few.rows)
        if (hipError_t e = p.type == F16 ? pa_few_f16(a, pl, s) : p.type == Q8_0 ? pa_few_q8(a, pl, s) : pa_few_q4(a, pl, s)) return e;
    if (y.join) {
        const int64_t rows = (int64_t)b.n_tok * a.n_head;
        if (rows <= 2048) hipLaunchKernelGGL(k_paged_join<true>, dim3((unsigned)rows, rows * (p.hd / 64) <= 512 ? p.hd / 64 : 1), dim3(256), 0, s, a, pl);
        else hipLaunchKernelGGL(k_paged_join<false>, dim3(ceil_div(rows, 256 / (p.hd / 4))), dim3(256), 0, s, a, pl);
        return hipGetLastError();
    }
    return hipSuccess;
}

}  // namespace g4
