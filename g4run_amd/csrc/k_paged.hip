// k_paged.hip -- the paged KV cache's attention call: how it is split over the two
// kernels (paged_attn.h), its workspace, and the join of the partial results.
#include <algorithm>

#include "paged_attn.h"

namespace g4 {

namespace {

int ceil_div(int64_t a, int64_t b) { return (int)((a + b - 1) / b); }

// Workgroups the many-row kernel's splits aim at, and positions of a split at
// least: a split of 128 rows writes and reads back as many bytes as it reads for
// 256 positions.
constexpr int MANY_WGS = 256, MANY_CHUNK = 256;

int many_splits(int64_t items, int span) {
    return std::max(1, std::min<int>((int)(MANY_WGS / std::max<int64_t>(items, 1)), ceil_div(span, MANY_CHUNK)));
}
void many_chunk(int64_t items, int span, int &n, int &chunk) {
    chunk = std::max(MANY_CHUNK, ceil_div(ceil_div(span, many_splits(items, span)), 32) * 32);
    n = std::max(1, ceil_div(span, chunk));
}

struct Layout {
    PagedPlan pl;
    bool few, many, join;
    size_t fo, oo, po, fml, oml, pml, total;
};
// window 0 gives the most workspace
Layout layout(const PagedPool &p, const PagedBatch &b, int grp, int window, bool bound) {
    Layout y;
    PagedPlan &pl = y.pl;
    const int64_t rows = (int64_t)b.n_tok * grp;             // of one KV head
    // Sequences of at most few_rows rows are the few-row kernel's: 8 (one matrix
    // instruction per operand) where no sequence can have more, else 16.
    pl.few_rows = grp > 16 ? 0 : (b.q_off ? rows : grp) <= 8 ? 8 : 16;
    if (b.n_prefix && pl.few_rows == 8 && rows > 8 && rows <= 16) pl.few_rows = 16;
    y.few = pl.few_rows > 0;
    const bool few_pre = b.n_prefix && y.few && rows <= pl.few_rows;
    const bool many_own = b.q_off ? b.n_tok > (y.few ? pl.few_rows / grp : 0) : !y.few;
    const bool many_pre = b.n_prefix && !few_pre;
    y.many = many_own || many_pre;
    // few: the most own positions of a sequence it takes (few_rows tokens at most)
    pl.grp_inv = 65536 / grp + 1;
    // a step is at least what a workgroup takes at once; up to 256 positions stay
    // one step, so that no join is launched for them
    pl.few_shift = b.max_len <= 256 && !b.n_prefix ? 8 : 7;
    const int64_t fspan = window ? std::min<int64_t>(b.max_len, (int64_t)window + 32 + 16) : b.max_len;
    int64_t steps;
    for (;; pl.few_shift++) {                                // counted in 32 bits on the device
        pl.few_unit = 1 << pl.few_shift;
        pl.few_pre = few_pre ? ceil_div(b.n_prefix, pl.few_unit) : 0;
        steps = ((int64_t)b.n_seq * std::max(1, ceil_div(fspan, pl.few_unit)) + pl.few_pre) * p.n_kv;
        if (steps < (1 << 30)) break;
    }
    pl.few_wgs = (int)std::min<int64_t>(PA_FEW_WGS, steps);
    // many: tiles of up to 128 rows (64 of heads of 512), evenly filled
    const int most = p.hd > 256 ? 64 : 128;
    const int64_t tiles = std::max<int64_t>(1, ceil_div(b.q_off || many_pre ? rows : grp, most));
    pl.many_rows = (int)std::min<int64_t>(most, ceil_div(ceil_div(b.q_off || many_pre ? rows : grp, tiles), 32) * 32);
    pl.own_slots = pl.pre_slots = pl.own_chunk = pl.pre_chunk = pl.npre = 0;
    pl.nown = 1;
    int64_t slots = 0;
    if (many_own) {
        const int least = b.q_off && y.few ? pl.few_rows / grp + 1 : 1;      // tokens of a sequence it takes
        slots = b.q_off ? ceil_div(rows, pl.many_rows) + std::min(b.n_seq, b.n_tok / least) : (int64_t)b.n_seq * ceil_div(grp, pl.many_rows);
        pl.own_slots = (int)slots;
        const int64_t span = window ? std::min<int64_t>(b.max_len, (int64_t)window + 32 + pl.many_rows / grp + 1) : b.max_len;
        many_chunk(slots * p.n_kv, (int)span, pl.nown, pl.own_chunk);
        if (bound) pl.nown = many_splits(slots * p.n_kv, b.max_len);
    }
    if (many_pre) {
        pl.pre_slots = ceil_div(rows, pl.many_rows);
        many_chunk((int64_t)pl.pre_slots * p.n_kv, b.n_prefix, pl.npre, pl.pre_chunk);
    }
    y.join = b.n_prefix || pl.nown > 1 || (y.few && fspan > pl.few_unit);
    const size_t all = (size_t)b.n_tok * p.n_kv * grp, few = y.few && y.join ? (size_t)pl.few_wgs * 2 * pl.few_rows : 0;
    const size_t own = b.n_prefix || pl.nown > 1 ? all * pl.nown : 0, pre = all * pl.npre;
    size_t at = 0;
    auto take = [&](size_t bytes) { const size_t here = at; at += (bytes + 255) & ~(size_t)255; return here; };
    y.fo = take(few * p.hd * 4);
    y.fml = take(few * sizeof(float2));
    y.oo = take(own * p.hd * 4);
    y.oml = take(own * sizeof(float2));
    y.po = take(pre * p.hd * 4);
    y.pml = take(pre * sizeof(float2));
    y.total = at;
    return y;
}

// One (token, head) row per workgroup: out = sum of exp2(m_k - M) O_k / sum of
// exp2(m_k - M) l_k over the row's partial results in a fixed order.  Groups of
// hd / 4 threads take every so-many-th of them.
__global__ __launch_bounds__(256) void k_paged_join(PagedAttn a, PagedPlan pl) {
    __shared__ float red[4];
    __shared__ float lg[16];                                 // at most 16 groups: hd >= 64
    __shared__ pa_v4f part[256];
    const int hd = a.p.hd, hd4 = hd / 4, groups = 256 / hd4, gi = threadIdx.x / hd4, e4 = threadIdx.x % hd4 * 4;
    const int tok = blockIdx.x / a.n_head, head = blockIdx.x - tok * a.n_head, kvh = head / a.grp;
    const int seq = paged_find(a.b, tok);
    if (seq >= a.b.n_seq) return;                            // behind the last sequence
    const PagedSeq sq = paged_seq(a.p, a.b, seq);
    const int i = tok - sq.t0;
    if (i < 0 || i >= sq.nq) return;
    const size_t row = (size_t)tok * a.n_head + head;
    const bool few = sq.nq * a.grp <= pl.few_rows;
    int mine, share = 1, fb = 0, fi0 = 0, nf = 0, nw = 0;    // own few pieces: first workgroup, their number; whole ones
    if (few || pl.few_pre) share = pa_share(pa_total(a, pl, mine));
    if (few) {
        const int all = pa_seq_steps(a, pl, sq);
        fb = pl.few_pre * a.p.n_kv + pa_before(a, pl, mine, seq) + kvh * all;
        fi0 = fb / share;
        nf = (fb + all - 1) / share - fi0 + 1;
        if (nf == 1) {
            if (a.b.n_prefix == 0) return;                   // written by the kernel
            nf = 0;
            nw = 1;
        }
    } else {
        int lo, hi;
        pa_tile_span(sq, a.grp, pl.many_rows, (i * a.grp + head % a.grp) / pl.many_rows, a.window, lo, hi);
        nw = pa_tile_chunks(sq, pl, lo, hi);
        if (pl.nown == 1 && a.b.n_prefix == 0) return;
    }
    int pb = 0, pi0 = 0, np = 0;
    if (pl.few_pre) {
        pb = kvh * pl.few_pre;
        pi0 = pb / share;
        np = (pb + pl.few_pre - 1) / share - pi0 + 1;
    }
    // partial result k: prefix pieces or chunks, then own pieces or chunks
    const int R = pl.few_rows, nq0 = np ? np : pl.npre, total = nq0 + nf + nw;
    auto at = [&](int k, const float *&o, const float2 *&ml) {
        if (k < nq0) {
            if (np) {
                const size_t s = (size_t)(2 * (pi0 + k) + (k == 0 && pb != pi0 * share)) * R + (size_t)tok * a.grp + head % a.grp;
                o = pl.fo + s * hd;
                ml = pl.fml + s;
            } else {
                const size_t s = row * pl.npre + k;
                o = pl.po + s * hd;
                ml = pl.pml + s;
            }
        } else if (nf) {
            const int n = k - nq0;
            const size_t s = (size_t)(2 * (fi0 + n) + (n == 0 && fb != fi0 * share)) * R + (size_t)i * a.grp + head % a.grp;
            o = pl.fo + s * hd;
            ml = pl.fml + s;
        } else {
            const size_t s = row * pl.nown + (k - nq0);
            o = pl.oo + s * hd;
            ml = pl.oml + s;
        }
    };
    float mm = -__builtin_inff();
    for (int k = threadIdx.x; k < total; k += 256) {
        const float *o;
        const float2 *ml;
        at(k, o, ml);
        mm = fmaxf(mm, ml->x);
    }
    mm = group_max<64>(mm);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = mm;
    __syncthreads();
    mm = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
    pa_v4f s = {0.0f, 0.0f, 0.0f, 0.0f};
    float l = 0.0f;
#pragma unroll 4
    for (int k = gi; k < total; k += groups) {
        const float *o;
        const float2 *ml;
        at(k, o, ml);
        const float2 x = *ml;
        const pa_v4f v = *(const pa_v4f *)(o + e4);
        const float f = x.x == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(x.x - mm);
        l += x.y == x.y ? f * x.y : x.y;                     // a bad page's NaN stays
        s += v * f;
    }
    part[threadIdx.x] = s;
    if (e4 == 0) lg[gi] = l;
    __syncthreads();
    if (gi) return;
    for (int k = 1; k < groups; k++) {
        s += part[k * hd4 + threadIdx.x];
        l += lg[k];
    }
    const bool none = !sq.bad && sq.len - sq.nq + i < 0;
    pa_store4(a.out + (size_t)tok * a.os + (size_t)head * hd + e4, none ? pa_v4f{0.0f, 0.0f, 0.0f, 0.0f} : s * (1.0f / l));
}

}  // namespace

size_t paged_attn_workspace(const PagedPool &p, const PagedBatch &b, int n_head) {
    return layout(p, b, n_head / p.n_kv, 0, true).total;
}

hipError_t launch_paged_attn(const PagedAttn &a, hipStream_t s) {
    const PagedPool &p = a.p;
    const PagedBatch &b = a.b;
    if (b.n_tok == 0 || b.n_seq == 0) return hipSuccess;
    Layout y = layout(p, b, a.grp, a.window, false);
    PagedPlan &pl = y.pl;
    pl.fo = (float *)(a.ws + y.fo);
    pl.oo = (float *)(a.ws + y.oo);
    pl.po = (float *)(a.ws + y.po);
    pl.fml = (float2 *)(a.ws + y.fml);
    pl.oml = (float2 *)(a.ws + y.oml);
    pl.pml = (float2 *)(a.ws + y.pml);
    if (y.many) {
        const int64_t blocks = ((int64_t)pl.own_slots * pl.nown + (int64_t)pl.pre_slots * pl.npre) * p.n_kv;
        if (blocks > 0xffffff) return hipErrorInvalidValue;
        if (hipError_t e = p.type == F16 ? pa_many_f16(a, pl, (unsigned)blocks, s)
                         : p.type == Q8_0 ? pa_many_q8(a, pl, (unsigned)blocks, s) : pa_many_q4(a, pl, (unsigned)blocks, s))
            return e;
    }
    if (y.few)
        if (hipError_t e = p.type == F16 ? pa_few_f16(a, pl, s) : p.type == Q8_0 ? pa_few_q8(a, pl, s) : pa_few_q4(a, pl, s)) return e;
    if (y.join) {
        hipLaunchKernelGGL(k_paged_join, dim3((unsigned)(b.n_tok * a.n_head)), dim3(256), 0, s, a, pl);
        return hipGetLastError();
    }
    return hipSuccess;
}

}  // namespace g4
