// k_paged.hip -- the paged KV cache's attention call: how it is split, and the
// join of the splits (the kernel itself: paged_attn.h).
#include <algorithm>

#include "paged_attn.h"

namespace g4 {

namespace {

int ceil_div(int64_t a, int64_t b) { return (int)((a + b - 1) / b); }

// Tiles as large as the rows that share a segment's keys: 8 rows cost one matrix
// instruction per operand, 16 and 32 two and share the loads.
int tile_variant(int64_t rows, int hd) { return rows <= 8 ? PA_ST : rows <= 16 || hd > 256 ? PA_T1 : PA_T2; }

// Splits of `items` tiles over `span` positions: enough workgroups to fill the
// chip, chunks of at least one 32-position step per wave.
constexpr int PA_STEP = 32 * PA_WAVES, PA_BLOCKS = 1024;
int most_splits(int64_t items, int span) { return std::max(1, std::min(ceil_div(PA_BLOCKS, std::max<int64_t>(items, 1)), ceil_div(span, PA_STEP))); }
void split(int64_t items, int span, int &n, int &chunk) {
    chunk = std::max(PA_STEP, ceil_div(ceil_div(span, most_splits(items, span)), PA_STEP) * PA_STEP);
    n = std::max(1, ceil_div(span, chunk));
}

struct Shape {
    int own_v, pre_v;
    int64_t own_slots, pre_slots;
};
Shape shape(const PagedPool &p, const PagedBatch &b, int grp) {
    Shape s;
    const int64_t rows = (int64_t)b.n_tok * grp;
    s.own_v = tile_variant(b.q_off ? rows / std::max(1, b.n_seq) : grp, p.hd);
    s.own_slots = b.q_off ? ceil_div(rows, pa_rows(s.own_v)) + b.n_seq : (int64_t)b.n_seq * ceil_div(grp, pa_rows(s.own_v));
    s.pre_v = tile_variant(rows, p.hd);
    s.pre_slots = b.n_prefix ? ceil_div(rows, pa_rows(s.pre_v)) : 0;
    return s;
}

size_t row_bytes(int hd) { return (size_t)hd * 4 + sizeof(float2); }

// out[row] = sum over the row's splits of exp2(m_k - M) O_k / sum of
// exp2(m_k - M) l_k, splits in order; one thread per 4 elements.
__global__ __launch_bounds__(256) void k_paged_join(PagedAttn a, PagedPlan pl, int R) {
    const int hd4 = a.p.hd / 4, per = 256 / hd4;
    const int64_t row = (int64_t)blockIdx.x * per + threadIdx.x / hd4;
    const int e4 = threadIdx.x % hd4 * 4;
    if (row >= (int64_t)a.b.n_tok * a.n_head) return;
    const int tok = (int)(row / a.n_head), head = (int)(row - (int64_t)tok * a.n_head);
    int seq = tok;
    if (a.b.q_off) {                                 // the last sequence that starts at or before the token
        int x = 0, y = a.b.n_seq + 1;
        while (y - x > 1) {
            const int z = (x + y) >> 1;
            if (a.b.q_off[z] <= tok) x = z;
            else y = z;
        }
        seq = x;
    }
    if (seq >= a.b.n_seq) return;                    // behind the last sequence
    const PagedSeq sq = paged_seq(a.p, a.b, seq);
    const int i = tok - sq.t0;
    if (i < 0 || i >= sq.nq) return;
    float *d = a.out + (size_t)tok * a.os + (size_t)head * a.p.hd + e4;
    pa_v4f s = {0.0f, 0.0f, 0.0f, 0.0f};
    if (sq.bad || sq.len - sq.nq + i >= 0) {
        const int tile = (i * a.grp + head % a.grp) / R;
        int lo, hi;
        pa_tile_span(sq, a.grp, R, tile, a.window, lo, hi);
        const int n = pl.npre + pa_tile_chunks(sq, pl, lo, hi);
        const size_t at = (size_t)row * pl.nsplit;
        float mm = -__builtin_inff(), l = 0.0f;
#pragma unroll 4
        for (int k = 0; k < n; k++) mm = fmaxf(mm, pl.ml[at + k].x);
#pragma unroll 4
        for (int k = 0; k < n; k++) {
            const float2 ml = pl.ml[at + k];
            const pa_v4f v = *(const pa_v4f *)(pl.po + (at + k) * a.p.hd + e4);
            const float f = ml.x == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(ml.x - mm);
            l += ml.y == ml.y ? f * ml.y : ml.y;     // a bad page's NaN stays
            s += v * f;
        }
        s *= 1.0f / l;
    }
    if (a.os % 4 == 0 && (uintptr_t)a.out % 16 == 0) *(pa_v4f *)d = s;
    else { d[0] = s[0]; d[1] = s[1]; d[2] = s[2]; d[3] = s[3]; }
}

hipError_t launch(const PagedAttn &a, const PagedPlan &pl, int v, int64_t blocks, hipStream_t s) {
    if (blocks == 0) return hipSuccess;
    if (blocks > 0x7fffffff) return hipErrorInvalidValue;
    return a.p.type == F16 ? pa_launch_f16(a, pl, v, (unsigned)blocks, s)
         : a.p.type == Q8_0 ? pa_launch_q8(a, pl, v, (unsigned)blocks, s) : pa_launch_q4(a, pl, v, (unsigned)blocks, s);
}

}  // namespace

size_t paged_attn_workspace(const PagedPool &p, const PagedBatch &b, int n_head) {
    const Shape sh = shape(p, b, n_head / p.n_kv);
    const int n = most_splits(sh.own_slots * p.n_kv, b.max_len) + (b.n_prefix ? most_splits(sh.pre_slots * p.n_kv, b.n_prefix) : 0);
    return n == 1 ? 0 : (size_t)b.n_tok * n_head * n * row_bytes(p.hd);
}

hipError_t launch_paged_attn(const PagedAttn &a, hipStream_t s) {
    const PagedPool &p = a.p;
    const PagedBatch &b = a.b;
    if (b.n_tok == 0 || b.n_seq == 0) return hipSuccess;
    const Shape sh = shape(p, b, a.grp);
    const int own_r = pa_rows(sh.own_v);
    // most own positions a tile attends: its first token's window rounded down
    // to 32, and its later tokens
    const int64_t span = a.window ? std::min<int64_t>(b.max_len, (int64_t)a.window + 32 + own_r / a.grp + 1) : b.max_len;
    PagedPlan pl;
    pl.own_slots = (int)sh.own_slots;
    split(sh.own_slots * p.n_kv, (int)span, pl.nown, pl.own_chunk);
    pl.pre_slots = (int)sh.pre_slots;
    pl.npre = 0;
    pl.pre_chunk = 0;
    if (b.n_prefix) split(sh.pre_slots * p.n_kv, b.n_prefix, pl.npre, pl.pre_chunk);
    pl.nsplit = pl.nown + pl.npre;
    pl.po = (float *)a.ws;
    pl.ml = (float2 *)(a.ws + (size_t)b.n_tok * a.n_head * pl.nsplit * p.hd * 4);
    const int64_t own = sh.own_slots * p.n_kv * pl.nown, pre = sh.pre_slots * p.n_kv * pl.npre;
    if (pre && sh.pre_v == sh.own_v) {
        if (hipError_t e = launch(a, pl, sh.own_v, pre + own, s)) return e;
    } else {
        PagedPlan part = pl;
        part.own_slots = 1;                          // prefix items alone
        if (hipError_t e = launch(a, part, sh.pre_v, pre, s)) return e;
        part = pl;
        part.pre_slots = 0;
        if (hipError_t e = launch(a, part, sh.own_v, own, s)) return e;
    }
    if (pl.nsplit > 1) {
        const int64_t rows = (int64_t)b.n_tok * a.n_head, per = 256 / (p.hd / 4);
        hipLaunchKernelGGL(k_paged_join, dim3((unsigned)((rows + per - 1) / per)), dim3(256), 0, s, a, pl, own_r);
        return hipGetLastError();
    }
    return hipSuccess;
}

}  // namespace g4
