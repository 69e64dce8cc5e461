// paged_split.h -- how an attention call over the paged KV cache is split over the
// two kernels (paged_attn.h), and its workspace.  Host code only.
#pragma once

#include <algorithm>

#include "paged_attn.h"

namespace g4 {

inline int pa_ceil_div(int64_t a, int64_t b) { return (int)((a + b - 1) / b); }

// A window that hides no position is none; with any other the device's sums of
// positions and windows fit 32 bits (a token before position 0 counts from below 0).
inline int paged_window(const PagedBatch &b, int window) { return window >= b.n_prefix + b.max_len ? 0 : window; }

struct PagedLayout {
    PagedPlan pl;
    bool join;
    size_t fo, fml, mo, mml, own, pre, wo, wml, total;
};
// of a batch with tokens and sequences; window 0 gives the most workspace
inline PagedLayout paged_layout(const PagedPool &p, const PagedBatch &b, int grp, int window) {
    PagedLayout y;
    PagedPlan &pl = y.pl;
    PagedList &few = pl.few, &many = pl.many;
    const int64_t rows = (int64_t)b.n_tok * grp;             // of one KV head
    pl.all = (int)(rows * p.n_kv);                           // up to 2^24
    pl.grp_inv = 65536 / grp + 1;
    many.toks = 1;
    many.toks_inv = 0;
    // Sequences of at most few.rows rows are the few-row kernel's: 8 (one matrix
    // instruction per operand) where no sequence can have more, else 16.
    // None where sequences have 64 tokens on average: the other kernel then takes the
    // short ones among them too, and a launch is saved (four prompts of up to 509: 80.8
    // us with that launch, 79.0 without).  The rule goes by the average, which the host
    // knows: single tokens over long caches beside one very long prompt are the many-row
    // kernel's too, where one takes about twice its time in the other.
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
    // 32 positions: 16 windows of 1024 take 19.3 us, with steps of 128 20.1); up to 256
    // positions stay one step, so that no join is launched for them.  A sequence's tile counts as
    // `lead` steps more, for its queries, first loads and results: 64 sequences of
    // 2000 of 4096 positions, 8 KV heads of 128, 8 bits, take 75 us with a lead of 1, 73
    // with 2, 93 without; a lead of 2 is slower where steps are few (the shares' last
    // step rounded up).  None where every step has its workgroup.
    int64_t steps;
    for (few.shift = b.max_len <= 256 && !b.n_prefix ? 8 : p.hd == 512 ? 5 : p.hd == 256 ? 6 : 7;; few.shift++) {       // counted in 32 bits on the device
        few.unit = 1 << few.shift;
        few.pre_steps = few_pre ? pa_ceil_div(b.n_prefix, few.unit) : 0;
        steps = ((int64_t)b.n_seq * std::max(1, pa_ceil_div(fspan, few.unit)) + few.pre_steps) * p.n_kv;
        if (steps < (1 << 27)) break;
    }
    few.wgs = (int)std::min<int64_t>(256 * pa_few_per_cu(p.type, p.hd, few.rows <= 8), steps);
    few.lead = steps > few.wgs ? 1 : 0;
    y.join = b.n_prefix || (few.rows && fspan > few.unit);
    // Many rows: tiles of whole tokens, up to 128 rows (64 of heads of 512), evenly
    // filled; as many workgroups as fit on the device at once.  Steps of 32 positions,
    // each its workgroup where they are few (24 rows of 256 over 76 positions: 22 us,
    // with shares of 2 at least 29.6).  A lead of 5 lies between what long and short
    // tiles want (leads of 4, 5, 6; 32 / 8 heads of 128, f16: one prompt of 2000 158,
    // 150, 141 us; four of 256 behind a prefix of 100 37.5, 37.6, 42.2; eight of 128 in
    // windows of 512 40.5, 39.8, 40.7).
    many.rows = 0;
    many.pre_tiles = many.lead = 0;
    if (many_own || many_pre) {
        const int most = paged_most_group(p.hd) / grp, toks = b.q_off || many_pre ? b.n_tok : 1;
        many.toks = pa_ceil_div(toks, pa_ceil_div(toks, most));
        many.toks_inv = many.toks == 1 ? 0 : (uint32_t)(0x100000000ull / many.toks + 1);
        many.rows = many.toks * grp;
        many.pre_tiles = many_pre ? pa_ceil_div(b.n_tok, many.toks) : 0;
        const int64_t own = !many_own ? 0 : b.q_off ? pa_ceil_div(b.n_tok, many.toks) + std::min(b.n_seq, b.n_tok / (few.toks + 1)) : b.n_seq;
        const int64_t mspan = span(many.toks);
        for (many.shift = 5;; many.shift++) {
            many.unit = 1 << many.shift;
            many.pre_steps = many_pre ? pa_ceil_div(b.n_prefix, many.unit) : 0;
            steps = (own * std::max(1, pa_ceil_div(mspan, many.unit)) + (int64_t)many.pre_tiles * many.pre_steps) * p.n_kv;
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
    y.wo = take(2 * whole * p.hd * 4);
    y.wml = take(2 * whole * sizeof(float2));
    y.total = at;
    return y;
}
// the plan of a call with its workspace at ws
inline PagedPlan paged_places(const PagedLayout &y, uint8_t *ws) {
    PagedPlan pl = y.pl;
    pl.few.o = (float *)(ws + y.fo);
    pl.few.ml = (float2 *)(ws + y.fml);
    pl.many.o = (float *)(ws + y.mo);
    pl.many.ml = (float2 *)(ws + y.mml);
    pl.own = y.join ? (uint2 *)(ws + y.own) : nullptr;
    pl.pre = (uint2 *)(ws + y.pre);
    pl.wo = (float *)(ws + y.wo);
    pl.wml = (float2 *)(ws + y.wml);
    return pl;
}

}  // namespace g4
