// paged_attn.h -- what the attention kernels over the paged KV cache share
// (g4h_paged_attn): operands, masks, the split of a call and its workspace.
//
// Mathematics: one pass over the positions with the running maximum and sum of
// a softmax, per tile of (token, query head) rows of one KV head.  Both products
// run on the f16 matrix cores with the scores transposed,
//   S^T [positions][rows] = K q^T, then O^T [elements][rows] += V^T P^T:
// a lane then holds scores of one row at positions whose order is that of the
// second product's operand, so the weights never leave their registers.
//
// Precision: sums, scores and weights in fp32.  K and V enter the products exactly
// (halves, or the integers of the block formats, their scales applied in fp32 to the
// scores and to the weights); what they are multiplied with enters as two halves,
// cut off.  A query row is scaled by a power of two to [2^14, 2^15): an element is
// off by up to 2^-21 of itself and 2^-38 of the row's largest (the halves' smallest
// step, 2^-24).  Weights are exp2(s - m + 6), for quantized values with m over s + the
// exponent of the position's largest scale, so that weight x scale does not overflow:
// one is off by up to 2^-21 of itself and 2^-30 of the row's largest (quantized:
// weight times scale by 2^-29 of the largest such product, scales below 2^-14
// counting as that).  Where one position has nearly all the weight and a value near
// zero, the others' cut is what the result's error is made of: weights of 2^-17 of
// the largest lose 6e-5 of themselves on average.  A third half of the weights would
// cost a quarter more matrix instructions.
//
// Two kernels share a call:
//   k_paged_few   row tiles of up to 16 rows (single tokens; the prefix of a small
//                 batch): bound by the cache's bytes.
//   k_paged_many  sequences of more rows (prompt chunks; the prefix of a large
//                 batch): bound by the matrix cores.  K and V pass through LDS
//                 once for up to 128 rows.
// Calls with trees of new tokens (PagedAttn::mask) take one of two:
//   k_paged_few   in a form whose rows look at their masks, where all tiles are small;
//   k_paged_tree  else (paged_tree.h): a few to 128 rows, bound by the cache's bytes
//                 (f16) or by what makes operands of them.
#pragma once

#include "paged.h"

namespace g4 {

typedef _Float16 pa_v8h __attribute__((ext_vector_type(8)));
typedef _Float16 pa_v2h __attribute__((ext_vector_type(2)));
typedef float pa_v4f __attribute__((ext_vector_type(4)));
typedef float pa_v16f __attribute__((ext_vector_type(16)));
typedef uint32_t pa_v4u __attribute__((ext_vector_type(4)));

// The split of a call.  Each kernel's work is one list of steps (`unit` positions
// of one row tile of one KV head: the prefix's tiles, then the sequences' in
// order), cut into equal shares for its workgroups; k_paged_tree's steps count by
// their tiles' rows, so that its shares take equal time.  A piece -- the part of a
// share that lies in one tile of one head -- is written out where it is the whole
// tile and there is no prefix; else its sums go to the workspace.  A whole tile's
// have a place by row, one for the prefix's tile and one for the row's own.  Of the
// other pieces a share holds two at most, its first and its last: slot 2 w for
// workgroup w's first piece, 2 w + 1 for its last.  The tile's first piece tells
// k_paged_join where its rows' pieces lie.  The functions of the split run on the
// host too, where a test follows every piece of a call.
struct PagedList {
    int rows;                        // rows of a tile; the few-row kernel: most rows of a sequence it takes
    int toks;                        // many: tokens of a tile, rows / grp; few: most tokens of a sequence
    uint32_t toks_inv;               // many: n / toks == umulhi(n, toks_inv) for n <= 2^24 (0: toks is 1)
    int wgs;                         // workgroups
    int unit, shift;                 // positions of a step, and their log2
    int lead;                        // steps that the start of a sequence's tile counts as
    int pre_tiles, pre_steps;        // the prefix's tiles (0: not this kernel's), and steps of each
    float *o;                        // [2 wgs][rows][hd] unnormalised sums
    float2 *ml;                      // [2 wgs][rows] maximum (log2), sum
};
struct PagedPlan {
    PagedList few, many;             // rows 0: the kernel does not run
    int all;                         // (token, head) rows of the call
    uint32_t grp_inv;                // rows to tokens: r / grp == r * grp_inv >> 16 for r < 16
    // where a (token, head) row's partial results lie, own positions and prefix:
    // count << 2 | whether it has no position << 1 | kernel (0 few), slot << 8 | row of
    // the tile; [0] count 0 where there is nothing to join: the row is written out,
    // or no sequence's
    uint2 *own, *pre;
    float *wo;                       // [2][token][head][hd] whole tiles' sums beside a prefix: own positions, the prefix
    float2 *wml;
};

// Weights are scaled by 2^6 over a maximum that may lag by 2^8: their low halves
// stay normal and the largest, 2^14 (times a scale below 1), finite.  Without the
// lag some row of a tile raises its maximum, and all sums are rescaled, in most of
// the first steps.
constexpr float PA_SHIFT = 6.0f, PA_LAG = 8.0f;

// A kernel's arguments, and a copy of them read again where it is asked for: what
// the outer loop over the pieces needs between two of them then stays in memory,
// not in registers (with all of it held, 40 vector registers more).
struct PagedCall {
    PagedAttn a;
    PagedPlan pl;
};
template <typename T>
__device__ __forceinline__ void pa_global(T *&p) {
    auto *g = (__attribute__((address_space(1))) T *)p;
    asm("" : "+s"(g));
    p = (T *)g;
}
template <bool TREE = false>
__device__ __forceinline__ PagedCall pa_fresh() {
    static_assert(sizeof(PagedCall) % 4 == 0, "read by dwords");
    auto *p = (const __attribute__((address_space(4))) uint32_t *)__builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(p));
    uint32_t w[sizeof(PagedCall) / 4];
#pragma unroll
    for (int i = 0; i < (int)(sizeof w / 4); i++) w[i] = p[i];
    PagedCall k = __builtin_bit_cast(PagedCall, w);
    // pointers to global memory, which arguments are known to be and loaded ones are
    // not: flat accesses would count as LDS accesses too
    pa_global(k.a.p.k);
    pa_global(k.a.p.v);
    pa_global(k.a.p.status);
    pa_global(k.a.q);
    pa_global(k.a.out);
    if constexpr (TREE) {                                    // (said of what a kernel does not use, it is held all the same)
        pa_global(k.a.mask);
        pa_global(k.a.depth);
    }
    pa_global(k.pl.few.o);
    pa_global(k.pl.few.ml);
    pa_global(k.pl.many.o);
    pa_global(k.pl.many.ml);
    pa_global(k.pl.own);
    pa_global(k.pl.pre);
    pa_global(k.pl.wo);
    pa_global(k.pl.wml);
    return k;
}
__device__ __forceinline__ int pa_thread() {
    int t = threadIdx.x;
    asm volatile("" : "+v"(t));
    return t;
}

__device__ __forceinline__ int pa_uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ uint32_t pa_pk(float a, float b) { return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(a, b)); }
__device__ __forceinline__ float pa_lo(uint32_t h) { return (float)__builtin_bit_cast(pa_v2h, h)[0]; }
__device__ __forceinline__ float pa_hi(uint32_t h) { return (float)__builtin_bit_cast(pa_v2h, h)[1]; }
__device__ __forceinline__ float pa_scale(const uint32_t *d, int b) { return (b & 1) ? pa_hi(d[b >> 1]) : pa_lo(d[b >> 1]); }
__device__ __forceinline__ pa_v4f pa_mma(pa_v8h a, pa_v8h b, pa_v4f c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ pa_v8h pa_op(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    const pa_v4u v = {a, b, c, d};
    return __builtin_bit_cast(pa_v8h, v);
}
// bytes u = quant + 128 in the low byte of each half (a half's subnormals
// u 2^-24) to quant * 2^-9, exactly
__device__ __forceinline__ uint32_t pa_q8(uint32_t x) {
    const pa_v2h k = {(_Float16)32768.0f, (_Float16)32768.0f}, c = {(_Float16)-0.25f, (_Float16)-0.25f};
    return __builtin_bit_cast(uint32_t, __builtin_elementwise_fma(__builtin_bit_cast(pa_v2h, x), k, c));
}
// nibbles K (of 4) of both halves, quant + 8, to quant, exactly: bits 0..3 under the
// exponent of 1024 are 1024 + x, bits 4..7 are 1024 + 16 x
template <int K>
__device__ __forceinline__ uint32_t pa_q4(uint32_t w) {
    const uint32_t y = K < 2 ? w : w >> 8;
    if constexpr (K % 2 == 0) {
        const pa_v2h c = {(_Float16)-1032.0f, (_Float16)-1032.0f};
        return __builtin_bit_cast(uint32_t, __builtin_bit_cast(pa_v2h, (y & 0x000f000fu) | 0x64006400u) + c);
    } else {
        const pa_v2h k = {(_Float16)0.0625f, (_Float16)0.0625f}, c = {(_Float16)-72.0f, (_Float16)-72.0f};
        return __builtin_bit_cast(uint32_t, __builtin_elementwise_fma(__builtin_bit_cast(pa_v2h, (y & 0x00f000f0u) | 0x64006400u), k, c));
    }
}
__device__ __forceinline__ uint32_t pa_q4(uint32_t w, int k) { return k == 0 ? pa_q4<0>(w) : k == 1 ? pa_q4<1>(w) : k == 2 ? pa_q4<2>(w) : pa_q4<3>(w); }

template <int N>
__device__ __forceinline__ void pa_load(uint32_t *d, const uint8_t *p) {
    if constexpr (N % 4 == 0) {
#pragma unroll
        for (int i = 0; i < N; i += 4) {
            const uint4 x = *(const uint4 *)(p + 4 * i);
            d[i] = x.x; d[i + 1] = x.y; d[i + 2] = x.z; d[i + 3] = x.w;
        }
    } else if constexpr (N == 2) {
        const uint2 x = *(const uint2 *)p;
        d[0] = x.x; d[1] = x.y;
    } else {
        static_assert(N == 1, "a lane's run is 1, 2 or a multiple of 4 dwords");
        d[0] = *(const uint32_t *)p;
    }
}

// Where a wave's next units (16 positions each) lie: lane 2 k + h holds unit
// first + stride * k + h of the segment -- its page id and its first row in the
// page -- so that 32 steps of two units cost one load, and reading a unit none.
struct PaUnits {
    int id, row;
};
__device__ __forceinline__ PaUnits pa_units(const PagedPool &p, const int *table, int first, int stride, int last, int kvh) {
    const int lane = threadIdx.x & 63, u = min(first + stride * (lane >> 1) + (lane & 1), last), ent = paged_entry(p, u);
    PaUnits x;
    x.id = paged_ld(table, ent);
    x.row = kvh * p.page + (u - ent * p.units) * 16;
    return x;
}
// before their first use (not with the load, which would be waited for there): the
// lanes whose page lies outside the pool, read as page 0 instead
__device__ __forceinline__ uint64_t pa_check(const PagedPool &p, PaUnits &x) {
    const bool out = (uint64_t)(int64_t)x.id >= (uint64_t)p.n_pages;
    if (out) x.id = 0;
    return __ballot(out);
}
// whether the lane's row, of positions [rlo, rhi], attends one of them; a page that
// it does not attend (before its window, say, and given away) may be any.  A window
// may hide the whole segment: rlo behind rhi
__device__ __forceinline__ bool pa_hits(uint64_t out, int first, int stride, int last, int rlo, int rhi) {
    bool hit = false;
    for (; out; out &= out - 1) {
        const int k = __ffsll((unsigned long long)out) - 1, pos = 16 * min(first + stride * (k >> 1) + (k & 1), last);
        hit |= max(rlo, pos) <= min(rhi, pos + 15);
    }
    return hit;
}
// 32 bits of a tree's mask row from bit `off` on (off may be anything): 0 outside of it
__device__ __forceinline__ uint32_t pa_bits(const uint32_t *mask, int words, int off) {
    const int w = off >> 5;
    const uint32_t lo = w >= 0 && w < words ? mask[w] : 0u, hi = w + 1 >= 0 && w + 1 < words ? mask[w + 1] : 0u;
    return (uint32_t)(((uint64_t)hi << 32 | lo) >> (off & 31));
}
// which of the 32 positions from base on a tree's row attends: cached ones in [rlo, rhi],
// new ones by its bits from base on, before end
__device__ __forceinline__ uint32_t pa_tree_seen(int base, int rlo, int rhi, uint32_t bits, int end) {
    auto below = [&](int pos) { return pos <= base ? 0u : pos >= base + 32 ? ~0u : (1u << (pos - base)) - 1; };
    return ((below(rhi + 1) & ~below(rlo)) | bits) & below(end);
}
// Whether a tree's row attends nothing: no position of the prefix, no cached one, no
// new token that has a position.  mask: its row.
__device__ __forceinline__ bool pa_tree_nothing(const PagedAttn &a, const PagedSeq &q, int tok, const uint32_t *mask) {
    const int first_new = q.len - q.nq;
    if (first_new + (tok - q.t0) < 0) return true;
    const int low = a.window ? first_new + paged_depth(a.depth[tok], q.nq) + 1 - a.window : -0x7fffffff;       // first position, the prefix's below 0
    if ((a.b.n_prefix > 0 && low < 0) || (first_new > 0 && low < first_new)) return false;
    for (int w = 0; w < a.words; w++) {
        const int n = q.nq - 32 * w, gone = -first_new - 32 * w;             // tokens from this word on; of them before position 0
        uint32_t bits = n >= 32 ? mask[w] : n > 0 ? mask[w] & ((1u << n) - 1) : 0u;
        if (gone > 0) bits = gone >= 32 ? 0u : bits & ~((1u << gone) - 1);
        if (bits) return false;
    }
    return true;
}
// pa_hits of a tree's row, by what pa_tree_seen says that it attends of the segment's
// `len` positions: a window may leave it no cached position (rlo behind rhi), and bits
// of tokens that the sequence does not have mean nothing.  bits(pos): its bits from pos on
template <typename F>
__device__ __forceinline__ bool pa_tree_hits(uint64_t out, int first, int stride, int len, int rlo, int rhi, F bits) {
    bool hit = false;
    for (; out; out &= out - 1) {
        const int k = __ffsll((unsigned long long)out) - 1, pos = 16 * min(first + stride * (k >> 1) + (k & 1), (len - 1) >> 4);
        hit |= (pa_tree_seen(pos, rlo, rhi, bits(pos), len) & 0xffffu) != 0;
    }
    return hit;
}
// the offset of a unit's rows in the pools and, quantized, of their scales
struct PaUnit {
    size_t row, sc;
};
template <int HD, int KVT>
__device__ __forceinline__ PaUnit pa_unit(const PagedPool &p, const PaUnits &us, int lane) {
    const uint32_t id = __builtin_amdgcn_readlane(us.id, lane), r = __builtin_amdgcn_readlane(us.row, lane);
    PaUnit x;
    x.row = (size_t)id * p.page_bytes + (size_t)r * paged_row_bytes(KVT, HD);
    x.sc = KVT == F16 ? 0 : (size_t)id * p.page_bytes + p.sc_off + (size_t)r * (HD / 16);
    return x;
}

// x = tanh(x) of a lane's N scores: an odd polynomial below 0.3 (next term 9e-3
// x^11, below 6e-8 x there), where 1 - exp would lose the small value
template <int N>
__device__ __forceinline__ void pa_tanh(float (&x)[N]) {
    float most = 0.0f;
    float p[N];
#pragma unroll
    for (int j = 0; j < N; j++) {
        const float x2 = x[j] * x[j];
        float y = __builtin_fmaf(x2, 62.0f / 2835.0f, -17.0f / 315.0f);
        y = __builtin_fmaf(x2, y, 2.0f / 15.0f);
        y = __builtin_fmaf(x2, y, -1.0f / 3.0f);
        p[j] = __builtin_fmaf(x[j] * x2, y, x[j]);
        most = fmaxf(most, fabsf(x[j]));
    }
    if (__any(most > 0.3f)) {
#pragma unroll
        for (int j = 0; j < N; j++) {
            const float ax = fabsf(x[j]), t = __builtin_amdgcn_exp2f(-2.885390081777927f * ax);
            const float r = copysignf((1.0f - t) * __builtin_amdgcn_rcpf(1.0f + t), x[j]);
            p[j] = ax > 0.3f ? r : p[j];                     // NaN: the polynomial's
        }
    }
#pragma unroll
    for (int j = 0; j < N; j++) x[j] = p[j];
}

// the end of the batch's tokens; n_seq: its sequences before the first torn one
__host__ __device__ __forceinline__ int pa_tokens(const PagedBatch &b, int n_seq) {
    if (n_seq == 0) return 0;
    return b.q_off ? paged_ld(b.q_off, n_seq) : min(n_seq, b.n_tok);
}
// first own position that tokens from `first` on attend, rounded down to 32
__host__ __device__ __forceinline__ int pa_low(int first, int window) { return window ? max(0, first + 1 - window) & ~31 : 0; }

// position of global token tok (prefix included), its sequence looked up; a tree's
// (depth given) as its depth says
__device__ __forceinline__ int pa_token_pos(const PagedPool &p, const PagedBatch &b, int n_seq, int tok, const int *depth = nullptr) {
    int s = tok;
    if (b.q_off) {
        int x = 0, y = n_seq;                                // last s with q_off[s] <= tok
        while (y - x > 1) {
            const int z = (x + y) >> 1;
            if (paged_ld(b.q_off, z) <= tok) x = z;
            else y = z;
        }
        s = x;
    }
    const PagedSeq o = paged_seq(p, b, s);
    return b.n_prefix + o.len - o.nq + (depth ? paged_depth(depth[tok], o.nq) : tok - o.t0);
}

// inclusive sum over the lanes of a wave: within each row of 16, then the rows'
// totals passed on
__device__ __forceinline__ int pa_scan(int v) {
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, false);      // row_shr:1
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false);      // row_bcast:15 into rows 1 and 3
    v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false);      // row_bcast:31 into rows 2 and 3
    return v;
}

// ---- the lists of steps ----
// Which sequences are a kernel's (MANY: more rows than the few-row kernel takes),
// their tiles, and a tile's positions [lo, hi] (own; lo a multiple of 32).
template <bool MANY>
__host__ __device__ __forceinline__ const PagedList &pa_list(const PagedPlan &pl) {
    if constexpr (MANY) return pl.many;
    else return pl.few;
}
template <bool MANY>
__host__ __device__ __forceinline__ int pa_tiles(const PagedPlan &pl, const PagedSeq &q) {
    if (q.nq <= pl.few.toks) return !MANY && q.nq > 0;
    if constexpr (!MANY) return 0;
    const uint32_t n = q.nq + pl.many.toks - 1;
    return pl.many.toks_inv ? (int)((uint64_t)n * pl.many.toks_inv >> 32) : (int)n;
}
// A tree's tokens (TREE) may all attend all new tokens, and start with the first one's window.
template <bool MANY, bool TREE = false>
__host__ __device__ __forceinline__ void pa_tile_span(const PagedAttn &a, const PagedPlan &pl, const PagedSeq &q, int tile, int &lo, int &hi) {
    const int first = q.len - q.nq + (MANY && !TREE ? tile * pl.many.toks : 0);
    lo = pa_low(first, a.window);
    hi = MANY && !TREE ? min(q.len, first + pl.many.toks) - 1 : q.len - 1;
}
template <bool MANY, bool TREE = false>
__host__ __device__ __forceinline__ int pa_tile_steps(const PagedAttn &a, const PagedPlan &pl, const PagedSeq &q, int tile) {
    if (q.bad) return 1;
    const PagedList &y = pa_list<MANY>(pl);
    int lo, hi;
    pa_tile_span<MANY, TREE>(a, pl, q, tile, lo, hi);
    return max(1, (hi - lo + y.unit) >> y.shift);
}
// k_paged_tree: what a step of a tile of up to 32 (k 0), up to 64 (1) and more rows
// counts as (pa_cost), and what a tile's start.  Its 8 waves take a step's rows
// and positions in 1, 2 or 4 turns, which hide behind f16's bytes more than behind
// fewer ones.  (Steps alike, a lead of 3 of them, against these, with drafts of 1 to 33
// tokens: 32 over up to 4096 positions, 8 / 4 heads of 256, 8 bits 114.6 and 94.5 us, f16
// 143.8 and 130.1; 24 over up to 6000, 32 / 8 heads of 128, 8 bits 181.6 and 137.0, 4 bits
// 198.5 and 144.2; 16 of up to 16 over 8192, f16, 69.5 and 67.0.)
__host__ __device__ constexpr int pt_cost(int type, int k) { return type == F16 ? k == 0 ? 4 : k == 1 ? 5 : 9 : k == 0 ? 3 : k == 1 ? 5 : 8; }
__host__ __device__ constexpr int pt_lead(int type) { return type == F16 ? 16 : 9; }

// What a step of a tile of `toks` tokens counts as: 1, but in k_paged_tree, whose time
// for a step goes by the rows (pt_cost).
template <bool MANY, bool TREE = false>
__host__ __device__ __forceinline__ int pa_cost(const PagedAttn &a, const PagedPlan &pl, int toks) {
    if constexpr (!MANY || !TREE) return 1;
    const int rows = toks * a.grp;
    return pt_cost(a.p.type, rows <= 32 ? 0 : rows <= 64 ? 1 : 2);
}
template <bool MANY, bool TREE = false>
__host__ __device__ __forceinline__ int pa_tile_cost(const PagedAttn &a, const PagedPlan &pl, const PagedSeq &q, int tile) {
    if constexpr (!MANY || !TREE) return 1;
    return pa_cost<MANY, TREE>(a, pl, min(q.nq - tile * pl.many.toks, pl.many.toks));
}
// steps of a sequence for one KV head, by what they count as
template <bool MANY, bool TREE = false>
__host__ __device__ __forceinline__ int pa_steps(const PagedAttn &a, const PagedPlan &pl, const PagedSeq &q) {
    const int tiles = pa_tiles<MANY>(pl, q);
    int n = 0;
    for (int t = 0; t < tiles; t++) n += pa_tile_steps<MANY, TREE>(a, pl, q, t) * pa_tile_cost<MANY, TREE>(a, pl, q, t);
    return n + tiles * pa_list<MANY>(pl).lead;
}
// All steps of the list (wave-uniform; the whole wave calls it), 64 sequences at a
// time; the lane's own of the first 64 in `mine`.  The batch ends at the first torn
// sequence, n_seq: offsets that descend would give tokens to several sequences, and
// more steps than the host counted.
template <bool MANY, bool TREE = false>
__device__ __forceinline__ int pa_total(const PagedAttn &a, const PagedPlan &pl, int &mine, int &n_seq) {
    const PagedList &y = pa_list<MANY>(pl);
    const int lane = threadIdx.x & 63;
    auto at = [&](int s0) {
        PagedSeq q = {0, 0, 0, false, false};
        if (s0 + lane < n_seq) q = paged_seq(a.p, a.b, s0 + lane);
        if (a.b.q_off) {
            const uint64_t torn = __ballot(q.torn);
            if (torn) {
                n_seq = s0 + __ffsll((unsigned long long)torn) - 1;
                if (s0 + lane >= n_seq) q.nq = 0;
            }
        }
        return pa_steps<MANY, TREE>(a, pl, q);
    };
    n_seq = a.b.n_seq;
    mine = at(0);
    int n = mine;
    for (int s0 = 64; s0 < n_seq; s0 += 64) n += at(s0);
    n_seq = pa_uniform(n_seq);
    n = pa_uniform(group_isum<64>(n));
    return (n + y.pre_tiles * y.pre_steps * pa_cost<MANY, TREE>(a, pl, y.toks)) * a.p.n_kv;
}
// The sequence whose steps hold step u (counted without the prefix's) and the
// number of steps before it.  A workgroup asks for ascending u: the search goes on
// from the 64 sequences where the last one ended.
struct PaFind {
    int s0 = 0, before = 0;
};
template <bool MANY, bool TREE = false>
__device__ __forceinline__ void pa_find_step(const PagedAttn &a, const PagedPlan &pl, int mine, int u, PaFind &from, int &seq, int &before) {
    const int lane = threadIdx.x & 63;
    for (; from.s0 < a.b.n_seq; from.s0 += 64) {
        const int n = (from.s0 == 0 ? mine : from.s0 + lane < a.b.n_seq ? pa_steps<MANY, TREE>(a, pl, paged_seq(a.p, a.b, from.s0 + lane)) : 0) * a.p.n_kv;
        const int incl = pa_scan(n);
        const uint64_t past = __ballot(from.before + incl > u);
        if (past) {
            const int l = __ffsll((unsigned long long)past) - 1;
            seq = from.s0 + l;
            before = from.before + __builtin_amdgcn_readlane(incl, l) - __builtin_amdgcn_readlane(n, l);
            return;
        }
        from.before += __builtin_amdgcn_readlane(incl, 63);
    }
    seq = a.b.n_seq;
    before = from.before;
}
__host__ __device__ __forceinline__ int pa_share(const PagedList &y, int total) { return (total + y.wgs - 1) / y.wgs; }
// Of trees no less than the dearest step: every share of a tile's then begins one.
__device__ __forceinline__ int pa_tree_share(const PagedAttn &a, const PagedPlan &pl, int total, int n_seq) {
    const PagedList &y = pl.many;
    int most = y.pre_tiles ? y.toks : 0;                     // tokens of a tile
    for (int s = threadIdx.x & 63; s < n_seq; s += 64) most = max(most, min(paged_seq(a.p, a.b, s).nq, y.toks));
    return max(pa_share(y, total), pa_cost<true, true>(a, pl, pa_uniform((int)wave_umax((uint32_t)most))));
}

// A piece: steps [step, step + n) of the `all` of one tile of one KV head.  (The
// lead comes before step 0, so the shares of the list stay contiguous.)
struct PaPiece {
    PagedSeq sq;                     // the prefix: all tokens of the batch
    int kvh, tile, step, n, all;
    int took;                        // of the share: n and what it holds of the lead; n is 0 where it ends in that (a tree: or begins behind its last step)
    int seglen, start, end;          // positions of the segment; the piece's [start, end)
    int hi0, hi1, lo0, lo1;          // the first and the last row's last and first positions (a tree: hi0 the first new token's,
                                     // hi1 the last's; lo0 and lo1 as if its depths were 0 and the most)
    int slot;                        // of its sums
    int after;                       // k_paged_tree: what lies between the piece's end and the last step's start
    const int *table;
    bool pre;
};
// steps that begin before `end`, `cost` apart; wave-uniform
__host__ __device__ __forceinline__ int pa_steps_in(int end, int cost) {
    const int n = (end + cost - 1) / cost;
#ifdef __HIP_DEVICE_COMPILE__
    return __builtin_amdgcn_readfirstlane(n);
#else
    return n;
#endif
}
// the piece at step u of a share [first, stop); find(u, seq, before) as pa_find_step
template <bool MANY, bool TREE = false, typename F>
__host__ __device__ __forceinline__ PaPiece pa_piece_by(const PagedAttn &a, const PagedPlan &pl, int n_seq, int wg, int u, int first, int stop, F find) {
    const PagedList &y = pa_list<MANY>(pl);
    const PagedBatch &b = a.b;
    PaPiece x;
    int cost = pa_cost<MANY, TREE>(a, pl, y.toks);
    const int pre_all = y.pre_tiles * y.pre_steps * cost * a.p.n_kv;
    x.pre = u < pre_all;
    int base, v, lead = 0;                                   // v: the step of the tile, its lead counted
    if (x.pre) {
        x.sq.t0 = 0;
        x.sq.nq = pa_tokens(b, n_seq);
        x.sq.len = x.seglen = b.n_prefix;
        x.sq.bad = false;
        x.all = y.pre_steps;
        const int t = u / (x.all * cost);
        v = u - t * x.all * cost;
        x.kvh = y.pre_tiles == 1 ? t : t / y.pre_tiles;
        x.tile = t - x.kvh * y.pre_tiles;
        x.table = b.prefix;
        x.hi0 = x.hi1 = x.seglen - 1;
        x.lo0 = base = 0;
        x.lo1 = a.window ? 0x7fffffff : 0;                   // row by row
    } else {
        lead = y.lead;
        int seq, before;
        find(u - pre_all, seq, before);
        x.sq = paged_seq(a.p, b, seq);
        v = u - pre_all - before;
        if constexpr (MANY) {
            const int tiles = pa_tiles<MANY>(pl, x.sq);
            int head = tiles * y.lead;                       // steps of one KV head
            for (int t = 0; t < tiles; t++) head += pa_tile_steps<MANY, TREE>(a, pl, x.sq, t) * pa_tile_cost<MANY, TREE>(a, pl, x.sq, t);
            for (x.kvh = 0; v >= head; x.kvh++) v -= head;
            for (x.tile = 0;; x.tile++) {
                x.all = pa_tile_steps<MANY, TREE>(a, pl, x.sq, x.tile);
                cost = pa_tile_cost<MANY, TREE>(a, pl, x.sq, x.tile);
                if (v < y.lead + x.all * cost) break;
                v -= y.lead + x.all * cost;
            }
        } else {
            x.all = pa_tile_steps<MANY, TREE>(a, pl, x.sq, 0);
            cost = 1;
            x.tile = 0;
            for (x.kvh = 0; v >= y.lead + x.all; x.kvh++) v -= y.lead + x.all;
        }
        pa_tile_span<MANY, TREE>(a, pl, x.sq, x.tile, base, x.hi1);
        x.hi0 = x.sq.len - x.sq.nq + (MANY && !TREE ? x.tile * pl.many.toks : 0);
        x.lo0 = a.window ? max(0, x.hi0 + 1 - a.window) : 0;
        x.lo1 = a.window ? max(0, x.hi1 + 1 - a.window) : 0;
        x.seglen = x.sq.bad ? 0 : x.sq.len;
        x.table = b.table + (size_t)seq * b.table_stride;
    }
    if constexpr (MANY && TREE) {
        x.took = min(lead + x.all * cost - v, stop - u);
        const int end = max(0, v + x.took - lead);           // steps that begin before it
        x.step = pa_steps_in(max(0, v - lead), cost);
        x.n = pa_steps_in(end, cost) - x.step;
        x.after = (x.all - 1) * cost - end;
    } else {
        x.step = max(0, v - lead);
        x.took = min(lead + x.all - v, stop - u);
        x.n = max(0, v + x.took - lead) - x.step;
    }
    x.start = base + (x.step << y.shift);
    x.end = min(x.start + (x.n << y.shift), min(x.hi1 + 1, x.seglen));
    x.slot = 2 * wg + (u != first);
    return x;
}
template <bool MANY, bool TREE = false>
__device__ __forceinline__ PaPiece pa_piece(const PagedAttn &a, const PagedPlan &pl, int mine, int n_seq, PaFind &from, int wg, int u, int first, int stop) {
    return pa_piece_by<MANY, TREE>(a, pl, n_seq, wg, u, first, stop, [&](int v, int &seq, int &before) { pa_find_step<MANY, TREE>(a, pl, mine, v, from, seq, before); });
}
// Where row r (of its tile) of a piece puts its sums: out (normalised), or `o` and
// `ml`; and, from a tile's first piece, where k_paged_join finds them.
struct PaSink {
    float *o;
    float2 *ml;
    bool out;
};
template <bool MANY, bool TREE = false>
__host__ __device__ __forceinline__ PaSink pa_sink(const PagedAttn &a, const PagedPlan &pl, const PaPiece &x, int share, int r, int tok, int head, uint32_t none, bool note) {
    const PagedList &y = pa_list<MANY>(pl);
    const size_t row = (size_t)tok * a.n_head + head;
    const bool whole = x.n == x.all;
    PaSink s;
    s.out = !x.pre && whole && a.b.n_prefix == 0;
    if (s.out) {
        s.o = a.out + (size_t)tok * a.os + (size_t)head * a.p.hd;
        s.ml = nullptr;
        if (note && pl.own) pl.own[row] = make_uint2(0, 0);
    } else if (whole) {
        const size_t at = row + (x.pre ? pl.all : 0);
        s.o = pl.wo + at * a.p.hd;
        s.ml = pl.wml + at;
        if (note) (x.pre ? pl.pre : pl.own)[row] = make_uint2(4 | none << 1 | MANY, ~0u);
    } else {
        const size_t at = (size_t)x.slot * y.rows + r;
        s.o = y.o + at * a.p.hd;
        s.ml = y.ml + at;
        if (note && x.step == 0) {
            // later pieces start the next workgroups' shares
            const int rest = x.all - x.n, count = MANY && TREE ? 2 + x.after / share : 1 + (rest + share - 1) / share;
            (x.pre ? pl.pre : pl.own)[row] = make_uint2((uint32_t)count << 2 | none << 1 | MANY, (uint32_t)x.slot << 8 | (uint32_t)r);
        }
    }
    return s;
}

// Rows of tokens that are no sequence's are noted too, so that k_paged_join goes by
// the notes alone; those from a torn sequence on become NaN.
__host__ __device__ __forceinline__ void pa_outside(const PagedAttn &a, const PagedPlan &pl, int n_seq, int thread, int threads) {
    const int before = n_seq && a.b.q_off ? paged_ld(a.b.q_off, 0) : 0, end = pa_tokens(a.b, n_seq);
    if (pl.own) {
        const int n = (before + a.b.n_tok - end) * a.n_head;             // up to 2^24
        for (int i = thread; i < n; i += threads) pl.own[i < before * a.n_head ? i : i + (end - before) * a.n_head] = make_uint2(0, 0);
    }
    if (n_seq < a.b.n_seq) {
        const int row = a.n_head * a.p.hd;
        for (int t = end; t < a.b.n_tok; t++)
            for (int e = thread; e < row; e += threads) a.out[(size_t)t * a.os + e] = __builtin_nanf("");
    }
}
// where partial result k of a row lies: the prefix's pieces, then the own ones
struct PaPart {
    const float *o;
    const float2 *ml;
};
__host__ __device__ __forceinline__ PaPart pa_part(const PagedAttn &a, const PagedPlan &pl, size_t row, uint2 pre, uint2 own, int k) {
    // both kernels' lists first: loaded where they are chosen, they are loads by lane
    const PagedList few = pl.few, many = pl.many;
    const float *const wo = pl.wo;
    const float2 *const wml = pl.wml;
    const int n_pre = pre.x >> 2, hd = a.p.hd;
    const bool in_pre = k < n_pre;
    const uint2 d = in_pre ? pre : own;
    if (!in_pre) k -= n_pre;
    const bool whole = d.y == ~0u, by_many = d.x & 1;
    const int w = min((int)(d.y >> 9) + k, (by_many ? many.wgs : few.wgs) - 1);
    const size_t slot = (size_t)(2 * w + (k == 0 ? d.y >> 8 & 1 : 0)) * (by_many ? many.rows : few.rows) + (d.y & 255);
    const size_t at = whole ? row + (in_pre ? pl.all : 0) : slot;
    return PaPart{(whole ? wo : by_many ? many.o : few.o) + at * hd, (whole ? wml : by_many ? many.ml : few.ml) + at};
}

// what one workgroup of a call does ahead of its pieces
__device__ __forceinline__ void pa_rest(const PagedAttn &a, const PagedPlan &pl, int n_seq) {
    const bool torn = n_seq < a.b.n_seq;
    if (torn && threadIdx.x == 0) paged_flag(a.p, PAGED_BAD_BATCH);
    if (torn || pl.own) pa_outside(a, pl, n_seq, threadIdx.x, blockDim.x);
}

// max of unsigned halves; the biased exponent of a (positive) half as a float
typedef unsigned short pa_v2s __attribute__((ext_vector_type(2)));
__device__ __forceinline__ uint32_t pa_pkmax(uint32_t x, uint32_t y) {
    return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(pa_v2s, x), __builtin_bit_cast(pa_v2s, y)));
}
__device__ __forceinline__ float pa_exponent(uint32_t h, int which) { return (float)((h >> (which ? 26 : 10)) & 31u); }
// A weight's offset from the running maximum: for quantized values that maximum is
// over s + the biased exponent (15 more than the exponent).
template <int KVT>
__device__ __forceinline__ constexpr float pa_shift_of() { return KVT == F16 ? PA_SHIFT : PA_SHIFT + 14.0f; }
// two halves, those that are not finite as 0
__device__ __forceinline__ uint32_t pa_finite(uint32_t x) {
    x = (x & 0x7c00u) == 0x7c00u ? x & 0xffff0000u : x;
    return (x & 0x7c000000u) == 0x7c000000u ? x & 0xffffu : x;
}
// a query row's power-of-two scaling: 2^sh times its largest magnitude am lies
// in [2^14, 2^15), within +-126; none for 0 and inf
__device__ __forceinline__ int pa_shift(float am) {
    return am > 0.0f && am < __builtin_inff() ? min(max(15 - __builtin_amdgcn_frexp_expf(am), -126), 126) : 0;
}
__device__ __forceinline__ void pa_split(float u, float v, uint32_t &hi, uint32_t &lo) {
    float minus = -1.0f;
    asm("" : "+s"(minus));                                   // or a conversion and a subtraction each
    hi = pa_pk(u, v);
    lo = pa_pk(__builtin_fmaf(pa_lo(hi), minus, u), __builtin_fmaf(pa_hi(hi), minus, v));
}
// two weights times two halves' scales, split
__device__ __forceinline__ void pa_split_scaled(float u, float v, uint32_t d, uint32_t &hi, uint32_t &lo) {
    const float x = __builtin_fmaf(pa_lo(d), u, 0.0f), y = __builtin_fmaf(pa_hi(d), v, 0.0f);
    pa_split(x, y, hi, lo);
}
// the high half of both where part is 0, the low half where it is -1
__device__ __forceinline__ uint32_t pa_half(float u, float v, float part) {
    const uint32_t hi = pa_pk(u, v);
    return pa_pk(__builtin_fmaf(pa_lo(hi), part, u), __builtin_fmaf(pa_hi(hi), part, v));
}
// factor from a raw score product to log2 units (before a cap: to tanh's argument)
template <int KVT>
__device__ __forceinline__ float pa_score_scale(const PagedAttn &a, int sh) {
    return __builtin_ldexpf(a.scale * (KVT == Q8_0 ? 512.0f : 1.0f) * (a.cap > 0.0f ? 1.0f / a.cap : 1.4426950408889634f), -sh);
}
__device__ __forceinline__ void pa_store4(float *to, pa_v4f s) {
    auto *d = (__attribute__((address_space(1))) float *)to;
    if (((uintptr_t)to & 15) == 0) *(__attribute__((address_space(1))) pa_v4f *)d = s;
    else { d[0] = s[0]; d[1] = s[1]; d[2] = s[2]; d[3] = s[3]; }
}

// The few-row kernel's workgroups per CU: what its registers allow, but for 4-bit
// heads of 128 and more, of which 3 would fit (16 windows of 1024, heads of 512: 19.7
// us with 3, 19.4 with 2).  3 of 8-bit heads of 128 fit with 32 bytes of spills: 73 us
// for 70, more results to join.
__host__ __device__ constexpr int pa_few_per_cu(int type, int hd, bool st) {
    return hd == 64 ? 4 : type == F16 && hd == 128 && st ? 3 : 2;
}

// k_paged_tree (paged_tree.h): rows of a tile at most, and the log2 of the positions
// that a workgroup takes at a time.  wide: for more query heads a KV head than its rows
__host__ __device__ constexpr int pt_rows(int hd, bool wide) { return (hd == 512 ? 32 : hd == 256 ? 64 : 128) << wide; }
__host__ __device__ constexpr int pt_shift(int type, int hd) { return hd <= 128 ? 7 : hd == 256 && type != F16 ? 6 : 5; }

// launches of one cache type; the few-row variants hold 8 or 16 rows
hipError_t pa_few_f16(const PagedAttn &a, const PagedPlan &pl, hipStream_t s);
hipError_t pa_few_q8(const PagedAttn &a, const PagedPlan &pl, hipStream_t s);
hipError_t pa_few_q4(const PagedAttn &a, const PagedPlan &pl, hipStream_t s);
hipError_t pa_many_f16(const PagedAttn &a, const PagedPlan &pl, hipStream_t s);
hipError_t pa_many_q8(const PagedAttn &a, const PagedPlan &pl, hipStream_t s);
hipError_t pa_many_q4(const PagedAttn &a, const PagedPlan &pl, hipStream_t s);
// and over trees of new tokens
hipError_t pa_tree_f16(const PagedAttn &a, const PagedPlan &pl, bool wide, hipStream_t s);
hipError_t pa_tree_q8(const PagedAttn &a, const PagedPlan &pl, bool wide, hipStream_t s);
hipError_t pa_tree_q4(const PagedAttn &a, const PagedPlan &pl, bool wide, hipStream_t s);
hipError_t pa_few_tree_f16(const PagedAttn &a, const PagedPlan &pl, hipStream_t s);
hipError_t pa_few_tree_q8(const PagedAttn &a, const PagedPlan &pl, hipStream_t s);
hipError_t pa_few_tree_q4(const PagedAttn &a, const PagedPlan &pl, hipStream_t s);

}  // namespace g4
