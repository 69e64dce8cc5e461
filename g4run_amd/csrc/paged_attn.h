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
// Precision: fp32.  K and V enter exactly (halves, or the integers of the block
// formats, their scales applied in fp32 to the scores and to the weights).  A
// query row is scaled by a power of two to [2^14, 2^15) and split into two
// halves (22 bits), a weight likewise.  Weights are exp2(s - m + 12), for
// quantized values with m over s + the exponent of the position's largest
// scale, so weight x scale neither overflows nor falls among the halves'
// subnormals while it matters.
//
// Two kernels share a call:
//   k_paged_few   row tiles of up to 16 rows (single tokens; the prefix of a small
//                 batch): bound by the cache's bytes.  The batch's positions are
//                 one list of steps, dealt evenly to the workgroups.
//   k_paged_many  sequences of more rows (prompt chunks; the prefix of a large
//                 batch): bound by the matrix cores.  K and V pass through LDS
//                 once for up to 128 rows.
// Partial results go through the workspace to k_paged_join.
#pragma once

#include "paged.h"

namespace g4 {

typedef _Float16 pa_v8h __attribute__((ext_vector_type(8)));
typedef _Float16 pa_v2h __attribute__((ext_vector_type(2)));
typedef float pa_v4f __attribute__((ext_vector_type(4)));
typedef float pa_v16f __attribute__((ext_vector_type(16)));
typedef uint32_t pa_v4u __attribute__((ext_vector_type(4)));

// The split of a call.  Partial results: the few-row kernel's [wgs][2][R] (a
// workgroup's first and last piece), and per row [nown] own chunks (a whole few-row
// sequence beside a prefix: chunk 0) and [npre] prefix chunks.
struct PagedPlan {
    int few_rows;                    // sequences of up to this many rows are the few-row kernel's
    int few_wgs, few_unit, few_shift;    // its workgroups; positions of a step, and their log2
    uint32_t grp_inv;                // rows to tokens: r / grp == r * grp_inv >> 16 for r < 16
    int few_pre;                     // whether the prefix is its too: steps of the prefix (0: no)
    int many_rows;                   // rows of a workgroup of the many-row kernel
    int own_slots, nown, own_chunk;  // its tiles of the sequences' own positions, and chunks
    int pre_slots, npre, pre_chunk;  // and of the prefix's
    float *fo, *oo, *po;             // unnormalised sums: few, own, prefix
    float2 *fml, *oml, *pml;         // maximum (log2), sum
};

constexpr float PA_SHIFT = 12.0f;    // weights are scaled by 2^12: their low halves stay normal

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
// halves 1024 + (quant + 8) to quant, exactly
__device__ __forceinline__ uint32_t pa_q4(uint32_t x) {
    const pa_v2h c = {(_Float16)-1032.0f, (_Float16)-1032.0f};
    return __builtin_bit_cast(uint32_t, __builtin_bit_cast(pa_v2h, x) + c);
}
__device__ __forceinline__ uint32_t pa_nib(uint32_t w, int k) { return ((w >> (4 * k)) & 0x000f000fu) | 0x64006400u; }

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
template <int KVT>
__device__ __forceinline__ PaUnits pa_units(const PagedPool &p, const int *table, int first, int stride, int last, int kvh, bool &bad) {
    const int lane = threadIdx.x & 63, u = min(first + stride * (lane >> 1) + (lane & 1), last), ent = paged_entry(p, u);
    PaUnits x;
    x.id = paged_ld(table, ent);
    x.row = kvh * p.page + (u - ent * p.units) * 16;
    if ((uint64_t)(int64_t)x.id >= (uint64_t)p.n_pages) { bad = true; x.id = 0; }
    return x;
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

// log2(e) cap tanh(x): an odd polynomial below 0.3 (next term 9e-3 x^11, below
// 6e-8 x there), where 1 - exp would lose the small value
__device__ __forceinline__ float pa_tanh(float x) {
    const float x2 = x * x;
    float p = __builtin_fmaf(x2, 62.0f / 2835.0f, -17.0f / 315.0f);
    p = __builtin_fmaf(x2, p, 2.0f / 15.0f);
    p = __builtin_fmaf(x2, p, -1.0f / 3.0f);
    p = __builtin_fmaf(x * x2, p, x);
    const float ax = fabsf(x);
    if (__any(ax > 0.3f)) {
        const float t = __builtin_amdgcn_exp2f(-2.885390081777927f * ax);
        const float r = (1.0f - t) * __builtin_amdgcn_rcpf(1.0f + t);
        p = ax > 0.3f ? copysignf(r, x) : p;
        p = x == x ? p : x;
    }
    return p;
}

// the batch's rows that attend the prefix
__device__ __forceinline__ int pa_tokens(const PagedBatch &b) {
    return b.q_off ? min(max(paged_ld(b.q_off, b.n_seq), 0), b.n_tok) : min(b.n_seq, b.n_tok);
}
// first own position that tokens from `first` on attend, rounded down to 32
__device__ __forceinline__ int pa_low(int first, int window) { return window ? max(0, first + 1 - window) & ~31 : 0; }

// position of global token tok (prefix included), its sequence looked up
__device__ __forceinline__ int pa_token_pos(const PagedPool &p, const PagedBatch &b, int tok) {
    int s = tok;
    if (b.q_off) {
        int x = 0, y = b.n_seq;                              // last s with q_off[s] <= tok
        while (y - x > 1) {
            const int z = (x + y) >> 1;
            if (paged_ld(b.q_off, z) <= tok) x = z;
            else y = z;
        }
        s = x;
    }
    const PagedSeq o = paged_seq(p, b, s);
    return b.n_prefix + o.len - o.nq + (tok - o.t0);
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

// ---- the few-row kernel's list of steps ----
__device__ __forceinline__ int pa_seq_steps(const PagedAttn &a, const PagedPlan &pl, const PagedSeq &q) {
    return q.bad ? 1 : max(1, (q.len - pa_low(q.len - q.nq, a.window) + pl.few_unit - 1) >> pl.few_shift);
}
// steps of sequence s for one KV head: 0 when it is not this kernel's
__device__ __forceinline__ int pa_steps(const PagedAttn &a, const PagedPlan &pl, int s) {
    const PagedSeq q = paged_seq(a.p, a.b, s);
    if (q.nq == 0 || q.nq * a.grp > pl.few_rows) return 0;
    return pa_seq_steps(a, pl, q);
}
// All steps of the call (wave-uniform; the whole wave calls it), 64 sequences
// at a time; the first 64 sequences' own in `mine`.
__device__ __forceinline__ int pa_total(const PagedAttn &a, const PagedPlan &pl, int &mine) {
    const int lane = threadIdx.x & 63;
    mine = lane < a.b.n_seq ? pa_steps(a, pl, lane) : 0;
    int n = mine;
    for (int s = 64 + lane; s < a.b.n_seq; s += 64) n += pa_steps(a, pl, s);
    n = pa_uniform(group_isum<64>(n));
    return (n + pl.few_pre) * a.p.n_kv;
}
// the sequence whose steps hold step u (counted without the prefix's) and the
// number of steps before it
__device__ __forceinline__ void pa_find_step(const PagedAttn &a, const PagedPlan &pl, int mine, int u, int &seq, int &before) {
    const int lane = threadIdx.x & 63;
    before = 0;
    for (int s0 = 0; s0 < a.b.n_seq; s0 += 64) {
        const int n = (s0 == 0 ? mine : s0 + lane < a.b.n_seq ? pa_steps(a, pl, s0 + lane) : 0) * a.p.n_kv;
        const int incl = pa_scan(n);
        const uint64_t past = __ballot(before + incl > u);
        if (past) {
            const int l = __ffsll((unsigned long long)past) - 1;
            seq = s0 + l;
            before += __builtin_amdgcn_readlane(incl, l) - __builtin_amdgcn_readlane(n, l);
            return;
        }
        before += __builtin_amdgcn_readlane(incl, 63);
    }
    seq = a.b.n_seq;
}
// the steps before sequence `seq` (wave-uniform)
__device__ __forceinline__ int pa_before(const PagedAttn &a, const PagedPlan &pl, int mine, int seq) {
    const int lane = threadIdx.x & 63;
    int n = lane < seq ? mine : 0;
    for (int s = 64 + lane; s < seq; s += 64) n += pa_steps(a, pl, s);
    return pa_uniform(group_isum<64>(n)) * a.p.n_kv;
}
// steps of a workgroup: fewer than PA_FEW_WGS workgroups are launched only where
// each step has one
constexpr int PA_FEW_WGS = 512;
__device__ __forceinline__ int pa_share(int total) { return max(1, (total + PA_FEW_WGS - 1) / PA_FEW_WGS); }

// ---- the many-row kernel's tiles ----
// The slot-th row tile (wave-uniform): sequences' tiles one after another.
// seq = n_seq when there are fewer.
__device__ __forceinline__ void pa_find_tile(const PagedAttn &a, const PagedPlan &pl, int slot, int &seq, int &tile) {
    const PagedBatch &b = a.b;
    const int R = pl.many_rows;
    if (!b.q_off) {
        const int per = (a.grp + R - 1) / R;
        seq = slot / per;
        tile = slot - seq * per;
        return;
    }
    const int lane = threadIdx.x & 63;
    int before = 0;
    for (int s0 = 0; s0 < b.n_seq; s0 += 64) {
        const int s = s0 + lane;
        int n = 0;
        if (s < b.n_seq) {
            const int nq = paged_seq(a.p, b, s).nq;
            if (nq > pl.few_rows / a.grp) n = (nq * a.grp + R - 1) / R;
        }
        const int incl = pa_scan(n);
        const uint64_t past = __ballot(before + incl > slot);
        if (past) {
            const int l = __ffsll((unsigned long long)past) - 1;
            seq = s0 + l;
            tile = slot - before - (__builtin_amdgcn_readlane(incl, l) - __builtin_amdgcn_readlane(n, l));
            return;
        }
        before += __builtin_amdgcn_readlane(incl, 63);
    }
    seq = b.n_seq;
    tile = 0;
}
// own positions of a row tile: [lo, hi], lo a multiple of 32; and its chunks
__device__ __forceinline__ void pa_tile_span(const PagedSeq &q, int grp, int R, int tile, int window, int &lo, int &hi) {
    lo = pa_low(q.len - q.nq + tile * R / grp, window);
    hi = q.len - q.nq + min(q.nq - 1, ((tile + 1) * R - 1) / grp);
}
__device__ __forceinline__ int pa_tile_chunks(const PagedSeq &q, const PagedPlan &pl, int lo, int hi) {
    return q.bad ? 1 : min(pl.nown, max(1, (hi + pl.own_chunk - lo) / pl.own_chunk));
}

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
    hi = pa_pk(u, v);
    lo = pa_pk(u - pa_lo(hi), v - pa_hi(hi));
}
// factor from a raw score product to log2 units (before a cap: to tanh's argument)
template <int KVT>
__device__ __forceinline__ float pa_score_scale(const PagedAttn &a, int sh) {
    return __builtin_ldexpf(a.scale * (KVT == Q8_0 ? 512.0f : 1.0f) * (a.cap > 0.0f ? 1.0f / a.cap : 1.4426950408889634f), -sh);
}
__device__ __forceinline__ void pa_store4(float *d, pa_v4f s) {
    if (((uintptr_t)d & 15) == 0) *(pa_v4f *)d = s;
    else { d[0] = s[0]; d[1] = s[1]; d[2] = s[2]; d[3] = s[3]; }
}

// launches of one cache type; the few-row variants hold 8 or 16 rows
hipError_t pa_few_f16(const PagedAttn &a, const PagedPlan &pl, hipStream_t s);
hipError_t pa_few_q8(const PagedAttn &a, const PagedPlan &pl, hipStream_t s);
hipError_t pa_few_q4(const PagedAttn &a, const PagedPlan &pl, hipStream_t s);
hipError_t pa_many_f16(const PagedAttn &a, const PagedPlan &pl, unsigned blocks, hipStream_t s);
hipError_t pa_many_q8(const PagedAttn &a, const PagedPlan &pl, unsigned blocks, hipStream_t s);
hipError_t pa_many_q4(const PagedAttn &a, const PagedPlan &pl, unsigned blocks, hipStream_t s);

}  // namespace g4
