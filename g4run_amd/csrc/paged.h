// paged.h -- what the kernels over the paged KV cache share: the pools' layout,
// the batch's description on the device and their launchers.
#pragma once

#include "kernels.h"

namespace g4 {

constexpr int PAGED_BAD_PAGE = 1, PAGED_BAD_BATCH = 2;   // G4H_PAGED_*
constexpr int PAGED_MAX_PAGE = 4096;                     // slots of a page
constexpr int PAGED_MAX_POS = 1 << 26;                   // positions of a sequence, of a prefix

// The pools (layout: include/g4hip.h).  Positions map to pages in units of 16:
// a page is `units` such units, and u / units == umulhi(u, inv) for u < 2^22
// (PAGED_MAX_POS / 16): inv = floor(2^32 / units) + 1 exceeds 2^32 / units by at
// most 1, so the quotient is exact while u * units < 2^32, and units <= 256.
// With units == 1 the inverse does not fit 32 bits and inv is 0: the quotient is u.
struct PagedPool {
    uint8_t *k, *v;
    int64_t n_pages;
    size_t page_bytes;
    int type, n_kv, hd, page, units;
    uint32_t inv;
    uint32_t sc_off;                 // quantized: offset of a page's scales
    int *status;
};
struct PagedBatch {
    int n_seq, n_tok;
    const int *q_off, *len, *table;
    int table_stride, max_len, n_prefix;
    const int *prefix;
};
struct PagedRope {
    int n_rot, interleaved;
    double log2_base;
    const float *factor;
};

__host__ __device__ constexpr int paged_row_bytes(int type, int hd) { return type == F16 ? hd * 2 : type == Q8_0 ? hd : hd / 2; }

// query heads of a KV head at most: a token's rows share a tile
__host__ __device__ constexpr int paged_most_group(int hd) { return hd > 256 ? 64 : 128; }

// page entry and slot of unit u
__device__ __forceinline__ int paged_entry(const PagedPool &p, int u) { return p.inv ? (int)__umulhi((uint32_t)u, p.inv) : u; }

__device__ __forceinline__ void paged_flag(const PagedPool &p, int bits) {
    if (p.status) atomicOr(p.status, bits);
}

// The batch's arrays do not change while a call runs: read through the constant
// address space, a wave-uniform index takes a scalar load, which does not wait
// behind the vector loads in flight.  (The host's twin of the split reads its own.)
__host__ __device__ __forceinline__ int paged_ld(const int *p, int64_t i) {
#ifdef __HIP_DEVICE_COMPILE__
    return ((const __attribute__((address_space(4))) int *)p)[i];
#else
    return p[i];
#endif
}

// A sequence as a call may use it: its tokens [t0, t0 + nq) within n_tok, its
// length; bad lengths and offsets are flagged by the caller.
struct PagedSeq {
    int t0, nq, len;
    bool bad, torn;                  // torn: by its offsets
};
__host__ __device__ __forceinline__ PagedSeq paged_seq(const PagedPool &p, const PagedBatch &b, int s) {
    PagedSeq r;
    r.len = paged_ld(b.len, s);
    r.torn = false;
    r.bad = r.len < 0 || r.len > b.max_len || (int64_t)r.len > (int64_t)b.table_stride * p.page;
    if (b.q_off) {
        const int a = paged_ld(b.q_off, s), e = paged_ld(b.q_off, s + 1);
        r.t0 = min(max(a, 0), b.n_tok);
        r.nq = min(max(e, r.t0), b.n_tok) - r.t0;
        r.torn = r.t0 != a || r.t0 + r.nq != e;
        r.bad |= r.torn;
    } else {
        r.t0 = s;
        r.nq = s < b.n_tok ? 1 : 0;
    }
    return r;
}

// The sequence of token t, found by one wave together: the last s with
// q_off[s] <= t, by 64 offsets at a time (4096 sequences: two reads); n_seq when t
// is behind all of them.
__device__ __forceinline__ int paged_find(const PagedBatch &b, int t) {
    if (!b.q_off) return t < b.n_seq ? t : b.n_seq;
    const int lane = threadIdx.x & 63;
    int lo = 0, hi = b.n_seq;                                // it is one of lo .. hi
    while (hi - lo > 64) {
        const int step = (hi - lo + 63) >> 6, s = lo + (lane + 1) * step;
        lo += step * __popcll(__ballot(s <= hi && paged_ld(b.q_off, min(s, hi)) <= t));
        hi = min(hi, lo + step - 1);
    }
    const int s = lo + 1 + lane;
    return lo + __popcll(__ballot(s <= hi && paged_ld(b.q_off, min(s, hi)) <= t));
}

// whether paged_find's sequence `seq` stands for none: t lies before all of them
__device__ __forceinline__ bool paged_before(const PagedSeq &q, int seq, int t) { return seq == 0 && !q.torn && t < q.t0; }

struct PagedAppend {
    PagedPool p;
    PagedBatch b;
    PagedRope r;
    int n_head, tokens;              // query heads; tokens per workgroup
    int rows;                        // rows (heads) per workgroup
    const float *q, *k, *v;
    float *q_out;
    size_t qs, qos, ks, vs;
};
hipError_t launch_paged_append(const PagedAppend &a, hipStream_t s);

struct PagedRead {
    PagedPool p;
    PagedBatch b;
    void *k_out, *v_out;
    int f16;
};
hipError_t launch_paged_read(const PagedRead &a, hipStream_t s);

struct PagedAttn {
    PagedPool p;
    PagedBatch b;
    int n_head, grp;
    const float *q;
    float *out;
    size_t qs, os;
    float scale, cap;
    int window;
    uint8_t *ws;
};
// workspace of a call: the workgroups' partial results and where each (token, head)
// row's lie, 0 where a call writes its outputs directly
size_t paged_attn_workspace(const PagedPool &p, const PagedBatch &b, int n_head);
hipError_t launch_paged_attn(PagedAttn a, hipStream_t s);

}  // namespace g4
