// paged_attn.h -- attention over the paged KV cache (g4h_paged_attn): the
// kernel template, instantiated per cache type by k_paged_f16 / q8 / q4.hip.
//
// Mathematics: one pass over the positions with the running maximum and sum of
// a softmax, per tile of (token, query head) rows of one KV head, 32 positions
// at a time on v_mfma_f32_16x16x32_f16:
//   S^T [positions][rows] = K q^T, then O^T [elements][rows] += V^T P^T.
// With the scores transposed, a lane holds 8 positions of one row (4 g + i of
// two 16-position units, row c: lane = 16 g + c), which is the second product's
// operand as it stands: the weights never leave their registers.
//
// Precision: fp32.  K and V enter exactly (halves, or the integers of the block
// formats, their scales applied in fp32 to the scores and to the weights).  A
// query row is scaled by a power of two to [2^14, 2^15) and split into two
// halves (22 bits), a weight likewise.  Up to 8 rows (decode) sit in a 16-row
// operand as high halves (columns 0..7) and low halves (8..15), so the second
// half costs no matrix instruction; larger tiles take two.  Weights are
// exp2(s - m + 12), for quantized values with m over s + the exponent of the
// position's largest scale, so weight x scale neither overflows nor falls
// among the halves' subnormals while it matters.
//
// Memory: K and V go from the pages to registers, each lane's loads being the
// operand's runs of bytes (the layout of the quantized rows is made for it); the
// f16 value rows are turned (8 positions x 2 elements) with v_perm_b32.
#pragma once

#include "paged.h"

namespace g4 {

typedef _Float16 pa_v8h __attribute__((ext_vector_type(8)));
typedef _Float16 pa_v2h __attribute__((ext_vector_type(2)));
typedef float pa_v4f __attribute__((ext_vector_type(4)));
typedef uint32_t pa_v4u __attribute__((ext_vector_type(4)));

// The split of a call (paged_plan): tiles of `rows` rows; own positions in
// `nown` chunks of `own_chunk`, the prefix's in `npre` of `pre_chunk`; partial
// results [n_tok * n_head][nsplit] in the workspace unless there is one split.
struct PagedPlan {
    int own_slots, nown, own_chunk;
    int pre_slots, npre, pre_chunk;
    int nsplit;
    float *po;                       // [row][nsplit][hd] unnormalised sums
    float2 *ml;                      // [row][nsplit] maximum (log2), sum
};

constexpr int PA_WAVES = 4;          // waves of a workgroup: they share its rows and take every fourth tile of 32 positions
constexpr float PA_SHIFT = 12.0f;    // weights are scaled by 2^12: their low halves stay normal

__device__ __forceinline__ int pa_uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ uint32_t pa_pk(float a, float b) { return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(a, b)); }
__device__ __forceinline__ float pa_lo(uint32_t h) { return (float)__builtin_bit_cast(pa_v2h, h)[0]; }
__device__ __forceinline__ float pa_hi(uint32_t h) { return (float)__builtin_bit_cast(pa_v2h, h)[1]; }
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

// the largest / smallest over the 16 rows of a lane group
__device__ __forceinline__ int pa_rmax(int v) {
    v = max(v, partner<1>(v));
    v = max(v, partner<2>(v));
    v = max(v, partner<4>(v));
    return max(v, partner<8>(v));
}

// Operands of 32 positions: raw bytes as loaded.
template <int HD, int KVT>
struct PaTile {
    static constexpr int KW = KVT == F16 ? HD / 16 : KVT == Q8_0 ? HD / 16 : HD / 32;    // dwords of a lane's key run (q8/q4); f16: 4 per step
    static constexpr int VW = KVT == F16 ? HD / 32 : KVT == Q8_0 ? HD / 64 : (HD >= 128 ? HD / 128 : 1);
    static constexpr int DW = HD / 64;                                                   // dwords of a row's scales
    uint32_t k[2][KVT == F16 ? HD / 8 : KW];   // [unit][dwords]
    uint32_t v[8][VW];                         // [position 4 t + i][dwords]
    uint32_t dk[KVT == F16 ? 1 : 8][DW], dv[KVT == F16 ? 1 : 8][DW];
};

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

// unit u (16 positions) of the segment: the offset of its rows of KV head kvh in
// the pools (row 0) and, quantized, of their scales
struct PaUnit {
    size_t row, sc;
};
template <int HD, int KVT>
__device__ __forceinline__ PaUnit pa_unit(const PagedPool &p, const int *table, int u, int last, int kvh, bool &bad) {
    u = min(u, last);
    const int ent = paged_entry(p, u);
    int id = table[ent];
    if ((uint64_t)(int64_t)id >= (uint64_t)p.n_pages) { bad = true; id = 0; }
    const uint32_t r = (uint32_t)kvh * p.page + (uint32_t)(u - ent * p.units) * 16;
    PaUnit x;
    x.row = (size_t)id * p.page_bytes + (size_t)r * paged_row_bytes(KVT, HD);
    x.sc = KVT == F16 ? 0 : (size_t)id * p.page_bytes + p.sc_off + (size_t)r * (HD / 16);
    return x;
}

template <int HD, int KVT>
__device__ __forceinline__ void pa_load_k(PaTile<HD, KVT> &t, const PagedPool &p, const PaUnit u[2], int c, int g) {
#pragma unroll
    for (int h = 0; h < 2; h++) {
        const uint8_t *row = p.k + u[h].row + (size_t)c * paged_row_bytes(KVT, HD);
        if constexpr (KVT == F16) {
#pragma unroll
            for (int s = 0; s < HD / 32; s++) pa_load<4>(t.k[h] + 4 * s, row + 64 * s + 16 * g);
        } else {
            pa_load<PaTile<HD, KVT>::KW>(t.k[h], row + 4 * PaTile<HD, KVT>::KW * g);
#pragma unroll
            for (int i = 0; i < 4; i++) pa_load<PaTile<HD, KVT>::DW>(t.dk[4 * h + i], p.k + u[h].sc + (4 * g + i) * (HD / 16));
        }
    }
}
template <int HD, int KVT>
__device__ __forceinline__ void pa_load_v(PaTile<HD, KVT> &t, const PagedPool &p, const PaUnit u[2], int c, int g) {
#pragma unroll
    for (int j = 0; j < 8; j++) {
        const int i = 4 * g + (j & 3);
        const uint8_t *row = p.v + u[j >> 2].row + (size_t)i * paged_row_bytes(KVT, HD);
        if constexpr (KVT == F16 && HD == 64) {
            pa_load<2>(t.v[j], row + 8 * c);
        } else if constexpr (KVT == F16) {
#pragma unroll
            for (int n = 0; n < HD / 128; n++) pa_load<4>(t.v[j] + 4 * n, row + 256 * n + 16 * c);
        } else if constexpr (KVT == Q4_0 && HD == 64) {
            t.v[j][0] = *(const uint16_t *)(row + 2 * c);
        } else {
            pa_load<PaTile<HD, KVT>::VW>(t.v[j], row + 4 * PaTile<HD, KVT>::VW * c);
        }
        if constexpr (KVT != F16) pa_load<PaTile<HD, KVT>::DW>(t.dv[j], p.v + u[j >> 2].sc + i * (HD / 16));
    }
}

// key operand of unit h, 32 elements s
template <int HD, int KVT>
__device__ __forceinline__ pa_v8h pa_key(const PaTile<HD, KVT> &t, int h, int s) {
    if constexpr (KVT == F16) return pa_op(t.k[h][4 * s], t.k[h][4 * s + 1], t.k[h][4 * s + 2], t.k[h][4 * s + 3]);
    else if constexpr (KVT == Q8_0) {
        const uint32_t a = t.k[h][2 * s], b = t.k[h][2 * s + 1];
        return pa_op(pa_q8(__builtin_amdgcn_perm(0, a, 0x0c010c00u)), pa_q8(__builtin_amdgcn_perm(0, a, 0x0c030c02u)),
                     pa_q8(__builtin_amdgcn_perm(0, b, 0x0c010c00u)), pa_q8(__builtin_amdgcn_perm(0, b, 0x0c030c02u)));
    } else {
        const uint32_t w = t.k[h][s];
        return pa_op(pa_q4(pa_nib(w, 0)), pa_q4(pa_nib(w, 1)), pa_q4(pa_nib(w, 2)), pa_q4(pa_nib(w, 3)));
    }
}
// value operand of the 16 elements m (pa_elem) over the 32 positions
template <int HD, int KVT>
__device__ __forceinline__ pa_v8h pa_value(const PaTile<HD, KVT> &t, int m) {
    uint32_t w[4];
#pragma unroll
    for (int k = 0; k < 4; k++) {
        if constexpr (KVT == F16) {
            const int d = HD == 64 ? m >> 1 : 4 * (m >> 3) + ((m & 7) >> 1);
            w[k] = __builtin_amdgcn_perm(t.v[2 * k + 1][d], t.v[2 * k][d], (m & 1) ? 0x07060302u : 0x05040100u);
        } else if constexpr (KVT == Q8_0) {
            const uint32_t b = m & 3;
            w[k] = pa_q8(__builtin_amdgcn_perm(t.v[2 * k + 1][m >> 2], t.v[2 * k][m >> 2], 0x0c000c00u | b | ((4 + b) << 16)));
        } else {
            const int d = m >> 3, n = m & 3;
            w[k] = pa_q4(__builtin_amdgcn_perm(pa_nib(t.v[2 * k + 1][d], n), pa_nib(t.v[2 * k][d], n), (m & 4) ? 0x07060302u : 0x05040100u));
        }
    }
    return pa_op(w[0], w[1], w[2], w[3]);
}
// element of a row that value tile m holds in its operand row x (0..15)
template <int HD, int KVT>
__device__ __forceinline__ int pa_elem(int m, int x) {
    return KVT != F16 ? 16 * m + x : HD == 64 ? 4 * x + m : 128 * (m >> 3) + 8 * x + (m & 7);
}
__device__ __forceinline__ float pa_scale(const uint32_t *d, int b) { return (b & 1) ? pa_hi(d[b >> 1]) : pa_lo(d[b >> 1]); }

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

// The slot-th row tile of the batch (wave-uniform): sequences' tiles one after
// another, counted 64 sequences at a time.  seq = n_seq when there are fewer.
__device__ __forceinline__ void pa_find_tile(const PagedPool &p, const PagedBatch &b, int grp, int R, int slot, int &seq, int &tile) {
    if (!b.q_off) {
        const int per = (grp + R - 1) / R;
        seq = slot / per;
        tile = slot - seq * per;
        return;
    }
    const int lane = threadIdx.x & 63;
    int before = 0;
    for (int s0 = 0; s0 < b.n_seq; s0 += 64) {
        const int s = s0 + lane;
        int n = 0;
        if (s < b.n_seq) n = (paged_seq(p, b, s).nq * grp + R - 1) / R;
        int incl = n;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const int o = __shfl_up(incl, d, 64);
            incl += lane >= d ? o : 0;
        }
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
    const int first = q.len - q.nq + tile * R / grp, last = q.len - q.nq + min(q.nq - 1, ((tile + 1) * R - 1) / grp);
    lo = window ? max(0, first + 1 - window) & ~31 : 0;
    hi = last;
}
__device__ __forceinline__ int pa_tile_chunks(const PagedSeq &q, const PagedPlan &pl, int lo, int hi) {
    return q.bad ? 1 : min(pl.nown, max(1, (hi + pl.own_chunk - lo) / pl.own_chunk));
}

// One workgroup: one row tile of one KV head against one chunk of positions.
// grid: pre_slots x n_kv x npre prefix items, then own_slots x n_kv x nown.
template <int HD, int KVT, int NT, bool ST>
__global__ __launch_bounds__(64 * PA_WAVES, (HD >= 256 && !ST) || HD == 512 ? 1 : 2) void k_paged_attn(PagedAttn a, PagedPlan pl) {
    constexpr int R = ST ? 8 : 16 * NT, NS = HD / 32, NM = HD / 16;
    constexpr float KS = KVT == Q8_0 ? 512.0f : 1.0f;        // pa_q8's 2^-9
    __shared__ float buf[PA_WAVES][8][HD + 4];
    __shared__ float2 wml[PA_WAVES][R];
    const int lane = threadIdx.x & 63, wave = pa_uniform(threadIdx.x >> 6), c = lane & 15, g = lane >> 4;
    const PagedPool &p = a.p;
    const PagedBatch &b = a.b;
    const int G = a.grp;

    // the item
    int item = blockIdx.x, split;
    const int npre_items = pl.pre_slots * p.n_kv * pl.npre;
    const bool pre = item < npre_items;
    if (!pre) item -= npre_items;
    const int slots = pre ? pl.pre_slots : pl.own_slots;
    const int tslot = item % slots;
    item /= slots;
    const int kvh = item % p.n_kv, chunk = item / p.n_kv;
    PagedSeq sq;
    int tile = tslot, seglen, start, end;
    const int *table;
    bool bad = false;
    if (pre) {
        sq.t0 = 0;
        sq.nq = b.q_off ? min(max(b.q_off[b.n_seq], 0), b.n_tok) : min(b.n_seq, b.n_tok);
        sq.bad = false;
        if (tile * R >= sq.nq * G) return;
        seglen = b.n_prefix;
        table = b.prefix;
        start = chunk * pl.pre_chunk;
        end = min(start + pl.pre_chunk, seglen);
        split = chunk;
        sq.len = seglen;
    } else {
        int seq;
        pa_find_tile(p, b, G, R, tslot, seq, tile);
        seq = pa_uniform(seq);
        tile = pa_uniform(tile);
        if (seq >= b.n_seq) return;
        sq = paged_seq(p, b, seq);
        if (tile * R >= sq.nq * G) return;
        if (sq.bad) bad = true;
        int lo, hi;
        pa_tile_span(sq, G, R, tile, a.window, lo, hi);
        if (chunk >= pa_tile_chunks(sq, pl, lo, hi)) return;
        if (sq.bad && threadIdx.x == 0) paged_flag(p, PAGED_BAD_BATCH);
        seglen = sq.bad ? 0 : sq.len;
        table = b.table + (size_t)seq * b.table_stride;
        start = lo + chunk * pl.own_chunk;
        end = min(start + pl.own_chunk, hi + 1);
        split = pl.npre + chunk;
    }

    // the lane's rows: positions [rlo, rhi] of this segment
    int rlo[NT], rhi[NT], mx_hi = -1, mn_hi = 0x7fffffff, mx_lo = 0, mn_lo = 0x7fffffff;
    pa_v8h q0[NT][NS], q1[ST ? 1 : NT][ST ? 1 : NS];
    float qs[NT];
#pragma unroll
    for (int t = 0; t < NT; t++) {
        const int r = tile * R + 16 * t + (ST ? c & 7 : c);
        const bool ok = r < sq.nq * G;
        const int i = ok ? r / G : 0, h = ok ? r - i * G : 0;
        const int tok = sq.t0 + i;
        if (pre) {
            rhi[t] = b.n_prefix - 1;
            rlo[t] = 0;
            if (a.window && ok) {                            // the token's own position is needed
                int s = tok;
                if (b.q_off) {
                    int x = 0, y = b.n_seq;                  // last s with q_off[s] <= tok
                    while (y - x > 1) {
                        const int z = (x + y) >> 1;
                        if (b.q_off[z] <= tok) x = z;
                        else y = z;
                    }
                    s = x;
                }
                const PagedSeq o = paged_seq(p, b, s);
                rlo[t] = max(0, b.n_prefix + o.len - o.nq + (tok - o.t0) + 1 - a.window);
            }
        } else {
            rhi[t] = sq.len - sq.nq + i;
            rlo[t] = a.window ? max(0, rhi[t] + 1 - a.window) : 0;
        }
        if (ok) {
            mx_hi = max(mx_hi, rhi[t]);
            mn_hi = min(mn_hi, rhi[t]);
            mx_lo = max(mx_lo, rlo[t]);
            mn_lo = min(mn_lo, rlo[t]);
        }
        // the query row: 8 elements of each 32, scaled by 2^sh, in two halves
        const float *qr = a.q + (size_t)tok * a.qs + (size_t)(kvh * G + h) * HD;
        float x[NS][8], am = 0.0f;
#pragma unroll
        for (int s = 0; s < NS; s++)
#pragma unroll
            for (int j = 0; j < 8; j++) {
                x[s][j] = ok ? qr[32 * s + 8 * g + j] : 0.0f;
                am = fmaxf(am, fabsf(x[s][j]));
            }
        am = fmaxf(am, partner<16>(am));
        am = fmaxf(am, partner<32>(am));
        // am in [2^e, 2^(e+1)): sh = 14 - e, within +-126; no scaling of 0, inf
        int sh = 0;
        if (am > 0.0f && am < __builtin_inff()) sh = min(max(15 - __builtin_amdgcn_frexp_expf(am), -126), 126);
        qs[t] = __builtin_ldexpf(a.scale * KS * (a.cap > 0.0f ? 1.0f / a.cap : 1.4426950408889634f), -sh);
#pragma unroll
        for (int s = 0; s < NS; s++) {
            uint32_t hi[4], lo[4];
#pragma unroll
            for (int k = 0; k < 4; k++) {
                const float u = __builtin_ldexpf(x[s][2 * k], sh), v = __builtin_ldexpf(x[s][2 * k + 1], sh);
                hi[k] = pa_pk(u, v);
                lo[k] = pa_pk(u - pa_lo(hi[k]), v - pa_hi(hi[k]));
            }
            if constexpr (ST) {
                q0[t][s] = c < 8 ? pa_op(hi[0], hi[1], hi[2], hi[3]) : pa_op(lo[0], lo[1], lo[2], lo[3]);
            } else {
                q0[t][s] = pa_op(hi[0], hi[1], hi[2], hi[3]);
                q1[t][s] = pa_op(lo[0], lo[1], lo[2], lo[3]);
            }
        }
    }
    mx_hi = pa_uniform(pa_rmax(mx_hi));
    mn_hi = pa_uniform(-pa_rmax(-mn_hi));
    mx_lo = pa_uniform(pa_rmax(mx_lo));
    mn_lo = pa_uniform(-pa_rmax(-mn_lo));
    end = min(end, min(mx_hi + 1, seglen));
    start = max(start, mn_lo & ~31);

    pa_v4f o[NT][NM];
    float m[NT], l[NT];
#pragma unroll
    for (int t = 0; t < NT; t++) {
        m[t] = -__builtin_inff();
        l[t] = 0.0f;
#pragma unroll
        for (int e = 0; e < NM; e++) o[t][e] = pa_v4f{0.0f, 0.0f, 0.0f, 0.0f};
    }
    const float capl = a.cap * 1.4426950408889634f;
    const int last = (seglen - 1) >> 4;

    for (int base = start + 32 * wave; base < end; base += 32 * PA_WAVES) {
        PaTile<HD, KVT> kv;
        const PaUnit u[2] = {pa_unit<HD, KVT>(p, table, base >> 4, last, kvh, bad), pa_unit<HD, KVT>(p, table, (base >> 4) + 1, last, kvh, bad)};
        pa_load_k<HD, KVT>(kv, p, u, c, g);
        pa_load_v<HD, KVT>(kv, p, u, c, g);
        const bool edge = base + 31 > mn_hi || base < mx_lo || base + 32 > seglen;
        float w[NT][8], ex[8];
        if constexpr (KVT != F16) {
            // exponent of the position's largest value scale
#pragma unroll
            for (int j = 0; j < 8; j++) {
                uint32_t dm = 0;
#pragma unroll
                for (int d = 0; d < HD / 64; d++) dm = max(dm, max(kv.dv[j][d] & 0x7fffu, (kv.dv[j][d] >> 16) & 0x7fffu));
                ex[j] = (float)__builtin_amdgcn_frexp_expf(h2f((uint16_t)dm));
            }
        }
#pragma unroll
        for (int t = 0; t < NT; t++) {
            // scores of the lane's row at positions base + 16 h + 4 g + i
            pa_v4f sc[2] = {{0.0f, 0.0f, 0.0f, 0.0f}, {0.0f, 0.0f, 0.0f, 0.0f}};
#pragma unroll
            for (int h = 0; h < 2; h++)
#pragma unroll
                for (int s = 0; s < NS; s++) {
                    const pa_v8h ko = pa_key<HD, KVT>(kv, h, s);
                    if constexpr (KVT == F16) {
                        sc[h] = pa_mma(ko, q0[t][s], sc[h]);
                        if constexpr (!ST) sc[h] = pa_mma(ko, q1[t][s], sc[h]);
                    } else {
                        pa_v4f d = pa_mma(ko, q0[t][s], pa_v4f{0.0f, 0.0f, 0.0f, 0.0f});
                        if constexpr (!ST) d = pa_mma(ko, q1[t][s], d);
#pragma unroll
                        for (int i = 0; i < 4; i++) sc[h][i] = __builtin_fmaf(pa_scale(kv.dk[4 * h + i], s), d[i], sc[h][i]);
                    }
                }
            float mt = -__builtin_inff();
#pragma unroll
            for (int j = 0; j < 8; j++) {
                float x = sc[j >> 2][j & 3];
                if constexpr (ST) x += xor8(x);
                x *= qs[t];
                if (a.cap > 0.0f) x = capl * pa_tanh(x);
                if (edge) {
                    const int pos = base + 16 * (j >> 2) + 4 * g + (j & 3);
                    x = pos >= rlo[t] && pos <= rhi[t] ? x : -__builtin_inff();
                }
                w[t][j] = x;
                mt = fmaxf(mt, KVT == F16 ? x : x + ex[j]);
            }
            mt = fmaxf(mt, partner<16>(mt));
            mt = fmaxf(mt, partner<32>(mt));
            const float mn = fmaxf(m[t], mt);
            if (__any(mn > m[t])) {
                const float cr = mn > m[t] ? __builtin_amdgcn_exp2f(m[t] - mn) : 1.0f;
                l[t] *= cr;
#pragma unroll
                for (int e = 0; e < NM; e++) o[t][e] *= cr;
                m[t] = mn;
            }
            const float mr = m[t] == -__builtin_inff() ? 0.0f : m[t] - PA_SHIFT;
#pragma unroll
            for (int j = 0; j < 8; j++) {
                w[t][j] = __builtin_amdgcn_exp2f(w[t][j] - mr);
                l[t] += w[t][j];
            }
        }
        // positions that no row of the tile attends may hold anything: zeros
        // for them; non-finite values that some rows attend and some do not
        // are taken out and added to those that do (rare, one by one)
        uint64_t odd = 0;
        if constexpr (KVT == F16) {
            if (edge) {
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    const int pos = base + 16 * (j >> 2) + 4 * g + (j & 3);
                    const bool dead = pos < mn_lo || pos > mx_hi || pos >= seglen;
                    uint32_t nf = 0;
#pragma unroll
                    for (int d = 0; d < PaTile<HD, KVT>::VW; d++) {
                        uint32_t x = dead ? 0u : kv.v[j][d];
                        const uint32_t a0 = (x & 0x7c00u) == 0x7c00u, a1 = (x & 0x7c000000u) == 0x7c000000u;
                        nf |= a0 | a1;
                        x = a0 ? x & 0xffff0000u : x;
                        kv.v[j][d] = a1 ? x & 0xffffu : x;
                    }
                    odd |= __ballot(nf);
                }
            }
        }
#pragma unroll
        for (int t = 0; t < NT; t++) {
            if constexpr (KVT == F16) {
                uint32_t ph[4], pl2[4];
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    const float x = w[t][2 * k], y = w[t][2 * k + 1];
                    ph[k] = pa_pk(x, y);
                    pl2[k] = pa_pk(x - pa_lo(ph[k]), y - pa_hi(ph[k]));
                    if constexpr (ST) ph[k] = c < 8 ? ph[k] : pl2[k];
                }
                const pa_v8h b0 = pa_op(ph[0], ph[1], ph[2], ph[3]), b1 = pa_op(pl2[0], pl2[1], pl2[2], pl2[3]);
#pragma unroll
                for (int e = 0; e < NM; e++) {
                    const pa_v8h va = pa_value<HD, KVT>(kv, e);
                    o[t][e] = pa_mma(va, b0, o[t][e]);
                    if constexpr (!ST) o[t][e] = pa_mma(va, b1, o[t][e]);
                }
            } else {
#pragma unroll
                for (int s = 0; s < NS; s++) {               // blocks of 32 elements: value tiles 2 s, 2 s + 1
                    uint32_t ph[4], pl2[4];
#pragma unroll
                    for (int k = 0; k < 4; k++) {
                        const float w0 = w[t][2 * k], w1 = w[t][2 * k + 1];
                        const float x = w0 == 0.0f ? 0.0f : w0 * pa_scale(kv.dv[2 * k], s), y = w1 == 0.0f ? 0.0f : w1 * pa_scale(kv.dv[2 * k + 1], s);
                        ph[k] = pa_pk(x, y);
                        pl2[k] = pa_pk(x - pa_lo(ph[k]), y - pa_hi(ph[k]));
                        if constexpr (ST) ph[k] = c < 8 ? ph[k] : pl2[k];
                    }
                    const pa_v8h b0 = pa_op(ph[0], ph[1], ph[2], ph[3]), b1 = pa_op(pl2[0], pl2[1], pl2[2], pl2[3]);
#pragma unroll
                    for (int e = 2 * s; e < 2 * s + 2; e++) {
                        const pa_v8h va = pa_value<HD, KVT>(kv, e);
                        o[t][e] = pa_mma(va, b0, o[t][e]);
                        if constexpr (!ST) o[t][e] = pa_mma(va, b1, o[t][e]);
                    }
                }
            }
        }
        if constexpr (KVT == F16) {
            if (odd) {
                for (int x = 0; x < 32; x++) {
                    const int pos = base + x;
                    if (pos < mn_lo || pos > mx_hi || pos >= seglen) continue;
                    const uint16_t *row = (const uint16_t *)(p.v + u[x >> 4].row) + (x & 15) * HD;
#pragma unroll
                    for (int t = 0; t < NT; t++) {
                        float wx = 0.0f;
#pragma unroll
                        for (int j = 0; j < 8; j++) {
                            const float v = __shfl(w[t][j], 16 * ((x & 15) >> 2) + c, 64);
                            if (j == 4 * (x >> 4) + (x & 3)) wx = v;
                        }
                        const bool sees = pos >= rlo[t] && pos <= rhi[t] && !(ST && c >= 8);
#pragma unroll
                        for (int e = 0; e < NM; e++)
#pragma unroll
                            for (int i = 0; i < 4; i++) {
                                const uint16_t hv = row[pa_elem<HD, KVT>(e, 4 * g + i)];
                                if (sees && (hv & 0x7c00) == 0x7c00) o[t][e][i] += wx * h2f(hv);
                            }
                    }
                }
            }
        }
    }
    if (__any(bad)) {
        if (lane == 0 && !sq.bad) paged_flag(p, PAGED_BAD_PAGE);
#pragma unroll
        for (int t = 0; t < NT; t++) l[t] = __builtin_nanf("");
    }

    // the waves' results joined in order, 8 rows at a time
#pragma unroll
    for (int t = 0; t < NT; t++) {
        l[t] += partner<16>(l[t]);
        l[t] += partner<32>(l[t]);
        if (lane < (ST ? 8 : 16)) wml[wave][16 * t + lane] = make_float2(m[t], l[t]);
        if constexpr (ST) {
#pragma unroll
            for (int e = 0; e < NM; e++)
#pragma unroll
                for (int i = 0; i < 4; i++) o[t][e][i] += xor8(o[t][e][i]);
        }
    }
    constexpr float VS = KVT == Q8_0 ? 512.0f : 1.0f;
#pragma unroll
    for (int k = 0; k < R / 8; k++) {
        if (k) __syncthreads();
        if ((c >> 3) == (k & 1)) {
#pragma unroll
            for (int e = 0; e < NM; e++)
#pragma unroll
                for (int i = 0; i < 4; i++) buf[wave][c & 7][pa_elem<HD, KVT>(e, 4 * g + i)] = o[ST ? 0 : k >> 1][e][i];
        }
        __syncthreads();
        for (int x = threadIdx.x; x < 8 * (HD / 4); x += 64 * PA_WAVES) {
            const int r8 = x / (HD / 4), e4 = x % (HD / 4) * 4, r = tile * R + 8 * k + r8;
            if (r >= sq.nq * G) continue;
            float mm = -__builtin_inff();
#pragma unroll
            for (int w = 0; w < PA_WAVES; w++) mm = fmaxf(mm, wml[w][8 * k + r8].x);
            float ls = 0.0f;
            pa_v4f s = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int w = 0; w < PA_WAVES; w++) {
                const float2 ml = wml[w][8 * k + r8];
                const float f = ml.x == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(ml.x - mm);
                ls += ml.y == ml.y ? f * ml.y : ml.y;        // a bad page's NaN stays
                const pa_v4f v = *(const pa_v4f *)&buf[w][r8][e4];
                s += v * f;
            }
            s *= VS;
            const int i = r / G, tok = sq.t0 + i, head = kvh * G + (r - i * G);
            if (pl.nsplit == 1) {
                const float inv = 1.0f / ls;
                s = !pre && !sq.bad && sq.len - sq.nq + i < 0 ? pa_v4f{0.0f, 0.0f, 0.0f, 0.0f} : s * inv;
                float *d = a.out + (size_t)tok * a.os + (size_t)head * HD + e4;
                d[0] = s[0]; d[1] = s[1]; d[2] = s[2]; d[3] = s[3];
            } else {
                const size_t row = (size_t)tok * a.n_head + head, at = row * pl.nsplit + split;
                *(pa_v4f *)(pl.po + at * HD + e4) = s;
                if (e4 == 0) pl.ml[at] = make_float2(mm, ls);
            }
        }
    }
}

// A tile variant of a cache type: its rows, and its launch.
enum { PA_ST = 0, PA_T1 = 1, PA_T2 = 2 };
__host__ __device__ constexpr int pa_rows(int v) { return v == PA_ST ? 8 : 16 * v; }

template <int KVT, int HD>
hipError_t pa_launch_hd(const PagedAttn &a, const PagedPlan &pl, int v, unsigned blocks, hipStream_t s) {
    const dim3 grid(blocks), wg(64 * PA_WAVES);
    if (v == PA_ST) hipLaunchKernelGGL((k_paged_attn<HD, KVT, 1, true>), grid, wg, 0, s, a, pl);
    else if (v == PA_T1) hipLaunchKernelGGL((k_paged_attn<HD, KVT, 1, false>), grid, wg, 0, s, a, pl);
    else if constexpr (HD <= 256) hipLaunchKernelGGL((k_paged_attn<HD, KVT, 2, false>), grid, wg, 0, s, a, pl);
    else return hipErrorInvalidValue;
    return hipGetLastError();
}
template <int KVT>
hipError_t pa_launch(const PagedAttn &a, const PagedPlan &pl, int v, unsigned blocks, hipStream_t s) {
    switch (a.p.hd) {
    case 64: return pa_launch_hd<KVT, 64>(a, pl, v, blocks, s);
    case 128: return pa_launch_hd<KVT, 128>(a, pl, v, blocks, s);
    case 256: return pa_launch_hd<KVT, 256>(a, pl, v, blocks, s);
    case 512: return pa_launch_hd<KVT, 512>(a, pl, v, blocks, s);
    }
    return hipErrorInvalidValue;
}
hipError_t pa_launch_f16(const PagedAttn &a, const PagedPlan &pl, int v, unsigned blocks, hipStream_t s);
hipError_t pa_launch_q8(const PagedAttn &a, const PagedPlan &pl, int v, unsigned blocks, hipStream_t s);
hipError_t pa_launch_q4(const PagedAttn &a, const PagedPlan &pl, int v, unsigned blocks, hipStream_t s);

}  // namespace g4
