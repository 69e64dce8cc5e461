// paged_few.h -- attention of a few rows over the paged KV cache (paged_attn.h):
// single tokens of many sequences, short drafts, the prefix of a small batch.
//
// Bound by the cache's bytes; over few positions by the chain of reads from the
// lengths to the pages to K, 6 us of it, and the join.  The workgroups all fit on
// the device at once, and their shares of the list of steps are equal, so ragged
// lengths leave none idle.  Reached: 32 sequences of up to 8192 positions, 8 q / 4
// kv heads of 256, f16: 101 us, 5.3 TB/s; 64 of up to 4096, 32 / 8 heads of 128, 8
// bits, capped: 72 to 75 us, 3.8 to 4.0 TB/s; 16 windows of 1024, 8 / 2 heads of 512,
// 4 bits: 19 us (joins included).
//
// A workgroup's 4 waves take 32 positions each of a step of 128, on
// v_mfma_f32_16x16x32_f16 with the rows as columns.  Up to 8 rows (ST) sit as
// high halves in columns 0..7 and low halves in 8..15: the second half costs no
// matrix instruction.  K and V go from the pages to registers, each lane's loads
// being the operand's runs of bytes (the layout of the quantized rows is made for
// it); f16 value rows are turned (8 positions x 2 elements) with v_perm_b32.  A
// step's K registers are loaded again as soon as its scores are taken, its V
// registers after the sums.  Heads of 256 and 512: two and four waves share 32
// positions, each with 128 of the elements, their scores added through LDS (whole
// heads of 256 in one wave's registers spilled: 32 sequences of up to 8192
// positions, 8 q / 4 kv heads, 188 us).
#pragma once

#include "paged_attn.h"

namespace g4 {

// Operands of 32 positions and HE elements of the head (one wave's): raw bytes.
template <int HE, int KVT>
struct PaTile {
    static constexpr int KW = KVT == Q4_0 ? HE / 32 : HE / 16;                           // dwords of a lane's key run (f16: of four)
    static constexpr int VW = KVT == F16 ? HE / 32 : KVT == Q8_0 ? HE / 64 : (HE >= 128 ? HE / 128 : 1);
    static constexpr int DW = HE / 64;                                                   // dwords of a row's scales
    uint32_t k[2][KVT == F16 ? HE / 8 : KW];   // [unit][dwords]
    uint32_t v[8][VW];                         // [position 4 t + i][dwords]
    uint32_t sc[KVT == F16 ? 1 : DW];          // of position lane % 32, K's in lanes 0..31, V's in the others
};
// The scales through LDS: one load of the wave brings all 64 rows', where a lane
// loading the 16 that it multiplies with took 17 of a step's 27 load instructions
// (64 sequences of up to 4096 positions, 8 KV heads of 128, 8 bits: 73 us, now 70).
template <int HE>
struct PaScales {
    uint32_t d[2][32][HE / 64];
    float e[32];                               // pa_exponent of V's largest
};

template <int N>
__device__ __forceinline__ void pa_read(uint32_t *d, const void *lds) {
#pragma unroll
    for (int i = 0; i < N; i += 4) {
        const pa_v4u x = ((const pa_v4u *)lds)[i / 4];
        d[i] = x[0]; d[i + 1] = x[1]; d[i + 2] = x[2]; d[i + 3] = x[3];
    }
}

template <int HD, int HE, int KVT>
__device__ __forceinline__ void pa_load_k(PaTile<HE, KVT> &t, const PagedPool &p, const PaUnit u[2], int c, int g, int ew) {
    using T = PaTile<HE, KVT>;
#pragma unroll
    for (int h = 0; h < 2; h++) {
        const uint8_t *row = p.k + u[h].row + c * paged_row_bytes(KVT, HD);
        if constexpr (KVT == F16) {
#pragma unroll
            for (int s = 0; s < HE / 32; s++) pa_load<4>(t.k[h] + 4 * s, row + 2 * HE * ew + 64 * s + 16 * g);
        } else {
            pa_load<T::KW>(t.k[h], row + 4 * T::KW * ((HD / HE) * g + ew));
        }
    }
}
template <int HD, int HE, int KVT>
__device__ __forceinline__ void pa_load_scales(PaTile<HE, KVT> &t, const PagedPool &p, const PaUnit u[2], int lane, int ew) {
    const uint8_t *pool = lane < 32 ? p.k : p.v;
    pa_load<PaTile<HE, KVT>::DW>(t.sc, pool + ((lane & 16) ? u[1].sc : u[0].sc) + ((lane & 15) * (HD / 16) + (HE / 16) * ew));
}
template <int HD, int HE, int KVT>
__device__ __forceinline__ void pa_load_v(PaTile<HE, KVT> &t, const PagedPool &p, const PaUnit u[2], int c, int g, int ew) {
    using T = PaTile<HE, KVT>;
#pragma unroll
    for (int j = 0; j < 8; j++) {
        const int i = 4 * g + (j & 3);
        const uint8_t *row = p.v + u[j >> 2].row + i * paged_row_bytes(KVT, HD);
        if constexpr (KVT == F16 && HE == 64) {
            pa_load<2>(t.v[j], row + 8 * c);
        } else if constexpr (KVT == F16) {
#pragma unroll
            for (int n = 0; n < HE / 128; n++) pa_load<4>(t.v[j] + 4 * n, row + 2 * HE * ew + 256 * n + 16 * c);
        } else if constexpr (KVT == Q4_0 && HE == 64) {
            t.v[j][0] = *(const uint16_t *)(row + 2 * c);
        } else {
            pa_load<T::VW>(t.v[j], row + 4 * T::VW * ((HD / HE) * c + ew));
        }
    }
}

// key operand of unit h, 32 elements s
template <int HE, int KVT>
__device__ __forceinline__ pa_v8h pa_key(const PaTile<HE, KVT> &t, int h, int s) {
    if constexpr (KVT == F16) return pa_op(t.k[h][4 * s], t.k[h][4 * s + 1], t.k[h][4 * s + 2], t.k[h][4 * s + 3]);
    else if constexpr (KVT == Q8_0) {
        const uint32_t a = t.k[h][2 * s], b = t.k[h][2 * s + 1];
        return pa_op(pa_q8(__builtin_amdgcn_perm(0, a, 0x0c010c00u)), pa_q8(__builtin_amdgcn_perm(0, a, 0x0c030c02u)),
                     pa_q8(__builtin_amdgcn_perm(0, b, 0x0c010c00u)), pa_q8(__builtin_amdgcn_perm(0, b, 0x0c030c02u)));
    } else {
        const uint32_t w = t.k[h][s];
        return pa_op(pa_q4<0>(w), pa_q4<1>(w), pa_q4<2>(w), pa_q4<3>(w));
    }
}
// value operand of the 16 elements m (pa_elem) over the 32 positions
template <int HE, int KVT>
__device__ __forceinline__ pa_v8h pa_value(const PaTile<HE, KVT> &t, int m) {
    uint32_t w[4];
#pragma unroll
    for (int k = 0; k < 4; k++) {
        if constexpr (KVT == F16) {
            const int d = HE == 64 ? m >> 1 : 4 * (m >> 3) + ((m & 7) >> 1);
            w[k] = __builtin_amdgcn_perm(t.v[2 * k + 1][d], t.v[2 * k][d], (m & 1) ? 0x07060302u : 0x05040100u);
        } else if constexpr (KVT == Q8_0) {
            const uint32_t b = m & 3;
            w[k] = pa_q8(__builtin_amdgcn_perm(t.v[2 * k + 1][m >> 2], t.v[2 * k][m >> 2], 0x0c000c00u | b | ((4 + b) << 16)));
        } else {
            const int d = m >> 3;
            w[k] = pa_q4(__builtin_amdgcn_perm(t.v[2 * k + 1][d], t.v[2 * k][d], (m & 4) ? 0x07060302u : 0x05040100u), m & 3);
        }
    }
    return pa_op(w[0], w[1], w[2], w[3]);
}
// element (of the wave's HE) that value tile m holds in its operand row x (0..15)
template <int HE, int KVT>
__device__ __forceinline__ int pa_elem(int m, int x) {
    return KVT != F16 ? 16 * m + x : HE == 64 ? 4 * x + m : 128 * (m >> 3) + 8 * x + (m & 7);
}

template <int HD, int KVT, bool ST, bool TREE>
__global__ __launch_bounds__(256, pa_few_per_cu(KVT, HD, ST)) void k_paged_few(PagedCall call) {
    constexpr int R = ST ? 8 : 16, HE = HD > 128 ? 128 : HD, ES = HD / HE, PW = 4 / ES, NS = HE / 32, NM = HE / 16;
    constexpr int QP = HD + 8;                               // padded query row
    constexpr size_t QB = 2 * R * QP * 2, OB = (size_t)PW * 8 * (HD + 4) * 4;
    __shared__ __align__(16) uint8_t lds[QB > OB ? QB : OB]; // the queries' halves [2][R][QP]; then sums [PW][8][HD + 4]
    __shared__ float qsc[R];
    __shared__ float2 wml[4][R];                             // two waves of one tile may differ in m (by their elements' scales)
    __shared__ __align__(16) float xs[ES > 1 ? 2 : 1][ES > 1 ? 4 : 1][ES > 1 ? 64 : 1][8];   // partial scores of the waves of one tile
    __shared__ __align__(16) PaScales<HE> scl[KVT == F16 ? 1 : 4];           // of a wave
    __shared__ int nothing[TREE ? R : 1];                    // whether a tree's row attends nothing
    _Float16 *const qh = (_Float16 *)lds;
    float *const buf = (float *)lds;

    int mine, n_seq;
    const int total = pa_total<false, TREE>(call.a, call.pl, mine, n_seq), share = pa_share(call.pl.few, total);
    const int first = blockIdx.x * share, stop = min(first + share, total);
    if (blockIdx.x == 0 && call.pl.many.rows == 0) pa_rest(call.a, call.pl, n_seq);
    PaFind from;
    for (int u = first; u < stop;) {
        const PagedCall call = pa_fresh<TREE>();
        const PagedAttn &a = call.a;
        const PagedPlan &pl = call.pl;
        const PagedPool &p = a.p;
        const PagedBatch &b = a.b;
        const int tid = pa_thread(), lane = tid & 63, wave = pa_uniform(tid >> 6), c = lane & 15, g = lane >> 4, ew = wave % ES, pw = wave / ES;
        const int G = a.grp, rc = ST ? c & 7 : c;
        const PaPiece x = pa_piece<false, TREE>(a, pl, mine, n_seq, from, blockIdx.x, u, first, stop);
        u += x.took;
        if (x.n == 0) break;                                 // the share ends in a tile's lead
        const PagedSeq &sq = x.sq;
        const int kvh = x.kvh, hi0 = x.hi0, lo0 = x.lo0, lo1 = x.lo1, start = x.start, end = x.end, rows = sq.nq * G;
        bool bad = sq.bad;
        if (bad && tid == 0) paged_flag(p, PAGED_BAD_BATCH);
        const bool tree = TREE && !x.pre;
        const bool mixed = tree || hi0 != x.hi1 || lo0 != lo1;           // whether the rows differ in what they attend
        const int full = tree ? hi0 - 1 : hi0;               // the last position that all rows attend, windows apart
        const int last = (x.seglen - 1) >> 4, iters = end > start ? (end - start + 32 * PW - 1) / (32 * PW) : 0;

        // queries: loaded first, ahead of the stream
        constexpr int LPR = 256 / R, QN = HD / (4 * LPR) > 0 ? HD / (4 * LPR) : 1;
        const int qr = tid / LPR, ql = tid % LPR;
        pa_v4f qv[QN];
        {
            const int i = (int)(qr * pl.grp_inv >> 16), h = qr - i * G;
            const float *src = a.q + (size_t)(sq.t0 + i) * a.qs + (size_t)(kvh * G + h) * HD;
            const bool al = ((uintptr_t)src & 15) == 0;
#pragma unroll
            for (int k = 0; k < QN; k++) {
                const int e = 4 * (ql + LPR * k);
                qv[k] = pa_v4f{0.0f, 0.0f, 0.0f, 0.0f};
                if (qr < rows && e < HD) {
                    if (al) qv[k] = *(const pa_v4f *)(src + e);
                    else qv[k] = pa_v4f{src[e], src[e + 1], src[e + 2], src[e + 3]};
                }
            }
        }
        // the lane's row: positions [rlo, rhi]
        int rlo = lo0, rhi = hi0;
        uint32_t bits = 0;                                   // a tree's row: its new tokens (16 at most), from position hi0 on
        if (rc < rows) {
            const int i = (int)(rc * pl.grp_inv >> 16);
            if (tree) {
                rhi = hi0 + i < 0 ? -1 : hi0 - 1;
                if (hi0 + i >= 0) bits = a.mask[(size_t)(sq.t0 + i) * a.words];
                rlo = a.window ? max(0, hi0 + paged_depth(a.depth[sq.t0 + i], sq.nq) + 1 - a.window) : 0;
            } else if (!x.pre) {
                rhi = hi0 + i;
                rlo = a.window ? max(0, rhi + 1 - a.window) : 0;
            } else if (a.window) {
                rlo = max(0, pa_token_pos(p, b, n_seq, sq.t0 + i, TREE ? a.depth : nullptr) + 1 - a.window);
            }
        }
        auto row_bits = [&](int pos) {                       // from position pos on
            const int off = pos - hi0;
            return off <= -32 || off >= 32 ? 0u : off < 0 ? bits << -off : bits >> off;
        };
        auto row_hits = [&](uint64_t out, int first, int stride) {
            if constexpr (TREE) return pa_tree_hits(out, first, stride, x.seglen, rlo, rhi, row_bits);
            else return pa_hits(out, first, stride, last, rlo, rhi);
        };

        PaTile<HE, KVT> kv;
        PaUnit un[2], nx[2];
        PaUnits us, more_us;                                 // of 32 steps, and of the next 32
        int base = start + 32 * pw;
        if (iters) {
            us = pa_units(p, x.table, base >> 4, 2 * PW, last, kvh);
            bad |= row_hits(pa_check(p, us), base >> 4, 2 * PW);
            nx[0] = pa_unit<HD, KVT>(p, us, 0);
            nx[1] = pa_unit<HD, KVT>(p, us, 1);
            if constexpr (KVT != F16) pa_load_scales<HD, HE, KVT>(kv, p, nx, lane, ew);
            pa_load_k<HD, HE, KVT>(kv, p, nx, c, g, ew);
            pa_load_v<HD, HE, KVT>(kv, p, nx, c, g, ew);
        }
        lds_barrier();                                       // the previous piece's sums are read
        if constexpr (TREE) {
            if (tid < R) {
                const int tok = sq.t0 + (int)(tid * pl.grp_inv >> 16);
                nothing[tid] = tid < rows && !x.pre && !sq.bad && pa_tree_nothing(a, sq, tok, a.mask + (size_t)tok * a.words);
            }
        }
        {
            float am = 0.0f;
#pragma unroll
            for (int k = 0; k < QN; k++)
#pragma unroll
                for (int i = 0; i < 4; i++) am = fmaxf(am, fabsf(qv[k][i]));
            am = group_max<LPR>(am);
            const int sh = pa_shift(am);
            if (ql == 0) qsc[qr] = pa_score_scale<KVT>(a, sh);
#pragma unroll
            for (int k = 0; k < QN; k++) {
                const int e = 4 * (ql + LPR * k);
                uint2 hi, lo;
                pa_split(__builtin_ldexpf(qv[k][0], sh), __builtin_ldexpf(qv[k][1], sh), hi.x, lo.x);
                pa_split(__builtin_ldexpf(qv[k][2], sh), __builtin_ldexpf(qv[k][3], sh), hi.y, lo.y);
                if (e < HD) {
                    *(uint2 *)(qh + qr * QP + e) = hi;
                    *(uint2 *)(qh + (R + qr) * QP + e) = lo;
                }
            }
        }
        lds_barrier();
        const _Float16 *const q0 = qh + ((ST && c >= 8 ? R : 0) + rc) * QP + HE * ew + 8 * g, *const q1 = qh + (R + rc) * QP + HE * ew + 8 * g;
        pa_v8h qa[NS], qb[ST ? 1 : NS];
#pragma unroll
        for (int s = 0; s < NS; s++) {
            qa[s] = *(const pa_v8h *)(q0 + 32 * s);
            if constexpr (!ST) qb[s] = *(const pa_v8h *)(q1 + 32 * s);
        }
        const float qs = qsc[rc], capl = a.cap * 1.4426950408889634f;

        const float part = c < 8 ? 0.0f : -1.0f;             // ST: the lane's half of a weight
        pa_v4f o[NM];
        float m = -__builtin_inff(), l = 0.0f;
#pragma unroll
        for (int e = 0; e < NM; e++) o[e] = pa_v4f{0.0f, 0.0f, 0.0f, 0.0f};

        for (int it = 0; it < iters; it++, base += 32 * PW) {
            const bool more = it + 1 < iters;
            un[0] = nx[0];
            un[1] = nx[1];
            if ((it & 31) == 31 && it + 1 < iters) {
                us = more_us;
                bad |= row_hits(pa_check(p, us), (base >> 4) + 2 * PW, 2 * PW);
            }
            if (more) {
                nx[0] = pa_unit<HD, KVT>(p, us, 2 * (it + 1) & 63);
                nx[1] = pa_unit<HD, KVT>(p, us, (2 * (it + 1) & 63) + 1);
            }
            if ((it & 31) == 0 && it + 32 < iters) more_us = pa_units(p, x.table, (base >> 4) + 64 * PW, 2 * PW, last, kvh);
            const bool edge = base + 31 > full || base < lo1 || base + 32 > end;
            const uint32_t att = TREE ? pa_tree_seen(base, rlo, rhi, row_bits(base), end) : 0u;
            auto seen = [&](int pos) { return (att >> (pos - base) & 1) != 0; };         // by a tree's row
            constexpr int DW = PaTile<HE, KVT>::DW;
            uint32_t dk[8][DW], dv[8][DW];                   // of the lane's 8 positions
            PaScales<HE> &sl = scl[KVT == F16 ? 0 : wave];
            if constexpr (KVT != F16) {
                // a wave's LDS accesses complete in order
                asm volatile("" ::: "memory");
#pragma unroll
                for (int d = 0; d < DW; d++) sl.d[lane >> 5][lane & 31][d] = kv.sc[d];
                uint32_t dm = kv.sc[0] & 0x7fff7fffu;
#pragma unroll
                for (int d = 1; d < DW; d++) dm = pa_pkmax(dm, kv.sc[d] & 0x7fff7fffu);
                if (lane >= 32) sl.e[lane & 31] = pa_exponent(max(dm << 16, dm), 1);
                asm volatile("" ::: "memory");
#pragma unroll
                for (int h = 0; h < 2; h++) pa_read<4 * DW>(dk[4 * h], sl.d[0][16 * h + 4 * g]);
            }
            // scores at positions base + 16 h + 4 g + i
            pa_v4f sc[2] = {{0.0f, 0.0f, 0.0f, 0.0f}, {0.0f, 0.0f, 0.0f, 0.0f}};
#pragma unroll
            for (int s = 0; s < NS; s++) {
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    const pa_v8h ko = pa_key<HE, KVT>(kv, h, s);
                    if constexpr (KVT == F16) {
                        sc[h] = pa_mma(ko, qa[s], sc[h]);
                        if constexpr (!ST) sc[h] = pa_mma(ko, qb[s], sc[h]);
                    } else {
                        pa_v4f d = pa_mma(ko, qa[s], pa_v4f{0.0f, 0.0f, 0.0f, 0.0f});
                        if constexpr (!ST) d = pa_mma(ko, qb[s], d);
#pragma unroll
                        for (int i = 0; i < 4; i++) sc[h][i] = __builtin_fmaf(pa_scale(dk[4 * h + i], s), d[i], sc[h][i]);
                    }
                }
            }
            __builtin_amdgcn_sched_barrier(0);               // the next keys go where these were
            if (more) {
                if constexpr (KVT != F16) pa_load_scales<HD, HE, KVT>(kv, p, nx, lane, ew);
                pa_load_k<HD, HE, KVT>(kv, p, nx, c, g, ew);
            }
            __builtin_amdgcn_sched_barrier(0);
            if constexpr (ES > 1) {
                *(pa_v4f *)xs[it & 1][wave][lane] = sc[0];
                *(pa_v4f *)(xs[it & 1][wave][lane] + 4) = sc[1];
                lds_barrier();
                const int w0 = wave & ~(ES - 1);
                sc[0] = *(const pa_v4f *)xs[it & 1][w0][lane];
                sc[1] = *(const pa_v4f *)(xs[it & 1][w0][lane] + 4);
#pragma unroll
                for (int k = 1; k < ES; k++) {
                    sc[0] += *(const pa_v4f *)xs[it & 1][w0 + k][lane];
                    sc[1] += *(const pa_v4f *)(xs[it & 1][w0 + k][lane] + 4);
                }
            }
            float w[8], mt = -__builtin_inff();
#pragma unroll
            for (int j = 0; j < 8; j++) {
                float y = sc[j >> 2][j & 3];
                if constexpr (ST) y += xor8(y);
                w[j] = y * qs;
            }
            if (a.cap > 0.0f) {
                if constexpr (ST) {                          // columns c and c ^ 8 hold the same scores: half of them each
                    float y[4];
#pragma unroll
                    for (int j = 0; j < 4; j++) y[j] = c < 8 ? w[j] : w[4 + j];
                    pa_tanh(y);
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        const float z = y[j] * capl, other = xor8(z);
                        w[j] = c < 8 ? z : other;
                        w[4 + j] = c < 8 ? other : z;
                    }
                } else {
                    pa_tanh(w);
#pragma unroll
                    for (int j = 0; j < 8; j++) w[j] *= capl;
                }
            }
            if (edge) {
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    const int pos = base + 16 * (j >> 2) + 4 * g + (j & 3);
                    w[j] = (TREE ? seen(pos) : pos >= rlo && pos <= rhi && pos < end) ? w[j] : -__builtin_inff();
                }
            }
            if constexpr (KVT == F16) {
#pragma unroll
                for (int j = 0; j < 8; j++) mt = fmaxf(mt, w[j]);
            } else {
                // + the exponent of the position's largest value scale
                const pa_v4f e[2] = {*(const pa_v4f *)&sl.e[4 * g], *(const pa_v4f *)&sl.e[16 + 4 * g]};
#pragma unroll
                for (int j = 0; j < 8; j++) mt = fmaxf(mt, w[j] + e[j >> 2][j & 3]);
#pragma unroll
                for (int h = 0; h < 2; h++) pa_read<4 * DW>(dv[4 * h], sl.d[1][16 * h + 4 * g]);
            }
            mt = fmaxf(mt, partner<16>(mt));
            mt = fmaxf(mt, partner<32>(mt));
            if (__any(mt > m + PA_LAG)) {
                const float mn = fmaxf(m, mt), cr = mn > m ? __builtin_amdgcn_exp2f(m - mn) : 1.0f;
                l *= cr;
#pragma unroll
                for (int e = 0; e < NM; e++) o[e] *= cr;
                m = mn;
            }
            const float mr = m == -__builtin_inff() ? 0.0f : m - pa_shift_of<KVT>();
#pragma unroll
            for (int j = 0; j < 8; j++) {
                w[j] = __builtin_amdgcn_exp2f(w[j] - mr);
                l += w[j];
            }
            // positions that no row of the tile attends may hold anything: zeros
            // for them; non-finite values that some rows attend and some do not
            // are taken out and added to those that do (rare, one by one)
            bool odd = false;
            if constexpr (KVT == F16) {
                if (edge) {
#pragma unroll
                    for (int j = 0; j < 8; j++) {
                        const int pos = base + 16 * (j >> 2) + 4 * g + (j & 3);
                        const uint32_t live = pos < lo0 || pos >= end ? 0u : ~0u;
#pragma unroll
                        for (int d = 0; d < PaTile<HE, KVT>::VW; d++) kv.v[j][d] &= live;
                    }
                    if (mixed) {
                        uint32_t nf = 0;                     // bit 15 or 31 where an exponent is all ones
#pragma unroll
                        for (int j = 0; j < 8; j++)
#pragma unroll
                            for (int d = 0; d < PaTile<HE, KVT>::VW; d++) nf |= (kv.v[j][d] & 0x7c007c00u) + 0x04000400u;
                        odd = __any(nf & 0x80008000u);
                        if (odd) {
#pragma unroll
                            for (int j = 0; j < 8; j++)
#pragma unroll
                                for (int d = 0; d < PaTile<HE, KVT>::VW; d++) kv.v[j][d] = pa_finite(kv.v[j][d]);
                        }
                    }
                }
                uint32_t ph[4], pq[4];
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    if constexpr (ST) ph[k] = pa_half(w[2 * k], w[2 * k + 1], part);
                    else pa_split(w[2 * k], w[2 * k + 1], ph[k], pq[k]);
                }
                const pa_v8h b0 = pa_op(ph[0], ph[1], ph[2], ph[3]), b1 = pa_op(pq[0], pq[1], pq[2], pq[3]);
#pragma unroll
                for (int e = 0; e < NM; e++) {
                    const pa_v8h va = pa_value<HE, KVT>(kv, e);
                    o[e] = pa_mma(va, b0, o[e]);
                    if constexpr (!ST) o[e] = pa_mma(va, b1, o[e]);
                }
            } else {
                // a scale of a position that the row does not attend may be anything
                if (edge) {
#pragma unroll
                    for (int j = 0; j < 8; j++) {
                        const int pos = base + 16 * (j >> 2) + 4 * g + (j & 3);
                        const uint32_t live = (TREE ? seen(pos) : pos >= rlo && pos <= rhi && pos < end) ? ~0u : 0u;
#pragma unroll
                        for (int d = 0; d < DW; d++) dv[j][d] &= live;
                    }
                }
#pragma unroll
                for (int s = 0; s < NS; s++) {               // blocks of 32 elements: value tiles 2 s, 2 s + 1
                    uint32_t ph[4], pq[4];
#pragma unroll
                    for (int k = 0; k < 4; k++) {
                        const float y = __builtin_fmaf(pa_scale(dv[2 * k], s), w[2 * k], 0.0f), z = __builtin_fmaf(pa_scale(dv[2 * k + 1], s), w[2 * k + 1], 0.0f);
                        if constexpr (ST) ph[k] = pa_half(y, z, part);
                        else pa_split(y, z, ph[k], pq[k]);
                    }
                    const pa_v8h b0 = pa_op(ph[0], ph[1], ph[2], ph[3]), b1 = pa_op(pq[0], pq[1], pq[2], pq[3]);
#pragma unroll
                    for (int e = 2 * s; e < 2 * s + 2; e++) {
                        const pa_v8h va = pa_value<HE, KVT>(kv, e);
                        o[e] = pa_mma(va, b0, o[e]);
                        if constexpr (!ST) o[e] = pa_mma(va, b1, o[e]);
                    }
                }
            }
            __builtin_amdgcn_sched_barrier(0);
            if (more) pa_load_v<HD, HE, KVT>(kv, p, nx, c, g, ew);
            __builtin_amdgcn_sched_barrier(0);
            if constexpr (KVT == F16) {
                if (odd) {
                    for (int k = 0; k < 32; k++) {
                        const int pos = base + k;
                        if (pos < lo0 || pos >= end) continue;
                        const uint16_t *row = (const uint16_t *)(p.v + (k < 16 ? un[0].row : un[1].row)) + (k & 15) * HD + HE * ew;
                        float wx = 0.0f;
#pragma unroll
                        for (int j = 0; j < 8; j++) {
                            const float v = __shfl(w[j], 16 * ((k & 15) >> 2) + c, 64);
                            if (j == 4 * (k >> 4) + (k & 3)) wx = v;
                        }
                        const bool sees = (TREE ? seen(pos) : pos >= rlo && pos <= rhi) && !(ST && c >= 8);
#pragma unroll
                        for (int e = 0; e < NM; e++)
#pragma unroll
                            for (int i = 0; i < 4; i++) {
                                const uint16_t hv = row[pa_elem<HE, KVT>(e, 4 * g + i)];
                                if (sees && (hv & 0x7c00) == 0x7c00) o[e][i] += wx * h2f(hv);
                                __builtin_amdgcn_sched_barrier(0);
                            }
                    }
                }
            }
        }
        bad &= rc < rows;
        if (__any(bad)) {
            if (lane == 0 && !sq.bad) paged_flag(p, PAGED_BAD_PAGE);
            if (bad) l = __builtin_nanf("");
        }

        // the position waves' results joined in order, 8 rows at a time
        l += partner<16>(l);
        l += partner<32>(l);
        if (lane < R) wml[wave][lane] = make_float2(m, l);
        if constexpr (ST) {
#pragma unroll
            for (int e = 0; e < NM; e++)
#pragma unroll
                for (int i = 0; i < 4; i++) o[e][i] += xor8(o[e][i]);
        }
        constexpr float VS = KVT == Q8_0 ? 512.0f : 1.0f;
#pragma unroll
        for (int k = 0; k < R / 8; k++) {
            lds_barrier();                                   // the queries (the previous rows' sums) are read
            if ((c >> 3) == k) {
#pragma unroll
                for (int e = 0; e < NM; e++)
#pragma unroll
                    for (int i = 0; i < 4; i++) buf[(pw * 8 + (c & 7)) * (HD + 4) + HE * ew + pa_elem<HE, KVT>(e, 4 * g + i)] = o[e][i];
            }
            lds_barrier();
            for (int y = tid; y < 8 * (HD / 4); y += 256) {
                const int r8 = y / (HD / 4), e4 = y % (HD / 4) * 4, r = 8 * k + r8;
                if (r >= rows) continue;
                float mm = -__builtin_inff();
#pragma unroll
                for (int w = 0; w < 4; w++) mm = fmaxf(mm, wml[w][r].x);
                float ls = 0.0f;
                pa_v4f s = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int w = 0; w < PW; w++) {
                    const float2 ml = wml[w * ES][r];
                    const float f = ml.x == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(ml.x - mm);
                    ls += ml.y == ml.y ? f * ml.y : ml.y;    // a bad page's NaN stays
                    const float mo = wml[w * ES + (ES > 1 ? e4 / HE : 0)][r].x;
                    s += *(const pa_v4f *)&buf[(w * 8 + r8) * (HD + 4) + e4] * (mo == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(mo - mm));
                }
                s *= VS;
                const int i = (int)(r * pl.grp_inv >> 16), tok = sq.t0 + i, head = kvh * G + (r - i * G);
                const bool none = TREE ? nothing[r] : !sq.bad && hi0 + i < 0;
                const PaSink to = pa_sink<false>(a, pl, x, share, r, tok, head, none, e4 == 0);
                if (to.out) {
                    s = none ? pa_v4f{0.0f, 0.0f, 0.0f, 0.0f} : s * (1.0f / ls);
                    pa_store4(to.o + e4, s);
                } else {
                    *(pa_v4f *)(to.o + e4) = s;
                    if (e4 == 0) *to.ml = make_float2(mm, ls);
                }
            }
        }
    }
}

template <int KVT, int HD, bool TREE>
hipError_t pa_few_hd(const PagedAttn &a, const PagedPlan &pl, hipStream_t s) {
    const dim3 grid(pl.few.wgs), wg(256);
    if (pl.few.rows <= 8) hipLaunchKernelGGL((k_paged_few<HD, KVT, true, TREE>), grid, wg, 0, s, PagedCall{a, pl});
    else hipLaunchKernelGGL((k_paged_few<HD, KVT, false, TREE>), grid, wg, 0, s, PagedCall{a, pl});
    return hipGetLastError();
}
template <int KVT, bool TREE = false>
hipError_t pa_few(const PagedAttn &a, const PagedPlan &pl, hipStream_t s) {
    switch (a.p.hd) {
    case 64: return pa_few_hd<KVT, 64, TREE>(a, pl, s);
    case 128: return pa_few_hd<KVT, 128, TREE>(a, pl, s);
    case 256: return pa_few_hd<KVT, 256, TREE>(a, pl, s);
    case 512: return pa_few_hd<KVT, 512, TREE>(a, pl, s);
    }
    return hipErrorInvalidValue;
}

}  // namespace g4
