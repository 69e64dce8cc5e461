// paged_many.h -- attention of many rows over the paged KV cache (paged_attn.h):
// prompt chunks, and the prefix of a large batch.
//
// Bound by the matrix cores (two instructions per operand pair: a query's and a
// weight's two halves) and, between them, by the softmax on the VALU.  A
// workgroup takes up to 128 rows of one KV head, 32 of a wave, against one chunk
// of positions, 32 at a time on v_mfma_f32_32x32x16_f16.  All its threads bring
// the next 32 positions' K and V from the pages to registers while the present
// ones are computed, then to LDS as operands: K rows as halves (the block
// formats' integers are halves too), V rows turned to 8 positions of one
// element, so each is converted once for all rows.  Heads of 512: two waves
// share 32 rows, each with half of the elements, their scores added through LDS.
#pragma once

#include "paged_attn.h"

namespace g4 {

__device__ __forceinline__ pa_v16f pa_mma32(pa_v8h a, pa_v8h b, pa_v16f c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }

// Operand order of 16 positions (step ks of 32): lane group g (lane / 32), j of
// its 8 halves -- the order in which a lane holds scores.
__device__ __forceinline__ int pm_pos(int ks, int g, int j) { return 16 * ks + 8 * (j >> 2) + 4 * g + (j & 3); }

// LDS of 32 positions: K [32][HD + 8] halves; V [ks][HD / 32][64 lanes][8]; the
// scales [HD / 32][32] of K and of V (quantized)
template <int HD, int KVT>
struct PmTile {
    _Float16 k[32][HD + 8];
    _Float16 v[2][HD / 32][64][8];
    uint16_t dk[KVT == F16 ? 1 : HD / 32][32], dv[KVT == F16 ? 1 : HD / 32][32];
};

// What a thread carries of the next 32 positions: KT runs of 16 bytes of K (4 for
// q4_0) and VT tasks of 8 positions of V.
template <int HD, int KVT>
struct PmStage {
    // K: runs of 16 bytes (f16: 8 elements, q8_0: 16), q4_0: 4 bytes (8 elements)
    static constexpr int KRUNS = KVT == F16 ? 32 * HD / 8 : KVT == Q8_0 ? 32 * HD / 16 : 32 * HD / 8;
    static constexpr int KT = (KRUNS + 255) / 256;
    static constexpr int KD = KVT == Q4_0 ? 1 : 4;           // dwords of a run
    // V: 8 positions of one (ks, g) x (f16: 4 elements, 8 bytes; q8_0: 4 bytes, q4_0: 2 bytes = 4 elements 16 apart)
    static constexpr int VE = 4;
    static constexpr int VTASKS = 4 * HD / VE;
    static constexpr int VT = (VTASKS + 255) / 256;
    static constexpr int VD = KVT == F16 ? 2 : 1;
    static constexpr int STASKS = KVT == F16 ? 0 : 2 * 32 * HD / 64;     // dwords of scales, K then V
    static constexpr int SCT = (STASKS + 255) / 256;
    uint32_t k[KT][KD], v[VT][8][VD], s[SCT ? SCT : 1];
};

template <int HD, int KVT>
__device__ __forceinline__ void pm_load(PmStage<HD, KVT> &t, const PagedPool &p, const PaUnit u[2]) {
    using T = PmStage<HD, KVT>;
    constexpr int RB = paged_row_bytes(KVT, HD);
#pragma unroll
    for (int n = 0; n < T::KT; n++) {
        const int x = threadIdx.x + 256 * n;
        if (T::KRUNS % 256 && x >= T::KRUNS) break;
        constexpr int per = RB / (4 * T::KD);
        const int pos = x / per, at = x % per;
        pa_load<T::KD>(t.k[n], p.k + (pos < 16 ? u[0].row : u[1].row) + (pos & 15) * RB + at * 4 * T::KD);
    }
#pragma unroll
    for (int n = 0; n < T::VT; n++) {
        const int x = threadIdx.x + 256 * n;
        if (T::VTASKS % 256 && x >= T::VTASKS) break;
        constexpr int per = HD / T::VE;
        const int kg = x / per, at = x % per;
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const int pos = pm_pos(kg >> 1, kg & 1, j);      // 16 ks ..: unit ks
            const uint8_t *row = p.v + u[0].row + (kg >> 1 ? u[1].row - u[0].row : 0) + (pos & 15) * RB;
            if constexpr (KVT == Q4_0) t.v[n][j][0] = *(const uint16_t *)(row + 2 * at);
            else pa_load<T::VD>(t.v[n][j], row + 4 * T::VD * at);
        }
    }
    if constexpr (T::SCT > 0) {
#pragma unroll
        for (int n = 0; n < T::SCT; n++) {
            const int x = threadIdx.x + 256 * n;
            if (T::STASKS % 256 && x >= T::STASKS) break;
            constexpr int per = HD / 64;
            const int pos = x / per % 32, at = x % per;
            const uint8_t *pool = x < T::STASKS / 2 ? p.k : p.v;
            t.s[n] = *(const uint32_t *)(pool + (pos < 16 ? u[0].sc : u[1].sc) + (pos & 15) * (HD / 16) + 4 * at);
        }
    }
}

// dead: positions that no row of the workgroup attends hold zeros (lo <= pos <
// hi counted from the tile's first); returns whether a value of a live position is
// not finite (edge tiles only: it is zero in LDS then)
template <int HD, int KVT>
__device__ __forceinline__ bool pm_store(PmTile<HD, KVT> &d, const PmStage<HD, KVT> &t, bool edge, int lo, int hi) {
    using T = PmStage<HD, KVT>;
    constexpr int RB = paged_row_bytes(KVT, HD);
    bool odd = false;
#pragma unroll
    for (int n = 0; n < T::KT; n++) {
        const int x = threadIdx.x + 256 * n;
        if (T::KRUNS % 256 && x >= T::KRUNS) break;
        constexpr int per = RB / (4 * T::KD);
        const int pos = x / per, at = x % per;
        if constexpr (KVT == F16) {
            *(pa_v4u *)&d.k[pos][8 * at] = pa_v4u{t.k[n][0], t.k[n][1], t.k[n][2], t.k[n][3]};
        } else if constexpr (KVT == Q8_0) {
            // bytes 16 at ..: group g4 = 16 at / (HD / 4), elements 32 s + 8 g4 + j of two s
            constexpr int G4 = HD / 64;                      // runs of a group
            const int g4 = at / G4, s0 = at % G4 * 2;
#pragma unroll
            for (int s = 0; s < 2; s++) {
                const uint32_t a = t.k[n][2 * s], b = t.k[n][2 * s + 1];
                *(pa_v4u *)&d.k[pos][32 * (s0 + s) + 8 * g4] =
                    pa_v4u{pa_q8(__builtin_amdgcn_perm(0, a, 0x0c010c00u)), pa_q8(__builtin_amdgcn_perm(0, a, 0x0c030c02u)),
                           pa_q8(__builtin_amdgcn_perm(0, b, 0x0c010c00u)), pa_q8(__builtin_amdgcn_perm(0, b, 0x0c030c02u))};
            }
        } else {
            const int g4 = at / (HD / 32), s = at % (HD / 32);
            const uint32_t w = t.k[n][0];
            *(pa_v4u *)&d.k[pos][32 * s + 8 * g4] = pa_v4u{pa_q4(pa_nib(w, 0)), pa_q4(pa_nib(w, 1)), pa_q4(pa_nib(w, 2)), pa_q4(pa_nib(w, 3))};
        }
    }
#pragma unroll
    for (int n = 0; n < T::VT; n++) {
        const int x = threadIdx.x + 256 * n;
        if (T::VTASKS % 256 && x >= T::VTASKS) break;
        constexpr int per = HD / T::VE;
        const int kg = x / per, at = x % per, ks = kg >> 1, g = kg & 1;
        uint32_t v[8][T::VD];
#pragma unroll
        for (int j = 0; j < 8; j++)
#pragma unroll
            for (int i = 0; i < T::VD; i++) v[j][i] = t.v[n][j][i];
        if constexpr (KVT == F16) {
            if (edge) {
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    const int pos = pm_pos(ks, g, j);
                    const bool dead = pos < lo || pos >= hi;
#pragma unroll
                    for (int i = 0; i < T::VD; i++) {
                        uint32_t y = dead ? 0u : v[j][i];
                        const bool a0 = (y & 0x7c00u) == 0x7c00u, a1 = (y & 0x7c000000u) == 0x7c000000u;
                        odd |= a0 | a1;
                        y = a0 ? y & 0xffff0000u : y;
                        v[j][i] = a1 ? y & 0xffffu : y;
                    }
                }
            }
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int e = 4 * at + i;
                pa_v4u w;
#pragma unroll
                for (int k = 0; k < 4; k++) w[k] = __builtin_amdgcn_perm(v[2 * k + 1][i >> 1], v[2 * k][i >> 1], (i & 1) ? 0x07060302u : 0x05040100u);
                *(pa_v4u *)d.v[ks][e >> 5][32 * g + (e & 31)] = w;
            }
        } else {
            // q8_0 bytes 4 at .. / q4_0 nibbles 4 at ..: c = 4 at / (HD / 16), tiles m0 .. m0 + 3, elements 16 m + c
            constexpr int per16 = HD / 64;
            const int c = at / per16, m0 = at % per16 * 4;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int e = 16 * (m0 + i) + c;
                pa_v4u w;
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    if constexpr (KVT == Q8_0)
                        w[k] = pa_q8(__builtin_amdgcn_perm(v[2 * k + 1][0], v[2 * k][0], 0x0c000c00u | i | ((4 + i) << 16)));
                    else
                        w[k] = pa_q4(__builtin_amdgcn_perm(pa_nib(v[2 * k + 1][0], i), pa_nib(v[2 * k][0], i), 0x05040100u));
                }
                *(pa_v4u *)d.v[ks][e >> 5][32 * g + (e & 31)] = w;
            }
        }
    }
    if constexpr (T::SCT > 0) {
#pragma unroll
        for (int n = 0; n < T::SCT; n++) {
            const int x = threadIdx.x + 256 * n;
            if (T::STASKS % 256 && x >= T::STASKS) break;
            constexpr int per = HD / 64;
            const int pos = x / per % 32, at = x % per;
            uint16_t(*to)[32] = x < T::STASKS / 2 ? d.dk : d.dv;
            to[2 * at][pos] = (uint16_t)t.s[n];
            to[2 * at + 1][pos] = (uint16_t)(t.s[n] >> 16);
        }
    }
    return odd;
}

// between a wave's own LDS writes and reads of what its other lanes wrote
__device__ __forceinline__ void pm_wave() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

// rows of 32 floats on their way between memory and operands, padded
constexpr int PM_COLS = 36, PM_TR = 32 * PM_COLS;

template <int HD, int KVT>
__global__ __launch_bounds__(256, HD >= 256 ? 1 : 2) void k_paged_many(PagedAttn a, PagedPlan pl) {
    constexpr int HE = HD > 256 ? 256 : HD, ES = HD / HE, NS = HE / 16, NE = HE / 32, NB = HD > 256 ? 1 : 2;   // NB: buffers
    constexpr size_t TB = sizeof(PmTile<HD, KVT>) * NB, RB = (size_t)4 * PM_TR * 4;
    __shared__ __align__(16) uint8_t lds[TB > RB ? TB : RB];  // the tiles; before and after them rows on their way (4 waves' PM_TR floats)
    PmTile<HD, KVT> *const tiles = (PmTile<HD, KVT> *)lds;
    __shared__ __align__(16) float xs[ES > 1 ? 4 : 1][ES > 1 ? 64 : 1][16];
    __shared__ int odds[3];                                  // by iteration: whether the tile held a non-finite value
    const int lane = threadIdx.x & 63, wave = pa_uniform(threadIdx.x >> 6), c = lane & 31, g = lane >> 5, ew = wave % ES, rw = wave / ES;
    const PagedPool &p = a.p;
    const PagedBatch &b = a.b;
    const int G = a.grp, R = pl.many.rows;

    // Workgroups of one XCD (every eighth) take neighbouring shares: row tiles
    // that read the same K and V find them in its L2.
    const int per = (pl.many.wgs + 7) >> 3, w = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
    int mine;
    const int total = pa_total<true>(a, pl, mine), share = pa_share(pl.many, total);
    const int first = w * share, stop = w < pl.many.wgs ? min(first + share, total) : 0;
    for (int u = first; u < stop;) {
        const PaPiece x = pa_piece<true>(a, pl, mine, w, u, first, stop);
        u += x.n;
        const PagedSeq &sq = x.sq;
        const int kvh = x.kvh, hi0 = x.hi0, lo0 = x.lo0, lo1 = x.lo1, start = x.start, end = x.end;
        bool bad = sq.bad;
        if (bad && threadIdx.x == 0) paged_flag(p, PAGED_BAD_BATCH);
        const int last = (x.seglen - 1) >> 4, iters = end > start ? (end - start + 31) / 32 : 0;

        // the lane's row, its positions [rlo, rhi], and its query in two halves
        const int r = x.tile * R + 32 * rw + c;
        const bool ok = 32 * rw < R && r < sq.nq * G;
        const bool busy = 32 * rw < R && x.tile * R + 32 * rw < sq.nq * G;   // whether the wave has rows
        const int ri = ok ? r / G : 0, head = kvh * G + (ok ? r - ri * G : 0), tok = sq.t0 + ri;
        int rlo = lo0, rhi = hi0;
        if (ok) {
            if (!x.pre) {
                rhi = sq.len - sq.nq + ri;
                rlo = a.window ? max(0, rhi + 1 - a.window) : 0;
            } else if (a.window) {
                rlo = max(0, pa_token_pos(p, b, tok) + 1 - a.window);
            }
        }
        PmStage<HD, KVT> st;
        PaUnits us, more_us;                                     // of 32 steps, and of the next 32
        PaUnit un[2], nx[2];
        if (iters) {
            us = pa_units<KVT>(p, x.table, start >> 4, 2, last, kvh, bad);
            nx[0] = pa_unit<HD, KVT>(p, us, 0);
            nx[1] = pa_unit<HD, KVT>(p, us, 1);
            pm_load<HD, KVT>(st, p, nx);
        }
        // The wave's 32 query rows, 32 elements at a time through its part of LDS:
        // whole lines from memory, then the operand's 8 elements of one row.
        pa_v8h q0[NS], q1[NS];
        float qs;
        {
            pa_v4f y[NE][4];                                     // rows 8 k + lane / 8, elements 32 e + 4 (lane % 8) ..
            float am[4];
            const float *src[4];
            const bool al = (((uintptr_t)a.q & 15) | (a.qs & 3)) == 0;
#pragma unroll
            for (int k = 0; k < 4; k++) {
                const int rr = x.tile * R + 32 * rw + 8 * k + (lane >> 3), i = rr / G;
                src[k] = 32 * rw < R && rr < sq.nq * G ? a.q + (size_t)(sq.t0 + i) * a.qs + (size_t)(kvh * G + rr - i * G) * HD + HE * ew + 4 * (lane & 7) : nullptr;
                am[k] = 0.0f;
            }
#pragma unroll
            for (int e = 0; e < NE; e++)
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    const float *d = src[k] + 32 * e;
                    y[e][k] = !src[k] ? pa_v4f{0.0f, 0.0f, 0.0f, 0.0f} : al ? *(const pa_v4f *)d : pa_v4f{d[0], d[1], d[2], d[3]};
                }
#pragma unroll
            for (int k = 0; k < 4; k++) {
#pragma unroll
                for (int e = 0; e < NE; e++)
                    am[k] = fmaxf(fmaxf(am[k], fmaxf(fabsf(y[e][k][0]), fabsf(y[e][k][1]))), fmaxf(fabsf(y[e][k][2]), fabsf(y[e][k][3])));
                am[k] = group_max<8>(am[k]);
            }
            float *const tr = (float *)lds + wave * PM_TR;
            __syncthreads();                                     // the previous piece's tiles and rows are used
#pragma unroll
            for (int k = 0; k < 4; k++)
                if ((lane & 7) == 0) tr[(8 * k + (lane >> 3)) * PM_COLS] = am[k];
            pm_wave();
            float mx = tr[c * PM_COLS];                          // the lane's row
            if constexpr (ES > 1) {                              // over both halves of the elements
                __syncthreads();
                mx = fmaxf(mx, ((float *)lds + (wave ^ 1) * PM_TR)[c * PM_COLS]);
                __syncthreads();
            }
            const int sh = pa_shift(mx);
            qs = pa_score_scale<KVT>(a, sh);
#pragma unroll
            for (int e = 0; e < NE; e++) {
                pm_wave();
#pragma unroll
                for (int k = 0; k < 4; k++) *(pa_v4f *)(tr + (8 * k + (lane >> 3)) * PM_COLS + 4 * (lane & 7)) = y[e][k];
                pm_wave();
#pragma unroll
                for (int s = 0; s < 2; s++) {
                    const pa_v4f u0 = *(const pa_v4f *)(tr + c * PM_COLS + 16 * s + 8 * g), u1 = *(const pa_v4f *)(tr + c * PM_COLS + 16 * s + 8 * g + 4);
                    uint32_t hi[4], lo[4];
                    pa_split(__builtin_ldexpf(u0[0], sh), __builtin_ldexpf(u0[1], sh), hi[0], lo[0]);
                    pa_split(__builtin_ldexpf(u0[2], sh), __builtin_ldexpf(u0[3], sh), hi[1], lo[1]);
                    pa_split(__builtin_ldexpf(u1[0], sh), __builtin_ldexpf(u1[1], sh), hi[2], lo[2]);
                    pa_split(__builtin_ldexpf(u1[2], sh), __builtin_ldexpf(u1[3], sh), hi[3], lo[3]);
                    q0[2 * e + s] = pa_op(hi[0], hi[1], hi[2], hi[3]);
                    q1[2 * e + s] = pa_op(lo[0], lo[1], lo[2], lo[3]);
                }
            }
        }
        const float capl = a.cap * 1.4426950408889634f;
        pa_v16f o[NE];
        float m = -__builtin_inff(), l = 0.0f;
#pragma unroll
        for (int e = 0; e < NE; e++)
#pragma unroll
            for (int i = 0; i < 16; i++) o[e][i] = 0.0f;
        __syncthreads();
        if (threadIdx.x < 3) odds[threadIdx.x] = 0;
        __syncthreads();

        for (int it = 0, turn = 0; it < iters; it++, turn = turn == 2 ? 0 : turn + 1) {
            const int base = start + 32 * it;
            const bool edge = base + 31 > hi0 || base < lo1 || base + 32 > end;
            PmTile<HD, KVT> &d = tiles[NB == 2 ? it & 1 : 0];
            if (NB == 1 && it) __syncthreads();                  // one buffer: the previous positions are used
            if (pm_store<HD, KVT>(d, st, edge, lo0 - base, end - base)) odds[turn] = 1;
            un[0] = nx[0];
            un[1] = nx[1];
            if ((it & 31) == 31) us = more_us;
            if (it + 1 < iters) {
                nx[0] = pa_unit<HD, KVT>(p, us, 2 * (it + 1) & 63);
                nx[1] = pa_unit<HD, KVT>(p, us, (2 * (it + 1) & 63) + 1);
                pm_load<HD, KVT>(st, p, nx);
            }
            if ((it & 31) == 0 && it + 32 < iters) more_us = pa_units<KVT>(p, x.table, (base >> 4) + 64, 2, last, kvh, bad);
            lds_barrier();
            const int odd = odds[turn];
            if (threadIdx.x == 0) odds[turn == 0 ? 2 : turn - 1] = 0;        // the iteration after the next's: written behind the next barrier
            if (!busy && ES == 1) continue;
            // scores at positions base + 8 (i / 4) + 4 g + i % 4
            pa_v16f sc;
#pragma unroll
            for (int i = 0; i < 16; i++) sc[i] = 0.0f;
            const _Float16 *kr = &d.k[c][HE * ew + 8 * g];
            if constexpr (KVT == F16) {
#pragma unroll
                for (int s = 0; s < NS; s++) {
                    const pa_v8h ko = *(const pa_v8h *)(kr + 16 * s);
                    sc = pa_mma32(ko, q0[s], sc);
                    sc = pa_mma32(ko, q1[s], sc);
                }
            } else {
#pragma unroll
                for (int s = 0; s < NE; s++) {
                    pa_v16f y;
#pragma unroll
                    for (int i = 0; i < 16; i++) y[i] = 0.0f;
#pragma unroll
                    for (int k = 2 * s; k < 2 * s + 2; k++) {
                        const pa_v8h ko = *(const pa_v8h *)(kr + 16 * k);
                        y = pa_mma32(ko, q0[k], y);
                        y = pa_mma32(ko, q1[k], y);
                    }
#pragma unroll
                    for (int k = 0; k < 4; k++) {
                        const uint2 dd = *(const uint2 *)&d.dk[NE * ew + s][8 * k + 4 * g];
                        sc[4 * k] = __builtin_fmaf(pa_lo(dd.x), y[4 * k], sc[4 * k]);
                        sc[4 * k + 1] = __builtin_fmaf(pa_hi(dd.x), y[4 * k + 1], sc[4 * k + 1]);
                        sc[4 * k + 2] = __builtin_fmaf(pa_lo(dd.y), y[4 * k + 2], sc[4 * k + 2]);
                        sc[4 * k + 3] = __builtin_fmaf(pa_hi(dd.y), y[4 * k + 3], sc[4 * k + 3]);
                    }
                }
            }
            if constexpr (ES > 1) {
#pragma unroll
                for (int k = 0; k < 4; k++) *(pa_v4f *)&xs[wave][lane][4 * k] = pa_v4f{sc[4 * k], sc[4 * k + 1], sc[4 * k + 2], sc[4 * k + 3]};
                lds_barrier();
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    const pa_v4f y = *(const pa_v4f *)&xs[wave ^ 1][lane][4 * k];
#pragma unroll
                    for (int i = 0; i < 4; i++) sc[4 * k + i] += y[i];
                }
            }
            float mt = -__builtin_inff();
#pragma unroll
            for (int i = 0; i < 16; i++) sc[i] *= qs;
            if (a.cap > 0.0f) {
#pragma unroll
                for (int i = 0; i < 16; i++) sc[i] = capl * pa_tanh(sc[i]);
            }
            if (edge) {
#pragma unroll
                for (int i = 0; i < 16; i++) {
                    const int pos = base + 8 * (i >> 2) + 4 * g + (i & 3);
                    sc[i] = pos >= rlo && pos <= rhi && pos < end ? sc[i] : -__builtin_inff();
                }
            }
            if constexpr (KVT == F16) {
#pragma unroll
                for (int i = 0; i < 16; i++) mt = fmaxf(mt, sc[i]);
            } else {
                // + the exponent of the position's largest value scale
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    uint2 y = make_uint2(0x00010001u, 0x00010001u);      // all zero: the smallest scale there is
#pragma unroll
                    for (int s = 0; s < HD / 32; s++) {
                        const uint2 z = *(const uint2 *)&d.dv[s][8 * k + 4 * g];
                        y.x = max(y.x & 0xffffu, z.x & 0x7fffu) | max(y.x & 0xffff0000u, z.x & 0x7fff0000u);
                        y.y = max(y.y & 0xffffu, z.y & 0x7fffu) | max(y.y & 0xffff0000u, z.y & 0x7fff0000u);
                    }
                    mt = fmaxf(mt, sc[4 * k] + (float)__builtin_amdgcn_frexp_expf(pa_lo(y.x)));
                    mt = fmaxf(mt, sc[4 * k + 1] + (float)__builtin_amdgcn_frexp_expf(pa_hi(y.x)));
                    mt = fmaxf(mt, sc[4 * k + 2] + (float)__builtin_amdgcn_frexp_expf(pa_lo(y.y)));
                    mt = fmaxf(mt, sc[4 * k + 3] + (float)__builtin_amdgcn_frexp_expf(pa_hi(y.y)));
                }
            }
            mt = fmaxf(mt, partner<32>(mt));
            if (__any(mt > m + PA_LAG)) {
                const float mn = fmaxf(m, mt), cr = mn > m ? __builtin_amdgcn_exp2f(m - mn) : 1.0f;
                l *= cr;
#pragma unroll
                for (int e = 0; e < NE; e++) o[e] *= cr;
                m = mn;
            }
            const float mr = m == -__builtin_inff() ? 0.0f : m - PA_SHIFT;
#pragma unroll
            for (int i = 0; i < 16; i++) {
                sc[i] = __builtin_amdgcn_exp2f(sc[i] - mr);
                l += sc[i];
            }
            if constexpr (KVT == F16) {
#pragma unroll
                for (int ks = 0; ks < 2; ks++) {
                    uint32_t hi[4], lo[4];
#pragma unroll
                    for (int k = 0; k < 4; k++) pa_split(sc[8 * ks + 2 * k], sc[8 * ks + 2 * k + 1], hi[k], lo[k]);
                    const pa_v8h b0 = pa_op(hi[0], hi[1], hi[2], hi[3]), b1 = pa_op(lo[0], lo[1], lo[2], lo[3]);
#pragma unroll
                    for (int e = 0; e < NE; e++) {
                        const pa_v8h va = *(const pa_v8h *)d.v[ks][NE * ew + e][lane];
                        o[e] = pa_mma32(va, b0, o[e]);
                        o[e] = pa_mma32(va, b1, o[e]);
                    }
                }
                if (odd) {
                    // non-finite values, zero in LDS, added to the rows that attend them
                    for (int k = 0; k < 32; k++) {
                        const int pos = base + k;
                        if (pos < lo0 || pos >= end) continue;
                        const uint16_t *row = (const uint16_t *)(p.v + (k < 16 ? un[0].row : un[1].row)) + (k & 15) * HD + HE * ew;
                        float wx = 0.0f;
#pragma unroll
                        for (int i = 0; i < 16; i++) {
                            const float v = __shfl(sc[i], 32 * ((k >> 2) & 1) + c, 64);
                            if (i == 4 * (k >> 3) + (k & 3)) wx = v;
                        }
                        const bool sees = pos >= rlo && pos <= rhi;
#pragma unroll
                        for (int e = 0; e < NE; e++)
#pragma unroll
                            for (int i = 0; i < 16; i++) {
                                const uint16_t hv = row[32 * e + 8 * (i >> 2) + 4 * g + (i & 3)];
                                if (sees && (hv & 0x7c00) == 0x7c00) o[e][i] += wx * h2f(hv);
                            }
                    }
                }
            } else {
#pragma unroll
                for (int e = 0; e < NE; e++) {
#pragma unroll
                    for (int ks = 0; ks < 2; ks++) {
                        uint32_t hi[4], lo[4];
#pragma unroll
                        for (int k = 0; k < 2; k++) {
                            const uint2 dd = *(const uint2 *)&d.dv[NE * ew + e][16 * ks + 8 * k + 4 * g];
                            const float w0 = sc[8 * ks + 4 * k], w1 = sc[8 * ks + 4 * k + 1], w2 = sc[8 * ks + 4 * k + 2], w3 = sc[8 * ks + 4 * k + 3];
                            pa_split(w0 == 0.0f ? 0.0f : w0 * pa_lo(dd.x), w1 == 0.0f ? 0.0f : w1 * pa_hi(dd.x), hi[2 * k], lo[2 * k]);
                            pa_split(w2 == 0.0f ? 0.0f : w2 * pa_lo(dd.y), w3 == 0.0f ? 0.0f : w3 * pa_hi(dd.y), hi[2 * k + 1], lo[2 * k + 1]);
                        }
                        const pa_v8h va = *(const pa_v8h *)d.v[ks][NE * ew + e][lane];
                        o[e] = pa_mma32(va, pa_op(hi[0], hi[1], hi[2], hi[3]), o[e]);
                        o[e] = pa_mma32(va, pa_op(lo[0], lo[1], lo[2], lo[3]), o[e]);
                    }
                }
            }
        }
        if (__any(bad)) {
            if (lane == 0 && !sq.bad) paged_flag(p, PAGED_BAD_PAGE);
            l = __builtin_nanf("");
        }
        l += partner<32>(l);
        // out through LDS as the queries came in
        float *const tr = (float *)lds + wave * PM_TR;
        __syncthreads();                                         // the tiles are used
        constexpr float VS = KVT == Q8_0 ? 512.0f : 1.0f;
        float *to[4];
        bool out = false;
        if (g == 0) {
            PaSink k = {nullptr, nullptr, false};
            if (ok) {
                k = pa_sink<true>(a, pl, x, share, r - x.tile * R, tok, head, ew == 0);
                if (!k.out && ew == 0) *k.ml = make_float2(m, l);
            }
            out = k.out;
            *(float **)(tr + c * PM_COLS) = k.o;
        }
        out = __any(out);
        pm_wave();
#pragma unroll
        for (int k = 0; k < 4; k++) to[k] = *(float **)(tr + (8 * k + (lane >> 3)) * PM_COLS);
        const bool none = out && !sq.bad && sq.len - sq.nq + ri < 0;
        const float f = none ? 0.0f : out ? VS / l : VS;
#pragma unroll
        for (int e = 0; e < NE; e++) {
            pm_wave();
#pragma unroll
            for (int k = 0; k < 4; k++) {
                const pa_v4f y = {o[e][4 * k], o[e][4 * k + 1], o[e][4 * k + 2], o[e][4 * k + 3]};
                *(pa_v4f *)(tr + c * PM_COLS + 8 * k + 4 * g) = none ? pa_v4f{0.0f, 0.0f, 0.0f, 0.0f} : y * f;
            }
            pm_wave();
#pragma unroll
            for (int k = 0; k < 4; k++)
                if (to[k]) pa_store4(to[k] + HE * ew + 32 * e + 4 * (lane & 7), *(const pa_v4f *)(tr + (8 * k + (lane >> 3)) * PM_COLS + 4 * (lane & 7)));
        }
    }
}

template <int KVT>
hipError_t pa_many(const PagedAttn &a, const PagedPlan &pl, hipStream_t s) {
    const dim3 grid((pl.many.wgs + 7) / 8 * 8), wg(256);
    switch (a.p.hd) {
    case 64: hipLaunchKernelGGL((k_paged_many<64, KVT>), grid, wg, 0, s, a, pl); break;
    case 128: hipLaunchKernelGGL((k_paged_many<128, KVT>), grid, wg, 0, s, a, pl); break;
    case 256: hipLaunchKernelGGL((k_paged_many<256, KVT>), grid, wg, 0, s, a, pl); break;
    case 512: hipLaunchKernelGGL((k_paged_many<512, KVT>), grid, wg, 0, s, a, pl); break;
    default: return hipErrorInvalidValue;
    }
    return hipGetLastError();
}

}  // namespace g4
