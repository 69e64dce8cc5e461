// paged_many.h -- attention of many rows over the paged KV cache (paged_attn.h):
// prompt chunks, and the prefix of a large batch.
//
// Bound by the matrix cores (two instructions per operand pair: a query's and a
// weight's two halves), by LDS, which feeds them at the same rate, and by the
// softmax on the VALU.  A workgroup of 8 waves takes up to 128 rows of one KV
// head, 16 of a wave, 32 positions at a time on v_mfma_f32_16x16x32_f16.  All its
// threads bring the next 32 positions' K and V from the pages to registers while
// the present ones are computed, then to LDS as operands: K rows as halves (the
// block formats' integers are halves too), V rows turned to 8 positions of one
// element, so each is converted once for all rows.  Two waves per SIMD cover each
// other's LDS reads and exponentials (4 waves of 32 rows on the 32x32x16 form read
// half of the LDS bytes, but left one wave per SIMD with its operands in
// accumulation registers: 4.3 us for 32 positions of 128 rows of 256).  Heads of
// 512: two waves share 16 rows, each with half of the elements, their scores added
// through LDS.
//
// 32 positions of 128 rows of 256 take 2.06 us of a workgroup per CU: the matrix
// cores at 1.04 PFLOP/s, a large f16 product of the library reaches 1.17.  A call of
// four prompts of up to 509 tokens behind up to 3800 positions, 8 q / 4 kv heads,
// capped, takes 79 us: the rest is each piece's start and end (8 us), the shares'
// rest, and the sums of the split tiles out and in again (about 60 MB each way, the join
// 11 us).  Few rows do not make a tile cheaper (20 rows of 256: 1.4 us for 32
// positions): it is then one wave's chain from the staging to its second product.
// Waves one stage apart by counters in LDS instead of a barrier gave 3 %, and spills
// with quantized pages.
#pragma once

#include "paged_attn.h"

namespace g4 {

constexpr int PM_THREADS = 512;

// The 8 positions (of 32) that lane group g (lane / 16) holds, j of 8: the order
// of a wave's scores and of the second product's operand.
__device__ __forceinline__ int pm_pos(int g, int j) { return 16 * (j >> 2) + 4 * g + (j & 3); }

// Where 8 elements of a K row lie in LDS: unit g of elements 32 s, row c of 16.  Rows
// are moved about by (s, g), so that neither the 16 lanes that write one row's units
// nor those that read 16 rows' meet in a bank.
__device__ __forceinline__ int pm_key(int c, int g, int s) { return 16 * g + (c ^ g ^ (4 * (s & 3))); }

// LDS of 32 positions: K as operands [2 s + half][64 units of 8 halves] (pm_key); V [32][HD + 16] halves, read
// transposed (ds_read_b64_tr_b16), quantized V [HD / 16][64 lanes][8] as operands;
// the scales [HD / 32][32] of K and of V, and each position's pa_exponent of its
// largest V scale (quantized)
template <int HD, int KVT>
struct PmTile {
    _Float16 k[HD / 16][64][8];
    _Float16 v[KVT == F16 ? 32 * (HD + 16) / 512 : HD / 16][64][8];
    uint16_t dk[KVT == F16 ? 1 : HD / 32][32], dv[KVT == F16 ? 1 : HD / 32][32];
    float ev[KVT == F16 ? 4 : 32];
};

// What a thread carries of the next 32 positions.
template <int HD, int KVT>
struct PmStage {
    // K: runs of 16 bytes (f16: 8 elements, q8_0: 16), q4_0: 4 bytes (8 elements)
    static constexpr int KRUNS = KVT == F16 ? 32 * HD / 8 : KVT == Q8_0 ? 32 * HD / 16 : 32 * HD / 8;
    static constexpr int KT = (KRUNS + PM_THREADS - 1) / PM_THREADS;
    static constexpr int KD = KVT == Q4_0 ? 1 : 4;           // dwords of a run
    // V: f16 runs as K's; else 8 positions of one g x 4 elements, 16 apart (q8_0 4 bytes, q4_0 2 bytes)
    static constexpr int VTASKS = KVT == F16 ? KRUNS : HD;
    static constexpr int VT = (VTASKS + PM_THREADS - 1) / PM_THREADS;
    static constexpr int STASKS = KVT == F16 ? 0 : 2 * 32 * HD / 64;     // dwords of scales, K then V
    static constexpr int SCT = (STASKS + PM_THREADS - 1) / PM_THREADS;
    uint32_t k[KT][KD], v[VT][KVT == F16 ? 4 : 8], s[SCT ? SCT : 1];
};

template <int HD, int KVT>
__device__ __forceinline__ void pm_load(PmStage<HD, KVT> &t, const PagedPool &p, const PaUnit u[2], int tid) {
    using T = PmStage<HD, KVT>;
    constexpr int RB = paged_row_bytes(KVT, HD);
#pragma unroll
    for (int n = 0; n < T::KT; n++) {
        const int x = tid + PM_THREADS * n;
        if (T::KRUNS % PM_THREADS && x >= T::KRUNS) break;
        constexpr int per = RB / (4 * T::KD), step = PM_THREADS / per;       // positions of one n
        const int pos = x / per, at = x % per;
        const uint32_t off = (pos & 15) * RB + at * 4 * T::KD;
        if constexpr (step <= 16) pa_load<T::KD>(t.k[n], p.k + (n * step < 16 ? u[0].row : u[1].row) + off);
        else pa_load<T::KD>(t.k[n], p.k + (pos < 16 ? u[0].row : u[1].row) + off);
    }
#pragma unroll
    for (int n = 0; n < T::VT; n++) {
        const int x = (KVT == F16 ? tid ^ 256 : tid) + PM_THREADS * n;   // heads of 64: half of the waves K, half V
        if (T::VTASKS % PM_THREADS && x >= T::VTASKS) break;
        if constexpr (KVT == F16) {
            constexpr int per = RB / 16;
            const int pos = x / per;
            pa_load<4>(t.v[n], p.v + (pos < 16 ? u[0].row : u[1].row) + (uint32_t)((pos & 15) * RB + x % per * 16));
        } else {
            constexpr int per = HD / 4;
            const int g = per % 64 == 0 ? pa_uniform(x / per) : x / per;
            const uint32_t off = x % per * (KVT == Q4_0 ? 2 : 4);
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const uint8_t *row = p.v + u[j >> 2].row + (uint32_t)(4 * g + (j & 3)) * RB;
                if constexpr (KVT == Q4_0) t.v[n][j] = *(const uint16_t *)(row + off);
                else t.v[n][j] = *(const uint32_t *)(row + off);
            }
        }
    }
    if constexpr (T::SCT > 0) {
#pragma unroll
        for (int n = 0; n < T::SCT; n++) {
            const int x = tid + PM_THREADS * n;
            if (T::STASKS % PM_THREADS && x >= T::STASKS) break;
            constexpr int per = HD / 64;
            const int pos = x / per % 32, at = x % per;
            const uint8_t *pool = x < T::STASKS / 2 ? p.k : p.v;
            t.s[n] = *(const uint32_t *)(pool + (pos < 16 ? u[0].sc : u[1].sc) + (pos & 15) * (HD / 16) + 4 * at);
        }
    }
}

// In edge tiles values of positions that no row of the workgroup attends (outside
// [lo, hi) counted from the tile's first) become 0, and so do non-finite ones;
// returns whether there was one of the latter.
template <int HD, int KVT>
__device__ __forceinline__ bool pm_store(PmTile<HD, KVT> &d, const PmStage<HD, KVT> &t, bool edge, int lo, int hi, int tid) {
    using T = PmStage<HD, KVT>;
    constexpr int RB = paged_row_bytes(KVT, HD);
    bool odd = false;
#pragma unroll
    for (int n = 0; n < T::KT; n++) {
        const int x = tid + PM_THREADS * n;
        if (T::KRUNS % PM_THREADS && x >= T::KRUNS) break;
        constexpr int per = RB / (4 * T::KD);
        const int pos = x / per, at = x % per;
        if constexpr (KVT == F16) {
            *(pa_v4u *)d.k[2 * (at >> 2) + (pos >> 4)][pm_key(pos & 15, at & 3, at >> 2)] = pa_v4u{t.k[n][0], t.k[n][1], t.k[n][2], t.k[n][3]};
        } else if constexpr (KVT == Q8_0) {
            // bytes 16 at ..: group g4 = 16 at / (HD / 4), elements 32 s + 8 g4 + j of two s
            constexpr int G4 = HD / 64;                      // runs of a group
            const int g4 = at / G4, s0 = at % G4 * 2;
#pragma unroll
            for (int s = 0; s < 2; s++) {
                const uint32_t a = t.k[n][2 * s], b = t.k[n][2 * s + 1];
                *(pa_v4u *)d.k[2 * (s0 + s) + (pos >> 4)][pm_key(pos & 15, g4, s0 + s)] =
                    pa_v4u{pa_q8(__builtin_amdgcn_perm(0, a, 0x0c010c00u)), pa_q8(__builtin_amdgcn_perm(0, a, 0x0c030c02u)),
                           pa_q8(__builtin_amdgcn_perm(0, b, 0x0c010c00u)), pa_q8(__builtin_amdgcn_perm(0, b, 0x0c030c02u))};
            }
        } else {
            const int g4 = at / (HD / 32), s = at % (HD / 32);
            const uint32_t w = t.k[n][0];
            *(pa_v4u *)d.k[2 * s + (pos >> 4)][pm_key(pos & 15, g4, s)] = pa_v4u{pa_q4<0>(w), pa_q4<1>(w), pa_q4<2>(w), pa_q4<3>(w)};
        }
    }
#pragma unroll
    for (int n = 0; n < T::VT; n++) {
        const int x = (KVT == F16 ? tid ^ 256 : tid) + PM_THREADS * n;
        if (T::VTASKS % PM_THREADS && x >= T::VTASKS) break;
        if constexpr (KVT == F16) {
            constexpr int per = RB / 16;
            const int pos = x / per, at = x % per;
            pa_v4u w = {t.v[n][0], t.v[n][1], t.v[n][2], t.v[n][3]};
            if (edge) {
                uint32_t nf = 0;                             // bit 15 or 31 where an exponent is all ones
                if (pos < lo || pos >= hi) w = pa_v4u{0, 0, 0, 0};
#pragma unroll
                for (int k = 0; k < 4; k++) nf |= (w[k] & 0x7c007c00u) + 0x04000400u;
                if (nf & 0x80008000u) {
                    odd = true;
#pragma unroll
                    for (int k = 0; k < 4; k++) w[k] = pa_finite(w[k]);
                }
            }
            *(pa_v4u *)(&d.v[0][0][0] + pos * (HD + 16) + 8 * at) = w;
        } else {
            // q8_0 bytes 4 at .. / q4_0 nibbles 4 at ..: c = 4 at / (HD / 16), tiles m0 .. m0 + 3, elements 16 m + c
            constexpr int per = HD / 4, per16 = HD / 64;
            const int g = per % 64 == 0 ? pa_uniform(x / per) : x / per, at = x % per, c = at / per16, m0 = at % per16 * 4;
            const uint32_t *v = t.v[n];
#pragma unroll
            for (int i = 0; i < 4; i++) {
                pa_v4u w;
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    if constexpr (KVT == Q8_0)
                        w[k] = pa_q8(__builtin_amdgcn_perm(v[2 * k + 1], v[2 * k], 0x0c000c00u | i | ((4 + i) << 16)));
                    else
                        w[k] = pa_q4(__builtin_amdgcn_perm(v[2 * k + 1], v[2 * k], 0x05040100u), i);
                }
                *(pa_v4u *)d.v[m0 + i][16 * g + c] = w;
            }
        }
    }
    if constexpr (T::SCT > 0) {
#pragma unroll
        for (int n = 0; n < T::SCT; n++) {
            const int x = tid + PM_THREADS * n;
            if (T::STASKS % PM_THREADS && x >= T::STASKS) break;
            constexpr int per = HD / 64;
            const int pos = x / per % 32, at = x % per;
            uint16_t(*to)[32] = x < T::STASKS / 2 ? d.dk : d.dv;
            to[2 * at][pos] = (uint16_t)t.s[n];
            to[2 * at + 1][pos] = (uint16_t)(t.s[n] >> 16);
            if (x >= T::STASKS / 2) {
                const uint32_t y = t.s[n] & 0x7fff7fffu;
                const float e = group_max<per>(pa_exponent(max(y << 16, y), 1));
                if (at == 0) d.ev[pos] = e;
            }
        }
    }
    return odd;
}

typedef short pa_v4s __attribute__((ext_vector_type(4)));
typedef short pa_v8s __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) pa_v4s *pa_lds4;
__device__ __forceinline__ pa_v8h pm_turned(const _Float16 *a, const _Float16 *b) {
    const pa_v4s x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((pa_lds4)a), y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((pa_lds4)b);
    return __builtin_bit_cast(pa_v8h, pa_v8s{x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w});
}
struct PmKey {
    pa_v8h x;
    uint2 d;
};
struct PmValue {
    pa_v8h x[2];
    uint2 d[2];
};

// read(i) brings operand i of N from LDS, use(i, operand) multiplies with it: reads
// run AHEAD of their use.  (Left to itself the compiler reads, waits and multiplies
// one by one: 130 cycles of LDS latency for 32 of matrix instructions.)
template <int N, int AHEAD, typename R, typename U>
__device__ __forceinline__ void pm_pipeline(R read, U use) {
    decltype(read(0)) x[AHEAD];
#pragma unroll
    for (int i = 0; i < AHEAD && i < N; i++) x[i] = read(i);
#pragma unroll
    for (int i = 0; i < N; i++) {
        __builtin_amdgcn_sched_barrier(0);
        const auto y = x[i % AHEAD];
        use(i, y);
        __builtin_amdgcn_sched_barrier(0);
        if (i + AHEAD < N) x[i % AHEAD] = read(i + AHEAD);
    }
}

// between a wave's own LDS writes and reads of what its other lanes wrote
__device__ __forceinline__ void pm_wave() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

// a wave's 16 rows of 32 floats on their way between memory and operands, padded
constexpr int PM_COLS = 36, PM_TR = 16 * PM_COLS;

template <int HD, int KVT>
__global__ __launch_bounds__(PM_THREADS, HD >= 128 ? 2 : 4) void k_paged_many(PagedCall call) {
    constexpr int HE = HD > 256 ? 256 : HD, ES = HD / HE, NS = HE / 32, NM = HE / 16, NB = HD > 256 ? 1 : 2, AHEAD = HD == 64 || HD == 512 ? 2 : 4, BLOCKS = HD > 64 ? 2 : 1;    // NB: buffers
    constexpr size_t TB = sizeof(PmTile<HD, KVT>) * NB, RB = (size_t)8 * PM_TR * 4;
    __shared__ __align__(16) uint8_t lds[TB > RB ? TB : RB]; // the tiles; before and after them rows on their way
    __shared__ __align__(16) float xs[ES > 1 ? 8 : 1][ES > 1 ? 64 : 1][8];   // partial scores of wave pairs
    __shared__ int odds[3];                                  // by iteration: whether the tile held a non-finite value
    PmTile<HD, KVT> *const tiles = (PmTile<HD, KVT> *)lds;

    // Workgroups of one XCD (every eighth) take neighbouring shares: row tiles
    // that read the same K and V find them in its L2.
    const int per = (call.pl.many.wgs + 7) >> 3, wg = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
    int mine, n_seq;
    const int total = pa_total<true>(call.a, call.pl, mine, n_seq), share = pa_share(call.pl.many, total);
    const int first = wg * share, stop = wg < call.pl.many.wgs ? min(first + share, total) : 0;
    if (blockIdx.x == 0) pa_rest(call.a, call.pl, n_seq);
    PaFind from;
    for (int u = first; u < stop;) {
        const PagedCall call = pa_fresh();
        const PagedAttn &a = call.a;
        const PagedPlan &pl = call.pl;
        const PagedPool &p = a.p;
        const PagedBatch &b = a.b;
        const int tid = pa_thread(), lane = tid & 63, wave = pa_uniform(tid >> 6), c = lane & 15, g = lane >> 4, ew = wave % ES, rw = wave / ES;
        const int G = a.grp, R = pl.many.rows;
        float *const tr = (float *)lds + wave * PM_TR;
        const float capl = a.cap * 1.4426950408889634f;
        const PaPiece x = pa_piece<true>(a, pl, mine, n_seq, from, wg, u, first, stop);
        u += x.took;
        if (x.n == 0) break;                                 // the share ends in a tile's lead
        const PagedSeq &sq = x.sq;
        const int kvh = x.kvh, hi0 = x.hi0, lo0 = x.lo0, lo1 = x.lo1, start = x.start, end = x.end, rows = min(sq.nq * G, (x.tile + 1) * R);     // the tile's rows end at `rows`
        bool bad = sq.bad;
        if (bad && tid == 0) paged_flag(p, PAGED_BAD_BATCH);
        const int last = (x.seglen - 1) >> 4, iters = end > start ? (end - start + 31) / 32 : 0;

        // The queries first (rows 8 k + lane / 8 of the wave's, elements 32 s + 4 (lane %
        // 8) ..): they are back with the page ids, and used while the first keys and values come.
        const int r0 = x.tile * R + 16 * rw;                 // the wave's rows: r0 ..
        pa_v4f y[NS][2];
        {
            const bool al = (((uintptr_t)a.q & 15) | (a.qs & 3)) == 0;
#pragma unroll
            for (int k = 0; k < 2; k++) {
                const int r = r0 + 8 * k + (lane >> 3), i = r / G;
                const bool in = r < rows;
                const float *src = a.q + (size_t)(sq.t0 + (in ? i : 0)) * a.qs + (size_t)(kvh * G + (in ? r - i * G : 0)) * HD + HE * ew + 4 * (lane & 7);
#pragma unroll
                for (int s = 0; s < NS; s++) {
                    const float *d = src + 32 * s;
                    y[s][k] = !in ? pa_v4f{0.0f, 0.0f, 0.0f, 0.0f} : al ? *(const pa_v4f *)d : pa_v4f{d[0], d[1], d[2], d[3]};
                }
            }
        }
        asm volatile("" ::: "memory");
        PmStage<HD, KVT> st;
        PaUnits us, more_us;                                 // of 32 steps, and of the next 32
        PaUnit un[2], nx[2];
        uint64_t outside = 0;                                // of the first 32 steps
        if (iters) {
            us = pa_units(p, x.table, start >> 4, 2, last, kvh);
            outside = pa_check(p, us);
            nx[0] = pa_unit<HD, KVT>(p, us, 0);
            nx[1] = pa_unit<HD, KVT>(p, us, 1);
            pm_load<HD, KVT>(st, p, nx, tid);
        }
        // busy: the wave has rows; the lane's: r0 + c
        const bool busy = r0 < rows, ok = r0 + c < rows;
        const int ri = ok ? (r0 + c) / G : 0, head = kvh * G + (ok ? r0 + c - ri * G : 0), tok = sq.t0 + ri;
        int rlo = lo0, rhi = hi0;                            // the lane's row attends [rlo, rhi]
        if (ok) {
            if (!x.pre) {
                rhi = sq.len - sq.nq + ri;
                rlo = a.window ? max(0, rhi + 1 - a.window) : 0;
            } else if (a.window) {
                rlo = max(0, pa_token_pos(p, b, n_seq, tok) + 1 - a.window);
            }
        }
        bad |= pa_hits(outside, start >> 4, 2, last, rlo, rhi);
        __syncthreads();                                     // the previous piece's tiles and rows are used
        // Queries, 32 elements at a time through the wave's part of LDS: whole lines
        // from memory, then the operand's 8 elements of one row.
        pa_v8h q0[NS], q1[NS];
        float qs;
        {
#pragma unroll
            for (int k = 0; k < 2; k++) {
                float am = 0.0f;
#pragma unroll
                for (int s = 0; s < NS; s++)
                    am = fmaxf(fmaxf(am, fmaxf(fabsf(y[s][k][0]), fabsf(y[s][k][1]))), fmaxf(fabsf(y[s][k][2]), fabsf(y[s][k][3])));
                am = group_max<8>(am);
                if ((lane & 7) == 0) tr[(8 * k + (lane >> 3)) * PM_COLS] = am;
            }
            pm_wave();
            float mx = tr[c * PM_COLS];                      // the lane's row
            if constexpr (ES > 1) {                          // over both halves of the elements
                __syncthreads();
                mx = fmaxf(mx, ((float *)lds + (wave ^ 1) * PM_TR)[c * PM_COLS]);
                __syncthreads();
            }
            const int sh = pa_shift(mx);
            qs = pa_score_scale<KVT>(a, sh);
#pragma unroll
            for (int s = 0; s < NS; s++) {
                pm_wave();
#pragma unroll
                for (int k = 0; k < 2; k++) *(pa_v4f *)(tr + (8 * k + (lane >> 3)) * PM_COLS + 4 * (lane & 7)) = y[s][k];
                pm_wave();
                const pa_v4f u0 = *(const pa_v4f *)(tr + c * PM_COLS + 8 * g), u1 = *(const pa_v4f *)(tr + c * PM_COLS + 8 * g + 4);
                uint32_t hi[4], lo[4];
                pa_split(__builtin_ldexpf(u0[0], sh), __builtin_ldexpf(u0[1], sh), hi[0], lo[0]);
                pa_split(__builtin_ldexpf(u0[2], sh), __builtin_ldexpf(u0[3], sh), hi[1], lo[1]);
                pa_split(__builtin_ldexpf(u1[0], sh), __builtin_ldexpf(u1[1], sh), hi[2], lo[2]);
                pa_split(__builtin_ldexpf(u1[2], sh), __builtin_ldexpf(u1[3], sh), hi[3], lo[3]);
                q0[s] = pa_op(hi[0], hi[1], hi[2], hi[3]);
                q1[s] = pa_op(lo[0], lo[1], lo[2], lo[3]);
            }
        }
        pa_v4f o[NM];
        float m = -__builtin_inff(), l = 0.0f;
#pragma unroll
        for (int e = 0; e < NM; e++) o[e] = pa_v4f{0.0f, 0.0f, 0.0f, 0.0f};
        if (tid < 3) odds[tid] = 0;
        __syncthreads();

        for (int it = 0, turn = 0; it < iters; it++, turn = turn == 2 ? 0 : turn + 1) {
            const int base = start + 32 * it;
            const bool edge = base + 31 > hi0 || base < lo1 || base + 32 > end;
            PmTile<HD, KVT> &d = tiles[NB == 2 ? it & 1 : 0];
            if (NB == 1 && it) __syncthreads();              // one buffer: the previous positions are used
            if (pm_store<HD, KVT>(d, st, edge, lo0 - base, end - base, tid)) odds[turn] = 1;
            un[0] = nx[0];
            un[1] = nx[1];
            if ((it & 31) == 31 && it + 1 < iters) {
                us = more_us;
                bad |= pa_hits(pa_check(p, us), (base + 32) >> 4, 2, last, rlo, rhi);
            }
            if (it + 1 < iters) {
                nx[0] = pa_unit<HD, KVT>(p, us, 2 * (it + 1) & 63);
                nx[1] = pa_unit<HD, KVT>(p, us, (2 * (it + 1) & 63) + 1);
                pm_load<HD, KVT>(st, p, nx, tid);
            }
            if ((it & 31) == 0 && it + 32 < iters) more_us = pa_units(p, x.table, (base >> 4) + 64, 2, last, kvh);
            lds_barrier();
            const int odd = odds[turn];
            if (tid == 0) odds[turn == 0 ? 2 : turn - 1] = 0;    // the iteration after the next's: written behind the next barrier
            if (!busy && ES == 1) continue;
            // scores of row c at positions base + pm_pos(g, j): high and low halves apart,
            // so that no instruction waits for the one before it
            pa_v4f sc[2] = {{0.0f, 0.0f, 0.0f, 0.0f}, {0.0f, 0.0f, 0.0f, 0.0f}}, s2[2] = {{0.0f, 0.0f, 0.0f, 0.0f}, {0.0f, 0.0f, 0.0f, 0.0f}};
            auto key = [&](int i) { return *(const pa_v8h *)d.k[2 * NS * ew + i][pm_key(c, g, i >> 1)]; };
            if constexpr (KVT == F16) {
                pm_pipeline<2 * NS, AHEAD>(key, [&](int i, pa_v8h ko) {
                    sc[i & 1] = pa_mma(ko, q0[i >> 1], sc[i & 1]);
                    s2[i & 1] = pa_mma(ko, q1[i >> 1], s2[i & 1]);
                });
                sc[0] += s2[0];
                sc[1] += s2[1];
            } else {
                // scaled one operand later, when the products are there
                uint2 before;
                auto scaled = [&](int h) {
                    sc[h][0] = __builtin_fmaf(pa_lo(before.x), s2[0][0], sc[h][0]);
                    sc[h][1] = __builtin_fmaf(pa_hi(before.x), s2[0][1], sc[h][1]);
                    sc[h][2] = __builtin_fmaf(pa_lo(before.y), s2[0][2], sc[h][2]);
                    sc[h][3] = __builtin_fmaf(pa_hi(before.y), s2[0][3], sc[h][3]);
                };
                pm_pipeline<2 * NS, AHEAD>([&](int i) { return PmKey{key(i), *(const uint2 *)&d.dk[NS * ew + (i >> 1)][16 * (i & 1) + 4 * g]}; }, [&](int i, PmKey k) {
                    const pa_v4f y = pa_mma(k.x, q1[i >> 1], pa_mma(k.x, q0[i >> 1], pa_v4f{0.0f, 0.0f, 0.0f, 0.0f}));
                    if (i) scaled(1 - (i & 1));
                    s2[0] = y;
                    before = k.d;
                });
                scaled(1);
            }
            if constexpr (ES > 1) {
                *(pa_v4f *)xs[wave][lane] = sc[0];
                *(pa_v4f *)(xs[wave][lane] + 4) = sc[1];
                lds_barrier();
                sc[0] += *(const pa_v4f *)xs[wave ^ 1][lane];
                sc[1] += *(const pa_v4f *)(xs[wave ^ 1][lane] + 4);
            }
            float w[8];
#pragma unroll
            for (int j = 0; j < 8; j++) w[j] = sc[j >> 2][j & 3] * qs;
            if (a.cap > 0.0f) {
                pa_tanh(w);
#pragma unroll
                for (int j = 0; j < 8; j++) w[j] *= capl;
            }
            if (edge) {
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    const int pos = base + pm_pos(g, j);
                    w[j] = pos >= rlo && pos <= rhi && pos < end ? w[j] : -__builtin_inff();
                }
            }
            float mt = -__builtin_inff();
            if constexpr (KVT == F16) {
#pragma unroll
                for (int j = 0; j < 8; j++) mt = fmaxf(mt, w[j]);
            } else {
                // + the exponent of the position's largest value scale
                const pa_v4f e[2] = {*(const pa_v4f *)&d.ev[4 * g], *(const pa_v4f *)&d.ev[16 + 4 * g]};
#pragma unroll
                for (int j = 0; j < 8; j++) mt = fmaxf(mt, w[j] + e[j >> 2][j & 3]);
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
            if constexpr (KVT == F16) {
                uint32_t hi[4], lo[4];
#pragma unroll
                for (int k = 0; k < 4; k++) pa_split(w[2 * k], w[2 * k + 1], hi[k], lo[k]);
                const pa_v8h b0 = pa_op(hi[0], hi[1], hi[2], hi[3]), b1 = pa_op(lo[0], lo[1], lo[2], lo[3]);
                pa_v8h before;                               // low halves one operand later
                // 16 lanes give 4 positions of 16 elements and get 4 positions of their own
                const _Float16 *const vt = &d.v[0][0][0] + (4 * g + (c >> 2)) * (HD + 16) + HE * ew + 4 * (c & 3);
                pm_pipeline<NM, AHEAD>([&](int e) { return pm_turned(vt + 16 * e, vt + 16 * (HD + 16) + 16 * e); }, [&](int e, pa_v8h va) {
                    o[e] = pa_mma(va, b0, o[e]);
                    if (e) o[e - 1] = pa_mma(before, b1, o[e - 1]);
                    before = va;
                });
                o[NM - 1] = pa_mma(before, b1, o[NM - 1]);
                if (odd) {
                    // non-finite values, zero in LDS, added to the rows that attend them
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
                        const bool sees = pos >= rlo && pos <= rhi;
#pragma unroll
                        for (int e = 0; e < NM; e++) {
                            const uint2 hv = *(const uint2 *)(row + 16 * e + 4 * g);
#pragma unroll
                            for (int i = 0; i < 4; i++) {
                                const uint32_t v = (i < 2 ? hv.x : hv.y) >> (16 * (i & 1)) & 0xffffu;
                                if (sees && (v & 0x7c00) == 0x7c00) o[e][i] += wx * h2f((uint16_t)v);
                            }
                            __builtin_amdgcn_sched_barrier(0);
                        }
                    }
                }
            } else {
                // a scale of a position that the row does not attend may be anything
                uint32_t live[4] = {~0u, ~0u, ~0u, ~0u};
                if (edge) {
#pragma unroll
                    for (int j = 0; j < 8; j++) {
                        const int pos = base + pm_pos(g, j);
                        if (!(pos >= rlo && pos <= rhi && pos < end)) live[j >> 1] &= j & 1 ? 0xffffu : 0xffff0000u;
                    }
                }
                // blocks of 32 elements: value tiles 2 s, 2 s + 1
                pm_pipeline<NS, BLOCKS>([&](int s) {
                    const uint16_t *dv = d.dv[NS * ew + s];
                    const pa_v8h(*v)[64] = (const pa_v8h(*)[64])d.v[NM * ew + 2 * s];
                    return PmValue{{v[0][lane], v[1][lane]}, {*(const uint2 *)&dv[4 * g], *(const uint2 *)&dv[16 + 4 * g]}};
                }, [&](int s, PmValue x) {
                    uint32_t hi[4], lo[4];
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        pa_split_scaled(w[4 * h], w[4 * h + 1], x.d[h].x & live[2 * h], hi[2 * h], lo[2 * h]);
                        pa_split_scaled(w[4 * h + 2], w[4 * h + 3], x.d[h].y & live[2 * h + 1], hi[2 * h + 1], lo[2 * h + 1]);
                    }
                    const pa_v8h b0 = pa_op(hi[0], hi[1], hi[2], hi[3]), b1 = pa_op(lo[0], lo[1], lo[2], lo[3]);
                    o[2 * s] = pa_mma(x.x[0], b0, o[2 * s]);
                    o[2 * s + 1] = pa_mma(x.x[1], b0, o[2 * s + 1]);
                    o[2 * s] = pa_mma(x.x[0], b1, o[2 * s]);
                    o[2 * s + 1] = pa_mma(x.x[1], b1, o[2 * s + 1]);
                });
            }
        }
        bad &= ok;
        if (__any(bad)) {
            if (lane == 0 && !sq.bad) paged_flag(p, PAGED_BAD_PAGE);
            if (bad) l = __builtin_nanf("");
        }
        l += partner<16>(l);
        l += partner<32>(l);
        // out through LDS as the queries came in
        __syncthreads();                                     // the tiles are used
        if (!busy) continue;
        const bool nowhere = !sq.bad && sq.len - sq.nq + ri < 0;
        float *to[2];
        bool out = false;
        if (g == 0) {
            PaSink k = {nullptr, nullptr, false};
            if (ok) {
                k = pa_sink<true>(a, pl, x, share, r0 + c - x.tile * R, tok, head, nowhere, ew == 0);
                if (!k.out && ew == 0) *k.ml = make_float2(m, l);
            }
            out = k.out;
            *(float **)(tr + c * PM_COLS) = k.o;
        }
        out = __any(out);
        pm_wave();
#pragma unroll
        for (int k = 0; k < 2; k++) to[k] = *(float **)(tr + (8 * k + (lane >> 3)) * PM_COLS);
        constexpr float VS = KVT == Q8_0 ? 512.0f : 1.0f;
        const bool none = out && nowhere;
        const float f = none ? 0.0f : out ? VS / l : VS;
#pragma unroll
        for (int s = 0; s < NS; s++) {                       // 32 elements at a time: value tiles 2 s, 2 s + 1
            pm_wave();
#pragma unroll
            for (int e = 0; e < 2; e++) *(pa_v4f *)(tr + c * PM_COLS + 16 * e + 4 * g) = none ? pa_v4f{0.0f, 0.0f, 0.0f, 0.0f} : o[2 * s + e] * f;
            pm_wave();
#pragma unroll
            for (int k = 0; k < 2; k++)
                if (to[k]) pa_store4(to[k] + HE * ew + 32 * s + 4 * (lane & 7), *(const pa_v4f *)(tr + (8 * k + (lane >> 3)) * PM_COLS + 4 * (lane & 7)));
        }
    }
}

template <int KVT>
hipError_t pa_many(const PagedAttn &a, const PagedPlan &pl, hipStream_t s) {
    const dim3 grid((pl.many.wgs + 7) / 8 * 8), wg(PM_THREADS);
    switch (a.p.hd) {
    case 64: hipLaunchKernelGGL((k_paged_many<64, KVT>), grid, wg, 0, s, PagedCall{a, pl}); break;
    case 128: hipLaunchKernelGGL((k_paged_many<128, KVT>), grid, wg, 0, s, PagedCall{a, pl}); break;
    case 256: hipLaunchKernelGGL((k_paged_many<256, KVT>), grid, wg, 0, s, PagedCall{a, pl}); break;
    case 512: hipLaunchKernelGGL((k_paged_many<512, KVT>), grid, wg, 0, s, PagedCall{a, pl}); break;
    default: return hipErrorInvalidValue;
    }
    return hipGetLastError();
}

}  // namespace g4
