// paged_tree.h -- attention of a tree's tokens over the paged KV cache
// (paged_attn.h): drafts of more than a token or two.
//
// Bound by the cache's bytes where sequences are long: a few rows of each have to be
// served as fast as its K and V arrive.  Pages go straight to LDS, as they are, into
// a ring of slots that the loads of the next positions are always filling.  A wave
// takes 16 rows and makes its operands from LDS, as k_paged_few from registers.
// Where a tile has fewer rows than the waves could take, the others take the same
// rows over other positions: a workgroup's 8 waves (heads of 256 and 512: 4 pairs and
// 2 fours, each wave with 128 of the elements, their scores added through LDS) are
// 1, 2, 4 or 8 row groups times as many position groups as are left, as the tile's
// rows need, so that drafts of all sizes share a call.  The position groups' sums are
// joined at a piece's end.  (A kernel with k_paged_few's register loads for more row
// groups took 91 us for 16 drafts of up to 16 tokens over 8192 positions, 32 / 8 heads
// of 128, f16; this one 67: 3.8 TB/s of pages in the call, 5.5 in its steps.  Two row
// groups a wave, one operand for both, halve the LDS traffic and the conversions of
// quantized rows, but a wave then starts and ends with twice the state: 82 us there.)
//
// Quantized rows are VALU work first (operands from integers, scales, splits), and no one
// limit: 32 drafts of up to 33 tokens over 4096 positions, 8 / 4 heads of 256, 8 bits,
// capped, take 90 us, their bytes 30.  The VALU issues in 55 % of the SIMDs' time there,
// the matrix cores are busy in 12 %, and the waves, two a SIMD with a barrier a step,
// wait 45 % of theirs.  (Without a cap 87; where the scores reach the cap, 97.)
#pragma once

#include <algorithm>
#include <type_traits>

#include "paged_few.h"
#include "paged_many.h"

namespace g4 {

// 16 (4) bytes of each lane to LDS, lane after lane from byte `lds` on.  No register
// is written, so nothing of it is the compiler's to wait for: who reads the bytes waits by
// count (pt_wait) and, for other waves' loads, at a barrier.  The compiler's own waits
// for its loads count these too and only wait longer.
__device__ __forceinline__ void pt_async16(const uint8_t *from, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off" ::"v"(from), "s"(pa_uniform(lds)) : "memory");
}
__device__ __forceinline__ void pt_async4(const int *from, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dword %0, off" ::"v"(from), "s"(pa_uniform(lds)) : "memory");
}
// until at most N of the wave's loads are under way
template <int N>
__device__ __forceinline__ void pt_wait() {
    static_assert(N < 64, "six bits");
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}
__device__ __forceinline__ uint32_t pt_lds(const void *p) { return (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) uint8_t *)p; }

// A slot: of each of TILES tiles of 32 positions the K rows, the V rows, then
// (quantized) their scales, K's and V's, all in order.  Within a row the 16-byte
// chunks are moved about by the row (chunk ^ key or value), so that the lanes that read
// one chunk of 16 rows, or 32 bytes of 4 rows (f16 V, read transposed), meet in no bank.
template <int HD, int KVT, bool WIDE>
struct PtShape {
    static constexpr int HE = HD <= 128 ? HD : WIDE ? 256 : 128, ES = HD / HE, ZW = 8 / ES;
    static constexpr int RB = paged_row_bytes(KVT, HD), CPR = RB / 16, WIN = RB < 256 ? 256 / RB : 1, FM = (CPR < 16 ? CPR : 16) - 1;
    static constexpr int SCB = KVT == F16 ? 0 : HD / 16;                                 // scale bytes of a row
    static constexpr int TILE = 64 * RB + 64 * SCB, TILES = HD <= 128 ? 4 : HD == 256 && KVT != F16 ? 2 : 1, SLOT = TILES * TILE;
    static constexpr int DEPTH = std::max(2, std::min(6, (ES > 1 ? 112 : 132) * 1024 / SLOT));        // slots
    static constexpr int LOADS = 2 * (RB / 32) * TILES, PER = LOADS >= 8 ? LOADS / 8 : 1;            // of 1 KB, K and V; a wave's
    static constexpr int SLOADS = KVT == F16 ? 0 : TILES * (HD == 512 ? 2 : 1);          // of scales, the last waves'
    static constexpr int TRB = 8 * PM_TR * 4, BP = HE + 4;
    static constexpr size_t RING = (size_t)DEPTH * SLOT, TRAT = SLOT >= TRB ? (size_t)(DEPTH - 1) * SLOT : RING, OB = (size_t)8 * 16 * BP * 4;
    static constexpr size_t LDS = std::max(std::max(RING, TRAT + TRB), OB);
    __device__ static __forceinline__ int key(int row) { return row / WIN & FM; }
    __device__ static __forceinline__ int value(int row) { return KVT == F16 ? 2 * (row / WIN) & FM : 0; }
};

// The wave's loads of the tiles whose units are lanes l0 .. of us.
template <typename S, int HD, int KVT>
__device__ __forceinline__ void pt_load(const PagedPool &p, const PaUnits &us, int l0, uint32_t slot, int wave, int lane) {
    constexpr int T = S::RB / 32;
    uintptr_t pk = (uintptr_t)p.k, pv = (uintptr_t)p.v;      // chosen between by value, not by place
    asm volatile("" : "+s"(pk), "+s"(pv));
#pragma unroll
    for (int n = 0; n < S::PER; n++) {
        const int idx = wave + 8 * n;
        if (S::LOADS < 8 && idx >= S::LOADS) break;
        const int q = idx / (2 * T), r = idx % (2 * T), w = r % T;
        const bool value = r >= T;
        const int i = 64 * w + lane, row = i / S::CPR, chunk = i % S::CPR ^ (value ? S::value(row) : S::key(row));
        size_t unit;
        if constexpr (S::RB >= 64) unit = pa_unit<HD, KVT>(p, us, l0 + 2 * q + pa_uniform(row >> 4)).row;
        else {
            const size_t u0 = pa_unit<HD, KVT>(p, us, l0 + 2 * q).row, u1 = pa_unit<HD, KVT>(p, us, l0 + 2 * q + 1).row;
            unit = row < 16 ? u0 : u1;
        }
        pt_async16((const uint8_t *)(value ? pv : pk) + unit + (uint32_t)((row & 15) * S::RB + 16 * chunk), slot + q * S::TILE + (value ? 32 * S::RB : 0) + 1024 * w);
    }
    if constexpr (S::SLOADS > 0) {
        if (wave >= 8 - S::SLOADS) {
            const int idx = 7 - wave, q = HD == 512 ? idx >> 1 : idx, part = HD == 512 ? idx & 1 : 0;
            const int at = 1024 * part + 16 * lane, seg = at / HD;                       // K's two units, V's two
            if (seg < 4) {
                const size_t s0 = pa_unit<HD, KVT>(p, us, l0 + 2 * q).sc, s1 = pa_unit<HD, KVT>(p, us, l0 + 2 * q + 1).sc;
                const uint8_t *const k = p.k + (seg & 1 ? s1 : s0), *const v = p.v + (seg & 1 ? s1 : s0);
                pt_async16((seg < 2 ? k : v) + at % HD, slot + q * S::TILE + 64 * S::RB + 1024 * part);
            }
        }
    }
}
// until the wave's loads of all but the last BEHIND slots are there
template <typename S, int BEHIND>
__device__ __forceinline__ void pt_arrived(int wave) {
    const bool kv = S::LOADS >= 8 || wave < S::LOADS, sc = S::SLOADS > 0 && wave >= 8 - S::SLOADS;
    if (kv && sc) pt_wait<BEHIND *(S::PER + 1)>();
    else if (kv) pt_wait<BEHIND * S::PER>();
    else if (sc) pt_wait<BEHIND>();
    else pt_wait<0>();                                       // page ids at most
}

constexpr int PT_BITS = 512;                     // words of a tile's masks kept in LDS

template <int HD, int KVT, bool WIDE>
__global__ __launch_bounds__(PM_THREADS, 2) void k_paged_tree(PagedCall call) {
    using S = PtShape<HD, KVT, WIDE>;
    constexpr int PG = S::TILES, HE = S::HE, ES = S::ES, ZW = S::ZW, NS = HE / 32, NM = HE / 16, RB = S::RB, BP = S::BP, TURN = 32 / PG;   // TURN: iterations of 64 units
    constexpr int AHEAD = HE == 64 ? 2 : 4;
    __shared__ __align__(16) uint8_t lds[S::LDS];            // the ring; before it, where it is filled last, queries on their way; after it sums
    __shared__ __align__(16) float xs[ES > 1 ? 8 : 1][ES > 1 ? PG : 1][ES > 1 ? 64 : 1][8];      // partial scores of the waves of one tile
    __shared__ __align__(16) float ex[KVT == F16 ? 1 : 8][ES > 1 ? PG : 1][32];            // of a wave and tile: pa_exponent of its positions' largest V scales
    __shared__ int ids[8][64];                               // of a wave: the next page ids
    __shared__ float2 wml[8][16];
    __shared__ uint32_t bits[PT_BITS];                       // the tile's masks
    __shared__ float part[8][16];                            // at the end: each wave's factor of its rows
    __shared__ float *dst[16 * ZW];                          // and where the rows go
    float *const buf = (float *)lds;

    // Workgroups of one XCD (every eighth) take neighbouring shares: row tiles
    // that read the same K and V find them in its L2.
    const int per = (call.pl.many.wgs + 7) >> 3, wg = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
    int mine, n_seq;
    const int total = pa_total<true, true>(call.a, call.pl, mine, n_seq), share = pa_tree_share(call.a, call.pl, total, n_seq);
    const int first = wg * share, stop = wg < call.pl.many.wgs ? min(first + share, total) : 0;
    if (blockIdx.x == 0) pa_rest(call.a, call.pl, n_seq);
    PaFind from;
    for (int u = first; u < stop;) {
        const PagedCall call = pa_fresh<true>();
        const PagedAttn &a = call.a;
        const PagedPlan &pl = call.pl;
        const PagedPool &p = a.p;
        const PagedBatch &b = a.b;
        const int tid = pa_thread(), lane = tid & 63, wave = pa_uniform(tid >> 6), c = lane & 15, g = lane >> 4, ew = wave % ES, z = wave / ES;
        const int G = a.grp, R = pl.many.rows;
        float *const tr = (float *)(lds + S::TRAT) + wave * PM_TR;
        const float capl = a.cap * 1.4426950408889634f;
        const PaPiece x = pa_piece<true, true>(a, pl, mine, n_seq, from, wg, u, first, stop);
        u += x.took;
        if (x.n == 0) continue;                              // the share ends in a tile's lead, or begins behind a last step
        const PagedSeq &sq = x.sq;
        const int kvh = x.kvh, hi0 = x.hi0, lo0 = x.lo0, lo1 = x.lo1, start = x.start, end = x.end, rows = min(sq.nq * G, (x.tile + 1) * R);     // the tile's rows end at `rows`
        // row groups: a power of two that the tile's rows need; position groups: the rest
        const int need = (rows - x.tile * R + 15) >> 4, rgl = need <= 1 ? 0 : 32 - __builtin_clz(need - 1), rw = z & ((1 << rgl) - 1), pg = z >> rgl;
        const int groups = min(ZW >> rgl, PG), turns = PG / groups;          // position groups (other waves have none); tiles of a slot for each: of heads of 256 and 512 one or two
        bool bad = sq.bad;
        if (bad && tid == 0) paged_flag(p, PAGED_BAD_BATCH);
        const int last = (x.seglen - 1) >> 4, iters = end > start ? (end - start + 32 * PG - 1) / (32 * PG) : 0;
        const bool tree = !x.pre;
        const int full = tree ? hi0 - 1 : hi0;               // the last position that all rows attend, windows apart

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
        // busy: the wave has rows; the lane's: r0 + c
        const bool busy = r0 < rows && pg < groups, ok = r0 + c < rows;
        const int ri = ok ? (r0 + c) / G : 0, tok = sq.t0 + ri;
        // it attends cached positions [rlo, full], and new tokens of its mask, from position hi0 on
        const int tok0 = x.tile * pl.many.toks, words = a.words, held = min(sq.nq - tok0, pl.many.toks) * words;
        const bool in_lds = tree && held <= PT_BITS;         // the tile's masks
        int rlo = lo0;
        const uint32_t *mask = nullptr;
        if (ok) {
            if (tree) {
                if (hi0 + ri >= 0) mask = in_lds ? bits + (ri - tok0) * words : a.mask + (size_t)tok * words;
                rlo = a.window ? max(0, hi0 + paged_depth(a.depth[tok], sq.nq) + 1 - a.window) : 0;
            } else if (a.window) {
                rlo = max(0, pa_token_pos(p, b, n_seq, tok, a.depth) + 1 - a.window);
            }
        }
        auto row_bits = [&](int pos) { return mask ? pa_bits(mask, words, pos - hi0) : 0u; };
        auto row_hits = [&](uint64_t out, int unit) { return out ? pa_tree_hits(out, unit, 2, x.seglen, rlo, full, row_bits) : false; };
        uint32_t my_bits = 0;
        if (in_lds && tid < held) my_bits = a.mask[(size_t)(sq.t0 + tok0) * words + tid];

        PaUnits us = {0, 0};                                 // 64 units; their successors' ids in ids[wave]
        uint64_t outside = 0;
        if (iters) {
            us = pa_units(p, x.table, start >> 4, 2, last, kvh);
            outside = pa_check(p, us);
        }
        // The masks before the barrier: the previous piece has met behind its last look at its
        // own, and this one's are there for all waves from the first units' check on.
        if (in_lds && tid < held) bits[tid] = my_bits;
        __syncthreads();                                     // the previous piece's sums are used
        // The queries, older than the page ids, are here too: said now, as a wait of the
        // compiler's for them behind the loads below would be for those as well.
#pragma unroll
        for (int s = 0; s < NS; s++)
#pragma unroll
            for (int k = 0; k < 2; k++) asm volatile("" : "+v"(y[s][k]));
        issue_order();
        // the ids of the 64 units from `unit` on, on their way
        auto ask = [&](int unit) { pt_async4(x.table + paged_entry(p, min(unit + lane, last)), pt_lds(ids[wave])); };
        const uint32_t ring = pt_lds(lds);
        int to = 0;                                          // the slot filled next
        auto load = [&](int it) {
            pt_load<S, HD, KVT>(p, us, 2 * PG * (it & (TURN - 1)), ring + to * S::SLOT, wave, lane);
            to = to + 1 == S::DEPTH ? 0 : to + 1;
        };
        if (iters > TURN) ask((start >> 4) + 64);
#pragma unroll
        for (int k = 0; k + 1 < S::DEPTH; k++)
            if (k < iters) load(k);
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
            if constexpr (ES > 1) {                          // over all parts of the elements
                __syncthreads();
#pragma unroll
                for (int k = 1; k < ES; k++) mx = fmaxf(mx, ((float *)(lds + S::TRAT) + (wave ^ k) * PM_TR)[c * PM_COLS]);
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
        bad |= row_hits(outside, start >> 4);
        pa_v4f o[NM];
        float m = -__builtin_inff(), l = 0.0f;
#pragma unroll
        for (int e = 0; e < NM; e++) o[e] = pa_v4f{0.0f, 0.0f, 0.0f, 0.0f};

        // the lane's places in a tile: K rows c and 16 + c, V rows (f16) 4 g + c / 4 and 16 more
        const uint32_t kc = S::key(c), vr = 4 * g + (c >> 2);
        int at = 0;                                          // the slot of this iteration
        for (int it = 0; it < iters; it++) {
            const uint8_t *const slot = lds + at * S::SLOT;
            at = at + 1 == S::DEPTH ? 0 : at + 1;
            // This iteration's bytes: the wave's own by count, the others' at the barrier,
            // behind which the slot of the iteration before is free.
            if (it + S::DEPTH - 1 <= iters) pt_arrived<S, S::DEPTH - 2>(wave);
            else pt_wait<0>();
            lds_barrier();
            const int far = it + S::DEPTH - 1;
            if (far < iters) {
                if ((far & (TURN - 1)) == 0) {
                    const int un = (start >> 4) + 2 * PG * far, unit = min(un + lane, last);
                    us.id = ids[wave][lane];                 // asked for TURN iterations ago
                    us.row = kvh * p.page + (unit - paged_entry(p, unit) * p.units) * 16;
                    bad |= row_hits(pa_check(p, us), un);
                    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
                    if (far + TURN < iters) ask(un + 64);
                }
                load(far);
            }
            if (!busy) {                                     // waves that share scores all meet
                if constexpr (ES > 1) lds_barrier();
                continue;
            }
            // NT tiles at once, q, q + groups: one exchange of scores and one maximum for both
            // (heads of 64 and 128 exchange none, and two at once spill: 113 us for 69)
            auto step = [&](auto nt, int q) {
                constexpr int NT = decltype(nt)::value, DW = HE / 64;        // DW: dwords of a row's scales
                const int base0 = start + 32 * (PG * it + q);
                const uint8_t *const d0 = slot + q * S::TILE;
                auto base_of = [&](int t) { return base0 + 32 * groups * t; };
                auto tile_of = [&](int t) { return d0 + t * groups * S::TILE; };
                const bool edge = base_of(NT - 1) + 31 > full || base0 < lo1 || base_of(NT - 1) + 32 > end;
                uint32_t att[NT];                            // which of these positions the row attends
#pragma unroll
                for (int t = 0; t < NT; t++)
                    att[t] = edge ? pa_tree_seen(base_of(t), rlo, full, base_of(t) + 31 >= hi0 ? row_bits(base_of(t)) : 0u, end) : ~0u;
                auto seen = [&](int t, int k) { return (att[t] >> k & 1) != 0; };        // position k of tile t
                // scores of row c at positions pm_pos(g, j)
                pa_v4f sc[NT][2];
#pragma unroll
                for (int t = 0; t < NT; t++) {
                    const uint8_t *const d = tile_of(t);
                    sc[t][0] = sc[t][1] = pa_v4f{0.0f, 0.0f, 0.0f, 0.0f};
                    if constexpr (KVT == F16) {
                        pa_v4f s2[2] = {{0.0f, 0.0f, 0.0f, 0.0f}, {0.0f, 0.0f, 0.0f, 0.0f}};
                        const uint8_t *const kr = d + c * RB + HE * 2 * ew;
                        const uint32_t k0 = 16 * (g ^ kc);
                        // high and low halves apart, so that no instruction waits for the one before it
                        pm_pipeline<2 * NS, AHEAD>([&](int i) { return *(const pa_v8h *)(kr + (i & 1) * 16 * RB + (k0 ^ (64 * (i >> 1)))); }, [&](int i, pa_v8h ko) {
                            sc[t][i & 1] = pa_mma(ko, q0[i >> 1], sc[t][i & 1]);
                            s2[i & 1] = pa_mma(ko, q1[i >> 1], s2[i & 1]);
                        });
                        sc[t][0] += s2[0];
                        sc[t][1] += s2[1];
                    } else {
                        // the lane's runs, as k_paged_few's
                        constexpr int KW = PaTile<HE, KVT>::KW;
                        PaTile<HE, KVT> kv;
                        uint32_t dk[8][DW];
#pragma unroll
                        for (int h = 0; h < 2; h++) {
                            const uint8_t *const kr = d + (16 * h + c) * RB;
                            const uint32_t byte = 4 * KW * ((HD / HE) * g + ew);
                            if constexpr (KW >= 4) {
#pragma unroll
                                for (int k = 0; k < KW / 4; k++) pa_load<4>(kv.k[h] + 4 * k, kr + 16 * ((byte / 16 + k) ^ kc));
                            } else pa_load<KW>(kv.k[h], kr + 16 * (byte / 16 ^ kc) + byte % 16);
                        }
                        const uint8_t *const sp = d + 64 * RB + HE / 16 * ew;
#pragma unroll
                        for (int j = 0; j < 8; j++) pa_load<DW>(dk[j], sp + pm_pos(g, j) * S::SCB);
                        // the largest V scale of each position, as an exponent: a position a lane
                        if (lane < 32) {
                            uint32_t w[DW], top = 0;
                            pa_load<DW>(w, sp + (32 + lane) * S::SCB);
#pragma unroll
                            for (int k = 0; k < DW; k++) top = pa_pkmax(top, w[k] & 0x7fff7fffu);
                            ex[wave][t][lane] = pa_exponent(max(top << 16, top), 1);
                        }
                        asm volatile("" ::: "memory");       // a wave's LDS accesses complete in order
#pragma unroll
                        for (int s = 0; s < NS; s++)
#pragma unroll
                            for (int h = 0; h < 2; h++) {
                                const pa_v8h ko = pa_key<HE, KVT>(kv, h, s);
                                const pa_v4f y = pa_mma(ko, q1[s], pa_mma(ko, q0[s], pa_v4f{0.0f, 0.0f, 0.0f, 0.0f}));
#pragma unroll
                                for (int i = 0; i < 4; i++) sc[t][h][i] = __builtin_fmaf(pa_scale(dk[4 * h + i], s), y[i], sc[t][h][i]);
                            }
                    }
                }
                if constexpr (ES > 1) {
#pragma unroll
                    for (int t = 0; t < NT; t++) {
                        *(pa_v4f *)xs[wave][t][lane] = sc[t][0];
                        *(pa_v4f *)(xs[wave][t][lane] + 4) = sc[t][1];
                    }
                    lds_barrier();
                    const int w0 = wave & ~(ES - 1);         // in one order for all of them
#pragma unroll
                    for (int t = 0; t < NT; t++) {
                        sc[t][0] = *(const pa_v4f *)xs[w0][t][lane];
                        sc[t][1] = *(const pa_v4f *)(xs[w0][t][lane] + 4);
#pragma unroll
                        for (int k = 1; k < ES; k++) {
                            sc[t][0] += *(const pa_v4f *)xs[w0 + k][t][lane];
                            sc[t][1] += *(const pa_v4f *)(xs[w0 + k][t][lane] + 4);
                        }
                    }
                }
                float w[NT][8], mt = -__builtin_inff();
                uint32_t live[NT];                           // bit j: the row attends position j
#pragma unroll
                for (int t = 0; t < NT; t++) {
#pragma unroll
                    for (int j = 0; j < 8; j++) w[t][j] = sc[t][j >> 2][j & 3] * qs;
                    if (a.cap > 0.0f) {
                        pa_tanh(w[t]);
#pragma unroll
                        for (int j = 0; j < 8; j++) w[t][j] *= capl;
                    }
                    // (positions pm_pos(g, j): 4 g .. 4 g + 3 and 16 further)
                    live[t] = (att[t] >> (4 * g) & 15) | (att[t] >> (4 * g + 12) & 240);
                    if (edge) {
#pragma unroll
                        for (int j = 0; j < 8; j++) w[t][j] = live[t] >> j & 1 ? w[t][j] : -__builtin_inff();
                    }
                    if constexpr (KVT == F16) {
#pragma unroll
                        for (int j = 0; j < 8; j++) mt = fmaxf(mt, w[t][j]);
                    } else {
                        // + the exponent of the position's largest value scale
                        const pa_v4f e[2] = {*(const pa_v4f *)&ex[wave][t][4 * g], *(const pa_v4f *)&ex[wave][t][16 + 4 * g]};
#pragma unroll
                        for (int j = 0; j < 8; j++) mt = fmaxf(mt, w[t][j] + e[j >> 2][j & 3]);
                    }
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
                for (int t = 0; t < NT; t++)
#pragma unroll
                    for (int j = 0; j < 8; j++) {
                        w[t][j] = __builtin_amdgcn_exp2f(w[t][j] - mr);
                        l += w[t][j];
                    }
#pragma unroll
                for (int t = 0; t < NT; t++) {
                    const uint8_t *const d = tile_of(t);
                    if constexpr (KVT == F16) {
                        uint32_t hi[4], lo[4];
#pragma unroll
                        for (int k = 0; k < 4; k++) pa_split(w[t][2 * k], w[t][2 * k + 1], hi[k], lo[k]);
                        const pa_v8h b0 = pa_op(hi[0], hi[1], hi[2], hi[3]), b1 = pa_op(lo[0], lo[1], lo[2], lo[3]);
                        const uint8_t *const vt = d + (32 + vr) * RB + HE * 2 * ew + 8 * (c & 1);
                        const uint32_t v0 = 16 * ((c & 3) >> 1 ^ S::value(vr));
                        // 16 lanes give 4 positions of 16 elements and get 4 positions of their own
                        auto turned = [&](int e) { return pm_turned((const _Float16 *)(vt + (v0 ^ (32 * e))), (const _Float16 *)(vt + 16 * RB + (v0 ^ (32 * e)))); };
                        if (edge) {
                            // Positions that no row of the tile attends may hold anything: zeros
                            // for them.  Non-finite values that some rows attend and some do not
                            // are taken out and added to those that do (rare, one by one).
                            uint32_t mask4[4], nf = 0;
#pragma unroll
                            for (int k = 0; k < 4; k++) {
                                const int pos = base_of(t) + pm_pos(g, 2 * k);
                                mask4[k] = (pos >= lo0 && pos < end ? 0xffffu : 0u) | (pos + 1 >= lo0 && pos + 1 < end ? 0xffff0000u : 0u);
                            }
#pragma unroll
                            for (int e = 0; e < NM; e++) {
                                pa_v4u va = __builtin_bit_cast(pa_v4u, turned(e));
#pragma unroll
                                for (int k = 0; k < 4; k++) {
                                    const uint32_t v = va[k] & mask4[k];
                                    nf |= (v & 0x7c007c00u) + 0x04000400u;               // bit 15 or 31 where an exponent is all ones
                                    va[k] = pa_finite(v);
                                }
                                const pa_v8h vo = __builtin_bit_cast(pa_v8h, va);
                                o[e] = pa_mma(vo, b0, o[e]);
                                o[e] = pa_mma(vo, b1, o[e]);
                            }
                            if (__any(nf & 0x80008000u)) {
                                for (int k = 0; k < 32; k++) {
                                    const int pos = base_of(t) + k;
                                    if (pos < lo0 || pos >= end) continue;
                                    const uint8_t *const row = d + (32 + k) * RB + HE * 2 * ew;
                                    const uint32_t f = S::value(k);
                                    float wx = 0.0f;
#pragma unroll
                                    for (int j = 0; j < 8; j++) {
                                        const float v = __shfl(w[t][j], 16 * ((k & 15) >> 2) + c, 64);
                                        if (j == 4 * (k >> 4) + (k & 3)) wx = v;
                                    }
                                    const bool sees = seen(t, k);
#pragma unroll
                                    for (int e = 0; e < NM; e++) {
                                        const uint2 hv = *(const uint2 *)(row + 16 * ((2 * e + (g >> 1)) ^ f) + 8 * (g & 1));
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
                            pa_v8h before;                   // low halves one operand later
                            pm_pipeline<NM, AHEAD>(turned, [&](int e, pa_v8h va) {
                                o[e] = pa_mma(va, b0, o[e]);
                                if (e) o[e - 1] = pa_mma(before, b1, o[e - 1]);
                                before = va;
                            });
                            o[NM - 1] = pa_mma(before, b1, o[NM - 1]);
                        }
                    } else {
                        constexpr int VW = PaTile<HE, KVT>::VW;
                        PaTile<HE, KVT> kv;
                        uint32_t dv[8][DW];
                        const uint8_t *const sp = d + 64 * RB + HE / 16 * ew;
#pragma unroll
                        for (int j = 0; j < 8; j++) {
                            const int pos = pm_pos(g, j);
                            const uint8_t *const row = d + (32 + pos) * RB;
                            if constexpr (KVT == Q4_0 && HE == 64) kv.v[j][0] = *(const uint16_t *)(row + 2 * c);
                            else pa_load<VW>(kv.v[j], row + 4 * VW * ((HD / HE) * c + ew));
                            pa_load<DW>(dv[j], sp + (32 + pos) * S::SCB);
                        }
                        // a scale of a position that the row does not attend may be anything
                        if (edge) {
#pragma unroll
                            for (int j = 0; j < 8; j++)
#pragma unroll
                                for (int k = 0; k < DW; k++) dv[j][k] = live[t] >> j & 1 ? dv[j][k] : 0u;
                        }
#pragma unroll
                        for (int s = 0; s < NS; s++) {       // blocks of 32 elements: value tiles 2 s, 2 s + 1
                            uint32_t hi[4], lo[4];
#pragma unroll
                            for (int k = 0; k < 4; k++)
                                pa_split(__builtin_fmaf(pa_scale(dv[2 * k], s), w[t][2 * k], 0.0f), __builtin_fmaf(pa_scale(dv[2 * k + 1], s), w[t][2 * k + 1], 0.0f), hi[k], lo[k]);
                            const pa_v8h b0 = pa_op(hi[0], hi[1], hi[2], hi[3]), b1 = pa_op(lo[0], lo[1], lo[2], lo[3]);
                            const pa_v8h x0 = pa_value<HE, KVT>(kv, 2 * s), x1 = pa_value<HE, KVT>(kv, 2 * s + 1);
                            o[2 * s] = pa_mma(x0, b0, o[2 * s]);
                            o[2 * s + 1] = pa_mma(x1, b0, o[2 * s + 1]);
                            o[2 * s] = pa_mma(x0, b1, o[2 * s]);
                            o[2 * s + 1] = pa_mma(x1, b1, o[2 * s + 1]);
                        }
                    }
                }
            };
            if constexpr (ES > 1 && PG > 1) {
                if (turns > 1) {
                    step(std::integral_constant<int, 2>(), pg & (groups - 1));
                    continue;
                }
            }
            for (int q = pg & (groups - 1); q < PG; q += groups)
                if (ES > 1 || start + 32 * (PG * it + q) < end) step(std::integral_constant<int, 1>(), q);
        }
        bad &= ok;
        if (__any(bad)) {
            if (lane == 0 && !sq.bad) paged_flag(p, PAGED_BAD_PAGE);
            if (bad) l = __builtin_nanf("");
        }
        l += partner<16>(l);
        l += partner<32>(l);
        // Out through LDS, the position groups' results joined in order.  A row a thread
        // finds its place meanwhile.
        constexpr float VS = KVT == Q8_0 ? 512.0f : 1.0f;
        const int r00 = x.tile * R, count = rows - r00;      // rows of the tile
        PaSink sink = {nullptr, nullptr, false};
        bool zero = false;
        if (tid < count) {
            const int i = (r00 + tid) / G, head = kvh * G + (r00 + tid - i * G), tok = sq.t0 + i;
            zero = tree && !sq.bad && pa_tree_nothing(a, sq, tok, in_lds ? bits + (i - tok0) * words : a.mask + (size_t)tok * words);
            sink = pa_sink<true, true>(a, pl, x, share, tid, tok, head, zero, true);
            dst[tid] = sink.o;
        }
        __syncthreads();                                     // the ring is used
        if (g == 0) wml[wave][c] = make_float2(m, l);
#pragma unroll
        for (int e = 0; e < NM; e++) *(pa_v4f *)&buf[(wave * 16 + c) * BP + 16 * e + 4 * g] = o[e];
        __syncthreads();
        // a row a thread: its waves' factors; then four elements a thread
        if (tid < count) {
            const int w0 = (tid >> 4) * ES, step = ES << rgl, cc = tid & 15;
            float mm = -__builtin_inff(), ls = 0.0f;
            for (int k = 0; k < groups; k++)
#pragma unroll
                for (int n = 0; n < ES; n++) mm = fmaxf(mm, wml[w0 + k * step + n][cc].x);
            auto factor = [&](int w) { const float v = wml[w][cc].x; return v == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(v - mm); };
            for (int k = 0; k < groups; k++) {
                const float v = wml[w0 + k * step][cc].y;
                ls += v == v ? factor(w0 + k * step) * v : v;            // a bad page's NaN stays
            }
            const float f = !sink.out ? VS : zero ? 0.0f : VS / ls;
            for (int k = 0; k < groups; k++)
#pragma unroll
                for (int n = 0; n < ES; n++) part[w0 + k * step + n][cc] = f * factor(w0 + k * step + n);
            if (!sink.out) *sink.ml = make_float2(mm, ls);
        }
        __syncthreads();
        for (int y = tid; y < count * (HD / 4); y += PM_THREADS) {
            const int r = y / (HD / 4), e4 = y % (HD / 4) * 4, ez = e4 / HE, w0 = (r >> 4) * ES + ez, step = ES << rgl;
            pa_v4f s = {0.0f, 0.0f, 0.0f, 0.0f};
            for (int k = 0; k < groups; k++) s += *(const pa_v4f *)&buf[((w0 + k * step) * 16 + (r & 15)) * BP + e4 - ez * HE] * part[w0 + k * step][r & 15];
            pa_store4(dst[r] + e4, s);
        }
    }
}


template <int KVT>
hipError_t pa_tree(const PagedAttn &a, const PagedPlan &pl, bool wide, hipStream_t s) {
    const dim3 grid((pl.many.wgs + 7) / 8 * 8), wg(PM_THREADS);
    switch (a.p.hd) {
    case 64: hipLaunchKernelGGL((k_paged_tree<64, KVT, false>), grid, wg, 0, s, PagedCall{a, pl}); break;
    case 128: hipLaunchKernelGGL((k_paged_tree<128, KVT, false>), grid, wg, 0, s, PagedCall{a, pl}); break;
    case 256:
        if (wide) hipLaunchKernelGGL((k_paged_tree<256, KVT, true>), grid, wg, 0, s, PagedCall{a, pl});
        else hipLaunchKernelGGL((k_paged_tree<256, KVT, false>), grid, wg, 0, s, PagedCall{a, pl});
        break;
    case 512:
        if (wide) hipLaunchKernelGGL((k_paged_tree<512, KVT, true>), grid, wg, 0, s, PagedCall{a, pl});
        else hipLaunchKernelGGL((k_paged_tree<512, KVT, false>), grid, wg, 0, s, PagedCall{a, pl});
        break;
    default: return hipErrorInvalidValue;
    }
    return hipGetLastError();
}

}  // namespace g4
