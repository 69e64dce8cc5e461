// k_paged_append.hip -- rows into and out of the paged KV cache: the rotation of
// queries and keys (model.c:359-367 over positions of a batch of sequences), the
// store of keys and values as f16 (RNE) or q8_0 / q4_0 blocks (model.c:583-589)
// in the pages' layout, and the way back.
//
// Bound by memory (8 bytes per query element, 4 + the row's type per key and
// value element) and, for a few tokens, by one dependent chain: the token's
// sequence, its length, its page.  A workgroup takes whole tokens: the angles of
// a token are computed once, into LDS, for all of its heads.  One token of 8 q / 4
// kv heads of 256: 2.8 us, a launch; 3800 of them in three prompts: 27.4 us, 4.0
// TB/s (a large copy reaches 4.8).
#include "paged.h"
#include "steps.h"

namespace g4 {

namespace {

__device__ __forceinline__ float4 pp_ld4(const float *p, bool al) {
    if (al) return *(const float4 *)p;
    return make_float4(p[0], p[1], p[2], p[3]);
}

// (cos, sin) of the pair of element e, the element of the pair's other half, and
// whether e is the pair's second one
struct PpPair {
    int i, other;
    bool second, turns;
};
__device__ __forceinline__ PpPair pp_pair(const PagedRope &r, int e) {
    PpPair x;
    x.turns = e < r.n_rot;
    const int half = r.n_rot >> 1;
    x.second = r.interleaved ? e & 1 : e >= half;
    x.i = r.interleaved ? e >> 1 : x.second ? e - half : e;
    x.other = r.interleaved ? e ^ 1 : x.second ? e - half : e + half;
    return x;
}
__device__ __forceinline__ float pp_turn(float v, float o, float cs, float sn, bool second) {
    // (a cos - b sin, b cos + a sin): o is b, or a
    return second ? __builtin_fmaf(o, sn, v * cs) : __builtin_fmaf(-o, sn, v * cs);
}

// HD elements of one row in 4-element groups.  Lane li of a row's LPR lanes
// holds group li (+ LPR).  In natural order group k is elements 4 k ..; in value
// order (quantized value rows, e = 16 m + c) it is elements 16 (4 m' + j) + c of
// c = k % 16, m' = k / 16, the four that share a dword or two bytes of the row.
template <int HD, int KVT>
__global__ __launch_bounds__(256) void k_paged_append(PagedAppend a) {
    constexpr int LPR = HD / 4 < 64 ? HD / 4 : 64, GPL = HD / 4 / LPR, RPW = 64 / LPR;   // lanes a row, groups a lane, rows a wave
    __shared__ float2 cs[HD / 2];
    const PagedPool &p = a.p;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, li = lane % LPR;
    const int half = a.r.n_rot >> 1, total = a.n_head + 2 * p.n_kv;
    const int row0 = blockIdx.y * a.rows, row1 = min(row0 + a.rows, total);
    double turns = 0.0;                              // a position's angle in turns, of pair threadIdx.x
    if ((int)threadIdx.x < half) {
        turns = exp2(-2.0 * threadIdx.x / a.r.n_rot * a.r.log2_base) * 0.15915494309189535;
        if (a.r.factor) turns /= (double)a.r.factor[threadIdx.x];
    }
    for (int t = blockIdx.x * a.tokens; t < min((blockIdx.x + 1) * a.tokens, (unsigned)a.b.n_tok); t++) {
        const int seq = paged_find(a.b, t);
        if (seq >= a.b.n_seq) return;                // behind the last sequence, as all later tokens
        const PagedSeq sq = paged_seq(p, a.b, seq);
        const int own = sq.len - sq.nq + (t - sq.t0);
        if (sq.bad || t < sq.t0 || t >= sq.t0 + sq.nq) {
            if (threadIdx.x == 0 && !paged_before(sq, seq, t)) paged_flag(p, PAGED_BAD_BATCH);
            continue;
        }
        if (own < 0) continue;
        const int ent = paged_entry(p, own >> 4), slot = own - ent * p.page;
        const int id = paged_ld(a.b.table, (int64_t)seq * a.b.table_stride + ent);
        const bool stored = (uint64_t)(int64_t)id < (uint64_t)p.n_pages;
        if (!stored && threadIdx.x == 0) paged_flag(p, PAGED_BAD_PAGE);
        if (half) {
            __syncthreads();                         // the previous token's angles are used
            if ((int)threadIdx.x < half) {
                const double x = turns * (double)((int64_t)a.b.n_prefix + own);
                const float f = (float)(2.0 * (x - rint(x)));
                float sn, cn;
                sincospif(f, &sn, &cn);
                cs[threadIdx.x] = make_float2(cn, sn);
            }
            __syncthreads();
        }
        for (int r0 = row0 + wave * RPW; r0 < row1; r0 += 4 * RPW) {
            const int row = r0 + lane / LPR;
            if (row >= row1) continue;
            const bool isq = row < a.n_head, isk = !isq && row < a.n_head + p.n_kv;
            const int h = isq ? row : isk ? row - a.n_head : row - a.n_head - p.n_kv;
            const float *src = (isq ? a.q + (size_t)t * a.qs : isk ? a.k + (size_t)t * a.ks : a.v + (size_t)t * a.vs) + (size_t)h * HD;
            const bool al = (((uintptr_t)src) & 15) == 0;
            const bool vorder = KVT != F16 && !isq && !isk;
            float v[GPL][4];
#pragma unroll
            for (int n = 0; n < GPL; n++) {
                const int k = li + n * LPR;
                if (vorder) {
#pragma unroll
                    for (int j = 0; j < 4; j++) v[n][j] = src[16 * (4 * (k >> 4) + j) + (k & 15)];
                } else {
                    const float4 x = pp_ld4(src + 4 * k, al);
                    v[n][0] = x.x; v[n][1] = x.y; v[n][2] = x.z; v[n][3] = x.w;
                }
            }
            if ((isq || isk) && half) {
                float w[GPL][4];
#pragma unroll
                for (int n = 0; n < GPL; n++) {
                    const int e = 4 * (li + n * LPR);
                    if (e >= a.r.n_rot) continue;
                    if (a.r.interleaved) {
#pragma unroll
                        for (int j = 0; j < 4; j++) w[n][j] = v[n][j ^ 1];
                    } else {
                        const float4 x = pp_ld4(src + pp_pair(a.r, e).other, al);
                        w[n][0] = x.x; w[n][1] = x.y; w[n][2] = x.z; w[n][3] = x.w;
                    }
                }
#pragma unroll
                for (int n = 0; n < GPL; n++) {
                    const int e = 4 * (li + n * LPR);
                    if (e >= a.r.n_rot) continue;
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        const PpPair x = pp_pair(a.r, e + j);
                        const float2 s = cs[x.i];
                        v[n][j] = pp_turn(v[n][j], w[n][j], s.x, s.y, x.second);
                    }
                }
            }
            if (isq) {
                float *dst = a.q_out + (size_t)t * a.qos + (size_t)h * HD;
                const bool da = (((uintptr_t)dst) & 15) == 0;
#pragma unroll
                for (int n = 0; n < GPL; n++) {
                    float *d = dst + 4 * (li + n * LPR);
                    if (da) *(float4 *)d = make_float4(v[n][0], v[n][1], v[n][2], v[n][3]);
                    else { d[0] = v[n][0]; d[1] = v[n][1]; d[2] = v[n][2]; d[3] = v[n][3]; }
                }
                continue;
            }
            uint8_t *page = (isk ? p.k : p.v) + (stored ? (size_t)id * p.page_bytes : 0);
            const uint32_t prow = (uint32_t)h * p.page + slot;
            uint8_t *dst = page + (size_t)prow * paged_row_bytes(KVT, HD);
            uint16_t *dsc = (uint16_t *)(page + p.sc_off + (size_t)prow * (HD / 16));
#pragma unroll
            for (int n = 0; n < GPL; n++) {
                const int k = li + n * LPR;
                if constexpr (KVT == F16) {
                    uint2 x;
                    x.x = f2h(v[n][0]) | ((uint32_t)f2h(v[n][1]) << 16);
                    x.y = f2h(v[n][2]) | ((uint32_t)f2h(v[n][3]) << 16);
                    if (stored) *(uint2 *)(dst + 8 * k) = x;
                } else if (isk) {
                    // block k / 8, its elements 4 (k % 8) ..: 8 lanes of the row
                    const int s = k >> 3, gq = (k & 7) >> 1, j0 = 4 * (k & 1);
                    if constexpr (KVT == Q8_0) {
                        uint16_t d16;
                        const uint32_t pk = q8_pack4(v[n], &d16) ^ 0x80808080u;
                        if (stored) {
                            *(uint32_t *)(dst + gq * (HD / 4) + 8 * s + j0) = pk;
                            if ((k & 7) == 0) dsc[s] = d16;
                        }
                    } else {
                        float ba = fabsf(v[n][0]), bv = v[n][0];
                        int be = 4 * k;
#pragma unroll
                        for (int j = 1; j < 4; j++)
                            if (fabsf(v[n][j]) > ba) { ba = fabsf(v[n][j]); bv = v[n][j]; be = 4 * k + j; }
#pragma unroll
                        for (int m = 1; m < 8; m <<= 1) {
                            const float oa = shfl_xor(ba, m), ov = shfl_xor(bv, m);
                            const int oe = shfl_xor(be, m);
                            if (oa > ba || (oa == ba && oe < be)) { ba = oa; bv = ov; be = oe; }
                        }
                        const float d = bv * -0.125f, id4 = d != 0.0f ? 1.0f / d : 0.0f;
                        uint32_t nib = 0;            // element j0 + j in nibble (j0 + j) / 2 + 4 (j & 1)
#pragma unroll
                        for (int j = 0; j < 4; j++)
                            nib |= (uint32_t)(min((int)__builtin_fmaf(v[n][j], id4, 8.5f), 15) & 15) << (4 * (((j0 + j) >> 1) + 4 * (j & 1)));
                        nib |= shfl_xor(nib, 1);
                        if (stored) {
                            if ((k & 1) == 0) *(uint32_t *)(dst + 4 * (gq * (HD / 32) + s)) = nib;
                            if ((k & 7) == 0) dsc[s] = f2h(d);
                        }
                    }
                } else {
                    // blocks 2 m' (elements j = 0, 1) and 2 m' + 1 (j = 2, 3) over the row's 16 lanes of one m'
                    const int c = k & 15, mq = k >> 4;
                    uint32_t pk = 0;
#pragma unroll
                    for (int half2 = 0; half2 < 2; half2++) {
                        const float x = v[n][2 * half2], y = v[n][2 * half2 + 1];
                        float d, id32;
                        if constexpr (KVT == Q8_0) {
                            const float am = group_max<16>(fmaxf(fabsf(x), fabsf(y)));
                            id32 = am != 0.0f ? 127.0f / am : 0.0f;
                            d = am * (1.0f / 127.0f);
                            pk |= (((uint32_t)(int)__builtin_rintf(x * id32) + 128) & 0xffu) << (16 * half2);
                            pk |= (((uint32_t)(int)__builtin_rintf(y * id32) + 128) & 0xffu) << (16 * half2 + 8);
                        } else {
                            float ba = fabsf(x), bv = x;
                            int be = c;
                            if (fabsf(y) > ba) { ba = fabsf(y); bv = y; be = 16 + c; }
#pragma unroll
                            for (int m = 1; m < 16; m <<= 1) {
                                const float oa = shfl_xor(ba, m), ov = shfl_xor(bv, m);
                                const int oe = shfl_xor(be, m);
                                if (oa > ba || (oa == ba && oe < be)) { ba = oa; bv = ov; be = oe; }
                            }
                            d = bv * -0.125f;
                            id32 = d != 0.0f ? 1.0f / d : 0.0f;
                            pk |= (uint32_t)(min((int)__builtin_fmaf(x, id32, 8.5f), 15) & 15) << (8 * half2);
                            pk |= (uint32_t)(min((int)__builtin_fmaf(y, id32, 8.5f), 15) & 15) << (8 * half2 + 4);
                        }
                        if (stored && c == 0) dsc[2 * mq + half2] = f2h(d);
                    }
                    if (stored) {
                        if constexpr (KVT == Q8_0) *(uint32_t *)(dst + c * (HD / 16) + 4 * mq) = pk;
                        else *(uint16_t *)(dst + c * (HD / 32) + 2 * mq) = (uint16_t)pk;
                    }
                }
            }
        }
    }
}

// One token, its rows' elements as values.  64 tokens of 8 heads of 128, 8 bits:
// 4.8 us with one element a thread and one workgroup a token, now 3.1.
template <int HD, int KVT>
__global__ __launch_bounds__(256) void k_paged_read(PagedRead a) {
    const PagedPool &p = a.p;
    const int t = blockIdx.x, seq = paged_find(a.b, t);
    if (seq >= a.b.n_seq) return;
    const PagedSeq sq = paged_seq(p, a.b, seq);
    const int own = sq.len - sq.nq + (t - sq.t0);
    if (sq.bad || t < sq.t0 || t >= sq.t0 + sq.nq) {
        if (threadIdx.x == 0 && !paged_before(sq, seq, t)) paged_flag(p, PAGED_BAD_BATCH);
        return;
    }
    if (own < 0) return;
    const int ent = paged_entry(p, own >> 4), slot = own - ent * p.page;
    const int id = paged_ld(a.b.table, (int64_t)seq * a.b.table_stride + ent);
    if ((uint64_t)(int64_t)id >= (uint64_t)p.n_pages) {
        if (threadIdx.x == 0) paged_flag(p, PAGED_BAD_PAGE);
        return;
    }
    // 4 elements at a time: neighbours, or of a quantized value row the four 16 apart
    // that share a dword or two bytes (e = 16 m + c)
    for (int x = blockIdx.y * 256 + threadIdx.x; x < p.n_kv * (HD / 2); x += 256 * gridDim.y) {
        const bool key = x < p.n_kv * (HD / 4);
        void *out = key ? a.k_out : a.v_out;
        if (!out) continue;
        const int at = key ? x : x - p.n_kv * (HD / 4), h = at / (HD / 4), k = at % (HD / 4);
        const uint8_t *page = (key ? p.k : p.v) + (size_t)id * p.page_bytes;
        const uint32_t prow = (uint32_t)h * p.page + slot;
        const uint8_t *row = page + (size_t)prow * paged_row_bytes(KVT, HD);
        int e = 4 * k, step = 1;
        float v[4];
        if constexpr (KVT == F16) {
            const uint2 w = *(const uint2 *)(row + 8 * k);
            v[0] = h2f((uint16_t)w.x); v[1] = h2f((uint16_t)(w.x >> 16)); v[2] = h2f((uint16_t)w.y); v[3] = h2f((uint16_t)(w.y >> 16));
        } else {
            const uint16_t *sc = (const uint16_t *)(page + p.sc_off) + (size_t)prow * (HD / 32);
            int q[4];
            float d0, d1;                                    // of elements 0, 1 and 2, 3
            if (key) {
                const int s = e >> 5, g = (e & 31) >> 3, j = e & 4;
                const uint32_t w = *(const uint32_t *)(row + (KVT == Q8_0 ? g * (HD / 4) + 8 * s + j : 4 * (g * (HD / 32) + s)));
                d0 = d1 = h2f(sc[s]);
#pragma unroll
                for (int i = 0; i < 4; i++) q[i] = KVT == Q8_0 ? (int)(w >> (8 * i) & 255) : (int)(w >> (2 * j + 4 * (i >> 1) + 16 * (i & 1)) & 15);
            } else {
                const int c = k & 15, m = k >> 4 << 2, n = c * (HD / 16) + m;
                const uint32_t w = KVT == Q8_0 ? *(const uint32_t *)(row + n) : *(const uint16_t *)(row + n / 2), d = *(const uint32_t *)(sc + m / 2);
                d0 = h2f((uint16_t)d);
                d1 = h2f((uint16_t)(d >> 16));
                e = 16 * m + c;
                step = 16;
#pragma unroll
                for (int i = 0; i < 4; i++) q[i] = KVT == Q8_0 ? (int)(w >> (8 * i) & 255) : (int)(w >> (4 * i) & 15);
            }
#pragma unroll
            for (int i = 0; i < 4; i++) v[i] = (float)(q[i] - (KVT == Q8_0 ? 128 : 8)) * (i < 2 ? d0 : d1);
        }
        const size_t o = ((size_t)t * p.n_kv + h) * HD + e;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            if (a.f16) ((uint16_t *)out)[o + step * i] = f2h(v[i]);
            else ((float *)out)[o + step * i] = v[i];
        }
    }
}

template <template <int, int> class L, typename A>
hipError_t by_shape(const A &a, hipStream_t s) {
#define G4_HD(T)                                          \
    switch (a.p.hd) {                                     \
    case 64: return L<64, T>::go(a, s);                   \
    case 128: return L<128, T>::go(a, s);                 \
    case 256: return L<256, T>::go(a, s);                 \
    case 512: return L<512, T>::go(a, s);                 \
    }                                                     \
    return hipErrorInvalidValue;
    if (a.p.type == F16) { G4_HD(F16) }
    if (a.p.type == Q8_0) { G4_HD(Q8_0) }
    G4_HD(Q4_0)
#undef G4_HD
}
template <int HD, int KVT>
struct Append {
    static hipError_t go(PagedAppend a, hipStream_t s) {
        // a workgroup's step covers 4 waves of rows.  Few tokens: one step per
        // workgroup, every row's loads in flight at once.  From 1024 workgroups
        // on, all rows of a token (its angles computed once), and several tokens.
        const int total = a.n_head + 2 * a.p.n_kv, step = 4 * (HD / 4 < 64 ? 256 / HD : 1);
        const int64_t steps = (total + step - 1) / step;
        a.rows = (int64_t)a.b.n_tok * steps <= 1024 ? step : total;
        a.tokens = a.rows == total ? std::max(1, std::min(4, a.b.n_tok / 2048)) : 1;
        const dim3 grid((a.b.n_tok + a.tokens - 1) / a.tokens, (total + a.rows - 1) / a.rows);
        hipLaunchKernelGGL((k_paged_append<HD, KVT>), grid, dim3(256), 0, s, a);
        return hipGetLastError();
    }
};
template <int HD, int KVT>
struct Read {
    static hipError_t go(const PagedRead &a, hipStream_t s) {
        const int64_t steps = (a.p.n_kv * (HD / 2) + 255) / 256;
        const dim3 grid(a.b.n_tok, a.b.n_tok * steps <= 1024 ? (unsigned)steps : 1);         // few tokens: every row's loads at once
        hipLaunchKernelGGL((k_paged_read<HD, KVT>), grid, dim3(256), 0, s, a);
        return hipGetLastError();
    }
};

}  // namespace

hipError_t launch_paged_append(const PagedAppend &a, hipStream_t s) {
    if (a.b.n_tok == 0 || a.b.n_seq == 0) return hipSuccess;
    return by_shape<Append>(a, s);
}
hipError_t launch_paged_read(const PagedRead &a, hipStream_t s) {
    if (a.b.n_tok == 0 || a.b.n_seq == 0) return hipSuccess;
    return by_shape<Read>(a, s);
}

}  // namespace g4
