// k_paged_move.hip -- rows moved within the paged KV caches of a model's layers:
// the accepted rows of a draft moved together (g4h_paged_keep), and the beams that
// a selection kept given tables and pages of their own (g4h_paged_fork).
//
// Copies: bound by memory where there is much of it (each byte read and written
// once: 32 new beams' pages of 64 x 4 heads of 256 in 26 f16 caches, 257 MB in 46 us,
// 5.6 TB/s), else by a launch and a chain of dependent reads (offsets and lengths, page
// ids, rows: 4 beams in 26 caches 5.7 us; one accepted path 4.5, 32 of them in 8-bit
// caches 7.9).  One launch serves all layers' caches of one shape.
#include <algorithm>

#include "paged.h"

namespace g4 {

namespace {

typedef uint32_t pv_v4 __attribute__((ext_vector_type(4)));      // (arrays of HIP's uint4 end up in LDS or scratch)

// The rows of one sequence and one cache's keys or values: a thread carries the same
// 16 bytes (of quantized rows' scales: 4) of every kept row, so that the moves of a
// thread need only be in their own order.  Entries ascend and entry k is at least k:
// where row k goes, no later row comes from.
__global__ __launch_bounds__(256) void k_paged_keep(PagedKeep a, PagedPools pools) {
    const PagedPool &p = a.p;
    const int s = blockIdx.x >> 1, lane = threadIdx.x & 63;
    const bool value = blockIdx.x & 1;
    const PagedSeq q = paged_seq(p, a.b, s);
    const int n = paged_ld(a.n_keep, s), first = q.len - q.nq;
    const bool leader = threadIdx.x == 0 && !value && blockIdx.y == 0;
    if (q.bad || n < 0 || n > a.most || n > q.nq) {
        if (leader) paged_flag(p, PAGED_BAD_BATCH);
        return;
    }
    if (n == 0 || first < 0) return;
    const int *const keep = a.keep + (int64_t)s * a.most, *const table = a.b.table + (int64_t)s * a.b.table_stride;
    uint8_t *const pool = value ? pools.v[blockIdx.y] : pools.k[blockIdx.y];
    const int rb = paged_row_bytes(p.type, p.hd), wide = rb / 16, narrow = p.type == F16 ? 0 : p.hd / 64, cols = wide + narrow;
    int before = -1;                                         // the last entry of the 64 before
    for (int k0 = 0; k0 < n; k0 += 64) {
        // the lanes' moves: where row first + from goes to row first + k
        const int k = k0 + lane;
        const int from = k < n ? keep[k] : 0x7fffffff, prev = __shfl_up(from, 1, 64);
        const uint64_t wrong = __ballot(k < n && (from <= (lane ? prev : before) || from >= q.nq));
        const int count = min(wrong ? __ffsll((unsigned long long)wrong) - 1 : 64, n - k0);
        bool moves = lane < count && from != k;
        size_t src = 0, dst = 0;
        int src_row = 0, dst_row = 0;
        if (moves) {
            const int x = first + from, y = first + k, xe = paged_entry(p, x >> 4), ye = paged_entry(p, y >> 4), xi = table[xe], yi = table[ye];
            if ((uint64_t)(int64_t)xi >= (uint64_t)p.n_pages || (uint64_t)(int64_t)yi >= (uint64_t)p.n_pages) {
                moves = false;
                if (!value && blockIdx.y == 0) paged_flag(p, PAGED_BAD_PAGE);
            } else {
                src = (size_t)xi * p.page_bytes;
                dst = (size_t)yi * p.page_bytes;
                src_row = x - xe * p.page;
                dst_row = y - ye * p.page;
            }
        }
        const uint64_t todo = __ballot(moves);
        // whole waves: all lanes have to be there where one's move is read (in divergent code
        // the reads became a loop over lanes: 13.6 us, with this 7.9)
        for (int x0 = threadIdx.x & ~63; x0 < p.n_kv * cols; x0 += 256) {
            const int x = min(x0 + lane, p.n_kv * cols - 1);
            const bool live = x == x0 + lane;
            const int h = x / cols, c = x - h * cols, row = h * p.page;
            const bool sc = c >= wide;
            const size_t at = sc ? p.sc_off + (size_t)row * (p.hd / 16) + (c - wide) * 4 : (size_t)row * rb + c * 16;
            auto place = [&](int l, size_t page, int r) {
                const size_t b = (size_t)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)page, l) | (size_t)(uint32_t)__builtin_amdgcn_readlane((int)(page >> 32), l) << 32;
                return b + (size_t)__builtin_amdgcn_readlane(r, l) * rb;
            };
            auto scales = [&](int l, size_t page, int r) {
                const size_t b = (size_t)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)page, l) | (size_t)(uint32_t)__builtin_amdgcn_readlane((int)(page >> 32), l) << 32;
                return b + (size_t)__builtin_amdgcn_readlane(r, l) * (p.hd / 16);
            };
            // eight rows read, then written: the last one again where fewer are left
            for (uint64_t left = todo; left;) {
                constexpr int N = 8;
                size_t f[N], t[N], fs[N], ts[N];
                int l = 0;
#pragma unroll
                for (int i = 0; i < N; i++) {
                    if (left) l = __ffsll((unsigned long long)left) - 1;
                    left &= left - 1;
                    f[i] = place(l, src, src_row);
                    t[i] = place(l, dst, dst_row);
                    fs[i] = scales(l, src, src_row);
                    ts[i] = scales(l, dst, dst_row);
                }
                if (!live) continue;
                if (sc) {
                    uint32_t v[N];
#pragma unroll
                    for (int i = 0; i < N; i++) v[i] = *(const uint32_t *)(pool + at + fs[i]);
#pragma unroll
                    for (int i = 0; i < N; i++) *(uint32_t *)(pool + at + ts[i]) = v[i];
                } else {
                    pv_v4 v[N];
#pragma unroll
                    for (int i = 0; i < N; i++) v[i] = *(const pv_v4 *)(pool + at + f[i]);
#pragma unroll
                    for (int i = 0; i < N; i++) *(pv_v4 *)(pool + at + t[i]) = v[i];
                }
            }
        }
        if (wrong) {
            if (leader) paged_flag(p, PAGED_BAD_BATCH);
            return;
        }
        before = __shfl(from, 63, 64);
    }
}

// Row i of the new table: the parent's whole pages, then a fresh page that takes the
// rows of its part-filled one.  blockIdx.x: row, KV head, keys or values; y: cache;
// z: piece of a page's run of rows.
constexpr int PF_BYTES = 256 * 4 * 16;
__global__ __launch_bounds__(256) void k_paged_fork(PagedFork a, PagedPools pools) {
    const PagedPool &p = a.p;
    const bool value = blockIdx.x & 1;
    const int x = blockIdx.x >> 1, h = x % p.n_kv, i = x / p.n_kv, piece = blockIdx.z;
    const bool leader = blockIdx.y == 0 && piece == 0 && !value && h == 0;
    const int up = paged_ld(a.parent, i), fresh = paged_ld(a.fresh, i);
    int len = 0;
    bool bad = up < -1 || up >= a.b.n_seq;
    if (up >= 0 && !bad) {
        len = paged_ld(a.b.len, up);
        bad = len < 0 || len > a.b.max_len || (int64_t)len > (int64_t)a.b.table_stride * p.page || (int64_t)len > (int64_t)a.out_stride * p.page;
    }
    if (bad || up < 0) {
        if (leader && threadIdx.x == 0) {
            if (bad) paged_flag(p, PAGED_BAD_BATCH);
            if (a.len_out) a.len_out[i] = 0;
        }
        return;
    }
    const int whole = len / p.page, part = len - whole * p.page;
    const int *const table = a.b.table + (int64_t)up * a.b.table_stride;
    if (leader && a.table_out) {
        int *const out = a.table_out + (int64_t)i * a.out_stride;
        for (int k = threadIdx.x; k < whole; k += 256) out[k] = table[k];
        if (threadIdx.x == 0 && whole < a.out_stride) out[whole] = fresh;
    }
    if (leader && threadIdx.x == 0 && a.len_out) a.len_out[i] = len;
    if (part == 0) return;
    const int from = paged_ld(table, whole);
    const bool bad_page = (uint64_t)(int64_t)from >= (uint64_t)p.n_pages || (uint64_t)(int64_t)fresh >= (uint64_t)p.n_pages;
    if (bad_page || from == fresh) {                         // a parent's own page goes on
        if (bad_page && leader && threadIdx.x == 0) paged_flag(p, PAGED_BAD_PAGE);
        return;
    }
    uint8_t *const pool = value ? pools.v[blockIdx.y] : pools.k[blockIdx.y];
    const int rb = paged_row_bytes(p.type, p.hd);
    const size_t src = (size_t)from * p.page_bytes, dst = (size_t)fresh * p.page_bytes, row = (size_t)h * p.page;
    const int n = part * rb / 16, at = piece * (PF_BYTES / 16) + threadIdx.x;            // up to 4096 * 64
    if (piece * (PF_BYTES / 16) < n) {
        const pv_v4 *const f = (const pv_v4 *)(pool + src + row * rb);
        pv_v4 *const t = (pv_v4 *)(pool + dst + row * rb);
        pv_v4 v[4];
#pragma unroll
        for (int k = 0; k < 4; k++) v[k] = f[min(at + 256 * k, n - 1)];
#pragma unroll
        for (int k = 0; k < 4; k++)
            if (at + 256 * k < n) t[at + 256 * k] = v[k];
    }
    if (p.type != F16 && piece == 0) {
        const size_t at = p.sc_off + row * (p.hd / 16);
        const uint32_t *const f = (const uint32_t *)(pool + src + at);
        uint32_t *const t = (uint32_t *)(pool + dst + at);
        for (int k = threadIdx.x; k < part * (p.hd / 64); k += 256) t[k] = f[k];
    }
}

}  // namespace

hipError_t launch_paged_keep(const PagedKeep &a, const PagedPools &pools, hipStream_t s) {
    if (a.b.n_tok == 0 || a.b.n_seq == 0 || a.n_cache == 0) return hipSuccess;
    hipLaunchKernelGGL(k_paged_keep, dim3(2 * a.b.n_seq, a.n_cache), dim3(256), 0, s, a, pools);
    return hipGetLastError();
}
hipError_t launch_paged_fork(const PagedFork &a, const PagedPools &pools, hipStream_t s) {
    if (a.n_out == 0 || a.n_cache == 0) return hipSuccess;
    const int bytes = std::min(a.p.page, std::max(1, a.b.max_len)) * paged_row_bytes(a.p.type, a.p.hd);
    const int pieces = std::max(1, (bytes + PF_BYTES - 1) / PF_BYTES);
    hipLaunchKernelGGL(k_paged_fork, dim3(2u * a.p.n_kv * a.n_out, a.n_cache, pieces), dim3(256), 0, s, a, pools);
    return hipGetLastError();
}

}  // namespace g4
