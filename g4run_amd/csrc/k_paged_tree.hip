// k_paged_tree.hip -- trees of drafted tokens (g4h_paged_tree): masks and depths
// from the tokens' parents, and the path that a greedy walk accepts.  Whole numbers
// only, a few bytes a token: both are bound by a launch and their chain of dependent
// reads (offsets, then the tokens' words), so a sequence's tokens go to LDS, or to
// one wave, at once (one draft: 2 us to build, 2.8 to accept; 32 drafts of 64: 4.2).
#include "paged.h"

namespace g4 {

namespace {

constexpr int PT_TOKENS = 32 * PAGED_TREE_WORDS;

__device__ __forceinline__ void pt_flag(int *status) {
    if (status) atomicOr(status, PAGED_BAD_BATCH);
}
struct PtSpan {
    int t0, nq;
    bool torn;
};
__device__ __forceinline__ PtSpan pt_span(const PagedBatch &b, int s) {
    if (!b.q_off) return PtSpan{s, s < b.n_tok ? 1 : 0, false};
    const int a = paged_ld(b.q_off, s), e = paged_ld(b.q_off, s + 1), t0 = min(max(a, 0), b.n_tok), nq = min(max(e, t0), b.n_tok) - t0;
    return PtSpan{t0, nq, t0 != a || t0 + nq != e};
}

// mask = the token's own bit and its ancestors', depth = their number.  A workgroup a
// sequence, its tokens in blocks of 32 (a mask's words).  First a thread a token: the
// token's line within its block, and the ancestor at which it leaves the block.  Then a
// thread a (token, word), from block to block down to the word's: at most 32 steps of
// each kind, where a line followed token by token takes a thousand.
__global__ __launch_bounds__(256) void k_paged_tree_build(PagedTreeBuild a) {
    __shared__ int up[PT_TOKENS], out[PT_TOKENS];
    __shared__ uint32_t line[PT_TOKENS];
    const PtSpan q = pt_span(a.b, blockIdx.x);
    const int most = 32 * a.words, n = min(q.nq, most);
    bool bad = q.torn || q.nq > most;
    for (int i = threadIdx.x; i < n; i += 256) {
        int x = a.parent[q.t0 + i];
        if (x < -1 || x >= i) {                              // as if it had none
            bad = true;
            x = -1;
        }
        up[i] = x;
    }
    if (__any(bad) && (threadIdx.x & 63) == 0) pt_flag(a.status);
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += 256) {
        uint32_t bits = 0;
        int j = i;
        for (; j >= 0 && j >> 5 == i >> 5; j = up[j]) bits |= 1u << (j & 31);            // descends: the block ends it
        line[i] = bits;
        out[i] = j;
    }
    __syncthreads();
    for (int64_t x = threadIdx.x; x < (int64_t)q.nq * a.words; x += 256) {
        const int i = (int)(x / a.words), w = (int)(x - (int64_t)i * a.words);
        uint32_t bits = 0;
        int depth = 0;
        if (i < n) {
            int j = i;
            for (depth = -1; j >= 0 && j >> 5 > w; j = out[j]) depth += __popc(line[j]);
            if (j >= 0 && j >> 5 == w) bits = line[j];
            depth += __popc(bits);                           // of word 0: all of them
        }
        a.mask[(size_t)(q.t0 + i) * a.words + w] = bits;
        if (w == 0) a.depth[q.t0 + i] = depth;
    }
}

// The walk from token 0: from node x to its first child whose token is the choice
// made at x.  A wave a sequence, 64 tokens looked at together.
__global__ __launch_bounds__(64) void k_paged_tree_accept(PagedTreeAccept a) {
    const int s = blockIdx.x, lane = threadIdx.x;
    const PtSpan q = pt_span(a.b, s);
    const int len = paged_ld(a.b.len, s);
    const bool bad = q.torn || len < 0 || len > a.b.max_len;
    if (bad && lane == 0) pt_flag(a.status);
    int *const keep = a.keep + (size_t)s * a.most;
    int n = 0, next = -1;
    if (!bad && q.nq > 0 && len >= q.nq) {
        int at = 0;
        for (n = 1;; n++) {
            if (lane == 0) keep[n - 1] = at;
            next = a.choice[q.t0 + at];
            if (n == a.most) break;
            int found = -1;
            for (int j0 = at + 1; j0 < q.nq && found < 0; j0 += 64) {
                const int j = j0 + lane;
                const uint64_t hit = __ballot(j < q.nq && a.parent[q.t0 + min(j, q.nq - 1)] == at && a.token[q.t0 + min(j, q.nq - 1)] == next);
                if (hit) found = j0 + __ffsll((unsigned long long)hit) - 1;
            }
            if (found < 0) break;
            at = found;                                      // ascends: the walk ends
        }
    }
    for (int k = n + lane; k < a.most; k += 64) keep[k] = -1;
    if (lane == 0) {
        a.n_keep[s] = n;
        if (a.next) a.next[s] = next;
        if (a.len_out) a.len_out[s] = bad ? 0 : max(0, len - q.nq) + n;
    }
}

}  // namespace

hipError_t launch_paged_tree_build(const PagedTreeBuild &a, hipStream_t s) {
    if (a.b.n_tok == 0 || a.b.n_seq == 0) return hipSuccess;
    hipLaunchKernelGGL(k_paged_tree_build, dim3(a.b.n_seq), dim3(256), 0, s, a);
    return hipGetLastError();
}
hipError_t launch_paged_tree_accept(const PagedTreeAccept &a, hipStream_t s) {
    if (a.b.n_seq == 0) return hipSuccess;
    hipLaunchKernelGGL(k_paged_tree_accept, dim3(a.b.n_seq), dim3(64), 0, s, a);
    return hipGetLastError();
}

}  // namespace g4
