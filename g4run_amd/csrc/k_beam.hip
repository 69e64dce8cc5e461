// k_beam.hip -- beam search's selection: of each group of beams, the n_out largest of
//   score_b + x_bv - log sum_u exp(x_bu)
// over beams b and tokens v.
//
// Within a row the order is that of its logits, so one pass over a row finds both
// what its normaliser is made of and its n_out best tokens; scores are only computed
// for those.  k_beam_rows reads the logits once, a workgroup a part of a row, and
// leaves the part's maximum, sum and n_out best; k_beam_join takes a row's from its
// parts', then a group's from its rows'.  Bound by the logits' bytes where they are
// many (16 groups of 8 beams of 262144, 16 outputs: 37 us of k_beam_rows, 3.6 TB/s, and
// 10 of k_beam_join, whose two merges are a chain of 32 rounds), by the two launches and
// the selection's chains where they are few (4 beams of 32768, 8 outputs: 6 and 6 us) or
// the outputs many: the first bound is loose, and candidates are ranked by comparing all
// with all (32 beams of 262144, both kernels: 8, 16, 32, 64 outputs 25, 35, 53, 245 us).
//
// Exactness: candidates are compared as (logit, lowest token) within a row and as
// (score in 64 bits, lowest beam) between rows.  Sums of exponentials are fp32, under
// each thread's running maximum, added up over the threads in a fixed order; over the
// parts, and scores, in 64 bits.
#include <algorithm>

#include "beam.h"

namespace g4 {

namespace {

// ascending with the value, -0 as +0; every finite value above 0
__device__ __forceinline__ uint32_t bs_order(float x) {
    const uint32_t u = __builtin_bit_cast(uint32_t, x + 0.0f);
    return u ^ ((uint32_t)((int32_t)u >> 31) | 0x80000000u);
}
__device__ __forceinline__ float bs_value(uint32_t o) {
    return __builtin_bit_cast(float, o ^ ((o >> 31) ? 0x80000000u : 0xffffffffu));
}
__device__ __forceinline__ uint64_t bs_order(double x) {
    const uint64_t u = __builtin_bit_cast(uint64_t, x + 0.0);
    return u ^ ((uint64_t)((int64_t)u >> 63) | 0x8000000000000000ull);
}
__device__ __forceinline__ double bs_value(uint64_t o) {
    return __builtin_bit_cast(double, o ^ ((o >> 63) ? 0x8000000000000000ull : 0xffffffffffffffffull));
}
// a candidate: 0 for what is none (NaN, -inf)
__device__ __forceinline__ uint64_t bs_key(float x, int v) {
    return x > -__builtin_inff() ? (uint64_t)bs_order(x) << 32 | (uint32_t)~v : 0;
}
// The largest of the wave's values and the first lane that has it: one round over the
// upper halves, a second where several lanes share the largest.
__device__ __forceinline__ uint64_t bs_largest(uint64_t v, int &lane) {
    const uint32_t hi = wave_umax((uint32_t)(v >> 32));
    uint64_t who = __ballot((uint32_t)(v >> 32) == hi);
    uint32_t lo;
    if (who & (who - 1)) {
        const bool tied = (uint32_t)(v >> 32) == hi;
        lo = wave_umax(tied ? (uint32_t)v : 0u);
        who = __ballot(tied && (uint32_t)v == lo);
        lane = __ffsll((unsigned long long)who) - 1;
    } else {
        lane = __ffsll((unsigned long long)who) - 1;
        lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)v, lane);
    }
    return (uint64_t)hi << 32 | lo;
}

// four elements from 4-byte aligned addresses on
typedef float bs_v4 __attribute__((ext_vector_type(4), aligned(4)));

constexpr int BR_CAP = 1024;                     // new candidates of a chunk

// A part of a row in chunks of 256 E elements, the next one's loads under way while one
// is looked through: thread t has a chunk's elements 4 (t + 256 i) + j.  Elements above
// the n_out-th best so far join the list, few after the first chunk; in the first one
// a wave's n_out-th largest thread maximum bounds the n_out-th largest element from
// below (each maximum is an element), and the best of four waves' bounds counts.
// (Parts of one chunk, each with a bound of its own: 2048 workgroups 42 us, 1024 of
// eight chunks 37.)
template <int E>
__global__ __launch_bounds__(256) void k_beam_rows(BeamSelect a) {
    __shared__ float red[8];
    __shared__ uint32_t bound[4];
    __shared__ int counts[2], ones[4];                       // of a chunk's candidates: one of the two, in turn
    __shared__ uint64_t cand[BR_CAP], best[2][BEAM_MOST];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, row = blockIdx.x, k = a.n_out;
    if (a.ended && a.ended[row]) return;                     // its logits do not count
    const int v0 = blockIdx.y * a.span, n = min(a.n_vocab - v0, a.span);
    const float *const x = a.x + (size_t)row * a.stride + v0;
    constexpr float LOWEST = -3.4028234664e38f;
    float e[E], more[E];
    auto load = [&](float(&to)[E], int c0) {
#pragma unroll
        for (int i = 0; i < E / 4; i++) {
            const int at = c0 + 4 * (tid + 256 * i);
            if (at + 3 < n) {
                const bs_v4 y = *(const bs_v4 *)(x + at);
                to[4 * i] = y.x; to[4 * i + 1] = y.y; to[4 * i + 2] = y.z; to[4 * i + 3] = y.w;
            } else {
#pragma unroll
                for (int j = 0; j < 4; j++) to[4 * i + j] = at + j < n ? x[at + j] : -__builtin_inff();
            }
        }
    };
    if (tid < 2) counts[tid] = 0;
    load(more, 0);
    float m = -__builtin_inff(), s = 0.0f, least = LOWEST;
    int kept = 0, side = 0, turn = 0;
    for (int c0 = 0; c0 < n; c0 += 256 * E, turn ^= 1) {
        // a thread that finds no candidate goes on while others still read that: the next
        // chunk counts elsewhere, and the one behind it after another barrier
        int &count = counts[turn];
#pragma unroll
        for (int i = 0; i < E; i++) e[i] = more[i];
        if (c0 + 256 * E < n) load(more, c0 + 256 * E);
        float cm = e[0];
#pragma unroll
        for (int i = 1; i < E; i++) cm = fmaxf(cm, e[i]);    // a NaN only where all are
        if (cm > m) {
            s *= __expf(m - cm);                             // from -inf: 0 (or a NaN's NaN)
            m = cm;
        }
        const float mm = m > -__builtin_inff() ? m : 0.0f;   // nothing but -inf and NaN
        float cs = 0.0f;                                     // a chunk's apart: few roundings in a long row
#pragma unroll
        for (int i = 0; i < E; i++) cs += __expf(e[i] - mm);
        s += cs;
        if (kept < k) {
            // the wave's k-th largest thread maximum, its upper half bit by bit
            const uint32_t mo = cm > -__builtin_inff() ? bs_order(cm) : 0u;
            uint32_t t = 0;
            for (int b = 31; b >= 16; b--) {
                const uint32_t u = t | 1u << b;
                if (__popcll(__ballot(mo >= u)) >= k) t = u;
            }
            if (lane == 0) bound[wave] = t;
            __syncthreads();
            t = max(max(bound[0], bound[1]), max(bound[2], bound[3]));
            least = t > bs_order(LOWEST) ? bs_value(t) : LOWEST;
        }
        auto key = [&](int i) { return bs_key(e[i], v0 + c0 + 4 * (tid + 256 * (i >> 2)) + (i & 3)); };
#pragma unroll
        for (int i = 0; i < E; i++) {
            if (e[i] >= least) {
                const int at = atomicAdd(&count, 1);
                if (at < BR_CAP) cand[at] = key(i);
            }
        }
        __syncthreads();
        int c = count;
        if (c > BR_CAP) {
            // too many alike: the k-th largest candidate itself, bit by bit
            uint64_t low = 0;
            for (int b = 63; b >= 0; b--) {
                const uint64_t u = low | 1ull << b;
                int n1 = 0;
#pragma unroll
                for (int i = 0; i < E; i++) n1 += key(i) >= u;
                n1 = group_isum<64>(n1);
                __syncthreads();
                if (lane == 0) ones[wave] = n1;
                __syncthreads();
                if (ones[0] + ones[1] + ones[2] + ones[3] >= k) low = u;
            }
            __syncthreads();
            if (tid == 0) count = 0;
            __syncthreads();
#pragma unroll
            for (int i = 0; i < E; i++) {
                const uint64_t y = key(i);
                if (y >= low && y) cand[atomicAdd(&count, 1)] = y;       // k of them: keys differ
            }
            __syncthreads();
            c = count;
        }
        if (c == 0) continue;
        // ranks among those kept and the new ones, by counting
        const uint64_t *const old = best[side];
        uint64_t *const now = best[side ^ 1];
        for (int i = tid; i < kept + c; i += 256) {
            const uint64_t y = i < kept ? old[i] : cand[i - kept];
            int rank = i < kept ? i : 0;
            if (i >= kept)
                for (int j = 0; j < kept; j++) rank += old[j] > y;
            for (int j = 0; j < c; j++) rank += cand[j] > y;
            if (rank < k) now[rank] = y;
        }
        __syncthreads();
        if (tid == 0) count = 0;
        kept = min(kept + c, k);
        side ^= 1;
        if (kept == k) {
            // only what is above the k-th: an equal one has a higher token
            const float kth = bs_value((uint32_t)(now[k - 1] >> 32));
            least = kth < __builtin_inff() ? bs_value(bs_order(kth) + 1) : __builtin_nanf("");
        }
        __syncthreads();
    }
    const float wm = group_max<64>(m);
    s = m > -__builtin_inff() ? s * __expf(m - wm) : s;
    s = group_sum<64>(s);
    if (lane == 0) {
        red[wave] = wm;
        red[4 + wave] = s;
    }
    __syncthreads();
    const size_t list = (size_t)row * a.lists + blockIdx.y;
    if (tid == 0) {
        const float top = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
        float sum = 0.0f;
        for (int w = 0; w < 4; w++) sum += red[w] > -__builtin_inff() ? red[4 + w] * __expf(red[w] - top) : red[4 + w];
        a.ms[list] = make_float2(top, sum);
    }
    for (int i = tid; i < k; i += 256) a.top[list * k + i] = i < kept ? best[side][i] : 0;
}

// The first entries of a lane's list in registers.
struct BsHeads {
    uint64_t h[4];
};
__device__ __forceinline__ BsHeads bs_heads(const uint64_t *list, bool is, int k) {
    BsHeads x;
#pragma unroll
    for (int i = 0; i < 4; i++) x.h[i] = is && i < k ? list[i] : 0;
    return x;
}
// The k largest of up to 64 descending lists of k, one a lane's, its first entries in
// x, by the whole wave: lane i gets the i-th, the list it is from and its place there.
// Ties go to the first list.
struct BsBest {
    uint64_t entry;
    int list, at;
};
__device__ __forceinline__ BsBest bs_merge(const uint64_t *list, BsHeads x, int k) {
    const int lane = threadIdx.x & 63;
    BsBest y = {0, 0, 0};
    int taken = 0;
    for (int i = 0; i < k; i++) {
        int who;
        const uint64_t best = bs_largest(x.h[0], who);
        if (best == 0) break;
        const int at = __builtin_amdgcn_readlane(taken, who);
        if (lane == i) y = BsBest{best, who, at};
        if (lane == who) {
            x.h[0] = x.h[1];
            x.h[1] = x.h[2];
            x.h[2] = x.h[3];
            x.h[3] = 0;
            if ((++taken & 3) == 0) {                        // four at a time: a load a round would be waited for in each
#pragma unroll
                for (int j = 0; j < 4; j++) x.h[j] = taken + j < k ? list[taken + j] : 0;
            }
        }
    }
    return y;
}

// A workgroup a group: its waves merge the rows' lists, all threads turn the rows' best
// into scores, the first wave merges the rows.
__global__ __launch_bounds__(1024) void k_beam_join(BeamSelect a) {
    extern __shared__ uint64_t tops[];                       // [beam][n_out] candidates, then their scores; behind them the tokens
    __shared__ double norm[BEAM_MOST];                       // what a logit's score is above it
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6, k = a.n_out, g = blockIdx.x;
    int *const tokens = (int *)(tops + a.n_beam * k);
    for (int b = wave; b < a.n_beam; b += waves) {
        const int row = g * a.n_beam + b;
        // all that the row needs at once: the first reads are what this kernel waits for
        const bool over = a.ended && a.ended[row];
        const float score = a.score[row];
        const float2 *const ms = a.ms + (size_t)row * a.lists;
        const uint64_t *const list = a.top + ((size_t)row * a.lists + min(lane, a.lists - 1)) * k;
        const float2 first = ms[min(lane, a.lists - 1)];     // lane: a list
        const BsHeads heads = bs_heads(list, lane < a.lists, k);
        if (over) {
            for (int i = lane; i < k; i += 64) tops[b * k + i] = i == 0 ? 1 : 0;
            if (lane == 0) norm[b] = score;
            continue;
        }
        const float m = group_max<64>(first.x);
        // (a NaN stays one)
        const double s = group_sum_t<64>(lane < a.lists && first.y != 0.0f ? (double)first.y * exp((double)first.x - (double)m) : 0.0);
        if (lane == 0) norm[b] = (double)score - ((double)m + log(s));
        const BsBest y = bs_merge(list, heads, k);
        if (lane < k) tops[b * k + lane] = y.entry;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < a.n_beam * k; i += blockDim.x) {
        const int b = i / k;
        const uint64_t y = tops[i];
        const double v = y == 1 ? norm[b] : norm[b] + (double)bs_value((uint32_t)(y >> 32));         // (1: no logit's)
        tops[i] = y && v > -__builtin_inf() ? bs_order(v) : 0;           // nor a NaN
        tokens[i] = y == 1 ? -1 : (int)~(uint32_t)y;
    }
    __syncthreads();
    if (wave) return;
    const bool mine = lane < a.n_beam;                       // lane: a beam
    const uint64_t *const list = tops + (mine ? lane : 0) * k;
    const BsBest y = bs_merge(list, bs_heads(list, mine, k), k);
    if (lane >= k) return;
    const size_t out = (size_t)g * k + lane;
    a.score_out[out] = y.entry ? (float)bs_value(y.entry) : -__builtin_inff();
    a.row_out[out] = y.entry ? g * a.n_beam + y.list : -1;
    a.token_out[out] = y.entry ? tokens[y.list * k + y.at] : -1;
}

// How a row is cut: 4 workgroups a CU in all where its parts stay 4096 tokens or more,
// else parts of 2048, one chunk of 8 elements a thread; never more parts than a wave of
// k_beam_join has lanes.
constexpr int BEAM_LISTS = 64;
struct BeamSplit {
    int lists, span, e;
};
BeamSplit beam_split(int rows, int n_vocab) {
    BeamSplit y;
    const int most = (n_vocab + 4095) / 4096, want = std::max(1, 1024 / std::max(1, rows)), small = (n_vocab + 2047) / 2048;
    y.e = want >= most && small <= BEAM_LISTS ? 8 : 16;
    const int lists = y.e == 8 ? small : std::min(std::min(want, most), BEAM_LISTS);
    y.span = ((n_vocab + lists - 1) / lists + 1023) / 1024 * 1024;
    y.lists = (n_vocab + y.span - 1) / y.span;
    return y;
}

// lists of any call of up to `rows` rows at most: fewer rows may be cut into more parts
size_t beam_lists_most(int rows, int n_vocab) {
    const int most = (n_vocab + 4095) / 4096, small = (n_vocab + 2047) / 2048;
    const int fine = small > BEAM_LISTS ? 0 : most == 1 ? rows : 1024 / most;            // rows up to which the parts are of 2048
    const size_t few = (size_t)std::min(rows, fine) * small;
    const size_t many = rows > fine ? std::min((size_t)rows * std::min(most, BEAM_LISTS), (size_t)std::max(1024, rows)) : 0;
    return std::max(few, many);
}
size_t beam_bytes(size_t lists, int n_out) { return lists * (sizeof(float2) + (size_t)n_out * sizeof(uint64_t)); }

}  // namespace

size_t beam_workspace(int n_group, int n_beam, int n_vocab, int n_out) {
    const int rows = n_group * n_beam;
    return beam_bytes((size_t)rows * beam_split(rows, n_vocab).lists, n_out);
}
size_t beam_workspace_most(int n_group, int n_beam, int n_vocab, int n_out) { return beam_bytes(beam_lists_most(n_group * n_beam, n_vocab), n_out); }
hipError_t launch_beam_select(BeamSelect a, uint8_t *ws, hipStream_t s) {
    const int rows = a.n_group * a.n_beam;
    if (rows == 0) return hipSuccess;
    const BeamSplit y = beam_split(rows, a.n_vocab);
    a.lists = y.lists;
    a.span = y.span;
    a.top = (uint64_t *)ws;
    a.ms = (float2 *)(ws + (size_t)rows * a.lists * a.n_out * sizeof(uint64_t));
    if (y.e == 16) hipLaunchKernelGGL(k_beam_rows<16>, dim3(rows, a.lists), dim3(256), 0, s, a);
    else hipLaunchKernelGGL(k_beam_rows<8>, dim3(rows, a.lists), dim3(256), 0, s, a);
    if (hipError_t err = hipGetLastError()) return err;
    const int waves = std::min(16, a.n_beam);
    hipLaunchKernelGGL(k_beam_join, dim3(a.n_group), dim3(64 * waves), (size_t)a.n_beam * a.n_out * (sizeof(uint64_t) + sizeof(int)), s, a);
    return hipGetLastError();
}

}  // namespace g4
