// k_beam.hip -- beam search's selection: of each group of beams, the n_out largest of
//   score_b + x_bv - log sum_u exp(x_bu)
// over beams b and tokens v.
//
// Within a row the order is that of its logits, so one pass over a row finds both
// what its normaliser is made of and its n_out best tokens; scores are only computed
// for those.  k_beam_rows reads the logits once, a workgroup a chunk of a row, and
// keeps per chunk the maximum, the sum and the n_out best; k_beam_join takes a row's
// from its chunks', then a group's from its rows'.  Bound by the logits' bytes where
// they are many, by the two launches and the selection's chains where they are few.
//
// Exactness: candidates are compared as (logit, lowest token) within a row and as
// (score in 64 bits, lowest beam) between rows.  Sums of exponentials are fp32
// within a thread's elements, the threads' fp32 sums added in a fixed order; chunks
// and scores in 64 bits.
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
__device__ __forceinline__ uint64_t wave_umax64(uint64_t v) {
    const uint32_t hi = wave_umax((uint32_t)(v >> 32));
    return (uint64_t)hi << 32 | wave_umax((uint32_t)(v >> 32) == hi ? (uint32_t)v : 0u);
}

// four elements from 4-byte aligned addresses on
typedef float bs_v4 __attribute__((ext_vector_type(4), aligned(4)));

constexpr int BR_CAP = 1024;                     // candidates kept for the ranking

// One chunk of 256 E elements: thread t has the elements 4 (t + 256 i) + j.  A wave's
// n_out largest thread maxima bound the chunk's n_out largest elements from below
// (each is an element): what reaches the best wave's bound is ranked by counting.
template <int E>
__global__ __launch_bounds__(256) void k_beam_rows(BeamSelect a) {
    __shared__ float red[8];
    __shared__ uint32_t bound[4];
    __shared__ int count, ones[4];
    __shared__ uint64_t cand[BR_CAP];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, row = blockIdx.x, k = a.n_out;
    if (a.ended && a.ended[row]) return;                     // its logits do not count
    const int v0 = blockIdx.y * 256 * E, n = min(a.n_vocab - v0, 256 * E);
    const float *const x = a.x + (size_t)row * a.stride + v0;
    float e[E];
#pragma unroll
    for (int i = 0; i < E / 4; i++) {
        const int at = 4 * (tid + 256 * i);
        if (at + 3 < n) {
            const bs_v4 y = *(const bs_v4 *)(x + at);
            e[4 * i] = y.x; e[4 * i + 1] = y.y; e[4 * i + 2] = y.z; e[4 * i + 3] = y.w;
        } else {
#pragma unroll
            for (int j = 0; j < 4; j++) e[4 * i + j] = at + j < n ? x[at + j] : -__builtin_inff();
        }
    }
    float m = e[0];
#pragma unroll
    for (int i = 1; i < E; i++) m = fmaxf(m, e[i]);          // a NaN only where all are
    // the wave's k-th largest thread maximum, bit by bit
    const uint32_t mo = m > -__builtin_inff() ? bs_order(m) : 0u;
    uint32_t t = 0;
    for (int b = 31; b >= 0; b--) {
        const uint32_t u = t | 1u << b;
        if (__popcll(__ballot(mo >= u)) >= k) t = u;
    }
    const float wm = group_max<64>(m);
    if (tid == 0) count = 0;
    if (lane == 0) {
        bound[wave] = t;
        red[wave] = wm;
    }
    __syncthreads();
    t = max(max(bound[0], bound[1]), max(bound[2], bound[3]));
    const float least = t > bs_order(-3.4028234664e38f) ? bs_value(t) : -3.4028234664e38f;
    m = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
    const float mm = m > -__builtin_inff() ? m : 0.0f;       // nothing but -inf and NaN
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < E; i++) s += __expf(e[i] - mm);
    s = group_sum<64>(s);
    if (lane == 0) red[4 + wave] = s;
    auto key = [&](int i) { return bs_key(e[i], v0 + 4 * (tid + 256 * (i >> 2)) + (i & 3)); };
#pragma unroll
    for (int i = 0; i < E; i++) {
        if (e[i] >= least) {
            const int at = atomicAdd(&count, 1);
            if (at < BR_CAP) cand[at] = key(i);
        }
    }
    __syncthreads();
    const size_t chunk = (size_t)row * a.chunks + blockIdx.y;
    if (tid == 0) a.ms[chunk] = make_float2(m, red[4] + red[5] + red[6] + red[7]);
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
        for (int i = 0; i < E; i++) {
            const uint64_t y = key(i);
            if (y >= low && y) cand[atomicAdd(&count, 1)] = y;  // k of them: keys differ
        }
        __syncthreads();
        c = count;
    }
    uint64_t *const top = a.top + chunk * k;
    for (int i = tid; i < c; i += 256) {
        const uint64_t y = cand[i];
        int rank = 0;
        for (int j = 0; j < c; j++) rank += cand[j] > y;
        if (rank < k) top[rank] = y;
    }
    for (int i = c + tid; i < k; i += 256) top[i] = 0;
}

// The k largest of `lists` descending lists of k in memory, lists l, l + 64, .. a
// lane's: k times the largest head.  put(i, candidate) for i < k, by the whole wave.
template <typename F>
__device__ __forceinline__ void bs_merge(const uint64_t *lists, int n, int k, F put) {
    const int lane = threadIdx.x & 63;
    if (n <= 64) {
        const uint64_t *at = lists + (size_t)min(lane, n - 1) * k, *const end = at + k;
        uint64_t head = lane < n ? *at : 0;
        for (int i = 0; i < k; i++) {
            const uint64_t best = wave_umax64(head);
            put(i, best);
            if (best == 0) continue;
            if (head == best) head = ++at < end ? *at : 0;
        }
        return;
    }
    // more lists than lanes: the best below the last one, looked for in all of the lane's
    uint64_t last = ~0ull;
    for (int i = 0; i < k; i++) {
        uint64_t mine = 0;
        if (last) {
            for (int l = lane; l < n; l += 64) {
                const uint64_t *at = lists + (size_t)l * k;
                int j = 0;
                while (j < k && at[j] >= last) j++;          // descending: the first below
                if (j < k && at[j] > mine) mine = at[j];
            }
        }
        last = wave_umax64(mine);
        put(i, last);
    }
}

// A workgroup a group: its waves merge the rows' chunks, then the first wave the rows.
__global__ __launch_bounds__(1024) void k_beam_join(BeamSelect a) {
    extern __shared__ uint64_t tops[];                       // [beam][n_out]
    __shared__ double norm[BEAM_MOST];                       // what a logit's score is above it
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6, k = a.n_out, g = blockIdx.x;
    for (int b = wave; b < a.n_beam; b += waves) {
        const int row = g * a.n_beam + b;
        if (a.ended && a.ended[row]) {
            for (int i = lane; i < k; i += 64) tops[b * k + i] = i == 0 ? 1 : 0;
            if (lane == 0) norm[b] = a.score[row];
            continue;
        }
        const float2 *const ms = a.ms + (size_t)row * a.chunks;
        float m = -__builtin_inff();
        for (int c = lane; c < a.chunks; c += 64) m = fmaxf(m, ms[c].x);
        m = group_max<64>(m);
        double s = 0.0;
        for (int c = lane; c < a.chunks; c += 64) {
            const float2 y = ms[c];
            s += y.y == 0.0f ? 0.0 : (double)y.y * exp((double)y.x - (double)m);        // a NaN stays
        }
        s = group_sum_t<64>(s);
        if (lane == 0) norm[b] = (double)a.score[row] - ((double)m + log(s));
        bs_merge(a.top + (size_t)row * a.chunks * k, a.chunks, k, [&](int i, uint64_t y) {
            if (lane == 0) tops[b * k + i] = y;
        });
    }
    __syncthreads();
    if (wave) return;
    // lane: a beam; its next candidate's score, and whether that is one
    const bool mine = lane < a.n_beam;
    const double base = mine ? norm[lane] : 0.0;
    const bool over = mine && a.ended && a.ended[g * a.n_beam + lane];
    int at = 0;
    auto next = [&]() -> uint64_t {
        if (!mine || at == k) return 0;
        const uint64_t y = tops[lane * k + at];
        if (y == 0) return 0;
        const double v = over ? base : base + (double)bs_value((uint32_t)(y >> 32));
        return v > -__builtin_inf() ? bs_order(v) : 0;       // nor a NaN
    };
    uint64_t head = next();
    for (int i = 0; i < k; i++) {
        const uint64_t best = wave_umax64(head);
        const uint64_t hit = __ballot(head == best);
        const int b = __ffsll((unsigned long long)hit) - 1;  // the lowest of equal ones
        const size_t out = (size_t)g * k + i;
        if (best == 0) {
            if (lane == 0) {
                a.score_out[out] = -__builtin_inff();
                a.row_out[out] = -1;
                a.token_out[out] = -1;
            }
            continue;
        }
        if (lane == b) {
            a.score_out[out] = (float)bs_value(best);
            a.row_out[out] = g * a.n_beam + b;
            a.token_out[out] = over ? -1 : (int)~(uint32_t)tops[lane * k + at];
            at++;
            head = next();
        }
    }
}

// Elements of a thread: 32 where that leaves two workgroups a CU, else 8.
int beam_elements(int rows, int n_vocab) { return (int64_t)rows * ((n_vocab + 8191) / 8192) >= 512 ? 32 : 8; }

}  // namespace

size_t beam_workspace(int n_group, int n_beam, int n_vocab, int n_out) {
    const int rows = n_group * n_beam, chunk = 256 * beam_elements(rows, n_vocab);
    const size_t chunks = (size_t)rows * ((n_vocab + chunk - 1) / chunk);
    return chunks * (sizeof(float2) + (size_t)n_out * sizeof(uint64_t));
}
hipError_t launch_beam_select(BeamSelect a, uint8_t *ws, hipStream_t s) {
    const int rows = a.n_group * a.n_beam, e = beam_elements(rows, a.n_vocab), chunk = 256 * e;
    if (rows == 0) return hipSuccess;
    a.chunks = (a.n_vocab + chunk - 1) / chunk;
    a.top = (uint64_t *)ws;
    a.ms = (float2 *)(ws + (size_t)rows * a.chunks * a.n_out * sizeof(uint64_t));
    if (e == 32) hipLaunchKernelGGL(k_beam_rows<32>, dim3(rows, a.chunks), dim3(256), 0, s, a);
    else hipLaunchKernelGGL(k_beam_rows<8>, dim3(rows, a.chunks), dim3(256), 0, s, a);
    if (hipError_t err = hipGetLastError()) return err;
    const int waves = std::min(16, a.n_beam);
    hipLaunchKernelGGL(k_beam_join, dim3(a.n_group), dim3(64 * waves), (size_t)a.n_beam * a.n_out * sizeof(uint64_t), s, a);
    return hipGetLastError();
}

}  // namespace g4
