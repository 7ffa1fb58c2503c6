/* How sure a recognizer is: log probabilities of given tokens, the entropy and
 * the most probable tokens of rows of logits. */
#include "q8_internal.h"

#include <hip/hip_runtime.h>

#include <algorithm>
#include <array>
#include <utility>

#pragma clang fp contract(off)

namespace pkq8 {

typedef float p4f __attribute__((ext_vector_type(4)));
typedef float p4f_u __attribute__((ext_vector_type(4), aligned(4)));

constexpr float kLog2e = 1.44269504088896340736f;

/* Part of a row's distribution: its largest logit, the sum of exp(x - top) over
 * the others (the largest itself would hide what the rest adds: a token of
 * probability 1 - 10^-9 has a log probability of -10^-9), and that of exp(x -
 * top) (x - top). */
struct Spread {
    float top, rest, slope;
};

/* Logits in the order that the alternatives have, as whole numbers: greater
 * first, of equals the lower id, NaN last. */
__device__ __forceinline__ uint32_t ordered(float x) {
    const uint32_t u = __float_as_uint(x + 0.0f);       /* -0 is 0 */
    return x != x ? 0 : (u & 0x80000000u) ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float of_ordered(uint32_t o) {
    return __uint_as_float(o & 0x80000000u ? o & 0x7fffffffu : ~o);
}
__device__ __forceinline__ uint64_t rank_key(float x, uint32_t id) {
    return (uint64_t)ordered(x) << 32 | (uint32_t)~id;
}
__device__ __forceinline__ uint32_t key_id(uint64_t k) { return ~(uint32_t)k; }

/* Over the wave, in every lane (all of them active): within 16 lanes by DPP,
 * then across the rows into lane 63. */
template <typename F>
__device__ __forceinline__ uint32_t over_wave(uint32_t v, uint32_t none, F f) {
    v = f(v, (uint32_t)__builtin_amdgcn_update_dpp((int)none, (int)v, 0xB1, 0xF, 0xF, false));
    v = f(v, (uint32_t)__builtin_amdgcn_update_dpp((int)none, (int)v, 0x4E, 0xF, 0xF, false));
    v = f(v, (uint32_t)__builtin_amdgcn_update_dpp((int)none, (int)v, 0x141, 0xF, 0xF, false));
    v = f(v, (uint32_t)__builtin_amdgcn_update_dpp((int)none, (int)v, 0x140, 0xF, 0xF, false));
    v = f(v, (uint32_t)__builtin_amdgcn_update_dpp((int)none, (int)v, 0x142, 0xA, 0xF, false));
    v = f(v, (uint32_t)__builtin_amdgcn_update_dpp((int)none, (int)v, 0x143, 0xC, 0xF, false));
    return (uint32_t)__builtin_amdgcn_readlane((int)v, 63);
}
__device__ __forceinline__ float wave_sum_f(float x) {
    return __uint_as_float(over_wave(__float_as_uint(x), 0, [](uint32_t a, uint32_t b) {
        return __float_as_uint(__uint_as_float(a) + __uint_as_float(b));
    }));
}
__device__ __forceinline__ float wave_max_f(float x) {
    return __uint_as_float(over_wave(__float_as_uint(x), 0xff800000u, [](uint32_t a, uint32_t b) {
        return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b)));
    }));
}
__device__ __forceinline__ uint32_t wave_max_u(uint32_t x) {
    return over_wave(x, 0, [](uint32_t a, uint32_t b) { return a > b ? a : b; });
}
__device__ __forceinline__ uint32_t wave_min_u(uint32_t x) {
    return over_wave(x, ~0u, [](uint32_t a, uint32_t b) { return a < b ? a : b; });
}
__device__ __forceinline__ uint64_t wave_max_key(uint64_t v) {
#pragma unroll
    for (int m = 32; m >= 1; m >>= 1) {
        const uint64_t o = __shfl_xor(v, m);
        v = o > v ? o : v;
    }
    return v;
}

__device__ __forceinline__ void prob_sync() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

/* The k greatest of a wave's many: each lane knows its own greatest, and what at
 * least k lanes reach with theirs has k at least that reach it, and few more as a
 * rule. Found by halving the range between the least and the greatest lane's, until
 * k to k + 4 lanes do. */
__device__ __forceinline__ uint32_t reached(uint32_t mine, uint32_t k) {
    uint32_t lo = wave_min_u(mine), hi = wave_max_u(mine);
    for (int n = 0; n < 20 && lo < hi; n++) {
        const uint32_t mid = hi - (hi - lo) / 2;
        const uint32_t lanes = (uint32_t)__builtin_popcountll(__ballot(mine >= mid));
        if (lanes >= k)
            lo = mid;
        else
            hi = mid - 1;
        if (lanes >= k && lanes <= k + 4)
            break;
    }
    return lo;
}

/* n keys, up to 64 of them in LDS in any order: the i-th greatest in lane i. */
__device__ __forceinline__ uint64_t sorted(uint64_t *list, uint32_t n) {
    const uint32_t lane = threadIdx.x & 63;
    prob_sync();
    const uint64_t key = lane < n ? list[lane] : 0;
    const uint32_t lo = (uint32_t)key, hi = (uint32_t)(key >> 32);
    uint32_t rank = 0;
    for (uint32_t i = 0; i < n; i++) {
        const uint64_t other = (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)hi, i) << 32 |
                               (uint32_t)__builtin_amdgcn_readlane((int)lo, i);
        rank += other > key;
    }
    if (lane < n)
        list[rank] = key;
    prob_sync();
    return lane < n ? list[lane] : 0;
}

/* Lanes whose entry is taken put it behind the n in the list, if it is up to 64. */
template <typename K>
__device__ __forceinline__ void gather(uint64_t *list, uint32_t &n, bool taken, K key) {
    const uint64_t who = __ballot(taken);
    if (who == 0)
        return;
    const uint32_t at = n + __builtin_amdgcn_mbcnt_hi((uint32_t)(who >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)who, 0));
    if (taken && at < 64)
        list[at] = key();
    n += (uint32_t)__builtin_popcountll(who);
}

/* A wave's columns [c0, c1) of a row: 16 bytes a lane in turn V times, then 4
 * bytes a lane S times (so 1025 columns are 17 values a lane and not 20);
 * -infinity past the end. */
template <int V, int S>
__device__ __forceinline__ void load_part(const float *x, uint32_t c0, uint32_t c1, float (&y)[4 * V + S]) {
    const uint32_t lane = threadIdx.x & 63;
#pragma unroll
    for (int j = 0; j < V; j++) {
        const uint32_t c = c0 + 4 * (64 * j + lane);
        p4f t = { -INFINITY, -INFINITY, -INFINITY, -INFINITY };
        if (S > 0 || c + 4 <= c1) {         /* the last columns are behind the whole ones */
            t = *(const p4f_u *)(x + c);
        } else if (c < c1) {
            t.x = x[c];
            if (c + 1 < c1)
                t.y = x[c + 1];
            if (c + 2 < c1)
                t.z = x[c + 2];
        }
#pragma unroll
        for (int e = 0; e < 4; e++)
            y[4 * j + e] = t[e];
    }
#pragma unroll
    for (int j = 0; j < S; j++) {
        const uint32_t c = c0 + 256 * V + 64 * j + lane;
        y[4 * V + j] = c < c1 ? x[c] : -INFINITY;
    }
}

template <int V>
__device__ __forceinline__ uint32_t column_of(uint32_t c0, int j, uint32_t lane) {
    return c0 + (j < 4 * V ? 4 * (64 * (j / 4) + lane) + j % 4 : 256 * V + 64 * (j - 4 * V) + lane);
}

/* A wave's columns: the spread, and the k greatest keys (0 where there are
 * fewer), the i-th in lane i. */
template <int V, int S>
__device__ __forceinline__ Spread part_of_row(const float (&x)[4 * V + S], const float *row, uint32_t c0, uint32_t c1,
                                              uint32_t k, uint64_t *list, uint64_t &best) {
    constexpr int E = 4 * V + S;
    Spread s;
    float top = -INFINITY;
#pragma unroll
    for (int j = 0; j < E; j++)
        top = fmaxf(top, x[j]);
    s.top = wave_max_f(top);
    const float base = s.top == -INFINITY ? 0.0f : s.top;
    float rest = 0.0f, slope = 0.0f;
    uint32_t tops = 0;                      /* logits that are the largest: all but one count among the rest */
#pragma unroll
    for (int j = 0; j < E; j++) {
        const float d = x[j] - base;
        float e = __builtin_amdgcn_exp2f(d * kLog2e);
        const bool is_top = x[j] == s.top;
        tops += (uint32_t)__builtin_popcountll(__ballot(is_top));
        e = is_top ? 0.0f : e;
        rest += e;
        slope = __builtin_fmaf(e, fmaxf(d, -1e30f), slope);
    }
    s.rest = wave_sum_f(rest) + (s.top == -INFINITY ? 0.0f : (float)(tops - 1)), s.slope = wave_sum_f(slope);
    best = 0;
    if (k == 0)
        return s;
    const float least = of_ordered(reached(ordered(top), k));
    uint32_t n = 0, lane = threadIdx.x & 63;
    asm volatile("" : "+v"(lane));          /* columns are made where one is taken: kept, they would cost half of the waves */
    if (least > -INFINITY)                  /* what is past the end is not */
#pragma unroll
        for (int j = 0; j < E; j++)
            gather(list, n, x[j] >= least, [&] { return rank_key(x[j], column_of<V>(c0, j, lane)); });
    if (n >= k && n <= 64) {
        best = sorted(list, n);
        return s;
    }
    /* many equal ones, or few that are numbers: one after another, from memory (kept in registers their keys would cost
     * every row half of its waves) */
    uint64_t last = ~0ull;
#pragma unroll 1
    for (uint32_t i = 0; i < k; i++) {
        uint64_t mine = 0;
#pragma unroll 1
        for (uint32_t c = c0 + (threadIdx.x & 63); c < c1; c += 64) {
            const uint64_t key = rank_key(row[c], c);
            mine = key < last && key > mine ? key : mine;
        }
        last = wave_max_key(mine);
        best = (threadIdx.x & 63) == i ? last : best;
    }
    return s;
}

struct Answer {
    float *lp, *entropy;
    int32_t *top;
    float *top_lp;
    uint32_t k;
    const float *x;
    uint64_t xs;
    uint32_t rows, cols;
    const int32_t *tokens;
    uint32_t m;
    /* the parts of a row that several workgroups have: part (row, n) */
    Spread *spread;
    uint64_t *keys;                         /* [part][k] */
    uint32_t parts;
};

/* A row's results from its whole spread; one wave. */
__device__ __forceinline__ void answer_row(const Answer &a, uint32_t row, const Spread &s, uint64_t best) {
    const uint32_t lane = threadIdx.x & 63;
    /* log of the sum, less the largest; with an infinity, or nothing above -infinity, there is no distribution */
    const float more = __builtin_fabsf(s.top) == INFINITY ? __builtin_nanf("") : log1pf(s.rest);
    const float *x = a.x + row * a.xs;
    for (uint32_t i = lane; i < a.m; i += 64) {
        const int32_t t = a.tokens[(uint64_t)row * a.m + i];
        a.lp[(uint64_t)row * a.m + i] = t == -1 ? 0.0f : (uint32_t)t < a.cols ? (x[t] - s.top) - more : __builtin_nanf("");
    }
    if (a.entropy && lane == 0)
        a.entropy[row] = more - s.slope / (1.0f + s.rest);
    if (lane < a.k) {
        const uint32_t id = key_id(best);
        a.top[(uint64_t)row * a.k + lane] = (int32_t)id;
        if (a.top_lp)
            a.top_lp[(uint64_t)row * a.k + lane] = (x[id] - s.top) - more;
    }
}

/* The parts of spreads as one, each lane its own part (n of them; 64 at most):
 * the part whose key is the greatest has the row's largest logit, the others'
 * largest count among the rest. */
__device__ __forceinline__ Spread joined_spread(Spread s, uint64_t key, bool live) {
    const uint64_t first = wave_max_key(live ? key : 0);
    Spread r;
    r.top = wave_max_f(live ? s.top : -INFINITY);
    const float d = s.top - (r.top == -INFINITY ? 0.0f : r.top), e = __builtin_amdgcn_exp2f(d * kLog2e);
    const float n = s.rest + (key == first ? 0.0f : 1.0f);
    r.rest = wave_sum_f(live ? n * e : 0.0f);
    r.slope = wave_sum_f(live && e > 0.0f ? s.slope * e + n * e * d : 0.0f);
    return r;
}

/* Rows of up to 2048 columns, 256 V + 64 S of them: a wave each. 45000 rows of
 * 1025 with 8 alternatives, 187 MB: 46 us, 4.1 TB/s of the 6.8 that reads reach;
 * instructions bound it (587 vector and 248 scalar ones a row and wave: all of the
 * cycles). 60 with 20 values a lane and
 * the ties' keys in registers; 68 with a wave's next row loaded under this one's
 * results (92 registers for 28, five waves a SIMD for eight); 113 with one
 * alternative after another out of all values. */
template <int V, int S>
__global__ __launch_bounds__(256) void answer_wave_kernel(Answer a) {
    __shared__ uint64_t list[4][64];
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), row = blockIdx.x * 4 + wave;
    if (row >= a.rows)
        return;
    float x[4 * V + S];
    load_part<V, S>(a.x + row * a.xs, 0, a.cols, x);
    uint64_t best;
    const Spread s = part_of_row<V, S>(x, a.x + row * a.xs, 0, a.cols, a.k, list[wave], best);
    answer_row(a, row, s, best);
}

/* A workgroup's run of 1024 V columns of a row, its four waves' parts met in
 * LDS; the row's results if it is the only one, else its part of them. 64 rows of
 * 131072 with 20 alternatives: 14.9 us, and 5.2 for the launch that meets the
 * parts (69 in all with one alternative after another). Bound by the chain of a
 * wave's steps: the loads, the sums over lanes, the alternatives' order. */
template <int V>
__global__ __launch_bounds__(256) void answer_part_kernel(Answer a) {
    __shared__ Spread spread[4];
    __shared__ uint64_t list[4][64], keys[4][kMostAlternatives], met[kMostAlternatives];
    const uint32_t part = blockIdx.x % a.parts, row = blockIdx.x / a.parts;
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6, k = max(a.k, 1u);
    const uint32_t c0 = min((part * 4 + wave) * (256 * V), a.cols), c1 = min(c0 + 256 * V, a.cols);
    float x[4 * V];
    load_part<V, 0>(a.x + row * a.xs, c0, c1, x);
    uint64_t best;
    const Spread s = part_of_row<V, 0>(x, a.x + row * a.xs, c0, c1, k, list[wave], best);
    if (lane < k)
        keys[wave][lane] = best;
    if (lane == 0)
        spread[wave] = s;
    if (threadIdx.x < k)
        met[threadIdx.x] = 0;
    __syncthreads();
    /* a key's place among all is its place in its own list and how many of the others' are greater */
    if (lane < k && best) {
        uint32_t rank = lane;
        for (uint32_t u = 1; u < 4; u++)
            for (uint32_t i = 0; i < k; i++)
                rank += keys[(wave + u) % 4][i] > best;
        if (rank < k)
            met[rank] = best;
    }
    __syncthreads();
    if (wave)
        return;
    const Spread all = joined_spread(spread[lane % 4], keys[lane % 4][0], lane < 4 && keys[lane % 4][0] != 0);
    best = lane < k ? met[lane] : 0;
    if (a.parts == 1) {
        answer_row(a, row, all, best);
        return;
    }
    if (lane == 0)
        a.spread[blockIdx.x] = all;
    if (lane < k)
        a.keys[(uint64_t)blockIdx.x * k + lane] = best;
}

/* A row's parts met, a wave a row. */
__global__ __launch_bounds__(64) void answer_join_kernel(Answer a) {
    constexpr int M = 8;
    __shared__ uint64_t list[64];
    const uint32_t row = blockIdx.x, lane = threadIdx.x, k = max(a.k, 1u), all_keys = a.parts * k;
    const Spread *spread = a.spread + (uint64_t)row * a.parts;
    const uint64_t *keys = a.keys + (uint64_t)row * a.parts * k;
    Spread all = { -INFINITY, 0.0f, 0.0f };
    uint64_t first = 0;
    for (uint32_t n0 = 0; n0 < a.parts; n0 += 63) {     /* what is met so far, and 63 parts more */
        const uint32_t n = n0 + lane - 1;
        const bool own = lane == 0;
        Spread s = all;
        uint64_t key = first;
        if (!own && n < a.parts)
            s = spread[n], key = keys[(uint64_t)n * k];
        const bool live = own ? n0 > 0 : n < a.parts && n < n0 + 63;
        all = joined_spread(s, key, live);
        first = wave_max_key(live ? key : 0);
    }
    uint64_t best = 0;
    for (uint32_t n0 = 0; a.k && n0 < all_keys; n0 += 64 * M) {     /* the greatest so far, and 64 M keys more */
        uint64_t key[M + 1], top = best;
        key[M] = best;
#pragma unroll
        for (int j = 0; j < M; j++) {
            const uint32_t n = n0 + 64 * j + lane;
            key[j] = n < all_keys ? keys[n] : 0;
            top = key[j] > top ? key[j] : top;
        }
        const uint64_t least = (uint64_t)reached((uint32_t)(top >> 32), k) << 32;
        uint32_t n = 0;
#pragma unroll
        for (int j = 0; j <= M; j++)
            gather(list, n, key[j] != 0 && key[j] >= least, [&] { return key[j]; });
        if (n >= k && n <= 64) {
            best = sorted(list, n);
        } else {
            uint64_t last = ~0ull;
            for (uint32_t i = 0; i < k; i++) {
                uint64_t mine = 0;
#pragma unroll
                for (int j = 0; j <= M; j++)
                    mine = key[j] < last && key[j] > mine ? key[j] : mine;
                last = wave_max_key(mine);
                best = lane == i ? last : lane > i ? 0 : best;
            }
        }
        best = lane < k ? best : 0;
        prob_sync();
    }
    answer_row(a, row, all, best);
}

/* ------------------------------------------------------------- launches --- */

static uint32_t answer_parts(uint32_t cols) { return cols <= 2048 ? 1 : (cols + 8191) / 8192; }

size_t answer_workspace(uint32_t rows, uint32_t cols, uint32_t k) {
    const uint32_t parts = answer_parts(cols);
    if (parts == 1)
        return 0;
    return (size_t)rows * parts * ((sizeof(Spread) + 15) / 16 * 16 + std::max(k, 1u) * sizeof(uint64_t)) + 16;
}

bool answer_fits(uint32_t rows, uint32_t cols) { return (uint64_t)rows * answer_parts(cols) < 1u << 24; }

/* The kernel of rows of 64 n columns, n from 1 to 32. */
using WaveKernel = void (*)(Answer);
template <int... N>
static constexpr std::array<WaveKernel, sizeof...(N)> wave_kernels(std::integer_sequence<int, N...>) {
    return { answer_wave_kernel<(N + 1) / 4, (N + 1) % 4>... };
}
static const std::array<WaveKernel, 32> kWaveKernels = wave_kernels(std::make_integer_sequence<int, 32>());

int launch_answer(const AnswerCall &c, hipStream_t s) {
    Answer a = {};
    a.lp = c.lp, a.entropy = c.entropy, a.top = c.top, a.top_lp = c.top_lp, a.k = c.k;
    a.x = c.x, a.xs = c.xs, a.rows = c.rows, a.cols = c.cols, a.tokens = c.tokens, a.m = c.m;
    a.parts = answer_parts(c.cols);
    a.keys = (uint64_t *)c.ws;
    a.spread = (Spread *)((char *)c.ws + (size_t)c.rows * a.parts * std::max(c.k, 1u) * sizeof(uint64_t));
    if (c.cols <= 2048) {
        const uint32_t sixtyfours = (c.cols + 63) / 64;
        kWaveKernels[sixtyfours - 1]<<<(c.rows + 3) / 4, 256, 0, s>>>(a);
    } else {
        answer_part_kernel<8><<<c.rows * a.parts, 256, 0, s>>>(a);
        if (a.parts > 1)
            answer_join_kernel<<<c.rows, 64, 0, s>>>(a);
    }
    return hipPeekAtLastError() == hipSuccess ? 0 : -1;
}

}  // namespace pkq8
