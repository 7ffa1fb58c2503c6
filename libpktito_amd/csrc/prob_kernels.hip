/* How sure a recognizer is: log probabilities of given tokens, the entropy and
 * the most probable tokens of rows of logits. */
#include "q8_internal.h"

#include <hip/hip_runtime.h>

#include <algorithm>

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

/* Logits in the order that the alternatives have: greater first, of equals the
 * lower id, NaN last. */
__device__ __forceinline__ uint64_t rank_key(float x, uint32_t id) {
    const uint32_t u = __float_as_uint(x + 0.0f);       /* -0 is 0 */
    const uint32_t order = x != x ? 0 : (u & 0x80000000u) ? ~u : u | 0x80000000u;
    return (uint64_t)order << 32 | (uint32_t)~id;
}
__device__ __forceinline__ uint32_t key_id(uint64_t k) { return ~(uint32_t)k; }

__device__ __forceinline__ float wave_sum_f(float v) {
#pragma unroll
    for (int m = 32; m >= 1; m >>= 1)
        v += __shfl_xor(v, m);
    return v;
}
__device__ __forceinline__ float wave_max_f(float v) {
#pragma unroll
    for (int m = 32; m >= 1; m >>= 1)
        v = fmaxf(v, __shfl_xor(v, m));
    return v;
}
__device__ __forceinline__ uint64_t wave_max_u(uint64_t v) {
#pragma unroll
    for (int m = 32; m >= 1; m >>= 1) {
        const uint64_t o = __shfl_xor(v, m);
        v = o > v ? o : v;
    }
    return v;
}

/* x of 4 V consecutive columns' values a wave, of lanes in turn 16 bytes each;
 * -infinity past the end. */
template <int V>
__device__ __forceinline__ void load_part(const float *x, uint32_t c0, uint32_t c1, float (&y)[4 * V]) {
    const uint32_t lane = threadIdx.x & 63;
#pragma unroll
    for (int j = 0; j < V; j++) {
        const uint32_t c = c0 + 4 * (64 * j + lane);
        p4f t = { -INFINITY, -INFINITY, -INFINITY, -INFINITY };
        if (c + 4 <= c1)
            t = *(const p4f_u *)(x + c);
        else if (c < c1) {
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
}

template <int V>
__device__ __forceinline__ uint32_t column_of(uint32_t c0, int j) {
    return c0 + 4 * (64 * (j / 4) + (threadIdx.x & 63)) + j % 4;
}

/* A wave's columns: the spread, and the k greatest keys (0 where there are
 * fewer), the i-th in lane i. */
template <int V>
__device__ __forceinline__ Spread part_of_row(const float (&x)[4 * V], uint32_t c0, uint32_t c1, uint32_t k, uint64_t &best) {
    uint64_t mine = 0;
    Spread s;
    float top = -INFINITY;
#pragma unroll
    for (int j = 0; j < 4 * V; j++) {
        const uint32_t c = column_of<V>(c0, j);
        const uint64_t key = c < c1 ? rank_key(x[j], c) : 0;
        mine = key > mine ? key : mine;
        top = fmaxf(top, x[j]);
    }
    s.top = wave_max_f(top);
    uint64_t last = wave_max_u(mine);
    best = last;
    const uint32_t first = key_id(last);
    const float base = s.top == -INFINITY ? 0.0f : s.top;
    float rest = 0.0f, slope = 0.0f;
#pragma unroll
    for (int j = 0; j < 4 * V; j++) {
        const uint32_t c = column_of<V>(c0, j);
        const float d = x[j] - base;
        float e = __builtin_amdgcn_exp2f(d * kLog2e);
        e = c >= c1 || c == first ? 0.0f : e;
        rest += e;
        slope = e > 0.0f ? __builtin_fmaf(e, d, slope) : slope;
    }
    s.rest = wave_sum_f(rest), s.slope = wave_sum_f(slope);
    for (uint32_t i = 1; i < k; i++) {
        mine = 0;
#pragma unroll
        for (int j = 0; j < 4 * V; j++) {
            const uint32_t c = column_of<V>(c0, j);
            const uint64_t key = c < c1 ? rank_key(x[j], c) : 0;
            mine = key < last && key > mine ? key : mine;
        }
        last = wave_max_u(mine);
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
    const uint64_t first = wave_max_u(live ? key : 0);
    Spread r;
    r.top = wave_max_f(live ? s.top : -INFINITY);
    const float d = s.top - (r.top == -INFINITY ? 0.0f : r.top), e = __builtin_amdgcn_exp2f(d * kLog2e);
    const float n = s.rest + (key == first ? 0.0f : 1.0f);
    r.rest = wave_sum_f(live ? n * e : 0.0f);
    r.slope = wave_sum_f(live && e > 0.0f ? s.slope * e + n * e * d : 0.0f);
    return r;
}

/* Rows of up to 256 V columns: a wave each. */
template <int V>
__global__ __launch_bounds__(256) void answer_wave_kernel(Answer a) {
    const uint32_t row = blockIdx.x * 4 + (threadIdx.x >> 6);
    if (row >= a.rows)
        return;
    float x[4 * V];
    load_part<V>(a.x + row * a.xs, 0, a.cols, x);
    uint64_t best;
    const Spread s = part_of_row<V>(x, 0, a.cols, a.k, best);
    answer_row(a, row, s, best);
}

/* The greatest k of n keys, the i-th in lane i. */
template <typename K>
__device__ __forceinline__ uint64_t greatest(uint32_t n, uint32_t k, K key) {
    const uint32_t lane = threadIdx.x & 63;
    uint64_t last = ~0ull, best = 0;
    for (uint32_t i = 0; i < max(k, 1u); i++) {
        uint64_t mine = 0;
        for (uint32_t j = lane; j < n; j += 64) {
            const uint64_t y = key(j);
            mine = y < last && y > mine ? y : mine;
        }
        last = wave_max_u(mine);
        best = lane == i ? last : best;
    }
    return best;
}

/* A workgroup's run of 1024 V columns of a row, its four waves' parts met in
 * LDS; the row's results if it is the only one, else its part of them. */
template <int V>
__global__ __launch_bounds__(256) void answer_part_kernel(Answer a) {
    __shared__ Spread spread[4];
    __shared__ uint64_t keys[4][32];
    const uint32_t part = blockIdx.x % a.parts, row = blockIdx.x / a.parts;
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const uint32_t c0 = min((part * 4 + wave) * (256 * V), a.cols), c1 = min(c0 + 256 * V, a.cols);
    float x[4 * V];
    load_part<V>(a.x + row * a.xs, c0, c1, x);
    uint64_t best;
    const Spread s = part_of_row<V>(x, c0, c1, max(a.k, 1u), best);
    if (lane < max(a.k, 1u))
        keys[wave][lane] = best;
    if (lane == 0)
        spread[wave] = s;
    __syncthreads();
    if (wave)
        return;
    const uint32_t k = max(a.k, 1u);
    const bool live = lane < 4 && keys[lane % 4][0] != 0;
    const Spread all = joined_spread(spread[lane % 4], keys[lane % 4][0], live);
    best = greatest(4 * k, k, [&](uint32_t j) { return keys[j / k][j % k]; });
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
    const uint32_t row = blockIdx.x, lane = threadIdx.x, k = max(a.k, 1u);
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
        first = wave_max_u(live ? key : 0);
    }
    const uint64_t best = greatest(a.parts * k, a.k, [&](uint32_t j) { return keys[j]; });
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

int launch_answer(const AnswerCall &c, hipStream_t s) {
    Answer a = {};
    a.lp = c.lp, a.entropy = c.entropy, a.top = c.top, a.top_lp = c.top_lp, a.k = c.k;
    a.x = c.x, a.xs = c.xs, a.rows = c.rows, a.cols = c.cols, a.tokens = c.tokens, a.m = c.m;
    a.parts = answer_parts(c.cols);
    a.keys = (uint64_t *)c.ws;
    a.spread = (Spread *)((char *)c.ws + (size_t)c.rows * a.parts * std::max(c.k, 1u) * sizeof(uint64_t));
    if (c.cols <= 2048) {
        const uint32_t grid = (c.rows + 3) / 4;
        switch ((c.cols + 255) / 256) {
        case 1: answer_wave_kernel<1><<<grid, 256, 0, s>>>(a); break;
        case 2: answer_wave_kernel<2><<<grid, 256, 0, s>>>(a); break;
        case 3: answer_wave_kernel<3><<<grid, 256, 0, s>>>(a); break;
        case 4: answer_wave_kernel<4><<<grid, 256, 0, s>>>(a); break;
        case 5: answer_wave_kernel<5><<<grid, 256, 0, s>>>(a); break;
        case 6: answer_wave_kernel<6><<<grid, 256, 0, s>>>(a); break;
        default: answer_wave_kernel<8><<<grid, 256, 0, s>>>(a); break;
        }
    } else {
        answer_part_kernel<8><<<c.rows * a.parts, 256, 0, s>>>(a);
        if (a.parts > 1)
            answer_join_kernel<<<c.rows, 64, 0, s>>>(a);
    }
    return hipPeekAtLastError() == hipSuccess ? 0 : -1;
}

}  // namespace pkq8
