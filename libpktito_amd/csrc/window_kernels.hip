/* Attention with a sliding window and sinks over whole segments: every row
 * attends the frames of a window around it and the segment's first few, so an
 * hour of audio in one piece costs its frames times the window. Products and
 * sums in 32 bits on the fp32 matrix instruction: it rounds as a fused multiply
 * and add does, takes floats of any magnitude as they are, and a product of
 * three bfloat16 pieces by three would gain a fifth of its time at best and lose
 * that in the cutting. */
#include "q8_internal.h"

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>

#pragma clang fp contract(off)

namespace pkq8 {

typedef float w4f __attribute__((ext_vector_type(4)));

struct WindowAttention {
    float *o;
    const float *q, *k, *v;
    uint64_t os, qs, ks, vs;
    const int32_t *row0;
    uint32_t B, rows, max_T, H, G;
    int32_t left, right, sinks;             /* clipped to what can occur */
    float scale;                            /* log2(e) / sqrt(dk) */
    const float *p, *bias_u, *bias_w;       /* p's first row the distance left's; NULL: no positions */
    uint32_t bw;                            /* its rows, left + right + 1 */
    uint32_t tiles;                         /* a segment's tiles of rows */
};

/* A workgroup's part: rows [i0, i0 + R) of a segment of T at row r0, one head. */
struct WindowTile {
    int32_t r0, T, i0;
    uint32_t h, g;
};

template <int R>
__device__ __forceinline__ bool window_tile(const WindowAttention &a, WindowTile &s) {
    uint32_t i = blockIdx.x;
    s.h = i % a.H, i /= a.H;
    s.g = s.h / (a.H / a.G);
    s.i0 = (int32_t)(i % a.tiles) * R;
    const uint32_t b = i / a.tiles;
    s.r0 = cache_clip(a.row0[b], 0, (int32_t)a.rows);
    s.T = cache_clip(cache_clip(a.row0[b + 1], 0, (int32_t)a.rows) - s.r0, 0, (int32_t)a.max_T);
    return s.i0 < s.T;
}

__device__ __forceinline__ w4f wmfma(float x, float y, w4f c) {
    return __builtin_amdgcn_mfma_f32_16x16x4f32(x, y, c, 0, 0, 0);
}

/* The instruction's reduction runs over 4 indices, one a quarter of the wave,
 * in any order that both operands follow. For the scores lane l takes
 * dimensions 16 t + 4 (l / 16) + i of key (or row of positions) l % 16, i in
 * four instructions one after another: a key's row is read 16 bytes a lane, and
 * so is the query's. Keys are the result's rows and queries its columns: a lane
 * holds scores of query l % 16 with keys 4 (l / 16) + r, which is where the
 * second product wants them (r again in four instructions), so no probability
 * crosses lanes. There the rows are dimensions, VW of them next to each other in
 * a lane over VW instructions. */
template <int NS>
struct WindowShape {
    static constexpr int dk = 32 * NS, NT = dk / 16;
    static constexpr int VW = NS % 2 ? 2 : 4, NB = dk / (16 * VW);
    typedef float vec __attribute__((ext_vector_type(VW)));
};

/* Sixteen queries' operands: with the content's bias and with the place's, in
 * powers of 2, and what a frame behind the window scores for its place (the
 * table's first row). */
template <int NS, bool POS>
struct WindowQueries {
    w4f c[2 * NS], p[POS ? 2 * NS : 1];
    float behind;

    __device__ __forceinline__ void load(const WindowAttention &a, const WindowTile &s, int32_t i) {
        constexpr uint32_t dk = 32 * NS;
        const uint32_t w = (threadIdx.x & 63) / 16;
        const float *src = a.q + (uint64_t)(s.r0 + min(i, s.T - 1)) * a.qs + s.h * dk + 4 * w;
        behind = 0.0f;
#pragma unroll
        for (int t = 0; t < 2 * NS; t++) {
            const w4f x = *(const w4f *)(src + 16 * t);
            if constexpr (POS) {
                const uint32_t d = s.h * dk + 4 * w + 16 * t;
                c[t] = (x + *(const w4f *)(a.bias_u + d)) * a.scale;
                p[t] = (x + *(const w4f *)(a.bias_w + d)) * a.scale;
                if (a.sinks) {
                    const w4f far = *(const w4f *)(a.p + d);
#pragma unroll
                    for (int j = 0; j < 4; j++)
                        behind = __builtin_fmaf(p[t][j], far[j], behind);
                }
            } else {
                c[t] = x * a.scale;
            }
        }
        if constexpr (POS) {
            behind += __shfl_xor(behind, 16);
            behind += __shfl_xor(behind, 32);
        }
    }
};

/* The running maximum follows the scores only when one is over it by more than
 * this many powers of two. */
constexpr float kWindowSlack = 8.0f;

/* Scores of a query with 16 KT frames, -infinity where not attended, into the
 * running softmax: the exponentials in their place. */
template <int KT, int NO>
__device__ __forceinline__ void window_softmax(w4f (&s)[KT], float &top, float &sum, w4f (&o)[NO]) {
    float best = -INFINITY;
#pragma unroll
    for (int i = 0; i < 4 * KT; i++)
        best = fmaxf(best, s[i / 4][i % 4]);
    if (__any(best > top + kWindowSlack)) {
        best = fmaxf(best, __shfl_xor(best, 16));
        best = fmaxf(best, __shfl_xor(best, 32));
        const float now = fmaxf(top, best);
        const float scale = __builtin_amdgcn_exp2f(top - (now == -INFINITY ? 0.0f : now));
        top = now;
        sum *= scale;
#pragma unroll
        for (int i = 0; i < NO; i++)
            o[i] *= scale;
    }
    const float base = top == -INFINITY ? 0.0f : top;
#pragma unroll
    for (int i = 0; i < 4 * KT; i++) {
        const float e = __builtin_amdgcn_exp2f(s[i / 4][i % 4] - base);
        sum += e;
        s[i / 4][i % 4] = e;
    }
}

__device__ __forceinline__ void wave_sync() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

/* Sixteen rows a workgroup, its waves a run of 32 frames each in turn, met in
 * LDS at the end: for calls of few tiles, where one wave's pass over a row's
 * frames is what takes time. Operands come straight from memory. A frame j's
 * place scores are products with 47 rows of the table, x = left - (row - j); a
 * lane's are another column's, so they pass through LDS. */
template <int NS, bool POS, int W>
__global__ __launch_bounds__(64 * W, 1) void window_few_kernel(WindowAttention a) {
    using S = WindowShape<NS>;
    constexpr int KT = 2, kKeys = 16 * KT, PT = KT + 1, kRow = 16 * PT + 4;
    __shared__ __attribute__((aligned(16))) float part[W][16][S::dk + 4];
    __shared__ __attribute__((aligned(16))) float place[POS ? W : 1][16][kRow];
    __shared__ float tops[W][16], sums[W][16];
    WindowTile s;
    if (!window_tile<16>(a, s))
        return;
    const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int32_t c = (int32_t)(lane % 16), w = (int32_t)(lane / 16), i = s.i0 + c;
    WindowQueries<NS, POS> q;
    q.load(a, s, i);
    float top = -INFINITY, sum = 0.0f;
    w4f o[2 * NS] = {};

    /* the runs that the tile reaches: the sinks' first, then the window's */
    const int32_t w0 = max(s.i0 - a.left, 0) / kKeys, w1 = min(s.i0 + 15 + a.right, s.T - 1) / kKeys + 1;
    const int32_t ns = min((min(a.sinks, s.T) + kKeys - 1) / kKeys, w0);
    const int32_t runs = ns + w1 - w0;
#pragma unroll 1
    for (int32_t n = (int32_t)wave; n < runs; n += W) {
        const int32_t j0 = kKeys * (n < ns ? n : n - ns + w0);
        w4f x[KT] = {};
#pragma unroll
        for (int kt = 0; kt < KT; kt++) {
            const float *src = a.k + (uint64_t)(s.r0 + min(j0 + 16 * kt + c, s.T - 1)) * a.ks + s.g * S::dk + 4 * w;
            w4f key[S::NT];
#pragma unroll
            for (int t = 0; t < S::NT; t++)
                key[t] = *(const w4f *)(src + 16 * t);
#pragma unroll
            for (int t = 0; t < S::NT; t++)
#pragma unroll
                for (int j = 0; j < 4; j++)
                    x[kt] = wmfma(key[t][j], q.c[t][j], x[kt]);
        }
        if constexpr (POS) {
            if (n >= ns) {
                const int32_t x0 = a.left - (s.i0 + 15) + j0;
#pragma unroll
                for (int pt = 0; pt < PT; pt++) {
                    const int32_t row = cache_clip(x0 + 16 * pt + c, 0, (int32_t)a.bw - 1);
                    const float *src = a.p + (uint64_t)(uint32_t)row * (a.H * S::dk) + s.h * S::dk + 4 * w;
                    w4f pos[S::NT], r = {};
#pragma unroll
                    for (int t = 0; t < S::NT; t++)
                        pos[t] = *(const w4f *)(src + 16 * t);
#pragma unroll
                    for (int t = 0; t < S::NT; t++)
#pragma unroll
                        for (int j = 0; j < 4; j++)
                            r = wmfma(pos[t][j], q.p[t][j], r);
                    *(w4f *)&place[wave][c][16 * pt + 4 * w] = r;
                }
                wave_sync();
#pragma unroll
                for (int kt = 0; kt < KT; kt++)
#pragma unroll
                    for (int r = 0; r < 4; r++) {
                        const float y = place[wave][c][15 - c + 16 * kt + 4 * w + r];
                        x[kt][r] += j0 + 16 * kt + 4 * w + r < i - a.left ? q.behind : y;
                    }
                wave_sync();
            } else {
#pragma unroll
                for (int kt = 0; kt < KT; kt++)
                    x[kt] += q.behind;
            }
        }
#pragma unroll
        for (int kt = 0; kt < KT; kt++)
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const int32_t j = j0 + 16 * kt + 4 * w + r;
                const bool seen = j < s.T && j <= i + a.right && (j >= i - a.left || j < a.sinks);
                x[kt][r] = seen ? x[kt][r] : -INFINITY;
            }
        typename S::vec v[KT][4][S::NB];
        float odd = 0.0f;                   /* NaN where a value is no number */
#pragma unroll
        for (int kt = 0; kt < KT; kt++)
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const int32_t j = min(j0 + 16 * kt + 4 * w + r, s.T - 1);
                const float *src = a.v + (uint64_t)(s.r0 + j) * a.vs + s.g * S::dk + S::VW * c;
#pragma unroll
                for (int b = 0; b < S::NB; b++) {
                    v[kt][r][b] = *(const typename S::vec *)(src + 16 * S::VW * b);
#pragma unroll
                    for (int e = 0; e < S::VW; e++)
                        odd = __builtin_fmaf(v[kt][r][b][e], 0.0f, odd);
                }
            }
        w4f prob[KT];
#pragma unroll
        for (int kt = 0; kt < KT; kt++)
            prob[kt] = x[kt];
        window_softmax<KT, 2 * NS>(prob, top, sum, o);
        if (__builtin_expect(__any(odd != odd), 0)) {
            /* An infinity or a NaN among the values may be only some rows': the others would get its product with
             * their 0. Those take the product without it, and each attended one is added to the rows that attend it. */
#pragma unroll
            for (int kt = 0; kt < KT; kt++)
#pragma unroll
                for (int r = 0; r < 4; r++)
#pragma unroll
                    for (int b = 0; b < S::NB; b++)
#pragma unroll
                        for (int e = 0; e < S::VW; e++) {
                            const float y = v[kt][r][b][e];
                            const bool bad = __builtin_fmaf(y, 0.0f, 0.0f) != 0.0f;
                            v[kt][r][b][e] = bad ? 0.0f : y;
                            uint64_t who = __ballot(bad);
                            while (who) {
                                const int from = __builtin_ctzll(who);
                                who &= who - 1;
                                const float value = __shfl(y, from);
                                const float mine = __shfl(prob[kt][r], 16 * (from / 16) + c);
                                const bool seen = __shfl((int)(x[kt][r] != -INFINITY), 16 * (from / 16) + c);
                                /* its dimension is row from % 16 of block (b, e), which lanes w = row / 4 hold */
                                const int row = from % 16;
#pragma unroll
                                for (int rr = 0; rr < 4; rr++)
                                    if (seen && row == 4 * w + rr)
                                        o[b * S::VW + e][rr] += mine * value;
                            }
                        }
        }
#pragma unroll
        for (int kt = 0; kt < KT; kt++)
#pragma unroll
            for (int r = 0; r < 4; r++)
#pragma unroll
                for (int b = 0; b < S::NB; b++)
#pragma unroll
                    for (int e = 0; e < S::VW; e++)
                        o[b * S::VW + e] = wmfma(v[kt][r][b][e], prob[kt][r], o[b * S::VW + e]);
    }
    sum += __shfl_xor(sum, 16);
    sum += __shfl_xor(sum, 32);
    if (w == 0)
        tops[wave][c] = top, sums[wave][c] = sum;
#pragma unroll
    for (int b = 0; b < S::NB; b++)
#pragma unroll
        for (int r = 0; r < 4; r++) {
            typename S::vec y;
#pragma unroll
            for (int e = 0; e < S::VW; e++)
                y[e] = o[b * S::VW + e][r];
            *(typename S::vec *)&part[wave][c][16 * S::VW * b + S::VW * (4 * w + r)] = y;
        }
    __syncthreads();
    for (uint32_t n = threadIdx.x; n < 16 * S::dk / 4; n += 64 * W) {
        const int32_t r = (int32_t)(n / (S::dk / 4)), d = (int32_t)(n % (S::dk / 4)) * 4;
        if (s.i0 + r >= s.T)
            continue;
        float m = -INFINITY, l = 0.0f;
        w4f y = {};
#pragma unroll
        for (int u = 0; u < W; u++)
            m = fmaxf(m, tops[u][r]);
        const float base = m == -INFINITY ? 0.0f : m;
#pragma unroll
        for (int u = 0; u < W; u++) {
            const float e = __builtin_amdgcn_exp2f(tops[u][r] - base);
            l += sums[u][r] * e;
            y += *(const w4f *)&part[u][r][d] * e;
        }
        *(w4f *)(a.o + (uint64_t)(s.r0 + s.i0 + r) * a.os + s.h * S::dk + d) = l == 0.0f ? w4f{} : y / l;
    }
}

/* ------------------------------------------------------------- launches --- */

constexpr uint64_t kMostWindowGroups = (1u << 24) - 1;

bool window_fits(uint32_t B, uint32_t max_T, uint32_t H) {
    return (uint64_t)((max_T + 15) / 16) * B * H <= kMostWindowGroups;
}

template <int NS>
static void window(WindowAttention &a, hipStream_t s) {
    a.tiles = (a.max_T + 15) / 16;
    const uint32_t grid = a.B * a.tiles * a.H;
    if (a.p)
        window_few_kernel<NS, true, 4><<<grid, 256, 0, s>>>(a);
    else
        window_few_kernel<NS, false, 4><<<grid, 256, 0, s>>>(a);
}

int launch_window(const WindowCall &c, hipStream_t s) {
    WindowAttention a = {};
    a.o = c.o, a.q = c.q, a.k = c.k, a.v = c.v;
    a.os = c.os, a.qs = c.qs, a.ks = c.ks, a.vs = c.vs;
    a.row0 = c.row0, a.B = c.B, a.rows = c.rows, a.max_T = c.max_T, a.H = c.H, a.G = c.G;
    a.left = c.left, a.right = c.right, a.sinks = c.sinks;
    a.scale = 1.44269504088896340736f / sqrtf((float)c.dk);
    a.p = c.p, a.bias_u = c.bias_u, a.bias_w = c.bias_w;
    a.bw = (uint32_t)c.left + (uint32_t)c.right + 1;
    switch (c.dk / 32) {
    case 1: window<1>(a, s); break;
    case 2: window<2>(a, s); break;
    case 3: window<3>(a, s); break;
    case 4: window<4>(a, s); break;
    default: return -2;
    }
    return hipPeekAtLastError() == hipSuccess ? 0 : -1;
}

}  // namespace pkq8
