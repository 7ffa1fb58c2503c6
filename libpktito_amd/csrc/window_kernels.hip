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
    const float *p, *bias_u, *bias_w;       /* p's first row the distance left's; NULL: no positions */
    const int32_t *row0;
    uint64_t os, qs, ks, vs;
    uint32_t B, rows, max_T, H, G;
    int32_t left, right, sinks;             /* clipped to what can occur */
    uint32_t bw;                            /* the rows of p, left + right + 1 */
    uint32_t tiles;                         /* a segment's tiles of rows */
    float scale;                            /* log2(e) / sqrt(dk) */
};

/* A wave's part: rows [i0, i0 + R) of a segment of T at row r0, one head; its
 * workgroup has N tiles one after another. */
struct WindowTile {
    int32_t r0, T, i0;
    uint32_t h, g;
};

template <int R, int N>
__device__ __forceinline__ bool window_tile(const WindowAttention &a, WindowTile &s, uint32_t tile) {
    uint32_t i = blockIdx.x;
    s.h = i % a.H, i /= a.H;
    s.g = s.h / (a.H / a.G);
    const uint32_t groups = (a.tiles + N - 1) / N;
    s.i0 = (int32_t)(i % groups * N + tile) * R;
    const uint32_t b = i / groups;
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
    w4f c[2 * NS];
    float behind;

    __device__ __forceinline__ void load(const WindowAttention &a, const WindowTile &s, int32_t i, w4f (*at_place)[64]) {
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
                const w4f p = (x + *(const w4f *)(a.bias_w + d)) * a.scale;
                at_place[t][threadIdx.x & 63] = p;
                if (a.sinks) {
                    const w4f far = *(const w4f *)(a.p + d);
#pragma unroll
                    for (int j = 0; j < 4; j++)
                        behind = __builtin_fmaf(p[j], far[j], behind);
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
        const float now = best > top + kWindowSlack ? best : top;   /* by the query's own scores: no other row's bits */
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

/* Sixteen rows a tile, W waves to a tile, each a run of its steps of 16 frames:
 * the sinks' steps first, then the window's, which begins at the tile's first
 * frame of it whatever that is a multiple of (no step is taken for alignment).
 * Operands come straight from memory: 24 KB a step for 96 matrix instructions,
 * whose 3072 cycles hide the loads of the step after, each issued into the
 * registers of this one's as those have been used.
 *
 * A frame j's place scores are products with the rows x = left - (row - j) of
 * the table, 31 of them for 16 rows and frames; the first 16 of those are the
 * step before's last, so each step makes 16 more. A lane's are another column's
 * than its scores', so they pass through LDS. */
template <int NS, bool POS, int W>
__global__ __launch_bounds__(W > 4 ? 64 * W : 256, 2) void window_kernel(WindowAttention a) {
    using S = WindowShape<NS>;
    constexpr int kWaves = W > 4 ? W : 4, kTiles = kWaves / W, kRow = 36;
    __shared__ __attribute__((aligned(16))) float place[POS ? kWaves : 1][16][kRow];
    __shared__ __attribute__((aligned(16))) float rows[kWaves][16][S::dk + 4];
    __shared__ w4f query[POS ? kWaves : 1][S::NT][64];      /* the place's operands, which registers have no room for */
    const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    WindowTile s;
    if (!window_tile<16, kTiles>(a, s, wave / W))
        return;
    const int32_t c = (int32_t)(lane % 16), w = (int32_t)(lane / 16), i = s.i0 + c;
    WindowQueries<NS, POS> q;
    q.load(a, s, i, query[POS ? wave : 0]);
    float top, sum;
    w4f o[2 * NS];

    /* the window's frames [lo, hi] of any of the rows, the sinks [0, far) before them, the steps of both */
    const int32_t lo = max(s.i0 - a.left, 0), hi = min(s.i0 + 15 + a.right, s.T - 1), far = min(a.sinks, lo);
    const int32_t ns = (far + 15) / 16, steps = ns + (hi - lo) / 16 + 1, each = (steps + W - 1) / W;
    const int32_t n0 = min((int32_t)(wave % W) * each, steps), n1 = min(n0 + each, steps);
    const int32_t last = min(i + a.right, s.T - 1);         /* the lane's query's */
    auto first_of = [&](int32_t n) { return n < ns ? 16 * n : lo + 16 * (n - ns); };

    w4f key[2][NS], pos[2][NS], before;
    typename S::vec v[4][S::NB];
    /* Sixteen rows of keys or of the table, 128 bytes of one to eight lanes (to a lane of its own the 16 bytes that the
     * instruction wants of it, each row's would be cache lookups of their own, four times as many), put where operands are
     * read from. Offsets from a step's first row are 32 bits, as no stride passes 2^25 floats. */
    const int32_t lr = (int32_t)(lane / 8), lc = 4 * (int32_t)(lane % 8);
    auto load_keys = [&](int32_t n) {
        const int32_t j0 = first_of(n);
        const float *src = a.k + (uint64_t)(s.r0 + j0) * a.ks + s.g * S::dk + lc;
#pragma unroll
        for (int half = 0; half < 2; half++) {
            const uint32_t off = (uint32_t)min(lr + 8 * half, s.T - 1 - j0) * (uint32_t)a.ks;
#pragma unroll
            for (int t = 0; t < NS; t++)
                key[half][t] = *(const w4f *)(src + off + 32 * t);
        }
    };
    auto put = [&](const w4f (&x)[2][NS]) {
        wave_sync();
#pragma unroll
        for (int half = 0; half < 2; half++)
#pragma unroll
            for (int t = 0; t < NS; t++)
                *(w4f *)&rows[wave][lr + 8 * half][lc + 32 * t] = x[half][t];
        wave_sync();
    };
    auto operand = [&](int t) { return *(const w4f *)&rows[wave][c][16 * t + 4 * w]; };
    const uint32_t value_off = 4 * (uint32_t)w * (uint32_t)a.vs + S::VW * c;
    auto load_values = [&](int32_t n) {
        const int32_t j0 = first_of(n);
        const float *src = a.v + (uint64_t)(s.r0 + j0) * a.vs + s.g * S::dk;
#pragma unroll
        for (int r = 0; r < 4; r++) {
            const uint32_t off = j0 + 15 < s.T ? value_off + r * (uint32_t)a.vs
                                               : (uint32_t)min(4 * w + r, s.T - 1 - j0) * (uint32_t)a.vs + S::VW * c;
#pragma unroll
            for (int b = 0; b < S::NB; b++)
                v[r][b] = *(const typename S::vec *)(src + off + 16 * S::VW * b);
        }
    };
    /* the table's rows x to x + 15 */
    auto load_places = [&](int32_t x) {
#pragma unroll
        for (int half = 0; half < 2; half++) {
            const uint32_t row = (uint32_t)cache_clip(x + lr + 8 * half, 0, (int32_t)a.bw - 1);
            const float *src = a.p + (uint64_t)row * (a.H * S::dk) + s.h * S::dk + lc;
#pragma unroll
            for (int t = 0; t < NS; t++)
                pos[half][t] = *(const w4f *)(src + 32 * t);
        }
    };
    auto places = [&]() {
        w4f r = {};
#pragma unroll
        for (int t = 0; t < S::NT; t++) {
            const w4f x = operand(t), y = query[wave][t][lane];
#pragma unroll
            for (int j = 0; j < 4; j++)
                r = wmfma(x[j], y[j], r);
        }
        return r;
    };
    /* the row of the table of the tile's last row and step n's first frame */
    auto place_of = [&](int32_t n) { return first_of(n) - (s.i0 + 15) + a.left; };

    /* A value that is an infinity or no number gives NaN to every row of the tile, those that do not attend it among them
     * (its product with their 0). So a pass that ends with one is made again with care. */
    bool careful = false;
    for (;;) {
    top = -INFINITY, sum = 0.0f;
#pragma unroll
    for (int n = 0; n < 2 * NS; n++)
        o[n] = w4f{};
    if (n0 < n1) {
        load_keys(n0);
        load_values(n0);
        if constexpr (POS) {
            const int32_t n = max(n0, ns);
            load_places(place_of(n));
            put(pos);
            before = places();
            load_places(place_of(n) + 16);
        }
    }
#pragma unroll 1
    for (int32_t n = n0; n < n1; n++) {
        const int32_t j0 = first_of(n), next = min(n + 1, n1 - 1);
        w4f x[1] = {};
        put(key);
        load_keys(next);
#pragma unroll
        for (int t = 0; t < S::NT; t++) {
            const w4f y = operand(t);
#pragma unroll
            for (int j = 0; j < 4; j++)
                x[0] = wmfma(y[j], q.c[t][j], x[0]);
        }
        w4f now = {};
        if constexpr (POS) {
            const int32_t x0 = place_of(n);
            put(pos);
            load_places(place_of(max(next, ns)) + 16);
            if (n >= ns && x0 + 16 < (int32_t)a.bw)
                now = places();
        }
        if (n < ns) {
            x[0] += q.behind;
#pragma unroll
            for (int r = 0; r < 4; r++)
                x[0][r] = j0 + 4 * w + r < far ? x[0][r] : -INFINITY;
        } else {
            if constexpr (POS) {
                *(w4f *)&place[wave][c][4 * w] = before;
                *(w4f *)&place[wave][c][16 + 4 * w] = now;
                before = now;
                wave_sync();
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    const float y = place[wave][c][15 - c + 4 * w + r];
                    x[0][r] += j0 + 4 * w + r < i - a.left ? q.behind : y;
                }
                wave_sync();
            }
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const int32_t j = j0 + 4 * w + r;
                const bool seen = (j <= last) & ((j >= i - a.left) | (j < a.sinks));
                x[0][r] = seen ? x[0][r] : -INFINITY;
            }
        }
        w4f prob[1] = { x[0] };
        window_softmax<1, 2 * NS>(prob, top, sum, o);
        if (__builtin_expect(careful, 0)) {
            /* the product without them, and each added to the rows that attend it */
#pragma unroll
            for (int r = 0; r < 4; r++)
#pragma unroll
                for (int b = 0; b < S::NB; b++)
#pragma unroll
                    for (int e = 0; e < S::VW; e++) {
                        const float y = v[r][b][e];
                        const bool bad = __builtin_fmaf(y, 0.0f, 0.0f) != 0.0f;
                        v[r][b][e] = bad ? 0.0f : y;
                        uint64_t who = __ballot(bad);
                        while (who) {
                            const int from = __builtin_ctzll(who);
                            who &= who - 1;
                            const float value = __shfl(y, from);
                            const float mine = __shfl(prob[0][r], 16 * (from / 16) + c);
                            const bool seen = __shfl((int)(x[0][r] != -INFINITY), 16 * (from / 16) + c);
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
        for (int r = 0; r < 4; r++)
#pragma unroll
            for (int b = 0; b < S::NB; b++)
#pragma unroll
                for (int e = 0; e < S::VW; e++)
                    o[b * S::VW + e] = wmfma(v[r][b][e], prob[0][r], o[b * S::VW + e]);
        load_values(next);
    }
    float odd = 0.0f;                       /* NaN where an output is no number */
#pragma unroll
    for (int n = 0; n < 2 * NS; n++)
#pragma unroll
        for (int r = 0; r < 4; r++)
            odd = __builtin_fmaf(o[n][r], 0.0f, odd);
    if (careful || !__any(odd != odd))
        break;
    careful = true;
    }
    sum += __shfl_xor(sum, 16);
    sum += __shfl_xor(sum, 32);
    /* a lane's outputs: VW dimensions next to each other from 16 VW b + VW (4 w + r) on */
    auto output = [&](int b, int r) {
        typename S::vec y;
#pragma unroll
        for (int e = 0; e < S::VW; e++)
            y[e] = o[b * S::VW + e][r];
        return y;
    };
    if constexpr (W == 1) {
        if (i >= s.T)
            return;
        const float scale = sum == 0.0f ? 0.0f : 1.0f / sum;
        float *to = a.o + (uint64_t)(s.r0 + i) * a.os + s.h * S::dk + S::VW * 4 * w;
#pragma unroll
        for (int b = 0; b < S::NB; b++)
#pragma unroll
            for (int r = 0; r < 4; r++)
                *(typename S::vec *)(to + 16 * S::VW * b + S::VW * r) = output(b, r) * scale;
    } else {
        __shared__ float tops[kWaves][16], sums[kWaves][16];
        if (w == 0)
            tops[wave][c] = top, sums[wave][c] = sum;
#pragma unroll
        for (int b = 0; b < S::NB; b++)
#pragma unroll
            for (int r = 0; r < 4; r++)
                *(typename S::vec *)&rows[wave][c][16 * S::VW * b + S::VW * (4 * w + r)] = output(b, r);
        __syncthreads();
        const uint32_t w0 = wave / W * W;
        for (uint32_t n = threadIdx.x % (64 * W); n < 16 * S::dk / 4; n += 64 * W) {
            const int32_t r = (int32_t)(n / (S::dk / 4)), d = (int32_t)(n % (S::dk / 4)) * 4;
            if (s.i0 + r >= s.T)
                continue;
            float m = -INFINITY, l = 0.0f;
            w4f y = {};
#pragma unroll
            for (int u = 0; u < W; u++)
                m = fmaxf(m, tops[w0 + u][r]);
            const float base = m == -INFINITY ? 0.0f : m;
#pragma unroll
            for (int u = 0; u < W; u++) {
                const float e = __builtin_amdgcn_exp2f(tops[w0 + u][r] - base);
                l += sums[w0 + u][r] * e;
                y += *(const w4f *)&rows[w0 + u][r][d] * e;
            }
            *(w4f *)(a.o + (uint64_t)(s.r0 + s.i0 + r) * a.os + s.h * S::dk + d) = l == 0.0f ? w4f{} : y / l;
        }
    }
}

/* ------------------------------------------------------------- launches --- */

constexpr uint64_t kMostWindowGroups = (1u << 24) - 1;

bool window_fits(uint32_t B, uint32_t max_T, uint32_t H) {
    return (uint64_t)((max_T + 15) / 16) * B * H <= kMostWindowGroups;
}

template <int NS, int W>
static void window(const WindowAttention &a, hipStream_t s) {
    constexpr uint32_t kTiles = W > 4 ? 1 : 4 / W;
    const uint32_t grid = a.B * ((a.tiles + kTiles - 1) / kTiles) * a.H;
    (a.p ? window_kernel<NS, true, W> : window_kernel<NS, false, W>)<<<grid, W > 4 ? 64 * W : 256, 0, s>>>(a);
}

template <int NS>
static void window(WindowAttention &a, hipStream_t s) {
    a.tiles = (a.max_T + 15) / 16;
    const char *e = getenv("PKW");
    switch (e ? atoi(e) : 4) {
    case 1: window<NS, 1>(a, s); break;
    case 2: window<NS, 2>(a, s); break;
    case 4: window<NS, 4>(a, s); break;
    default: window<NS, 8>(a, s); break;
    }
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
