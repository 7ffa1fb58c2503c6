/* Attention with a sliding window and sinks over whole segments: every row
 * attends the frames of a window around it and the segment's first few, so an
 * hour of audio in one piece costs its frames times the window. Products and
 * sums in 32 bits, whatever the floats' magnitudes: on the fp32 matrix
 * instruction, which rounds as a fused multiply and add does, or where many rows
 * can share the cutting on the bfloat16 one. */
#include "pieces.h"
#include "q8_internal.h"

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <type_traits>

#pragma clang fp contract(off)

namespace pkq8 {

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

__device__ __forceinline__ v4f wmfma(float x, float y, v4f c) {
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
    v4f c[2 * NS];
    float behind;

    __device__ __forceinline__ void load(const WindowAttention &a, const WindowTile &s, int32_t i, v4f (*at_place)[64]) {
        constexpr uint32_t dk = 32 * NS;
        const uint32_t w = (threadIdx.x & 63) / 16;
        const float *src = a.q + (uint64_t)(s.r0 + min(i, s.T - 1)) * a.qs + s.h * dk + 4 * w;
        behind = 0.0f;
#pragma unroll
        for (int t = 0; t < 2 * NS; t++) {
            const v4f x = *(const v4f *)(src + 16 * t);
            if constexpr (POS) {
                const uint32_t d = s.h * dk + 4 * w + 16 * t;
                c[t] = (x + *(const v4f *)(a.bias_u + d)) * a.scale;
                const v4f p = (x + *(const v4f *)(a.bias_w + d)) * a.scale;
                at_place[t][threadIdx.x & 63] = p;
                if (a.sinks) {
                    const v4f far = *(const v4f *)(a.p + d);
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
__device__ __forceinline__ void window_softmax(v4f (&s)[KT], float &top, float &sum, v4f (&o)[NO]) {
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

/* A row by itself in 64 bits, dimension lane + 64 n of it in y[n]: for the outputs that 32 bits do not hold on their way.
 * Sums of weights and values are before their division up to 2^8 (the slack) and the frames' number times the
 * greatest value, and scores may be beyond floats. Frames whose score is -infinity have no part, and a row without
 * others is 0. Two walks over the frames, a frame a lane for the scores, a dimension a lane for the values: about fifty
 * times what the row costs beside others (the hour below with values of 1e37 in every row 37 ms; where all are no
 * numbers the walks end early). */
template <int NS, bool POS>
__device__ __forceinline__ void window_row(const WindowAttention &a, const WindowTile &s, int32_t i, float (&y)[(NS + 1) / 2]) {
    constexpr int dk = 32 * NS, N = (NS + 1) / 2;
    const int32_t lane = (int32_t)(threadIdx.x & 63);
    const int32_t lo = max(i - a.left, 0), far = min(a.sinks, lo), n = far + min(i + a.right, s.T - 1) - lo + 1;
    const float *q = a.q + (uint64_t)(s.r0 + i) * a.qs + s.h * dk;
    auto frame_of = [&](int32_t k) { return k < far ? k : lo + k - far; };
    auto score_of = [&](int32_t j) {
        const float *key = a.k + (uint64_t)(s.r0 + j) * a.ks + s.g * dk;
        const float *place = a.p + (uint64_t)(uint32_t)max(j - i + a.left, 0) * (a.H * dk) + s.h * dk;
        double score = 0.0;
#pragma unroll 1
        for (int d = 0; d < dk; d += 4) {
            const v4f x = *(const v4f *)(q + d), k = *(const v4f *)(key + d);
            v4f u = {}, w = {}, p = {};
            if constexpr (POS) {
                u = *(const v4f *)(a.bias_u + s.h * dk + d), w = *(const v4f *)(a.bias_w + s.h * dk + d);
                p = *(const v4f *)(place + d);
            }
#pragma unroll
            for (int e = 0; e < 4; e++) {
                score = __builtin_fma((double)x[e] + u[e], (double)k[e], score);
                if constexpr (POS)
                    score = __builtin_fma((double)x[e] + w[e], (double)p[e], score);
            }
        }
        return score * a.scale;
    };
    double top = -INFINITY, sum = 0.0, o[N] = {};
    bool none = false;                      /* a score is no number: no output is */
#pragma unroll 1
    for (int32_t k = 0; k < n && !none; k += 64) {
        const double score = score_of(frame_of(min(k + lane, n - 1)));
        none = __any(score != score);
        top = fmax(top, score);
    }
#pragma unroll
    for (int m = 32; m >= 1; m >>= 1)
        top = fmax(top, __shfl_xor(top, m));
    if (none || __builtin_fabs(top) == INFINITY) {
#pragma unroll
        for (int u = 0; u < N; u++)
            y[u] = !none && top < 0.0 ? 0.0f : __builtin_nanf("");
        return;
    }
    bool all = false;                       /* every output is no number already */
#pragma unroll 1
    for (int32_t k = 0; k < n && !all; k += 64) {
        const double e = k + lane < n ? exp2(score_of(frame_of(min(k + lane, n - 1))) - top) : 0.0;
        sum += e;
#pragma unroll 1
        for (int32_t l = 0; l < 64; l++) {
            const double weight = __shfl(e, l);
            if (weight == 0.0)
                continue;
            const float *v = a.v + (uint64_t)(s.r0 + frame_of(k + l)) * a.vs + s.g * dk;
#pragma unroll
            for (int u = 0; u < N; u++)
                if (lane + 64 * u < dk)
                    o[u] = __builtin_fma(weight, (double)v[lane + 64 * u], o[u]);
        }
        bool mine = true;
#pragma unroll
        for (int u = 0; u < N; u++)
            mine &= o[u] != o[u] || lane + 64 * u >= dk;
        all = __all(mine);
    }
#pragma unroll
    for (int m = 32; m >= 1; m >>= 1)
        sum += __shfl_xor(sum, m);
#pragma unroll
    for (int u = 0; u < N; u++)
        y[u] = (float)(o[u] / sum);
}

/* The lowest 16 bits: the queries that any of a wave's lanes, a query each 16 of them, is in. */
__device__ __forceinline__ uint32_t queries_of(bool mine) {
    const uint64_t lanes = __ballot(mine);
    return (uint32_t)(lanes | lanes >> 16 | lanes >> 32 | lanes >> 48) & 0xffff;
}

__device__ __forceinline__ void wave_sync() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

/* Sixteen rows a tile, W waves to a tile, each a run of its steps of 16 frames:
 * the sinks' steps first, then the window's, which begins at the tile's first
 * frame of it whatever that is a multiple of (no step is taken for alignment).
 * Operands come from memory, 24 KB a step, each load issued into the registers
 * of the step before as those have been used.
 *
 * A frame j's place scores are products with the rows x = left - (row - j) of
 * the table, 31 of them for 16 rows and frames; the first 16 of those are the
 * step before's last, so each step makes 16 more. A lane's are another column's
 * than its scores', so they pass through LDS.
 *
 * An hour (45000 frames, 8 heads of 128, 128 + 128 + 1 frames and 16 sinks, 75.6
 * GFLOP): 799 us, 95 TFLOP/s of the 154 that an fp32 product reaches. The matrix
 * instructions are busy 65% of it, two waves a SIMD or one (4900 and 5400 clocks a
 * step, of which 3100 are theirs). What holds them up is the loads, 24 a step whose
 * results pass into registers: without them the same products take 630; without
 * masks, places' skew and exponentials 765. Keys by lanes that use them took 910 (53
 * cache lookups a load, 16 now). Measured and no faster: loads straight to LDS, a step
 * ahead (840), the sinks merged into the window's steps (820), two chains of products
 * side by side (805), the shared cutting of the kernel below (820: four barriers a
 * step), 32 rows a wave cut into pieces in its registers (850, a wave a SIMD). */
template <int NS, bool POS, int W>
__global__ __launch_bounds__(256, 2) void window_kernel(WindowAttention a) {
    using S = WindowShape<NS>;
    static_assert(W == 1 || W == 4, "a workgroup's four waves have a tile each, or one");
    constexpr int kWaves = 4, kTiles = kWaves / W, kRow = 36;
    __shared__ __attribute__((aligned(16))) float place[POS ? kWaves : 1][16][kRow];
    __shared__ __attribute__((aligned(16))) float rows[kWaves][16][S::dk + 4];
    __shared__ v4f query[POS ? kWaves : 1][S::NT][64];      /* the place's operands, which registers have no room for */
    const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    WindowTile s;
    if (!window_tile<16, kTiles>(a, s, wave / W))
        return;
    const int32_t c = (int32_t)(lane % 16), w = (int32_t)(lane / 16), i = s.i0 + c;
    /* the window's frames [lo, hi] of any of the rows, the sinks [0, far) before them, the steps of both */
    const int32_t lo = max(s.i0 - a.left, 0), hi = min(s.i0 + 15 + a.right, s.T - 1), far = min(a.sinks, lo);
    const int32_t ns = (far + 15) / 16, steps = ns + (hi - lo) / 16 + 1, each = (steps + W - 1) / W;
    const int32_t n0 = min((int32_t)(wave % W) * each, steps), n1 = min(n0 + each, steps);
    const int32_t last = min(i + a.right, s.T - 1);         /* the lane's query's */
    auto first_of = [&](int32_t n) { return n < ns ? 16 * n : lo + 16 * (n - ns); };

    v4f key[2][NS], pos[2][NS], before;
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
                key[half][t] = *(const v4f *)(src + off + 32 * t);
        }
    };
    auto put = [&](const v4f (&x)[2][NS]) {
        wave_sync();
#pragma unroll
        for (int half = 0; half < 2; half++)
#pragma unroll
            for (int t = 0; t < NS; t++)
                *(v4f *)&rows[wave][lr + 8 * half][lc + 32 * t] = x[half][t];
        wave_sync();
    };
    auto operand = [&](int t) { return *(const v4f *)&rows[wave][c][16 * t + 4 * w]; };
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
                pos[half][t] = *(const v4f *)(src + 32 * t);
        }
    };
    auto places = [&]() {
        v4f r = {};
#pragma unroll
        for (int t = 0; t < S::NT; t++) {
            const v4f x = operand(t), y = query[wave][t][lane];
#pragma unroll
            for (int j = 0; j < 4; j++)
                r = wmfma(x[j], y[j], r);
        }
        return r;
    };
    /* the row of the table of the tile's last row and step n's first frame */
    auto place_of = [&](int32_t n) { return first_of(n) - (s.i0 + 15) + a.left; };

    /* the first loads of all */
    const int32_t x0 = place_of(max(n0, ns));
    auto begin = [&]() {
        if constexpr (POS)
            load_places(x0);
        load_keys(n0);
        load_values(n0);
    };
    if (n0 < n1)
        begin();
    WindowQueries<NS, POS> q;
    q.load(a, s, i, query[POS ? wave : 0]);
    float top, sum, odd;                    /* odd: NaN where an output is no number */
    v4f o[2 * NS];
    /* A value that is an infinity or no number gives NaN to every row of the tile, those that do not attend it among them
     * (its product with their 0). So a pass that ends with one is made again with care. */
    bool careful = false;
    for (;;) {
        top = -INFINITY, sum = 0.0f;
#pragma unroll
        for (int n = 0; n < 2 * NS; n++)
            o[n] = v4f{};
        if constexpr (POS) {
            if (n0 < n1) {
                put(pos);
                load_places(x0 + 16);
                before = places();
            }
        }
#pragma unroll 1
        for (int32_t n = n0; n < n1; n++) {
            const int32_t j0 = first_of(n), next = min(n + 1, n1 - 1);
            v4f x = {};
            put(key);
            load_keys(next);
#pragma unroll
            for (int t = 0; t < S::NT; t++) {
                const v4f y = operand(t);
#pragma unroll
                for (int j = 0; j < 4; j++)
                    x = wmfma(y[j], q.c[t][j], x);
            }
            v4f now = {};
            if constexpr (POS) {
                const int32_t x0 = place_of(n);
                put(pos);
                load_places(place_of(max(next, ns)) + 16);
                if (n >= ns && x0 + 16 < (int32_t)a.bw)
                    now = places();
            }
            if (n < ns) {
                x += q.behind;
#pragma unroll
                for (int r = 0; r < 4; r++)
                    x[r] = j0 + 4 * w + r < far ? x[r] : -INFINITY;
            } else {
                if constexpr (POS) {
                    *(v4f *)&place[wave][c][4 * w] = before;
                    *(v4f *)&place[wave][c][16 + 4 * w] = now;
                    before = now;
                    wave_sync();
#pragma unroll
                    for (int r = 0; r < 4; r++) {
                        const float y = place[wave][c][15 - c + 4 * w + r];
                        x[r] += j0 + 4 * w + r < i - a.left ? q.behind : y;
                    }
                    wave_sync();
                }
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    const int32_t j = j0 + 4 * w + r;
                    const bool seen = (j <= last) & ((j >= i - a.left) | (j < a.sinks));
                    x[r] = seen ? x[r] : -INFINITY;
                }
            }
            v4f prob[1] = { x };
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
                                const bool seen = __shfl((int)(x[r] != -INFINITY), 16 * (from / 16) + c);
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
        sum += __shfl_xor(sum, 16);
        sum += __shfl_xor(sum, 32);
        if constexpr (W == 1) {
            const float scale = 1.0f / sum;                 /* of no weight at all: the outputs' 0 times an infinity */
#pragma unroll
            for (int n = 0; n < 2 * NS; n++)
                o[n] *= scale;
        }
        odd = 0.0f;
#pragma unroll
        for (int n = 0; n < 2 * NS; n++)
#pragma unroll
            for (int r = 0; r < 4; r++)
                odd = __builtin_fmaf(o[n][r], 0.0f, odd);
        if (careful || !__any(i < s.T && odd != odd))
            break;
        careful = true;
        begin();
    }
    /* a lane's outputs: VW dimensions next to each other from 16 VW b + VW (4 w + r) on */
    auto output = [&](int b, int r) {
        typename S::vec y;
#pragma unroll
        for (int e = 0; e < S::VW; e++)
            y[e] = o[b * S::VW + e][r];
        return y;
    };
    if constexpr (W == 1) {
        /* outputs that are no number even so: from their row by itself */
        for (uint32_t rows = queries_of(i < s.T && odd != odd); rows; rows &= rows - 1) {
            const int32_t r = __builtin_ctz(rows);
            float y[(NS + 1) / 2];
            window_row<NS, POS>(a, s, s.i0 + r, y);
#pragma unroll
            for (int b = 0; b < S::NB; b++)
#pragma unroll
                for (int e = 0; e < S::VW; e++)
#pragma unroll
                    for (int k = 0; k < 4; k++) {
                        const float again = __shfl(y[16 * S::VW * b / 64], 16 * S::VW * b % 64 + S::VW * (4 * w + k) + e);
                        const float mine = o[b * S::VW + e][k];
                        o[b * S::VW + e][k] = c == r && __builtin_fmaf(mine, 0.0f, 0.0f) != 0.0f ? again : mine;
                    }
        }
        if (i >= s.T)
            return;
        float *to = a.o + (uint64_t)(s.r0 + i) * a.os + s.h * S::dk + S::VW * 4 * w;
#pragma unroll
        for (int b = 0; b < S::NB; b++)
#pragma unroll
            for (int r = 0; r < 4; r++)
                *(typename S::vec *)(to + 16 * S::VW * b + S::VW * r) = output(b, r);
    } else {
        constexpr int kEach = (16 * S::dk / 4 + 255) / 256;
        __shared__ float tops[kWaves][16], sums[kWaves][16];
        __shared__ uint32_t odd_rows;
        if (threadIdx.x == 0)
            odd_rows = 0;
        if (w == 0)
            tops[wave][c] = top, sums[wave][c] = sum;
#pragma unroll
        for (int b = 0; b < S::NB; b++)
#pragma unroll
            for (int r = 0; r < 4; r++)
                *(typename S::vec *)&rows[wave][c][16 * S::VW * b + S::VW * (4 * w + r)] = output(b, r);
        __syncthreads();
        v4f y[kEach];
#pragma unroll
        for (int n = 0; n < kEach; n++) {
            const uint32_t at = threadIdx.x + 256 * n;
            const int32_t r = (int32_t)(at / (S::dk / 4)), d = (int32_t)(at % (S::dk / 4)) * 4;
            if (at >= 16 * S::dk / 4 || s.i0 + r >= s.T)
                continue;
            float m = -INFINITY, l = 0.0f, e[W];
#pragma unroll
            for (int u = 0; u < W; u++)
                m = fmaxf(m, tops[u][r]);
            const float base = m == -INFINITY ? 0.0f : m;
#pragma unroll
            for (int u = 0; u < W; u++) {
                e[u] = __builtin_amdgcn_exp2f(tops[u][r] - base);
                l += sums[u][r] * e[u];
            }
            y[n] = v4f{};
            const float scale = 1.0f / l;
#pragma unroll
            for (int u = 0; u < W; u++)
                y[n] += *(const v4f *)&rows[u][r][d] * (e[u] * scale);
            float none = 0.0f;
#pragma unroll
            for (int k = 0; k < 4; k++)
                none = __builtin_fmaf(y[n][k], 0.0f, none);
            if (none != none)
                atomicOr(&odd_rows, 1u << r);
        }
        __syncthreads();
        float *again = (float *)query;
        static_assert(sizeof query >= 16 * S::dk * sizeof(float), "a tile's rows fit");
        for (uint32_t of = odd_rows; of; of &= of - 1) {
            const int32_t r = __builtin_ctz(of);
            if (r % kWaves != (int32_t)wave)
                continue;
            float x[(NS + 1) / 2];
            window_row<NS, POS>(a, s, s.i0 + r, x);
#pragma unroll
            for (int u = 0; u < (NS + 1) / 2; u++)
                if ((int)lane + 64 * u < S::dk)
                    again[r * S::dk + (int)lane + 64 * u] = x[u];
        }
        if (odd_rows)
            __syncthreads();
#pragma unroll
        for (int n = 0; n < kEach; n++) {
            const uint32_t at = threadIdx.x + 256 * n;
            const int32_t r = (int32_t)(at / (S::dk / 4)), d = (int32_t)(at % (S::dk / 4)) * 4;
            if (at >= 16 * S::dk / 4 || s.i0 + r >= s.T)
                continue;
            if (odd_rows >> r & 1)
#pragma unroll
                for (int k = 0; k < 4; k++)
                    y[n][k] = __builtin_fmaf(y[n][k], 0.0f, 0.0f) != 0.0f ? again[r * S::dk + d + k] : y[n][k];
            *(v4f *)(a.o + (uint64_t)(s.r0 + s.i0 + r) * a.os + s.h * S::dk + d) = y[n];
        }
    }
}

/* Floats from here on round to a bfloat16 infinity. Values of them are taken
 * apart from the others. */
constexpr float kNoPieces = 0x1.ffp127f;

/* Keys are cut at 2^-40 of what they are and queries at 2^40 of it: every finite
 * key has pieces then, and what pieces end at, 2^-133, is 2^-173 of a query and
 * 2^-93 of a key. Against the greatest key that is 2^-45 of a score, and against
 * queries under this bound 2^-43. Queries from it on are taken as no number, which
 * gives each of their scores the care below. */
constexpr float kKeyScale = 0x1p-40f, kQueryScale = 0x1p40f, kMostQuery = 0x1p90f;

/* Values are cut at 2^16 of what they are: the last bit of the smallest, 2^-149,
 * is then a bfloat16's 2^-133. */
constexpr float kValueScale = 0x1p16f;

/* The six products of pieces that count, the smallest first. */
__device__ __forceinline__ v4f product(const Pieces &x, const Pieces &y, v4f acc) {
    acc = mfma(x.p[2], y.p[0], acc);
    acc = mfma(x.p[1], y.p[1], acc);
    acc = mfma(x.p[0], y.p[2], acc);
    acc = mfma(x.p[1], y.p[0], acc);
    acc = mfma(x.p[0], y.p[1], acc);
    return mfma(x.p[0], y.p[0], acc);
}

/* Many rows without positions: 64 rows a workgroup, 16 a wave, 32 frames a step
 * for all of them, on the bfloat16 matrix cores with every float in three pieces
 * (pieces.h): six products take three eighths of the fp32 instructions' time. The
 * cutting takes 11 vector instructions for two floats, more than the products if
 * each wave cut what it uses: so the workgroup cuts a step's keys and values once,
 * into the operands' own order in LDS, and its four waves read them there. Raw,
 * they are loaded a step ahead.
 *
 * Reductions run over 32 indices, eight a quarter of the wave. Scores: lane l
 * has dimensions 32 s + 8 (l / 16) + i of key l % 16 of a run of 16 (two runs a
 * step), queries are the columns. A lane's scores are then its query's with
 * frames 4 (l / 16) + r of both runs, the eight that it gives the second product,
 * whose rows are dimensions 32 b + 2 (l % 16) + d of instruction (b, d).
 *
 * Four segments of 2001 to 3000 frames, 16 heads of 64 to 4 kept ones, 512 frames
 * and 8 sinks, 19.6 GFLOP: 150 to 156 us by the machine, 126 to 131 TFLOP/s (220 us
 * with fp32 instructions); with 2000 frames 390 us, 131 TFLOP/s. Two products' chains
 * side by side were no faster. */
template <int NS>
__global__ __launch_bounds__(256, 2) void window_many_kernel(WindowAttention a) {
    constexpr int dk = 32 * NS, kChunks = 4 * NS;
    constexpr int kEach = (32 * kChunks + 255) / 256;       /* eights of dimensions that a thread cuts */
    __shared__ v8bf key[2][NS][3][64];
    __shared__ v8bf value[NS][2][3][64];
    __shared__ uint32_t odd_step;                           /* the step whose values hold what has no pieces, and one */
    __shared__ uint32_t again;
    WindowTile s;
    if (!window_tile<64, 1>(a, s, 0))
        return;
    const uint32_t lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int32_t c = (int32_t)(lane % 16), w = (int32_t)(lane / 16), iw = s.i0 + 16 * (int32_t)wave, i = iw + c;

    Pieces q[NS];                           /* scores in powers of 2 */
    const float *query = a.q + (uint64_t)(s.r0 + min(i, s.T - 1)) * a.qs + s.h * dk + 8 * w;
    const float query_scale = a.scale * kQueryScale;
#pragma unroll
    for (int t = 0; t < NS; t++) {
        const v4f x = *(const v4f *)(query + 32 * t) * query_scale, y = *(const v4f *)(query + 32 * t + 4) * query_scale;
        float z[8] = { x[0], x[1], x[2], x[3], y[0], y[1], y[2], y[3] };
#pragma unroll
        for (int e = 0; e < 8; e++)
            z[e] = __builtin_fabsf(z[e]) < kMostQuery ? z[e] : __builtin_nanf("");
        q[t] = cut_near(z);
    }
    float top, sum, odd;                    /* odd: NaN where an output is no number */
    v4f o[2 * NS];

    /* the window's frames [lo, hi] of any of the rows, the sinks [0, far) before them, the steps of both */
    const int32_t lo = max(s.i0 - a.left, 0), hi = min(s.i0 + 63 + a.right, s.T - 1), far = min(a.sinks, lo);
    const int32_t ns = (far + 31) / 32, steps = ns + (hi - lo) / 32 + 1;
    auto first_of = [&](int32_t n) { return n < ns ? 32 * n : lo + 32 * (n - ns); };

    /* a step's raw rows: eights of dimensions of a row by threads side by side; of values two dimensions of eight frames,
     * which become an operand as they are */
    v4f raw[kEach][2];
    v2f_c raw_v[8];
    auto load_keys = [&](int32_t j0) {
        const float *src = a.k + (uint64_t)(s.r0 + j0) * a.ks + s.g * dk;
#pragma unroll
        for (int e = 0; e < kEach; e++) {
            const uint32_t n = threadIdx.x + 256 * e;
            const uint32_t off = (uint32_t)min((int32_t)(n / kChunks), s.T - 1 - j0) * (uint32_t)a.ks + 8 * (n % kChunks);
            raw[e][0] = *(const v4f *)(src + off);
            raw[e][1] = *(const v4f *)(src + off + 4);
        }
    };
    auto load_values = [&](int32_t j0) {
        const float *src = a.v + (uint64_t)(s.r0 + j0) * a.vs + s.g * dk + 32 * (wave % NS) + 2 * c;
#pragma unroll
        for (int k = 0; k < 8; k++)
            raw_v[k] = *(const v2f_c *)(src + (uint32_t)min(16 * (k / 4) + 4 * w + k % 4, s.T - 1 - j0) * (uint32_t)a.vs);
    };
    /* rows cut into operands: chunk n % kChunks of row n / kChunks, at a place of its run of 16 that lets threads side by
     * side write to banks of their own */
    auto slot_of = [&](uint32_t row, uint32_t chunk) {
        return 16 * (chunk % 4) + (row % 16 ^ (chunk * (NS == 1 ? 4 : NS == 2 ? 2 : 1)) % 16);
    };
    auto put = [&](const v4f (&x)[kEach][2]) {
#pragma unroll
        for (int e = 0; e < kEach; e++) {
            const uint32_t n = threadIdx.x + 256 * e, row = n / kChunks, chunk = n % kChunks;
            const v4f u = x[e][0] * kKeyScale, v = x[e][1] * kKeyScale;
            const float z[8] = { u[0], u[1], u[2], u[3], v[0], v[1], v[2], v[3] };
            const Pieces y = cut_near(z);
            if (32 * kChunks % 256 == 0 || n < 32 * kChunks)
#pragma unroll
                for (int k = 0; k < 3; k++)
                    key[row / 16][chunk / 4][k][slot_of(row, chunk)] = y.p[k];
        }
    };
    auto operand = [&](int kt, int t) {
        Pieces x;
#pragma unroll
        for (int k = 0; k < 3; k++)
            x.p[k] = key[kt][t][k][slot_of((uint32_t)c, 4 * t + (uint32_t)w)];
        return x;
    };
    auto put_values = [&]() {
        if (wave < NS)
#pragma unroll
            for (int d = 0; d < 2; d++) {
                float z[8];
#pragma unroll
                for (int k = 0; k < 8; k++)
                    z[k] = raw_v[k][d] * kValueScale;
                const Pieces y = cut_near(z);
#pragma unroll
                for (int k = 0; k < 3; k++)
                    value[wave][d][k][lane] = y.p[k];
            }
    };
    /* With care: an infinity or a NaN among the values, or a float that has no pieces, may be only some rows': the others
     * got its product with their 0. So the product is made without it, and the step told. */
    auto leave_out = [&](int32_t n) {
        bool odd = false;
#pragma unroll
        for (int k = 0; k < 8; k++)
#pragma unroll
            for (int d = 0; d < 2; d++) {
                const bool has = __builtin_fabsf(raw_v[k][d] * kValueScale) < kNoPieces;
                odd |= !has;
                raw_v[k][d] = has ? raw_v[k][d] : 0.0f;
            }
        if (odd)
            odd_step = (uint32_t)n + 1;
    };
    /* of the lane's eight of a step's 32 frames that of frame k, as the query's lane has it */
    auto of_frame = [&](const v4f (&x)[2], int32_t k) {
        float y = x[0][0];
#pragma unroll
        for (int n = 1; n < 8; n++)
            y = k / 16 * 4 + k % 4 == n ? x[n / 4][n % 4] : y;
        return __shfl(y, 16 * (k / 4 % 4) + c);
    };
    auto add_left_out = [&](int32_t j0, const v4f (&x)[2], const v4f (&e)[2]) {
#pragma unroll 1
        for (int32_t k = 0; k < 32 && j0 + k < s.T; k++) {
            const float mine = of_frame(e, k), score = of_frame(x, k);
            const float *src = a.v + (uint64_t)(s.r0 + j0 + k) * a.vs + s.g * dk + 8 * w;
            if (score != -INFINITY)
#pragma unroll
                for (int b = 0; b < NS; b++)
#pragma unroll
                    for (int r = 0; r < 4; r++)
#pragma unroll
                        for (int d = 0; d < 2; d++) {
                            const float y = src[32 * b + 2 * r + d] * kValueScale;
                            if (!(__builtin_fabsf(y) < kNoPieces))
                                o[2 * b + d][r] += mine * y;
                        }
        }
    };
    /* Scores that are no number are made again from the floats themselves: an infinite key has pieces that are none, and
     * its score may be -infinity. */
    auto score_again = [&](int32_t j0, v4f (&x)[2]) {
        uint32_t none = 0;
#pragma unroll
        for (int n = 0; n < 8; n++)
            none |= x[n / 4][n % 4] != x[n / 4][n % 4] ? 1u << n : 0;
        if (!__any(none))
            return;
#pragma unroll 1
        for (int32_t k = 0; k < 32 && j0 + k < s.T; k++) {
            const int32_t at = k / 16 * 4 + k % 4;
            const bool mine = w == k / 4 % 4 && (none >> at & 1);
            if (!__any(mine))
                continue;
            const float *key = a.k + (uint64_t)(s.r0 + j0 + k) * a.ks + s.g * dk + 8 * w;
            float score = 0.0f;
#pragma unroll 1
            for (int t = 0; t < 2 * NS; t++) {
                const v4f y = *(const v4f *)(query + 32 * (t / 2) + t % 2 * 4) * a.scale;
                const v4f z = *(const v4f *)(key + 32 * (t / 2) + t % 2 * 4);
#pragma unroll
                for (int e = 0; e < 4; e++)
                    score = __builtin_fmaf(y[e], z[e], score);
            }
            score += __shfl_xor(score, 16);
            score += __shfl_xor(score, 32);
#pragma unroll
            for (int n = 0; n < 8; n++)
                x[n / 4][n % 4] = mine && n == at ? score : x[n / 4][n % 4];
        }
    };
    if (threadIdx.x == 0)
        odd_step = again = 0;
    auto pass = [&](auto careful) {
        top = -INFINITY, sum = 0.0f;
#pragma unroll
        for (int n = 0; n < 2 * NS; n++)
            o[n] = v4f{};
        if constexpr (!careful) {
            load_keys(first_of(0));
            load_values(first_of(0));
        }
#pragma unroll 1
        for (int32_t n = 0; n < steps; n++) {
            const int32_t j0 = first_of(n), next = first_of(min(n + 1, steps - 1));
            if constexpr (careful) {                /* not ahead: the care needs the registers */
                load_keys(j0);
                load_values(j0);
            }
            __syncthreads();
            put(raw);
            if constexpr (careful)
                leave_out(n);
            put_values();
            if constexpr (!careful) {
                load_keys(next);
                load_values(next);
            }
            __syncthreads();
            /* whether any of the wave's rows attends any of the frames */
            const bool busy = n < ns || (j0 + 31 >= iw - a.left && j0 <= iw + 15 + a.right) || j0 < a.sinks;
            if (!busy)
                continue;
            v4f x[2] = {};
#pragma unroll
            for (int kt = 0; kt < 2; kt++)
#pragma unroll
                for (int t = 0; t < NS; t++)
                    x[kt] = product(operand(kt, t), q[t], x[kt]);
            if (n < ns) {
#pragma unroll
                for (int k = 0; k < 8; k++)
                    x[k / 4][k % 4] = j0 + 16 * (k / 4) + 4 * w + k % 4 < far ? x[k / 4][k % 4] : -INFINITY;
            } else if (j0 < iw + 15 - a.left || j0 + 31 > min(iw + a.right, s.T - 1)) {
                const int32_t last = min(i + a.right, s.T - 1);
#pragma unroll
                for (int k = 0; k < 8; k++) {
                    const int32_t j = j0 + 16 * (k / 4) + 4 * w + k % 4;
                    const bool seen = (j <= last) & ((j >= i - a.left) | (j < a.sinks));
                    x[k / 4][k % 4] = seen ? x[k / 4][k % 4] : -INFINITY;
                }
            }
            if constexpr (careful)
                score_again(j0, x);
            v4f e[2] = { x[0], x[1] };
            window_softmax<2, 2 * NS>(e, top, sum, o);
            if constexpr (careful)
                if (odd_step == (uint32_t)n + 1)
                    add_left_out(j0, x, e);
            const float z[8] = { e[0][0], e[0][1], e[0][2], e[0][3], e[1][0], e[1][1], e[1][2], e[1][3] };
            const Pieces prob = cut_near(z);
#pragma unroll
            for (int b = 0; b < NS; b++)
#pragma unroll
                for (int d = 0; d < 2; d++) {
                    Pieces y;
#pragma unroll
                    for (int k = 0; k < 3; k++)
                        y.p[k] = value[b][d][k][lane];
                    o[2 * b + d] = product(y, prob, o[2 * b + d]);
                }
        }
        sum += __shfl_xor(sum, 16);
        sum += __shfl_xor(sum, 32);
        const float scale = 1.0f / sum * (1.0f / kValueScale);      /* of no weight at all: the outputs' 0 times an infinity */
        odd = 0.0f;
#pragma unroll
        for (int n = 0; n < 2 * NS; n++) {
            o[n] *= scale;
#pragma unroll
            for (int r = 0; r < 4; r++)
                odd = __builtin_fmaf(o[n][r], 0.0f, odd);
        }
    };
    pass(std::false_type());
    /* An infinity or a NaN among the outputs: once more then, with care, and what is none even so from its row by itself. */
    if (i < s.T && odd != odd)
        again = 1;
    __syncthreads();
    if (__builtin_expect(again, 0)) {
        pass(std::true_type());
        for (uint32_t rows = queries_of(i < s.T && odd != odd); rows; rows &= rows - 1) {
            const int32_t row = __builtin_ctz(rows);
            float y[(NS + 1) / 2];
            window_row<NS, false>(a, s, iw + row, y);
#pragma unroll
            for (int b = 0; b < NS; b++)
#pragma unroll
                for (int r = 0; r < 4; r++)
#pragma unroll
                    for (int d = 0; d < 2; d++) {
                        const float y1 = __shfl(y[b / 2], 32 * (b % 2) + 8 * w + 2 * r + d), mine = o[2 * b + d][r];
                        o[2 * b + d][r] = c == row && __builtin_fmaf(mine, 0.0f, 0.0f) != 0.0f ? y1 : mine;
                    }
        }
    }
    if (i >= s.T)
        return;
    float *to = a.o + (uint64_t)(s.r0 + i) * a.os + s.h * dk + 8 * w;
#pragma unroll
    for (int b = 0; b < NS; b++)
#pragma unroll
        for (int r = 0; r < 4; r += 2)
            *(v4f *)(to + 32 * b + 2 * r) = v4f{ o[2 * b][r], o[2 * b + 1][r], o[2 * b][r + 1], o[2 * b + 1][r + 1] };
}

/* ------------------------------------------------------------- launches --- */

constexpr uint64_t kMostWindowGroups = (1u << 24) - 1;

bool window_fits(uint32_t B, uint32_t max_T, uint32_t H) {
    return (uint64_t)((max_T + 15) / 16) * B * H <= kMostWindowGroups;
}

/* A SIMD's waves hardly overlap here (an fp32 matrix instruction holds up every
 * vector one: four of those between two make 53 clocks of its 32), so what counts
 * is how many waves the fullest SIMD has and how many steps each takes, with
 * three for what comes before and after them. Four waves a tile of 8 heads of
 * 128 with 129 + 128 frames of window: 192 tiles 18.8 us, one wave 43.2; 512 31.3
 * and 44.0; 752 51.0 and 44.2; 1024 56.0 and 45.5; 3000 151 and 120. With 70 + 13
 * frames: 512 19.2 and 23.1, 752 32.5 and 24.0; with 511: 752 70.6 and 77.1, 1504
 * 120 and 136, 3000 232 and 219. */
static bool tile_split(uint64_t tiles, uint64_t steps) {
    return (4 * tiles + 1023) / 1024 * ((steps + 3) / 4 + 3) <= (tiles + 1023) / 1024 * (steps + 3);
}

/* Without positions four waves a tile, or from this many tiles on 64 rows a
 * workgroup. Heads of 128 with 257 frames: 752 tiles 31.1 and 31.9 us, 1024 36.1 and
 * 32.1, 3000 91.7 and 67.6; heads of 64: 1024 18.6 and 21.2, 1504 25.7 and 26.6,
 * 3000 47.8 and 35.5; of 96 1024 30.7 and 26.3; of 32 1504 17.1 and 20.6, 3000 29.9
 * and 26.8. */
constexpr uint64_t many_from(int NS) { return NS >= 3 ? 1024 : 2048; }

template <int NS>
static void window(WindowAttention &a, hipStream_t s) {
    a.tiles = (a.max_T + 15) / 16;
    /* segments are up to max_T long, and together no more than the rows */
    const uint64_t tiles = std::min((uint64_t)a.B * a.tiles, (uint64_t)a.rows / 16 + a.B) * a.H;
    const uint32_t reach = std::min((uint32_t)(a.left + a.right) + 16, a.max_T + 15);
    if (a.p) {
        if (tile_split(tiles, reach / 16 + ((uint32_t)a.sinks + 15) / 16))
            window_kernel<NS, true, 4><<<a.B * a.tiles * a.H, 256, 0, s>>>(a);
        else
            window_kernel<NS, true, 1><<<a.B * ((a.tiles + 3) / 4) * a.H, 256, 0, s>>>(a);
    } else if (tiles < many_from(NS)) {
        window_kernel<NS, false, 4><<<a.B * a.tiles * a.H, 256, 0, s>>>(a);
    } else {
        a.tiles = (a.max_T + 63) / 64;
        window_many_kernel<NS><<<a.B * a.tiles * a.H, 256, 0, s>>>(a);
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
