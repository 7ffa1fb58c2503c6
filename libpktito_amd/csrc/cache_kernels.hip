/* The 4-bit cache of keys and values (cache_layout.h has its layout): the
 * write of a chunk's keys and values, their read-back, the attention of a
 * chunk's rows to everything kept, and the move of pages. */
#include "cache_layout.h"
#include "q8_device.h"
#include "q8_internal.h"

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>

#pragma clang fp contract(off)

namespace pkq8 {

typedef __bf16 v2bf __attribute__((ext_vector_type(2)));
typedef __bf16 v8bf __attribute__((ext_vector_type(8)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef float v4f_u __attribute__((ext_vector_type(4), aligned(4)));
typedef float v2f_c __attribute__((ext_vector_type(2)));
typedef uint32_t v4u __attribute__((ext_vector_type(4)));
typedef uint32_t v2u __attribute__((ext_vector_type(2)));

__device__ __forceinline__ CacheSpan span_of(const CacheStreams &s, uint32_t b) {
    return cache_span(s, s.row0[b], s.row0[b + 1], s.len[b]);
}

/* An 8 x 8 square of codes turned over: dword i's nibble n and dword n's
 * nibble i change places. Eight frames' codes of eight dimensions become eight
 * dimensions' codes of eight frames, and back. */
__device__ __forceinline__ void turn(uint32_t (&a)[8]) {
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const uint32_t t = (a[i] >> 16 ^ a[i + 4]) & 0x0000ffffu;
        a[i + 4] ^= t, a[i] ^= t << 16;
    }
#pragma unroll
    for (int i = 0; i < 8; i++)
        if (!(i & 2)) {
            const uint32_t t = (a[i] >> 8 ^ a[i + 2]) & 0x00ff00ffu;
            a[i + 2] ^= t, a[i] ^= t << 8;
        }
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
        const uint32_t t = (a[i] >> 4 ^ a[i + 1]) & 0x0f0f0f0fu;
        a[i + 1] ^= t, a[i] ^= t << 4;
    }
}

/* Eight values' codes at scale d. The hardware's rounding to e2m1 takes x / d
 * only as a rounded product with 1 / d, off by up to 2^-23 of itself; where it
 * gives one code a little below and a little above, that is the code, and
 * elsewhere (one value in 10^5, every tie among them) the exact comparisons
 * decide: 5 instructions a value in place of 18. */
__device__ __forceinline__ uint32_t codes(v4f a, v4f b, float d) {
    const float id = 1.0f / d;
    uint32_t c[2];
#pragma unroll
    for (int i = 0; i < 2; i++) {
        const float s = id * (i ? 1.0f + 0x1p-20f : 1.0f - 0x1p-20f);
        const v4f x = a * s, y = b * s;
        c[i] = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0u, x[0], x[1], 1.0f, 0);
        c[i] = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c[i], x[2], x[3], 1.0f, 1);
        c[i] = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c[i], y[0], y[1], 1.0f, 2);
        c[i] = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c[i], y[2], y[3], 1.0f, 3);
    }
    if (c[0] != c[1]) {
        c[0] = 0;
#pragma unroll
        for (int j = 0; j < 4; j++)
            c[0] |= cache_code(a[j], d) << 4 * j | cache_code(b[j], d) << (16 + 4 * j);
    }
    /* no sign without a magnitude */
    const uint32_t some = (c[0] | c[0] >> 1 | c[0] >> 2) & 0x11111111u;
    return c[0] & (0x77777777u | some << 3);
}

/* The part of a stream's frames [len, len + T) that a workgroup has: page pg of
 * the stream, frames [f0, f1) of it, the page's record if it has one. */
struct PagePart {
    CacheSpan sp;
    int32_t base, f0, f1, id;
    uint8_t *rec;
};

__device__ __forceinline__ bool part_of(uint8_t *data, uint32_t pages, uint32_t G, uint32_t dk, const CacheStreams &st,
                                        PagePart &p) {
    const uint32_t g = blockIdx.x, b = blockIdx.z;
    p.sp = span_of(st, b);
    const int32_t pg = p.sp.len / (int32_t)kPage + (int32_t)blockIdx.y;
    p.base = pg * (int32_t)kPage;
    p.f0 = max(p.sp.len - p.base, 0), p.f1 = min(p.sp.len + p.sp.T - p.base, (int32_t)kPage);
    if (p.f0 >= p.f1)
        return false;
    p.id = pg < (int32_t)st.max_pages ? st.table[(uint64_t)b * st.max_pages + pg] : -1;
    p.rec = cache_page_ok(p.id, pages) ? data + ((uint64_t)p.id * G + g) * cache_record(dk) : nullptr;
    return true;
}

constexpr uint32_t kCodeRow = kMaxCacheDk / 8 + 1;  /* dwords of a frame's codes in LDS, and one against bank conflicts */

/* ---------------------------------------------------------------- write --- */

/* A workgroup writes one page's part of a stream's new frames for one kept
 * head: 16 lanes a frame, eight dimensions a lane, so that a frame's largest
 * magnitude is four steps over its lanes and its codes a dword a lane. Every
 * load is issued before the first code is made. Keys go straight to their
 * rows. Values are turned over in LDS, eight frames by eight dimensions a
 * thread, into the record's own order, and stored 16 bytes a lane; what a
 * chunk covers in part keeps its other frames' codes (a lane's 16 bytes read,
 * merged and stored by it alone, so a frame that shares a byte with the one
 * before it is no race).
 *
 * 48 segments of 250 to 384 frames, 142 MB: 36 us, 3.9 TB/s, a third of it the
 * codes' instructions; a wave a frame and two dimensions a lane took 61, exact
 * comparisons alone 41. 64 streams of two frames: 5 us, three round trips (the
 * stream, its page and rows, the codes around the new ones). */
__global__ __launch_bounds__(256) void cache_write_kernel(uint8_t *data, uint32_t pages, uint32_t G, uint32_t dk,
                                                          CacheStreams st, const float *__restrict__ k, uint64_t ks,
                                                          const float *__restrict__ v, uint64_t vs) {
    __shared__ uint32_t code[kPage][kCodeRow];
    __shared__ v4u image[kPage * kMaxCacheDk / 2 / 16];
    PagePart p;
    if (!part_of(data, pages, G, dk, st, p))
        return;
    const uint32_t part = threadIdx.x % 16, g = blockIdx.x;
    const bool in = part < dk / 8;
    const int32_t fa = p.f0 + (int32_t)(threadIdx.x / 16);
    v4f x[2][4][2] = {};
#pragma unroll
    for (int i = 0; i < 4; i++)
        if (in && fa + 16 * i < p.f1) {
            const uint64_t row = (uint64_t)(p.sp.r0 + p.base + fa + 16 * i - p.sp.len);
            const v4f *kp = (const v4f *)(k + row * ks + g * dk + 8 * part);
            const v4f *vp = (const v4f *)(v + row * vs + g * dk + 8 * part);
            x[0][i][0] = __builtin_nontemporal_load(kp), x[0][i][1] = __builtin_nontemporal_load(kp + 1);
            x[1][i][0] = __builtin_nontemporal_load(vp), x[1][i][1] = __builtin_nontemporal_load(vp + 1);
        }
    if (!p.rec)
        return;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const int32_t f = fa + 16 * i;
        if (f - (int32_t)(threadIdx.x / 16) >= p.f1)
            break;                          /* all of the workgroup's, so the lanes stay together */
#pragma unroll
        for (int which = 0; which < 2; which++) {
            const v4f a = x[which][i][0], b = x[which][i][1];
            int top = 0;
#pragma unroll
            for (int j = 0; j < 4; j++)
                top = max(top, max(mag_bits(a[j]), mag_bits(b[j])));
            const uint32_t bf = cache_scale((uint32_t)group_max_nonneg<16>(top));
            const float d = cache_scale_value(bf);
            const uint32_t c = bf ? codes(a, b, d) : 0;
            if (f < p.f1) {
                if (in && which == 0)
                    *(uint32_t *)(p.rec + cache_key_at(dk, f) + 4 * part) = c;
                else if (in)
                    code[f][part] = c;
                if (part == 0)
                    *(uint16_t *)(p.rec + (which ? cache_value_scale_at(dk, f) : cache_key_scale_at(dk, f))) =
                        (uint16_t)bf;
            }
        }
    }
    __syncthreads();
    /* a thread's square: dimensions 8 e to 8 e + 7 of the eight frames of (gg, w) */
    if (threadIdx.x < dk) {
        const uint32_t e = threadIdx.x / 8, gg = threadIdx.x % 2, w = threadIdx.x / 2 % 4;
        uint32_t a[8];
#pragma unroll
        for (uint32_t n = 0; n < 8; n++)
            a[n] = code[cache_frame_of(gg, w, n)][e];       /* frames that are not the call's: never kept below */
        turn(a);
#pragma unroll
        for (uint32_t n = 0; n < 8; n++)
            ((uint32_t *)image)[cache_value_dword(8 * e + n, gg, w) / 4] = a[n];
    }
    __syncthreads();
    /* a lane's 16 bytes: dimensions c and c + 16, frames of (0, w) and (1, w) */
    if (threadIdx.x < 2 * dk) {
        const uint32_t w = threadIdx.x / 16 % 4;
        uint32_t mask[2] = { 0, 0 };
#pragma unroll
        for (uint32_t n = 0; n < 16; n++) {
            const int32_t f = (int32_t)cache_frame_of(n / 8, w, n % 8);
            mask[n / 8] |= f >= p.f0 && f < p.f1 ? 15u << 4 * (n % 8) : 0;
        }
        if (mask[0] | mask[1]) {
            v4u *at = (v4u *)(p.rec + cache_values_at(dk)) + threadIdx.x;
            v4u now = image[threadIdx.x];
            if (~mask[0] | ~mask[1]) {
                const v4u old = *at;
#pragma unroll
                for (int i = 0; i < 4; i++)
                    now[i] = (now[i] & mask[i % 2]) | (old[i] & ~mask[i % 2]);
            }
            *at = now;
        }
    }
}

/* ----------------------------------------------------------------- read --- */

/* The write's way back: a workgroup reads one page's part of a stream's frames
 * [len, len + T) for one kept head. Frames of a hole read as zeros, and so do
 * frames past the table. 48 segments, 142 MB: 26 us, 5.4 TB/s (57 with a value
 * a thread). */
__global__ __launch_bounds__(256) void cache_read_kernel(uint8_t *data, uint32_t pages, uint32_t G, uint32_t dk,
                                                         CacheStreams st, float *__restrict__ k, uint64_t ks,
                                                         float *__restrict__ v, uint64_t vs) {
    __shared__ uint32_t code[kPage][kCodeRow];
    __shared__ v4u image[kPage * kMaxCacheDk / 2 / 16];
    PagePart p;
    if (!part_of(data, pages, G, dk, st, p))
        return;
    const uint32_t part = threadIdx.x % 16, g = blockIdx.x;
    const int32_t fa = p.f0 + (int32_t)(threadIdx.x / 16);
    uint32_t kc[4] = {}, ks_bf[4] = {}, vs_bf[4] = {};
    if (p.rec) {
        if (threadIdx.x < 2 * dk)
            image[threadIdx.x] = ((const v4u *)(p.rec + cache_values_at(dk)))[threadIdx.x];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int32_t f = fa + 16 * i;
            if (part < dk / 8 && f < p.f1) {
                kc[i] = *(const uint32_t *)(p.rec + cache_key_at(dk, f) + 4 * part);
                ks_bf[i] = *(const uint16_t *)(p.rec + cache_key_scale_at(dk, f));
                vs_bf[i] = *(const uint16_t *)(p.rec + cache_value_scale_at(dk, f));
            }
        }
        __syncthreads();
        if (threadIdx.x < dk) {
            const uint32_t e = threadIdx.x / 8, gg = threadIdx.x % 2, w = threadIdx.x / 2 % 4;
            uint32_t a[8];
#pragma unroll
            for (uint32_t n = 0; n < 8; n++)
                a[n] = ((const uint32_t *)image)[cache_value_dword(8 * e + n, gg, w) / 4];
            turn(a);
#pragma unroll
            for (uint32_t n = 0; n < 8; n++)
                code[cache_frame_of(gg, w, n)][e] = a[n];
        }
        __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const int32_t f = fa + 16 * i;
        if (part >= dk / 8 || f >= p.f1)
            continue;
        const uint64_t row = (uint64_t)(p.sp.r0 + p.base + f - p.sp.len);
        const uint32_t vc = p.rec ? code[f][part] : 0;
        const float kd = cache_scale_value(ks_bf[i]), vd = cache_scale_value(vs_bf[i]);
#pragma unroll
        for (int which = 0; which < 2; which++) {
            const uint32_t c = which ? vc : kc[i];
            const float d = which ? vd : kd;
            const v2f_c y0 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, 1.0f, 0);
            const v2f_c y1 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, 1.0f, 1);
            const v2f_c y2 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, 1.0f, 2);
            const v2f_c y3 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, 1.0f, 3);
            v4f *to = (v4f *)((which ? v + row * vs : k + row * ks) + g * dk + 8 * part);
            to[0] = v4f{ y0.x * d, y0.y * d, y1.x * d, y1.y * d };
            to[1] = v4f{ y2.x * d, y2.y * d, y3.x * d, y3.y * d };
        }
    }
}

/* ------------------------------------------------------------ attention --- */

/* Products in 32 bits on the bfloat16 matrix cores. A level has 2 significant
 * bits, so it is a bfloat16 as it stands; the other operand (a query, a
 * probability times its value's scale) is a float cut into three bfloat16 of
 * 8 bits each, whose sum is the float exactly (truncation leaves 16 bits
 * after the first piece and 8 after the second). Three products of exact
 * terms, added in 32 bits: what an fp32 product of the same values gives, at
 * a third of the bfloat16 rate, five times the fp32 matrix rate. */
struct Pieces {
    v8bf p[3];
};

__device__ __forceinline__ Pieces cut(const float (&x)[8]) {
    Pieces r;
    uint32_t w[3][4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        float a = x[2 * i], b = x[2 * i + 1];
#pragma unroll
        for (int n = 0; n < 3; n++) {
            const uint32_t ua = __float_as_uint(a), ub = __float_as_uint(b);
            w[n][i] = __builtin_amdgcn_perm(ub, ua, 0x07060302u);
            a -= __uint_as_float(ua & 0xffff0000u);
            b -= __uint_as_float(ub & 0xffff0000u);
        }
    }
#pragma unroll
    for (int n = 0; n < 3; n++)
        r.p[n] = __builtin_bit_cast(v8bf, v4u{ w[n][0], w[n][1], w[n][2], w[n][3] });
    return r;
}

/* eight codes as bfloat16 levels */
__device__ __forceinline__ v8bf levels(uint32_t w) {
    const v2bf a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, 1.0f, 0);
    const v2bf b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, 1.0f, 1);
    const v2bf c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, 1.0f, 2);
    const v2bf d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, 1.0f, 3);
    return v8bf{ a.x, a.y, b.x, b.y, c.x, c.y, d.x, d.y };
}

__device__ __forceinline__ v4f mfma(v8bf a, v8bf b, v4f c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

struct CacheAttention {
    float *o;
    const float *q;
    uint64_t os, qs;
    const uint8_t *data;                    /* the layer's records */
    uint32_t pages, G, H, dk;
    CacheStreams st;
    int32_t left, right;                    /* clipped to what can occur */
    float scale;                            /* 1 / sqrt(dk) */
    /* positions (p NULL: none), p's first row the distance left's */
    const float *p, *bias_u, *bias_w;
    float *place;                           /* the position scores, [rows][H][place_stride(bw)] */
    uint32_t bw;
    void *pieces;                           /* the table cut beforehand, [H][tiles of 16][steps][3][64 lanes] of 16 bytes */
    /* a stream's tiles of rows a kept head, workgroups that share a tile's pages, what they leave each other */
    uint32_t tiles, splits;
    float *parts;
};

__device__ __forceinline__ uint64_t unit_of(const CacheAttention &a, uint32_t b, uint32_t tile, uint32_t g) {
    return ((uint64_t)b * a.tiles + tile) * a.G + g;
}

/* Floats cut for a product of floats with floats: each piece the nearest
 * bfloat16 of what the ones before leave, so that the second is at most 2^-8
 * of the float's power of two, the third 2^-17, and the three sum to it exactly
 * (down to 2^-126, where pieces end). Of the nine products of two floats'
 * pieces the six largest are taken: those left out are 2^-24 of the product at
 * most, as much as a 32-bit product's own rounding. Whatever the other
 * dimensions hold: a row has no exponent in common. */
__device__ __forceinline__ Pieces cut_near(const float (&x)[8]) {
    Pieces r;
    uint32_t w[3][4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        v2f_c a = { x[2 * i], x[2 * i + 1] };
#pragma unroll
        for (int n = 0; n < 3; n++) {
            w[n][i] = __builtin_bit_cast(uint32_t, __builtin_convertvector(a, v2bf));
            a.x -= __uint_as_float(w[n][i] << 16);
            a.y -= __uint_as_float(w[n][i] & 0xffff0000u);
        }
    }
#pragma unroll
    for (int n = 0; n < 3; n++)
        r.p[n] = __builtin_bit_cast(v8bf, v4u{ w[n][0], w[n][1], w[n][2], w[n][3] });
    return r;
}

/* Sixteen rows of the positions' table for one head as the matrix
 * instruction's operand: lane l has dimensions 32 s + 8 (l / 16) of row l % 16
 * in step s. */
template <int NS>
struct PlaceTile {
    v4f p[NS][2];

    __device__ __forceinline__ void load(const CacheAttention &a, uint32_t h, uint32_t x) {
        const uint32_t lane = threadIdx.x & 63, dk = 32 * NS;
        const v4f *src = (const v4f *)(a.p + (uint64_t)min(x + lane % 16, a.bw - 1) * (a.H * dk) + h * dk + lane / 16 * 8);
#pragma unroll
        for (int s = 0; s < NS; s++)
            p[s][0] = src[8 * s], p[s][1] = src[8 * s + 1];
    }

    __device__ __forceinline__ void pieces(Pieces (&out)[NS]) const {
#pragma unroll
        for (int s = 0; s < NS; s++) {
            const float x[8] = { p[s][0][0], p[s][0][1], p[s][0][2], p[s][0][3], p[s][1][0], p[s][1][1], p[s][1][2], p[s][1][3] };
            out[s] = cut_near(x);
        }
    }
};

/* The table cut once for a call whose rows would do it many times over: a wave
 * a tile of a head, its operands 1 KB in a row each. */
template <int NS>
__global__ __launch_bounds__(256) void cache_cut_kernel(CacheAttention a) {
    const uint32_t tiles = (a.bw + 15) / 16, lane = threadIdx.x & 63;
    const uint32_t h = blockIdx.y, tile = blockIdx.x * 4 + (threadIdx.x >> 6);
    if (tile >= tiles)
        return;
    PlaceTile<NS> t;
    t.load(a, h, 16 * tile);
    Pieces ph[NS];
    t.pieces(ph);
    v8bf *to = (v8bf *)a.pieces + ((uint64_t)h * tiles + tile) * (NS * 3 * 64) + lane;
#pragma unroll
    for (int s = 0; s < NS; s++)
#pragma unroll
        for (int n = 0; n < 3; n++)
            to[64 * (3 * s + n)] = ph[s].p[n];
}

/* The maximum over the wave, in every lane (all of them active). */
__device__ __forceinline__ int wave_max(int v) {
    v = max(v, __builtin_amdgcn_update_dpp(v, v, 0xB1, 0xF, 0xF, false));
    v = max(v, __builtin_amdgcn_update_dpp(v, v, 0x4E, 0xF, 0xF, false));
    v = max(v, __builtin_amdgcn_update_dpp(v, v, 0x141, 0xF, 0xF, false));
    v = max(v, __builtin_amdgcn_update_dpp(v, v, 0x140, 0xF, 0xF, false));
    v = max(v, __builtin_amdgcn_update_dpp(v, v, 0x142, 0xA, 0xF, false));
    v = max(v, __builtin_amdgcn_update_dpp(v, v, 0x143, 0xC, 0xF, false));
    return __builtin_amdgcn_readlane(v, 63);
}

/* The position scores (q + w) . p, scaled as the softmax takes them (in powers
 * of 2), of every row at every distance that it needs, into the workspace:
 * the same rows of p serve every stream, so this is one product of all rows by
 * the table, read once, where the attention reads its own stream's pages only.
 * A workgroup of four waves takes 16 RT rows of a head, cut into the matrix
 * instruction's operands in LDS, and walks `steps` runs of 64 MT distances; a
 * wave takes MT tiles of 16 of each, so that an operand read from LDS serves
 * MT. PRE: the table's rows come cut.
 *
 * At 2624 rows by up to 3750 distances it takes 121 us, 110 at best (and the
 * cutting 11), for 280 MB of scores: its products alone take 91 at the 1134
 * TFLOP/s that a bfloat16 product of 8192 cubed reaches here, and the matrix
 * cores are busy half of its cycles. Of two float16 pieces with an exponent a
 * row three products do, in 97 us, but what is small beside its row's largest
 * loses its bits. At 256 rows by 4500 it takes 28 us, and at few rows a chain of
 * two memory round trips and a launch, 7. The shapes of a workgroup are within a
 * few us of each other: 8 waves, 128 rows and two tiles a wave 132 us, three
 * tiles 126, 96 rows and 6 waves 147. Measured and taken back: a lane's four
 * scores stored at the frames' own places (16 bytes at any multiple of 4: each
 * step twice as long), one float a lane stored there (as long as now, and the
 * attention no faster), stores through the caches (the attention of 256 streams
 * 171 -> 190 us). */

/* waves a SIMD: registers for three where a wave keeps two tiles of the table, as
 * LDS has room for (48 KB a workgroup of 64 rows of 128) */
constexpr int kPlaceWaves = 4;
constexpr int place_residency(int MT) { return MT == 1 ? 4 : 3; }

template <int NS, int RT, int MT, bool PRE>
__global__ __launch_bounds__(64 * kPlaceWaves, place_residency(MT)) void cache_place_kernel(CacheAttention a, int32_t steps) {
    constexpr int W = kPlaceWaves;
    constexpr int kRows = 16 * RT, kRun = 16 * MT * W, kThreads = 64 * W, kFill = kRows * 16 / kThreads;
    __shared__ v8bf frag[RT][NS][3][64];
    __shared__ int32_t need[W][2];
    const uint32_t h = blockIdx.y, n0 = blockIdx.z * kRows;
    const int32_t x0 = (int32_t)blockIdx.x * (kRun * steps), x1 = min(x0 + kRun * steps, (int32_t)a.bw);
    const uint32_t dk = 32 * NS, stride = place_stride(a.bw);
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6, w = lane / 16;
    const uint32_t rows = min((uint32_t)kRows, a.st.rows - n0);

    /* the rows' queries, 16 lanes a row: in flight while the streams are looked through */
    const uint32_t part = threadIdx.x % 16, row_a = threadIdx.x / 16;
    v4f qv[kFill][2] = {}, bias[2] = {};
    if (part < 4 * NS) {
#pragma unroll
        for (int i = 0; i < kFill; i++) {
            const v4f *src = (const v4f *)(a.q + (uint64_t)(n0 + min(row_a + 4 * W * i, rows - 1)) * a.qs + h * dk + 8 * part);
            qv[i][0] = src[0], qv[i][1] = src[1];
        }
        const v4f *b = (const v4f *)(a.bias_w + h * dk + 8 * part);
        bias[0] = b[0], bias[1] = b[1];
    }
    /* the distances that any of the rows needs */
    int32_t lo = INT32_MAX, hi = -INT32_MAX;
    for (uint32_t b = threadIdx.x; b < a.st.B; b += kThreads) {
        const CacheSpan sp = span_of(a.st, b);
        const int32_t r0 = max(sp.r0, (int32_t)n0), r1 = min(sp.r0 + sp.T, (int32_t)(n0 + kRows));
        if (r0 >= r1)
            continue;
        lo = min(lo, place_lo(sp, r1, a.left));
        hi = max(hi, place_hi(sp, r0, a.left));
    }
    lo = -wave_max(-lo), hi = wave_max(hi);
    if (lane == 0)
        need[wave][0] = lo, need[wave][1] = hi;
    const float c2 = a.scale * 1.44269504088896340736f;     /* scores in powers of 2 */
#pragma unroll
    for (int i = 0; i < kFill; i++) {
        const uint32_t row = row_a + 4 * W * i;
        float x[8];
#pragma unroll
        for (int j = 0; j < 8; j++)
            x[j] = (qv[i][j / 4][j % 4] + bias[j / 4][j % 4]) * c2;
        const Pieces c = cut_near(x);
        if (part < 4 * NS) {                /* a row's parts in different banks */
#pragma unroll
            for (int n = 0; n < 3; n++)
                frag[row / 16][part / 4][n][16 * (part % 4) + (row % 16 ^ part)] = c.p[n];
        }
    }
    __syncthreads();
    int32_t from = need[0][0], to = need[0][1];
#pragma unroll
    for (int i = 1; i < W; i++)
        from = min(from, need[i][0]), to = max(to, need[i][1]);
#pragma unroll 1
    for (int32_t x = x0 + 16 * MT * (int32_t)wave; x < x1 && x <= to; x += kRun) {
        if (from >= x + 16 * MT)
            continue;
        Pieces ph[MT][NS];
        if constexpr (PRE) {
            const uint32_t tiles = (a.bw + 15) / 16;
#pragma unroll
            for (int i = 0; i < MT; i++) {
                const uint32_t tile = min((uint32_t)x / 16 + i, tiles - 1);
                const v8bf *src = (const v8bf *)a.pieces + ((uint64_t)h * tiles + tile) * (NS * 3 * 64) + lane;
#pragma unroll
                for (int s = 0; s < NS; s++)
#pragma unroll
                    for (int n = 0; n < 3; n++)
                        ph[i][s].p[n] = src[64 * (3 * s + n)];
            }
        } else {
            PlaceTile<NS> t[MT];
#pragma unroll
            for (int i = 0; i < MT; i++)
                t[i].load(a, h, (uint32_t)x + 16 * i);
#pragma unroll
            for (int i = 0; i < MT; i++)
                t[i].pieces(ph[i]);
        }
#pragma unroll 1
        for (uint32_t rt = 0; 16 * rt < rows; rt++) {
            v4f acc[MT] = {};
#pragma unroll
            for (int s = 0; s < NS; s++) {
                const uint32_t at = 16 * w + (lane % 16 ^ (4 * s + w));
                const v8bf q0 = frag[rt][s][0][at], q1 = frag[rt][s][1][at], q2 = frag[rt][s][2][at];
#pragma unroll
                for (int i = 0; i < MT; i++)
                    acc[i] = mfma(ph[i][s].p[2], q0, acc[i]);
#pragma unroll
                for (int i = 0; i < MT; i++)
                    acc[i] = mfma(ph[i][s].p[1], q1, acc[i]);
#pragma unroll
                for (int i = 0; i < MT; i++)
                    acc[i] = mfma(ph[i][s].p[0], q2, acc[i]);
#pragma unroll
                for (int i = 0; i < MT; i++)
                    acc[i] = mfma(ph[i][s].p[1], q0, acc[i]);
#pragma unroll
                for (int i = 0; i < MT; i++)
                    acc[i] = mfma(ph[i][s].p[0], q1, acc[i]);
#pragma unroll
                for (int i = 0; i < MT; i++)
                    acc[i] = mfma(ph[i][s].p[0], q0, acc[i]);
            }
            const uint32_t row = 16 * rt + lane % 16;
            float *to_row = a.place + ((uint64_t)(n0 + row) * a.H + h) * stride + kPlacePad + x + 4 * w;
            if (row < rows) {
#pragma unroll
                for (int i = 0; i < MT; i++)
                    __builtin_nontemporal_store(acc[i], (v4f *)(to_row + 16 * i));
            }
        }
    }
}

/* Which rows of a stream and kept head a workgroup attends for, and which of
 * their pages: a stream's rows for a kept head are its frames, each with the
 * H / G heads that share the kept one; `splits` workgroups share a tile's
 * pages in runs. */
struct Share {
    CacheSpan sp;
    uint32_t g, b, grp, split;
    int32_t nrows, rr0;                     /* the stream's rows, the tile's first */
    int32_t pa, pb;                         /* the workgroup's pages, [pa, pb) of the stream */
    uint64_t unit;                          /* the tile among all of the call's */
};

template <int R>
__device__ __forceinline__ bool share_of(const CacheAttention &a, Share &s, uint32_t splits) {
    uint32_t i = blockIdx.x;
    s.g = i % a.G, i /= a.G;
    s.split = i % splits, i /= splits;
    const uint32_t tile = i % a.tiles;
    s.b = i / a.tiles;
    s.sp = span_of(a.st, s.b);
    s.grp = a.H / a.G;
    s.nrows = s.sp.T * (int32_t)s.grp;
    s.rr0 = (int32_t)tile * R;
    if (s.rr0 >= s.nrows)
        return false;
    const int32_t t0 = s.rr0 / (int32_t)s.grp, t1 = min(s.rr0 + R - 1, s.nrows - 1) / (int32_t)s.grp;
    const int32_t j0 = cache_lo(s.sp.len + t0, a.left), j1 = cache_hi(s.sp.len + t1, a.right, s.sp.total);
    const int32_t p0 = j0 / (int32_t)kPage, p1 = j1 < j0 ? p0 : j1 / (int32_t)kPage + 1;
    const int32_t each = (p1 - p0 + (int32_t)splits - 1) / (int32_t)splits;
    s.pa = min(p0 + (int32_t)s.split * each, p1);
    s.pb = min(s.pa + each, p1);
    s.unit = unit_of(a, s.b, tile, s.g);
    return true;
}

/* the wave's number in its workgroup, known to be the same in all its lanes */
__device__ __forceinline__ uint32_t wave_id() { return __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); }

/* The pages that a wave takes, every W-th of its workgroup of W waves: 64 table
 * entries at a time, one a lane, those that are no page of the pool passed
 * over. */
template <int W>
struct Walk {
    int32_t first, ids;
    uint64_t left;

    __device__ __forceinline__ Walk(const CacheAttention &a, const Share &s)
        : first(s.pa + (int32_t)wave_id() - W * 64), ids(0), left(0) {}

    /* the next page and its place in the pool; false, and pg and id as they were, after the last */
    __device__ __forceinline__ bool next(const CacheAttention &a, const Share &s, int32_t &pg, int32_t &id) {
        while (left == 0) {
            if (first + W * 64 >= s.pb)
                return false;
            first += W * 64;
            const int32_t mine = first + W * (int32_t)(threadIdx.x & 63);
            ids = mine < s.pb ? a.st.table[(uint64_t)s.b * a.st.max_pages + mine] : -1;
            left = __ballot(cache_page_ok(ids, a.pages));
        }
        const int at = __builtin_ctzll(left);
        left &= left - 1;
        pg = first + W * at;
        id = __builtin_amdgcn_readlane(ids, at);
        return true;
    }
};

__device__ __forceinline__ float bf_lo(uint32_t u) { return __uint_as_float(u << 16); }
__device__ __forceinline__ float bf_hi(uint32_t u) { return __uint_as_float(u & 0xffff0000u); }
__device__ __forceinline__ float bf_of(v2u u, int r) { return r % 2 ? bf_hi(u[r / 2]) : bf_lo(u[r / 2]); }

/* The maximum and the sum over each 16 lanes, in all of them. */
__device__ __forceinline__ float row_max(float v) {
    v = fmaxf(v, __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0xB1, 0xF, 0xF, false)));
    v = fmaxf(v, __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x4E, 0xF, 0xF, false)));
    v = fmaxf(v, __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x141, 0xF, 0xF, false)));
    return fmaxf(v, __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x140, 0xF, 0xF, false)));
}
__device__ __forceinline__ float row_sum(float v) {
    v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0xB1, 0xF, 0xF, false));
    v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x4E, 0xF, 0xF, false));
    v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x141, 0xF, 0xF, false));
    return v + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x140, 0xF, 0xF, false));
}

/* Parts of softmaxes over disjoint frames, n of them with their maxima and
 * sums, as one: sum(part e^(top - m)) / sum(sum e^(top - m)). Parts that
 * attended nothing have a maximum of -infinity and a sum of 0; a NaN among
 * the scores is in the sum and stays. */
template <int N, typename P>
__device__ __forceinline__ v4f joined(int n, P part, float &m, float &l) {
    m = -INFINITY;
    l = 0.0f;
    float top, sum;
    v4f y = { 0.0f, 0.0f, 0.0f, 0.0f }, o;
#pragma unroll N
    for (int i = 0; i < n; i++) {
        part(i, top, sum, nullptr);
        m = fmaxf(m, top);
    }
    const float base = m == -INFINITY ? 0.0f : m;
#pragma unroll N
    for (int i = 0; i < n; i++) {
        part(i, top, sum, &o);
        const float e = __builtin_amdgcn_exp2f(top - base);
        l += sum * e;
        y += o * e;
    }
    return y;
}

__device__ __forceinline__ v4f normal(v4f y, float l) {
    return l == 0.0f ? v4f{ 0.0f, 0.0f, 0.0f, 0.0f } : y / l;
}

/* The workgroup's waves met: into the outputs, or with several splits into
 * the workspace (R rows of dk sums, then R pairs of maximum and sum). */
template <int R, int NS, int W>
__device__ __forceinline__ void finish(const CacheAttention &a, const Share &s, float (*part)[R][32 * NS + 4],
                                       float (*tops)[R], float (*sums)[R]) {
    constexpr uint32_t dk = 32 * NS;
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < R * dk / 4; i += 64 * W) {
        const uint32_t r = i / (dk / 4), c = i % (dk / 4) * 4;
        const int32_t rr = s.rr0 + (int32_t)r;
        if (rr >= s.nrows)
            continue;
        float m, l;
        const v4f y = joined<W>(W, [&](int n, float &top, float &sum, v4f *o) {
            top = tops[n][r], sum = sums[n][r];
            if (o)
                *o = *(const v4f *)&part[n][r][c];
        }, m, l);
        if (a.splits == 1) {
            const uint64_t row = (uint64_t)(s.sp.r0 + rr / (int32_t)s.grp);
            *(v4f *)(a.o + row * a.os + (s.g * s.grp + (uint32_t)rr % s.grp) * dk + c) = normal(y, l);
        } else {
            float *w = a.parts + (s.unit * a.splits + s.split) * (R * (dk + 2));
            *(v4f *)(w + r * dk + c) = y;
            if (c == 0) {
                w[R * dk + 2 * r] = m;
                w[R * dk + 2 * r + 1] = l;
            }
        }
    }
}

/* The splits of each tile met, a workgroup a row: its threads in groups of
 * dk / 4, a group every so many splits, four dimensions a thread. */
template <int R, int NS>
__global__ __launch_bounds__(256) void cache_join_kernel(CacheAttention a) {
    constexpr uint32_t dk = 32 * NS, kCols = dk / 4, kGroups = 256 / kCols;
    __shared__ v4f part[kGroups][kCols];
    __shared__ float tops[kGroups], sums[kGroups];
    Share s;
    if (!share_of<R>(a, s, 1))
        return;
    const uint32_t r = blockIdx.y, group = threadIdx.x / kCols, c = threadIdx.x % kCols;
    const int32_t rr = s.rr0 + (int32_t)r;
    if (rr >= s.nrows)
        return;
    const float *w = a.parts + s.unit * a.splits * (R * (dk + 2));
    float m, l;
    if (group < kGroups) {
        const int n = group < a.splits ? (int)((a.splits - group + kGroups - 1) / kGroups) : 0;
        part[group][c] = joined<4>(n, [&](int i, float &top, float &sum, v4f *o) {
            const float *p = w + (uint64_t)(group + (uint32_t)i * kGroups) * (R * (dk + 2));
            top = p[R * dk + 2 * r], sum = p[R * dk + 2 * r + 1];
            if (o)
                *o = *(const v4f *)(p + r * dk + 4 * c);
        }, m, l);
        if (c == 0)
            tops[group] = m, sums[group] = l;
    }
    __syncthreads();
    if (group)
        return;
    const v4f y = joined<(int)kGroups>((int)kGroups, [&](int i, float &top, float &sum, v4f *o) {
        top = tops[i], sum = sums[i];
        if (o)
            *o = part[i][c];
    }, m, l);
    const uint64_t row = (uint64_t)(s.sp.r0 + rr / (int32_t)s.grp);
    *(v4f *)(a.o + row * a.os + (s.g * s.grp + (uint32_t)rr % s.grp) * dk + 4 * c) = normal(y, l);
}

/* The maximum that a softmax's exponentials are taken against follows the
 * scores only when one is over it by more than this many powers of two: until
 * then no lane asks another, and sums reach 2^8 times what they would, which
 * 32-bit floats hold as well. */
constexpr float kSlack = 8.0f;

/* Up to four rows of a stream and kept head (a step of a frame or a few), where
 * the cache's bytes are what takes time. A row's three pieces are three rows
 * of the matrix instruction's 16 (row 4 i + n piece n of query i), so one
 * product takes them all, and the keys are its columns: a lane's four sums
 * are one query's pieces of one key, added in place, and every lane has
 * scores of its own to make a softmax of (of the columns' other use, queries,
 * each would be made four times over). Tile kt's column c is key 4 c + kt, so
 * a lane's four scores are neighbours in memory: their scales and position
 * scores are one load each. The probabilities cross lanes once, cut, through
 * LDS, to be the second product's rows as the queries were the first's.
 *
 * Position scores come from the workspace, or with one row a stream and few
 * streams (kOwn) from the table itself: a quarter of the lanes' dimensions
 * each, four keys a lane, as 32-bit products.
 *
 * 256 streams of 3000 to 4500 frames, 8 heads of 128: 172 us for 1.02 GB, 5.9
 * TB/s of the 6.8 that reads reach (612 us with the kernel below, which makes
 * each score for 16 columns). What else counts: values loaded past the caches
 * (187 -> 172; the keys too 180), three waves a SIMD (four, at 128 registers,
 * spill: 233). Short calls take 10 to 12 us whatever their bytes: a launch,
 * the stream, its table, a page's loads and three pages a wave. */
enum { kNone, kMade, kOwn };
template <int NS, int POS, int W>
__global__ __launch_bounds__(64 * W) void cache_few_kernel(CacheAttention a) {
    constexpr uint32_t dk = 32 * NS, record = kPage * dk + 4 * kPage;
    constexpr uint32_t kRow = 72;           /* bfloat16 a row of pieces: 64 and a pad against bank conflicts */
    __shared__ float part[W][4][dk + 4], tops[W][4], sums[W][4];
    __shared__ __attribute__((aligned(16))) uint16_t prob[W][12][kRow];
    Share s;
    if (!share_of<4>(a, s, a.splits))
        return;
    const uint32_t lane = threadIdx.x & 63, wave = wave_id(), w = lane / 16, c = lane % 16;

    const float c2 = a.scale * 1.44269504088896340736f;     /* scores in powers of 2 */
    v8bf q[NS];
    {
        const int32_t i = (int32_t)(c / 4);
        const uint32_t n = c % 4;
        const uint32_t m1 = n >= 1 ? 0xffff0000u : 0, m2 = n >= 2 ? 0xffff0000u : 0;
        const bool live = i < s.nrows && n < 3;
        const int32_t ic = min(i, s.nrows - 1);
        const uint64_t row = (uint64_t)(s.sp.r0 + ic / (int32_t)s.grp);
        const uint32_t h = s.g * s.grp + (uint32_t)ic % s.grp;
#pragma unroll
        for (int st = 0; st < NS; st++) {
            const uint32_t d = h * dk + w * (8 * NS) + 8 * st;
            const v4f *src = (const v4f *)(a.q + row * a.qs + d);
            v4f s0 = src[0], s1 = src[1];
            if constexpr (POS != kNone) {
                const v4f *bias = (const v4f *)(a.bias_u + d);
                s0 += bias[0], s1 += bias[1];
            }
            uint32_t u[8];
#pragma unroll
            for (int j = 0; j < 8; j++) {
                float x = (j < 4 ? s0[j % 4] : s1[j % 4]) * c2;
                x -= __uint_as_float(__float_as_uint(x) & m1);
                x -= __uint_as_float(__float_as_uint(x) & m2);
                u[j] = live ? __float_as_uint(x) : 0;
            }
            v4u packed;
#pragma unroll
            for (int j = 0; j < 4; j++)
                packed[j] = __builtin_amdgcn_perm(u[2 * j + 1], u[2 * j], 0x07060302u);
            q[st] = __builtin_bit_cast(v8bf, packed);
        }
    }
    /* the lane's query in the softmax */
    const bool mine = (int32_t)w < s.nrows;
    const int32_t wi = min((int32_t)w, s.nrows - 1);
    const int32_t pos = s.sp.len + wi / (int32_t)s.grp;
    const int32_t lo = cache_lo(pos, a.left), hi = mine ? cache_hi(pos, a.right, s.sp.total) : -1;
    const float *place = nullptr;
    if constexpr (POS == kMade)
        place = a.place + ((uint64_t)(s.sp.r0 + wi / (int32_t)s.grp) * a.H + s.g * s.grp + (uint32_t)wi % s.grp) *
                              place_stride(a.bw) + kPlacePad + (a.left - pos) + 4 * c;

    float top = -INFINITY, sum = 0.0f;
    v4f o[2 * NS] = {};

    /* a page's keys, and its values: the next page's are loaded as soon as this one's have been used, into the
     * registers that they leave (after the last page, once more its own) */
    uint32_t kw[4][NS];
    v4u vw[NS];
    v2u ks, vs;
    v4f add = { 0.0f, 0.0f, 0.0f, 0.0f };
    v4f pw[4][2 * NS], own[2 * NS];
    if constexpr (POS == kOwn) {
#pragma unroll
        for (int i = 0; i < 2 * NS; i++) {
            const uint32_t d = s.g * dk + w * (8 * NS) + 4 * i;
            own[i] = (*(const v4f *)(a.q + (uint64_t)s.sp.r0 * a.qs + d) + *(const v4f *)(a.bias_w + d)) * c2;
        }
    }
    auto record_of = [&](int32_t id) { return a.data + ((uint64_t)(uint32_t)id * a.G + s.g) * record; };
    auto load_keys = [&](const uint8_t *rec, int32_t pg) {
#pragma unroll
        for (int kt = 0; kt < 4; kt++)
#pragma unroll
            for (int st = 0; st < NS; st++)
                kw[kt][st] = ((const uint32_t *)(rec + cache_key_at(dk, 4 * c + kt) + w * (4 * NS)))[st];
        ks = *(const v2u *)(rec + cache_key_scale_at(dk, 4 * c));
        if constexpr (POS == kMade)
            add = *(const v4f_u *)(place + pg * (int32_t)kPage);
        if constexpr (POS == kOwn) {
#pragma unroll
            for (int kt = 0; kt < 4; kt++) {
                const int32_t x = min(max(pg * (int32_t)kPage + 4 * (int32_t)c + kt - pos + a.left, 0), (int32_t)a.bw - 1);
                const v4f *src = (const v4f *)(a.p + (uint64_t)(uint32_t)x * (a.H * dk) + s.g * dk + w * (8 * NS));
#pragma unroll
                for (int i = 0; i < 2 * NS; i++)
                    pw[kt][i] = src[i];
            }
        }
    };
    auto load_values = [&](const uint8_t *rec) {
#pragma unroll
        for (int i = 0; i < NS; i++)
            vw[i] = __builtin_nontemporal_load((const v4u *)(rec + cache_values_at(dk) + 1024 * i + 16 * lane));
        vs = *(const v2u *)(rec + cache_value_scale_at(dk, 4 * c));
    };

    Walk<W> walk(a, s);
    int32_t pg = 0, id = 0;
    bool more = walk.next(a, s, pg, id);
    if (more) {
        load_keys(record_of(id), pg);
        load_values(record_of(id));
    }
    while (more) {
        float x[4], best = -INFINITY;
        const int32_t j = pg * (int32_t)kPage + 4 * (int32_t)c;
        v4f acc[4] = {};                    /* four chains side by side: a product waits for the one before it in its own */
#pragma unroll
        for (int st = 0; st < NS; st++)
#pragma unroll
            for (int kt = 0; kt < 4; kt++)
                acc[kt] = mfma(q[st], levels(kw[kt][st]), acc[kt]);
        if constexpr (POS == kOwn) {
#pragma unroll
            for (int kt = 0; kt < 4; kt++) {
                float d = 0.0f;
#pragma unroll
                for (int i = 0; i < 8 * NS; i++)
                    d = __builtin_fmaf(own[i / 4][i % 4], pw[kt][i / 4][i % 4], d);
                d += __shfl_xor(d, 16);
                add[kt] = d + __shfl_xor(d, 32);
            }
        }
#pragma unroll
        for (int kt = 0; kt < 4; kt++) {
            const float v = __builtin_fmaf((acc[kt][2] + acc[kt][1]) + acc[kt][0], bf_of(ks, kt), add[kt]);
            x[kt] = j + kt >= lo && j + kt <= hi ? v : -INFINITY;
            best = fmaxf(best, x[kt]);
        }
        more = walk.next(a, s, pg, id);
        const uint8_t *rec = record_of(id);
        load_keys(rec, pg);
        if (__any(best > top + kSlack)) {
            const float now = fmaxf(top, row_max(best));
            const float scale = __builtin_amdgcn_exp2f(top - (now == -INFINITY ? 0.0f : now));
            top = now;
            sum *= scale;
#pragma unroll
            for (int i = 0; i < 2 * NS; i++)
                o[i] *= scale;
        }
        const float base = top == -INFINITY ? 0.0f : top;
        uint32_t u[3][4];
#pragma unroll
        for (int kt = 0; kt < 4; kt++) {
            const float e = __builtin_amdgcn_exp2f(x[kt] - base);
            sum += e;
            /* a frame that is not attended may have a scale that was never written */
            float y = x[kt] == -INFINITY ? 0.0f : e * bf_of(vs, kt);
#pragma unroll
            for (int n = 0; n < 3; n++) {
                u[n][kt] = __float_as_uint(y);
                y -= __uint_as_float(u[n][kt] & 0xffff0000u);
            }
        }
        /* key 4 c + kt = 32 g + 16 h + 4 w' + kt with c = 8 g + 4 h + w': the eight frames that quarter w' of the
         * second product takes are in a row */
#pragma unroll
        for (int n = 0; n < 3; n++)
            *(v2u *)&prob[wave][3 * w + n][32 * (c / 8) + 8 * (c % 4) + 4 * (c / 4 % 2)] =
                v2u{ __builtin_amdgcn_perm(u[n][1], u[n][0], 0x07060302u),
                     __builtin_amdgcn_perm(u[n][3], u[n][2], 0x07060302u) };
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int gg = 0; gg < 2; gg++) {
            const v8bf pr = __builtin_bit_cast(v8bf, *(const v4u *)&prob[wave][3 * (c / 4) + min(c % 4, 2u)][32 * gg + 8 * w]);
#pragma unroll
            for (int dt = 0; dt < 2 * NS; dt++)
                o[dt] = mfma(pr, levels(vw[dt / 2][2 * (dt % 2) + gg]), o[dt]);
        }
        load_values(rec);
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
    }
    sum = row_sum(sum);
    if (c == 0) {
        tops[wave][w] = top;
        sums[wave][w] = sum;
    }
#pragma unroll
    for (int dt = 0; dt < 2 * NS; dt++)
        part[wave][w][16 * dt + c] = (o[dt][2] + o[dt][1]) + o[dt][0];
    finish<4, NS, W>(a, s, part, tops, sums);
}

/* More rows: 16 a workgroup, its four waves a page each in turn with the
 * running maximum and sum of a softmax, a query a column and its pieces three
 * products one after another. A lane's scores are a query's, and stay where
 * the second product takes them.
 *
 * Four files of 500 to 750 rows after 2200 to 3000 frames, 8 heads of 128:
 * 135 us (123 at best), 243 TFLOP/s as an fp32 product counts them. Instructions
 * bound it: of 525 vector ones a page and 16 rows 96 are products, which keep the
 * matrix cores busy 44% of the cycles, and the others issue in 49%, with two waves
 * a SIMD (235 registers) to overlap them. Measured and no faster, at best: a
 * page's first product under the page before's softmax (130), the products at
 * another wave priority (127, 129), the queries' pieces in LDS (126; for three
 * waves, 250: spills), eight waves (147; where 16 streams of 14 rows leave half
 * the CUs idle, eight take 12.8 and four 14.5). */
template <int NS, bool POS, int W>
__global__ __launch_bounds__(64 * W) void cache_many_kernel(CacheAttention a) {
    constexpr uint32_t dk = 32 * NS, record = kPage * dk + 4 * kPage;
    __shared__ float part[W][16][dk + 4], tops[W][16], sums[W][16];
    Share sh;
    if (!share_of<16>(a, sh, a.splits))
        return;
    const CacheSpan &sp = sh.sp;
    const uint32_t lane = threadIdx.x & 63, wave = wave_id(), w = lane / 16;
    const int32_t rr = min(sh.rr0 + (int32_t)(lane % 16), sh.nrows - 1);
    const int32_t t = rr / (int32_t)sh.grp;
    const uint32_t h = sh.g * sh.grp + (uint32_t)rr % sh.grp;
    const uint64_t row = (uint64_t)(sp.r0 + t);
    const int32_t pos = sp.len + t;
    const int32_t lo = cache_lo(pos, a.left), hi = cache_hi(pos, a.right, sp.total);

    const float c2 = a.scale * 1.44269504088896340736f;     /* scores in powers of 2 */
    Pieces q[NS];
#pragma unroll
    for (int s = 0; s < NS; s++) {
        const uint32_t c = h * dk + w * (8 * NS) + 8 * s;
        const v4f *src = (const v4f *)(a.q + row * a.qs + c);
        v4f s0 = src[0], s1 = src[1];
        if constexpr (POS) {
            const v4f *bias = (const v4f *)(a.bias_u + c);
            s0 += bias[0], s1 += bias[1];
        }
        s0 *= c2, s1 *= c2;
        const float x[8] = { s0[0], s0[1], s0[2], s0[3], s1[0], s1[1], s1[2], s1[3] };
        q[s] = cut(x);
    }
    const float *place = nullptr;
    if constexpr (POS)
        place = a.place + (row * a.H + h) * place_stride(a.bw) + kPlacePad + (a.left - pos) + 4 * w;

    /* frames that every row of the tile attends */
    const int32_t t1 = min(sh.rr0 + 15, sh.nrows - 1) / (int32_t)sh.grp;
    const int32_t all_lo = cache_lo(sp.len + t1, a.left);
    const int32_t all_hi = cache_hi(sp.len + sh.rr0 / (int32_t)sh.grp, a.right, sp.total);
    float top = -INFINITY, sum = 0.0f;
    v4f o[2 * NS] = {};

    /* loads ahead as in cache_few_kernel */
    uint32_t kw[4][NS];
    v4u vw[NS];
    v2u ks[4], vs[4];
    v4f add[4] = {};
    auto record_of = [&](int32_t id) { return a.data + ((uint64_t)(uint32_t)id * a.G + sh.g) * record; };
    auto load_keys = [&](const uint8_t *rec, int32_t pg) {
#pragma unroll
        for (int kt = 0; kt < 4; kt++) {
#pragma unroll
            for (int st = 0; st < NS; st++)
                kw[kt][st] = ((const uint32_t *)(rec + cache_key_at(dk, 16 * kt + lane % 16) + w * (4 * NS)))[st];
            ks[kt] = *(const v2u *)(rec + cache_key_scale_at(dk, 16 * kt + 4 * w));
            if constexpr (POS)
                add[kt] = *(const v4f_u *)(place + pg * (int32_t)kPage + 16 * kt);
        }
    };
    auto load_values = [&](const uint8_t *rec) {
#pragma unroll
        for (int i = 0; i < NS; i++)
            vw[i] = *(const v4u *)(rec + cache_values_at(dk) + 1024 * i + 16 * lane);
#pragma unroll
        for (int kt = 0; kt < 4; kt++)
            vs[kt] = *(const v2u *)(rec + cache_value_scale_at(dk, 16 * kt + 4 * w));
    };

    Walk<W> walk(a, sh);
    int32_t pg = 0, id = 0;
    bool more = walk.next(a, sh, pg, id);
    if (more) {
        load_keys(record_of(id), pg);
        load_values(record_of(id));
    }
    while (more) {
        float s[4][4], best = -INFINITY;
        const int32_t j = pg * (int32_t)kPage + 4 * (int32_t)w;
        const bool inside = pg * (int32_t)kPage >= all_lo && pg * (int32_t)kPage + (int32_t)kPage - 1 <= all_hi;
        v4f acc[4] = {};                    /* four chains side by side: a product waits for the one before it in its own */
#pragma unroll
        for (int st = 0; st < NS; st++) {
            v8bf k[4];
#pragma unroll
            for (int kt = 0; kt < 4; kt++)
                k[kt] = levels(kw[kt][st]);
#pragma unroll
            for (int n = 2; n >= 0; n--)
#pragma unroll
                for (int kt = 0; kt < 4; kt++)
                    acc[kt] = mfma(k[kt], q[st].p[n], acc[kt]);
        }
#pragma unroll
        for (int i = 0; i < 16; i++)
            s[i / 4][i % 4] = __builtin_fmaf(acc[i / 4][i % 4], bf_of(ks[i / 4], i % 4), add[i / 4][i % 4]);
        if (!inside) {
#pragma unroll
            for (int i = 0; i < 16; i++) {
                const int32_t f = j + 16 * (i / 4) + i % 4;
                s[i / 4][i % 4] = f >= lo && f <= hi ? s[i / 4][i % 4] : -INFINITY;
            }
        }
        more = walk.next(a, sh, pg, id);
        const uint8_t *rec = record_of(id);
        load_keys(rec, pg);
#pragma unroll
        for (int i = 0; i < 16; i++)
            best = fmaxf(best, s[i / 4][i % 4]);
        if (__any(best > top + kSlack)) {
            best = fmaxf(best, __shfl_xor(best, 16));
            best = fmaxf(best, __shfl_xor(best, 32));
            const float now = fmaxf(top, best);
            const float scale = __builtin_amdgcn_exp2f(top - (now == -INFINITY ? 0.0f : now));
            top = now;
            sum *= scale;
#pragma unroll
            for (int i = 0; i < 2 * NS; i++)
                o[i] *= scale;
        }
        const float base = top == -INFINITY ? 0.0f : top;
#pragma unroll
        for (int gg = 0; gg < 2; gg++) {
            float x[8];
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const int kt = 2 * gg + i / 4, r = i % 4;
                const float e = __builtin_amdgcn_exp2f(s[kt][r] - base);
                sum += e;
                x[i] = e * bf_of(vs[kt], r);
            }
            if (!inside) {
                /* a frame that is not attended may have a scale that was never written */
#pragma unroll
                for (int i = 0; i < 8; i++)
                    x[i] = s[2 * gg + i / 4][i % 4] == -INFINITY ? 0.0f : x[i];
            }
            const Pieces pr = cut(x);
            v8bf val[2 * NS];
#pragma unroll
            for (int dt = 0; dt < 2 * NS; dt++)
                val[dt] = levels(vw[dt / 2][2 * (dt % 2) + gg]);
#pragma unroll
            for (int n = 2; n >= 0; n--)
#pragma unroll
                for (int dt = 0; dt < 2 * NS; dt++)
                    o[dt] = mfma(val[dt], pr.p[n], o[dt]);
        }
        load_values(rec);
    }
    sum += __shfl_xor(sum, 16);
    sum += __shfl_xor(sum, 32);
    if (w == 0) {
        tops[wave][lane % 16] = top;
        sums[wave][lane % 16] = sum;
    }
#pragma unroll
    for (int dt = 0; dt < 2 * NS; dt++)
        *(v4f *)&part[wave][lane % 16][16 * dt + 4 * w] = o[dt];
    finish<16, NS, W>(a, sh, part, tops, sums);
}

/* ----------------------------------------------------------------- move --- */

/* Pairs (from, to) of pages by value, so that a call needs no device memory
 * of its own (a kernel's arguments are 4 KB at most); more take several
 * launches. */
constexpr int kMovePairs = 448;
struct MovePairs {
    int32_t from[kMovePairs], to[kMovePairs];
};

/* A page of a layer is one contiguous run of G records: kMoveParts workgroups a
 * page and layer, eight 16-byte loads a lane in flight. The row of workgroups
 * behind the last pair lets the tables follow, each entry against all pairs in
 * LDS (a page is moved at most once, so at most one is its). 300 pages of 24
 * layers, 973 MB read and written: 175 us, 5.6 TB/s, where torch's copy of 4
 * GiB reaches 4.8 (four workgroups a page, one load in flight: 200, and 23 for
 * the tables in a launch of their own). */
constexpr int kMoveParts = 2;
__global__ __launch_bounds__(256) void cache_move_kernel(uint8_t *__restrict__ dst, uint64_t dlayer,
                                                         const uint8_t *__restrict__ src, uint64_t slayer,
                                                         uint32_t page_bytes, MovePairs m, uint32_t pairs,
                                                         int32_t *__restrict__ table, uint64_t entries) {
    if (blockIdx.y == pairs) {
        __shared__ __attribute__((aligned(16))) int32_t from[kMovePairs], to[kMovePairs];
        for (uint32_t i = threadIdx.x; i < kMovePairs; i += 256) {
            from[i] = i < pairs ? m.from[i] : -1;
            to[i] = m.to[i];
        }
        __syncthreads();
        const uint64_t step = (uint64_t)gridDim.x * gridDim.z * 256;
        for (uint64_t i = ((uint64_t)blockIdx.z * gridDim.x + blockIdx.x) * 256 + threadIdx.x; i < entries; i += step) {
            const int32_t old = table[i];
            int32_t at = -1;
            if (old >= 0) {
                for (uint32_t q = 0; q < pairs; q += 4) {
                    const int4 f = *(const int4 *)&from[q];
                    at = f.x == old ? (int32_t)q : f.y == old ? (int32_t)q + 1 : f.z == old ? (int32_t)q + 2
                       : f.w == old ? (int32_t)q + 3 : at;
                }
            }
            if (at >= 0)
                table[i] = to[at];
        }
        return;
    }
    const v4u *from = (const v4u *)(src + blockIdx.z * slayer + (uint64_t)m.from[blockIdx.y] * page_bytes);
    v4u *to = (v4u *)(dst + blockIdx.z * dlayer + (uint64_t)m.to[blockIdx.y] * page_bytes);
    const uint32_t n = page_bytes / 16, step = kMoveParts * 256;
    uint32_t i = blockIdx.x * 256 + threadIdx.x;
    for (; i + 7 * step < n; i += 8 * step) {
        v4u x[8];
#pragma unroll
        for (int j = 0; j < 8; j++)
            x[j] = __builtin_nontemporal_load(from + i + j * step);
#pragma unroll
        for (int j = 0; j < 8; j++)
            __builtin_nontemporal_store(x[j], to + i + j * step);
    }
    for (; i < n; i += step)
        to[i] = from[i];
}

/* ------------------------------------------------------------- launches --- */

/* A write or read has a workgroup for every page that a stream's frames can
 * touch, a kept head; those that find nothing of theirs end at once, 0.42 ns
 * apart (16.8 million take 7.0 ms). 2^28 of them, a tenth of a second, are the
 * most that are launched: counts that no call's rows could fill (65535 streams
 * with a max_T of 2^21 would end them for minutes). */
static uint32_t span_pages(const CacheStreams &st) { return (st.max_T + kPage - 2) / kPage + 1; }

bool cache_span_fits(const CacheStreams &st, uint32_t G) {
    return (uint64_t)span_pages(st) * st.B * G <= 1u << 28;
}

int launch_cache_write(uint8_t *data, uint32_t pages, uint32_t G, uint32_t dk, const CacheStreams &st, const float *k,
                       uint64_t ks, const float *v, uint64_t vs, hipStream_t s) {
    const dim3 grid(G, span_pages(st), st.B);
    cache_write_kernel<<<grid, 256, 0, s>>>(data, pages, G, dk, st, k, ks, v, vs);
    return hipPeekAtLastError() == hipSuccess ? 0 : -1;
}

int launch_cache_read(const uint8_t *data, uint32_t pages, uint32_t G, uint32_t dk, const CacheStreams &st, float *k,
                      uint64_t ks, float *v, uint64_t vs, hipStream_t s) {
    const dim3 grid(G, span_pages(st), st.B);
    cache_read_kernel<<<grid, 256, 0, s>>>((uint8_t *)data, pages, G, dk, st, k, ks, v, vs);
    return hipPeekAtLastError() == hipSuccess ? 0 : -1;
}

/* workgroups of 256 in a launch's first dimension, under 2^32 threads */
constexpr uint64_t kMostGroups = (1u << 24) - 1;

/* How a call's rows are dealt. Tiles of four rows where a stream has at most
 * four a kept head, else of 16. With up to 256 tiles, a workgroup a CU, the
 * waves that a CU holds are found in two ways: workgroups of eight waves, which
 * meet in LDS, where a wave then takes a page or more (four rows' pages are
 * short work, so 10 pages of 128 dimensions or 20 of 64), and splits of a
 * tile's pages, joined for 4 to 5 us by a launch of their own, from 32 pages
 * on, so many that a wave takes two pages or more. As many splits of four waves
 * as two a CU allow only where that is an odd number, so that those of eight
 * waves leave CUs idle, and against none from 120 pages on (100 of 16 rows).
 *
 * Heads of 128, four rows: 256 tiles of 33 pages 16.2 us with eight waves, 16.7
 * with four, 19.4 in two splits of four; 192 of 16 8.6 and 9.0 (heads of 64 7.7
 * and 7.3); 32 of 70 unsplit with four 23.7, in eight splits 10.7, in nine 11.5.
 * 16 rows: 256 of 33 19.4 with eight, in two splits of four 26.4; 192 of 24 15.1
 * with eight and 15.8 with four, of 8 9.2 and 9.1; 320 of 24 27.4 and 22.8 (more
 * tiles than CUs). 152 tiles of four rows unsplit with eight waves and in three
 * splits of four: 100 pages 26.1 and 27.5, 120 30.3 and 30.6, 300 66 and 62 (136
 * tiles of 120 30.5 and 28.7, 168 30.7 and 32.7; heads of 64 22.4 and 21.5). 136
 * tiles of 16 rows: 80 pages 31.3 and 29.6, 120 42 and 36.5 (heads of 64 21.8 and
 * 22.8, 29.2 and 27.2; of 32 17.8 and 20.1, 24.4 and 24.6). 96 tiles in two of
 * eight and in five of four: 33 pages 12.1 and 12.0, 300 42.2 and 42.5 (16 rows 56
 * and 50; heads of 32 29.8 and 25.4). One frame against 704 pages of one stream:
 * 16.4 in 32 splits of eight waves, unsplit 141, with four waves 200. */
struct Deal {
    uint32_t rows, tiles, splits;           /* rows a tile, a stream's tiles a kept head, a tile's splits */
    uint32_t pages;                         /* pages a tile can reach */
    uint32_t waves;                         /* waves a workgroup of the attention */
    uint64_t units;
    bool own;                               /* a row's position scores made where they are used */
};

/* A row's position scores are made where they are used for single rows of few
 * streams with a narrow window: a launch fewer. A call of one row by 71
 * distances takes 7.7 us so and 10.0 with a launch of their own, by 181 11.5 and
 * 11.7; 16 rows by 71 8.0 and 9.8, by 181 12.1 and 11.6; 64 rows by 71 14.3 and
 * 12.4 (each stream reads the table itself, in pieces of 16 bytes). */
static Deal deal(const CacheStreams &st, uint32_t G, uint32_t H, uint32_t dk, int32_t left, int32_t right) {
    Deal d;
    const uint32_t rows = st.max_T * (H / G);
    d.rows = rows <= 4 ? 4 : 16;
    d.tiles = (rows + d.rows - 1) / d.rows;
    d.units = (uint64_t)st.B * G * d.tiles;
    d.pages = cache_tile_pages(st.max_pages, left, right);
    d.own = rows == 1 && st.B <= 16 && left + right < 100;
    d.splits = 1, d.waves = 4;
    if (d.units == 0 || d.units > 256)
        return d;
    const uint32_t eights = (uint32_t)(256 / d.units), fours = (uint32_t)(512 / d.units);
    const bool odd = fours % 2 && d.pages >= (eights > 1 ? 32 : d.rows == 4 ? 120 : 100);
    if (d.pages >= 32)
        d.splits = std::min({ odd ? fours : eights, (d.pages + 7) / 8, 128u });
    if (!odd && (d.rows == 4 ? (uint64_t)d.pages * dk > 1280u * d.splits : d.pages > 8 * d.splits))
        d.waves = 8;
    return d;
}

/* From this many scores a head on, the position scores are made of a table cut
 * beforehand: a launch more, and 64 rows' share of the cutting less for each 64
 * rows. Whole calls of 8 heads of 128 with it and without: 2624 rows by 3750
 * distances 260 and 267 us, 1000 by 3450 105 and 117, 1920 by 2280 134 and 152;
 * 1000 by 2300 56 and 52, 600 by 2600 67 and 64, 600 by 1500 38 and 36. */
static bool place_cut(uint32_t rows, uint32_t bw) { return (uint64_t)rows * bw >= 2600000; }

static size_t pieces_bytes(uint32_t H, uint32_t bw, uint32_t dk) {
    return (size_t)H * ((bw + 15) / 16) * 16 * (6 * dk);
}

/* The workspace's parts, in bytes, one after another (each a multiple of 16). */
struct Space {
    size_t place, pieces, parts;
};

static Space space(const CacheStreams &st, uint32_t H, uint32_t dk, bool positions, uint32_t bw, const Deal &d) {
    Space s = { 0, 0, 0 };
    if (positions && !d.own) {
        s.place = (size_t)st.rows * H * place_stride(bw) * sizeof(float);
        s.pieces = place_cut(st.rows, bw) ? pieces_bytes(H, bw, dk) : 0;
    }
    if (d.splits > 1)
        s.parts = (size_t)d.units * d.splits * d.rows * (dk + 2) * sizeof(float);
    return s;
}

size_t cache_attention_workspace(const CacheStreams &st, uint32_t G, uint32_t H, uint32_t dk, bool positions,
                                 int32_t left, int32_t right) {
    const Space s = space(st, H, dk, positions, (uint32_t)left + (uint32_t)right + 1, deal(st, G, H, dk, left, right));
    return s.place + s.pieces + s.parts;
}

bool cache_attention_fits(const CacheStreams &st, uint32_t G, uint32_t H, uint32_t dk, int32_t left, int32_t right) {
    const Deal d = deal(st, G, H, dk, left, right);
    return d.units <= kMostGroups / d.splits;
}

bool cache_places_fit(const CacheStreams &st, uint32_t H, int32_t left, int32_t right) {
    const uint32_t bw = (uint32_t)left + (uint32_t)right + 1;
    const uint64_t row = (uint64_t)H * place_stride(bw) * sizeof(float);        /* under 2^50 */
    return (bw - 1) / 64 < kMostGroups && (st.rows == 0 || row <= (1ull << 48) / st.rows);
}

template <int NS, int RT, int MT, bool PRE>
static void place(const CacheAttention &a, hipStream_t s) {
    /* Runs one after another in a workgroup, whose rows' operands are then made once for all of them, as many as take the
     * fewest steps in a row over the rounds of workgroups that the chip holds, those operands counted as a step (2624
     * rows by 3750: 154 us with one run, 134 with two, 125 with five, which it takes; 160 rows by 900: 8.7 with one,
     * which it takes, 11.9 with two, 21.0 with five). */
    constexpr uint32_t kRun = 16 * MT * kPlaceWaves, kHeld = 256 * 4 * place_residency(MT) / kPlaceWaves;
    const uint32_t runs = (a.bw + kRun - 1) / kRun, blocks = (a.st.rows + 16 * RT - 1) / (16 * RT);
    auto rounds = [&](uint32_t n) { return ((uint64_t)((runs + n - 1) / n) * a.H * blocks + kHeld - 1) / kHeld * (n + 1); };
    uint32_t steps = 1;
    for (uint32_t n = 2; n <= 8; n++)
        steps = rounds(n) < rounds(steps) ? n : steps;
    cache_place_kernel<NS, RT, MT, PRE><<<dim3((runs + steps - 1) / steps, a.H, blocks), 64 * kPlaceWaves, 0, s>>>(a, (int32_t)steps);
}

template <int NS>
static void attend(const CacheAttention &a, const Deal &d, hipStream_t s) {
    if (a.p && !d.own) {
        if (place_cut(a.st.rows, a.bw)) {
            cache_cut_kernel<NS><<<dim3(((a.bw + 15) / 16 + 3) / 4, a.H), 256, 0, s>>>(a);
            place<NS, 4, 2, true>(a, s);
        } else if (a.st.rows <= 16 || (uint64_t)((a.st.rows + 15) / 16) * ((a.bw + 15) / 16) * a.H <= 4096) {
            /* up to four tiles of 16 by 16 a SIMD: one workgroup's pass from the table's rows to the last store is what
             * takes time, and 16 rows have the shortest (128 rows by 751 distances 7.4 us, with 64 rows 8.4; 256 by
             * 4500 47 and 29) */
            place<NS, 1, 1, false>(a, s);
        } else {
            place<NS, 4, 2, false>(a, s);
        }
    }
    const uint32_t grid = (uint32_t)(d.units * d.splits);
    const uint32_t threads = 64 * d.waves;
    if (d.rows == 4 && a.p && d.own)
        cache_few_kernel<NS, kOwn, 4><<<grid, threads, 0, s>>>(a);
    else if (d.rows == 4 && a.p)
        (d.waves == 8 ? cache_few_kernel<NS, kMade, 8> : cache_few_kernel<NS, kMade, 4>)<<<grid, threads, 0, s>>>(a);
    else if (d.rows == 4)
        (d.waves == 8 ? cache_few_kernel<NS, kNone, 8> : cache_few_kernel<NS, kNone, 4>)<<<grid, threads, 0, s>>>(a);
    else if (a.p)
        (d.waves == 8 ? cache_many_kernel<NS, true, 8> : cache_many_kernel<NS, true, 4>)<<<grid, threads, 0, s>>>(a);
    else
        (d.waves == 8 ? cache_many_kernel<NS, false, 8> : cache_many_kernel<NS, false, 4>)<<<grid, threads, 0, s>>>(a);
    if (d.splits > 1) {
        if (d.rows == 4)
            cache_join_kernel<4, NS><<<dim3(grid / d.splits, std::min(d.rows, a.st.max_T * (a.H / a.G))), 256, 0, s>>>(a);
        else
            cache_join_kernel<16, NS><<<dim3(grid / d.splits, std::min(d.rows, a.st.max_T * (a.H / a.G))), 256, 0, s>>>(a);
    }
}

int launch_cache_attention(const CacheAttentionCall &c, hipStream_t s) {
    CacheAttention a = {};
    a.o = c.o, a.os = c.os, a.q = c.q, a.qs = c.qs;
    a.data = c.data, a.pages = c.pages, a.G = c.G, a.H = c.H, a.dk = c.dk;
    a.st = c.st;
    a.left = c.left, a.right = c.right;
    a.scale = 1.0f / sqrtf((float)c.dk);
    a.p = c.p, a.bias_u = c.bias_u, a.bias_w = c.bias_w;
    a.bw = (uint32_t)c.left + (uint32_t)c.right + 1;
    const Deal d = deal(c.st, c.G, c.H, c.dk, c.left, c.right);
    a.tiles = d.tiles, a.splits = d.splits;
    const Space sp = space(c.st, c.H, c.dk, c.p != nullptr, a.bw, d);
    a.place = (float *)c.ws;
    a.pieces = (char *)c.ws + sp.place;
    a.parts = (float *)((char *)c.ws + sp.place + sp.pieces);
    switch (c.dk / 32) {
    case 1: attend<1>(a, d, s); break;
    case 2: attend<2>(a, d, s); break;
    case 3: attend<3>(a, d, s); break;
    case 4: attend<4>(a, d, s); break;
    default: return -2;
    }
    return hipPeekAtLastError() == hipSuccess ? 0 : -1;
}

int launch_cache_move(uint8_t *dst, uint64_t dlayer, const uint8_t *src, uint64_t slayer, uint32_t layers,
                      uint32_t page_bytes, const int32_t *pairs, uint32_t n, int32_t *table, uint64_t entries,
                      hipStream_t s) {
    for (uint32_t p0 = 0; p0 < n; p0 += kMovePairs) {
        const uint32_t m = n - p0 < (uint32_t)kMovePairs ? n - p0 : (uint32_t)kMovePairs;
        MovePairs mp = {};
        for (uint32_t i = 0; i < m; i++) {
            mp.from[i] = pairs[2 * (p0 + i)];
            mp.to[i] = pairs[2 * (p0 + i) + 1];
        }
        const uint32_t follow = table && entries ? 1 : 0;
        cache_move_kernel<<<dim3(kMoveParts, m + follow, layers), 256, 0, s>>>(dst, dlayer, src, slayer, page_bytes, mp,
                                                                              m, table, entries);
    }
    return hipPeekAtLastError() == hipSuccess ? 0 : -1;
}

}  // namespace pkq8
