/* The 4-bit cache of keys and values: where each frame's codes and scales
 * lie, how a value becomes a code, and what a stream's descriptor says after
 * its bounds are checked. Plain arithmetic with no device calls, so the host
 * tests compile it too; the kernels (cache_kernels.hip) take every address
 * and every bound from here.
 *
 * A page holds 64 frames of one stream. Its record for one layer and one
 * kept head of dk dimensions (32, 64, 96 or 128):
 *
 *   keys    64 rows of dk / 2 bytes, dimension 2 b in byte b's low nibble,
 *           2 b + 1 in its high one
 *   values  dimension c of frame 32 g + 16 h + 4 w + r (g, h < 2; w, r < 4)
 *           in nibble 4 h + r of the dword at
 *           1024 (c / 32) + 16 (16 w + c % 16) + 8 (c / 16 % 2) + 4 g
 *   scales  64 bfloat16 of the keys, then 64 of the values
 *
 * Both orders are the matrix instruction's. v_mfma_f32_16x16x32_bf16 takes
 * from lane l eight consecutive reduction indices 8 (l / 16) of row l % 16.
 * For the scores the reduction runs over dimensions, in any order the
 * queries follow too: lane l takes dk / 4 dimensions of key l % 16, which a
 * row-major key holds in dk / 8 consecutive bytes. For the output it runs
 * over frames, and the scores leave the first product as four consecutive
 * frames 4 (l / 16) of a 16-frame tile a lane: two tiles give a lane its
 * eight frames {16 h + 4 w + r}, so the values of dimension c and those
 * frames are one dword, a lane's four dwords (two dimensions 16 apart, two
 * 32-frame groups) are 16 bytes, and a wave's are 1 KB in a row. No value
 * crosses lanes between the two products.
 *
 * A code is a sign (8) and one of the levels 0, 1/2, 1, 3/2, 2, 3, 4, 6 (the
 * 4-bit float e2m1, which the hardware turns into bfloat16 pairs in one
 * instruction), times the scale of its frame and head. One scale for a
 * frame's whole head, not one for each 32 values: it then multiplies a
 * score (keys) or a probability (values) once in 32 bits, and the products
 * run on the bare levels. It is a bfloat16: its 8 bits cost at most 1/256 of
 * a step, and being the least one that holds the largest magnitude under the
 * last level, it clips nothing. */
#ifndef PK_CACHE_LAYOUT_H
#define PK_CACHE_LAYOUT_H

#include <stddef.h>
#include <stdint.h>
#include <string.h>

#ifdef __HIPCC__
#include <hip/hip_runtime.h>
#define PK_HD __host__ __device__ __forceinline__
#else
#define PK_HD static inline
#endif

namespace pkq8 {

constexpr uint32_t kPage = 64;              /* frames a page */
constexpr uint32_t kMaxCacheDk = 128;

PK_HD bool cache_dk_ok(uint32_t dk) { return dk >= 32 && dk <= kMaxCacheDk && dk % 32 == 0; }

/* bytes of one (layer, page, head) record, and the offsets in it */
PK_HD uint32_t cache_record(uint32_t dk) { return kPage * dk + 4 * kPage; }
PK_HD uint32_t cache_key_at(uint32_t dk, uint32_t f) { return f * (dk / 2); }
PK_HD uint32_t cache_values_at(uint32_t dk) { return kPage * dk / 2; }
PK_HD uint32_t cache_value_dword(uint32_t c, uint32_t g, uint32_t w) {
    return 1024 * (c / 32) + 16 * (16 * w + c % 16) + 8 * (c / 16 % 2) + 4 * g;
}
PK_HD uint32_t cache_key_scale_at(uint32_t dk, uint32_t f) { return kPage * dk + 2 * f; }
PK_HD uint32_t cache_value_scale_at(uint32_t dk, uint32_t f) { return kPage * dk + 2 * kPage + 2 * f; }

/* the frame of nibble i of a value dword, in its page */
PK_HD uint32_t cache_frame_of(uint32_t g, uint32_t w, uint32_t i) { return 32 * g + 16 * (i / 4) + 4 * w + i % 4; }

PK_HD uint32_t bits_of(float x) {
    uint32_t u;
    memcpy(&u, &x, 4);
    return u;
}
PK_HD float float_of(uint32_t u) {
    float x;
    memcpy(&x, &u, 4);
    return x;
}

/* The scale's bfloat16 for a head whose largest magnitude has the bits mb (a
 * NaN's above an infinity's above every number's): the least d with 6 d >=
 * it; 0 (all codes zero) for a NaN, an infinity or anything of 2^127 and more
 * (6 d could pass the largest float), and under 2^-121. 6 d is exact in 32
 * bits, so d is the same however it is computed: the quotient's truncation
 * is at most a step off either way. */
PK_HD uint32_t cache_scale(uint32_t mb) {
    if (mb >= 0x7f000000u || mb < 0x03000000u)
        return 0;
    const float top = float_of(mb);
    uint32_t d = bits_of(top / 6.0f) & 0xffff0000u;
    if (6.0f * float_of(d) >= top)
        d -= 0x10000u;
    if (6.0f * float_of(d) < top)
        d += 0x10000u;
    return d >> 16;
}

PK_HD float cache_scale_value(uint32_t bf) { return float_of(bf << 16); }

/* x's code at scale d > 0: the nearest level, of two as near the one with the
 * even code. Levels' midpoints have 3 significant bits and d 8, so every
 * product is exact and so is every comparison. */
PK_HD uint32_t cache_code(float x, float d) {
    const uint32_t u = bits_of(x);
    const float a = float_of(u & 0x7fffffffu);
    const uint32_t c = (uint32_t)(a > 0.25f * d) + (uint32_t)(a >= 0.75f * d) + (uint32_t)(a > 1.25f * d) +
                       (uint32_t)(a >= 1.75f * d) + (uint32_t)(a > 2.5f * d) + (uint32_t)(a >= 3.5f * d) +
                       (uint32_t)(a > 5.0f * d);
    return c ? c | (u >> 28 & 8) : 0;
}

/* a code's level: 0, 0.5, 1, 1.5, 2, 3, 4, 6 with the sign bit 8 */
PK_HD float cache_level(uint32_t code) {
    const uint32_t m = code & 7;
    const float v = m < 4 ? 0.5f * (float)m : (float)(m < 6 ? m - 2 : 2 * m - 8);
    return code & 8 ? -v : v;
}

/* The streams of a call as the kernels see them (device pointers), and one
 * stream's part of it with every bound applied: rows [r0, r0 + T) of the
 * call, of frames [len, len + T) of the stream, total the frames that its
 * table can hold of them. Whatever the arrays hold, 0 <= r0, r0 + T <= rows,
 * T <= max_T and len, total <= 64 max_pages. */
struct CacheStreams {
    const int32_t *table;                   /* [B][max_pages] */
    const int32_t *len;                     /* [B] */
    const int32_t *row0;                    /* [B + 1] */
    uint32_t B, max_pages, rows, max_T;
};

struct CacheSpan {
    int32_t r0, T, len, total;
};

PK_HD int32_t cache_clip(int32_t v, int32_t lo, int32_t hi) { return v < lo ? lo : v > hi ? hi : v; }

PK_HD CacheSpan cache_span(const CacheStreams &s, int32_t row0, int32_t row1, int32_t len) {
    const int32_t rows = (int32_t)s.rows, cap = (int32_t)(s.max_pages * kPage);
    CacheSpan p;
    p.r0 = cache_clip(row0, 0, rows);
    p.T = cache_clip(cache_clip(row1, 0, rows) - p.r0, 0, (int32_t)s.max_T);
    p.len = cache_clip(len, 0, cap);
    p.total = cache_clip(p.len + p.T, 0, cap);
    return p;
}

/* whether a table's entry is a page of the pool; others are holes, whose
 * frames are neither written nor attended */
PK_HD bool cache_page_ok(int32_t id, uint32_t pages) { return (uint32_t)id < pages; }

/* The furthest back that a row of a call can attend. A stream's frames may
 * outgrow its table: then the last rows lie past every frame that the table
 * holds, and the first of those is this far behind. */
PK_HD int32_t cache_most_left(uint32_t max_pages, uint32_t max_T) {
    return (int32_t)(max_pages * kPage - 1 + max_T);
}

/* The frames a row at position pos attends: [lo, hi], empty if lo > hi. */
PK_HD int32_t cache_lo(int32_t pos, int32_t left) { return pos > left ? pos - left : 0; }
PK_HD int32_t cache_hi(int32_t pos, int32_t right, int32_t total) {
    const int64_t h = (int64_t)pos + right;
    return h < (int64_t)total - 1 ? (int32_t)h : total - 1;
}

/* The pages that a tile of rows reaches, at most: its rows' positions are up
 * to 15 apart, so its frames are at most left + right + 16 in a row, which
 * touch one page more than they fill. */
PK_HD uint32_t cache_tile_pages(uint32_t max_pages, int32_t left, int32_t right) {
    const uint64_t n = ((uint64_t)left + (uint64_t)right + 16 + kPage - 2) / kPage + 1;
    return n < max_pages ? (uint32_t)n : max_pages;
}

/* The position scores' workspace: a row's bw + 2 kPlacePad floats a head,
 * score of distance x at kPlacePad + x, x = frame - (pos - left). A tile of
 * 16 rows reads whole pages for all of them: a page's first frame is up to 63
 * before the first row's lo and the rows' positions up to 15 apart, so x runs
 * from -78 to bw + 77, inside the row's pads. They are written 32 at a time,
 * up to 31 past bw. */
constexpr uint32_t kPlacePad = 80;
PK_HD uint32_t place_stride(uint32_t bw) { return (bw + 2 * kPlacePad + 15) / 16 * 16; }

/* the distances x that the call's rows [r0, r1) of a stream need, all of its
 * frames: the last row's of frame 0, the first one's of the last frame (which
 * is under max_T ahead of it, so that left is added to a small number) */
PK_HD int32_t place_lo(const CacheSpan &sp, int32_t r1, int32_t left) { return left - (sp.len + r1 - 1 - sp.r0); }
PK_HD int32_t place_hi(const CacheSpan &sp, int32_t r0, int32_t left) {
    return left + (sp.total - 1 - (sp.len + r0 - sp.r0));
}

}  // namespace pkq8

#endif
