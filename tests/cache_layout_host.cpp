/* csrc/cache_layout.h as the host tests call it. */
#include "cache_layout.h"

using namespace pkq8;

extern "C" {

uint32_t t_scale(float top) { return cache_scale(bits_of(top) & 0x7fffffffu); }
uint32_t t_code(float x, float d) { return cache_code(x, d); }
float t_level(uint32_t c) { return cache_level(c); }
uint32_t t_record(uint32_t dk) { return cache_record(dk); }
uint32_t t_key_at(uint32_t dk, uint32_t f) { return cache_key_at(dk, f); }
uint32_t t_value_dword(uint32_t dk, uint32_t c, uint32_t g, uint32_t w) {
    return cache_values_at(dk) + cache_value_dword(c, g, w);
}
uint32_t t_frame_of(uint32_t g, uint32_t w, uint32_t i) { return cache_frame_of(g, w, i); }
uint32_t t_key_scale_at(uint32_t dk, uint32_t f) { return cache_key_scale_at(dk, f); }
uint32_t t_value_scale_at(uint32_t dk, uint32_t f) { return cache_value_scale_at(dk, f); }
int t_page_ok(int32_t id, uint32_t pages) { return cache_page_ok(id, pages); }
uint32_t t_tile_pages(uint32_t max_pages, int32_t left, int32_t right) { return cache_tile_pages(max_pages, left, right); }
uint32_t t_place_stride(uint32_t bw) { return place_stride(bw); }
uint32_t t_place_pad(void) { return kPlacePad; }
int32_t t_lo(int32_t pos, int32_t left) { return cache_lo(pos, left); }
int32_t t_hi(int32_t pos, int32_t right, int32_t total) { return cache_hi(pos, right, total); }

void t_span(uint32_t max_pages, uint32_t rows, uint32_t max_T, int32_t row0, int32_t row1, int32_t len, int32_t *out) {
    CacheStreams s = {};
    s.max_pages = max_pages, s.rows = rows, s.max_T = max_T;
    const CacheSpan p = cache_span(s, row0, row1, len);
    out[0] = p.r0, out[1] = p.T, out[2] = p.len, out[3] = p.total;
}

/* out: the call's r0, T, len, total, then the distances that its rows [a, b) need with this left */
int32_t t_most_left(uint32_t max_pages, uint32_t max_T) { return cache_most_left(max_pages, max_T); }
void t_places(uint32_t max_pages, uint32_t rows, uint32_t max_T, int32_t row0, int32_t row1, int32_t len, int32_t a,
              int32_t b, int32_t left, int32_t *out) {
    CacheStreams s = {};
    s.max_pages = max_pages, s.rows = rows, s.max_T = max_T;
    const CacheSpan p = cache_span(s, row0, row1, len);
    out[0] = p.r0, out[1] = p.T, out[2] = p.len, out[3] = p.total;
    out[4] = place_lo(p, p.r0 + b, left), out[5] = place_hi(p, p.r0 + a, left);
}

}
