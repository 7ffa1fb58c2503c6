/* The plan of a step of a cache's streams, made where it is used: what each
 * stream brings becomes its rows of the call, pages behind the window go back to
 * the pool, and new frames get pages of it. */
#include "q8_internal.h"

#include <hip/hip_runtime.h>

#pragma clang fp contract(off)

namespace pkq8 {

constexpr uint32_t kPlanThreads = 1024, kPlanWaves = kPlanThreads / 64;

/* The sum of v over a wave's lanes up to this one: within 16 lanes by shifts,
 * then the rows' last lanes to the rows behind. */
__device__ __forceinline__ uint32_t wave_scan(uint32_t v) {
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x111, 0xF, 0xF, false);
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x112, 0xF, 0xF, false);
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x114, 0xF, 0xF, false);
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x118, 0xF, 0xF, false);
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x142, 0xA, 0xF, false);
    v += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x143, 0xC, 0xF, false);
    return v;
}

/* N sums side by side of v over the threads up to this one, and over all. */
template <int N>
__device__ __forceinline__ void scan(uint32_t (&v)[N], uint32_t (&all)[N], uint32_t (*lds)[kPlanWaves]) {
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    __syncthreads();                        /* lds may still be read from the scan before */
#pragma unroll
    for (int n = 0; n < N; n++) {
        v[n] = wave_scan(v[n]);
        if (lane == 63)
            lds[n][wave] = v[n];
    }
    __syncthreads();
#pragma unroll
    for (int n = 0; n < N; n++) {
        const uint32_t of_waves = wave_scan(lds[n][lane % kPlanWaves]);      /* in the first row: those up to a wave */
        all[n] = (uint32_t)__builtin_amdgcn_readlane((int)of_waves, kPlanWaves - 1);
        const uint32_t w = __builtin_amdgcn_readfirstlane(wave);
        v[n] += w ? (uint32_t)__builtin_amdgcn_readlane((int)of_waves, w - 1) : 0;
    }
}

/* Which thread's run holds the n-th of all: the first whose inclusive sum is over n. */
__device__ __forceinline__ uint32_t run_of(const uint32_t *ends, uint32_t n) {
    uint32_t at = 0;
#pragma unroll
    for (uint32_t step = kPlanThreads / 2; step >= 1; step >>= 1)
        at += ends[at + step - 1] <= n ? step : 0;
    return at;
}

__device__ __forceinline__ int32_t slot_at(const PlanCall &p, uint32_t b, uint32_t f) {
    const int32_t id = p.table[(uint64_t)b * p.max_pages + f / kPage];
    return cache_page_ok(id, p.pages) ? (int32_t)(kPage * (uint32_t)id + f % kPage) : -1;
}

/* One workgroup, a thread a stream, 1024 streams at a time. The columns that
 * streams give back, and those that they take, are runs of different lengths:
 * all of them one after another are dealt to the threads, which find whose run
 * theirs is among the runs' ends, so a stream of an hour that ends is as quick
 * as many that give a page each, and pages enter and leave the queue in the order
 * of streams and columns whatever the threads do. With up to 1024 streams and
 * 4096 rows the rows' slots are made the same way; else by a launch behind.
 *
 * All of it is latency: 256 streams of one or two frames take 5.4 us, a chain
 * of what the streams bring, the table's entries given back, the queue's taken
 * and the sums between them (8 us with sums through LDS one at a time, and 3 for
 * a launch for the slots). */
template <bool SLOTS>
__global__ __launch_bounds__(kPlanThreads) void plan_kernel(PlanCall p) {
    __shared__ uint32_t sums[4][kPlanWaves];
    __shared__ uint32_t ends[kPlanThreads], from[kPlanThreads];
    __shared__ uint32_t row_ends[SLOTS ? kPlanThreads : 1], frames[SLOTS ? kPlanThreads : 1];
    const uint32_t tid = threadIdx.x;
    const int32_t cap = (int32_t)(p.max_pages * kPage);
    uint32_t head = (uint32_t)p.pool[0], free_pages = min((uint32_t)max(p.pool[1], 0), p.pages);
    head = head < p.pages ? head : 0;
    int32_t *ring = p.pool + 2;

    /* rows, and the pages given back */
    uint64_t rows = 0, asked = 0;           /* wanted of the streams before */
    uint32_t start = 0, T = 0;              /* the thread's stream's, of the last 1024 */
    for (uint32_t b0 = 0; b0 < p.B; b0 += kPlanThreads) {
        const uint32_t b = b0 + tid;
        const bool live = b < p.B;
        const uint32_t add = live ? (uint32_t)max(p.add[b], 0) : 0;
        const bool fresh = live && p.fresh && p.fresh[b] != 0;
        const int32_t had = live ? cache_clip(p.state[2 * (uint64_t)b], 0, cap) : 0;
        const int32_t gone = live ? max(p.state[2 * (uint64_t)b + 1], 0) : 0;
        start = fresh ? 0 : (uint32_t)had;
        const uint32_t want = min(add, min(p.max_T, (uint32_t)cap - start));
        const int32_t behind = p.left < 0 ? 0 : (int32_t)(max((int64_t)start - p.left, (int64_t)0) / kPage);
        const int32_t c0 = fresh ? 0 : max(gone, (int32_t)p.kept), c1 = fresh ? (had + (int32_t)kPage - 1) / (int32_t)kPage : behind;
        const uint32_t n = live ? (uint32_t)max(c1 - c0, 0) : 0;
        /* up to 2^31 each: 1024 of up to 2^21 rows, the columns of a table, halves of what is asked */
        uint32_t v[4] = { want, n, add & 0xffff, add >> 16 }, all[4];
        scan<4>(v, all, sums);
        const uint64_t upto = rows + v[0];
        const uint32_t r1 = (uint32_t)min(upto, (uint64_t)p.rows), r0 = (uint32_t)min(upto - want, (uint64_t)p.rows);
        rows += all[0];
        asked += all[2] + ((uint64_t)all[3] << 16);
        T = r1 - r0;
        if (live) {
            p.len[b] = (int32_t)start;
            if (b == 0)
                p.row0[0] = 0;
            p.row0[b + 1] = (int32_t)r1;
            p.state[2 * (uint64_t)b] = (int32_t)(start + T);
            p.state[2 * (uint64_t)b + 1] = fresh ? 0 : max(gone, behind);
        }
        if constexpr (SLOTS)
            row_ends[tid] = r1, frames[tid] = start + T - r1;       /* a row's frame, less its number (modulo 2^32) */
        ends[tid] = v[1];
        from[tid] = (uint32_t)c0 + n - v[1];                        /* a run's column, less its number among all */
        __syncthreads();
        for (uint32_t f = 0; f < all[1]; f += kPlanThreads) {
            const uint32_t at = f + tid;
            int32_t id = -1;
            if (at < all[1]) {
                const uint32_t who = run_of(ends, at);
                int32_t *entry = p.table + (uint64_t)(b0 + who) * p.max_pages + (from[who] + at);
                id = *entry;
                *entry = -1;
            }
            const bool held = cache_page_ok(id, p.pages);
            uint32_t rank[1] = { held }, given[1];
            scan<1>(rank, given, sums);
            if (held && free_pages + rank[0] <= p.pages)
                ring[(head + free_pages + rank[0] - 1) % p.pages] = id;
            free_pages = min(free_pages + given[0], p.pages);
        }
    }

    /* pages for new frames */
    uint32_t taken = 0;                     /* by the streams before */
    for (uint32_t b0 = 0; b0 < p.B; b0 += kPlanThreads) {
        if (p.B > kPlanThreads) {
            __syncthreads();
            const uint32_t b = b0 + tid;
            start = b < p.B ? (uint32_t)p.len[b] : 0;
            T = b < p.B ? (uint32_t)(p.row0[b + 1] - p.row0[b]) : 0;
        }
        const uint32_t c0 = (start + kPage - 1) / kPage, c1 = (start + T + kPage - 1) / kPage;
        uint32_t v[1] = { c1 - c0 }, all[1];
        scan<1>(v, all, sums);              /* its barriers also end the reads of `ends` and the writes of the ring */
        ends[tid] = v[0];
        from[tid] = c1 - v[0];
        __syncthreads();
        for (uint32_t at = tid; at < all[0]; at += kPlanThreads) {
            const uint32_t who = run_of(ends, at), n = taken + at;
            p.table[(uint64_t)(b0 + who) * p.max_pages + (from[who] + at)] = n < free_pages ? ring[(head + n) % p.pages] : -1;
        }
        taken += all[0];
    }
    if constexpr (SLOTS) {
        __syncthreads();
        const uint32_t in = (uint32_t)min(rows, (uint64_t)p.rows);
        for (uint32_t r = tid; r < p.rows; r += kPlanThreads) {
            const uint32_t who = r < in ? run_of(row_ends, r) : 0;
            p.slot[r] = r < in ? slot_at(p, who, frames[who] + r) : -1;
        }
    }
    if (tid == 0) {
        const uint32_t got = min(taken, free_pages);
        const uint64_t in = min(rows, (uint64_t)p.rows), out = asked - in;
        p.pool[0] = (int32_t)((head + (uint64_t)got) % p.pages);
        p.pool[1] = (int32_t)(free_pages - got);
        if (p.B == 0)
            p.row0[0] = 0;
        p.told[0] = (int32_t)in;
        p.told[1] = (int32_t)min(out, (uint64_t)INT32_MAX);
        p.told[2] = (int32_t)(taken - got);
        p.told[3] = (int32_t)(free_pages - got);
    }
}

/* Each row's place in the pool: 64 times its page, and its frame in it. */
__global__ __launch_bounds__(256) void slot_kernel(PlanCall p) {
    const uint32_t r = blockIdx.x * 256 + threadIdx.x;
    if (r >= p.rows)
        return;
    int32_t slot = -1;
    if (p.B && (int32_t)r < p.row0[p.B]) {
        uint32_t lo = 0, hi = p.B - 1;      /* the last stream that begins at r or before */
        while (lo < hi) {
            const uint32_t mid = (lo + hi + 1) / 2;
            if (p.row0[mid] <= (int32_t)r)
                lo = mid;
            else
                hi = mid - 1;
        }
        slot = slot_at(p, lo, (uint32_t)p.len[lo] + r - (uint32_t)p.row0[lo]);
    }
    p.slot[r] = slot;
}

int launch_plan(const PlanCall &c, hipStream_t s) {
    if (c.slot && c.B <= kPlanThreads && c.rows <= 4 * kPlanThreads) {
        plan_kernel<true><<<1, kPlanThreads, 0, s>>>(c);
    } else {
        plan_kernel<false><<<1, kPlanThreads, 0, s>>>(c);
        if (c.slot && c.rows)
            slot_kernel<<<(c.rows + 255) / 256, 256, 0, s>>>(c);
    }
    return hipPeekAtLastError() == hipSuccess ? 0 : -1;
}

}  // namespace pkq8
