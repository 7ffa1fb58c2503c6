/* The plan of a step of a cache's streams, made where it is used: what each
 * stream brings becomes its rows of the call, pages behind the window go back to
 * the pool, and new frames get pages of it. */
#include "q8_internal.h"

#include <hip/hip_runtime.h>

#pragma clang fp contract(off)

namespace pkq8 {

constexpr uint32_t kPlanThreads = 1024, kPlanWaves = kPlanThreads / 64;

/* The sum of v over the threads up to this one, and over all of them. */
template <typename T>
__device__ __forceinline__ T scan(T v, T *lds, T &all) {
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (uint32_t d = 1; d < 64; d <<= 1) {
        const T o = __shfl_up(v, d);
        v += lane >= d ? o : 0;
    }
    __syncthreads();                        /* lds may still be read from the scan before */
    if (lane == 63)
        lds[wave] = v;
    __syncthreads();
    T before = 0;
    all = 0;
#pragma unroll
    for (uint32_t i = 0; i < kPlanWaves; i++) {
        before += i < wave ? lds[i] : 0;
        all += lds[i];
    }
    return v + before;
}

/* Which thread's run holds the n-th of all: the first whose inclusive sum is over n. */
__device__ __forceinline__ uint32_t run_of(const uint32_t *ends, uint32_t n) {
    uint32_t at = 0;
#pragma unroll
    for (uint32_t step = kPlanThreads / 2; step >= 1; step >>= 1)
        at += ends[at + step - 1] <= n ? step : 0;
    return at;
}

/* One workgroup, a thread a stream, 1024 streams at a time. The columns that
 * streams give back, and those that they take, are runs of different lengths:
 * all of them one after another are dealt to the threads, which find whose run
 * theirs is among the runs' ends, so a stream of an hour that ends is as quick
 * as many that give a page each, and pages enter and leave the queue in the order
 * of streams and columns whatever the threads do. */
__global__ __launch_bounds__(kPlanThreads) void plan_kernel(PlanCall p) {
    __shared__ uint64_t sums[kPlanWaves];
    __shared__ uint32_t small[kPlanWaves];
    __shared__ uint32_t ends[kPlanThreads], from[kPlanThreads];
    const uint32_t tid = threadIdx.x;
    const int32_t cap = (int32_t)(p.max_pages * kPage);
    uint32_t head = (uint32_t)p.pool[0], free_pages = min((uint32_t)max(p.pool[1], 0), p.pages);
    head = head < p.pages ? head : 0;
    int32_t *ring = p.pool + 2;

    /* rows, and the pages given back */
    uint64_t rows = 0, asked = 0;           /* wanted of the streams before */
    for (uint32_t b0 = 0; b0 < p.B; b0 += kPlanThreads) {
        const uint32_t b = b0 + tid;
        const bool live = b < p.B;
        const int32_t add = live ? max(p.add[b], 0) : 0;
        const bool fresh = live && p.fresh && p.fresh[b] != 0;
        const int32_t had = live ? cache_clip(p.state[2 * (uint64_t)b], 0, cap) : 0;
        const int32_t gone = live ? max(p.state[2 * (uint64_t)b + 1], 0) : 0;
        const int32_t start = fresh ? 0 : had;
        const int32_t want = min(add, min((int32_t)p.max_T, cap - start));
        uint64_t all;
        const uint64_t upto = rows + scan<uint64_t>((uint64_t)want, sums, all);
        const int32_t r1 = (int32_t)min(upto, (uint64_t)p.rows), r0 = (int32_t)min(upto - want, (uint64_t)p.rows);
        rows += all;
        scan<uint64_t>((uint64_t)add, sums, all);
        asked += all;
        const int32_t behind = p.left < 0 ? 0 : (int32_t)(max((int64_t)start - p.left, (int64_t)0) / kPage);
        const int32_t c0 = fresh ? 0 : max(gone, (int32_t)p.kept), c1 = fresh ? (had + (int32_t)kPage - 1) / (int32_t)kPage : behind;
        if (live) {
            p.len[b] = start;
            if (b == 0)
                p.row0[0] = 0;
            p.row0[b + 1] = r1;
            p.state[2 * (uint64_t)b] = start + (r1 - r0);
            p.state[2 * (uint64_t)b + 1] = fresh ? 0 : max(gone, behind);
        }
        const uint32_t n = live ? (uint32_t)max(c1 - c0, 0) : 0;
        uint32_t total;
        const uint32_t end = scan<uint32_t>(n, small, total);
        ends[tid] = end;
        from[tid] = (uint32_t)c0 + n - end;             /* a run's column, less its number among all (modulo 2^32) */
        __syncthreads();
        for (uint32_t f = 0; f < total; f += kPlanThreads) {
            const uint32_t at = f + tid;
            int32_t id = -1;
            if (at < total) {
                const uint32_t who = run_of(ends, at);
                int32_t *entry = p.table + (uint64_t)(b0 + who) * p.max_pages + (from[who] + at);
                id = *entry;
                *entry = -1;
            }
            const bool held = cache_page_ok(id, p.pages);
            uint32_t given;
            const uint32_t rank = scan<uint32_t>(held, small, given);
            if (held && free_pages + rank <= p.pages)
                ring[(head + free_pages + rank - 1) % p.pages] = id;
            free_pages = min(free_pages + given, p.pages);
        }
        __syncthreads();
    }
    __syncthreads();

    /* pages for new frames */
    uint32_t taken = 0;                     /* by the streams before */
    for (uint32_t b0 = 0; b0 < p.B; b0 += kPlanThreads) {
        const uint32_t b = b0 + tid;
        const bool live = b < p.B;
        const uint32_t start = live ? (uint32_t)p.len[b] : 0, r1 = live ? (uint32_t)p.row0[b + 1] : 0;
        const uint32_t T = live ? r1 - (uint32_t)p.row0[b] : 0;
        const uint32_t c0 = (start + kPage - 1) / kPage, c1 = (start + T + kPage - 1) / kPage;
        uint32_t total;
        const uint32_t end = scan<uint32_t>(c1 - c0, small, total);
        __syncthreads();
        ends[tid] = end;
        from[tid] = c1 - end;
        __syncthreads();
        for (uint32_t at = tid; at < total; at += kPlanThreads) {
            const uint32_t who = run_of(ends, at), n = taken + at;
            p.table[(uint64_t)(b0 + who) * p.max_pages + (from[who] + at)] = n < free_pages ? ring[(head + n) % p.pages] : -1;
        }
        taken += total;
        __syncthreads();
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
        const uint32_t f = (uint32_t)p.len[lo] + r - (uint32_t)p.row0[lo];
        const int32_t id = p.table[(uint64_t)lo * p.max_pages + f / kPage];
        slot = cache_page_ok(id, p.pages) ? (int32_t)(kPage * (uint32_t)id + f % kPage) : -1;
    }
    p.slot[r] = slot;
}

int launch_plan(const PlanCall &c, hipStream_t s) {
    plan_kernel<<<1, kPlanThreads, 0, s>>>(c);
    if (c.slot && c.rows)
        slot_kernel<<<(c.rows + 255) / 256, 256, 0, s>>>(c);
    return hipPeekAtLastError() == hipSuccess ? 0 : -1;
}

}  // namespace pkq8
