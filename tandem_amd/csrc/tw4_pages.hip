// The bookkeeping of a step over a paged cache, on the GPU, from the lengths of the batch's requests: request i has c_i
// tokens in the cache and brings n_i more. With page size P, pages_i(x) = min(ceil(x / P), W) and W the width of the table,
//
//   start_i = n_0 + .. + n_(i-1)                      the request's first row among the step's tokens
//   len_i   = c_i + n_i
//   first_i = taken + sum over j < i of (pages_j(len_j) - pages_j(c_j))
//   table[i][pages_i(c_i) + j] = free[first_i + j]    for its j-th new page (-1 past the end of the list)
//   position of row t of request i = c_i + t - start_i
//   slot = table[i][position / P] P + position % P    (-1: no page, one past 2^31 slots, or a row behind the last request)
//   taken <- min(first_last, length of the list)
//
// It moves a few KB and is bound by a launch and three dependent round trips to memory (lengths, the list's entries, the table's): one
// request 3.3 us, 512 in decode 5.0, 64 prompts of 350 tokens on average 7.4. One workgroup does the scan and the tables, and for up to
// kInline rows the rows too: one launch for a decode step (against 4.7 us for one request in two). Past that a second launch spreads the
// rows over the GPU, finding each row's request by bisection in the starts: 8 requests of 1000 tokens take 6.3 us in two launches and 7.3 in
// one, but called eagerly 16.7 and 15.1, for the host's second launch; 16000 tokens take 6.4 and 12.1.
#include "tw4_attn.h"

namespace tw4 {

constexpr int kThreads = 1024, kPerThread = 4, kMaxBatch = kThreads * kPerThread, kInline = 8192;

struct PageArgs {
    const int32_t* context;
    const int32_t* fresh;
    int32_t* table;
    int64_t table_stride;
    const int32_t* free_pages;
    const int32_t* taken;
    int32_t* taken_out;
    int32_t* starts;
    int32_t* lens;
    int32_t* positions;
    int32_t* slots;
    int32_t* counts;
    int32_t* advance;  // tw4_plan_step: the requests' lengths for the next step, else null
    int batch, tokens, width, n_free, shift;
};

// The last i with starts[i] <= at, starts[0] = 0 (requests without tokens come before the one that has the row).
__device__ __forceinline__ int request_of(const int32_t* starts, int batch, int at) {
    int lo = 0, hi = batch;  // starts[lo] <= at, starts[hi] > at or hi = batch
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (starts[mid] <= at) lo = mid; else hi = mid;
    }
    return lo;
}

__device__ __forceinline__ int pages_of(int64_t tokens, const PageArgs& a) {
    return static_cast<int>(min((tokens + (1 << a.shift) - 1) >> a.shift, static_cast<int64_t>(a.width)));
}

// Row t's position and slot; context(i): the tokens request i had.
template <typename F>
__device__ __forceinline__ void place_row(const PageArgs& a, const int32_t* starts, F context, int t) {
    int pos = 0, slot = -1;
    if (t < starts[a.batch]) {
        const int i = request_of(starts, a.batch, t);
        pos = context(i) + (t - starts[i]);
        const int page = pos >> a.shift;
        const int id = static_cast<uint32_t>(page) < static_cast<uint32_t>(a.width) ? a.table[i * a.table_stride + page] : -1;
        if (id >= 0 && id <= 0x7FFFFFFF >> a.shift) slot = (id << a.shift) + (pos & ((1 << a.shift) - 1));
    }
    a.positions[t] = pos;
    a.slots[t] = slot;
}

// Sums over the workgroup of two values per thread, exclusive prefixes in `x`, `y`, totals in `tx`, `ty`.
__device__ __forceinline__ void scan2(int& x, int& y, int& tx, int& ty, int (*part)[2]) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int sx = x, sy = y;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int ox = __shfl_up(sx, d), oy = __shfl_up(sy, d);
        if (lane >= d) sx += ox, sy += oy;
    }
    if (lane == 63) part[wave][0] = sx, part[wave][1] = sy;
    __syncthreads();
    int bx = 0, by = 0;
    tx = ty = 0;
#pragma unroll
    for (int w = 0; w < kThreads / 64; ++w) {
        if (w == wave) bx = tx, by = ty;
        tx += part[w][0], ty += part[w][1];
    }
    x = bx + sx - x;
    y = by + sy - y;
}

// STEP: the table is a cache's own, so an entry behind a request's length is a page it already has (its length was taken back): it
// stays, and only entries that are none (-1) take pages, in the order of their places. Tokens behind row a.tokens - 1 are not computed in
// this step, so starts and lengths end there too: they come again, and find the pages they were given. One request in decode takes 3.0-3.2 us,
// 0.1 more than without STEP, 64 prompts of 40 tokens 0.5 more: a round trip to the entries and a scan of what they lack.
template <bool STEP>
__global__ void __launch_bounds__(kThreads) pages_kernel(PageArgs a, int rows) {
    __shared__ int part[kThreads / 64][2];
    __shared__ int32_t starts[kMaxBatch + 1], first[kMaxBatch + 1], context[kMaxBatch];
    const int tid = threadIdx.x, base = tid * kPerThread;
    int n[kPerThread], need[kPerThread], sum_n = 0, sum_need = 0;
    const int taken = min(max(*a.taken, 0), a.n_free);
#pragma unroll
    for (int j = 0; j < kPerThread; ++j) {
        const int i = base + j;
        n[j] = need[j] = 0;
        if (i < a.batch) {
            const int c = max(a.context[i], 0);
            n[j] = max(a.fresh[i], 0);
            need[j] = pages_of(static_cast<int64_t>(c) + n[j], a) - pages_of(c, a);
            context[i] = c;
            sum_n += n[j], sum_need += need[j];
        }
    }
    int total, pages;
    scan2(sum_n, sum_need, total, pages, part);
#pragma unroll
    for (int j = 0; j < kPerThread; ++j) {
        const int i = base + j;
        if (i < a.batch) {
            starts[i] = sum_n, first[i] = sum_need;
            // the lengths' arrays may be one: read above, written here
            if constexpr (STEP) {
                const int from = min(sum_n, a.tokens), to = min(sum_n + n[j], a.tokens);
                a.starts[i] = from;
                a.lens[i] = a.advance[i] = context[i] + (to - from);
            } else {
                a.starts[i] = sum_n;
                a.lens[i] = context[i] + n[j];
            }
            sum_n += n[j], sum_need += need[j];
        }
    }
    if (tid == 0) {
        starts[a.batch] = total, first[a.batch] = pages;
        a.starts[a.batch] = STEP ? min(total, a.tokens) : total;
    }
    __syncthreads();
    int missing = 0;  // of the places so far; without STEP all are
    if constexpr (STEP) {
        const int lane = tid & 63, wave = tid >> 6;
        for (int p0 = 0; p0 < pages; p0 += kThreads) {
            const int p = p0 + tid;
            int32_t* entry = nullptr;
            if (p < pages) {
                const int i = request_of(first, a.batch, p);
                entry = a.table + i * a.table_stride + pages_of(context[i], a) + (p - first[i]);
            }
            const bool none = entry && *entry < 0;
            const uint64_t all = __ballot(none);
            if (lane == 0) part[wave][0] = __popcll(all);
            __syncthreads();
            int before = missing;
#pragma unroll
            for (int w = 0; w < kThreads / 64; ++w) {
                if (w < wave) before += part[w][0];
                missing += part[w][0];
            }
            const int64_t from = static_cast<int64_t>(taken) + before + __popcll(all & ((1ULL << lane) - 1));
            if (none) *entry = from < a.n_free ? a.free_pages[from] : -1;
            __syncthreads();
        }
    } else {
        missing = pages;
        for (int p = tid; p < pages; p += kThreads) {
            const int i = request_of(first, a.batch, p);
            const int from = taken + p;
            a.table[i * a.table_stride + pages_of(context[i], a) + (p - first[i])] = from < a.n_free ? a.free_pages[from] : -1;
        }
    }
    if (tid == 0) {
        const int given = min(missing, a.n_free - taken);
        *a.taken_out = taken + given;
        a.counts[0] = total, a.counts[1] = given, a.counts[2] = missing - given;
        a.counts[3] = max(total - a.tokens, 0);
    }
    if (rows == 0) return;
    __threadfence_block();
    __syncthreads();
    for (int t = tid; t < rows; t += kThreads) place_row(a, starts, [&](int i) { return context[i]; }, t);
}

__global__ void __launch_bounds__(256) rows_kernel(PageArgs a) {
    const int t = blockIdx.x * 256 + threadIdx.x;
    // what a request had is its length less its rows: the context's array may be the lengths'
    if (t < a.tokens) place_row(a, a.starts, [&](int i) { return a.lens[i] - (a.starts[i + 1] - a.starts[i]); }, t);
}

// The pages of the listed requests go back to the front of what is left of the free list, each request's (1024 of them at a time) before
// those of the one before it;
// their rows of the table become -1 and their lengths 0. WHOLE: every page of the row, not those of the request's length only.
// It is bound by two barriers and a round trip to memory for each 1024 columns of each request, one after another: with 512 columns one
// request 1.7 us, 8 6.6, 64 47-49; with 2501 3.2, 19 and 142. One workgroup all the same: it runs when requests end, not in every step.
template <bool WHOLE>
__global__ void __launch_bounds__(kThreads) release_kernel(const int32_t* ended, int count, int32_t* table, int64_t table_stride,
                                                           int width, int32_t* lens, int batch, int32_t* free_pages, int n_free,
                                                           int32_t* taken, int shift) {
    __shared__ int part[kThreads / 64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int left = min(max(*taken, 0), n_free);
    for (int e = 0; e < count; ++e) {
        const int i = ended[e];
        if (i < 0 || i >= batch) continue;  // uniform
        const int held = WHOLE ? width
                               : static_cast<int>(min((static_cast<int64_t>(max(lens[i], 0)) + (1 << shift) - 1) >> shift,
                                                      static_cast<int64_t>(width)));
        for (int p0 = 0; p0 < width; p0 += kThreads) {
            const int p = p0 + static_cast<int>(threadIdx.x);
            const int id = p < held ? table[i * table_stride + p] : -1;
            if (p < width) table[i * table_stride + p] = -1;
            const uint64_t have = __ballot(id >= 0);
            if (lane == 0) part[wave] = __popcll(have);
            __syncthreads();
            int before = 0, sum = 0;
            for (int w = 0; w < kThreads / 64; ++w) {
                if (w < wave) before += part[w];
                sum += part[w];
            }
            before += __popcll(have & ((1ULL << lane) - 1));
            if (id >= 0 && left - sum + before >= 0) free_pages[left - sum + before] = id;
            left = max(left - sum, 0);
            __syncthreads();
        }
        if (threadIdx.x == 0) lens[i] = 0;
        __syncthreads();  // the same request again: nothing is left of it
    }
    if (threadIdx.x == 0) *taken = left;
}

}  // namespace tw4

using namespace tw4;

static int plan(const char* who, PageArgs a, int page_size, hipStream_t st) {
    a.shift = page_shift(page_size);
    TW4_REQUIRE(a.shift >= 0, TW4_EINVAL, "%s: page_size 16, 32, 64, 128 or 256 (%d)", who, page_size);
    TW4_REQUIRE(a.batch >= 1 && a.batch <= kMaxBatch, TW4_EINVAL, "%s: 1 to %d requests (%d)", who, kMaxBatch, a.batch);
    TW4_REQUIRE(a.tokens >= 0 && a.tokens < 1 << 30, TW4_EINVAL, "%s: 0 <= tokens < 2^30 (%d)", who, a.tokens);
    TW4_REQUIRE(a.width >= 0 && a.n_free >= 0 && a.table_stride >= a.width && static_cast<int64_t>(a.batch) * a.width < 1LL << 31,
                TW4_EINVAL, "%s: a table of fewer than 2^31 entries whose rows do not overlap (width %d, stride %lld)", who,
                a.width, static_cast<long long>(a.table_stride));
    TW4_REQUIRE(a.context && a.fresh && a.taken && a.taken_out && a.starts && a.lens && a.counts && (a.table || !a.width) &&
                    (a.free_pages || !a.n_free) && ((a.positions && a.slots) || !a.tokens),
                TW4_EINVAL, "%s: null pointer", who);
    const bool one = a.tokens <= kInline;
    if (a.advance)
        pages_kernel<true><<<1, kThreads, 0, st>>>(a, one ? a.tokens : 0);
    else
        pages_kernel<false><<<1, kThreads, 0, st>>>(a, one ? a.tokens : 0);
    TW4_LAUNCH_CHECK("plan_pages: launch");
    if (!one) {
        rows_kernel<<<(a.tokens + 255) / 256, 256, 0, st>>>(a);
        TW4_LAUNCH_CHECK("plan_pages: launch");
    }
    return TW4_OK;
}

extern "C" int tw4_plan_pages(const int32_t* context, const int32_t* fresh, int32_t* table, int64_t table_stride, int width,
                              const int32_t* free_pages, int n_free, const int32_t* taken, int32_t* taken_out, int page_size,
                              int32_t* starts, int32_t* lens, int32_t* positions, int32_t* slots, int32_t* counts, int batch,
                              int tokens, void* stream) {
    return plan("plan_pages",
                PageArgs{context, fresh, table, table_stride, free_pages, taken, taken_out, starts, lens, positions, slots, counts,
                         nullptr, batch, tokens, width, n_free, 0},
                page_size, static_cast<hipStream_t>(stream));
}

extern "C" int tw4_plan_step(int32_t* context, const int32_t* fresh, int32_t* table, int64_t table_stride, int width,
                             const int32_t* free_pages, int n_free, int32_t* taken, int page_size, int32_t* starts, int32_t* lens,
                             int32_t* positions, int32_t* slots, int32_t* counts, int batch, int tokens, void* stream) {
    TW4_REQUIRE(lens != context, TW4_EINVAL, "plan_step: the step's lengths and the requests' must be two arrays");
    return plan("plan_step",
                PageArgs{context, fresh, table, table_stride, free_pages, taken, taken, starts, lens, positions, slots, counts,
                         context, batch, tokens, width, n_free, 0},
                page_size, static_cast<hipStream_t>(stream));
}

static int release(const char* who, bool whole, const int32_t* ended, int count, int32_t* table, int64_t table_stride, int width,
                   int32_t* lens, int batch, int32_t* free_pages, int n_free, int32_t* taken, int page_size, hipStream_t st) {
    const int shift = page_shift(page_size);
    TW4_REQUIRE(shift >= 0, TW4_EINVAL, "%s: page_size 16, 32, 64, 128 or 256 (%d)", who, page_size);
    TW4_REQUIRE(count >= 0 && batch >= 1 && width >= 0 && n_free >= 0 && table_stride >= width, TW4_EINVAL,
                "%s: bad sizes (%d of %d requests, width %d)", who, count, batch, width);
    if (count == 0) return TW4_OK;
    TW4_REQUIRE(ended && (table || !width) && lens && taken && (free_pages || !n_free), TW4_EINVAL, "%s: null pointer", who);
    if (whole)
        release_kernel<true><<<1, kThreads, 0, st>>>(ended, count, table, table_stride, width, lens, batch, free_pages, n_free, taken, shift);
    else
        release_kernel<false><<<1, kThreads, 0, st>>>(ended, count, table, table_stride, width, lens, batch, free_pages, n_free, taken, shift);
    TW4_LAUNCH_CHECK("release_pages: launch");
    return TW4_OK;
}

extern "C" int tw4_release_pages(const int32_t* ended, int count, int32_t* table, int64_t table_stride, int width,
                                 int32_t* lens, int batch, int32_t* free_pages, int n_free, int32_t* taken, int page_size,
                                 void* stream) {
    return release("release_pages", false, ended, count, table, table_stride, width, lens, batch, free_pages, n_free, taken, page_size,
                   static_cast<hipStream_t>(stream));
}

extern "C" int tw4_release_lanes(const int32_t* ended, int count, int32_t* table, int64_t table_stride, int width,
                                 int32_t* lens, int batch, int32_t* free_pages, int n_free, int32_t* taken, int page_size,
                                 void* stream) {
    return release("release_lanes", true, ended, count, table, table_stride, width, lens, batch, free_pages, n_free, taken, page_size,
                   static_cast<hipStream_t>(stream));
}
