// Page bookkeeping of a batch of requests on gfx950: block tables, slot map,
// positions and newest rows of a step, built from the requests' lengths, and
// the plain append of a step's K and V rows through the slot map.
//
// With L_b the committed tokens of request b, n_b its new ones, P tokens a
// page and F free pages:
//   off_b   = n_0 + .. + n_{b-1}            first row of request b
//   held_b  = ceil(L_b / P)                 pages it holds
//   need_b  = ceil((L_b + n_b) / P) - held_b
//   first_b = need_0 + .. + need_{b-1}
//   table[b][held_b + i] = free[F - 1 - (first_b + i)],  0 <= i < need_b
//   row t in [off_b, off_b + n_b): position p = L_b + t - off_b,
//   slot = table[b][p div P] * P + p mod P.
// Both sums run in request order, so a step's result is the same in every
// run. Nothing that a step reads is written by it (the table's new entries
// lie behind the held ones, the free list stands until the commit), so its
// workgroups need no order among them and a repeated step repeats its result.
#include "context.hpp"
#include "paged.hpp"

#include <algorithm>
#include <cstdio>

namespace pcl {

constexpr int kPageThreads = 256;

enum { kCountFree, kCountRows, kCountTaken, kCountState, kCounters };

struct PageParams {
    int32_t *lengths, *table, *free_pages, *counters, *step_lengths, *newest;
    int32_t *slots, *positions, *row_request;
    const int32_t *in; // new tokens, kept tokens or finished flags per request
    int64_t table_stride;
    int requests, pages, step_rows;
    uint32_t page_tokens, max_tokens; // tokens a request may hold
    int *err;
};

// Tokens request i holds, or ~0 when its length is outside the table.
__device__ __forceinline__ uint32_t held_tokens(const PageParams &p, const int32_t *lengths,
                                                int i)
{
    const int32_t n = lengths[i];
    return n >= 0 && (uint32_t)n <= p.max_tokens ? (uint32_t)n : ~0u;
}

// Four words at any word's address.
typedef int32_t int4w __attribute__((ext_vector_type(4), aligned(4)));

__device__ __forceinline__ bool in_pools(const PageParams &p, int32_t page)
{
    return page >= 0 && page < p.pages;
}

// The first workgroup writes the words of each request and the counters, the
// others have one thread per row of the step; every workgroup forms the sums over
// all requests by itself (they are a few loads a thread). The rows look at their
// own pages, the first workgroup at every page under a new token: with one outside
// the pools the step does not stand (the look at 64000 pages beside 1024000 rows
// costs 0.5 us of 17). A decode step is a chain of latencies: the lengths' load,
// the two scans in one 64-bit sum, the search, the page's load. Profiled durations:
// 3.9 us for 64 requests, 5.5 us for 512 requests and 7163 rows, 5.0 us for 96
// prompts of 136277 rows; a call takes 7.7 us, the host's time.
__global__ __launch_bounds__(kPageThreads) void page_step_kernel(PageParams p)
{
    extern __shared__ uint32_t offsets[]; // rows [requests + 1], pages [requests]
    __shared__ uint64_t waves[kPageThreads / 64];
    uint32_t *row_off = offsets, *page_off = offsets + p.requests + 1;
    const int tid = threadIdx.x;
    const bool books = blockIdx.x == 0;
    const int per = (p.requests + kPageThreads - 1) / kPageThreads;
    const int i0 = min(tid * per, p.requests), i1 = min(i0 + per, p.requests);
    const int free_count = p.counters[kCountFree];
    uint64_t sum = 0; // rows in the low half, pages in the high half
    uint32_t held_page = 0; // (a negative number is the largest)
    bool bad = false;
    for (int i = i0; i < i1; ++i) {
        const uint32_t len = held_tokens(p, p.lengths, i);
        const int32_t n = p.in[i];
        const bool fits = len != ~0u && n >= 0 && n <= p.step_rows &&
                          (uint32_t)n <= p.max_tokens - len;
        bad |= !fits;
        const uint32_t rows = fits ? (uint32_t)n : 0;
        const uint32_t need =
            fits ? pages_of(len + rows, p.page_tokens) - pages_of(len, p.page_tokens) : 0;
        row_off[i] = rows;
        page_off[i] = need;
        sum += (uint64_t)need << 32 | rows;
        // the step goes on in a held page (its number is looked at behind the sums)
        if (books && rows && len % p.page_tokens)
            held_page = max(held_page,
                            (uint32_t)p.table[i * p.table_stride + len / p.page_tokens]);
    }
    uint64_t total;
    uint64_t at = block_offsets(sum, waves, &total);
    for (int i = i0; i < i1; ++i) {
        const uint32_t rows = row_off[i], need = page_off[i];
        row_off[i] = (uint32_t)at;
        page_off[i] = (uint32_t)(at >> 32);
        at += (uint64_t)need << 32 | rows;
    }
    const uint32_t rows = (uint32_t)total, taken = (uint32_t)(total >> 32);
    if (tid == 0)
        row_off[p.requests] = rows;
    const bool had = free_count >= 0 && free_count <= p.pages && (int64_t)taken <= free_count;
    bad |= !had || rows > (uint32_t)p.step_rows;
    bool damaged = held_page >= (uint32_t)p.pages;
    // (the first words ahead of the barrier: a decode step takes no more)
    if (books && had && (uint32_t)tid < taken)
        damaged |= !in_pools(p, p.free_pages[free_count - 1 - tid]);
    const bool ok = !__syncthreads_or(bad);

    if (books) {
        for (int i = tid; i < p.requests; i += kPageThreads) {
            const uint32_t n = ok ? row_off[i + 1] - row_off[i] : 0;
            p.step_lengths[i] = (int32_t)((uint32_t)p.lengths[i] + n);
            p.newest[i] = n ? (int32_t)(row_off[i] + n - 1) : -1;
        }
        // the other words, four to a load (past the last four those again)
        constexpr uint32_t kAhead = 4, kRound = 4 * kAhead * kPageThreads;
        for (uint32_t u0 = 0; ok && u0 + kPageThreads < taken; u0 += kRound) {
            int4w words[kAhead];
#pragma unroll
            for (uint32_t j = 0; j < kAhead; ++j)
                words[j] = *(const int4w *)(p.free_pages + free_count - taken +
                                            min(u0 + 4 * (j * kPageThreads + tid), taken - 4));
#pragma unroll
            for (uint32_t j = 0; j < kAhead; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    damaged |= !in_pools(p, words[j][e]);
        }
        damaged = __syncthreads_or(damaged);
        if (tid == 0) {
            p.counters[kCountRows] = ok ? (int32_t)rows : 0;
            p.counters[kCountTaken] = ok ? (int32_t)taken : 0;
            p.counters[kCountState] = ok && !damaged;
            if (!ok || damaged)
                atomicOr(p.err, kErrPages);
        }
        return;
    }
    const uint32_t t = (blockIdx.x - 1) * kPageThreads + tid;
    if (t >= (uint32_t)p.step_rows)
        return;
    int32_t slot = -1, position = -1, request = -1;
    if (ok && t < rows) {
        request = find_range(row_off, p.requests, t);
        const uint32_t len = (uint32_t)p.lengths[request];
        const uint32_t pos = len + (t - row_off[request]);
        const uint32_t column = pos / p.page_tokens, held = pages_of(len, p.page_tokens);
        int32_t *entry = p.table + request * p.table_stride + column;
        const int32_t page =
            column < held
                ? *entry
                : p.free_pages[free_count - 1 - (int)(page_off[request] + column - held)];
        const bool in = in_pools(p, page); // else the table or free list is damaged
        position = (int32_t)pos;
        // a new page's first token is its first row (a number outside the pools
        // leaves no earlier request's page in its place)
        if (column >= held && pos % p.page_tokens == 0)
            *entry = in ? page : -1;
        if (in)
            slot = page * (int32_t)p.page_tokens + (int32_t)(pos % p.page_tokens);
    }
    p.slots[t] = slot;
    p.positions[t] = position;
    p.row_request[t] = request;
}

// Finds out whether the `total` pages returned(u) of a release can go back: each
// lies in the pools and no other returned(u) and none of the `held` pages kept(v)
// is the same one, for a page that block tables share would come to be free while
// a request holds it, or free twice. The top bit of word w of free_pages marks page
// w while the workgroup looks (page numbers leave it clear; behind the list it is
// cleared first). free_pages' first free_count words are left as they were. Ends
// with a barrier.
template <int THREADS, typename Returned, typename Kept>
__device__ __forceinline__ bool pages_can_return(const PageParams &p, int free_count,
                                                 uint32_t total, uint32_t held,
                                                 Returned returned, Kept kept)
{
    constexpr int32_t kMark = INT32_MIN;
    const uint32_t tid = threadIdx.x;
    constexpr int kAhead = 8; // words a thread has in flight
    bool bad = false;
    for (int64_t w0 = tid; w0 < p.pages; w0 += kAhead * THREADS) {
        int32_t word[kAhead];
#pragma unroll
        for (int j = 0; j < kAhead; ++j)
            word[j] = w0 + j * THREADS < p.pages ? p.free_pages[w0 + j * THREADS] : 0;
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
            const int64_t w = w0 + j * THREADS;
            if (word[j] >= 0)
                continue;
            if (w < free_count)
                bad = true; // no page number
            else
                p.free_pages[w] = word[j] & ~kMark;
        }
    }
    if (__syncthreads_or(bad))
        return false;
    for (uint32_t u = tid; u < total; u += THREADS) {
        const int32_t page = returned(u);
        bad |= !in_pools(p, page) || atomicOr(p.free_pages + page, kMark) < 0;
    }
    __syncthreads();
    for (uint32_t v = tid; v < held; v += THREADS) {
        const int32_t page = kept(v);
        bad |= in_pools(p, page) && __hip_atomic_load(p.free_pages + page, __ATOMIC_RELAXED,
                                                      __HIP_MEMORY_SCOPE_AGENT) < 0;
    }
    __syncthreads();
    for (uint32_t u = tid; u < total; u += THREADS) {
        const int32_t page = returned(u);
        if (in_pools(p, page))
            atomicAnd(p.free_pages + page, ~kMark);
    }
    return !__syncthreads_or(bad);
}

// The pages behind the kept ones of every request go back on the free list,
// in the order of the requests and of their pages: one workgroup. KEEP: the
// step's commit (`in`: the tokens kept of each request's new ones, null for
// all); otherwise the release of the requests whose flag is set. Where a page
// cannot go back nothing changes. Profiled durations: 3.7 us for the commit of 64
// requests; a release of nobody 4.2 us, of one of 96 prompts (90 pages of 8484)
// 19 us, of all of them 30 us, of 256 requests of 250 pages 0.19 ms: three looks
// at every page that goes back, one at every page that stays and one at every word
// of the list, 1024 at a time.
template <bool KEEP> constexpr int kReturnThreads = KEEP ? kPageThreads : 1024;

template <bool KEEP>
__global__ __launch_bounds__(kReturnThreads<KEEP>) void page_return_kernel(PageParams p)
{
    constexpr int kThreads = kReturnThreads<KEEP>;
    // before each request, and in all: the pages that go back [requests + 1] and
    // (a release) the pages that stay [requests + 1]
    extern __shared__ uint32_t offsets[];
    __shared__ uint64_t waves[kThreads / 64];
    uint32_t *stay_off = offsets + p.requests + 1;
    const int tid = threadIdx.x;
    if (KEEP && p.counters[kCountState] != 1)
        return; // no step stands
    const int per = (p.requests + kThreads - 1) / kThreads;
    const int i0 = min(tid * per, p.requests), i1 = min(i0 + per, p.requests);
    const int64_t free_count = (int64_t)p.counters[kCountFree] - (KEEP ? p.counters[kCountTaken] : 0);
    uint64_t sum = 0, stay_sum = 0; // (lengths that are wrong may add up past 2^32)
    bool bad = false;
    // tokens request i holds before the call (with the step's) and after it
    auto tokens = [&](int i, uint32_t *now, uint32_t *after) {
        const uint32_t len = held_tokens(p, p.lengths, i);
        *now = KEEP ? held_tokens(p, p.step_lengths, i) : len;
        bool in = len != ~0u && *now != ~0u && *now >= len;
        if (KEEP) {
            const int32_t kept = p.in ? p.in[i] : (int32_t)(*now - len);
            in = in && kept >= 0 && (uint32_t)kept <= *now - len;
            *after = len + (uint32_t)kept;
        } else {
            *after = p.in[i] ? 0 : len;
        }
        return in;
    };
    for (int i = i0; i < i1; ++i) {
        uint32_t now, after;
        const bool in = tokens(i, &now, &after);
        bad |= !in;
        const uint32_t stay = in ? pages_of(after, p.page_tokens) : 0;
        const uint32_t n = in ? pages_of(now, p.page_tokens) - stay : 0;
        offsets[i] = n;
        sum += n;
        if (!KEEP) {
            stay_off[i] = stay;
            stay_sum += stay;
        }
    }
    uint64_t all, stay_all = 0;
    auto add_up = [&](uint32_t *off, uint64_t mine, uint64_t *whole) {
        uint64_t at = block_offsets(mine, waves, whole);
        for (int i = i0; i < i1; ++i) {
            const uint32_t n = off[i];
            off[i] = (uint32_t)at;
            at += n;
        }
        if (tid == 0)
            off[p.requests] = (uint32_t)*whole;
    };
    add_up(offsets, sum, &all);
    if (!KEEP && all)
        add_up(stay_off, stay_sum, &stay_all);
    const uint32_t total = (uint32_t)all;
    // (more than 2^31 pages stay only where tables share them)
    bad |= free_count < 0 || free_count + (int64_t)all > p.pages || stay_all > INT32_MAX;
    auto refused = [&]() {
        const bool any = __syncthreads_or(bad);
        if (any && tid == 0)
            atomicOr(p.err, kErrPages);
        return any;
    };
    if (refused())
        return;
    if (total) {
        auto page_at = [&](uint32_t u) { // page u of those that go back
            const int i = find_range(offsets, p.requests, u);
            uint32_t now, after = 0;
            if (KEEP)
                tokens(i, &now, &after);
            return p.table[i * p.table_stride + pages_of(after, p.page_tokens) + (u - offsets[i])];
        };
        if constexpr (KEEP) {
            for (uint32_t u = tid; u < total; u += kThreads)
                bad |= !in_pools(p, page_at(u));
        } else {
            bad = !pages_can_return<kThreads>(
                p, (int)free_count, total, (uint32_t)stay_all, page_at, [&](uint32_t v) {
                    const int i = find_range(stay_off, p.requests, v);
                    return p.table[i * p.table_stride + (v - stay_off[i])];
                });
        }
        if (refused())
            return;
        for (uint32_t u = tid; u < total; u += kThreads)
            p.free_pages[free_count + u] = page_at(u);
    }
    __syncthreads(); // the lengths are read above
    for (int i = i0; i < i1; ++i) {
        uint32_t now, after;
        tokens(i, &now, &after);
        p.lengths[i] = (int32_t)after;
    }
    if (tid == 0) {
        p.counters[kCountFree] = (int32_t)(free_count + total);
        p.counters[kCountState] = 0;
    }
}

// An empty batch: no tokens, every page free (page 0 is taken first), no step.
__global__ __launch_bounds__(kPageThreads) void page_reset_kernel(PageParams p)
{
    const int64_t step = (int64_t)gridDim.x * kPageThreads;
    const int64_t t0 = (int64_t)blockIdx.x * kPageThreads + threadIdx.x;
    for (int64_t i = t0; i < p.requests * p.table_stride; i += step)
        p.table[i] = -1;
    for (int64_t i = t0; i < p.pages; i += step)
        p.free_pages[i] = p.pages - 1 - (int32_t)i;
    for (int64_t i = t0; i < p.requests; i += step) {
        p.lengths[i] = 0;
        p.step_lengths[i] = 0;
        p.newest[i] = -1;
    }
    for (int64_t i = t0; i < p.step_rows; i += step) {
        p.slots[i] = -1;
        p.positions[i] = -1;
        p.row_request[i] = -1;
    }
    if (t0 < kCounters)
        p.counters[t0] = t0 == kCountFree ? p.pages : 0;
}

struct RowsParams {
    const float *keys, *values; // [n][width]
    void *k, *v;                // pools
    const int32_t *slots;
    int n, width;
    int total; // slots of the pools
    int *err;
};

// One wave per row and array, eight 16-byte loads a lane in flight. HBM-bound on
// a prompt's rows: 3001 rows of 2 x 512 into f32 pages, 49 MB read and written,
// 10.8 us (4.5 TB/s; a plain copy of 4 GiB reaches 4.7).
template <typename T>
__global__ __launch_bounds__(256) void paged_rows_kernel(RowsParams p)
{
    constexpr int kAhead = 8; // 16-byte pieces a lane has in flight
    const int lane = threadIdx.x & 63;
    const int row = blockIdx.x * 4 + (threadIdx.x >> 6);
    if (row >= p.n)
        return;
    const float *src = (blockIdx.y ? p.values : p.keys) + (int64_t)row * p.width;
    T *pool = static_cast<T *>(blockIdx.y ? p.v : p.k);
    const int slot = p.slots[row];
    if (slot < 0)
        return;
    if (slot >= p.total) {
        if (lane == 0)
            atomicOr(p.err, kErrPages);
        return;
    }
    T *dst = pool + (int64_t)slot * p.width;
    for (int c = 4 * lane; c < p.width; c += 256 * kAhead) {
        f4 v[kAhead];
#pragma unroll
        for (int i = 0; i < kAhead; ++i)
            v[i] = c + 256 * i < p.width ? ldg4_stream(src + c + 256 * i) : f4{};
#pragma unroll
        for (int i = 0; i < kAhead; ++i)
            if (c + 256 * i < p.width)
                store_row4(dst + c + 256 * i, v[i]);
    }
}

bool valid_pools(const pcl_page_pools &s)
{
    return s.k && s.v && (s.type == PCL_CACHE_F32 || s.type == PCL_CACHE_BF16) && s.pages > 0 &&
           s.page_tokens > 0 && s.page_tokens <= kMaxPageTokens &&
           s.pages <= kMaxSlots / s.page_tokens && s.kvheads > 0 && s.kvheads <= 4096 &&
           s.dim > 0 && s.dim % 16 == 0 && s.dim <= 512 &&
           ((uintptr_t)s.k | (uintptr_t)s.v) % 16 == 0;
}

} // namespace pcl

namespace {

using pcl::PageParams;

int launched(const char *what)
{
    const hipError_t e = hipGetLastError();
    if (e == hipSuccess)
        return PCL_OK;
    std::fprintf(stderr, "pcl_page: %s: %s\n", what, hipGetErrorString(e));
    return PCL_NON_FINITE_VALUE;
}

int page_params(pcl_context *ctx, const pcl_page_batch *b, PageParams *p)
{
    if (!ctx || !b || b->requests <= 0 || b->requests > pcl::kMaxRequests || b->table_stride <= 0 ||
        b->table_stride > pcl::kMaxSlots || b->page_tokens <= 0 ||
        b->page_tokens > pcl::kMaxPageTokens || b->pages <= 0 ||
        b->pages > pcl::kMaxSlots / b->page_tokens || b->step_rows <= 0 ||
        b->step_rows > pcl::kMaxStepRows)
        return PCL_INVALID_SHAPE;
    const void *words[] = {b->lengths,      b->table,  b->free_pages, b->counters,   b->step_lengths,
                           b->newest,       b->slots,  b->positions,  b->row_request};
    for (const void *w : words)
        if (!w || (uintptr_t)w % 4)
            return PCL_INVALID_SHAPE;
    p->lengths = b->lengths;
    p->table = b->table;
    p->free_pages = b->free_pages;
    p->counters = b->counters;
    p->step_lengths = b->step_lengths;
    p->newest = b->newest;
    p->slots = b->slots;
    p->positions = b->positions;
    p->row_request = b->row_request;
    p->in = nullptr;
    p->table_stride = b->table_stride;
    p->requests = (int)b->requests;
    p->pages = (int)b->pages;
    p->step_rows = (int)b->step_rows;
    p->page_tokens = (uint32_t)b->page_tokens;
    p->max_tokens =
        (uint32_t)std::min<int64_t>(b->table_stride * b->page_tokens, pcl::kMaxSlots);
    p->err = ctx->err;
    (void)hipSetDevice(ctx->device);
    return PCL_OK;
}

} // namespace

extern "C" {

int pcl_page_reset(pcl_context *ctx, const pcl_page_batch *batch)
{
    PageParams p;
    const int rc = page_params(ctx, batch, &p);
    if (rc != PCL_OK)
        return rc;
    const int64_t words = std::max<int64_t>(
        {batch->requests * batch->table_stride, batch->pages, batch->step_rows});
    const int64_t groups = std::min<int64_t>((words + 255) / 256, 1024);
    pcl::page_reset_kernel<<<(unsigned)groups, pcl::kPageThreads, 0, ctx->stream>>>(p);
    return launched("reset");
}

int pcl_page_step(pcl_context *ctx, const pcl_page_batch *batch, const int32_t *new_tokens)
{
    PageParams p;
    const int rc = page_params(ctx, batch, &p);
    if (rc != PCL_OK)
        return rc;
    if (!new_tokens || (uintptr_t)new_tokens % 4)
        return PCL_INVALID_SHAPE;
    p.in = new_tokens;
    const int groups = 1 + (p.step_rows + pcl::kPageThreads - 1) / pcl::kPageThreads;
    const size_t lds = (2 * (size_t)p.requests + 1) * sizeof(uint32_t);
    pcl::page_step_kernel<<<groups, pcl::kPageThreads, lds, ctx->stream>>>(p);
    return launched("step");
}

int pcl_page_commit(pcl_context *ctx, const pcl_page_batch *batch, const int32_t *kept)
{
    PageParams p;
    const int rc = page_params(ctx, batch, &p);
    if (rc != PCL_OK)
        return rc;
    if ((uintptr_t)kept % 4)
        return PCL_INVALID_SHAPE;
    p.in = kept;
    const size_t lds = ((size_t)p.requests + 1) * sizeof(uint32_t);
    pcl::page_return_kernel<true><<<1, pcl::kReturnThreads<true>, lds, ctx->stream>>>(p);
    return launched("commit");
}

int pcl_page_release(pcl_context *ctx, const pcl_page_batch *batch, const int32_t *finished)
{
    PageParams p;
    const int rc = page_params(ctx, batch, &p);
    if (rc != PCL_OK)
        return rc;
    if (!finished || (uintptr_t)finished % 4)
        return PCL_INVALID_SHAPE;
    p.in = finished;
    const size_t lds = 2 * ((size_t)p.requests + 1) * sizeof(uint32_t);
    pcl::page_return_kernel<false><<<1, pcl::kReturnThreads<false>, lds, ctx->stream>>>(p);
    return launched("release");
}

int pcl_paged_append(pcl_context *ctx, const pcl_page_pools *pools, const int32_t *slots,
                     const float *keys, const float *values, int64_t n)
{
    if (!ctx || !pools || !pcl::valid_pools(*pools) || n < 0 || n > pcl::kMaxStepRows)
        return PCL_INVALID_SHAPE;
    if (n == 0)
        return PCL_OK;
    if (!slots || !keys || !values || (uintptr_t)slots % 4 ||
        ((uintptr_t)keys | (uintptr_t)values) % 16)
        return PCL_INVALID_SHAPE;
    pcl::RowsParams p;
    p.keys = keys;
    p.values = values;
    p.k = pools->k;
    p.v = pools->v;
    p.slots = slots;
    p.n = (int)n;
    p.width = (int)(pools->kvheads * pools->dim);
    p.total = (int)(pools->pages * pools->page_tokens);
    p.err = ctx->err;
    (void)hipSetDevice(ctx->device);
    const dim3 grid((unsigned)((n + 3) / 4), 2);
    if (pools->type == PCL_CACHE_F32)
        pcl::paged_rows_kernel<float><<<grid, 256, 0, ctx->stream>>>(p);
    else
        pcl::paged_rows_kernel<__bf16><<<grid, 256, 0, ctx->stream>>>(p);
    return launched("append");
}

} // extern "C"
