// Drafted trees and shared pages of a batch on gfx950: what each new token of a
// step sees of the others, which rows a verified branch moves, requests that begin
// as copies of others, pages given back where nobody else holds them, and copies
// of rows in the pages of several layers.
//
// With L_b the held tokens of request b, n_b its new ones of the standing step, P
// tokens a page and par the parent of a new token among its request's (-1: it
// follows the held ones):
//   branch(i) = {i} + branch(par(i)),  position(i) = L_b + |branch(i)| - 1,
//   a verified branch c_0 < c_1 < ..: row at position L_b + c_k to L_b + k;
//   request f that begins as a copy of s: table[f][j] = table[s][j] for the whole
//   pages j < L_s div P, and a page of its own for the L_s mod P tokens behind;
//   pages that go back: those of the finished requests' tables that no other
//   request's holds.
// All but the copies are short, bound by their chains of dependent loads and by the
// launch (MI355X, profiled durations): masks of 16 trees of 12 and of 256 of 64, 3.0 and
// 3.8 us; accepted branches 3.2 and 3.4; a fork 4.4 (32 requests from 8 of up to 4000
// tokens, pages of 16) and 6.0 (480 from 16 of up to 8192, pages of 8); their releases 8.0
// in one workgroup, 1.8 + 4.4 + 4.4 in three launches. Copies of 192 part-filled pages of
// 64 tokens in four layers of 2 x 512, f32, 402 MB read and written, 89 us (4.5 TB/s; a
// plain copy of 4 GiB 4.7), of 64 branches of up to 5 rows in six layers 6.3 us.
#include "context.hpp"
#include "page_batch.hpp"
#include "paged.hpp"

#include <algorithm>
#include <cstdio>

namespace pcl {

constexpr int64_t kMaxTreeWords = 8;

struct TreeStepParams {
    PageParams b;
    const int32_t *parents;
    int32_t *positions;
    uint64_t *masks;
    int words;
};

// Request i's part of the standing step: its new tokens, and the row of the first;
// 0 new tokens where it has none or they do not fit the step (*bad).
__device__ __forceinline__ int step_tokens(const PageParams &p, int i, int *first, bool *bad)
{
    const uint32_t len = held_tokens(p, p.lengths, i), after = held_tokens(p, p.step_lengths, i);
    const int32_t last = p.newest[i];
    *first = 0;
    if (last < 0)
        return 0;
    const int64_t n = (int64_t)after - len, row = last - n + 1;
    if (len == ~0u || after == ~0u || n <= 0 || row < 0 || last >= p.step_rows) {
        *bad = true;
        return 0;
    }
    *first = (int)row;
    return (int)n;
}

// One workgroup per request; a thread walks up its token's branch in LDS. Rows
// behind the step's last are dealt over the workgroups.
template <int WORDS>
__global__ __launch_bounds__(64 * WORDS) void page_tree_kernel(TreeStepParams t)
{
    constexpr int kThreads = 64 * WORDS;
    __shared__ int16_t parents[kThreads];
    const PageParams &p = t.b;
    const int b = blockIdx.x, i = threadIdx.x;
    const bool stands = p.counters[kCountState] == kStepStands;
    const int rows = stands ? min(max(p.counters[kCountRows], 0), p.step_rows) : 0;
    for (int r = rows + b * kThreads + i; r < p.step_rows; r += gridDim.x * kThreads) {
        t.positions[r] = -1;
        for (int w = 0; w < t.words; ++w)
            t.masks[(int64_t)r * t.words + w] = 0;
    }
    if (!stands)
        return;
    int first;
    bool bad = false;
    const int n = step_tokens(p, b, &first, &bad);
    const int held = p.lengths[b];
    if (n > 64 * t.words) {
        // no tree of so many tokens: each sees the held ones alone
        bad = true;
        for (int j = i; j < n; j += kThreads) {
            t.positions[first + j] = held + j;
            for (int w = 0; w < t.words; ++w)
                t.masks[(int64_t)(first + j) * t.words + w] = 0;
        }
    } else if (n > 0) {
        int parent = i < n ? t.parents[first + i] : -1;
        // (a parent that does not come before its token is none)
        if (parent < -1 || parent >= i) {
            bad |= i < n;
            parent = -1;
        }
        parents[i] = (int16_t)parent;
        __syncthreads();
        if (i < n) {
            uint64_t mask[WORDS] = {};
            int depth = -1;
            for (int at = i; at >= 0; at = parents[at], ++depth)
#pragma unroll
                for (int w = 0; w < WORDS; ++w)
                    mask[w] |= at / 64 == w ? (uint64_t)1 << (at % 64) : 0;
            t.positions[first + i] = held + depth;
#pragma unroll
            for (int w = 0; w < WORDS; ++w)
                if (w < t.words)
                    t.masks[(int64_t)(first + i) * t.words + w] = mask[w];
        }
    }
    if (bad)
        atomicOr(p.err, kErrPages);
}

struct AcceptParams {
    PageParams b;
    const int32_t *paths, *counts;
    int32_t *from, *to;
    int depth;
};

constexpr int kAcceptWaves = 4;

// One wave per request. A branch that is not one leaves the step not standing, so
// that no commit counts its tokens.
__global__ __launch_bounds__(64 * kAcceptWaves) void page_accept_kernel(AcceptParams a)
{
    const PageParams &p = a.b;
    const int b = blockIdx.x * kAcceptWaves + (threadIdx.x >> 6), lane = threadIdx.x & 63;
    if (b >= p.requests)
        return;
    const bool stands = p.counters[kCountState] == kStepStands;
    int first;
    bool bad = false;
    const int n = stands ? step_tokens(p, b, &first, &bad) : 0;
    const int held = p.lengths[b];
    const int count = stands ? a.counts[b] : 0;
    bad |= count < 0 || count > min(n, a.depth);
    for (int k0 = 0; k0 < a.depth; k0 += 64) {
        const int k = k0 + lane;
        int from = -1, to = -1;
        if (!bad && k < count) {
            const int64_t at = (int64_t)b * a.depth + k;
            const int c = a.paths[at], before = k ? a.paths[at - 1] : -1;
            if (c <= before || c >= n) {
                bad = true;
            } else if (c != k) {
                const int32_t *table = p.table + b * p.table_stride;
                const uint32_t x = (uint32_t)(held + c), y = (uint32_t)(held + k);
                const int32_t px = table[x / p.page_tokens], py = table[y / p.page_tokens];
                if (in_pools(p, px) && in_pools(p, py)) {
                    from = px * (int32_t)p.page_tokens + (int32_t)(x % p.page_tokens);
                    to = py * (int32_t)p.page_tokens + (int32_t)(y % p.page_tokens);
                } else {
                    bad = true;
                }
            }
        }
        if (k < a.depth) {
            a.from[(int64_t)b * a.depth + k] = from;
            a.to[(int64_t)b * a.depth + k] = to;
        }
    }
    if (!__any(bad))
        return;
    // none of its rows moves
    for (int k = lane; k < a.depth; k += 64) {
        a.from[(int64_t)b * a.depth + k] = -1;
        a.to[(int64_t)b * a.depth + k] = -1;
    }
    if (lane == 0) {
        atomicOr(p.err, kErrPages);
        p.counters[kCountState] = kStepNone;
    }
}

struct ForkParams {
    PageParams b; // in: the source of each request
    int32_t *from, *to, *rows;
};

// The first workgroup writes the words of each request and the counters; workgroup
// 1 + b the table of request b where it begins as a copy, and its part of the rows,
// which a fork has none of. Every workgroup forms the sum of the new pages over all
// requests by itself, as a step's do.
__global__ __launch_bounds__(kPageThreads) void page_fork_kernel(ForkParams f)
{
    extern __shared__ uint32_t page_off[]; // [requests + 1] new pages before each
    __shared__ uint32_t waves[kPageThreads / 64];
    const PageParams &p = f.b;
    const int tid = threadIdx.x;
    const int per = (p.requests + kPageThreads - 1) / kPageThreads;
    const int i0 = min(tid * per, p.requests), i1 = min(i0 + per, p.requests);
    const int free_count = p.counters[kCountFree];
    // the tokens that request i begins with, ~0 where it cannot; 0 without a source
    auto tokens = [&](int i) {
        const int32_t source = p.in[i];
        const uint32_t len = held_tokens(p, p.lengths, i);
        if (source < 0)
            return len == ~0u ? len : 0u;
        if (source >= p.requests || len != 0 || p.in[source] >= 0)
            return ~0u;
        return held_tokens(p, p.lengths, source);
    };
    uint32_t sum = 0;
    bool bad = false;
    for (int i = i0; i < i1; ++i) {
        const uint32_t n = tokens(i);
        bad |= n == ~0u;
        const uint32_t need = n != ~0u && n % p.page_tokens ? 1 : 0;
        page_off[i] = need;
        sum += need;
    }
    uint32_t taken;
    uint32_t at = block_offsets(sum, waves, &taken);
    for (int i = i0; i < i1; ++i) {
        const uint32_t need = page_off[i];
        page_off[i] = at;
        at += need;
    }
    if (tid == 0)
        page_off[p.requests] = taken;
    const bool had = free_count >= 0 && free_count <= p.pages && (int64_t)taken <= free_count;
    bad |= !had;
    const bool ok = !__syncthreads_or(bad);

    if (blockIdx.x == 0) {
        bool damaged = false;
        for (int i = tid; i < p.requests; i += kPageThreads) {
            const int32_t source = p.in[i];
            const uint32_t n = ok ? tokens(i) : 0;
            int32_t from = -1, to = -1, rows = 0;
            if (ok && source >= 0 && n % p.page_tokens) {
                const int32_t old = p.table[source * p.table_stride + n / p.page_tokens];
                const int32_t page = p.free_pages[free_count - 1 - (int)page_off[i]];
                if (in_pools(p, old) && in_pools(p, page)) {
                    from = old * (int32_t)p.page_tokens;
                    to = page * (int32_t)p.page_tokens;
                    rows = (int32_t)(n % p.page_tokens);
                } else {
                    damaged = true; // in the source's table or the free list
                }
            }
            p.step_lengths[i] = ok && source >= 0 ? (int32_t)n : p.lengths[i];
            p.newest[i] = -1;
            f.from[i] = from;
            f.to[i] = to;
            f.rows[i] = rows;
        }
        damaged = __syncthreads_or(damaged);
        if (tid == 0) {
            p.counters[kCountRows] = 0;
            p.counters[kCountTaken] = ok ? (int32_t)taken : 0;
            p.counters[kCountState] = ok && !damaged ? kForkStands : kStepNone;
            if (!ok || damaged)
                atomicOr(p.err, kErrPages);
        }
        return;
    }
    const int b = blockIdx.x - 1;
    for (int64_t t = (int64_t)b * kPageThreads + tid; t < p.step_rows;
         t += (int64_t)p.requests * kPageThreads) {
        p.slots[t] = -1;
        p.positions[t] = -1;
        p.row_request[t] = -1;
    }
    const int32_t source = p.in[b];
    if (!ok || source < 0)
        return;
    const uint32_t n = tokens(b), whole = n / p.page_tokens;
    const int32_t *theirs = p.table + source * p.table_stride;
    int32_t *mine = p.table + b * p.table_stride;
    for (uint32_t c = tid; c < whole; c += kPageThreads)
        mine[c] = theirs[c];
    if (tid == 0 && n % p.page_tokens) {
        const int32_t page = p.free_pages[free_count - 1 - (int)page_off[b]];
        mine[whole] = in_pools(p, page) ? page : -1;
    }
}

// A release's pages are marked, and those that the finished requests hold and the
// others do not go back, the highest first.
struct ReleaseParams {
    PageParams b; // in: finished flags
    uint8_t *gone, *kept; // [marks] a byte a page: of a finished request, of another
    uint32_t *refuse;     // set where a length or page is out of range
    int64_t marks;        // pages, to whole 32 bytes
};

// Marks request b's pages by `threads` threads from thread t on; true where it or
// one of them is out of range (a page that stays is not looked at).
template <typename Mark>
__device__ __forceinline__ bool mark_pages(const PageParams &p, int b, int t, int threads, Mark mark)
{
    const bool gone = p.in[b] != 0;
    const uint32_t len = held_tokens(p, p.lengths, b);
    if (len == ~0u)
        return true;
    bool bad = false;
    const uint32_t pages = pages_of(len, p.page_tokens);
    for (uint32_t c = t; c < pages; c += threads) {
        const int32_t page = p.table[b * p.table_stride + c];
        if (in_pools(p, page))
            mark(page, gone);
        else
            bad |= gone;
    }
    return bad;
}

// The end of a release by one workgroup: checks the free list against the marks,
// then appends the pages in descending order; count(i) and pages(i, f) are those of
// the i-th group of 32 marks from the highest on.
template <int THREADS, typename Gone, typename Bits>
__device__ __forceinline__ void give_back(const PageParams &p, bool bad, int groups,
                                          uint32_t *waves, Gone gone, Bits bits)
{
    const int tid = threadIdx.x;
    const int free_count = p.counters[kCountFree];
    bad |= free_count < 0 || free_count > p.pages;
    // a page of the free list is nobody's
    for (int i = tid; !bad && i < free_count; i += THREADS) {
        const int32_t page = p.free_pages[i];
        bad |= !in_pools(p, page) || gone(page);
    }
    const int per = (groups + THREADS - 1) / THREADS;
    const int i0 = min(tid * per, groups), i1 = min(i0 + per, groups);
    uint32_t mine = 0;
    for (int i = i0; i < i1; ++i)
        mine += __popc(bits(groups - 1 - i));
    uint32_t total;
    uint32_t at = block_offsets(mine, waves, &total);
    bad |= (int64_t)free_count + total > p.pages;
    if (__syncthreads_or(bad)) {
        if (tid == 0)
            atomicOr(p.err, kErrPages);
        return;
    }
    for (int i = i0; i < i1 && mine; ++i) {
        const int g = groups - 1 - i;
        for (uint32_t b = bits(g); b;) {
            const int top = 31 - __clz(b);
            p.free_pages[free_count + at++] = 32 * g + top;
            b &= ~(1u << top);
        }
    }
    for (int i = tid; i < p.requests; i += THREADS)
        if (p.in[i])
            p.lengths[i] = 0;
    if (tid == 0) {
        p.counters[kCountFree] = (int32_t)(free_count + total);
        p.counters[kCountState] = kStepNone;
    }
}

constexpr int kReleaseThreads = 1024;
// Pages (a bit each) and table entries of a release by one workgroup.
constexpr int kReleaseBits = 1 << 17, kReleaseEntries = 1 << 14;

// Small batches: one workgroup, the marks as bits in LDS. The requests' words are read
// at once, then a wave takes the tables of kReleaseAhead requests at a time, so that
// their loads do not wait for each other's (32 forks of 8 prompts of up to 4000 tokens,
// pages of 16: 8.0 us, 8.9 with a table after another).
constexpr int kReleaseAhead = 4;

__global__ __launch_bounds__(kReleaseThreads) void release_small_kernel(PageParams p)
{
    constexpr int kWaves = kReleaseThreads / 64;
    extern __shared__ uint32_t marks[]; // [2][groups], and [requests] pages, gone in bit 31
    __shared__ uint32_t waves[kWaves];
    const int groups = (p.pages + 31) / 32, lane = threadIdx.x & 63;
    uint32_t *const held = marks + 2 * groups;
    bool bad = false;
    for (int i = threadIdx.x; i < p.requests; i += kReleaseThreads) {
        const uint32_t len = held_tokens(p, p.lengths, i);
        bad |= len == ~0u;
        held[i] = (len == ~0u ? 0 : pages_of(len, p.page_tokens)) | (p.in[i] ? 1u << 31 : 0);
    }
    for (int i = threadIdx.x; i < 2 * groups; i += kReleaseThreads)
        marks[i] = 0;
    __syncthreads();
    auto mark = [&](int32_t page, bool gone) { // (a page that stays is not looked at)
        if (in_pools(p, page))
            atomicOr(&marks[(gone ? 0 : groups) + page / 32], 1u << (page % 32));
        else
            bad |= gone;
    };
    for (int b0 = threadIdx.x >> 6; b0 < p.requests; b0 += kReleaseAhead * kWaves) {
        uint32_t words[kReleaseAhead];
        int32_t page[kReleaseAhead];
#pragma unroll
        for (int u = 0; u < kReleaseAhead; ++u) {
            const int b = b0 + u * kWaves;
            words[u] = b < p.requests ? held[b] : 0;
            page[u] = 0;
            if (lane < (int)(words[u] & ~(1u << 31)))
                page[u] = p.table[b * p.table_stride + lane];
        }
#pragma unroll
        for (int u = 0; u < kReleaseAhead; ++u) {
            const int pages = (int)(words[u] & ~(1u << 31));
            const bool gone = words[u] >> 31;
            if (lane < pages)
                mark(page[u], gone);
            for (int c = 64 + lane; c < pages; c += 64)
                mark(p.table[(b0 + u * kWaves) * p.table_stride + c], gone);
        }
    }
    __syncthreads();
    give_back<kReleaseThreads>(
        p, bad, groups, waves, [&](int page) { return marks[page / 32] >> (page % 32) & 1; },
        [&](int g) { return marks[g] & ~marks[groups + g]; });
}

__global__ __launch_bounds__(kPageThreads) void release_clear_kernel(ReleaseParams r)
{
    const int64_t step = (int64_t)gridDim.x * kPageThreads;
    int4 *words = reinterpret_cast<int4 *>(r.gone); // (and kept behind it)
    for (int64_t i = (int64_t)blockIdx.x * kPageThreads + threadIdx.x; i < 2 * r.marks / 16;
         i += step) {
        words[i] = int4{0, 0, 0, 0};
        if (i == 0)
            *r.refuse = 0;
    }
}

// Large ones: a workgroup a request. Many requests may hold a page: they store the
// same byte, which needs no atomic (as bits, 480 forks of 16 prompts took 112 us here,
// one cache line's atomics one after another).
__global__ __launch_bounds__(kPageThreads) void release_mark_kernel(ReleaseParams r)
{
    if (mark_pages(r.b, blockIdx.x, threadIdx.x, kPageThreads,
                   [&](int page, bool gone) { (gone ? r.gone : r.kept)[page] = 1; }))
        atomicOr(r.refuse, 1u);
}

__global__ __launch_bounds__(kReleaseThreads) void release_return_kernel(ReleaseParams r)
{
    __shared__ uint32_t waves[kReleaseThreads / 64];
    const int groups = (int)(r.marks / 32);
    // 32 bytes of 0 and 1 as bits
    auto bits = [&](int g) {
        uint32_t x = 0;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int4 a = reinterpret_cast<const int4 *>(r.gone)[2 * g + h];
            const int4 k = reinterpret_cast<const int4 *>(r.kept)[2 * g + h];
            const uint32_t w[4] = {(uint32_t)(a.x & ~k.x), (uint32_t)(a.y & ~k.y),
                                   (uint32_t)(a.z & ~k.z), (uint32_t)(a.w & ~k.w)};
#pragma unroll
            for (int i = 0; i < 4; ++i) // byte j's bit 0 to bit j
                x |= ((w[i] & 0x01010101u) * 0x10204080u >> 28) << (16 * h + 4 * i);
        }
        return x;
    };
    give_back<kReleaseThreads>(r.b, *r.refuse != 0, groups, waves,
                               [&](int page) { return r.gone[page] != 0; }, bits);
}

// Layers that one launch copies in.
constexpr int kCopyLayers = 64;

struct CopyLayer {
    char *k, *v;
    uint32_t row_bytes;
};

struct CopyParams {
    CopyLayer layer[kCopyLayers];
    const int32_t *from, *to, *rows;
    int entries;
    int total; // slots of the pools
    int *err;
};

constexpr int kCopyThreads = 256;
constexpr int kCopyAhead = 8; // 16-byte pieces a lane has in flight

__device__ __forceinline__ f4 load16(const char *p)
{
    return *(gf4_cptr)p;
}

__device__ __forceinline__ void store16(char *p, f4 v)
{
    *(gf4_ptr)p = v;
}

// Entries of one list of its own: blockIdx.x the entry, y the layer and array, z a
// share of the bytes, which lie in a row.
__global__ __launch_bounds__(kCopyThreads) void copy_runs_kernel(CopyParams p)
{
    const int from = p.from[blockIdx.x], to = p.to[blockIdx.x];
    const int rows = p.rows ? p.rows[blockIdx.x] : 1;
    if (from < 0 || to < 0 || rows <= 0)
        return;
    if (rows > p.total || from > p.total - rows || to > p.total - rows) {
        if (threadIdx.x == 0)
            atomicOr(p.err, kErrPages);
        return;
    }
    const CopyLayer &y = p.layer[blockIdx.y / 2];
    char *pool = blockIdx.y % 2 ? y.v : y.k;
    const char *src = pool + (int64_t)from * y.row_bytes;
    char *dst = pool + (int64_t)to * y.row_bytes;
    const int64_t bytes = (int64_t)rows * y.row_bytes;
    constexpr int64_t kRound = 16 * kCopyThreads * kCopyAhead;
    for (int64_t c = (int64_t)blockIdx.z * kRound + 16 * threadIdx.x; c < bytes;
         c += gridDim.z * kRound) {
        f4 v[kCopyAhead];
#pragma unroll
        for (int i = 0; i < kCopyAhead; ++i)
            v[i] = load16(src + min(c + 16 * kCopyThreads * i, bytes - 16));
#pragma unroll
        for (int i = 0; i < kCopyAhead; ++i)
            if (c + 16 * kCopyThreads * i < bytes)
                store16(dst + c + 16 * kCopyThreads * i, v[i]);
    }
}

// Lists of single rows, in the order of their entries: blockIdx.x the list, a
// thread a 16-byte column of the rows. A batch of rows is read before it is
// written: no entry reads a row that an earlier one of its list writes.
__global__ __launch_bounds__(kCopyThreads) void copy_lists_kernel(CopyParams p)
{
    const CopyLayer &y = p.layer[blockIdx.y / 2];
    char *pool = blockIdx.y % 2 ? y.v : y.k;
    const int32_t *from = p.from + (int64_t)blockIdx.x * p.entries;
    const int32_t *to = p.to + (int64_t)blockIdx.x * p.entries;
    for (uint32_t c = 16 * threadIdx.x; c < y.row_bytes; c += 16 * kCopyThreads)
        for (int e0 = 0; e0 < p.entries; e0 += kCopyAhead) {
            f4 v[kCopyAhead];
            int at[kCopyAhead];
            bool bad = false;
#pragma unroll
            for (int i = 0; i < kCopyAhead; ++i) {
                const int e = min(e0 + i, p.entries - 1);
                int f = from[e];
                at[i] = e0 + i < p.entries && f >= 0 ? to[e] : -1;
                if (at[i] >= 0 && (at[i] >= p.total || f >= p.total)) {
                    bad = true;
                    at[i] = -1;
                }
                f = at[i] < 0 ? 0 : f;
                v[i] = load16(pool + (int64_t)f * y.row_bytes + c);
            }
            if (bad && threadIdx.x == 0)
                atomicOr(p.err, kErrPages);
#pragma unroll
            for (int i = 0; i < kCopyAhead; ++i)
                if (at[i] >= 0)
                    store16(pool + (int64_t)at[i] * y.row_bytes + c, v[i]);
        }
}

} // namespace pcl

namespace {

using pcl::PageParams;

// Bytes of a kind of a release's marks.
int64_t mark_bytes(const pcl_page_batch *b)
{
    return (b->pages + 31) / 32 * 32;
}

// One workgroup does as long as it has some 16 table entries a thread to look at. Calls in
// a row, one workgroup and three launches, of a release in which nobody ended and of a
// fork with its commit and release: 40 requests of 250 entries 6.2 and 8.5, 16.0 and 16.6
// us; of 32 entries 5.0 and 9.1, 13.0 and 17; at the border 64 of 250 7.6 and 9.1, 17.4 and
// 16.9, 16 of 1000 (the lives alone) 18.2 and 17.7, 8 of 1875 22 and 19.7.
bool release_is_small(const pcl_page_batch *b)
{
    return b->pages <= pcl::kReleaseBits &&
           b->table_stride <= pcl::kReleaseEntries / b->requests;
}

size_t release_bytes(const pcl_page_batch *b)
{
    return release_is_small(b) ? 0 : 2 * mark_bytes(b) + 16;
}

} // namespace

extern "C" {

int pcl_page_tree_masks(pcl_context *ctx, const pcl_page_batch *batch, const pcl_page_tree *tree)
{
    pcl::TreeStepParams t;
    const int rc = pcl::page_params(ctx, batch, &t.b);
    if (rc != PCL_OK)
        return rc;
    if (!tree || tree->words <= 0 || tree->words > pcl::kMaxTreeWords || !tree->parents ||
        !tree->positions || !tree->masks ||
        ((uintptr_t)tree->parents | (uintptr_t)tree->positions) % 4 || (uintptr_t)tree->masks % 8)
        return PCL_INVALID_SHAPE;
    t.parents = tree->parents;
    t.positions = tree->positions;
    t.masks = tree->masks;
    t.words = (int)tree->words;
    if (t.words == 1)
        pcl::page_tree_kernel<1><<<t.b.requests, 64, 0, ctx->stream>>>(t);
    else if (t.words == 2)
        pcl::page_tree_kernel<2><<<t.b.requests, 128, 0, ctx->stream>>>(t);
    else
        pcl::page_tree_kernel<8><<<t.b.requests, 512, 0, ctx->stream>>>(t);
    return pcl::page_launched("tree");
}

int pcl_page_accept(pcl_context *ctx, const pcl_page_batch *batch, const int32_t *paths,
                    const int32_t *counts, int64_t depth, int32_t *from, int32_t *to)
{
    pcl::AcceptParams a;
    const int rc = pcl::page_params(ctx, batch, &a.b);
    if (rc != PCL_OK)
        return rc;
    if (!paths || !counts || !from || !to || depth <= 0 || depth > pcl::kMaxStepRows ||
        depth > pcl::kMaxSlots / batch->requests ||
        ((uintptr_t)paths | (uintptr_t)counts | (uintptr_t)from | (uintptr_t)to) % 4)
        return PCL_INVALID_SHAPE;
    a.paths = paths;
    a.counts = counts;
    a.from = from;
    a.to = to;
    a.depth = (int)depth;
    const int groups = (a.b.requests + pcl::kAcceptWaves - 1) / pcl::kAcceptWaves;
    pcl::page_accept_kernel<<<groups, 64 * pcl::kAcceptWaves, 0, ctx->stream>>>(a);
    return pcl::page_launched("accept");
}

int pcl_page_fork(pcl_context *ctx, const pcl_page_batch *batch, const int32_t *sources,
                  int32_t *from, int32_t *to, int32_t *rows)
{
    pcl::ForkParams f;
    const int rc = pcl::page_params(ctx, batch, &f.b);
    if (rc != PCL_OK)
        return rc;
    if (!sources || !from || !to || !rows ||
        ((uintptr_t)sources | (uintptr_t)from | (uintptr_t)to | (uintptr_t)rows) % 4)
        return PCL_INVALID_SHAPE;
    f.b.in = sources;
    f.from = from;
    f.to = to;
    f.rows = rows;
    const size_t lds = ((size_t)f.b.requests + 1) * sizeof(uint32_t);
    pcl::page_fork_kernel<<<1 + f.b.requests, pcl::kPageThreads, lds, ctx->stream>>>(f);
    return pcl::page_launched("fork");
}

size_t pcl_page_release_workspace_bytes(const pcl_page_batch *batch)
{
    if (!batch || pcl::check_batch(*batch) != PCL_OK)
        return 0;
    return pcl::workspace_bytes_for(release_bytes(batch));
}

int pcl_page_release_shared(pcl_context *ctx, const pcl_page_batch *batch, const int32_t *finished)
{
    pcl::ReleaseParams r;
    int rc = pcl::page_params(ctx, batch, &r.b);
    if (rc != PCL_OK)
        return rc;
    if (!finished || (uintptr_t)finished % 4)
        return PCL_INVALID_SHAPE;
    r.b.in = finished;
    if (release_is_small(batch)) {
        const size_t lds =
            (2 * (size_t)((batch->pages + 31) / 32) + batch->requests) * sizeof(uint32_t);
        pcl::release_small_kernel<<<1, pcl::kReleaseThreads, lds, ctx->stream>>>(r.b);
        return pcl::page_launched("shared release");
    }
    float *body = nullptr;
    rc = pcl::workspace_body(ctx, release_bytes(batch), &body);
    if (rc != PCL_OK)
        return rc;
    r.marks = mark_bytes(batch);
    r.gone = reinterpret_cast<uint8_t *>(body);
    r.kept = r.gone + r.marks;
    r.refuse = reinterpret_cast<uint32_t *>(r.kept + r.marks);
    const int groups = (int)std::min<int64_t>(
        (r.marks / 8 + pcl::kPageThreads - 1) / pcl::kPageThreads, 1024);
    pcl::release_clear_kernel<<<groups, pcl::kPageThreads, 0, ctx->stream>>>(r);
    pcl::release_mark_kernel<<<r.b.requests, pcl::kPageThreads, 0, ctx->stream>>>(r);
    pcl::release_return_kernel<<<1, pcl::kReleaseThreads, 0, ctx->stream>>>(r);
    return pcl::page_launched("shared release");
}

int pcl_paged_copy(pcl_context *ctx, const pcl_page_pools *pools, int64_t layers,
                   const int32_t *from, const int32_t *to, const int32_t *rows, int64_t lists,
                   int64_t entries)
{
    if (!ctx || !pools || layers < 0 || layers > 4096 || lists < 0 || entries < 0 ||
        lists > pcl::kMaxStepRows || entries > pcl::kMaxStepRows || (rows && entries > 1))
        return PCL_INVALID_SHAPE;
    for (int64_t i = 0; i < layers; ++i)
        if (!pcl::valid_pools(pools[i]) || pools[i].pages != pools[0].pages ||
            pools[i].page_tokens != pools[0].page_tokens)
            return PCL_INVALID_SHAPE;
    if (layers == 0 || lists == 0 || entries == 0)
        return PCL_OK;
    if (!from || !to || ((uintptr_t)from | (uintptr_t)to | (uintptr_t)rows) % 4 ||
        entries > pcl::kMaxSlots / lists)
        return PCL_INVALID_SHAPE;
    (void)hipSetDevice(ctx->device);
    pcl::CopyParams p;
    p.from = from;
    p.to = to;
    p.rows = rows;
    p.entries = (int)entries;
    p.total = (int)(pools[0].pages * pools[0].page_tokens);
    p.err = ctx->err;
    for (int64_t l0 = 0; l0 < layers; l0 += pcl::kCopyLayers) {
        const int n = (int)std::min<int64_t>(layers - l0, pcl::kCopyLayers);
        int64_t widest = 0;
        for (int i = 0; i < n; ++i) {
            const pcl_page_pools &s = pools[l0 + i];
            const int64_t bytes = s.kvheads * s.dim * (s.type == PCL_CACHE_F32 ? 4 : 2);
            p.layer[i] = {static_cast<char *>(s.k), static_cast<char *>(s.v), (uint32_t)bytes};
            widest = std::max(widest, bytes);
        }
        if (entries == 1) {
            // shares of a page's bytes, as many as an entry may have rounds
            constexpr int64_t kRound = 16 * pcl::kCopyThreads * pcl::kCopyAhead;
            const int64_t most = rows ? widest * pools[0].page_tokens : widest;
            const dim3 grid((unsigned)lists, 2 * n,
                            (unsigned)std::min<int64_t>((most + kRound - 1) / kRound, 16));
            pcl::copy_runs_kernel<<<grid, pcl::kCopyThreads, 0, ctx->stream>>>(p);
        } else {
            const dim3 grid((unsigned)lists, 2 * n);
            pcl::copy_lists_kernel<<<grid, pcl::kCopyThreads, 0, ctx->stream>>>(p);
        }
    }
    return pcl::page_launched("copy");
}

} // extern "C"
