// What the paged attention's chunk kernels and its combine share: the launch's
// parameters and the keys of a request.
#pragma once

#include "attention_device.hpp"
#include "item_claims.hpp"

#include <cstdint>

namespace pcl {

struct PagedParams {
    const float *q;
    int64_t q_stride;
    const void *k, *v;
    const int32_t *table, *lengths, *rows;
    int64_t table_stride;
    int64_t row_stride; // values between consecutive slots (kvheads * dim)
    float *out;
    int64_t o_stride;
    float *ws_o, *ws_ml; // [chunk][qheads][dim], [chunk][qheads][2]
    int4 *ws_req;        // [requests] for the combine: chunks before it, its chunks,
                         // its first chunk, its row (a tree launch: its first row, its
                         // chunks, its held tokens, its new ones)
    int *err;
    int requests, q_rows, max_length, window, pages;
    uint32_t page_tokens;
    int qheads, kvheads, group, units, dim;
    float q_scale, softcap, inv_softcap;
};

// The keys a request's newest token attends, [first, len), none for a request
// without a row or keys.
struct RequestKeys {
    int row, first, len;
};

__device__ __forceinline__ int first_key(const PagedParams &p, int len)
{
    return p.window && len > p.window ? len - p.window : 0;
}

__device__ __forceinline__ RequestKeys request_keys(const PagedParams &p, int i, bool *bad)
{
    RequestKeys r;
    r.row = p.rows ? p.rows[i] : i;
    r.len = p.lengths[i];
    if (r.row < 0 || r.len <= 0) {
        r.len = 0;
    } else if (r.row >= p.q_rows || r.len > p.max_length) {
        *bad = true;
        r.len = 0;
    }
    r.first = first_key(p, r.len);
    return r;
}

__device__ __forceinline__ int request_chunks(const RequestKeys &r)
{
    return r.len ? (r.len - 1) / kChunk + 1 - r.first / kChunk : 0;
}

// Division of a value below 2^31 by a divisor of the launch, at most 2^12: with s =
// ceil(log2 d) - 1 and mul = ceil(2^(32 + s) / d), (x mul) >> (32 + s) is exact as
// mul d - 2^(32 + s) < d <= 2^(s + 1) and x below 2^31 (1: x itself).
struct Divisor {
    uint32_t mul, shift; // mul 0: by 1
};

inline Divisor divisor(uint32_t d)
{
    if (d == 1)
        return {0, 0};
    uint32_t s = 0;
    while ((2u << s) < d)
        ++s;
    return {(uint32_t)((((uint64_t)1 << (32 + s)) + d - 1) / d), s};
}

__device__ __forceinline__ uint32_t divided(uint32_t x, const Divisor &d)
{
    return d.mul ? __umulhi(x, d.mul) >> d.shift : x;
}

// An item of a launch of many rows: the chunks of a span, or one, of one request, KV
// head and unit of query rows.
struct PlanItem {
    int b, kh;
    int row, held, n;     // as TreeItem's
    int first_row, nrows; // of the unit
    int from, to;         // the first and the last key that any row may attend
    int chunk, chunks;    // first one, and how many (0: no key, nothing to do)
    int slot;             // partial (of a row's) of the last chunk, the result's
    int only;             // the chunks are all of the request's
    int spare[3];
};

struct PlanHead {
    int items, uneven; // uneven: some have several chunks
    int taken[kItemParts]; // items of each part that are taken
    int spare[6];
};

static_assert(sizeof(PlanItem) == 64 && sizeof(PlanHead) == 64, "whole scalar loads");

// Of a launch over every new token of a step (lengths: with the step's tokens).
struct TreeParams : PagedParams {
    const int32_t *held, *newest;  // [requests] tokens before the step, row of the last one
    const uint64_t *masks;         // [q_rows][mask_words], or null: a chain
    const int32_t *positions;      // [q_rows], with masks and a window
    int mask_words, max_new;
    int row_chunks; // partials of a row: chunks that one request may have
    // of a launch of many rows, written by its plan kernel: the items behind their
    // count, and of every request the first chunk that is an item of its own, those
    // before it being of whole spans (null: every chunk is an item)
    PlanHead *plan;
    int32_t *split; // [requests]
    int max_items;
    Divisor by_group, by_kvheads, by_page_tokens;
};

// A request's keys [0, len), the tokens that it held before the step, and the
// step's row of its first new token; none (held = len) for a request without one.
struct TreeKeys {
    int row, held, len;
};

// The first key that any new token attends: their positions start at the held
// tokens' count.
__device__ __forceinline__ int first_tree_key(const TreeParams &p, int position)
{
    return p.window && position >= p.window ? position - p.window + 1 : 0;
}

__device__ __forceinline__ TreeKeys tree_keys(const TreeParams &p, int i, bool *bad)
{
    TreeKeys r;
    const int last = p.newest[i];
    r.held = p.held[i];
    r.len = p.lengths[i];
    const int64_t n = (int64_t)r.len - r.held;
    r.row = (int)(last - n + 1);
    if (last < 0 || n == 0) {
        r.held = r.len = 0;
    } else if (r.held < 0 || n < 0 || r.len > p.max_length || n > p.max_new ||
               last - n + 1 < 0 || last >= p.q_rows || (p.masks && n > 64 * p.mask_words)) {
        *bad = true;
        r.held = r.len = 0;
    }
    return r;
}

__device__ __forceinline__ int tree_chunks(const TreeParams &p, const TreeKeys &r)
{
    return r.len > r.held ? (r.len - 1) / kChunk + 1 - first_tree_key(p, r.held) / kChunk : 0;
}

// The kernel of a tree launch: units of `rows` query rows, 4 or 8 (paged_kv.hpp, with
// `buffers` in a wave's ring) or 16, 32 or 48 (paged_rows.hpp, `buffers` 0).
struct TreeVariant {
    int rows, buffers;
};

// Which one a launch of at most `chunks` chunks takes on a device of `cus` CUs; `rows`:
// query rows of a KV head that one request has at most.
TreeVariant tree_variant(int64_t dim, int64_t chunks, int64_t kvheads, int64_t rows, int64_t cus);

// The chunk kernel of a launch of at most `chunks` chunks, at padded head dim
// DK (64, 128, 256 or 512, a source file each).
template <int DK>
hipError_t launch_paged_kv(const PagedParams &p, bool bf16, int64_t chunks, hipStream_t stream);
template <int DK>
hipError_t launch_paged_tree(const TreeParams &p, const TreeVariant &v, bool bf16, int64_t rows,
                             int64_t chunks, hipStream_t stream);
template <int DK>
hipError_t launch_paged_rows(const TreeParams &p, int unit, bool bf16, int64_t rows,
                             int64_t chunks, hipStream_t stream);

} // namespace pcl
