// What the kernels of a batch's page bookkeeping share: its arrays and their ranges.
#pragma once

#include "context.hpp"
#include "paged.hpp"

namespace pcl {

constexpr int kPageThreads = 256;

enum { kCountFree, kCountRows, kCountTaken, kCountState, kCounters };
enum { kStepNone, kStepStands, kForkStands };

struct PageParams {
    int32_t *lengths, *table, *free_pages, *counters, *step_lengths, *newest;
    int32_t *slots, *positions, *row_request;
    const int32_t *in; // new tokens, kept tokens, finished flags or sources per request
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

__device__ __forceinline__ bool in_pools(const PageParams &p, int32_t page)
{
    return page >= 0 && page < p.pages;
}

// Checks of a batch's fields alone; its parameters on the context's device; the
// status of the launch behind them.
int check_batch(const pcl_page_batch &b);
int page_params(pcl_context *ctx, const pcl_page_batch *b, PageParams *p);
int page_launched(const char *what);

} // namespace pcl
