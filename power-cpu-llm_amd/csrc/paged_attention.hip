// Attention of one new token of every request over a paged KV cache: checks,
// workspace and launches, and the ordered merge of the chunk partials
// (paged_kv.hpp has the mathematics and the chunk kernel).
#include "context.hpp"
#include "launch.hpp"
#include "paged.hpp"
#include "paged_combine.hpp"
#include "paged_params.hpp"

#include <algorithm>
#include <cmath>
#include <cstdio>

namespace pcl {

// Requests of one chunk are written already.
template <int BATCH>
__global__ __launch_bounds__(kCombineMost) void paged_combine_kernel(PagedParams p, CombineShape c)
{
    const int4 req = p.ws_req[blockIdx.x]; // (one load; all that a request's lanes need)
    if (req.y <= 1)
        return;
    const RowParts r = {(uint32_t)req.x, req.z, req.z + req.y, req.z, 0};
    combine_row<BATCH>(p, c, r, blockIdx.y * c.heads, 4 * c.lanes * blockIdx.z,
                       [&](int h, int d, const Merged4 &t) {
                           write_merged(p, t,
                                        p.out + req.w * p.o_stride + (int64_t)h * p.dim + d);
                       });
}

static hipError_t launch_paged_combine(const PagedParams &p, int64_t chunks, hipStream_t stream)
{
    const CombineShape c = combine_shape(p, p.requests, chunks);
    const dim3 grid = combine_grid(p, c, (unsigned)p.requests);
    const int threads = c.lanes * c.spans * c.heads;
    if (c.spans >= 16)
        paged_combine_kernel<16><<<grid, threads, 0, stream>>>(p, c);
    else
        paged_combine_kernel<8><<<grid, threads, 0, stream>>>(p, c);
    return hipGetLastError();
}

// Chunks that one request may have. (A window is any positive int64_t: it is
// held to the longest request before anything is added to it.)
static int64_t most_chunks(const pcl_paged_desc &d)
{
    const int64_t all = (d.max_length + kChunk - 1) / kChunk;
    const int64_t window = std::min(d.window, d.max_length);
    return window ? std::min(all, (window + kChunk - 2) / kChunk + 1) : all;
}

static int check_paged(const pcl_paged_desc &d)
{
    const pcl_page_pools &s = d.pools;
    if (!valid_pools(s) || d.qheads <= 0 || d.qheads % s.kvheads != 0 || d.qheads > 4096 ||
        d.requests < 0 || d.requests > kMaxRequests || d.window < 0)
        return PCL_INVALID_SHAPE;
    if (!(d.softcap >= 0.0f) || !std::isfinite(d.softcap) || !std::isfinite(d.q_scale) ||
        (d.softcap > 0.0f && (!std::isnormal(d.softcap) || !std::isnormal(1.0f / d.softcap))))
        return PCL_INVALID_PARAMETER;
    if (d.requests == 0)
        return PCL_OK;
    if (!d.q || !d.out || !d.table || !d.lengths || d.table_stride <= 0 ||
        d.table_stride > kMaxSlots || d.max_length <= 0 || d.max_length > kMaxSlots - kChunk ||
        d.max_length > d.table_stride * s.page_tokens || d.q_rows <= 0 ||
        d.q_rows > kMaxStepRows || d.q_stride < d.qheads * s.dim || d.q_stride % 4 != 0 ||
        d.o_stride < d.qheads * s.dim || d.o_stride % 4 != 0 ||
        (!d.rows && d.q_rows < d.requests))
        return PCL_INVALID_SHAPE;
    if (((uintptr_t)d.q | (uintptr_t)d.out) % 16 ||
        ((uintptr_t)d.table | (uintptr_t)d.lengths | (uintptr_t)d.rows) % 4)
        return PCL_INVALID_SHAPE;
    // item indices of the whole batch stay below 2^31
    if (most_chunks(d) > kMaxSlots / (d.requests * d.qheads))
        return PCL_INVALID_SHAPE;
    return PCL_OK;
}

// Workspace bytes: four words of every request, then their chunk partials at the
// requests' longest (none where no request can have two chunks).
static size_t paged_bytes(const pcl_paged_desc &d)
{
    if (d.requests == 0)
        return 0;
    const int64_t each = most_chunks(d);
    const size_t parts = each > 1 ? (size_t)(d.requests * each) * d.qheads : 0;
    return d.requests * sizeof(int4) + parts * (d.pools.dim + 2) * sizeof(float);
}

} // namespace pcl

extern "C" {

size_t pcl_paged_workspace_bytes(const pcl_paged_desc *desc)
{
    if (!desc || pcl::check_paged(*desc) != PCL_OK)
        return 0;
    return pcl::workspace_bytes_for(pcl::paged_bytes(*desc));
}

int pcl_paged_attention(pcl_context *ctx, const pcl_paged_desc *desc)
{
    if (!ctx || !desc)
        return PCL_INVALID_SHAPE;
    const pcl_paged_desc &d = *desc;
    int rc = pcl::check_paged(d);
    if (rc != PCL_OK || d.requests == 0)
        return rc;
    (void)hipSetDevice(ctx->device);
    float *body = nullptr;
    rc = pcl::workspace_body(ctx, pcl::paged_bytes(d), &body);
    if (rc != PCL_OK)
        return rc;
    const pcl_page_pools &s = d.pools;
    const int64_t each = pcl::most_chunks(d);
    const int64_t group = d.qheads / s.kvheads;
    pcl::PagedParams p;
    p.q = d.q;
    p.q_stride = d.q_stride;
    p.k = s.k;
    p.v = s.v;
    p.table = d.table;
    p.lengths = d.lengths;
    p.rows = d.rows;
    p.table_stride = d.table_stride;
    p.row_stride = s.kvheads * s.dim;
    p.out = d.out;
    p.o_stride = d.o_stride;
    const int64_t parts = each > 1 ? d.requests * each * d.qheads : 0;
    p.ws_req = reinterpret_cast<int4 *>(body);
    p.ws_o = body + 4 * d.requests;
    p.ws_ml = p.ws_o + parts * s.dim;
    p.err = ctx->err;
    p.requests = (int)d.requests;
    p.q_rows = (int)d.q_rows;
    p.max_length = (int)d.max_length;
    p.window = (int)std::min(d.window, d.max_length);
    p.pages = (int)s.pages;
    p.page_tokens = (uint32_t)s.page_tokens;
    p.qheads = (int)d.qheads;
    p.kvheads = (int)s.kvheads;
    p.group = (int)group;
    p.units = 1;
    p.dim = (int)s.dim;
    p.q_scale = d.q_scale;
    p.softcap = d.softcap;
    p.inv_softcap = d.softcap > 0.0f ? 1.0f / d.softcap : 0.0f;
    const int64_t chunks = d.requests * each;
    const bool bf16 = s.type == PCL_CACHE_BF16;
    int span = pcl::open_timed_span(ctx, 0);
    hipError_t e = p.dim <= 64    ? pcl::launch_paged_kv<64>(p, bf16, chunks, ctx->stream)
                   : p.dim <= 128 ? pcl::launch_paged_kv<128>(p, bf16, chunks, ctx->stream)
                   : p.dim <= 256 ? pcl::launch_paged_kv<256>(p, bf16, chunks, ctx->stream)
                                  : pcl::launch_paged_kv<512>(p, bf16, chunks, ctx->stream);
    pcl::close_timed_span(ctx, span);
    if (e == hipSuccess && each > 1) {
        span = pcl::open_timed_span(ctx, 1);
        e = pcl::launch_paged_combine(p, each, ctx->stream);
        pcl::close_timed_span(ctx, span);
    }
    if (e != hipSuccess) {
        std::fprintf(stderr, "pcl_paged_attention: launch: %s\n", hipGetErrorString(e));
        return PCL_NON_FINITE_VALUE;
    }
    return PCL_OK;
}

} // extern "C"
