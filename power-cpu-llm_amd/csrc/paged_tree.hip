// Attention of every new token of a step over a paged KV cache: checks, workspace
// and launches, and the ordered merge of the chunk partials (paged_kv.hpp has the
// mathematics and the chunk kernel).
#include "context.hpp"
#include "launch.hpp"
#include "paged.hpp"
#include "paged_combine.hpp"
#include "paged_params.hpp"

#include <algorithm>
#include <cmath>
#include <cstdio>

namespace pcl {

constexpr int64_t kMaxMaskWords = 8;
// Workgroups of the combine's grid; each goes on to rows past them. (Prompt parts of
// 4 x 512 tokens, 16 heads, behind up to 8192 keys: 95 us with a workgroup for every
// row and head, 111 us with 2048 workgroups for 16 rows each.)
constexpr unsigned kCombineGroups = 65536;

// Rows of requests of one chunk are written already, and so is nothing of a row
// that attends no key. A chain's token has partials of its own chunks alone.
template <int BATCH>
__global__ __launch_bounds__(kCombineMost) void tree_combine_kernel(TreeParams p, CombineShape c)
{
    const int b = blockIdx.x % p.requests;
    const int4 req = p.ws_req[b];
    if (req.y <= 1)
        return;
    const int row0 = req.x, held = req.z, n = req.w;
    const int first = first_tree_key(p, held) / kChunk, end = first + req.y;
    const int split = p.plan ? p.split[b] : 0;
    if (split == end && (end - 1) / kSpanChunks == first / kSpanChunks)
        return; // one span: written already
    for (int i = blockIdx.x / p.requests; i < n; i += gridDim.x / p.requests) {
        int c0 = first, c1 = c0 + req.y;
        if (!p.masks) {
            c0 = first_tree_key(p, held + i) / kChunk;
            c1 = (held + i) / kChunk + 1;
        }
        const RowParts r = {(uint32_t)((row0 + i) * p.row_chunks), c0, c1, first, split};
        combine_row<BATCH>(p, c, r, blockIdx.y * c.heads, 4 * c.lanes * blockIdx.z,
                           [&](int h, int d, const Merged4 &t) {
                               if (t.L != 0.f)
                                   write_merged(p, t,
                                                p.out + (row0 + i) * p.o_stride +
                                                    (int64_t)h * p.dim + d);
                           });
    }
}

// `rows`: of the launch, at most.
static hipError_t launch_tree_combine(const TreeParams &p, int64_t rows, int64_t chunks,
                                      hipStream_t stream)
{
    const CombineShape c = combine_shape(p, rows, chunks);
    dim3 grid = combine_grid(p, c, (unsigned)p.requests);
    const unsigned each = grid.x * grid.y * grid.z;
    grid.x *= std::max(1u, std::min((unsigned)p.max_new, kCombineGroups / each));
    const int threads = c.lanes * c.spans * c.heads;
    if (c.spans >= 16)
        tree_combine_kernel<16><<<grid, threads, 0, stream>>>(p, c);
    else
        tree_combine_kernel<8><<<grid, threads, 0, stream>>>(p, c);
    return hipGetLastError();
}

// Chunks that one request may have: a window's keys begin that far before its
// first new token.
static int64_t most_chunks(const pcl_paged_tree_desc &d)
{
    const int64_t all = (d.max_length + kChunk - 1) / kChunk;
    if (!d.window)
        return all;
    const int64_t keys = std::min(d.window, d.max_length) + std::min(d.max_new, d.max_length) - 1;
    return std::min(all, (keys + kChunk - 2) / kChunk + 1);
}

// New tokens of the whole launch, at most.
static int64_t most_rows(const pcl_paged_tree_desc &d)
{
    return std::min(d.q_rows, d.requests * std::min(d.max_new, d.max_length));
}

// Query rows of a KV head and request up to which no launch is one of many rows.
constexpr int64_t kFewRows = 8;

// Units of 4 or 8 rows where a request has no more, or where they leave at most an item
// per CU, each with a CU to itself (one request of 8 new tokens behind 1000 keys, f32: 21
// us and 26 in units of sixteen rows at 16 x 8 x 256 heads, 29 and 54 at 16 x 2 x 512, 21
// and 27 at 32 x 8 x 128, both 23 at 16 x 4 x 64; of 40 behind 500: 26 and 45, 36 and 57,
// both 43, 31 and 37; padded, the 8 behind 1000: 23 and 35 at 10 x 2 x 80, 22 and 27 at 16 x
// 8 x 144, 35 and 56 at 16 x 2 x 400, but 25 and 24 at 16 x 4 x 48 and the same at 16 and 32
// dims, of 40 behind 500 33 and 29: not below 64). Two buffers of the ring where an item of
// a whole head dim has a CU to itself (PagedCfg has both sides). Otherwise the fewest units that hold a request's rows, and the smallest
// such units: no matrix instruction runs on rows that none has (64 trees of 16 at 32 x 8 x
// 128, 64 rows in two units of 32: 577 us; as 48 and 16: 759 us). The largest unit is what
// the LDS of a CU holds beside the rings (512) and what its registers do (64 rows at head
// dim 128 spilled 43 to 157 of them: prompt parts 2290 us, 2146 with 48; trees of 12 at 32
// x 8 x 128, f32, 513 and 385 us). Units of 32 instead of 48 at head dim 256, with two
// buffers: prompt parts 2250 us (2064).
TreeVariant tree_variant(int64_t dim, int64_t chunks, int64_t kvheads, int64_t rows, int64_t cus)
{
    const bool whole = dim == 64 || dim == 128 || dim == 256 || dim == 512; // not padded
    for (const int unit : {4, (int)kFewRows}) {
        const bool few = chunks * kvheads * ((rows + unit - 1) / unit) <= cus;
        if (rows <= unit || (few && dim >= 64))
            return {unit, few && whole ? 2 : 1};
    }
    const int64_t most = dim > 256 ? 32 : 48;
    const int64_t units = (rows + most - 1) / most, unit = (rows + units - 1) / units;
    return {unit > 32 ? 48 : unit > 16 ? 32 : 16, 0};
}

static int check_tree(const pcl_paged_tree_desc &d)
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
    if (!d.q || !d.out || !d.table || !d.lengths || !d.step_lengths || !d.newest ||
        d.table_stride <= 0 || d.table_stride > kMaxSlots || d.max_length <= 0 ||
        d.max_length > kMaxSlots - kChunk || d.max_length > d.table_stride * s.page_tokens ||
        d.max_new <= 0 || d.max_new > kMaxStepRows || d.q_rows <= 0 ||
        d.q_rows > kMaxStepRows || d.q_stride < d.qheads * s.dim || d.q_stride % 4 != 0 ||
        d.o_stride < d.qheads * s.dim || d.o_stride % 4 != 0)
        return PCL_INVALID_SHAPE;
    if (d.masks ? d.mask_words <= 0 || d.mask_words > kMaxMaskWords || (d.window && !d.positions)
                : d.mask_words != 0 || d.positions != nullptr)
        return PCL_INVALID_SHAPE;
    if (((uintptr_t)d.q | (uintptr_t)d.out) % 16 || (uintptr_t)d.masks % 8 ||
        ((uintptr_t)d.table | (uintptr_t)d.lengths | (uintptr_t)d.step_lengths |
         (uintptr_t)d.newest | (uintptr_t)d.positions) %
            4)
        return PCL_INVALID_SHAPE;
    // item and partial indices of the whole batch stay below 2^31 (an item has a
    // row at least, or ends a request's)
    if (most_chunks(d) > kMaxSlots / ((d.q_rows + d.requests) * d.qheads))
        return PCL_INVALID_SHAPE;
    return PCL_OK;
}

// Items of a launch of many rows, at most (a unit has sixteen rows at least, and every
// request may end in part of one); 0 where no launch of the shape is one on any device.
static int64_t most_items(const pcl_paged_tree_desc &d)
{
    const int64_t group = d.qheads / d.pools.kvheads;
    if (std::min(d.max_new, d.max_length) * group <= kFewRows)
        return 0;
    return most_chunks(d) * d.pools.kvheads * (most_rows(d) * group / 16 + d.requests);
}

static size_t split_bytes(const pcl_paged_tree_desc &d) // (whole 16 bytes)
{
    return (size_t)((d.requests + 3) / 4) * 16;
}

// Workspace bytes: the plan, four words of every request, then the rows' chunk
// partials at the requests' longest (none where no request can have two chunks).
static size_t tree_bytes(const pcl_paged_tree_desc &d)
{
    if (d.requests == 0)
        return 0;
    const int64_t each = most_chunks(d);
    const size_t parts = each > 1 ? (size_t)(d.q_rows * each) * d.qheads : 0;
    const int64_t items = most_items(d);
    return (items ? sizeof(PlanHead) + items * sizeof(PlanItem) + split_bytes(d) : 0) +
           d.requests * sizeof(int4) + parts * (d.pools.dim + 2) * sizeof(float);
}

} // namespace pcl

extern "C" {

size_t pcl_paged_tree_workspace_bytes(const pcl_paged_tree_desc *desc)
{
    if (!desc || pcl::check_tree(*desc) != PCL_OK)
        return 0;
    return pcl::workspace_bytes_for(pcl::tree_bytes(*desc));
}

int pcl_paged_tree_attention(pcl_context *ctx, const pcl_paged_tree_desc *desc)
{
    if (!ctx || !desc)
        return PCL_INVALID_SHAPE;
    const pcl_paged_tree_desc &d = *desc;
    int rc = pcl::check_tree(d);
    if (rc != PCL_OK || d.requests == 0)
        return rc;
    (void)hipSetDevice(ctx->device);
    float *body = nullptr;
    rc = pcl::workspace_body(ctx, pcl::tree_bytes(d), &body);
    if (rc != PCL_OK)
        return rc;
    const pcl_page_pools &s = d.pools;
    const int64_t each = pcl::most_chunks(d);
    const int64_t parts = each > 1 ? d.q_rows * each * d.qheads : 0;
    pcl::TreeParams p;
    p.q = d.q;
    p.q_stride = d.q_stride;
    p.k = s.k;
    p.v = s.v;
    p.table = d.table;
    p.lengths = d.step_lengths;
    p.rows = nullptr;
    p.table_stride = d.table_stride;
    p.row_stride = s.kvheads * s.dim;
    p.out = d.out;
    p.o_stride = d.o_stride;
    const int64_t items = pcl::most_items(d);
    p.max_items = (int)items;
    const int64_t rows = std::min(d.max_new, d.max_length) * (d.qheads / s.kvheads);
    const int64_t chunks = d.requests * each;
    const pcl::TreeVariant v =
        pcl::tree_variant(s.dim, chunks, s.kvheads, rows, pcl::device_cus());
    const bool many = !v.buffers;
    p.plan = many ? reinterpret_cast<pcl::PlanHead *>(body) : nullptr;
    p.split = many ? reinterpret_cast<int32_t *>(body + 16 * (1 + items)) : nullptr;
    body += items ? 16 * (1 + items) + pcl::split_bytes(d) / sizeof(float) : 0;
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
    p.group = (int)(d.qheads / s.kvheads);
    p.units = 1;
    p.dim = (int)s.dim;
    p.q_scale = d.q_scale;
    p.softcap = d.softcap;
    p.inv_softcap = d.softcap > 0.0f ? 1.0f / d.softcap : 0.0f;
    p.held = d.lengths;
    p.newest = d.newest;
    p.masks = d.masks;
    p.positions = d.positions;
    p.mask_words = (int)d.mask_words;
    p.max_new = (int)std::min(d.max_new, d.max_length);
    p.row_chunks = (int)each;
    p.by_group = pcl::divisor((uint32_t)p.group);
    p.by_kvheads = pcl::divisor((uint32_t)p.kvheads);
    p.by_page_tokens = pcl::divisor(p.page_tokens);
    const bool bf16 = s.type == PCL_CACHE_BF16;
    int span = pcl::open_timed_span(ctx, 0);
    const auto launch = p.dim <= 64    ? pcl::launch_paged_tree<64>
                        : p.dim <= 128 ? pcl::launch_paged_tree<128>
                        : p.dim <= 256 ? pcl::launch_paged_tree<256>
                                       : pcl::launch_paged_tree<512>;
    hipError_t e = launch(p, v, bf16, rows, chunks, ctx->stream);
    pcl::close_timed_span(ctx, span);
    if (e == hipSuccess && each > 1) {
        span = pcl::open_timed_span(ctx, 1);
        e = pcl::launch_tree_combine(p, pcl::most_rows(d), each, ctx->stream);
        pcl::close_timed_span(ctx, span);
    }
    if (e != hipSuccess) {
        std::fprintf(stderr, "pcl_paged_tree_attention: launch: %s\n", hipGetErrorString(e));
        return PCL_NON_FINITE_VALUE;
    }
    return PCL_OK;
}

} // extern "C"
