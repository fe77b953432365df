// Attention of one new token of every request over a paged KV cache: checks,
// workspace and launches, and the ordered merge of the chunk partials
// (paged_kv.hpp has the mathematics and the chunk kernel).
#include "context.hpp"
#include "launch.hpp"
#include "paged.hpp"
#include "paged_params.hpp"

#include <algorithm>
#include <cmath>
#include <cstdio>

namespace pcl {

// The ordered merge of a request's chunk partials. LANES lanes hold four dims
// each of one query head; SPANS such groups merge a span of 16 chunks each,
// ascending from (-inf, 0, 0), in batches of BATCH loads, and the first group
// folds the spans in ascending order. Requests of one chunk are written already.
constexpr int kCombineMost = 256; // threads of a workgroup, at most

struct CombineShape {
    int lanes, spans, heads; // powers of two; heads: query heads of a workgroup
};

template <int BATCH>
__global__ __launch_bounds__(kCombineMost) void paged_combine_kernel(PagedParams p, CombineShape c)
{
    __shared__ f4 so[kCombineMost];
    __shared__ float sm[kCombineMost], sl[kCombineMost];
    const int4 req = p.ws_req[blockIdx.x]; // (one load; all that a request's lanes need)
    if (req.y <= 1)
        return;
    const uint32_t base = (uint32_t)req.x;
    const int c0 = req.z, c1 = c0 + req.y; // the request's chunks
    const int s0 = c0 / kSpanChunks, s1 = (c1 - 1) / kSpanChunks + 1;
    const int tid = threadIdx.x;
    const int q = tid % c.lanes, gi = tid / c.lanes % c.spans;
    const int h = blockIdx.y * c.heads + tid / (c.lanes * c.spans);
    const int d = 4 * (c.lanes * blockIdx.z + q);
    const bool in = h < p.qheads && d < p.dim;
    const int64_t row = in ? h : 0;
    const int at = in ? d : 0;
    Merged4 t = {kNegInf, 0.f, f4{0.f, 0.f, 0.f, 0.f}};
    for (int r0 = s0; r0 < s1; r0 += c.spans) {
        Merged4 s = {kNegInf, 0.f, f4{0.f, 0.f, 0.f, 0.f}};
        if (r0 + gi < s1) {
            const int e = min((r0 + gi + 1) * kSpanChunks, c1);
            for (int a = max((r0 + gi) * kSpanChunks, c0); a < e; a += BATCH) {
                f2 ml[BATCH];
                f4 ov[BATCH];
#pragma unroll
                for (int i = 0; i < BATCH; ++i) {
                    const int64_t part =
                        (int64_t)(base + (uint32_t)(min(a + i, e - 1) - c0)) * p.qheads + row;
                    ml[i] = ldg2(p.ws_ml + 2 * part);
                    ov[i] = ldg4(p.ws_o + part * p.dim + at);
                }
#pragma unroll
                for (int i = 0; i < BATCH; ++i) {
                    // chunks past the span merge as empty parts (no-ops)
                    const bool here = a + i < e;
                    merge_into4(s, here ? ml[i].x : kNegInf, here ? ml[i].y : 0.f,
                                here ? ov[i] : f4{0.f, 0.f, 0.f, 0.f});
                }
            }
        }
        if (c.spans == 1) {
            merge_into4(t, s.M, s.L, s.acc);
            continue;
        }
        so[tid] = s.acc;
        sm[tid] = s.M;
        sl[tid] = s.L;
        __syncthreads();
        if (gi == 0)
            for (int i = 0; i < min(s1 - r0, c.spans); ++i)
                merge_into4(t, sm[tid + i * c.lanes], sl[tid + i * c.lanes],
                            so[tid + i * c.lanes]);
        __syncthreads();
    }
    if (gi != 0 || !in)
        return;
    f4 v;
    bool nonfinite = false;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        v[j] = t.acc[j] / t.L;
        nonfinite |= !is_finite(v[j]);
    }
    stg4(p.out + req.w * p.o_stride + (int64_t)h * p.dim + d, v);
    if (nonfinite)
        atomicOr(p.err, kErrOutput);
}

// Groups of the combine: as many spans at once as some four thousand waves
// allow (one long request: 32, each a round trip or two; 64 requests of 16
// heads of 256 dims: 4), the fewer the wider. In groups of 8 lanes and 32 spans
// throughout, 256 requests of up to 2048 keys took 48 us here (5.6 now), 64 of up to
// 8192 keys 27 us (5.6). Batches of 16 loads from 4 spans on were 1 to 3 us slower
// (146 registers against 114), 2048 or 8192 waves within 1 us.
static hipError_t launch_paged_combine(const PagedParams &p, int64_t chunks, hipStream_t stream)
{
    auto pow2_to = [](int64_t n, int most) { // the least power of two >= n, at most `most`
        int x = 1;
        while (x < n && x < most)
            x *= 2;
        return x;
    };
    const int quads = p.dim / 4;
    const int64_t lanes = (int64_t)p.requests * p.qheads * quads;
    CombineShape c;
    c.spans = pow2_to(chunks / kSpanChunks + 1, 32);
    while (c.spans > 1 && c.spans * lanes > 4096 * 64)
        c.spans /= 2;
    c.lanes = std::min(pow2_to(quads, 64), kCombineMost / c.spans);
    c.heads = std::max(1, 64 / (c.spans * c.lanes));
    const dim3 grid((unsigned)p.requests, (unsigned)((p.qheads + c.heads - 1) / c.heads),
                    (unsigned)((quads + c.lanes - 1) / c.lanes));
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
