// The ordered merge of the paged attention's chunk partials, for launches of one
// new token of every request and of all of a step's.
#pragma once

#include "launch.hpp"
#include "paged_params.hpp"

#include <algorithm>

namespace pcl {

// LANES lanes hold four dims each of one query head; SPANS such groups merge a
// span of 16 chunks each, ascending from (-inf, 0, 0), in batches of BATCH loads,
// and the first group folds the spans in ascending order.
constexpr int kCombineMost = 256; // threads of a workgroup, at most

struct CombineShape {
    int lanes, spans, heads; // powers of two; heads: query heads of a workgroup
};

// A row's partials: chunk c's of [c0, c1) is base + c - first. The chunks of a span
// that ends at `split` or before it are merged already, into the place of the last one.
struct RowParts {
    uint32_t base;
    int c0, c1;
    int first, split;
};

// Merges them for the workgroup's heads and dims and calls write(head, dim, the
// merged state).
template <int BATCH, typename Write>
__device__ __forceinline__ void combine_row(const PagedParams &p, const CombineShape &c,
                                            const RowParts &r, int head0, int dim0, Write write)
{
    __shared__ f4 so[kCombineMost];
    __shared__ float sm[kCombineMost], sl[kCombineMost];
    const int c0 = r.c0, c1 = r.c1; // the row's chunks
    const int s0 = c0 / kSpanChunks, s1 = (c1 - 1) / kSpanChunks + 1;
    const int tid = threadIdx.x;
    const int q = tid % c.lanes, gi = tid / c.lanes % c.spans;
    const int h = head0 + tid / (c.lanes * c.spans);
    const int d = dim0 + 4 * q;
    const bool in = h < p.qheads && d < p.dim;
    const int64_t row = in ? h : 0;
    const int at = in ? d : 0;
    Merged4 t = {kNegInf, 0.f, f4{0.f, 0.f, 0.f, 0.f}};
    for (int r0 = s0; r0 < s1; r0 += c.spans) {
        Merged4 s = {kNegInf, 0.f, f4{0.f, 0.f, 0.f, 0.f}};
        if (r0 + gi < s1) {
            int e = min((r0 + gi + 1) * kSpanChunks, c1);
            int a = max((r0 + gi) * kSpanChunks, c0);
            if (a < r.split) {
                e = min((r0 + gi + 1) * kSpanChunks, r.split);
                a = e - 1;
            }
            for (; a < e; a += BATCH) {
                f2 ml[BATCH];
                f4 ov[BATCH];
#pragma unroll
                for (int i = 0; i < BATCH; ++i) {
                    const int64_t part =
                        (int64_t)(r.base + (uint32_t)(min(a + i, e - 1) - r.first)) * p.qheads + row;
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
    if (gi == 0 && in)
        write(h, d, t);
}

// The merged state's output, to `to`.
__device__ __forceinline__ void write_merged(const PagedParams &p, const Merged4 &t, float *to)
{
    f4 v;
    bool nonfinite = false;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        v[j] = t.acc[j] / t.L;
        nonfinite |= !is_finite(v[j]);
    }
    stg4(to, v);
    if (nonfinite)
        atomicOr(p.err, kErrOutput);
}

// Groups of the combine of `rows` rows (a request's new tokens): as many spans at
// once as some four thousand waves allow (one long request: 32, each a round trip
// or two; 64 requests of 16 heads of 256 dims: 4), the fewer the wider. In groups
// of 8 lanes and 32 spans throughout, 256 requests of up to 2048 keys took 48 us
// here (5.6 now), 64 of up to 8192 keys 27 us (5.6). Batches of 16 loads from 4 spans
// on were 1 to 3 us slower (146 registers against 114), 2048 or 8192 waves within 1
// us.
inline CombineShape combine_shape(const PagedParams &p, int64_t rows, int64_t chunks)
{
    auto pow2_to = [](int64_t n, int most) { // the least power of two >= n, at most `most`
        int x = 1;
        while (x < n && x < most)
            x *= 2;
        return x;
    };
    const int quads = p.dim / 4;
    const int64_t lanes = rows * p.qheads * quads;
    CombineShape c;
    c.spans = pow2_to(chunks / kSpanChunks + 1, 32);
    while (c.spans > 1 && c.spans * lanes > 4096 * 64)
        c.spans /= 2;
    c.lanes = std::min(pow2_to(quads, 64), kCombineMost / c.spans);
    c.heads = std::max(1, 64 / (c.spans * c.lanes));
    return c;
}

inline dim3 combine_grid(const PagedParams &p, const CombineShape &c, unsigned x)
{
    const int quads = p.dim / 4;
    return dim3(x, (unsigned)((p.qheads + c.heads - 1) / c.heads),
                (unsigned)((quads + c.lanes - 1) / c.lanes));
}

} // namespace pcl
