// What the paged attention's chunk kernels and its combine share: the launch's
// parameters and the keys of a request.
#pragma once

#include "attention_device.hpp"

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
                         // its first chunk, its row
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

// The chunk kernel of a launch of at most `chunks` chunks, at padded head dim
// DK (64, 128, 256 or 512, a source file each).
template <int DK>
hipError_t launch_paged_kv(const PagedParams &p, bool bf16, int64_t chunks, hipStream_t stream);

} // namespace pcl
