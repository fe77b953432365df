// What the paged cache's kernels share: page arithmetic, row types and the
// device error bit of bad page data.
#pragma once

#include "attention_device.hpp"
#include "pcl_attention.h"

#include <cstdint>

namespace pcl {

// A step that does not fit, or a length, row, slot or page outside its range.
constexpr int kErrPages = 32;

// Bounds of the host's checks. Kernels keep one word per request in LDS; a
// slot (page * page_tokens + offset) stays within an int32.
constexpr int64_t kMaxRequests = 2048;
constexpr int64_t kMaxPageTokens = 4096;
constexpr int64_t kMaxStepRows = ((int64_t)1 << 20) - 1;
constexpr int64_t kMaxSlots = ((int64_t)1 << 31) - 1;

// Checks of the pools' fields alone (pointers and sizes).
bool valid_pools(const pcl_page_pools &pools);

// Pages that hold `tokens` tokens.
__host__ __device__ __forceinline__ uint32_t pages_of(uint32_t tokens, uint32_t page_tokens)
{
    return tokens ? (tokens - 1) / page_tokens + 1 : 0;
}

// The index i of ascending offsets (off[0] = 0, off[n] > x) with
// off[i] <= x < off[i + 1].
__device__ __forceinline__ int find_range(const uint32_t *off, int n, uint32_t x)
{
    int lo = 0, hi = n; // off[lo] <= x < off[hi]
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (off[mid] <= x)
            lo = mid;
        else
            hi = mid;
    }
    return lo;
}

// Exclusive sum of v over the threads of a workgroup of whole waves (at most
// 16), and the total; `waves` holds a word per wave. A barrier on either
// side keeps `waves` free for the next call.
template <typename T>
__device__ __forceinline__ T block_offsets(T v, T *waves, T *total)
{
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int count = blockDim.x >> 6;
    T x = v;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const T y = __shfl_up(x, o);
        if (lane >= o)
            x += y;
    }
    if (lane == 63)
        waves[wave] = x;
    __syncthreads();
    T before = 0, all = 0;
    for (int i = 0; i < count; ++i) {
        const T n = waves[i];
        before += i < wave ? n : 0;
        all += n;
    }
    __syncthreads();
    *total = all;
    return before + x - v;
}

// bf16 words to f32 (exact): the low and the high half of a 32-bit word.
__device__ __forceinline__ float bf16_low(uint32_t w)
{
    return __uint_as_float(w << 16);
}

__device__ __forceinline__ float bf16_high(uint32_t w)
{
    return __uint_as_float(w & 0xffff0000u);
}

// Four f32 values into a row of the pages: as they are, or rounded to bf16
// (nearest, ties to even: off by at most 2^-8 of the value).
__device__ __forceinline__ void store_row4(float *at, f4 v)
{
    stg4(at, v);
}

__device__ __forceinline__ void store_row4(__bf16 *at, f4 v)
{
    typedef __bf16 b4 __attribute__((ext_vector_type(4)));
    *(__attribute__((address_space(1))) b4 *)at = __builtin_convertvector(v, b4);
}

} // namespace pcl
