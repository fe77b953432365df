// Attention of one new token of every request over a paged KV cache on
// gfx950, split over the cache's length in 256-key chunks and joined.
//
// For request b with L keys, newest row r, query head h of KV head kh:
//   s_t = cap(q_scale * q[r][h] . K[slot_t][kh]),  max(0, L - window) <= t < L
//   out[r][h] = sum_t exp(s_t - max s) V[slot_t][kh] / sum_t exp(s_t - max s)
// with slot_t = table[b][t div P] * P + t mod P. The arithmetic is the
// canonical one of attention_device.hpp over the request's own key indices,
// so a request's output has the bits of the contiguous kernels over the same
// rows (bf16 pages: over the rows widened to f32, which is exact), whatever
// else is in the batch.
//
// The lengths live on the device, so the launch is a fixed grid whose
// workgroups form the chunk counts' sums over the requests themselves and
// take (chunk, KV head, 16-row unit) items in turn. An item's chunk is scored
// by NW waves (8 / NW tiles each), the running maxima meet in LDS, and every
// wave then runs the P.V chains of its DK / NW output dims over all eight
// tiles. A request of one chunk is written at once; the others leave chunk
// partials in the workspace for paged_combine_kernel.
#include "context.hpp"
#include "launch.hpp"
#include "paged.hpp"

#include <algorithm>
#include <atomic>
#include <cmath>
#include <cstdio>

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
    uint32_t *ws_off;    // [requests + 1] chunks before a request
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
    r.first = p.window && r.len > p.window ? r.len - p.window : 0;
    return r;
}

__device__ __forceinline__ int request_chunks(const RequestKeys &r)
{
    return r.len ? (r.len - 1) / kChunk + 1 - r.first / kChunk : 0;
}

// Chunks before each request, into off[requests + 1] (LDS), by the whole
// workgroup; ends with a barrier.
__device__ __forceinline__ void chunk_offsets(const PagedParams &p, uint32_t *off, uint32_t *waves)
{
    const int threads = blockDim.x;
    const int per = (p.requests + threads - 1) / threads;
    const int i0 = min((int)threadIdx.x * per, p.requests), i1 = min(i0 + per, p.requests);
    uint32_t sum = 0;
    bool bad = false;
    for (int i = i0; i < i1; ++i) {
        const uint32_t n = request_chunks(request_keys(p, i, &bad));
        off[i] = n;
        sum += n;
    }
    uint32_t total;
    uint32_t at = block_offsets(sum, waves, &total);
    for (int i = i0; i < i1; ++i) {
        const uint32_t n = off[i];
        off[i] = at;
        at += n;
    }
    if (threadIdx.x == 0)
        off[p.requests] = total;
    if (bad && blockIdx.x == 0)
        atomicOr(p.err, kErrPages);
    __syncthreads();
}

// Eight consecutive values of a K row (16 or 32 bytes), widened to f32.
template <typename T> struct Piece8;
template <> struct Piece8<float> {
    f4 v[2];
    __device__ __forceinline__ void load(const float *p)
    {
        v[0] = ldg4_stream(p);
        v[1] = ldg4_stream(p + 4);
    }
    __device__ __forceinline__ float operator[](int j) const { return v[j >> 2][j & 3]; }
};
typedef uint32_t u4 __attribute__((ext_vector_type(4)));
typedef uint32_t u2 __attribute__((ext_vector_type(2)));
template <> struct Piece8<__bf16> {
    u4 v;
    __device__ __forceinline__ void load(const __bf16 *p)
    {
        v = __builtin_nontemporal_load((const __attribute__((address_space(1))) u4 *)p);
    }
    __device__ __forceinline__ float operator[](int j) const
    {
        return j & 1 ? bf16_high(v[j >> 1]) : bf16_low(v[j >> 1]);
    }
};

// N consecutive values of a V row, widened to f32.
template <typename T, int N> struct PieceN;
template <int N> struct PieceN<float, N> {
    float v[N];
    __device__ __forceinline__ void load(const float *p)
    {
        if constexpr (N >= 4) {
#pragma unroll
            for (int i = 0; i < N / 4; ++i) {
                const f4 x = ldg4_stream(p + 4 * i);
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    v[4 * i + e] = x[e];
            }
        } else if constexpr (N == 2) {
            const f2 x = ldg2(p);
            v[0] = x.x;
            v[1] = x.y;
        } else {
            v[0] = ldg(p);
        }
    }
    __device__ __forceinline__ float operator[](int j) const { return v[j]; }
};
template <int N> struct PieceN<__bf16, N> {
    uint32_t v[(N + 1) / 2];
    __device__ __forceinline__ void load(const __bf16 *p)
    {
        if constexpr (N == 8) {
            const u4 x = __builtin_nontemporal_load((const __attribute__((address_space(1))) u4 *)p);
#pragma unroll
            for (int e = 0; e < 4; ++e)
                v[e] = x[e];
        } else if constexpr (N == 4) {
            const u2 x = __builtin_nontemporal_load((const __attribute__((address_space(1))) u2 *)p);
            v[0] = x.x;
            v[1] = x.y;
        } else if constexpr (N == 2) {
            v[0] = *(const __attribute__((address_space(1))) uint32_t *)p;
        } else {
            v[0] = *(const __attribute__((address_space(1))) uint16_t *)p;
        }
    }
    __device__ __forceinline__ float operator[](int j) const
    {
        return j & 1 ? bf16_high(v[j >> 1]) : bf16_low(v[j >> 1]);
    }
};

template <int DK, int NW> struct PagedCfg {
    static constexpr int kThreads = 64 * NW;
    static constexpr int NU = DK / 32;                  // score chain steps
    static constexpr int TPW = kTilesPerChunk / NW;     // tiles a wave scores
    static constexpr int VD = DK / NW;                  // output dims of a wave
    static constexpr int VW = VD / 16;                  // output blocks of a wave
    static constexpr int kQ = DK + 4;                   // padded Q row
    static_assert(VW >= 1 && VW * 16 * NW == DK, "whole 16-dim output blocks");
};

// FULL: the head dim equals the padded head dim DK.
template <int DK, typename T, bool FULL, bool CAP, int NW>
__global__ __launch_bounds__(64 * NW) void paged_kv_kernel(PagedParams p)
{
    using C = PagedCfg<DK, NW>;
    constexpr int NU = C::NU, TPW = C::TPW, VW = C::VW;
    __shared__ __attribute__((aligned(16))) float qs[kRows * C::kQ];
    __shared__ float ps[kTilesPerChunk][8][64];
    __shared__ float tmx[kTilesPerChunk][kRows], trs[kTilesPerChunk][kRows];
    __shared__ int32_t slots[kChunk];
    __shared__ uint32_t waves[NW];
    extern __shared__ uint32_t off[];
    const int tid = threadIdx.x;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int lane = tid & 63, col = lane & 15, g = lane >> 4;

    chunk_offsets(p, off, waves);
    if (blockIdx.x == 0)
        for (int i = tid; i <= p.requests; i += C::kThreads)
            p.ws_off[i] = off[i];
    const int per_chunk = p.kvheads * p.units;
    const int64_t items = (int64_t)off[p.requests] * per_chunk;

    for (int64_t item = blockIdx.x; item < items; item += gridDim.x) {
        const uint32_t ci = (uint32_t)(item / per_chunk);
        const int rest = (int)(item % per_chunk);
        const int kh = rest / p.units, unit = rest % p.units;
        const int b = find_range(off, p.requests, ci);
        bool unused = false;
        const RequestKeys rk = request_keys(p, b, &unused);
        const int c0 = rk.first / kChunk;
        const int cbase = (c0 + (int)(ci - off[b])) * kChunk;
        const bool only = off[b + 1] - off[b] == 1; // the request's only chunk
        // chunk-relative keys [lo, hi] are attended
        const int lo = max(rk.first - cbase, 0), hi = min(rk.len - 1 - cbase, kChunk - 1);

        __syncthreads(); // the last item's LDS is read
        // slots of the chunk's keys; a key outside [lo, hi] reads the nearest
        // one inside (its score and probability are not used)
        for (int i = tid; i < kChunk; i += C::kThreads) {
            const uint32_t t = (uint32_t)(cbase + min(max(i, lo), hi));
            int page = p.table[b * p.table_stride + t / p.page_tokens];
            if (page < 0 || page >= p.pages) {
                atomicOr(p.err, kErrPages);
                page = 0;
            }
            slots[i] = page * (int32_t)p.page_tokens + (int32_t)(t % p.page_tokens);
        }
        // the unit's query rows, scaled; zero past the group and the head dim
        const int h0 = kh * p.group + unit * kRows;
        const int nrows = min(p.group - unit * kRows, kRows);
        for (int i = tid; i < kRows * (DK / 4); i += C::kThreads) {
            const int r = i / (DK / 4), d = 4 * (i % (DK / 4));
            const bool in = r < nrows && (FULL || d < p.dim);
            const f4 x = ldg4(p.q + rk.row * p.q_stride + (in ? (int64_t)(h0 + r) * p.dim + d : 0));
            *(f4 *)(qs + r * C::kQ + d) = in ? x * p.q_scale : f4{0.f, 0.f, 0.f, 0.f};
        }
        __syncthreads();

        const T *kp = static_cast<const T *>(p.k) + (int64_t)kh * p.dim;
        const T *vp = static_cast<const T *>(p.v) + (int64_t)kh * p.dim;
        const bool rin = col < nrows;

        float s[TPW][2][4];
        bool bad = false;
#pragma unroll
        for (int tt = 0; tt < TPW; ++tt) {
            const int t = w * TPW + tt;
            const bool any = kTile * t <= hi && kTile * t + kTile - 1 >= lo;
            float tm = kNegInf;
            if (any) {
#pragma unroll
                for (int blk = 0; blk < 2; ++blk) {
                    const T *row = kp + (int64_t)slots[kTile * t + 16 * blk + col] * p.row_stride;
                    Piece8<T> kb[NU];
#pragma unroll
                    for (int u = 0; u < NU; ++u) {
                        const int d = 32 * u + 8 * g;
                        kb[u].load(row + (FULL || d < p.dim ? d : 0));
                    }
                    f4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int u = 0; u < NU; ++u) {
                        const int d = 32 * u + 8 * g;
                        const f4 qa = *(const f4 *)(qs + col * C::kQ + d);
                        const f4 qb = *(const f4 *)(qs + col * C::kQ + d + 4);
#pragma unroll
                        for (int jj = 0; jj < 8; ++jj) {
                            const float k = kb[u][jj];
                            acc = mfma(FULL || d < p.dim ? k : 0.f, jj < 4 ? qa[jj] : qb[jj - 4],
                                       acc);
                        }
                    }
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const float x = acc[r];
                        s[tt][blk][r] =
                            CAP ? soft_cap(x, p.softcap, p.inv_softcap) : x;
                        const int key = kTile * t + 16 * blk + 4 * g + r;
                        const bool ok = key >= lo && key <= hi;
                        bad |= ok && rin && !is_finite(s[tt][blk][r]);
                        tm = ok ? fmaxf(tm, s[tt][blk][r]) : tm;
                    }
                }
                tm = max_xor16(tm);
                tm = max_xor32(tm);
            }
            if (g == 0)
                tmx[t][col] = tm;
        }
        __syncthreads(); // every tile's maximum
        float tmr[kTilesPerChunk];
#pragma unroll
        for (int t = 0; t < kTilesPerChunk; ++t)
            tmr[t] = tmx[t][col];
        {
            float m = kNegInf;
#pragma unroll
            for (int t = 0; t < kTilesPerChunk; ++t) {
                m = fmaxf(m, tmr[t]);
                if (t / TPW != w)
                    continue;
                if (!(kTile * t <= hi && kTile * t + kTile - 1 >= lo))
                    continue;
                bool ok[2][4];
#pragma unroll
                for (int blk = 0; blk < 2; ++blk)
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const int key = kTile * t + 16 * blk + 4 * g + r;
                        ok[blk][r] = key >= lo && key <= hi;
                    }
                float pr[2][4];
                const float rs = tile_probs(s[t % TPW], ok, safe_max(m), pr);
#pragma unroll
                for (int blk = 0; blk < 2; ++blk)
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        ps[t][4 * blk + r][lane] = pr[blk][r];
                if (g == 0)
                    trs[t][col] = rs;
            }
        }
        if (bad)
            atomicOr(p.err, kErrScore);
        __syncthreads(); // every tile's probabilities and row sums

        // the l chain and the P.V chains of the wave's output blocks; block x:
        // A operand V[key][d0 + VW col + x], so O[x][i] is dim
        // d0 + VW (4g + i) + x of row col
        const int d0 = C::VD * w;
        const int vd = d0 + VW * col;
        const bool vin = FULL || vd < p.dim;
        float m = kNegInf, l = 0.f;
        f4 O[VW];
#pragma unroll
        for (int x = 0; x < VW; ++x)
            O[x] = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int t = 0; t < kTilesPerChunk; ++t) {
            if (!(kTile * t <= hi && kTile * t + kTile - 1 >= lo))
                continue;
            PieceN<T, VW> vr[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int key = kTile * t + 16 * (e >> 2) + 4 * g + (e & 3);
                vr[e].load(vp + (int64_t)slots[key] * p.row_stride + (vin ? vd : 0));
            }
            const float mn = fmaxf(m, tmr[t]);
            const float ms = safe_max(mn);
            const float alpha = fexp(m - ms);
            l = __builtin_fmaf(l, alpha, trs[t][col]);
            m = mn;
#pragma unroll
            for (int x = 0; x < VW; ++x)
                O[x] = O[x] * alpha;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float pe = ps[t][e][lane];
#pragma unroll
                for (int x = 0; x < VW; ++x)
                    O[x] = mfma(vr[e][x], pe, O[x]);
            }
        }

        if (!rin)
            continue;
        // lane (col, g): the 4 VW dims from d0 + 4 VW g of row col
        const int dg = d0 + 4 * VW * g;
        const int h = h0 + col;
        const int64_t part = (int64_t)ci * p.qheads + h;
        float *dst = only ? p.out + rk.row * p.o_stride + (int64_t)h * p.dim + dg
                          : p.ws_o + part * p.dim + dg;
        bool nonfinite = false;
#pragma unroll
        for (int k = 0; k < VW; ++k) {
            if (!FULL && dg + 4 * k >= p.dim)
                continue;
            f4 v;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int n = 4 * k + e;
                v[e] = O[n % VW][n / VW];
                if (only) {
                    v[e] = v[e] / l;
                    nonfinite |= !is_finite(v[e]);
                }
            }
            stg4(dst + 4 * k, v);
        }
        if (nonfinite)
            atomicOr(p.err, kErrOutput);
        if (!only && w == 0 && g == 0) {
            stg(p.ws_ml + 2 * part, m);
            stg(p.ws_ml + 2 * part + 1, l);
        }
    }
}

// The ordered merge of a request's chunk partials for one query head and a
// slab of 4 LANES dims: groups of LANES lanes merge a span of 16 chunks each,
// ascending from (-inf, 0, 0), and leave it in LDS, then the first group folds
// the spans in ascending order. Requests of one chunk are written already.
constexpr int kPagedLanes = 8;
constexpr int kPagedSpans = 32; // spans per round

__global__ __launch_bounds__(kPagedLanes * kPagedSpans) void paged_combine_kernel(PagedParams p)
{
    constexpr int L = kPagedLanes;
    __shared__ f4 so[kPagedSpans][L];
    __shared__ float sm[kPagedSpans], sl[kPagedSpans];
    const int b = blockIdx.x, h = blockIdx.y;
    const uint32_t base = p.ws_off[b];
    const int nch = (int)(p.ws_off[b + 1] - base);
    if (nch <= 1)
        return;
    bool unused = false;
    const RequestKeys rk = request_keys(p, b, &unused);
    const int c0 = rk.first / kChunk, c1 = c0 + nch; // the request's chunks
    const int s0 = c0 / kSpanChunks, s1 = (c1 - 1) / kSpanChunks + 1;
    const int gi = threadIdx.x / L, q = threadIdx.x % L;
    const int d = 4 * L * blockIdx.z + 4 * q;
    const bool din = d < p.dim;
    Merged4 t = {kNegInf, 0.f, f4{0.f, 0.f, 0.f, 0.f}};
    for (int r0 = s0; r0 < s1; r0 += kPagedSpans) {
        const int n = min(s1 - r0, kPagedSpans);
        if (gi < n) {
            const int a = max((r0 + gi) * kSpanChunks, c0), e = min((r0 + gi + 1) * kSpanChunks, c1);
            f2 ml[kSpanChunks];
            f4 ov[kSpanChunks];
#pragma unroll
            for (int i = 0; i < kSpanChunks; ++i) {
                const int64_t part =
                    (int64_t)(base + (uint32_t)((a + i < e ? a + i : a) - c0)) * p.qheads + h;
                ml[i] = ldg2(p.ws_ml + 2 * part);
                ov[i] = ldg4(p.ws_o + part * p.dim + (din ? d : 0));
            }
            Merged4 s = {kNegInf, 0.f, f4{0.f, 0.f, 0.f, 0.f}};
#pragma unroll
            for (int i = 0; i < kSpanChunks; ++i) {
                const bool in = a + i < e;
                merge_into4(s, in ? ml[i].x : kNegInf, in ? ml[i].y : 0.f,
                            in ? ov[i] : f4{0.f, 0.f, 0.f, 0.f});
            }
            so[gi][q] = s.acc;
            if (q == 0) {
                sm[gi] = s.M;
                sl[gi] = s.L;
            }
        }
        __syncthreads();
        if (gi == 0)
            for (int i = 0; i < n; ++i)
                merge_into4(t, sm[i], sl[i], so[i][q]);
        __syncthreads();
    }
    if (gi != 0 || !din)
        return;
    f4 v;
    bool nonfinite = false;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        v[j] = t.acc[j] / t.L;
        nonfinite |= !is_finite(v[j]);
    }
    stg4(p.out + rk.row * p.o_stride + (int64_t)h * p.dim + d, v);
    if (nonfinite)
        atomicOr(p.err, kErrOutput);
}

constexpr int kPagedGroupsPerCu = 4;

template <int DK, typename T, bool FULL, bool CAP>
static hipError_t launch_paged(const PagedParams &p, int64_t items, hipStream_t stream)
{
    constexpr int NW = DK == 64 ? 4 : 4;
    const int cus = std::max(device_cus(), 1);
    const int64_t grid = std::max<int64_t>(1, std::min<int64_t>(items, kPagedGroupsPerCu * cus));
    const size_t lds = ((size_t)p.requests + 1) * sizeof(uint32_t);
    paged_kv_kernel<DK, T, FULL, CAP, NW><<<(unsigned)grid, 64 * NW, lds, stream>>>(p);
    return hipGetLastError();
}

template <int DK, typename T> static hipError_t launch_paged(const PagedParams &p, int64_t items,
                                                             hipStream_t stream)
{
    if (p.softcap > 0.f)
        return p.dim == DK ? launch_paged<DK, T, true, true>(p, items, stream)
                           : launch_paged<DK, T, false, true>(p, items, stream);
    return p.dim == DK ? launch_paged<DK, T, true, false>(p, items, stream)
                       : launch_paged<DK, T, false, false>(p, items, stream);
}

template <typename T>
static hipError_t launch_paged(const PagedParams &p, int64_t items, hipStream_t stream)
{
    return p.dim <= 64    ? launch_paged<64, T>(p, items, stream)
           : p.dim <= 128 ? launch_paged<128, T>(p, items, stream)
           : p.dim <= 256 ? launch_paged<256, T>(p, items, stream)
                          : launch_paged<512, T>(p, items, stream);
}

// Chunks that one request may have.
static int64_t most_chunks(const pcl_paged_desc &d)
{
    const int64_t all = (d.max_length + kChunk - 1) / kChunk;
    return d.window ? std::min(all, (d.window + kChunk - 2) / kChunk + 1) : all;
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
    // chunk indices of the whole batch stay below 2^31
    if (most_chunks(d) > kMaxSlots / d.requests)
        return PCL_INVALID_SHAPE;
    return PCL_OK;
}

// Workspace bytes: the chunk partials of every request at its longest (none
// where no request can have two chunks), then the chunk offsets.
static size_t paged_bytes(const pcl_paged_desc &d)
{
    if (d.requests == 0)
        return 0;
    const int64_t each = most_chunks(d);
    const size_t parts = each > 1 ? (size_t)(d.requests * each) * d.qheads : 0;
    return parts * (d.pools.dim + 2) * sizeof(float) + (d.requests + 1) * sizeof(uint32_t);
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
    p.ws_o = body;
    p.ws_ml = body + parts * s.dim;
    p.ws_off = reinterpret_cast<uint32_t *>(body + parts * (s.dim + 2));
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
    p.units = (int)((group + pcl::kRows - 1) / pcl::kRows);
    p.dim = (int)s.dim;
    p.q_scale = d.q_scale;
    p.softcap = d.softcap;
    p.inv_softcap = d.softcap > 0.0f ? 1.0f / d.softcap : 0.0f;
    const int64_t items = d.requests * each * s.kvheads * p.units;
    hipError_t e = s.type == PCL_CACHE_F32 ? pcl::launch_paged<float>(p, items, ctx->stream)
                                           : pcl::launch_paged<__bf16>(p, items, ctx->stream);
    if (e == hipSuccess && each > 1) {
        const dim3 grid((unsigned)d.requests, (unsigned)d.qheads,
                        (unsigned)((s.dim + 4 * pcl::kPagedLanes - 1) / (4 * pcl::kPagedLanes)));
        pcl::paged_combine_kernel<<<grid, pcl::kPagedLanes * pcl::kPagedSpans, 0, ctx->stream>>>(p);
        e = hipGetLastError();
    }
    if (e != hipSuccess) {
        std::fprintf(stderr, "pcl_paged_attention: launch: %s\n", hipGetErrorString(e));
        return PCL_NON_FINITE_VALUE;
    }
    return PCL_OK;
}

} // extern "C"
