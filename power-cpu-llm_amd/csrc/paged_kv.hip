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
// take (chunk, KV head, unit of query rows) items in turn. Scores: a lane is a
// key, its K row loaded by itself and multiplied with four query rows a matrix
// instruction. The running maxima meet in LDS, and every wave then runs the
// P.V chains of its own output dims over the whole chunk, a lane holding VL of
// them. A request of one chunk is written at once; the others leave chunk
// partials in the workspace for paged_combine_kernel.
//
// A lane's K row is read 16 bytes at a time, eight loads to a 128-byte line, so
// these are plain loads: streaming ones left nothing of a line in the L1 cache
// and read it again for each (64 requests of up to 8192 keys, 16 x 8 x 256 heads
// in bf16: 4.6 times the lines and 345 us, plain 209 us).
#include "context.hpp"
#include "launch.hpp"
#include "paged.hpp"

#include <algorithm>
#include <atomic>
#include <cmath>
#include <cstdio>
#include <type_traits>

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

// f(std::integral_constant<int, i>) for i = 0 .. N - 1, in order.
template <int N, int I = 0, typename F> __device__ __forceinline__ void each(F &&f)
{
    if constexpr (I < N) {
        f(std::integral_constant<int, I>{});
        each<N, I + 1>(f);
    }
}

// acc + a b for 64 columns and four rows: every lane is a column with its own
// b, the four rows' a are those of lanes 4 BLOCK .. 4 BLOCK + 3. The f32 MFMAs
// are chains of fmas over their k slots (checked bit for bit on MI355X), so 4 of
// these in the order of the slots equal one v_mfma_f32_16x16x4f32 of the
// canonical chains, at an eighth of its matrix time for four rows.
template <int BLOCK> __device__ __forceinline__ f4 mfma_rows4(float a, float b, f4 acc)
{
    return __builtin_amdgcn_mfma_f32_4x4x1f32(a, b, acc, 4, BLOCK, 0);
}

// Head dim of the n-th step of the canonical score chain (u, jj, g), and the
// key of a tile at the n-th step of the canonical P.V chain (b, r, g).
__host__ __device__ constexpr int chain_dim(int n)
{
    return 32 * (n / 32) + 8 * (n % 4) + n % 32 / 4;
}

__host__ __device__ constexpr int chain_key(int n)
{
    return 16 * (n / 16) + 4 * (n % 4) + n % 16 / 4;
}

template <int CTRL> __device__ __forceinline__ float dpp(float x)
{
    return __uint_as_float(
        __builtin_amdgcn_update_dpp(0, __float_as_uint(x), CTRL, 0xf, 0xf, true));
}

constexpr int kDppXor1 = 0xb1, kDppXor2 = 0x4e, kDppMirror16 = 0x140, kDppMirror8 = 0x141;

// The maximum of 32 lanes (a tile's keys), on each of them.
__device__ __forceinline__ float max_tile(float x)
{
    x = fmaxf(x, dpp<kDppXor1>(x));
    x = fmaxf(x, dpp<kDppXor2>(x));
    x = fmaxf(x, dpp<kDppMirror8>(x));
    x = fmaxf(x, dpp<kDppMirror16>(x));
    return max_xor16(x);
}

// The canonical row sum of 32 lanes: the tree over the key's bits 0, 1, 4, 2
// and 3 (a mirror of 8 or 16 lanes is the flip of bit 2 or 3 once the lanes
// below that bit agree).
__device__ __forceinline__ float sum_tile(float x)
{
    x = x + dpp<kDppXor1>(x);
    x = x + dpp<kDppXor2>(x);
    x = add_xor16(x);
    x = x + dpp<kDppMirror8>(x);
    return x + dpp<kDppMirror16>(x);
}

typedef uint32_t u4 __attribute__((ext_vector_type(4)));
typedef uint32_t u2 __attribute__((ext_vector_type(2)));
typedef const __attribute__((address_space(1))) u4 *gu4_cptr;
typedef const __attribute__((address_space(1))) u2 *gu2_cptr;
typedef const __attribute__((address_space(1))) uint32_t *gu1_cptr;
typedef const __attribute__((address_space(1))) uint16_t *gu16_cptr;

// Value j of loaded words, widened to f32.
template <typename T> __device__ __forceinline__ float value_of(const uint32_t *words, int j)
{
    if constexpr (sizeof(T) == 4)
        return __uint_as_float(words[j]);
    else
        return j & 1 ? bf16_high(words[j / 2]) : bf16_low(words[j / 2]);
}

// One lane's N consecutive values of a V row.
template <typename T, int N> struct Values {
    static constexpr int kWords = (N * (int)sizeof(T) + 3) / 4;
    uint32_t w[kWords];
    __device__ __forceinline__ void load(const T *p)
    {
        if constexpr (kWords == 4) {
            const u4 x = __builtin_nontemporal_load((gu4_cptr)p);
#pragma unroll
            for (int e = 0; e < 4; ++e)
                w[e] = x[e];
        } else if constexpr (kWords == 2) {
            const u2 x = __builtin_nontemporal_load((gu2_cptr)p);
            w[0] = x.x;
            w[1] = x.y;
        } else if constexpr (N * sizeof(T) == 4) {
            w[0] = __builtin_nontemporal_load((gu1_cptr)p);
        } else {
            w[0] = __builtin_nontemporal_load((gu16_cptr)p);
        }
    }
};

// Shape of a workgroup: NW waves, 64 KG keys scored by each; the first PVW of
// them run the P.V chains of 64 VL output dims. R sets of four query rows.
template <int DK, typename T, int R> struct PagedCfg {
    static constexpr int NW = DK >= 256 ? 4 : DK / 64;
    static constexpr int VL = DK / 64 / NW;
    static constexpr int PVW = NW;
    static constexpr int KG = 4 / NW;
    static constexpr int kThreads = 64 * NW;
    // K in pieces of a 128-byte line of each of 64 rows, KB of them in flight
    static constexpr int kLine = 128 / (int)sizeof(T);
    static constexpr int KP = DK / kLine; // pieces of a row
    static constexpr int KB = KP < 2 ? KP : 2;
    // V tiles in flight
    static constexpr int VB = 2;
    static constexpr int kRowsUnit = 4 * R;
};

// LDS of a workgroup: the query rows and the probabilities in the order in
// which the MFMAs' A registers take them, and each tile's per-row words.
template <int DK, int R> struct PagedLds {
    float q[R][DK][4];                  // [row set][chain step][row]
    float p[R][kTilesPerChunk][kTile][4]; // [row set][tile][chain step][row]
    f4 max[kTilesPerChunk][R], alpha[kTilesPerChunk][R], sum[kTilesPerChunk][R];
    int32_t slots[kChunk];
};

// FULL: the head dim equals the padded head dim DK.
template <int DK, typename T, bool FULL, bool CAP, int R>
__global__ __launch_bounds__((PagedCfg<DK, T, R>::kThreads)) void paged_kv_kernel(PagedParams p)
{
    using C = PagedCfg<DK, T, R>;
    constexpr int KG = C::KG, KP = C::KP, KB = C::KB, VL = C::VL, VB = C::VB;
    __shared__ __attribute__((aligned(16))) PagedLds<DK, R> s;
    __shared__ uint32_t waves[C::NW];
    extern __shared__ uint32_t off[];
    const int tid = threadIdx.x;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int lane = tid & 63;

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
        const int cbase = (rk.first / kChunk + (int)(ci - off[b])) * kChunk;
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
            s.slots[i] = page * (int32_t)p.page_tokens + (int32_t)(t % p.page_tokens);
        }
        // the unit's query rows, scaled; zero past the group and the head dim
        const int h0 = kh * p.group + unit * C::kRowsUnit;
        const int nrows = min(p.group - unit * C::kRowsUnit, C::kRowsUnit);
        for (int i = tid; i < R * DK; i += C::kThreads) {
            const int r = i / (DK / 4), d = 4 * (i % (DK / 4));
            const bool in = r < nrows && (FULL || d < p.dim);
            f4 x = ldg4(p.q + rk.row * p.q_stride + (in ? (int64_t)(h0 + r) * p.dim + d : 0));
            x = in ? x * p.q_scale : f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int k = (d + e) % 32; // 8 g + jj
                s.q[r / 4][(d & ~31) + 4 * (k % 8) + k / 8][r % 4] = x[e];
            }
        }
        __syncthreads();

        const T *kp = static_cast<const T *>(p.k) + (int64_t)kh * p.dim;
        const T *vp = static_cast<const T *>(p.v) + (int64_t)kh * p.dim;

        // scores: lane = key
        f4 acc[KG][R];
        bool bad = false;
#pragma unroll
        for (int kg = 0; kg < KG; ++kg) {
            const int k0 = 64 * (w * KG + kg);
            if (k0 > hi || k0 + 63 < lo)
                continue;
            const T *row = kp + (int64_t)s.slots[k0 + lane] * p.row_stride;
            uint32_t kb[KB][32];
            auto load = [&](int i, uint32_t *to) {
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const int d = C::kLine * i + e * (16 / (int)sizeof(T));
                    const bool in = FULL || d < p.dim;
                    const u4 x = *(gu4_cptr)(row + (in ? d : 0)); // (not streamed, see above)
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        to[4 * e + j] = in ? x[j] : 0u;
                }
            };
#pragma unroll
            for (int i = 0; i < KB; ++i)
                load(i, kb[i]);
#pragma unroll
            for (int r = 0; r < R; ++r)
                acc[kg][r] = f4{0.f, 0.f, 0.f, 0.f};
            each<KP>([&](auto ic) {
                constexpr int i = decltype(ic)::value;
                uint32_t *words = kb[i % KB];
#pragma unroll
                for (int m = 0; m < C::kLine / 16; ++m) {
                    float a[R];
#pragma unroll
                    for (int r = 0; r < R; ++r)
                        a[r] = s.q[r][C::kLine * i + 16 * m + lane / 4][lane % 4];
                    each<16>([&](auto nc) {
                        constexpr int n = decltype(nc)::value;
                        const float k = value_of<T>(words, chain_dim(16 * m + n));
#pragma unroll
                        for (int r = 0; r < R; ++r)
                            acc[kg][r] = mfma_rows4<n>(a[r], k, acc[kg][r]);
                    });
                }
                __builtin_amdgcn_sched_barrier(0);
                if constexpr (i + KB < KP)
                    load(i + KB, words);
                __builtin_amdgcn_sched_barrier(0);
            });
            const int key = k0 + lane;
            const bool ok = key >= lo && key <= hi;
#pragma unroll
            for (int r = 0; r < R; ++r) {
                f4 tm;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    float x = acc[kg][r][e];
                    x = CAP ? soft_cap(x, p.softcap, p.inv_softcap) : x;
                    bad |= ok && 4 * r + e < nrows && !is_finite(x);
                    x = ok ? x : kNegInf;
                    acc[kg][r][e] = x;
                    tm[e] = max_tile(x);
                }
                if ((lane & 31) == 0)
                    s.max[key / kTile][r] = tm;
            }
        }
        if (bad)
            atomicOr(p.err, kErrScore);
        const int t0 = lo / kTile, t1 = hi / kTile; // tiles with attended keys
        __syncthreads(); // every tile's maximum

        // probabilities against the running maximum at the lane's tile
#pragma unroll
        for (int kg = 0; kg < KG; ++kg) {
            const int k0 = 64 * (w * KG + kg);
            if (k0 > hi || k0 + 63 < lo)
                continue;
            const int key = k0 + lane, t = key / kTile;
            const bool ok = key >= lo && key <= hi;
#pragma unroll
            for (int r = 0; r < R; ++r) {
                f4 before, m; // running maxima before and at the tile
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    before[e] = kNegInf;
                for (int i = t0; i < k0 / kTile; ++i) {
                    const f4 x = s.max[i][r];
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        before[e] = fmaxf(before[e], x[e]);
                }
                const f4 first = s.max[k0 / kTile][r], mine = s.max[t][r];
                f4 pr, sum, alpha;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    if (t > k0 / kTile && t0 <= k0 / kTile)
                        before[e] = fmaxf(before[e], first[e]);
                    m[e] = fmaxf(before[e], mine[e]);
                    const float ms = safe_max(m[e]);
                    pr[e] = ok ? fexp(acc[kg][r][e] - ms) : 0.f;
                    alpha[e] = fexp(before[e] - ms);
                    sum[e] = sum_tile(pr[e]);
                }
                const int k = key % kTile;
                *(f4 *)s.p[r][t][(k & 16) + 4 * (k & 3) + (k >> 2 & 3)] = pr;
                if ((lane & 31) == 0) {
                    s.alpha[t][r] = alpha;
                    s.sum[t][r] = sum;
                }
            }
        }
        __syncthreads(); // every tile's probabilities, row sums and factors

        if (w >= C::PVW)
            continue;
        // the l chain and the P.V chains of the lane's VL output dims
        const int vd = (64 * w + lane) * VL;
        const T *vlane = vp + (FULL || vd < p.dim ? vd : 0);
        f4 l[R], O[R][VL];
#pragma unroll
        for (int r = 0; r < R; ++r) {
            l[r] = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int x = 0; x < VL; ++x)
                O[r][x] = f4{0.f, 0.f, 0.f, 0.f};
        }
        Values<T, VL> vb[VB][kTile];
        auto load_v = [&](int t, Values<T, VL> *to) {
            const int slots = s.slots[kTile * t + (lane & 31)];
#pragma unroll
            for (int n = 0; n < kTile; ++n) {
                const int slot = __builtin_amdgcn_readlane(slots, chain_key(n));
                to[n].load(vlane + (int64_t)slot * p.row_stride);
            }
        };
        auto attend = [&](int t, const Values<T, VL> *v) {
#pragma unroll
            for (int r = 0; r < R; ++r) {
                const f4 alpha = s.alpha[t][r], sum = s.sum[t][r];
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    l[r][e] = __builtin_fmaf(l[r][e], alpha[e], sum[e]);
#pragma unroll
                for (int x = 0; x < VL; ++x)
                    O[r][x] = O[r][x] * alpha;
            }
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                float a[R];
#pragma unroll
                for (int r = 0; r < R; ++r)
                    a[r] = s.p[r][t][16 * half + lane / 4][lane % 4];
                each<16>([&](auto nc) {
                    constexpr int n = decltype(nc)::value;
#pragma unroll
                    for (int x = 0; x < VL; ++x)
#pragma unroll
                        for (int r = 0; r < R; ++r)
                            O[r][x] = mfma_rows4<n>(
                                a[r], value_of<T>(v[16 * half + n].w, x), O[r][x]);
                });
            }
        };
        // VB tiles in flight; tiles past the last repeat it (not attended)
#pragma unroll
        for (int i = 0; i < VB; ++i)
            load_v(min(t0 + i, t1), vb[i]);
        for (int t = t0; t <= t1; t += VB) {
#pragma unroll
            for (int i = 0; i < VB; ++i) {
                __builtin_amdgcn_sched_barrier(0);
                if (t + i <= t1)
                    attend(t + i, vb[i]);
                __builtin_amdgcn_sched_barrier(0);
                load_v(min(t + i + VB, t1), vb[i]);
            }
        }

        if (!FULL && vd >= p.dim)
            continue;
        f4 mlast[R];
        bool nonfinite = false;
#pragma unroll
        for (int r = 0; r < R; ++r) {
            mlast[r] = s.max[t0][r];
            for (int i = t0 + 1; i <= t1; ++i) {
                const f4 x = s.max[i][r];
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    mlast[r][e] = fmaxf(mlast[r][e], x[e]);
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if (4 * r + e >= nrows)
                    continue;
                const int h = h0 + 4 * r + e;
                const int64_t part = (int64_t)ci * p.qheads + h;
                float *dst = only ? p.out + rk.row * p.o_stride + (int64_t)h * p.dim + vd
                                  : p.ws_o + part * p.dim + vd;
#pragma unroll
                for (int x = 0; x < VL; ++x) {
                    const float v = only ? O[r][x][e] / l[r][e] : O[r][x][e];
                    nonfinite |= only && !is_finite(v);
                    stg(dst + x, v);
                }
                if (!only && w == 0 && lane == 0) {
                    stg(p.ws_ml + 2 * part, mlast[r][e]);
                    stg(p.ws_ml + 2 * part + 1, l[r][e]);
                }
            }
        }
        if (nonfinite)
            atomicOr(p.err, kErrOutput);
    }
}

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
    const int b = blockIdx.x;
    const uint32_t base = p.ws_off[b];
    const int nch = (int)(p.ws_off[b + 1] - base);
    if (nch <= 1)
        return;
    bool unused = false;
    const RequestKeys rk = request_keys(p, b, &unused);
    const int c0 = rk.first / kChunk, c1 = c0 + nch; // the request's chunks
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
    stg4(p.out + rk.row * p.o_stride + (int64_t)h * p.dim + d, v);
    if (nonfinite)
        atomicOr(p.err, kErrOutput);
}

// Groups of the combine: as many spans at once as some four thousand waves
// allow (one long request: 32, each a round trip or two; 64 requests of 16
// heads of 256 dims: 4), the fewer the wider.
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

constexpr int kPagedGroupsPerCu = 4;

template <int DK, typename T, bool FULL, bool CAP, int R>
static hipError_t launch_paged(PagedParams p, int64_t chunks, hipStream_t stream)
{
    using C = PagedCfg<DK, T, R>;
    p.units = (p.group + C::kRowsUnit - 1) / C::kRowsUnit;
    const int64_t items = chunks * p.kvheads * p.units;
    const int cus = std::max(device_cus(), 1);
    const int64_t grid = std::max<int64_t>(1, std::min<int64_t>(items, kPagedGroupsPerCu * cus));
    const size_t lds = ((size_t)p.requests + 1) * sizeof(uint32_t);
    paged_kv_kernel<DK, T, FULL, CAP, R><<<(unsigned)grid, C::kThreads, lds, stream>>>(p);
    return hipGetLastError();
}

template <int DK, typename T, bool FULL, bool CAP>
static hipError_t launch_paged(const PagedParams &p, int64_t chunks, hipStream_t stream)
{
    return p.group <= 4   ? launch_paged<DK, T, FULL, CAP, 1>(p, chunks, stream)
           : p.group <= 8 ? launch_paged<DK, T, FULL, CAP, 2>(p, chunks, stream)
                          : launch_paged<DK, T, FULL, CAP, 4>(p, chunks, stream);
}

template <int DK, typename T> static hipError_t launch_paged(const PagedParams &p, int64_t chunks,
                                                             hipStream_t stream)
{
    if (p.softcap > 0.f)
        return p.dim == DK ? launch_paged<DK, T, true, true>(p, chunks, stream)
                           : launch_paged<DK, T, false, true>(p, chunks, stream);
    return p.dim == DK ? launch_paged<DK, T, true, false>(p, chunks, stream)
                       : launch_paged<DK, T, false, false>(p, chunks, stream);
}

template <typename T>
static hipError_t launch_paged(const PagedParams &p, int64_t chunks, hipStream_t stream)
{
    return p.dim <= 64    ? launch_paged<64, T>(p, chunks, stream)
           : p.dim <= 128 ? launch_paged<128, T>(p, chunks, stream)
           : p.dim <= 256 ? launch_paged<256, T>(p, chunks, stream)
                          : launch_paged<512, T>(p, chunks, stream);
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
    p.units = 1;
    p.dim = (int)s.dim;
    p.q_scale = d.q_scale;
    p.softcap = d.softcap;
    p.inv_softcap = d.softcap > 0.0f ? 1.0f / d.softcap : 0.0f;
    const int64_t chunks = d.requests * each;
    hipError_t e = s.type == PCL_CACHE_F32 ? pcl::launch_paged<float>(p, chunks, ctx->stream)
                                           : pcl::launch_paged<__bf16>(p, chunks, ctx->stream);
    if (e == hipSuccess && each > 1)
        e = pcl::launch_paged_combine(p, each, ctx->stream);
    if (e != hipSuccess) {
        std::fprintf(stderr, "pcl_paged_attention: launch: %s\n", hipGetErrorString(e));
        return PCL_NON_FINITE_VALUE;
    }
    return PCL_OK;
}

} // extern "C"
