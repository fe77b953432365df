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
// The lengths live on the device, so the launch is a fixed grid of as many
// workgroups as the device holds at once, which form the chunk counts' sums over
// the requests themselves and take (chunk, KV head, unit of query rows) items
// in turn. Scores: a lane is a key. P.V: a lane is VL output dims, and every wave
// runs the chains of its own dims over the whole chunk. A matrix instruction
// multiplies four query rows with 64 keys or dims, so a decode's few rows per
// KV head do not pay for sixteen. A request of one chunk is written at once; the
// others leave chunk partials in the workspace for paged_combine_kernel.
//
// Bound by HBM where the lengths add up to some hundred MB (MI355X, cold inputs;
// a call with its combine, the figures in brackets without): 64 requests of up
// to 8192 keys, 16 x 8 x 256 heads in bf16, 0.86 GB, 150 us (143: 6.0 TB/s); 16 of
// up to 32768, 16 x 2 x 512, f32, 1.71 GB, 300 us (289: 5.9 TB/s); 32 with a
// 1024-key window, 16 x 8 x 256, f32, 0.54 GB, 96 us (91: 5.9 TB/s); one of 131072,
// 16 x 2 x 512, bf16, 0.54 GB, 109 us (98: 5.5 TB/s, two rounds of items); 256 of
// up to 2048, 32 x 8 x 128, bf16, 0.45 GB, 101 us (95: 4.7 TB/s, most items are
// partial chunks of 128 KiB at most). Below that by the chain of an item: the
// lengths, the table, K, two meetings of the waves, V (one request of 100 keys:
// 11.3 us).
//
// How it came there (the first case): canonical 16 x 16 x 4 MFMAs fed from
// registers 291 us; 4 x 4 x 1 ones, a lane loading its own key's row, 345 us with
// streaming loads (a line was fetched again for each of its eight 16-byte loads,
// 4.6 times the lines) and 209 us with plain ones; the combine's shape 191 us;
// K and V through LDS by 16-byte copies of whole lines (a V row's load by a lane
// a dim cost some 70 cycles of address arithmetic a key) 182 us; nontemporal
// copies 166 us; four waves a workgroup and one buffer each 155 us.
#pragma once

#include "launch.hpp"
#include "paged.hpp"
#include "paged_params.hpp"

#include <algorithm>
#include <atomic>
#include <type_traits>

namespace pcl {

// Words that a workgroup keeps of every request, in dynamic LDS: the chunks
// before it (and the total behind the last), its length and its row.
struct RequestWords {
    uint32_t *off;
    int32_t *len, *row;
};

__device__ __forceinline__ RequestWords request_words(uint32_t *lds, int requests)
{
    int32_t *words = reinterpret_cast<int32_t *>(lds);
    return {lds, words + requests + 1, words + 2 * requests + 1};
}

constexpr size_t request_words_bytes(int requests)
{
    return (3 * (size_t)requests + 1) * sizeof(uint32_t);
}

// Fills them by the whole workgroup; ends with a barrier.
__device__ __forceinline__ void fill_request_words(const PagedParams &p, const RequestWords &r,
                                                   uint32_t *waves)
{
    const int threads = blockDim.x;
    const int per = (p.requests + threads - 1) / threads;
    const int i0 = min((int)threadIdx.x * per, p.requests), i1 = min(i0 + per, p.requests);
    uint32_t sum = 0;
    bool bad = false;
    for (int i = i0; i < i1; ++i) {
        const RequestKeys k = request_keys(p, i, &bad);
        const uint32_t n = request_chunks(k);
        r.off[i] = n;
        r.len[i] = k.len;
        r.row[i] = k.row;
        sum += n;
    }
    uint32_t total;
    uint32_t at = block_offsets(sum, waves, &total);
    for (int i = i0; i < i1; ++i) {
        const uint32_t n = r.off[i];
        r.off[i] = at;
        at += n;
    }
    if (threadIdx.x == 0)
        r.off[p.requests] = total;
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
// canonical chains, at a quarter of its matrix time: the same rate, and no rows
// of the sixteen left unused by four.
template <int BLOCK> __device__ __forceinline__ f4 mfma_rows4(float a, float b, f4 acc)
{
    return __builtin_amdgcn_mfma_f32_4x4x1f32(a, b, acc, 4, BLOCK, 0);
}

// Head dim of the n-th step of the canonical score chain (u, jj, g), and the
// key of a tile at the n-th step of the canonical P.V chain (b, r, g); the
// latter is its own inverse.
__host__ __device__ constexpr int chain_dim(int n)
{
    return 32 * (n / 32) + 8 * (n % 4) + n % 32 / 4;
}

__host__ __device__ constexpr int chain_key(int n)
{
    return (n & 16) + 4 * (n & 3) + (n >> 2 & 3);
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

// A workgroup barrier for LDS contents that leaves loads from memory in flight
// (__syncthreads waits for them too). The empty statements keep the compiler
// from moving memory accesses across it.
__device__ __forceinline__ void lds_barrier()
{
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

typedef uint32_t u4 __attribute__((ext_vector_type(4)));
typedef uint32_t u2 __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) void *lds_ptr;
typedef const __attribute__((address_space(1))) void *global_ptr;

// Cache policy of a copy that is read once (the nontemporal bit): the lines'
// fill takes no place from the partials and the tables. 64 requests of up to
// 8192 keys, 16 x 8 x 256, bf16: 182 -> 166 us; a 1024-key window of 32, f32: 108
// -> 99 us.
constexpr int kStreamed = 2;

// Value j of loaded words, widened to f32.
template <typename T> __device__ __forceinline__ float value_of(const uint32_t *words, int j)
{
    if constexpr (sizeof(T) == 4)
        return __uint_as_float(words[j]);
    else
        return j & 1 ? bf16_high(words[j / 2]) : bf16_low(words[j / 2]);
}

// Shape of a workgroup: NW waves, 64 KG keys scored by each, then the P.V
// chains of 64 VL output dims by each. R sets of four query rows.
//
// K and V reach a wave through a ring of its own in LDS: NB buffers of 8 KiB,
// copied from memory with no register in between, eight loads of 1 KiB each. A
// unit is a 128-byte line of the K rows of 64 keys, or the wave's dims of the V
// rows of kKeysV keys. One buffer where many workgroups share a CU: a unit is
// read into registers, and its buffer filled again, before it is multiplied,
// and less LDS lets more waves cover for each other (64 requests of up to 8192
// keys, 16 x 8 x 256, bf16: 155 us with one, 161 with two, 191 with three
// buffers; one of 131072, 16 x 2 x 512: 109, 127 and 129 us). Two where every
// item has a CU to itself (4 requests of up to 600 keys, 16 x 8 x 256, f32: 24.4
// with one, 20.5 us with two).
template <int DK, typename T, int R> struct PagedCfg {
    static constexpr int NW = DK >= 256 ? 4 : DK / 64;
    static constexpr int VL = DK / 64 / NW;
    static constexpr int KG = 4 / NW;
    static constexpr int kThreads = 64 * NW;
    static constexpr int kLine = 128 / (int)sizeof(T); // dims of a K unit
    static constexpr int KP = DK / kLine;              // K units of a key group
    static constexpr int UK = KG * KP;
    static constexpr int kRowV = 64 * VL * (int)sizeof(T); // bytes of a V row of the wave
    static constexpr int kLanesV = kRowV / 16;             // lanes that copy it
    static constexpr int kKeysV = 8192 / kRowV;
    static constexpr int NQ = R * DK / kThreads; // query quads of a thread
    static constexpr int kRowsUnit = 4 * R;
    static_assert(UK >= 2 && kKeysV >= 16 && kKeysV <= 64, "units of 16 to 64 keys");
};

template <typename C, int NB> constexpr size_t ring_bytes()
{
    return (size_t)C::NW * NB * 8192;
}

// LDS of a workgroup: the query rows and the probabilities in the order in
// which the MFMAs' A registers take them, and each tile's per-row words.
template <int DK, int R> struct PagedLds {
    float q[R][DK][4];                    // [row set][chain step][row]
    float p[R][kTilesPerChunk][kTile][4]; // [row set][tile][chain step][row]
    f4 max[kTilesPerChunk][R], alpha[kTilesPerChunk][R], sum[kTilesPerChunk][R];
    f4 last[R];                           // the chunk's maximum
    int32_t slots[2][kChunk];             // of this item and the next
};

// find_range for a whole wave with one x: the lanes look at 64 offsets at once,
// two LDS round trips instead of one for each bit of n (n at most 64 x 64): 256
// requests of up to 2048 keys 101.4 -> 100.2 us.
__device__ __forceinline__ int find_range_wave(const uint32_t *off, int n, uint32_t x)
{
    static_assert(kMaxRequests <= 64 * 64, "two rounds of 64 offsets");
    const int lane = threadIdx.x & 63;
    const int step = (n + 63) / 64;
    // the samples are ascending: those at or below x come first
    const int i = lane * step;
    const int s = __popcll(__ballot(i < n && off[min(i, n)] <= x)) - 1;
    if (step == 1)
        return s;
    const int j = s * step + lane;
    return s * step + __popcll(__ballot(lane < step && j < n && off[min(j, n)] <= x)) - 1;
}

// A (chunk, KV head, unit of query rows) of one request.
struct PagedItem {
    uint32_t ci; // chunk of the batch
    int b, kh, unit;
    int cbase;   // its first key
    int lo, hi;  // chunk-relative keys [lo, hi] are attended
};

__device__ __forceinline__ PagedItem find_item(const PagedParams &p, const RequestWords &r,
                                               uint32_t item)
{
    const uint32_t per_chunk = (uint32_t)(p.kvheads * p.units);
    PagedItem x;
    x.ci = item / per_chunk;
    const int rest = (int)(item % per_chunk);
    x.kh = rest / p.units;
    x.unit = rest % p.units;
    x.b = __builtin_amdgcn_readfirstlane(find_range_wave(r.off, p.requests, x.ci));
    const int len = __builtin_amdgcn_readfirstlane(r.len[x.b]);
    const int first = first_key(p, len);
    const uint32_t before = __builtin_amdgcn_readfirstlane(r.off[x.b]);
    x.cbase = (first / kChunk + (int)(x.ci - before)) * kChunk;
    x.lo = max(first - x.cbase, 0);
    x.hi = min(len - 1 - x.cbase, kChunk - 1);
    return x;
}

// FULL: the head dim equals the padded head dim DK. Every wave keeps memory
// busy through an item: the next item's pages and query are requested ahead of
// the scores, the first V before the softmax, the next item's K with the last V.
//
// Three waves a SIMD (168 registers, no spill) for four query rows: 1 % faster
// than the two or three that the compiler left room for; eight rows would spill.
template <int DK, typename T, bool FULL, int R, int NB>
__global__ __launch_bounds__((PagedCfg<DK, T, R>::kThreads),
                             (FULL && R == 1 && NB == 1 ? 3 : 1)) void paged_kv_kernel(PagedParams p)
{
    using C = PagedCfg<DK, T, R>;
    constexpr int KG = C::KG, KP = C::KP, UK = C::UK, VL = C::VL, NQ = C::NQ;
    __shared__ __attribute__((aligned(16))) PagedLds<DK, R> s;
    __shared__ uint32_t waves[C::NW];
    extern __shared__ __attribute__((aligned(16))) uint32_t dyn[];
    const RequestWords req = request_words(dyn + ring_bytes<C, NB>() / 4, p.requests);
    const int tid = threadIdx.x;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int lane = tid & 63;

    fill_request_words(p, req, waves);
    if (blockIdx.x == 0)
        for (int i = tid; i < p.requests; i += C::kThreads)
            p.ws_req[i] = int4{(int)req.off[i], (int)(req.off[i + 1] - req.off[i]),
                               first_key(p, req.len[i]) / kChunk, req.row[i]};
    const uint32_t items = __builtin_amdgcn_readfirstlane(req.off[p.requests]) *
                           (uint32_t)(p.kvheads * p.units);
    if (blockIdx.x >= items)
        return;

    // An item's page numbers of the thread's keys and its part of the unit's
    // query rows, requested (fetch) and then left in LDS (store).
    struct Fetched {
        int page[KG];
        f4 q[NQ];
    };
    // a key outside [lo, hi] reads the nearest one inside (its score and
    // probability are not used)
    auto position = [&](const PagedItem &x, int kg) {
        const int key = 64 * (w * KG + kg) + lane;
        return (uint32_t)(x.cbase + min(max(key, x.lo), x.hi));
    };
    auto fetch = [&](const PagedItem &x, Fetched &f) {
#pragma unroll
        for (int kg = 0; kg < KG; ++kg)
            f.page[kg] = p.table[x.b * p.table_stride + position(x, kg) / p.page_tokens];
        const int row = __builtin_amdgcn_readfirstlane(req.row[x.b]);
        const int h0 = x.kh * p.group + x.unit * C::kRowsUnit;
        const int nrows = min(p.group - x.unit * C::kRowsUnit, C::kRowsUnit);
        const float *q = p.q + row * p.q_stride + (int64_t)h0 * p.dim;
#pragma unroll
        for (int i = 0; i < NQ; ++i) {
            const int r = (tid + C::kThreads * i) / (DK / 4);
            const int d = 4 * ((tid + C::kThreads * i) % (DK / 4));
            f.q[i] = ldg4(q + (r < nrows && (FULL || d < p.dim) ? r * p.dim + d : 0));
        }
    };
    auto store = [&](const PagedItem &x, const Fetched &f, int32_t *slots) {
#pragma unroll
        for (int kg = 0; kg < KG; ++kg) {
            int page = f.page[kg];
            if (page < 0 || page >= p.pages) {
                atomicOr(p.err, kErrPages);
                page = 0;
            }
            slots[64 * (w * KG + kg) + lane] =
                page * (int32_t)p.page_tokens + (int32_t)(position(x, kg) % p.page_tokens);
        }
        // scaled; zero past the group and the head dim
        const int nrows = min(p.group - x.unit * C::kRowsUnit, C::kRowsUnit);
#pragma unroll
        for (int i = 0; i < NQ; ++i) {
            const int r = (tid + C::kThreads * i) / (DK / 4);
            const int d = 4 * ((tid + C::kThreads * i) % (DK / 4));
            const bool in = r < nrows && (FULL || d < p.dim);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int k = d % 32 + e; // 8 g + jj
                s.q[r / 4][(d & ~31) + 4 * (k % 8) + k / 8][r % 4] =
                    in ? f.q[i][e] * p.q_scale : 0.f;
            }
        }
    };
    // The wave's ring: buffer `at` takes the unit issued next and holds, until
    // then, the one consumed next. Exactly one unit is issued for each one
    // consumed, so NB - 1 of them are behind the one waited for.
    uint32_t *const ring = dyn + (size_t)w * NB * 2048;
    int at = 0;
    const uint32_t row_bytes = (uint32_t)(p.row_stride * sizeof(T));
    // Where a unit's eight copies read.
    struct Sources {
        const char *from[8];
    };
    // Key group kg's K rows 8 e + lane / 8, each at the lane's 16-byte piece of the
    // line's: the pieces of row r lie in the order piece ^ (r & 7), so that a
    // lane's reads of its own row fall in other banks than its neighbours'.
    const int piece = (lane % 8 ^ lane / 8) * (16 / (int)sizeof(T));
    auto rows_k = [&](const int32_t *slots, int kh, int kg) {
        const char *base =
            static_cast<const char *>(p.k) + ((int64_t)kh * p.dim + piece) * sizeof(T);
        const int32_t *mine = slots + 64 * (w * KG + kg) + lane / 8;
        Sources c;
#pragma unroll
        for (int e = 0; e < 8; ++e)
            c.from[e] = base + (uint64_t)(uint32_t)mine[8 * e] * row_bytes;
        return c;
    };
    // line `line` of those rows (a piece past the head dim: the row's first one)
    auto line_k = [&](const Sources &rows, int line) {
        const int d = C::kLine * line;
        const int64_t step = (FULL || d + piece < p.dim ? d : -piece) * (int64_t)sizeof(T);
        Sources c;
#pragma unroll
        for (int e = 0; e < 8; ++e)
            c.from[e] = rows.from[e] + step;
        return c;
    };
    // V unit i of the tiles from t0 to t1 (past them the last tile again): its
    // keys in the order of the P.V chain
    auto sources_v = [&](const int32_t *slots, int kh, int t0, int t1, int i) {
        const int d = 64 * VL * w + lane % C::kLanesV * (16 / (int)sizeof(T));
        const char *base = static_cast<const char *>(p.v) +
                           ((int64_t)kh * p.dim + (FULL || d < p.dim ? d : 0)) * sizeof(T);
        Sources c;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const int n = C::kKeysV * i + (e * 64 + lane) / C::kLanesV; // chain step from tile t0 on
            const int t = min(t0 + n / kTile, t1), k = n % kTile;
            c.from[e] = base + (uint64_t)(uint32_t)slots[kTile * t + chain_key(k)] * row_bytes;
        }
        return c;
    };
    auto issue = [&](const Sources &c) {
#pragma unroll
        for (int e = 0; e < 8; ++e)
            __builtin_amdgcn_global_load_lds((global_ptr)c.from[e],
                                             (lds_ptr)(ring + at * 2048 + e * 256), 16, 0,
                                             kStreamed);
    };
    // the consumed unit's contents are there; then, read, its buffer is free
    auto wait_unit = [&]() {
        __builtin_amdgcn_s_waitcnt(waitcnt_vm(8 * (NB - 1)));
        asm volatile("" ::: "memory");
    };
    auto free_unit = [&]() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); };

    PagedItem x = find_item(p, req, blockIdx.x);
    {
        Fetched f;
        fetch(x, f);
        store(x, f, s.slots[0]);
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < NB; ++i, at = at + 1 == NB ? 0 : at + 1)
        issue(line_k(rows_k(s.slots[0], x.kh, i / KP), i % KP));

    int buf = 0;
    for (uint32_t item = blockIdx.x;; buf ^= 1) {
        const uint32_t next = item + gridDim.x;
        const bool more = next < items;
        // (without a next item this one is requested again, and not used)
        const PagedItem y = find_item(p, req, more ? next : item);
        Fetched f;
        fetch(y, f);
        const int h0 = x.kh * p.group + x.unit * C::kRowsUnit;
        const int nrows = min(p.group - x.unit * C::kRowsUnit, C::kRowsUnit);
        const int t0 = x.lo / kTile, t1 = x.hi / kTile; // tiles with attended keys

        // scores: lane = key
        f4 acc[KG][R];
        bool bad = false;
        // The copies behind a consumed unit go out once it is read, from sources
        // worked out during the unit before; the query is read ahead of the wait
        // (16 requests of up to 8192 keys, 32 query heads and one KV head of 128
        // dims, bf16: 50 -> 42 us; one request of 300 keys, 16 x 2 x 512: 32 -> 31).
        Sources rows = rows_k(s.slots[buf], x.kh, NB / KP % KG);
        Sources c = NB < UK ? line_k(rows, NB % KP) : sources_v(s.slots[buf], x.kh, t0, t1, 0);
        each<UK>([&](auto ic) {
            constexpr int i = decltype(ic)::value, kg = i / KP, M = C::kLine / 16;
            const int k0 = 64 * (w * KG + kg);
            if (i % KP == 0) {
#pragma unroll
                for (int r = 0; r < R; ++r)
                    acc[kg][r] = f4{0.f, 0.f, 0.f, 0.f};
            }
            float a[M][R];
#pragma unroll
            for (int m = 0; m < M; ++m)
#pragma unroll
                for (int r = 0; r < R; ++r)
                    a[m][r] = s.q[r][C::kLine * (i % KP) + 16 * m + lane / 4][lane % 4];
            wait_unit();
            uint32_t kw[32];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const u4 v = *(const u4 *)(ring + at * 2048 + 32 * lane + 4 * (j ^ (lane & 7)));
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    kw[4 * j + e] = FULL || C::kLine * (i % KP) + j * (16 / (int)sizeof(T)) < p.dim
                                        ? v[e]
                                        : 0u;
            }
            free_unit();
            issue(c);
            at = at + 1 == NB ? 0 : at + 1;
            constexpr int n1 = i + 1 + NB; // the unit that the next consumed one makes room for
            if constexpr (i + 1 < UK) {
                if constexpr (n1 < UK) {
                    if constexpr (n1 % KP == 0)
                        rows = rows_k(s.slots[buf], x.kh, n1 / KP);
                    c = line_k(rows, n1 % KP);
                } else {
                    c = sources_v(s.slots[buf], x.kh, t0, t1, n1 - UK);
                }
            }
            if (k0 <= x.hi && k0 + 63 >= x.lo) {
                each<M>([&](auto mc) {
                    constexpr int m = decltype(mc)::value;
                    each<16>([&](auto nc) {
                        constexpr int n = decltype(nc)::value;
                        const float k = value_of<T>(kw, chain_dim(16 * m + n));
#pragma unroll
                        for (int r = 0; r < R; ++r)
                            acc[kg][r] = mfma_rows4<n>(a[m][r], k, acc[kg][r]);
                    });
                });
            }
        });

#pragma unroll
        for (int kg = 0; kg < KG; ++kg) {
            const int k0 = 64 * (w * KG + kg);
            if (k0 > x.hi || k0 + 63 < x.lo)
                continue;
            const int key = k0 + lane;
            const bool ok = key >= x.lo && key <= x.hi;
#pragma unroll
            for (int r = 0; r < R; ++r) {
                f4 tm;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    float v = acc[kg][r][e];
                    v = p.softcap > 0.f ? soft_cap(v, p.softcap, p.inv_softcap) : v;
                    bad |= ok && 4 * r + e < nrows && !is_finite(v);
                    v = ok ? v : kNegInf;
                    acc[kg][r][e] = v;
                    tm[e] = max_tile(v);
                }
                if ((lane & 31) == 0)
                    s.max[key / kTile][r] = tm;
            }
        }
        if (bad)
            atomicOr(p.err, kErrScore);
        lds_barrier(); // every tile's maximum; the query is used

        // probabilities against the running maximum at the lane's tile
#pragma unroll
        for (int kg = 0; kg < KG; ++kg) {
            const int k0 = 64 * (w * KG + kg);
            if (k0 > x.hi || k0 + 63 < x.lo)
                continue;
            const int key = k0 + lane, t = key / kTile;
            const bool ok = key >= x.lo && key <= x.hi;
#pragma unroll
            for (int r = 0; r < R; ++r) {
                f4 before, m; // running maxima before and at the tile
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    before[e] = kNegInf;
                for (int i = t0; i < k0 / kTile; ++i) {
                    const f4 v = s.max[i][r];
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        before[e] = fmaxf(before[e], v[e]);
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
                *(f4 *)s.p[r][t][chain_key(key % kTile)] = pr;
                if ((lane & 31) == 0) {
                    s.alpha[t][r] = alpha;
                    s.sum[t][r] = sum;
                }
                // the last tile's running maximum is the chunk's
                if (t == t1 && (lane & 31) == 0)
                    s.last[r] = m;
            }
        }
        store(y, f, s.slots[buf ^ 1]);
        lds_barrier(); // probabilities, row sums and factors; the next query

        // the l chain and the P.V chains of the lane's VL output dims
        f4 l[R], O[R][VL];
#pragma unroll
        for (int r = 0; r < R; ++r) {
            l[r] = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int v = 0; v < VL; ++v)
                O[r][v] = f4{0.f, 0.f, 0.f, 0.f};
        }
        // 16 chain steps of tile t, its first or second half; a: their
        // probabilities, word(n): the words of step n
        auto attend = [&](int t, int half, const float (&a)[R], auto word) {
            if (half == 0) {
#pragma unroll
                for (int r = 0; r < R; ++r) {
                    const f4 alpha = s.alpha[t][r], sum = s.sum[t][r];
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        l[r][e] = __builtin_fmaf(l[r][e], alpha[e], sum[e]);
#pragma unroll
                    for (int j = 0; j < VL; ++j)
                        O[r][j] = O[r][j] * alpha;
                }
            }
            each<16>([&](auto nc) {
                constexpr int n = decltype(nc)::value;
                const uint32_t *v = word(n);
#pragma unroll
                for (int j = 0; j < VL; ++j)
#pragma unroll
                    for (int r = 0; r < R; ++r)
                        O[r][j] = mfma_rows4<n>(a[r], value_of<T>(v, j), O[r][j]);
            });
        };
        constexpr int WV = (VL * (int)sizeof(T) + 3) / 4; // words of a lane's values
        const int units = ((t1 - t0 + 1) * kTile + C::kKeysV - 1) / C::kKeysV;
        const int rounds = max(units, NB);
        // the unit that V unit i makes room for
        auto behind_v = [&](int i) {
            const int n = i + NB - rounds; // the next item's first units follow this one's
            return n < 0 ? sources_v(s.slots[buf], x.kh, t0, t1, i + NB)
                         : line_k(rows_k(s.slots[buf ^ 1], y.kh, n / KP), n % KP);
        };
        c = behind_v(0);
        for (int i = 0; i < rounds; ++i) {
            float a[C::kKeysV / 16][R];
#pragma unroll
            for (int h = 0; h < C::kKeysV / 16; ++h) {
                const int n = C::kKeysV * i + 16 * h, t = min(t0 + n / kTile, t1);
#pragma unroll
                for (int r = 0; r < R; ++r)
                    a[h][r] = s.p[r][t][n % kTile + lane / 4][lane % 4];
            }
            wait_unit();
            uint32_t vw[C::kKeysV][WV];
#pragma unroll
            for (int n = 0; n < C::kKeysV; ++n) {
                const char *row = reinterpret_cast<const char *>(ring + at * 2048) + n * C::kRowV;
                if constexpr (WV == 2) {
                    const u2 v = *(const u2 *)(row + 8 * lane);
                    vw[n][0] = v.x;
                    vw[n][1] = v.y;
                } else if constexpr (VL * sizeof(T) == 4) {
                    vw[n][0] = *(const uint32_t *)(row + 4 * lane);
                } else {
                    vw[n][0] = *(const uint16_t *)(row + 2 * lane);
                }
            }
            free_unit();
            issue(c);
            at = at + 1 == NB ? 0 : at + 1;
            if (i + 1 < rounds)
                c = behind_v(i + 1);
            if (i < units) {
#pragma unroll
                for (int h = 0; h < C::kKeysV / 16; ++h) {
                    const int n = C::kKeysV * i + 16 * h, t = t0 + n / kTile;
                    if (C::kKeysV > kTile && t > t1)
                        continue;
                    const int half = C::kKeysV < kTile ? i % 2 : h % 2;
                    attend(t, half, a[h], [&](int k) { return vw[16 * h + k]; });
                }
            }
        }

        const int vd = (64 * w + lane) * VL;
        const bool only = req.off[x.b + 1] - req.off[x.b] == 1; // the request's only chunk
        bool nonfinite = false;
        if (FULL || vd < p.dim) {
#pragma unroll
            for (int r = 0; r < R; ++r)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    if (4 * r + e >= nrows)
                        continue;
                    const int h = h0 + 4 * r + e;
                    const int64_t part = (int64_t)x.ci * p.qheads + h;
                    float *dst = only ? p.out + req.row[x.b] * p.o_stride + (int64_t)h * p.dim + vd
                                      : p.ws_o + part * p.dim + vd;
#pragma unroll
                    for (int j = 0; j < VL; ++j) {
                        const float v = only ? O[r][j][e] / l[r][e] : O[r][j][e];
                        nonfinite |= only && !is_finite(v);
                        stg(dst + j, v);
                    }
                    if (!only && w == 0 && lane == 0) {
                        stg(p.ws_ml + 2 * part, s.last[r][e]);
                        stg(p.ws_ml + 2 * part + 1, l[r][e]);
                    }
                }
        }
        if (nonfinite)
            atomicOr(p.err, kErrOutput);
        if (!more)
            break;
        item = next;
        x = y;
    }
    // no copy may land in LDS that another workgroup owns by then
    __builtin_amdgcn_s_waitcnt(waitcnt_vm(0));
}

// Workgroups of a kernel that a CU holds at once, for batches of up to
// kFewRequests (asked once per device) and for larger ones (asked per call:
// the request words take more LDS).
constexpr int kFewRequests = 256;

template <int DK, typename T, bool FULL, int R, int NB>
static hipError_t resident_groups(int requests, int *groups)
{
    using C = PagedCfg<DK, T, R>;
    const auto kernel = (const void *)paged_kv_kernel<DK, T, FULL, R, NB>;
    static std::atomic<int> known[kMaxDevices];
    int dev = 0;
    hipError_t e = hipGetDevice(&dev);
    if (e != hipSuccess)
        return e;
    if (dev < 0 || dev >= kMaxDevices)
        return hipErrorInvalidDevice;
    *groups = known[dev].load(std::memory_order_acquire);
    if (*groups > 0 && requests <= kFewRequests)
        return hipSuccess;
    constexpr size_t ring = ring_bytes<C, NB>();
    static_assert(sizeof(PagedLds<DK, R>) + 64 + ring + request_words_bytes(kMaxRequests) <=
                      160 * 1024,
                  "the LDS of a CU");
    if (*groups == 0) {
        // more than 64 KiB of LDS in all must be allowed once per device
        e = hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize,
                                (int)(ring + request_words_bytes(kMaxRequests)));
        if (e != hipSuccess)
            return e;
    }
    const int most = requests <= kFewRequests ? kFewRequests : requests;
    e = hipOccupancyMaxActiveBlocksPerMultiprocessor(groups, kernel, C::kThreads,
                                                     ring + request_words_bytes(most));
    if (e != hipSuccess)
        return e;
    *groups = std::max(*groups, 1);
    if (requests <= kFewRequests)
        known[dev].store(*groups, std::memory_order_release);
    return hipSuccess;
}

template <int DK, typename T, bool FULL, int R, int NB>
static hipError_t launch_paged(const PagedParams &p, int64_t items, hipStream_t stream)
{
    using C = PagedCfg<DK, T, R>;
    int groups = 0;
    const hipError_t e = resident_groups<DK, T, FULL, R, NB>(p.requests, &groups);
    if (e != hipSuccess)
        return e;
    const int64_t grid = std::min<int64_t>(items, (int64_t)groups * std::max(device_cus(), 1));
    paged_kv_kernel<DK, T, FULL, R, NB>
        <<<(unsigned)grid, C::kThreads, ring_bytes<C, NB>() + request_words_bytes(p.requests),
           stream>>>(p);
    return hipGetLastError();
}

template <int DK, typename T, bool FULL, int R>
static hipError_t launch_paged(PagedParams p, int64_t chunks, hipStream_t stream)
{
    p.units = (p.group + PagedCfg<DK, T, R>::kRowsUnit - 1) / PagedCfg<DK, T, R>::kRowsUnit;
    // (the items at the requests' longest)
    const int64_t items = chunks * p.kvheads * p.units;
    if constexpr (FULL && R <= 2) {
        if (items <= device_cus())
            return launch_paged<DK, T, FULL, R, 2>(p, items, stream);
    }
    return launch_paged<DK, T, FULL, R, 1>(p, items, stream);
}

template <int DK, typename T, bool FULL>
static hipError_t launch_paged(const PagedParams &p, int64_t chunks, hipStream_t stream)
{
    return p.group <= 4   ? launch_paged<DK, T, FULL, 1>(p, chunks, stream)
           : p.group <= 8 ? launch_paged<DK, T, FULL, 2>(p, chunks, stream)
                          : launch_paged<DK, T, FULL, 4>(p, chunks, stream);
}

template <int DK, typename T>
static hipError_t launch_paged(const PagedParams &p, int64_t chunks, hipStream_t stream)
{
    return p.dim == DK ? launch_paged<DK, T, true>(p, chunks, stream)
                       : launch_paged<DK, T, false>(p, chunks, stream);
}

template <int DK>
hipError_t launch_paged_kv(const PagedParams &p, bool bf16, int64_t chunks, hipStream_t stream)
{
    return bf16 ? launch_paged<DK, __bf16>(p, chunks, stream)
                : launch_paged<DK, float>(p, chunks, stream);
}

} // namespace pcl
