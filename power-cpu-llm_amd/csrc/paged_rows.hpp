// Attention of a step's new tokens over a paged KV cache where a KV head has more
// than eight query rows: units of 16 U rows, 256-key chunks, on 16 x 16 x 4 f32 MFMAs.
//
// For new token i of request b (L held tokens, row r), query head h of KV head kh:
//   s_t = cap(q_scale * q[r][h] . K[slot_t][kh])  over the keys t that it attends,
//   out[r][h] = sum_t exp(s_t - max s) V[slot_t][kh] / sum_t exp(s_t - max s),
// keys [0, L + i], or with masks [0, L) and L + j for each bit j; in a window those
// less than `window` positions before it. The arithmetic is that of paged_kv.hpp.
//
// Eight waves (four below head dim 256) score 32 keys (64) each against all the
// unit's rows and leave the probabilities in LDS; then each runs the P.V chains of its
// share of the dims over the whole chunk. So each byte of K and V is read from LDS
// once, by one wave, and feeds U instructions of 16 rows; a lane of the result is a
// row, and a tile's maximum and sum take two exchanges between lanes (a lane a key, as
// in paged_kv.hpp, takes five). The probabilities of all waves meet in LDS: three
// barriers a chunk.
//
// Bound by the matrix instructions and the phases between them (MI355X, cold inputs;
// calls in a row, each with its plan and merge, and in brackets the multiply-adds of
// whole units at 154 TFLOP/s, which a large f32 product of the library reaches):
//   64 trees of up to 8 over up to 8192 keys, 16 x 8 x 256 heads, bf16, 0.86 GB: 246 us
//     (96), matrix pipes 47 % busy; 203 us where all pages are the same one;
//   32 trees of up to 24, 1024-key window, 16 x 8 x 256, f32, 0.54 GB: 193 us (106);
//   16 trees of up to 12 over up to 32K keys, 16 x 2 x 512, f32, 1.7 GB: 897 us (537);
//   256 chains of up to 4 over up to 2048 keys, 32 x 8 x 128, bf16, 0.44 GB: 165 us (62);
//   4 prompt parts of up to 512 over up to 8192 keys, 16 x 8 x 256, bf16: 1.87 ms (1.16).
// The launch's words, two items and two chunks' words take more scalar registers than a
// wave has: 136 to 208 of them lie in lanes of vector registers.
// Of a chunk at 48 rows the scores take 43 % (83 % of it matrix instructions), the
// softmax 10 %, P.V 45 % (79 %) and the output 2 %.
//
// How it came there (the first, fourth and last case): units of 16 rows on 4 x 4 x 1
// MFMAs 298, - and 3164 us; 16 x 16 x 4 on four waves 227, 180 and 2385 us; eight waves,
// with which two workgroups have a CU's registers at one 16 of rows, and the query
// copied into LDS as it is, 222, 168 and 2054 us; a chunk's softmax from one read of
// its maxima and items as workgroups come to them 237, 170 and 1881 us with their plan;
// whole spans as items 248, 173 and 1857 us (the third case 1002 -> 882 us), half lines
// of K up to head dim 128 165 us; an item's claim and the next chunk's words behind the
// scores 245 and 162 us (246, 165 and 1868 since, the third case 897).
#pragma once

#include "paged_kv.hpp"

namespace pcl {

// Units of the ring that a wave's part of a K line comes in, and units that the ring
// holds. Up to head dim 128 a wave has 64 keys: a unit is 32 of them, so that fewer
// registers hold a unit's values (64 rows spilled 157 of them with whole lines, 74 with
// halves), and a ring of three keeps more copies in flight at 128 (256 chains of up to 4,
// 16 rows, 173 us with whole lines, 165 with halves; prompt parts of 512 tokens at 32 x 8
// x 128, bf16, 2237 us with two halves, 2129 with three; at 64 as fast, and 32 rows have
// two workgroups a CU with two). Above, halves cost more than they bring (window trees
// 194 -> 210 us, prompt parts 1857 -> 1925 us with three of them).
constexpr int rows_parts(int dk)
{
    return dk <= 128 ? 2 : 1;
}

constexpr int rows_buffers(int dk)
{
    return dk == 128 ? 3 : rows_parts(dk);
}

// Eight waves of 32 keys at head dims 256 and 512, four of 64 below (a wave's part of
// a V row is 16 dims at least; four waves at 256 took 2385 us for the prompt parts).
// Units of the ring are a 128-byte line of the wave's K rows, or of half of them, or its
// dims of some V rows.
template <int DK, typename T, int U> struct RowsCfg {
    static constexpr int NW = DK >= 256 ? 8 : 4;
    static constexpr int kThreads = 64 * NW;
    static constexpr int kRowsUnit = 16 * U;
    static constexpr int KW = kChunk / NW;             // keys of a wave
    static constexpr int TW = KW / kTile;              // tiles of them
    static constexpr int kParts = rows_parts(DK);      // K units of a line
    static constexpr int BU = KW / 16 / kParts;        // 16-key blocks of one
    static constexpr int kUnit = 128 * 16 * BU;        // bytes of a ring unit
    static constexpr int NE = kUnit / 1024;            // copies of one
    static constexpr int kLine = 128 / (int)sizeof(T); // dims of a K unit
    static constexpr int kLines = (DK + kLine - 1) / kLine;
    static constexpr int UK = kLines * kParts;         // K units
    static constexpr int SU = kLine / 32;              // score chain steps (32 dims) of a unit
    static constexpr int VL = DK / 16 / NW;            // 16-dim blocks of a wave's dims
    static constexpr int kRowV = 16 * VL * (int)sizeof(T); // bytes of a V row of the wave
    static constexpr int kLanesV = kRowV / 16;         // lanes that copy it
    static constexpr int kKeysV = kUnit / kRowV < kChunk ? kUnit / kRowV : kChunk;
    static_assert(kKeysV >= 16, "units of 16 keys and more");
    static_assert(VL == 1 || VL == 2 || VL == 4, "a lane's values are one read");
};

template <int DK, int U> struct RowsLds {
    f4 q[U][DK / 32][2][64];              // [rows][32 dims][half of a lane's eight][lane]
    f4 p[U][kTilesPerChunk][2][64];       // [rows][tile][16 keys][lane]
    float max[16 * U][kTilesPerChunk];    // -inf outside the attended tiles
    f2 factors[kTilesPerChunk][16 * U];   // alpha and the row sum
    int32_t slots[2][kChunk];             // of this chunk and the next
    int32_t live[2][kTilesPerChunk];      // tiles with a key that any row attends
    uint32_t taken;                       // the item behind the next one
    uint32_t part; // whose items the workgroup takes (a register's use costs spills)
};

// The LDS of a CU, less the kernel's static words.
constexpr size_t kRowsLds = 160 * 1024 - 64;

template <int DK, typename T, int U, int NB> constexpr size_t rows_lds_bytes()
{
    return sizeof(RowsLds<DK, U>) + (size_t)NB * RowsCfg<DK, T, U>::kUnit * RowsCfg<DK, T, U>::NW;
}

// What a lane requests of an item's trees: of its row in each 16 of the unit's the
// 64 mask bits of the wave's keys (two words) and the position; and of its key.
template <int U> struct RowsFetched {
    uint64_t mask[U][2];
    int position[U], key;
};

// The lane's row in 16 rows rg of the unit: the new token (the last one's past the
// rows).
__device__ __forceinline__ int row_token(const TreeParams &p, const TreeItem &x, int rg)
{
    return (int)divided(x.first_row + min(16 * rg + (int)(threadIdx.x & 15), x.nrows - 1),
                        p.by_group);
}

template <int U>
__device__ __forceinline__ void fetch_rows(const TreeParams &p, const TreeItem &x, int k0,
                                           RowsFetched<U> &f)
{
#pragma unroll
    for (int rg = 0; rg < U; ++rg) {
        f.mask[rg][0] = f.mask[rg][1] = 0;
        f.position[rg] = 0;
    }
    f.key = 0;
    if (!p.masks)
        return;
    const int n0 = x.cbase + k0 - x.held; // new token of the wave's first key
    if (n0 + 63 >= 0 && n0 < x.n) {
        const int w0 = n0 < 0 ? -1 : n0 / 64;
#pragma unroll
        for (int rg = 0; rg < U; ++rg) {
            if (16 * rg >= x.nrows)
                continue;
            const uint64_t *row =
                p.masks + (int64_t)(x.row + row_token(p, x, rg)) * p.mask_words;
#pragma unroll
            for (int h = 0; h < 2; ++h)
                if (w0 + h >= 0 && w0 + h < p.mask_words)
                    f.mask[rg][h] = row[w0 + h];
        }
    }
    if (!p.window)
        return;
#pragma unroll
    for (int rg = 0; rg < U; ++rg)
        if (16 * rg < x.nrows)
            f.position[rg] = p.positions[x.row + row_token(p, x, rg)];
    const int n = n0 + (int)(threadIdx.x & 63);
    if (n >= 0 && n < x.n)
        f.key = p.positions[x.row + n];
}

// Bits [lo, hi] of 64 (none where hi < lo; lo and hi any).
__device__ __forceinline__ uint64_t bit_range(int lo, int hi)
{
    lo = max(lo, 0);
    hi = min(hi, 63);
    return hi < lo ? 0 : ~(uint64_t)0 >> (63 - (hi - lo)) << lo;
}

// The wave's keys k0 .. k0 + 63 that the lane's rows attend, bit k for key k0 + k.
template <int U>
__device__ __forceinline__ void attended_keys(const TreeParams &p, const TreeItem &x, int k0,
                                              const RowsFetched<U> &f, uint64_t (&see)[U])
{
    const int n0 = x.cbase + k0 - x.held;
    const uint64_t in = x.empty ? 0 : bit_range(x.lo - k0, x.hi - k0);
    const uint64_t held = bit_range(0, -n0 - 1); // keys held before the step
#pragma unroll
    for (int rg = 0; rg < U; ++rg) {
        see[rg] = 0;
        if (16 * rg >= x.nrows)
            continue;
        const int token = row_token(p, x, rg); // (past the rows the last one's again)
        if (!p.masks) {
            const int to = x.held + token, from = first_tree_key(p, to);
            see[rg] = in & bit_range(from - x.cbase - k0, to - x.cbase - k0);
            continue;
        }
        // the mask's bits from n0 on
        const int s = n0 & 63;
        const uint64_t bits =
            s ? f.mask[rg][0] >> s | f.mask[rg][1] << (64 - s) : f.mask[rg][0];
        see[rg] = in & (held | (bits & ~held));
        if (p.window)
            see[rg] &= ~held | bit_range(first_tree_key(p, f.position[rg]) - x.cbase - k0, 63);
    }
    // a window that is shorter than the trees
    if (p.masks && p.window && x.n > p.window && n0 + 63 >= 0) {
        for (int k = max(-n0, 0); k < 64; ++k) {
            const int at = __builtin_amdgcn_readlane(f.key, k);
#pragma unroll
            for (int rg = 0; rg < U; ++rg)
                if (f.position[rg] - at >= p.window)
                    see[rg] &= ~((uint64_t)1 << k);
        }
    }
}

// The bits that any lane with another lane % 16 has, on all of them.
__device__ __forceinline__ uint32_t or_rows(uint32_t x)
{
    x |= __builtin_amdgcn_update_dpp(0, x, kDppXor1, 0xf, 0xf, true);
    x |= __builtin_amdgcn_update_dpp(0, x, kDppXor2, 0xf, 0xf, true);
    x |= __builtin_amdgcn_update_dpp(0, x, kDppMirror8, 0xf, 0xf, true);
    x |= __builtin_amdgcn_update_dpp(0, x, kDppMirror16, 0xf, 0xf, true);
    return x;
}

// The items of a launch. A span of a request, over a unit, is one item while that
// leaves the workgroups evenly loaded: its chunks are merged in registers, in their
// order, and it leaves one partial (none where it is all of the request). The rest are
// items of a chunk each, which come last and fill what the spans leave uneven: with T
// chunks in all, W workgroups and no span longer than s chunks, the spans are the first
// W (where T >= s W) and those that begin in the first T - s W chunks. With the combine,
// against a chunk each (MI355X): trees of 12 tokens behind up to 32K keys of d512 (T = 19
// W) 0.89 and 0.99 ms, prompt parts of 512 tokens (T = 55 W) 1.86 and 1.91 ms, at 32 x 8 x
// 128 2.13 and 2.35 ms. (W floor(T / (s W)) spans left workgroups unevenly loaded: 2.01
// ms; spans in the first T - s W / 2 chunks as well, 2.03 ms, and 257 us instead of 194
// for windows of T = 5 W; in the first T - 2 s W 1.83 and 2.20 ms.)
constexpr int kPlanThreads = 256;

// The requests' words: items of spans and of chunks before each (over the KV heads),
// its tokens with the step's and without, its first row, and its first chunk that is
// an item of its own.
struct PlanWords {
    uint32_t *spans, *singles;
    int32_t *len, *held, *row, *split;
};

constexpr size_t plan_words_bytes(int requests)
{
    return (6 * (size_t)requests + 2) * sizeof(uint32_t);
}

// The last request of [0, requests) whose items begin at n or before it.
__device__ __forceinline__ int plan_request(const uint32_t *off, int requests, uint32_t n)
{
    int lo = 0;
    for (int hi = requests; hi - lo > 1;) {
        const int mid = (lo + hi) / 2;
        if (off[mid] <= n)
            lo = mid;
        else
            hi = mid;
    }
    return lo;
}

// block_offsets of two values, and b's total.
__device__ __forceinline__ void block_offsets2(uint64_t a, uint64_t b,
                                               uint64_t (&waves)[2][kPlanThreads / 64],
                                               uint64_t *a_at, uint64_t *b_at, uint64_t *total)
{
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    uint64_t x = a, y = b;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const uint64_t xo = __shfl_up(x, o), yo = __shfl_up(y, o);
        if (lane >= o) {
            x += xo;
            y += yo;
        }
    }
    if (lane == 63) {
        waves[0][wave] = x;
        waves[1][wave] = y;
    }
    __syncthreads();
    x -= a;
    y -= b;
    *total = 0;
#pragma unroll
    for (int i = 0; i < kPlanThreads / 64; ++i) {
        x += i < wave ? waves[0][i] : 0;
        y += i < wave ? waves[1][i] : 0;
        *total += waves[1][i];
    }
    __syncthreads();
    *a_at = x;
    *b_at = y;
}

template <int UNIT>
__global__ __launch_bounds__(kPlanThreads) void paged_plan_kernel(TreeParams p, int workgroups)
{
    extern __shared__ uint32_t dyn[];
    __shared__ uint64_t waves[2][kPlanThreads / 64];
    __shared__ int longest;
    const int n = p.requests;
    int32_t *words = reinterpret_cast<int32_t *>(dyn) + 2 * (n + 1);
    const PlanWords r = {dyn, dyn + n + 1, words, words + n, words + 2 * n, words + 3 * n};
    const int tid = threadIdx.x;
    const int per = (n + kPlanThreads - 1) / kPlanThreads;
    const int i0 = min(tid * per, n), i1 = min(i0 + per, n);
    const uint32_t kvheads = (uint32_t)p.kvheads;
    auto units_of = [&](int m) { return ((uint32_t)m * (uint32_t)p.group + UNIT - 1) / UNIT; };
    auto spans_of = [](int first, int chunks) {
        return chunks ? (first + chunks - 1) / kSpanChunks - first / kSpanChunks + 1 : 0;
    };
    if (tid == 0)
        longest = 1;
    __syncthreads();
    uint64_t chunk_sum = 0, span_sum = 0; // (requests that share rows may add up past 2^32)
    bool bad = false;
    int most = 0;
    for (int i = i0; i < i1; ++i) {
        const TreeKeys k = tree_keys(p, i, &bad);
        r.len[i] = k.len;
        r.held[i] = k.held;
        r.row[i] = k.row;
        const int chunks = tree_chunks(p, k), first = first_tree_key(p, k.held) / kChunk;
        const int spans = spans_of(first, chunks);
        chunk_sum += (uint64_t)chunks * units_of(k.len - k.held) * kvheads;
        span_sum += (uint64_t)spans * units_of(k.len - k.held) * kvheads;
        const int begin = min(kSpanChunks - first % kSpanChunks, chunks);
        most = max(most, spans > 2 ? kSpanChunks : max(begin, chunks - begin));
    }
    if (most > 1)
        atomicMax(&longest, most);
    uint64_t spans_at, chunks_at, total; // (barriers: longest)
    block_offsets2(span_sum, chunk_sum, waves, &spans_at, &chunks_at, &total);
    const bool fits = total <= (uint64_t)p.max_items;
    bad |= !fits;
    const uint64_t round = (uint64_t)longest * (uint32_t)workgroups;
    const uint64_t by_count = total >= round ? (uint32_t)workgroups : 0;
    const uint64_t by_chunks = total > round ? total - round : 0;
    span_sum = chunk_sum = 0;
    for (int i = i0; i < i1; ++i) {
        const TreeKeys k = {r.row[i], r.held[i], r.len[i]};
        const int chunks = fits ? tree_chunks(p, k) : 0;
        const int first = first_tree_key(p, k.held) / kChunk, spans = spans_of(first, chunks);
        const uint32_t units = units_of(k.len - k.held), each = units * kvheads;
        int whole = 0; // spans that are items
        if (spans) {
            const uint64_t a = by_count > spans_at ? (by_count - spans_at) / each : 0;
            const uint64_t left = by_chunks > chunks_at ? (by_chunks - chunks_at) / each : 0;
            const uint64_t b = left ? (first % kSpanChunks + left - 1) / kSpanChunks + 1 : 0;
            whole = (int)min(max(a, b), (uint64_t)spans);
        }
        const int split =
            whole ? min((first / kSpanChunks + whole) * kSpanChunks, first + chunks) : first;
        spans_at += (uint64_t)spans * each;
        chunks_at += (uint64_t)chunks * each;
        r.split[i] = split;
        r.spans[i] = whole * each;
        r.singles[i] = (first + chunks - split) * each;
        span_sum += r.spans[i];
        chunk_sum += r.singles[i];
        if (blockIdx.x == 0) {
            p.ws_req[i] = int4{k.row, chunks, k.held, k.len - k.held};
            p.split[i] = split;
        }
    }
    // (at most max_items together: halves of a word)
    uint64_t both, before = block_offsets(span_sum << 32 | chunk_sum, waves[0], &both);
    for (int i = i0; i < i1; ++i) {
        const uint32_t a = r.spans[i], b = r.singles[i];
        r.spans[i] = (uint32_t)(before >> 32);
        r.singles[i] = (uint32_t)before;
        before += (uint64_t)a << 32 | b;
    }
    const uint32_t spans = (uint32_t)(both >> 32), all = spans + (uint32_t)both;
    if (tid == 0 && blockIdx.x == 0) {
        p.plan->items = (int)all;
        p.plan->uneven = spans != 0;
        // (the first one of a workgroup is its own)
        for (int i = 0; i < (int)kItemParts; ++i)
            p.plan->taken[i] =
                workgroups % (int)kItemParts ? workgroups : workgroups / (int)kItemParts;
    }
    if (bad && blockIdx.x == 0)
        atomicOr(p.err, kErrPages);
    __syncthreads();
    PlanItem *out = reinterpret_cast<PlanItem *>(p.plan + 1);
    for (uint32_t i = blockIdx.x * kPlanThreads + tid; i < all; i += gridDim.x * kPlanThreads) {
        // units of a span or chunk and KV head side by side: they share its keys
        const bool span = i < spans;
        const uint32_t at = span ? i : i - spans;
        const uint32_t *off = span ? r.spans : r.singles;
        PlanItem x;
        x.b = plan_request(off, n, at);
        const TreeKeys k = {r.row[x.b], r.held[x.b], r.len[x.b]};
        x.row = k.row;
        x.held = k.held;
        x.n = k.len - k.held;
        const uint32_t rest = at - off[x.b], units = units_of(x.n);
        const int unit = (int)(rest % units);
        x.kh = (int)(rest / units % kvheads);
        const int part = (int)(rest / units / kvheads);
        x.first_row = unit * UNIT;
        x.nrows = min(x.n * p.group - x.first_row, UNIT);
        x.from = first_tree_key(p, k.held);
        const int first = x.from / kChunk, end = (k.len - 1) / kChunk + 1;
        x.to = k.len - 1;
        if (!p.masks) {
            x.from = first_tree_key(p, k.held + x.first_row / p.group);
            x.to = k.held + (x.first_row + x.nrows - 1) / p.group;
        }
        const int g0 = span ? (first / kSpanChunks + part) * kSpanChunks : r.split[x.b] + part;
        const int g1 = min(g0 + (span ? kSpanChunks : 1), end);
        const int c0 = max(g0, x.from / kChunk), c1 = min(g1, x.to / kChunk + 1);
        x.chunk = c0;
        x.chunks = max(c1 - c0, 0);
        x.slot = g1 - 1 - first;
        x.only = max(g0, first) == first && g1 == end;
        x.spare[0] = x.spare[1] = x.spare[2] = 0;
        out[i] = x;
    }
}

// Words of the plan, by scalar loads (the same for the whole wave).
typedef int32_t int16w __attribute__((ext_vector_type(16)));
typedef const __attribute__((address_space(4))) int16w *plan_ptr;

__device__ __forceinline__ PlanItem plan_item(plan_ptr at)
{
    const int16w w = *at;
    return {w[0], w[1], w[2], w[3], w[4],  w[5],  w[6],
            w[7], w[8], w[9], w[10], w[11], w[12], {0, 0, 0}};
}

// Chunk k of an item.
__device__ __forceinline__ TreeItem chunk_item(const PlanItem &i, int k)
{
    TreeItem x;
    x.b = i.b;
    x.kh = i.kh;
    x.held = i.held;
    x.n = i.n;
    x.row = i.row;
    x.first_row = i.first_row;
    x.nrows = i.nrows;
    x.unit = 0;
    x.ci = (uint32_t)i.slot;
    x.only = i.only;
    x.empty = false;
    x.cbase = (i.chunk + k) * kChunk;
    x.lo = max(i.from - x.cbase, 0);
    x.hi = min(i.to - x.cbase, kChunk - 1);
    return x;
}

// Four waves a SIMD, two workgroups a CU, where one 16 of rows leaves room for them
// (128 registers; 64 trees of bf16 219 us, 254 us at the 148 that the compiler took).
// (48 rows at padded head dim 128, bf16, spill 4 registers at 256; with the one workgroup
// that the LDS holds as the bound the compiler holds sums in AGPRs and copies them: prompt
// parts of 512 tokens at 32 x 8 x 112, bf16, 2276 us and 2180, at 128 2262 and 2124; units
// of 32 rows 2350.)
template <int DK, typename T, bool FULL, int U, int NB>
__global__ __launch_bounds__((RowsCfg<DK, T, U>::kThreads),
                             (DK == 256 && U == 1 ? 4 : 2)) void tree_rows_kernel(TreeParams p)
{
    using C = RowsCfg<DK, T, U>;
    constexpr int NW = C::NW, KW = C::KW, TW = C::TW, UK = C::UK, VL = C::VL, SU = C::SU;
    static_assert(NB <= UK, "the ring holds units of one K row");
    extern __shared__ __attribute__((aligned(16))) uint32_t dyn[];
    using Lds = RowsLds<DK, U>;
    Lds &s = *reinterpret_cast<Lds *>(dyn);
    uint32_t *const rings = dyn + sizeof(Lds) / 4;
    const int tid = threadIdx.x;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int lane = tid & 63, col = lane & 15, g = lane >> 4;
    const int k0 = KW * w; // the wave's keys

    // Workgroups take items as they come to them: chunks differ in their keys, and items
    // in their chunks. An XCD's workgroups take those of its part, whose units share its
    // L2 (item_claims.hpp); where items differ in their chunks they go on to the others'
    // (prompt parts 1.87 ms, 1.9 to 2.0 without; where each is one chunk it costs: 64 trees
    // 246 -> 258 us, 256 chains 165 -> 180). One is taken while the one before the last
    // runs, so that nobody waits for the counter.
    const plan_ptr plan = (plan_ptr)p.plan;
    const uint32_t items = (uint32_t)(*plan)[0];
    const uint32_t parts = gridDim.x % kItemParts ? 1 : kItemParts;
    const ItemClaims claims = {items, gridDim.x, gridDim.x / parts,
                               parts > 1 && (*plan)[1] != 0};
    // (by thread 0)
    auto add = [&](uint32_t part) { return (uint32_t)atomicAdd(&p.plan->taken[part], 1); };
    auto settle = [&](uint32_t n) { // item n of the workgroup's part, or another's
        return claims.settle(
            claims.place(s.part, n), s.part,
            [&](uint32_t part) {
                return (uint32_t)__hip_atomic_load(&p.plan->taken[part], __ATOMIC_RELAXED,
                                                   __HIP_MEMORY_SCOPE_AGENT);
            },
            add);
    };
    // (an item past the last has no chunks, and is not skipped)
    auto load_item = [&](uint32_t n) {
        PlanItem i;
        i.chunks = -1;
        if (n < items)
            i = plan_item(plan + 1 + n);
        return i;
    };
    auto taken_item = [&]() { // by the whole workgroup, behind a barrier
        PlanItem i = load_item(__builtin_amdgcn_readfirstlane(s.taken));
        while (i.chunks == 0) { // (a chain's early units have none of the last keys)
            __syncthreads();
            if (tid == 0)
                s.taken = settle(add(s.part));
            __syncthreads();
            i = load_item(__builtin_amdgcn_readfirstlane(s.taken));
        }
        return i;
    };
    if (tid == 0) {
        s.part = blockIdx.x % parts;
        s.taken = claims.place(s.part, blockIdx.x / parts);
    }
    __syncthreads();
    PlanItem now = taken_item();
    if (now.chunks < 0)
        return;
    __syncthreads();
    if (tid == 0)
        s.taken = settle(add(s.part));
    PlanItem next; // (taken below)
    int chunk = 0; // of `now`

    struct Fetched {
        int page;
        RowsFetched<U> tree;
    };
    auto position = [&](const TreeItem &x) {
        return (uint32_t)(x.cbase + min(max(k0 + lane % KW, x.lo), x.hi));
    };
    auto fetch = [&](const TreeItem &x, Fetched &f) {
        f.page = p.table[x.b * p.table_stride + divided(position(x), p.by_page_tokens)];
        fetch_rows(p, x, k0, f.tree);
    };
    // The unit's query rows into LDS: a copy is four of the eight dims of a lane, for 16
    // rows and 32 dims. Rows past the last are the last one's, dims past the head dim
    // the first ones.
    auto issue_q = [&](const TreeItem &x) {
        const float *row[U];
#pragma unroll
        for (int rg = 0; rg < U; ++rg) {
            const int token = row_token(p, x, rg);
            const int head = x.first_row + min(16 * rg + col, x.nrows - 1) - token * p.group;
            row[rg] = p.q + (x.row + token) * p.q_stride +
                      (int64_t)(x.kh * p.group + head) * p.dim;
        }
        constexpr int kPart = DK / 16 / NW; // copies of 16 rows by a wave
#pragma unroll
        for (int rg = 0; rg < U; ++rg)
#pragma unroll
            for (int i = 0; i < kPart; ++i) {
                const int n = w * kPart + i, u = n / 2, hh = n % 2;
                const int d = 32 * u + 8 * g + 4 * hh;
                __builtin_amdgcn_global_load_lds(
                    (global_ptr)(row[rg] + (FULL || d < p.dim ? d : 0)),
                    (lds_ptr)(&s.q[rg][u][hh][0]), 16, 0, 0);
            }
    };
    // Scales the wave's copies where they lie, once they are there.
    auto scale_q = [&]() {
        constexpr int kPart = DK / 16 / NW;
#pragma unroll
        for (int rg = 0; rg < U; ++rg)
#pragma unroll
            for (int i = 0; i < kPart; ++i) {
                const int n = w * kPart + i, u = n / 2, hh = n % 2;
                const f4 v = s.q[rg][u][hh][lane] * p.q_scale;
                s.q[rg][u][hh][lane] =
                    FULL || 32 * u + 8 * g + 4 * hh < p.dim ? v : f4{0.f, 0.f, 0.f, 0.f};
            }
    };
    uint64_t see[U], see_next[U]; // the wave's keys that the lane's rows attend
    // A chunk's slots and live tiles. A key that no row attends takes the slot of one of
    // the wave's that some row does, so that no value is multiplied that the rows' own
    // results do not hold; tiles without one are copied, but not multiplied.
    auto store = [&](const TreeItem &x, const Fetched &f, int to) {
        int page = f.page;
        if (page < 0 || page >= p.pages) {
            atomicOr(p.err, kErrPages);
            page = 0;
        }
        const uint32_t t = position(x);
        int slot = page * (int32_t)p.page_tokens +
                   (int32_t)(t - divided(t, p.by_page_tokens) * p.page_tokens);
        attended_keys(p, x, k0, f.tree, see_next);
        uint64_t any = 0;
#pragma unroll
        for (int rg = 0; rg < U; ++rg)
            any |= see_next[rg];
        any = (uint64_t)or_rows((uint32_t)(any >> 32)) << 32 | or_rows((uint32_t)any);
        const int spare = __builtin_amdgcn_readlane(slot, any ? __builtin_ctzll(any) & (KW - 1) : 0);
        if (!(any >> lane & 1))
            slot = spare;
        if (lane < KW)
            s.slots[to][k0 + lane] = slot;
        if (lane < TW)
            s.live[to][TW * w + lane] = (uint32_t)(any >> (kTile * lane)) != 0;
    };
    // (paged_kv.hpp has the ring and its units)
    constexpr int kWords = C::kUnit / 4;
    uint32_t *const ring = rings + (size_t)w * NB * kWords;
    int at = 0;
    const uint32_t row_bytes = (uint32_t)(p.row_stride * sizeof(T));
    struct Sources {
        const char *from[C::NE];
    };
    const int piece = (lane % 8 ^ lane / 8) * (16 / (int)sizeof(T));
    auto rows_k = [&](const int32_t *slots, int kh, int part) {
        const char *base =
            static_cast<const char *>(p.k) + ((int64_t)kh * p.dim + piece) * sizeof(T);
        const int32_t *mine = slots + k0 + 16 * C::BU * part + lane / 8;
        Sources c;
#pragma unroll
        for (int e = 0; e < C::NE; ++e)
            c.from[e] = base + (uint64_t)(uint32_t)mine[8 * e] * row_bytes;
        return c;
    };
    auto line_k = [&](const Sources &rows, int line) {
        const int d = C::kLine * line;
        const int64_t step = (FULL || d + piece < p.dim ? d : -piece) * (int64_t)sizeof(T);
        Sources c;
#pragma unroll
        for (int e = 0; e < C::NE; ++e)
            c.from[e] = rows.from[e] + step;
        return c;
    };
    auto sources_v = [&](const int32_t *slots, int kh, int t0, int t1, int i) {
        const int d = 16 * VL * w + lane % C::kLanesV * (16 / (int)sizeof(T));
        const char *base = static_cast<const char *>(p.v) +
                           ((int64_t)kh * p.dim + (FULL || d < p.dim ? d : 0)) * sizeof(T);
        Sources c;
#pragma unroll
        for (int e = 0; e < C::NE; ++e) {
            const int n = C::kKeysV * i + (e * 64 + lane) / C::kLanesV; // chain step from tile t0 on
            const int t = min(t0 + n / kTile, t1), k = n % kTile;
            c.from[e] = base + (uint64_t)(uint32_t)slots[kTile * t + chain_key(k)] * row_bytes;
        }
        return c;
    };
    auto issue = [&](const Sources &c) {
#pragma unroll
        for (int e = 0; e < C::NE; ++e)
            __builtin_amdgcn_global_load_lds((global_ptr)c.from[e],
                                             (lds_ptr)(ring + at * kWords + e * 256), 16, 0,
                                             U == 1 ? kStreamed : 0);
    };
    auto wait_unit = [&]() {
        __builtin_amdgcn_s_waitcnt(waitcnt_vm(C::NE * (NB - 1)));
        asm volatile("" ::: "memory");
    };
    auto free_unit = [&]() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); };
    auto next_buffer = [&]() { at = at + 1 == NB ? 0 : at + 1; };

    TreeItem x = chunk_item(now, 0);
    {
        Fetched f;
        issue_q(x);
        fetch(x, f);
        store(x, f, 0);
    }
    __builtin_amdgcn_s_waitcnt(waitcnt_vm(0)); // the query's copies
    scale_q();
    __syncthreads();
    next = taken_item();
    {
#pragma unroll
        for (int i = 0; i < NB; ++i) {
            issue(line_k(rows_k(s.slots[0], x.kh, i % C::kParts), i / C::kParts));
            next_buffer();
        }
    }

    // the item's chunks merged so far
    float M1[U], L1[U];
    f4 merged[U][VL];
    for (int buf = 0;; buf ^= 1) {
        const bool last_chunk = chunk + 1 == now.chunks;
        const bool more = !last_chunk || next.chunks > 0;
        const bool new_q = last_chunk && more;
        // (without a next chunk this one's first units are copied again, and not used)
        TreeItem y = x;
        if (more)
            y = last_chunk ? chunk_item(next, 0) : chunk_item(now, chunk + 1);
        const int behind = more ? buf ^ 1 : buf; // the next chunk's slots
#pragma unroll
        for (int rg = 0; rg < U; ++rg)
            see[rg] = see_next[rg];
        const int groups = (x.nrows + 15) / 16;
        const int t0 = x.lo / kTile, t1 = x.hi / kTile; // tiles with attended keys
        const bool mine = k0 <= x.hi && k0 + KW - 1 >= x.lo;

        // scores: D of 16 keys x 16 rows
        f4 acc[U][2 * TW];
#pragma unroll
        for (int rg = 0; rg < U; ++rg)
#pragma unroll
            for (int b = 0; b < 2 * TW; ++b)
                acc[rg][b] = f4{0.f, 0.f, 0.f, 0.f};
        Sources rows[C::kParts];
#pragma unroll
        for (int part = 0; part < C::kParts; ++part)
            rows[part] = rows_k(s.slots[buf], x.kh, part);
        // the unit n units behind line `line`'s first
        auto unit_behind = [&](int line, auto nc) {
            constexpr int n = decltype(nc)::value;
            const int i = line + n / C::kParts;
            return i < C::kLines ? line_k(rows[n % C::kParts], i)
                                 : sources_v(s.slots[buf], x.kh, t0, t1, line * C::kParts + n - UK);
        };
        Sources c = unit_behind(0, std::integral_constant<int, NB>{});
#pragma unroll 1
        for (int i = 0; i < C::kLines; ++i) {
            f4 q[U][SU][2]; // read ahead of the wait
#pragma unroll
            for (int rg = 0; rg < U; ++rg)
#pragma unroll
                for (int u = 0; u < SU; ++u)
#pragma unroll
                    for (int hh = 0; hh < 2; ++hh) {
                        const int n = min(SU * i + u, DK / 32 - 1);
                        q[rg][u][hh] = s.q[rg][n][hh][lane];
                    }
            pcl::each<C::kParts>([&](auto pc) {
                constexpr int part = decltype(pc)::value;
                wait_unit();
                u4 kw[C::BU][2];
#pragma unroll
                for (int b = 0; b < C::BU; ++b)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        // f32: halves of a lane's eight dims; bf16: the eight of two steps
                        const int j = sizeof(T) == 4 ? 2 * g + h : 4 * h + g;
                        const int d = C::kLine * i + j * (16 / (int)sizeof(T));
                        u4 v = *(const u4 *)(ring + at * kWords + 32 * (16 * b + col) +
                                             4 * (j ^ (col & 7)));
                        if (!FULL && d >= p.dim)
                            v = u4{0u, 0u, 0u, 0u};
                        kw[b][h] = v;
                    }
                free_unit();
                issue(c);
                next_buffer();
                if (part + 1 < C::kParts || i + 1 < C::kLines)
                    c = unit_behind(i, std::integral_constant<int, part + 1 + NB>{});
                if (!mine)
                    return;
                // (bf16: widened once for all rows)
                float k[SU][C::BU][8];
#pragma unroll
                for (int u = 0; u < SU; ++u)
#pragma unroll
                    for (int b = 0; b < C::BU; ++b)
#pragma unroll
                        for (int jj = 0; jj < 8; ++jj) {
                            if constexpr (sizeof(T) == 4)
                                k[u][b][jj] = __uint_as_float(kw[b][jj / 4][jj % 4]);
                            else
                                k[u][b][jj] = jj % 2 ? bf16_high(kw[b][u][jj / 2])
                                                     : bf16_low(kw[b][u][jj / 2]);
                        }
#pragma unroll
                for (int rg = 0; rg < U; ++rg) {
                    if (rg >= groups)
                        continue;
#pragma unroll
                    for (int u = 0; u < SU; ++u) {
                        if (SU * i + u >= DK / 32)
                            continue;
#pragma unroll
                        for (int jj = 0; jj < 8; ++jj)
#pragma unroll
                            for (int b = 0; b < C::BU; ++b)
                                acc[rg][C::BU * part + b] =
                                    mfma(k[u][b][jj], q[rg][u][jj / 4][jj % 4],
                                         acc[rg][C::BU * part + b]);
                    }
                }
            });
        }

        // The claim of an item and the next chunk's words return during the softmax and
        // P.V: ahead of the scores the first wait for a unit's copies waits for them too.
        uint32_t behind_next = 0;
        if (new_q && tid == 0)
            behind_next = add(s.part);
        Fetched f;
        if (more)
            fetch(y, f);

        // `whole`: every row of the unit attends all of the wave's keys, as mostly
        uint64_t seen = ~(uint64_t)0;
#pragma unroll
        for (int rg = 0; rg < U; ++rg)
            seen &= rg < groups ? see[rg] : ~(uint64_t)0;
        const bool whole = __all((seen << (64 - KW)) == ~(uint64_t)0 << (64 - KW));
        auto ok_of = [&](auto all, int rg, int t, bool ok[2][4]) { // of the wave's tile t
#pragma unroll
            for (int b = 0; b < 2; ++b)
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    ok[b][r] = decltype(all)::value ||
                               ((uint32_t)(see[rg] >> (32 * t)) >> (16 * b + 4 * g + r) & 1);
        };
        auto maxima = [&](auto all) {
            float zero = 0.f; // a NaN once an attended score is not finite
#pragma unroll
            for (int rg = 0; rg < U; ++rg) {
                if (rg >= groups)
                    continue;
#pragma unroll
                for (int t = 0; t < TW; ++t) {
                    bool ok[2][4];
                    float v[2][4];
                    ok_of(all, rg, t, ok);
#pragma unroll
                    for (int b = 0; b < 2; ++b)
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            v[b][r] = acc[rg][2 * t + b][r];
                            if (p.softcap > 0.f)
                                v[b][r] = soft_cap(v[b][r], p.softcap, p.inv_softcap);
                            acc[rg][2 * t + b][r] = v[b][r];
                            zero = __builtin_fmaf(ok[b][r] ? v[b][r] : 0.f, 0.f, zero);
                        }
                    const float m = tile_max(v, ok);
                    if (g == 0)
                        s.max[16 * rg + col][TW * w + t] = m;
                }
            }
            if (zero != 0.f)
                atomicOr(p.err, kErrScore);
        };
        if (whole)
            maxima(std::true_type{});
        else
            maxima(std::false_type{});
        lds_barrier(); // every tile's maximum; the query is used
        if (new_q)
            issue_q(y);

        float last[U]; // the chunk's maximum
        auto probabilities = [&](auto all) {
#pragma unroll
            for (int rg = 0; rg < U; ++rg) {
                last[rg] = kNegInf;
                if (rg >= groups)
                    continue;
                float tm[kTilesPerChunk];
                *(f4 *)tm = *(const f4 *)&s.max[16 * rg + col][0];
                *(f4 *)(tm + 4) = *(const f4 *)&s.max[16 * rg + col][4];
                float before = kNegInf;
#pragma unroll
                for (int t = 0; t < kTilesPerChunk; ++t) {
                    before = t < TW * w ? fmaxf(before, tm[t]) : before;
                    last[rg] = fmaxf(last[rg], tm[t]);
                }
#pragma unroll
                for (int t = 0; t < TW; ++t) {
                    const int tile = TW * w + t;
                    bool ok[2][4];
                    float v[2][4], pr[2][4];
                    ok_of(all, rg, t, ok);
                    float m = before;
#pragma unroll
                    for (int i = 0; i < kTilesPerChunk; ++i)
                        m = i == tile ? fmaxf(m, tm[i]) : m;
#pragma unroll
                    for (int b = 0; b < 2; ++b)
#pragma unroll
                        for (int r = 0; r < 4; ++r)
                            v[b][r] = acc[rg][2 * t + b][r];
                    const float ms = safe_max(m);
                    const float sum = tile_probs(v, ok, ms, pr);
#pragma unroll
                    for (int b = 0; b < 2; ++b)
                        s.p[rg][tile][b][lane] = f4{pr[b][0], pr[b][1], pr[b][2], pr[b][3]};
                    if (g == 0)
                        s.factors[tile][16 * rg + col] = f2{fexp(before - ms), sum};
                    before = m;
                }
            }
        };
        if (whole)
            probabilities(std::true_type{});
        else
            probabilities(std::false_type{});
        if (more)
            store(y, f, buf ^ 1);
        lds_barrier(); // probabilities, row sums and factors
        const uint32_t live = (uint32_t)__ballot(lane < kTilesPerChunk && s.live[buf][lane % 8]);

        // the l chain and the P.V chains of the wave's dims: D of 16 dims x 16 rows
        float l[U];
        f4 O[U][VL];
#pragma unroll
        for (int rg = 0; rg < U; ++rg) {
            l[rg] = 0.f;
#pragma unroll
            for (int j = 0; j < VL; ++j)
                O[rg][j] = f4{0.f, 0.f, 0.f, 0.f};
        }
        const int units = ((t1 - t0 + 1) * kTile + C::kKeysV - 1) / C::kKeysV;
        const int rounds = max(units, NB);
        auto behind_v = [&](int i) {
            const int n = i + NB - rounds; // the next item's first units follow this one's
            return n < 0 ? sources_v(s.slots[buf], x.kh, t0, t1, i + NB)
                         : line_k(rows_k(s.slots[behind], y.kh, n % C::kParts), n / C::kParts);
        };
        c = behind_v(0);
        // The probabilities and factors of the 16 keys behind n of the tiles' from t0 on,
        // for all rows (of keys past the last tile: any).
        struct Weights {
            f4 p[U];
            f2 factors[U];
        };
        auto weights = [&](int n, int b) {
            const int t = min(t0 + n / kTile, kTilesPerChunk - 1);
            Weights x;
#pragma unroll
            for (int rg = 0; rg < U; ++rg) {
                x.p[rg] = s.p[rg][t][b][lane];
                if (b == 0)
                    x.factors[rg] = s.factors[t][16 * rg + col];
            }
            return x;
        };
#pragma unroll 1
        for (int i = 0; i < rounds; ++i) {
            // 16 keys at a time: four chain steps of 4 keys (r), each with the lane's
            // own key and VL dims
            constexpr int WV = (VL * (int)sizeof(T) + 3) / 4; // words of a lane's values
            constexpr int kSixteens = C::kKeysV / 16, kHeld = kSixteens < 4 ? kSixteens : 4;
            auto half = [&](int h) { return C::kKeysV < kTile ? i % 2 : h % 2; };
            Weights x[2];
            x[0] = weights(C::kKeysV * i, half(0));
            wait_unit();
#pragma unroll 1
            for (int h0 = 0; h0 < kSixteens; h0 += kHeld) {
                uint32_t vw[kHeld][4][WV];
#pragma unroll
                for (int h = 0; h < kHeld; ++h)
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const char *row = reinterpret_cast<const char *>(ring + at * kWords) +
                                          (16 * (h0 + h) + 4 * r + g) * C::kRowV;
                        if constexpr (WV == 4) {
                            const u4 v = *(const u4 *)(row + 16 * col);
#pragma unroll
                            for (int e = 0; e < 4; ++e)
                                vw[h][r][e] = v[e];
                        } else if constexpr (WV == 2) {
                            const u2 v = *(const u2 *)(row + 8 * col);
                            vw[h][r][0] = v.x;
                            vw[h][r][1] = v.y;
                        } else if constexpr (VL * sizeof(T) == 4) {
                            vw[h][r][0] = *(const uint32_t *)(row + 4 * col);
                        } else {
                            vw[h][r][0] = *(const uint16_t *)(row + 2 * col);
                        }
                    }
                if (h0 + kHeld >= kSixteens) {
                    free_unit();
                    issue(c);
                    next_buffer();
                    if (i + 1 < rounds)
                        c = behind_v(i + 1);
                }
                if (i >= units)
                    continue;
#pragma unroll
                for (int h = 0; h < kHeld; ++h) {
                    const int n = C::kKeysV * i + 16 * (h0 + h), t = t0 + n / kTile;
                    // the next one's behind these products (of this unit)
                    if (h + 1 < kHeld || kHeld < kSixteens)
                        x[(h + 1) % 2] = weights(n + 16, half(h + 1));
                    if ((C::kKeysV > kTile && t > t1) || !(live >> t & 1))
                        continue;
#pragma unroll
                    for (int rg = 0; rg < U; ++rg) {
                        if (rg >= groups)
                            continue;
                        if (half(h) == 0) {
                            const f2 f = x[h % 2].factors[rg];
                            l[rg] = __builtin_fmaf(l[rg], f.x, f.y);
#pragma unroll
                            for (int j = 0; j < VL; ++j)
                                O[rg][j] = O[rg][j] * f.x;
                        }
#pragma unroll
                        for (int r = 0; r < 4; ++r)
#pragma unroll
                            for (int j = 0; j < VL; ++j)
                                O[rg][j] = mfma(value_of<T>(vw[h][r], j), x[h % 2].p[rg][r], O[rg][j]);
                    }
                }
            }
        }

        // (the next query's copies are older than its first units')
        __builtin_amdgcn_s_waitcnt(waitcnt_vm(C::NE * NB));
        if (new_q)
            scale_q();

        // a row without a key in the chunk merges as an empty part
        const bool merging = now.chunks > 1;
        if (merging) {
#pragma unroll
            for (int rg = 0; rg < U; ++rg) {
                if (chunk == 0) {
                    M1[rg] = kNegInf;
                    L1[rg] = 0.f;
#pragma unroll
                    for (int j = 0; j < VL; ++j)
                        merged[rg][j] = f4{0.f, 0.f, 0.f, 0.f};
                }
                const bool some = l[rg] != 0.f;
                const MergeFactors mf = merge_factors(M1[rg], last[rg]);
                L1[rg] = merge_value(L1[rg], l[rg], mf);
                M1[rg] = mf.m;
#pragma unroll
                for (int j = 0; j < VL; ++j)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        merged[rg][j][e] =
                            merge_value(merged[rg][j][e], some ? O[rg][j][e] : 0.f, mf);
            }
        }
        // D's row 4 g + e of block j is the dim that lane 4 g + e of the operand had:
        // a lane has 4 VL dims in a row
        const int d0 = 16 * VL * w + 4 * VL * g;
        bool nonfinite = false;
        if (last_chunk) {
#pragma unroll
            for (int rg = 0; rg < U; ++rg) {
                const int r = 16 * rg + col;
                if (r >= x.nrows)
                    continue;
                const int f0 = x.first_row + r, token = (int)divided(f0, p.by_group);
                const int head = x.kh * p.group + f0 - token * p.group;
                const int64_t part = ((int64_t)(x.row + token) * p.row_chunks + x.ci) * p.qheads + head;
                const float sum = merging ? L1[rg] : l[rg];
                const bool some = sum != 0.f; // a key that the row attends
                float *dst = x.only ? p.out + (x.row + token) * p.o_stride + (int64_t)head * p.dim
                                    : p.ws_o + part * p.dim;
                if (x.only && !some)
                    continue;
#pragma unroll
                for (int k = 0; k < VL; ++k) {
                    if (!FULL && d0 + 4 * k >= p.dim)
                        continue;
                    f4 v;
#pragma unroll
                    for (int a = 0; a < 4; ++a) {
                        const int j = (4 * k + a) % VL, e = (4 * k + a) / VL;
                        const float o = merging ? merged[rg][j][e] : O[rg][j][e];
                        v[a] = x.only ? o / sum : some ? o : 0.f;
                        nonfinite |= x.only && !is_finite(v[a]);
                    }
                    stg4(dst + d0 + 4 * k, v);
                }
                if (!x.only && w == 0 && g == 0) {
                    stg(p.ws_ml + 2 * part, merging ? M1[rg] : last[rg]);
                    stg(p.ws_ml + 2 * part + 1, sum);
                }
            }
        }
        if (nonfinite)
            atomicOr(p.err, kErrOutput);
        if (!more)
            break;
        if (new_q && tid == 0)
            s.taken = settle(behind_next);
        lds_barrier(); // the next query
        x = y;
        ++chunk;
        if (last_chunk) {
            now = next;
            next = taken_item();
            chunk = 0;
        }
    }
    // no copy may land in LDS that another workgroup owns by then
    __builtin_amdgcn_s_waitcnt(waitcnt_vm(0));
}

// Workgroups that a CU holds at once, asked once per device.
template <int DK, typename T, bool FULL, int U, int NB> static hipError_t resident_rows(int *groups)
{
    const auto kernel = (const void *)tree_rows_kernel<DK, T, FULL, U, NB>;
    static std::atomic<int> known[kMaxDevices];
    int dev = 0;
    hipError_t e = hipGetDevice(&dev);
    if (e != hipSuccess)
        return e;
    if (dev < 0 || dev >= kMaxDevices)
        return hipErrorInvalidDevice;
    *groups = known[dev].load(std::memory_order_acquire);
    if (*groups > 0)
        return hipSuccess;
    constexpr size_t bytes = rows_lds_bytes<DK, T, U, NB>();
    static_assert(bytes <= kRowsLds, "the LDS of a CU");
    e = hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
    if (e == hipSuccess)
        e = hipOccupancyMaxActiveBlocksPerMultiprocessor(groups, kernel,
                                                         RowsCfg<DK, T, U>::kThreads, bytes);
    if (e != hipSuccess)
        return e;
    *groups = std::max(*groups, 1);
    known[dev].store(*groups, std::memory_order_release);
    return hipSuccess;
}

template <int DK, typename T, bool FULL, int U>
static hipError_t launch_rows(const TreeParams &p, int64_t rows, int64_t chunks, hipStream_t stream)
{
    constexpr int NB = rows_buffers(DK);
    int groups = 0;
    const hipError_t e = resident_rows<DK, T, FULL, U, NB>(&groups);
    if (e != hipSuccess)
        return e;
    // (the items at the requests' longest)
    const int64_t units = (rows + 16 * U - 1) / (16 * U);
    const int64_t items = std::min<int64_t>(chunks * p.kvheads * units, p.max_items);
    const int64_t grid = std::min<int64_t>(items, (int64_t)groups * std::max(device_cus(), 1));
    const int64_t plans = std::min<int64_t>((items + kPlanThreads - 1) / kPlanThreads, 256);
    paged_plan_kernel<16 * U>
        <<<(unsigned)plans, kPlanThreads, plan_words_bytes(p.requests), stream>>>(p, (int)grid);
    tree_rows_kernel<DK, T, FULL, U, NB>
        <<<(unsigned)grid, RowsCfg<DK, T, U>::kThreads, rows_lds_bytes<DK, T, U, NB>(), stream>>>(p);
    return hipGetLastError();
}

template <int DK, typename T, bool FULL>
static hipError_t launch_rows(const TreeParams &p, int unit, int64_t rows, int64_t chunks,
                              hipStream_t stream)
{
    if constexpr (DK < 512) { // (tree_variant)
        if (unit == 48)
            return launch_rows<DK, T, FULL, 3>(p, rows, chunks, stream);
    }
    return unit == 32 ? launch_rows<DK, T, FULL, 2>(p, rows, chunks, stream)
                      : launch_rows<DK, T, FULL, 1>(p, rows, chunks, stream);
}

template <int DK>
hipError_t launch_paged_rows(const TreeParams &p, int unit, bool bf16, int64_t rows,
                             int64_t chunks, hipStream_t stream)
{
    if (p.dim == DK)
        return bf16 ? launch_rows<DK, __bf16, true>(p, unit, rows, chunks, stream)
                    : launch_rows<DK, float, true>(p, unit, rows, chunks, stream);
    return bf16 ? launch_rows<DK, __bf16, false>(p, unit, rows, chunks, stream)
                : launch_rows<DK, float, false>(p, unit, rows, chunks, stream);
}

} // namespace pcl
