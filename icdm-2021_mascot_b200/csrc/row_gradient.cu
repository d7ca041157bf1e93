// Sums by row: the gradient of a row lookup, and the gradients of the preference loss in both factor tables.
//
// Both are  out[r] = scale * sum over the entries e of row r of value(e),  where an entry is a place that looked a row up, and
// a value a row of its own: a gradient row (lookup), or c * (Q[i] - Q[j]) for the user and +-c * P[u] for the two items of a
// pair.  Atomic additions would settle the order of a sum by chance; here the entries are sorted by row, stably, and then
// summed in that order, in fp32:
//
//   sort     least significant digit first, on (row, entry) pairs of 32 bits each.  All entries of both tables are sorted at once,
//            the items' rows counted behind the users'.  Up to kSmall entries one block does all passes in shared
//            memory; more take count / scan / scatter kernels for each digit.
//   reduce   the sorted entries are cut into chunks of equal length, a team of lanes for each, so that a popular row is
//            shared by many teams and many unpopular ones by one.  A row that lies within a chunk is written at once; of one that
//            goes on in the next chunk or comes from the one before, the chunk's part is left in the workspace.
//   combine  adds these parts up in the order of the chunks, and clears rows that no entry names.
#include <algorithm>

#include "row_ops.h"

namespace mascot {
namespace {

constexpr int kSortBlock = 256, kSortItems = 16, kTile = kSortBlock * kSortItems;     // entries of a block of the sort
constexpr int kMaxDigitBits = 10, kMaxBins = 1 << kMaxDigitBits;
constexpr int kScanTiles = 32;                  // up to so many tiles the scatter kernel adds their counts up itself
constexpr int kSmallBlock = 1024, kSmallItems = 12;
constexpr uint32_t kSmall = kSmallBlock * kSmallItems;
constexpr int kSmallDigitBits = 8;
constexpr int kReduceBlock = 256, kCombineBlock = 1024;
constexpr uint32_t kLongSpan = 64;              // chunks of one row that a warp still adds up alone

// What is summed: where entries come from and what their values are.
struct Job {
    Ids ids[3];                                 // lookup: one; pairs: users, preferred, other
    uint32_t per;                               // ids of one kind: entry e is id e % per of kind e / per
    uint32_t kinds;                             // 1: lookup, 3: pairs
    uint32_t n;                                 // entries: kinds * per
    uint32_t rows[2];                           // of the table; of both tables
    uint32_t total;                             // all rows; the sort key of an entry that names none
    const void* src[2];                         // lookup: gradient rows; pairs: P, Q
    size_t src_stride[2];
    const float* coef;
    void* out[2];
    size_t out_stride[2];
    uint32_t width, chunk_log2;
    float scale;
    int accumulate;
    uint32_t* flags;
};

struct Space {                                  // the workspace, see carve()
    uint32_t *key[2], *val[2], *counts, *totals;
    float *head, *tail;                         // [chunks][pitch]
    uint8_t* touched;                           // a byte per row
    uint32_t pitch, chunks, tiles;
};

// ---- sort --------------------------------------------------------------------------------------------------

// Row of entry e, or `total`.
__device__ __forceinline__ uint32_t entry_key(const Job& j, uint32_t e, bool& bad) {
    if (j.kinds == 1) {
        const uint32_t r = row_of(j.ids[0], e, j.rows[0], bad);
        return r == kNoRow ? j.total : r;
    }
    const uint32_t kind = e / j.per, b = e - kind * j.per;
    const uint32_t u = row_of(j.ids[0], b, j.rows[0], bad), p = row_of(j.ids[1], b, j.rows[1], bad), o = row_of(j.ids[2], b, j.rows[1], bad);
    if (u == kNoRow || p == kNoRow || o == kNoRow) return j.total;
    return kind == 0 ? u : j.rows[0] + (kind == 1 ? p : o);
}

__device__ __forceinline__ void clear_touched(uint8_t* touched, uint32_t rows, size_t first, size_t step) {
    for (size_t w = first; w < ((size_t)rows + 15) / 16; w += step) reinterpret_cast<uint4*>(touched)[w] = make_uint4(0, 0, 0, 0);
}

// Stable ranks of a warp's keys among the keys with the same digit that the warp has met so far; `count` is the
// warp's own row of counters, zero at first.
__device__ __forceinline__ uint32_t warp_rank(uint32_t digit, bool there, uint16_t* count, uint32_t lane) {
    const uint32_t peers = __match_any_sync(0xffffffffu, there ? digit : 0xffffffffu);
    uint32_t before = 0;
    const uint32_t below = __popc(peers & ((1u << lane) - 1u));
    if (there) before = count[digit];
    __syncwarp();
    if (there && below == 0) count[digit] = (uint16_t)(before + __popc(peers));
    __syncwarp();
    return before + below;
}

// Exclusive scan over `bins` values in shared memory by a whole block, in place; bins at most 4 * blockDim.x.
__device__ __forceinline__ void block_scan(uint32_t* v, int bins, uint32_t* warp_sums) {
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5, warps = blockDim.x >> 5;
    uint32_t x[4], sum = 0;
#pragma unroll
    for (int k = 0; k < 4; k++) { const int b = 4 * t + k; x[k] = b < bins ? v[b] : 0u; sum += x[k]; }
    uint32_t inc = sum;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) { const uint32_t y = __shfl_up_sync(0xffffffffu, inc, d); if (lane >= d) inc += y; }
    if (lane == 31) warp_sums[warp] = inc;
    __syncthreads();
    if (warp == 0) {
        const uint32_t mine = lane < warps ? warp_sums[lane] : 0u;
        uint32_t s = mine;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) { const uint32_t y = __shfl_up_sync(0xffffffffu, s, d); if (lane >= d) s += y; }
        if (lane < warps) warp_sums[lane] = s - mine;
    }
    __syncthreads();
    uint32_t run = warp_sums[warp] + inc - sum;
#pragma unroll
    for (int k = 0; k < 4; k++) { const int b = 4 * t + k; if (b < bins) v[b] = run; run += x[k]; }
    __syncthreads();
}

// One block, everything in shared memory: keys and values twice, counters of 32 warps.  What bounds it is the latency of a
// pass (about 1.5 us of ranking); a sort over many blocks costs three launches a digit.
__global__ void __launch_bounds__(kSmallBlock) small_sort_kernel(const Job j, const Space s, int passes, int bits) {
    extern __shared__ uint32_t mem[];
    uint32_t* key[2] = {mem, mem + kSmall};
    uint32_t* val[2] = {mem + 2 * kSmall, mem + 3 * kSmall};
    uint16_t* const count = reinterpret_cast<uint16_t*>(mem + 4 * kSmall);
    uint32_t* const bins_at = mem + 4 * kSmall + 32 * (1 << kSmallDigitBits) / 2;
    uint32_t* const warp_sums = bins_at + (1 << kSmallDigitBits);
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5, bins = 1 << bits;
    if (!j.accumulate) clear_touched(s.touched, j.total, t, kSmallBlock);
    bool bad = false;
    for (uint32_t e = t; e < j.n; e += kSmallBlock) { key[0][e] = entry_key(j, e, bad); val[0][e] = e; }
    if (bad && j.flags) atomicOr(j.flags, (uint32_t)MASCOT_FLAG_BAD_ID);
    const uint32_t per_warp = ((j.n + 1023) / 1024) * 32, first = warp * per_warp;       // a warp's entries, in order
    uint16_t* const mine = count + (warp << bits);
    int from = 0;
    for (int p = 0; p < passes; p++, from ^= 1) {
        for (int b = lane; b < bins; b += 32) mine[b] = 0;
        __syncthreads();
        uint32_t rank[kSmallItems];
#pragma unroll
        for (int k = 0; k < kSmallItems; k++) {
            if (k * 32u >= per_warp) break;
            const uint32_t e = first + k * 32 + lane;
            const bool there = e < j.n;
            const uint32_t d = there ? key[from][e] >> (p * bits) & (bins - 1) : 0u;
            rank[k] = warp_rank(d, there, mine, lane);
        }
        __syncthreads();
        for (int b = t; b < bins; b += kSmallBlock) {           // counters become offsets of the warps within a bin
            uint32_t sum = 0;
            for (int w = 0; w < 32; w++) { uint16_t* const c = count + (w << bits) + b; const uint32_t x = *c; *c = (uint16_t)sum; sum += x; }
            bins_at[b] = sum;
        }
        __syncthreads();
        block_scan(bins_at, bins, warp_sums);
#pragma unroll
        for (int k = 0; k < kSmallItems; k++) {
            if (k * 32u >= per_warp) break;
            const uint32_t e = first + k * 32 + lane;
            if (e < j.n) {
                const uint32_t x = key[from][e], d = x >> (p * bits) & (bins - 1), at = bins_at[d] + mine[d] + rank[k];
                key[from ^ 1][at] = x;
                val[from ^ 1][at] = val[from][e];
            }
        }
        __syncthreads();
    }
    for (uint32_t e = t; e < j.n; e += kSmallBlock) { s.key[0][e] = key[from][e]; s.val[0][e] = val[from][e]; }
}

// Counts of the digits of a tile, [bin][tile].  The first pass makes the keys, and keeps them.
template <bool FIRST>
__global__ void __launch_bounds__(kSortBlock) count_kernel(const Job j, const Space s, int from, int shift, int bits) {
    __shared__ uint32_t hist[kMaxBins];
    const int bins = 1 << bits;
    for (int b = threadIdx.x; b < bins; b += kSortBlock) hist[b] = 0;
    if (FIRST && !j.accumulate) clear_touched(s.touched, j.total, (size_t)blockIdx.x * kSortBlock + threadIdx.x, (size_t)gridDim.x * kSortBlock);
    __syncthreads();
    bool bad = false;
#pragma unroll 4
    for (int k = 0; k < kSortItems; k++) {
        const uint32_t e = blockIdx.x * kTile + k * kSortBlock + threadIdx.x;
        if (e >= j.n) break;
        uint32_t key;
        if (FIRST) { key = entry_key(j, e, bad); s.key[0][e] = key; }
        else key = s.key[from][e];
        atomicAdd(&hist[key >> shift & (bins - 1)], 1u);
    }
    if (FIRST && bad && j.flags) atomicOr(j.flags, (uint32_t)MASCOT_FLAG_BAD_ID);
    __syncthreads();
    for (int b = threadIdx.x; b < bins; b += kSortBlock) s.counts[(size_t)b * s.tiles + blockIdx.x] = hist[b];
}

// A warp per bin: counts of the tiles become offsets within the bin, the sums go to totals.
__global__ void __launch_bounds__(256) scan_kernel(const Space s, int bins) {
    const int bin = (blockIdx.x * 256 + threadIdx.x) >> 5, lane = threadIdx.x & 31;
    if (bin >= bins) return;
    uint32_t* const c = s.counts + (size_t)bin * s.tiles;
    uint32_t run = 0;
    for (uint32_t t0 = 0; t0 < s.tiles; t0 += 128) {
        uint32_t x[4], sum = 0;
#pragma unroll
        for (int k = 0; k < 4; k++) { const uint32_t t = t0 + 4 * lane + k; x[k] = t < s.tiles ? c[t] : 0u; sum += x[k]; }
        uint32_t inc = sum;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) { const uint32_t y = __shfl_up_sync(0xffffffffu, inc, d); if (lane >= d) inc += y; }
        uint32_t at = run + inc - sum;
#pragma unroll
        for (int k = 0; k < 4; k++) { const uint32_t t = t0 + 4 * lane + k; if (t < s.tiles) c[t] = at; at += x[k]; }
        run += __shfl_sync(0xffffffffu, inc, 31);
    }
    if (lane == 0) s.totals[bin] = run;
}

// Moves a tile's entries to their places.  Ranks within a warp by matching digits, in the order of the entries; warps and tiles by
// their counts.
template <bool FIRST>
__global__ void __launch_bounds__(kSortBlock) scatter_kernel(const Job j, const Space s, int from, int shift, int bits, bool scanned) {
    extern __shared__ uint32_t mem[];                           // offsets of the bins, then the warps' counters
    __shared__ uint32_t warp_sums[kSortBlock / 32];
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5, bins = 1 << bits;
    uint32_t* const base = mem;
    uint16_t* const count = reinterpret_cast<uint16_t*>(mem + bins), *const mine = count + (warp << bits);
    for (int b = t; b < bins * (kSortBlock / 32) / 2; b += kSortBlock) reinterpret_cast<uint32_t*>(count)[b] = 0;
    uint32_t within[kMaxBins / kSortBlock];                     // entries of the bin in the tiles before
#pragma unroll
    for (int k = 0; k < kMaxBins / kSortBlock; k++) {
        const int b = t + k * kSortBlock;
        within[k] = 0;
        if (b < bins) {
            const uint32_t* const c = s.counts + (size_t)b * s.tiles;
            uint32_t sum = 0;
            if (scanned) { within[k] = c[blockIdx.x]; sum = s.totals[b]; }
            else for (uint32_t q = 0; q < s.tiles; q++) { if (q == blockIdx.x) within[k] = sum; sum += c[q]; }
            base[b] = sum;
        }
    }
    __syncthreads();
    block_scan(base, bins, warp_sums);
#pragma unroll
    for (int k = 0; k < kMaxBins / kSortBlock; k++) { const int b = t + k * kSortBlock; if (b < bins) base[b] += within[k]; }
    const uint32_t first = blockIdx.x * kTile + warp * (32 * kSortItems);
    uint32_t key[kSortItems], rank[kSortItems];
#pragma unroll
    for (int k = 0; k < kSortItems; k++) { const uint32_t e = first + k * 32 + lane; key[k] = e < j.n ? s.key[from][e] : 0u; }
#pragma unroll
    for (int k = 0; k < kSortItems; k++) rank[k] = warp_rank(key[k] >> shift & (bins - 1), first + k * 32 + lane < j.n, mine, lane);
    __syncthreads();
    for (int b = t; b < bins; b += kSortBlock) {
        uint32_t sum = 0;
#pragma unroll
        for (int w = 0; w < kSortBlock / 32; w++) { uint16_t* const c = count + (w << bits) + b; const uint32_t x = *c; *c = (uint16_t)sum; sum += x; }
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kSortItems; k++) {
        const uint32_t e = first + k * 32 + lane;
        if (e < j.n) {
            const uint32_t d = key[k] >> shift & (bins - 1), at = base[d] + mine[d] + rank[k];
            s.key[from ^ 1][at] = key[k];
            s.val[from ^ 1][at] = FIRST ? e : s.val[from][e];
        }
    }
}

// ---- sums --------------------------------------------------------------------------------------------------

template <typename Out, int N>
__device__ __forceinline__ void write_row(const Job& j, uint32_t row, uint32_t col, const float (&sum)[N]) {
    const bool second = row >= j.rows[0];
    Out* const at = static_cast<Out*>(j.out[second]) + (size_t)(second ? row - j.rows[0] : row) * j.out_stride[second] + col;
    Piece<Out, N> r;
    if (j.accumulate) {
        r = *reinterpret_cast<const Piece<Out, N>*>(at);
#pragma unroll
        for (int k = 0; k < N; k++) r.v[k] = from_float<Out>(fmaf(sum[k], j.scale, as_float(r.v[k])));
    } else {
#pragma unroll
        for (int k = 0; k < N; k++) r.v[k] = from_float<Out>(sum[k] * j.scale);
    }
    store_piece<Out, N>(at, r);
}

// An entry's value: c * (row a - row b), without b where that is null, and plain where there is no coefficient.
template <typename T> struct Value { const T *a, *b; float c; };
template <typename T, bool PAIRS>
__device__ __forceinline__ Value<T> value_of(const Job& j, uint32_t e, uint32_t col) {
    Value<T> v{nullptr, nullptr, 1.f};
    if (!PAIRS) { v.a = static_cast<const T*>(j.src[0]) + (size_t)e * j.src_stride[0] + col; return v; }
    const uint32_t kind = e >= 2 * j.per ? 2 : e >= j.per ? 1 : 0, b = e - kind * j.per;
    bool bad = false;
    v.c = __ldg(j.coef + b);
    if (kind == 0) {
        const uint32_t p = row_of(j.ids[1], b, j.rows[1], bad), o = row_of(j.ids[2], b, j.rows[1], bad);
        v.a = static_cast<const T*>(j.src[1]) + p * j.src_stride[1] + col;
        v.b = static_cast<const T*>(j.src[1]) + o * j.src_stride[1] + col;
    } else {
        const uint32_t u = row_of(j.ids[0], b, j.rows[0], bad);
        v.a = static_cast<const T*>(j.src[0]) + u * j.src_stride[0] + col;
        if (kind == 2) v.c = -v.c;
    }
    if (v.c == 0.f) v.a = nullptr;                              // whatever the rows hold
    return v;
}

constexpr int kBatch = 4;                       // entries whose rows a team has in flight

template <typename T, typename Out, int N, bool PAIRS>
__global__ void __launch_bounds__(kReduceBlock) reduce_kernel(const Job j, const Space s, const uint32_t* key, const uint32_t* val, int team_log2) {
    const uint32_t chunk = (blockIdx.x * kReduceBlock + threadIdx.x) >> team_log2, tl = threadIdx.x & ((1u << team_log2) - 1);
    const uint32_t col = ((blockIdx.y << team_log2) + tl) * N;
    if (chunk >= s.chunks || col >= j.width) return;
    const uint32_t begin = chunk << j.chunk_log2, end = min(j.n, begin + (1u << j.chunk_log2));
    const uint32_t before = begin ? __ldg(key + begin - 1) : kNoRow, after = end < j.n ? __ldg(key + end) : kNoRow;
    uint32_t row = __ldg(key + begin);
    float sum[N] = {};
    const auto flush = [&](uint32_t r) {
        if (r >= j.total) return;
        if (r == before || r == after) {                       // part of a row that other chunks share
            float* const part = (r == before ? s.head : s.tail) + (size_t)chunk * s.pitch + col;
#pragma unroll
            for (int k = 0; k < N; k++) part[k] = sum[k];
        } else write_row<Out, N>(j, r, col, sum);
        if (r != before && !j.accumulate && col == 0) s.touched[r] = 1;
    };
    for (uint32_t e0 = begin; e0 < end && row < j.total; e0 += kBatch) {
        const uint4 k4 = __ldg(reinterpret_cast<const uint4*>(key + e0)), v4 = __ldg(reinterpret_cast<const uint4*>(val + e0));
        const uint32_t keys[kBatch] = {k4.x, k4.y, k4.z, k4.w}, vals[kBatch] = {v4.x, v4.y, v4.z, v4.w};
        Value<T> v[kBatch];
        Piece<T, N> a[kBatch], b[kBatch];
#pragma unroll
        for (int k = 0; k < kBatch; k++) {
            v[k] = Value<T>{nullptr, nullptr, 0.f};
            if (e0 + k < end && keys[k] < j.total) v[k] = value_of<T, PAIRS>(j, vals[k], col);
        }
#pragma unroll
        for (int k = 0; k < kBatch; k++) {
            if (v[k].a) a[k] = load_piece<T, N>(v[k].a);
            if (PAIRS && v[k].b && v[k].a) b[k] = load_piece<T, N>(v[k].b);
        }
#pragma unroll
        for (int k = 0; k < kBatch; k++) {
            if (e0 + k >= end) break;
            if (keys[k] != row) {
                flush(row);
                row = keys[k];
#pragma unroll
                for (int x = 0; x < N; x++) sum[x] = 0.f;
            }
            if (v[k].a) {
#pragma unroll
                for (int x = 0; x < N; x++) {
                    if (!PAIRS) sum[x] += as_float(a[k].v[x]);
                    else sum[x] = fmaf(v[k].c, v[k].b ? as_float(a[k].v[x]) - as_float(b[k].v[x]) : as_float(a[k].v[x]), sum[x]);
                }
            }
        }
    }
    flush(row);
}

// The first position behind the entries of `row`, searched from `at`, which is one of them.
__device__ __forceinline__ uint32_t row_end(const uint32_t* key, uint32_t at, uint32_t n, uint32_t row) {
    uint32_t lo = at, hi = n;                                   // key[lo] == row, key[hi] > row
    while (hi - lo > 1) {
        const uint32_t mid = lo + (hi - lo) / 2;
        if (__ldg(key + mid) == row) lo = mid; else hi = mid;
    }
    return hi;
}

// Blocks below `combine_blocks`: a warp per chunk adds up the row that begins in it and goes on behind it.  A row over
// more than kLongSpan chunks is added up by all warps of the block, a slice each: only one row a block can be that long, since it
// covers all chunks of the block behind its first.  The other blocks clear the rows that no entry names, a warp for 32 of them.
template <typename Out, int N>
__global__ void __launch_bounds__(kCombineBlock) combine_kernel(const Job j, const Space s, const uint32_t* key, uint32_t combine_blocks) {
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    if (blockIdx.x >= combine_blocks) {
        const uint32_t row0 = (blockIdx.x - combine_blocks) * kCombineBlock + warp * 32;
        const bool clear = row0 + lane < j.total && (j.n == 0 || s.touched[row0 + lane] == 0);
        uint32_t todo = __ballot_sync(0xffffffffu, clear);
        while (todo) {
            const uint32_t r = row0 + __ffs(todo) - 1;
            todo &= todo - 1;
            const bool second = r >= j.rows[0];
            Out* const at = static_cast<Out*>(j.out[second]) + (size_t)(second ? r - j.rows[0] : r) * j.out_stride[second];
            for (uint32_t c = lane * N; c < j.width; c += 32 * N) {
                Piece<Out, N> zero;
#pragma unroll
                for (int k = 0; k < N; k++) zero.v[k] = from_float<Out>(0.f);
                store_piece<Out, N>(at + c, zero);
            }
        }
        return;
    }
    __shared__ float slice[kCombineBlock / 32][32 * N];
    __shared__ uint32_t long_chunk, long_count, long_row;
    if (threadIdx.x == 0) long_count = 0;
    __syncthreads();
    const uint32_t chunk = blockIdx.x * (kCombineBlock / 32) + warp;
    uint32_t row = kNoRow, count = 0;                           // chunks that follow
    if (chunk < s.chunks) {
        const uint32_t begin = chunk << j.chunk_log2, end = min(j.n, begin + (1u << j.chunk_log2));
        if (end < j.n) {
            row = __ldg(key + end - 1);
            const bool mine = row < j.total && __ldg(key + end) == row && (begin == 0 || __ldg(key + begin - 1) != row);
            if (mine) count = ((row_end(key, end, j.n, row) - 1) >> j.chunk_log2) - chunk;
        }
    }
    if (count > kLongSpan && lane == 0) { long_chunk = chunk; long_count = count; long_row = row; }
    if (count && count <= kLongSpan) {
        for (uint32_t c = lane * N; c < j.width; c += 32 * N) {
            float sum[N];
#pragma unroll
            for (int k = 0; k < N; k++) sum[k] = s.tail[(size_t)chunk * s.pitch + c + k];
#pragma unroll 4
            for (uint32_t q = 1; q <= count; q++) {
                const float* const part = s.head + (size_t)(chunk + q) * s.pitch + c;
#pragma unroll
                for (int k = 0; k < N; k++) sum[k] += part[k];
            }
            write_row<Out, N>(j, row, c, sum);
        }
    }
    __syncthreads();
    const uint32_t all = long_count;
    if (all == 0) return;
    const uint32_t per = (all + kCombineBlock / 32 - 1) / (kCombineBlock / 32), q0 = 1 + warp * per, q1 = min(all + 1, q0 + per);
    for (uint32_t c0 = 0; c0 < j.width; c0 += 32 * N) {
        const uint32_t c = c0 + lane * N;
        float sum[N] = {};
        if (c < j.width) {
            if (warp == 0) {
#pragma unroll
                for (int k = 0; k < N; k++) sum[k] = s.tail[(size_t)long_chunk * s.pitch + c + k];
            }
#pragma unroll 8
            for (uint32_t q = q0; q < q1; q++) {
                const float* const part = s.head + (size_t)(long_chunk + q) * s.pitch + c;
#pragma unroll
                for (int k = 0; k < N; k++) sum[k] += part[k];
            }
        }
#pragma unroll
        for (int k = 0; k < N; k++) slice[warp][lane * N + k] = sum[k];
        __syncthreads();
        if (warp == 0 && c < j.width) {
            for (int w = 1; w < kCombineBlock / 32; w++)
#pragma unroll
                for (int k = 0; k < N; k++) sum[k] += slice[w][lane * N + k];
            write_row<Out, N>(j, long_row, c, sum);
        }
        __syncthreads();
    }
}

// ---- host ---------------------------------------------------------------------------------------------------

// Entries of a chunk: enough chunks to fill the GPU, and no more parts than that needs.
int chunk_log2(uint64_t n) { return n < (1u << 17) ? 4 : n < (1u << 20) ? 5 : n < (1u << 22) ? 6 : 7; }
int bits_for(uint64_t keys) { int b = 1; while (b < 32 && (1ull << b) < keys) b++; return b; }      // of the largest key, keys - 1

size_t carve(uint64_t n, uint64_t total, uint32_t width, char* base, Space* s) {
    const auto up = [](size_t x) { return (x + 255) / 256 * 256; };
    size_t at = 0;
    const auto take = [&](size_t bytes) { char* const p = base ? base + at : nullptr; at += up(bytes); return p; };
    Space sp = {};
    if (n) {
        sp.tiles = (uint32_t)((n + kTile - 1) / kTile);
        sp.chunks = (uint32_t)((n + (1u << chunk_log2(n)) - 1) >> chunk_log2(n));
        sp.pitch = (width + 3) / 4 * 4;
        for (int k = 0; k < 2; k++) {
            sp.key[k] = reinterpret_cast<uint32_t*>(take(4 * n));
            sp.val[k] = reinterpret_cast<uint32_t*>(take(4 * n));
        }
        sp.counts = reinterpret_cast<uint32_t*>(take(4 * (size_t)sp.tiles * kMaxBins));
        sp.totals = reinterpret_cast<uint32_t*>(take(4 * kMaxBins));
        sp.head = reinterpret_cast<float*>(take(4 * (size_t)sp.chunks * sp.pitch));
        sp.tail = reinterpret_cast<float*>(take(4 * (size_t)sp.chunks * sp.pitch));
        sp.touched = reinterpret_cast<uint8_t*>(take(total));
    }
    if (s) *s = sp;
    return at;
}

// Sorts the entries; *which tells which of the two buffers holds them.
cudaError_t sort_entries(const Job& j, const Space& s, int* which, cudaStream_t st) {
    const int key_bits = bits_for((uint64_t)j.total + 1);
    if (j.n <= kSmall) {
        const int passes = (key_bits + kSmallDigitBits - 1) / kSmallDigitBits, bits = (key_bits + passes - 1) / passes;
        constexpr size_t smem = 4 * 4 * (size_t)kSmall + 32 * 2 * (1 << kSmallDigitBits) + 4 * (1 << kSmallDigitBits) + 4 * 32;
        const cudaError_t e = cudaFuncSetAttribute(small_sort_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        if (e != cudaSuccess) return e;
        small_sort_kernel<<<1, kSmallBlock, smem, st>>>(j, s, passes, bits);
        *which = 0;
        return cudaGetLastError();
    }
    const int passes = (key_bits + kMaxDigitBits - 1) / kMaxDigitBits, bits = (key_bits + passes - 1) / passes, bins = 1 << bits;
    const bool scanned = s.tiles > kScanTiles;
    const size_t smem = 4 * (size_t)bins + 2 * (size_t)bins * (kSortBlock / 32);
    for (int p = 0; p < passes; p++) {
        if (p == 0) count_kernel<true><<<s.tiles, kSortBlock, 0, st>>>(j, s, 0, 0, bits);
        else count_kernel<false><<<s.tiles, kSortBlock, 0, st>>>(j, s, p & 1, p * bits, bits);
        if (scanned) scan_kernel<<<(bins + 7) / 8, 256, 0, st>>>(s, bins);
        if (p == 0) scatter_kernel<true><<<s.tiles, kSortBlock, smem, st>>>(j, s, 0, 0, bits, scanned);
        else scatter_kernel<false><<<s.tiles, kSortBlock, smem, st>>>(j, s, p & 1, p * bits, bits, scanned);
    }
    *which = passes & 1;
    return cudaGetLastError();
}

template <typename T, typename Out, bool PAIRS>
cudaError_t sum_entries(const Job& j, const Space& s, int which, bool aligned, cudaStream_t st) {
    const uint32_t n_per = aligned ? 4 : 1, pieces = (j.width + n_per - 1) / n_per;
    int log2 = 0;
    while (log2 < 5 && (1u << log2) < pieces) log2++;
    const uint32_t teams_per_block = kReduceBlock >> log2;
    const dim3 grid((s.chunks + teams_per_block - 1) / teams_per_block, (pieces + (1u << log2) - 1) >> log2);
    const uint32_t combine_blocks = s.chunks > 1 ? (s.chunks + kCombineBlock / 32 - 1) / (kCombineBlock / 32) : 0;
    const uint32_t clear_blocks = j.accumulate ? 0 : (uint32_t)(((uint64_t)j.total + kCombineBlock - 1) / kCombineBlock);
    if (j.n) {
        if (aligned) reduce_kernel<T, Out, 4, PAIRS><<<grid, kReduceBlock, 0, st>>>(j, s, s.key[which], s.val[which], log2);
        else reduce_kernel<T, Out, 1, PAIRS><<<grid, kReduceBlock, 0, st>>>(j, s, s.key[which], s.val[which], log2);
    }
    if (combine_blocks + clear_blocks) {
        if (aligned) combine_kernel<Out, 4><<<combine_blocks + clear_blocks, kCombineBlock, 0, st>>>(j, s, s.key[which], combine_blocks);
        else combine_kernel<Out, 1><<<combine_blocks + clear_blocks, kCombineBlock, 0, st>>>(j, s, s.key[which], combine_blocks);
    }
    return cudaGetLastError();
}

int check_workspace(uint64_t n, uint64_t total, uint32_t width, void* workspace, uint64_t bytes) {
    const size_t need = carve(n, total, width, nullptr, nullptr);
    if (need == 0) return MASCOT_OK;
    if (!workspace || bytes < need) return fail(nullptr, MASCOT_ERR_BAD_ARG, "workspace: smaller than the *_workspace call says");
    if (reinterpret_cast<uintptr_t>(workspace) % 16) return fail(nullptr, MASCOT_ERR_BAD_ARG, "workspace: must be 16-byte aligned");
    return MASCOT_OK;
}

}  // namespace
}  // namespace mascot

using namespace mascot;

extern "C" {

int mascot_rows_gradient_workspace(uint64_t count, uint64_t rows, uint32_t width, uint64_t* bytes) {
    if (!bytes || count >= kMaxRows || rows >= kMaxRows || width == 0 || width > kMaxWidth) return fail(nullptr, MASCOT_ERR_BAD_ARG, "null pointer or size out of range");
    *bytes = carve(count, rows, width, nullptr, nullptr);
    return MASCOT_OK;
}

int mascot_pair_gradient_workspace(uint64_t count, uint64_t n_users, uint64_t n_items, uint32_t width, uint64_t* bytes) {
    if (!bytes || count >= kMaxRows || n_users >= kMaxRows || n_items >= kMaxRows || width == 0 || width > kMaxWidth || 3 * count >= kMaxRows || n_users + n_items >= kMaxRows)
        return fail(nullptr, MASCOT_ERR_BAD_ARG, "null pointer or size out of range");
    *bytes = carve(3 * count, n_users + n_items, width, nullptr, nullptr);
    return MASCOT_OK;
}

int mascot_rows_gradient(const mascot_rows* grad, const mascot_ids* ids, float scale, const mascot_rows* out, int accumulate, void* workspace,
                         uint64_t workspace_bytes, uint32_t* flags, void* stream) {
    ROW_CHECK(check_rows("grad", grad, false));
    ROW_CHECK(check_ids("ids", ids));
    ROW_CHECK(check_rows("out", out, false));
    if (grad->width != out->width) return fail(nullptr, MASCOT_ERR_BAD_ARG, "out: width is not the gradient's");
    if (grad->rows != ids->count) return fail(nullptr, MASCOT_ERR_BAD_ARG, "grad: must have a row for each id");
    ROW_CHECK(check_workspace(ids->count, out->rows, out->width, workspace, workspace_bytes));
    const size_t id_bytes = ids->count * ids->bits / 8;
    ROW_CHECK(check_distinct("grad", grad, "out", out));
    ROW_CHECK(check_distinct("ids", ids->data, id_bytes, "out", out));
    ROW_CHECK(check_distinct("workspace", workspace, workspace_bytes, "out", out));
    ROW_CHECK(check_distinct("workspace", workspace, workspace_bytes, "grad", grad));
    ROW_CHECK(check_distinct("workspace", workspace, workspace_bytes, "ids", ids->data, id_bytes));
    ROW_CHECK(check_distinct("workspace", workspace, workspace_bytes, "flags", flags, 4));
    ROW_CHECK(check_distinct("flags", flags, 4, "out", out));
    if (ids->count == 0 && (accumulate || out->rows == 0)) return MASCOT_OK;
    ROW_CHECK(check_device());
    if (ids->count) {
        ROW_CHECK(check_memory("grad", grad->data));
        ROW_CHECK(check_memory("ids", ids->data));
        ROW_CHECK(check_memory("workspace", workspace));
    }
    if (out->rows) ROW_CHECK(check_memory("out", out->data));
    ROW_CHECK(check_memory("flags", flags));
    Job j = {};
    j.ids[0] = ids_of(*ids);
    j.per = j.n = (uint32_t)ids->count;
    j.kinds = 1;
    j.rows[0] = j.total = (uint32_t)out->rows;
    j.src[0] = grad->data; j.src_stride[0] = grad->stride;
    j.out[0] = out->data; j.out_stride[0] = out->stride;
    j.width = out->width;
    j.chunk_log2 = chunk_log2(j.n);
    j.scale = scale; j.accumulate = accumulate != 0; j.flags = flags;
    Space s;
    carve(j.n, j.total, j.width, static_cast<char*>(workspace), &s);
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    int which = 0;
    if (j.n) CU(nullptr, sort_entries(j, s, &which, st));
    const bool aligned = aligned_rows(*grad, 4) && aligned_rows(*out, 4);
    const cudaError_t launched = with_type(grad->type, [&](auto* t) {
        return with_type(out->type, [&](auto* o) {
            return sum_entries<std::remove_pointer_t<decltype(t)>, std::remove_pointer_t<decltype(o)>, false>(j, s, which, aligned, st);
        });
    });
    CU(nullptr, launched);
    return MASCOT_OK;
}

int mascot_pair_gradient(const mascot_rows* P, const mascot_rows* Q, const mascot_ids* users, const mascot_ids* preferred, const mascot_ids* other,
                         const float* coef, float scale, const mascot_rows* dP, const mascot_rows* dQ, int accumulate, void* workspace,
                         uint64_t workspace_bytes, uint32_t* flags, void* stream) {
    const struct { const char* what; const mascot_rows* m; } mats[] = {{"P", P}, {"Q", Q}, {"dP", dP}, {"dQ", dQ}};
    const struct { const char* what; const mascot_ids* ids; } idss[] = {{"users", users}, {"preferred", preferred}, {"other", other}};
    for (const auto& m : mats) ROW_CHECK(check_rows(m.what, m.m, false));
    for (const auto& x : idss) ROW_CHECK(check_ids(x.what, x.ids));
    if (P->width != Q->width || P->type != Q->type) return fail(nullptr, MASCOT_ERR_BAD_ARG, "P and Q must have one width and one type");
    if (dP->rows != P->rows || dQ->rows != Q->rows || dP->width != P->width || dQ->width != P->width || dP->type != dQ->type)
        return fail(nullptr, MASCOT_ERR_BAD_ARG, "dP and dQ must have the shapes of P and Q, and one type");
    if (users->count != preferred->count || users->count != other->count) return fail(nullptr, MASCOT_ERR_BAD_ARG, "users, preferred and other must have one count");
    const uint64_t n = users->count, total = P->rows + Q->rows;
    if (3 * n >= kMaxRows || total >= kMaxRows) return fail(nullptr, MASCOT_ERR_BAD_ARG, "three times the pairs, and the rows of both tables, must be below 2^31 - 1");
    if (n && !coef) return fail(nullptr, MASCOT_ERR_BAD_ARG, "coef: null pointer");
    if (reinterpret_cast<uintptr_t>(coef) % 4) return fail(nullptr, MASCOT_ERR_BAD_ARG, "coef: address is not a multiple of the element's size");
    ROW_CHECK(check_workspace(3 * n, total, P->width, workspace, workspace_bytes));
    ROW_CHECK(check_distinct("dP", dP, "dQ", dQ));
    for (const auto* out : {dP, dQ}) {
        const char* const name = out == dP ? "dP" : "dQ";
        ROW_CHECK(check_distinct("P", P, name, out));
        ROW_CHECK(check_distinct("Q", Q, name, out));
        for (const auto& x : idss) ROW_CHECK(check_distinct(x.what, x.ids->data, n * x.ids->bits / 8, name, out));
        ROW_CHECK(check_distinct("coef", coef, n * 4, name, out));
        ROW_CHECK(check_distinct("flags", flags, 4, name, out));
    }
    for (const auto& m : mats) ROW_CHECK(check_distinct("workspace", workspace, workspace_bytes, m.what, m.m));
    for (const auto& x : idss) ROW_CHECK(check_distinct("workspace", workspace, workspace_bytes, x.what, x.ids->data, n * x.ids->bits / 8));
    ROW_CHECK(check_distinct("workspace", workspace, workspace_bytes, "coef", coef, n * 4));
    ROW_CHECK(check_distinct("workspace", workspace, workspace_bytes, "flags", flags, 4));
    if (n == 0 && (accumulate || total == 0)) return MASCOT_OK;
    ROW_CHECK(check_device());
    for (const auto& m : mats) if (m.m->rows) ROW_CHECK(check_memory(m.what, m.m->data));
    if (n) {
        for (const auto& x : idss) ROW_CHECK(check_memory(x.what, x.ids->data));
        ROW_CHECK(check_memory("coef", coef));
        ROW_CHECK(check_memory("workspace", workspace));
    }
    ROW_CHECK(check_memory("flags", flags));
    Job j = {};
    j.ids[0] = ids_of(*users); j.ids[1] = ids_of(*preferred); j.ids[2] = ids_of(*other);
    j.per = (uint32_t)n; j.kinds = 3; j.n = (uint32_t)(3 * n);
    j.rows[0] = (uint32_t)P->rows; j.rows[1] = (uint32_t)Q->rows; j.total = (uint32_t)total;
    j.src[0] = P->data; j.src[1] = Q->data;
    j.src_stride[0] = P->stride; j.src_stride[1] = Q->stride;
    j.coef = coef;
    j.out[0] = dP->data; j.out[1] = dQ->data;
    j.out_stride[0] = dP->stride; j.out_stride[1] = dQ->stride;
    j.width = P->width;
    j.chunk_log2 = chunk_log2(j.n);
    j.scale = scale; j.accumulate = accumulate != 0; j.flags = flags;
    Space s;
    carve(j.n, j.total, j.width, static_cast<char*>(workspace), &s);
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    int which = 0;
    if (j.n) CU(nullptr, sort_entries(j, s, &which, st));
    const bool aligned = aligned_rows(*P, 4) && aligned_rows(*Q, 4) && aligned_rows(*dP, 4) && aligned_rows(*dQ, 4);
    const cudaError_t launched = with_type(P->type, [&](auto* t) {
        return with_type(dP->type, [&](auto* o) {
            return sum_entries<std::remove_pointer_t<decltype(t)>, std::remove_pointer_t<decltype(o)>, true>(j, s, which, aligned, st);
        });
    });
    CU(nullptr, launched);
    return MASCOT_OK;
}

}  // extern "C"
