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
#include <initializer_list>

#include "launch_cache.h"
#include "row_ops.h"

namespace mascot {
namespace {

constexpr int kSortBlock = 512, kSortItems = 16, kTile = kSortBlock * kSortItems, kSortWarps = kSortBlock / 32;     // entries of a block of the sort
constexpr int kMaxDigitBits = 10, kMaxBins = 1 << kMaxDigitBits;
constexpr int kScanTiles = 32;                  // up to so many tiles the scatter kernel adds their counts up itself
constexpr int kSmallBlock = 1024, kSmallItems = 12, kSmallWarps = kSmallBlock / 32;
constexpr uint32_t kSmall = kSmallBlock * kSmallItems;
constexpr int kSmallDigitBits = 8, kSmallBins = 1 << kSmallDigitBits;
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
    uint32_t *key, *counts, *totals;            // rows of the entries as they come; [tiles][bins]; [bins]
    uint2* entry[2];                            // (row, entry)
    uint4* pair;                                // user, preferred, other, bits of coef
    float *head, *tail;                         // [chunks][pitch]
    uint8_t* touched;                           // a byte per row
    uint32_t pitch, chunks, tiles;
};

// ---- sort --------------------------------------------------------------------------------------------------

// Row of entry e, or `total`.  Pairs: the entry of the user also leaves the pair's rows where the sums find them.
__device__ __forceinline__ uint32_t entry_key(const Job& j, const Space& s, uint32_t e, bool& bad) {
    if (j.kinds == 1) {
        const uint32_t r = row_of(j.ids[0], e, j.rows[0], bad);
        return r == kNoRow ? j.total : r;
    }
    const uint32_t kind = e >= 2 * j.per ? 2 : e >= j.per ? 1 : 0, b = e - kind * j.per;
    const uint32_t u = row_of(j.ids[0], b, j.rows[0], bad), p = row_of(j.ids[1], b, j.rows[1], bad), o = row_of(j.ids[2], b, j.rows[1], bad);
    if (kind == 0) s.pair[b] = make_uint4(u, p, o, __float_as_uint(__ldg(j.coef + b)));
    if (u == kNoRow || p == kNoRow || o == kNoRow) return j.total;
    return kind == 0 ? u : j.rows[0] + (kind == 1 ? p : o);
}

__device__ __forceinline__ void clear_touched(uint8_t* touched, uint32_t rows, size_t first, size_t step) {
    for (size_t w = first; w < ((size_t)rows + 15) / 16; w += step) reinterpret_cast<uint4*>(touched)[w] = make_uint4(0, 0, 0, 0);
}

// Stable ranks of a warp's keys among the keys with the same digit that the warp has met so far; `count` is the
// warp's own row of counters, zero at first.
__device__ __forceinline__ uint32_t warp_rank(uint32_t digit, bool there, int bits, uint16_t* count, uint32_t lane) {
    uint32_t peers = __ballot_sync(0xffffffffu, there);
    for (int b = 0; b < bits; b++) {
        const uint32_t set = __ballot_sync(0xffffffffu, digit >> b & 1);
        peers &= digit >> b & 1 ? set : ~set;
    }
    const uint32_t below = __popc(peers & ((1u << lane) - 1u));
    uint32_t before = 0;
    if (there) before = count[digit];
    __syncwarp();
    if (there && below == 0) count[digit] = (uint16_t)(before + __popc(peers));
    __syncwarp();
    return before + below;
}

// Counters of `warps` warps, [warp][bins], become offsets of the warps within a bin, for two bins (2 b, 2 b + 1) at once; their sums come back.
__device__ __forceinline__ uint32_t warp_offsets(uint16_t* count, int warps, int bins, int b) {
    uint32_t sum = 0;                                           // two halves that never carry: at most 12288 entries
    for (int w = 0; w < warps; w++) {
        uint32_t* const c = reinterpret_cast<uint32_t*>(count + w * bins) + b;
        const uint32_t x = *c;
        *c = sum;
        sum += x;
    }
    return sum;
}

// Exclusive scan over `bins` values in shared memory by a whole block, in place; bins at most 2 * blockDim.x.
__device__ __forceinline__ void block_scan(uint32_t* v, int bins, uint32_t* warp_sums) {
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5, warps = blockDim.x >> 5;
    uint32_t x[2], sum = 0;
#pragma unroll
    for (int k = 0; k < 2; k++) { const int b = 2 * t + k; x[k] = b < bins ? v[b] : 0u; sum += x[k]; }
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
    for (int k = 0; k < 2; k++) { const int b = 2 * t + k; if (b < bins) v[b] = run; run += x[k]; }
    __syncthreads();
}

constexpr size_t kSmallSmem = 8 * (size_t)kSmall + 2 * (size_t)kSmallWarps * kSmallBins + 4 * kSmallBins + 4 * 32;

// One block: entries stay in registers while they are ranked and go through shared memory to their next place.  A sort over
// many blocks costs two launches a digit at least.
__global__ void __launch_bounds__(kSmallBlock) small_sort_kernel(const Job j, const Space s, int passes, int bits) {
    extern __shared__ uint2 at[];
    uint16_t* const count = reinterpret_cast<uint16_t*>(at + kSmall);
    uint32_t* const start = reinterpret_cast<uint32_t*>(count + kSmallWarps * kSmallBins), *const warp_sums = start + kSmallBins;
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5, bins = 1 << bits;
    if (!j.accumulate) clear_touched(s.touched, j.total, t, kSmallBlock);
    const uint32_t rounds = (j.n + kSmallBlock - 1) / kSmallBlock, first = warp * rounds * 32 + lane;      // a warp's entries, in order
    bool bad = false;
    uint2 e[kSmallItems];
#pragma unroll
    for (int k = 0; k < kSmallItems; k++) {
        const uint32_t i = first + k * 32;
        e[k] = make_uint2(0, i);
        if (k < rounds && i < j.n) e[k].x = entry_key(j, s, i, bad);
    }
    if (bad && j.flags) atomicOr(j.flags, (uint32_t)MASCOT_FLAG_BAD_ID);
    uint16_t* const mine = count + (warp << bits);
    for (int p = 0; p < passes; p++) {
        for (int b = lane; b < bins / 2; b += 32) reinterpret_cast<uint32_t*>(mine)[b] = 0;
        __syncwarp();
        uint32_t rank[kSmallItems];
#pragma unroll
        for (int k = 0; k < kSmallItems; k++)
            if (k < rounds) rank[k] = warp_rank(e[k].x >> (p * bits) & (bins - 1), first + k * 32 < j.n, bits, mine, lane);
        __syncthreads();
        for (int b = t; b < bins / 2; b += kSmallBlock) {
            const uint32_t sums = warp_offsets(count, kSmallWarps, bins, b);
            start[2 * b] = sums & 0xffff;
            start[2 * b + 1] = sums >> 16;
        }
        __syncthreads();
        block_scan(start, bins, warp_sums);
#pragma unroll
        for (int k = 0; k < kSmallItems; k++)
            if (k < rounds && first + k * 32 < j.n) { const uint32_t d = e[k].x >> (p * bits) & (bins - 1); at[start[d] + mine[d] + rank[k]] = e[k]; }
        __syncthreads();
        if (p + 1 < passes) {
#pragma unroll
            for (int k = 0; k < kSmallItems; k++) if (k < rounds && first + k * 32 < j.n) e[k] = at[first + k * 32];
            // `at` is written again only behind the next pass's barriers
        }
    }
    for (uint32_t i = t; i < j.n; i += kSmallBlock) s.entry[0][i] = at[i];
}

// Counts of the digits of a tile, [tile][bin].  The first pass makes the keys, and keeps them.
template <bool FIRST>
__global__ void __launch_bounds__(kSortBlock) count_kernel(const Job j, const Space s, int from, int shift, int bits) {
    __shared__ uint32_t hist[kMaxBins];
    const int bins = 1 << bits;
    for (int b = threadIdx.x; b < bins; b += kSortBlock) hist[b] = 0;
    if (FIRST && !j.accumulate) clear_touched(s.touched, j.total, (size_t)blockIdx.x * kSortBlock + threadIdx.x, (size_t)gridDim.x * kSortBlock);
    bool bad = false;
    uint32_t key[kSortItems];
#pragma unroll
    for (int k = 0; k < kSortItems; k++) {
        const uint32_t e = blockIdx.x * kTile + k * kSortBlock + threadIdx.x;
        if (e < j.n) key[k] = FIRST ? entry_key(j, s, e, bad) : s.entry[from][e].x;
    }
    if (FIRST && bad && j.flags) atomicOr(j.flags, (uint32_t)MASCOT_FLAG_BAD_ID);
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kSortItems; k++) {
        const uint32_t e = blockIdx.x * kTile + k * kSortBlock + threadIdx.x;
        if (e < j.n) {
            if (FIRST) s.key[e] = key[k];
            atomicAdd(&hist[key[k] >> shift & (bins - 1)], 1u);
        }
    }
    __syncthreads();
    for (int b = threadIdx.x; b < bins; b += kSortBlock) s.counts[(size_t)blockIdx.x * bins + b] = hist[b];
}

// A block for 32 bins, a warp for a run of tiles: counts of the tiles become offsets within the bin, the sums go to totals.
__global__ void __launch_bounds__(1024) scan_kernel(const Space s, int bins) {
    __shared__ uint32_t sums[32][32];
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5, bin = blockIdx.x * 32 + lane;
    const uint32_t per = (s.tiles + 31) / 32, t0 = min(s.tiles, warp * per), t1 = min(s.tiles, t0 + per);
    uint32_t sum = 0;
    if (bin < bins) {
#pragma unroll 8
        for (uint32_t t = t0; t < t1; t++) sum += s.counts[(size_t)t * bins + bin];
    }
    sums[warp][lane] = sum;
    __syncthreads();
    uint32_t run = 0;
    for (uint32_t w = 0; w < 32; w++) { const uint32_t x = sums[w][lane]; if (w < warp) run += x; else if (w == 31) break; }
    if (bin >= bins) return;
#pragma unroll 8
    for (uint32_t t = t0; t < t1; t++) {
        const uint32_t x = s.counts[(size_t)t * bins + bin];
        s.counts[(size_t)t * bins + bin] = run;
        run += x;
    }
    if (warp == 31) s.totals[bin] = run;
}

// Moves a tile's entries to their places: ranked by warps in the order of the entries, put in order in shared memory, and written from
// there, so that the entries of a bin leave as one run.
template <bool FIRST>
__global__ void __launch_bounds__(kSortBlock) scatter_kernel(const Job j, const Space s, int from, int shift, int bits, bool scanned) {
    extern __shared__ uint2 at[];                               // entries in their order; the warps' counters; the bins' offsets
    __shared__ uint32_t warp_sums[32];
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5, bins = 1 << bits;
    uint16_t* const count = reinterpret_cast<uint16_t*>(at + kTile), *const mine = count + (warp << bits);
    uint32_t* const start = reinterpret_cast<uint32_t*>(count + (kSortWarps << bits)), *const base = start + bins;
    for (int b = lane; b < bins / 2; b += 32) reinterpret_cast<uint32_t*>(mine)[b] = 0;
    const uint32_t first = blockIdx.x * kTile + warp * (32 * kSortItems) + lane;
    uint2 e[kSortItems];
#pragma unroll
    for (int k = 0; k < kSortItems; k++) {
        const uint32_t i = first + k * 32;
        e[k] = make_uint2(0, i);
        if (i < j.n) { if (FIRST) e[k].x = s.key[i]; else e[k] = s.entry[from][i]; }
    }
    uint32_t within[kMaxBins / kSortBlock];                     // entries of the bin in the tiles before
#pragma unroll
    for (int k = 0; k < kMaxBins / kSortBlock; k++) {
        const int b = t + k * kSortBlock;
        within[k] = 0;
        if (b < bins) {
            uint32_t sum = 0;
            if (scanned) { within[k] = s.counts[(size_t)blockIdx.x * bins + b]; sum = s.totals[b]; }
            else {
#pragma unroll 8
                for (uint32_t q = 0; q < s.tiles; q++) { if (q == blockIdx.x) within[k] = sum; sum += s.counts[(size_t)q * bins + b]; }
            }
            base[b] = sum;
        }
    }
    __syncwarp();
    uint32_t rank[kSortItems];
#pragma unroll
    for (int k = 0; k < kSortItems; k++) rank[k] = warp_rank(e[k].x >> shift & (bins - 1), first + k * 32 < j.n, bits, mine, lane);
    __syncthreads();
    for (int b = t; b < bins / 2; b += kSortBlock) {
        const uint32_t sums = warp_offsets(count, kSortWarps, bins, b);
        start[2 * b] = sums & 0xffff;
        start[2 * b + 1] = sums >> 16;
    }
    block_scan(base, bins, warp_sums);
    block_scan(start, bins, warp_sums);
#pragma unroll
    for (int k = 0; k < kMaxBins / kSortBlock; k++) { const int b = t + k * kSortBlock; if (b < bins) base[b] += within[k] - start[b]; }
#pragma unroll
    for (int k = 0; k < kSortItems; k++)
        if (first + k * 32 < j.n) { const uint32_t d = e[k].x >> shift & (bins - 1); at[start[d] + mine[d] + rank[k]] = e[k]; }
    __syncthreads();
    const uint32_t here = min((uint32_t)kTile, j.n - blockIdx.x * kTile);
#pragma unroll 4
    for (uint32_t i = t; i < here; i += kSortBlock) { const uint2 x = at[i]; s.entry[from ^ 1][i + base[x.x >> shift & (bins - 1)]] = x; }
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

// A team's lanes take a group of entries each, one round trip for all of them, and hand them round; the rows of BATCH
// entries are in flight at once.  What bounds it is those rows: random ones, from HBM or L2.
template <typename T, typename Out, int N, bool PAIRS>
__global__ void __launch_bounds__(kReduceBlock) reduce_kernel(const Job j, const Space s, const uint2* entry, int team_log2) {
    constexpr int BATCH = PAIRS ? 4 : 8;
    const uint32_t team = 1u << team_log2, tl = threadIdx.x & (team - 1);
    const uint32_t chunk = (blockIdx.x * kReduceBlock + threadIdx.x) >> team_log2, col = ((blockIdx.y << team_log2) + tl) * N;
    const bool writes = chunk < s.chunks && col < j.width;
    const uint32_t begin = min(j.n, chunk << j.chunk_log2), end = min(j.n, begin + (1u << j.chunk_log2));
    const uint32_t before = chunk < s.chunks && begin ? __ldg(&entry[begin - 1].x) : kNoRow, after = end < j.n ? __ldg(&entry[end].x) : kNoRow;
    const T* const src0 = static_cast<const T*>(j.src[0]) + col, *const src1 = static_cast<const T*>(j.src[1]) + col;
    uint32_t row = kNoRow;
    float sum[N] = {};
    const auto flush = [&]() {
        if (row >= j.total || !writes) return;
        if (row == before || row == after) {                   // part of a row that other chunks share
            float* const part = (row == before ? s.head : s.tail) + (size_t)chunk * s.pitch + col;
#pragma unroll
            for (int k = 0; k < N; k++) part[k] = sum[k];
        } else write_row<Out, N>(j, row, col, sum);
        if (row != before && !j.accumulate && col == 0) s.touched[row] = 1;
    };
    for (uint32_t g = begin; __any_sync(0xffffffffu, g < end); g += team) {
        uint2 mine = make_uint2(j.total, 0);
        if (g + tl < end) mine = __ldg(entry + g + tl);
        uint32_t my_a = mine.y, my_b = kNoRow;
        float my_c = 1.f;
        if (PAIRS && mine.x < j.total) {
            const uint32_t kind = mine.y >= 2 * j.per ? 2 : mine.y >= j.per ? 1 : 0;
            const uint4 p = __ldg(s.pair + (mine.y - kind * j.per));
            my_c = kind == 2 ? -__uint_as_float(p.w) : __uint_as_float(p.w);
            my_a = kind ? p.x : p.y;
            if (kind == 0) my_b = p.z;
        }
        for (uint32_t k0 = 0; k0 < team; k0 += BATCH) {
            if (!__any_sync(0xffffffffu, g + k0 < end)) break;
            uint32_t key[BATCH], b_row[BATCH];
            float c[BATCH];
            Piece<T, N> a[BATCH], b[BATCH];
#pragma unroll
            for (int k = 0; k < BATCH; k++) {
                key[k] = __shfl_sync(0xffffffffu, mine.x, k0 + k, team);
                const uint32_t a_row = __shfl_sync(0xffffffffu, my_a, k0 + k, team);
                c[k] = PAIRS ? __shfl_sync(0xffffffffu, my_c, k0 + k, team) : 1.f;
                b_row[k] = PAIRS ? __shfl_sync(0xffffffffu, my_b, k0 + k, team) : kNoRow;
                if (key[k] >= j.total || !writes) c[k] = 0.f;   // coef 0: whatever the rows hold
                if (c[k] != 0.f) {
                    a[k] = load_piece<T, N>(!PAIRS || b_row[k] == kNoRow ? src0 + a_row * j.src_stride[0] : src1 + a_row * j.src_stride[1]);
                    if (PAIRS && b_row[k] != kNoRow) b[k] = load_piece<T, N>(src1 + b_row[k] * j.src_stride[1]);
                }
            }
#pragma unroll
            for (int k = 0; k < BATCH; k++) {
                if (key[k] != row) {
                    flush();
                    row = key[k];
#pragma unroll
                    for (int x = 0; x < N; x++) sum[x] = 0.f;
                }
                if (c[k] != 0.f) {
#pragma unroll
                    for (int x = 0; x < N; x++) {
                        if (!PAIRS) sum[x] += as_float(a[k].v[x]);
                        else sum[x] = fmaf(c[k], b_row[k] != kNoRow ? as_float(a[k].v[x]) - as_float(b[k].v[x]) : as_float(a[k].v[x]), sum[x]);
                    }
                }
            }
        }
    }
    flush();
}

// The first position behind the entries of `row`, searched by a warp from `at`, which is one of them: 32 places at a time.
__device__ __forceinline__ uint32_t row_end(const uint2* entry, uint32_t at, uint32_t n, uint32_t row, uint32_t lane) {
    uint32_t lo = at, hi = n;                                   // the entry at lo is one, that at hi is none
    while (hi - lo > 1) {
        const uint32_t step = (hi - lo + 31) / 32, mid = lo + lane * step;      // lane 0: lo
        const uint32_t in = __popc(__ballot_sync(0xffffffffu, mid < hi && __ldg(&entry[mid].x) == row));      // the first `in` places
        hi = min(hi, lo + in * step);
        lo += (in - 1) * step;
    }
    return hi;
}

// Blocks below `combine_blocks`: a warp per chunk adds up the row that begins in it and goes on behind it.  A row over
// more than kLongSpan chunks is added up by all warps of the block, a slice each: only one row a block can be that long, since it
// covers all chunks of the block behind its first.  The other blocks clear the rows that no entry names, a warp for 32 of them.
template <typename Out, int N>
__global__ void __launch_bounds__(kCombineBlock) combine_kernel(const Job j, const Space s, const uint2* entry, uint32_t combine_blocks) {
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
            row = __ldg(&entry[end - 1].x);
            const uint32_t next = __ldg(&entry[end].x), before = begin ? __ldg(&entry[begin - 1].x) : kNoRow;
            if (row < j.total && next == row && before != row) {
                // most rows end in the next 32 chunks: lane q looks at the end of chunk q + 1 behind this one
                const uint64_t last = ((uint64_t)(chunk + 2 + lane) << j.chunk_log2) - 1;
                const uint32_t through = __ballot_sync(0xffffffffu, last + 1 < j.n && __ldg(&entry[last].x) == row && __ldg(&entry[last + 1].x) == row);
                count = through != 0xffffffffu ? __ffs(~through) : ((row_end(entry, end, j.n, row, lane) - 1) >> j.chunk_log2) - chunk;
            }
        }
    }
    if (count > kLongSpan && lane == 0) { long_chunk = chunk; long_count = count; long_row = row; }
    if (count && count <= kLongSpan) {
        for (uint32_t c = lane * N; c < j.width; c += 32 * N) {
            float sum[N];
#pragma unroll
            for (int k = 0; k < N; k++) sum[k] = s.tail[(size_t)chunk * s.pitch + c + k];
#pragma unroll 8
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
int chunk_log2(uint64_t n) { return n < (1u << 17) ? 4 : n < (1u << 19) ? 5 : n < (1u << 21) ? 6 : 7; }
int bits_for(uint64_t keys) { int b = 1; while (b < 32 && (1ull << b) < keys) b++; return b; }      // of the largest key, keys - 1

size_t carve(uint64_t n, uint64_t total, uint32_t width, bool pairs, char* base, Space* s) {
    size_t at = 0;
    const auto take = [&](size_t bytes) { char* const p = base ? base + at : nullptr; at += (bytes + 255) / 256 * 256; return p; };
    Space sp = {};
    if (n) {
        sp.tiles = (uint32_t)((n + kTile - 1) / kTile);
        sp.chunks = (uint32_t)((n + (1u << chunk_log2(n)) - 1) >> chunk_log2(n));
        sp.pitch = (width + 3) / 4 * 4;
        const bool small = n <= kSmall;
        sp.entry[0] = reinterpret_cast<uint2*>(take(8 * n));
        sp.entry[1] = reinterpret_cast<uint2*>(take(small ? 0 : 8 * n));
        sp.key = reinterpret_cast<uint32_t*>(take(small ? 0 : 4 * n));
        sp.counts = reinterpret_cast<uint32_t*>(take(small ? 0 : 4 * (size_t)sp.tiles * kMaxBins));
        sp.totals = reinterpret_cast<uint32_t*>(take(small ? 0 : 4 * kMaxBins));
        sp.pair = reinterpret_cast<uint4*>(take(pairs ? 16 * (n / 3) : 0));
        sp.head = reinterpret_cast<float*>(take(4 * (size_t)sp.chunks * sp.pitch));
        sp.tail = reinterpret_cast<float*>(take(4 * (size_t)sp.chunks * sp.pitch));
        sp.touched = reinterpret_cast<uint8_t*>(take(total));
    }
    if (s) *s = sp;
    return at;
}

// Raises a kernel's limit of dynamic shared memory, once for a device.
template <class Kernel>
cudaError_t allow_smem(Kernel kernel, size_t bytes, LaunchCache& cache) {
    int dev = 0, fit = 0;
    const cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    return (cudaError_t)cache.lookup(dev, 0, 0, bytes, [&](size_t most) { return (int)cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)most); },
                                     [](int, size_t, int*) { return 0; }, &fit);
}

constexpr size_t scatter_smem(int bins) { return 8 * (size_t)kTile + 2 * (size_t)bins * kSortWarps + 8 * (size_t)bins; }

// Sorts the entries; *which tells which of the two buffers holds them.
cudaError_t sort_entries(const Job& j, const Space& s, int* which, cudaStream_t st) {
    static LaunchCache small_cache, first_cache, next_cache;
    const int key_bits = bits_for((uint64_t)j.total + 1);
    if (j.n <= kSmall) {
        const int passes = (key_bits + kSmallDigitBits - 1) / kSmallDigitBits, bits = (key_bits + passes - 1) / passes;
        const cudaError_t e = allow_smem(small_sort_kernel, kSmallSmem, small_cache);
        if (e != cudaSuccess) return e;
        small_sort_kernel<<<1, kSmallBlock, kSmallSmem, st>>>(j, s, passes, bits);
        *which = 0;
        return cudaGetLastError();
    }
    const int passes = (key_bits + kMaxDigitBits - 1) / kMaxDigitBits, bits = (key_bits + passes - 1) / passes, bins = 1 << bits;
    const bool scanned = s.tiles > kScanTiles;
    cudaError_t e = allow_smem(scatter_kernel<true>, scatter_smem(kMaxBins), first_cache);
    if (e == cudaSuccess) e = allow_smem(scatter_kernel<false>, scatter_smem(kMaxBins), next_cache);
    if (e != cudaSuccess) return e;
    for (int p = 0; p < passes; p++) {
        const int from = p & 1;                                 // the first pass takes its entries from `key` and leaves them in entry[1]
        if (p == 0) count_kernel<true><<<s.tiles, kSortBlock, 0, st>>>(j, s, from, 0, bits);
        else count_kernel<false><<<s.tiles, kSortBlock, 0, st>>>(j, s, from, p * bits, bits);
        if (scanned) scan_kernel<<<(bins + 31) / 32, 1024, 0, st>>>(s, bins);
        if (p == 0) scatter_kernel<true><<<s.tiles, kSortBlock, scatter_smem(bins), st>>>(j, s, from, 0, bits, scanned);
        else scatter_kernel<false><<<s.tiles, kSortBlock, scatter_smem(bins), st>>>(j, s, from, p * bits, bits, scanned);
    }
    *which = passes & 1;
    return cudaGetLastError();
}

template <typename T, typename Out, int N, bool PAIRS>
cudaError_t sum_pieces(const Job& j, const Space& s, int which, cudaStream_t st) {
    const uint32_t pieces = (j.width + N - 1) / N;
    int log2 = 3;
    while (log2 < 5 && (1u << log2) < pieces) log2++;
    const uint32_t teams_per_block = kReduceBlock >> log2;
    const dim3 grid((s.chunks + teams_per_block - 1) / teams_per_block, (pieces + (1u << log2) - 1) >> log2);
    const uint32_t combine_blocks = s.chunks > 1 ? (s.chunks + kCombineBlock / 32 - 1) / (kCombineBlock / 32) : 0;
    const uint32_t clear_blocks = j.accumulate ? 0 : (uint32_t)(((uint64_t)j.total + kCombineBlock - 1) / kCombineBlock);
    if (j.n) reduce_kernel<T, Out, N, PAIRS><<<grid, kReduceBlock, 0, st>>>(j, s, s.entry[which], log2);
    if (combine_blocks + clear_blocks) combine_kernel<Out, (N < 4 ? N : 4)><<<combine_blocks + clear_blocks, kCombineBlock, 0, st>>>(j, s, s.entry[which], combine_blocks);
    return cudaGetLastError();
}

// `pieces`: elements that all rows may be moved in.
template <typename T, typename Out, bool PAIRS>
cudaError_t sum_entries(const Job& j, const Space& s, int which, uint32_t pieces, cudaStream_t st) {
    if (sizeof(T) == 2 && pieces == 8) return sum_pieces<T, Out, (sizeof(T) == 2 ? 8 : 4), PAIRS>(j, s, which, st);
    return pieces >= 4 ? sum_pieces<T, Out, 4, PAIRS>(j, s, which, st) : sum_pieces<T, Out, 1, PAIRS>(j, s, which, st);
}
uint32_t pieces_of(std::initializer_list<const mascot_rows*> all) {
    uint32_t n = 8;
    for (const mascot_rows* m : all) n = aligned_rows(*m, n) ? n : aligned_rows(*m, 4) ? 4 : 1;
    return n;
}

int check_workspace(uint64_t n, uint64_t total, uint32_t width, bool pairs, void* workspace, uint64_t bytes) {
    const size_t need = carve(n, total, width, pairs, nullptr, nullptr);
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
    *bytes = carve(count, rows, width, false, nullptr, nullptr);
    return MASCOT_OK;
}

int mascot_pair_gradient_workspace(uint64_t count, uint64_t n_users, uint64_t n_items, uint32_t width, uint64_t* bytes) {
    if (!bytes || count >= kMaxRows || n_users >= kMaxRows || n_items >= kMaxRows || width == 0 || width > kMaxWidth || 3 * count >= kMaxRows || n_users + n_items >= kMaxRows)
        return fail(nullptr, MASCOT_ERR_BAD_ARG, "null pointer or size out of range");
    *bytes = carve(3 * count, n_users + n_items, width, true, nullptr, nullptr);
    return MASCOT_OK;
}

int mascot_rows_gradient(const mascot_rows* grad, const mascot_ids* ids, float scale, const mascot_rows* out, int accumulate, void* workspace,
                         uint64_t workspace_bytes, uint32_t* flags, void* stream) {
    ROW_CHECK(check_rows("grad", grad, false));
    ROW_CHECK(check_ids("ids", ids));
    ROW_CHECK(check_rows("out", out, false));
    if (grad->width != out->width) return fail(nullptr, MASCOT_ERR_BAD_ARG, "out: width is not the gradient's");
    if (grad->rows != ids->count) return fail(nullptr, MASCOT_ERR_BAD_ARG, "grad: must have a row for each id");
    ROW_CHECK(check_workspace(ids->count, out->rows, out->width, false, workspace, workspace_bytes));
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
    carve(j.n, j.total, j.width, false, static_cast<char*>(workspace), &s);
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    int which = 0;
    if (j.n) CU(nullptr, sort_entries(j, s, &which, st));
    const uint32_t pieces = pieces_of({grad, out});
    const cudaError_t launched = with_type(grad->type, [&](auto* t) {
        return with_type(out->type, [&](auto* o) {
            return sum_entries<std::remove_pointer_t<decltype(t)>, std::remove_pointer_t<decltype(o)>, false>(j, s, which, pieces, st);
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
    ROW_CHECK(check_workspace(3 * n, total, P->width, true, workspace, workspace_bytes));
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
    carve(j.n, j.total, j.width, true, static_cast<char*>(workspace), &s);
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    int which = 0;
    if (j.n) CU(nullptr, sort_entries(j, s, &which, st));
    const uint32_t pieces = pieces_of({P, Q, dP, dQ});
    const cudaError_t launched = with_type(P->type, [&](auto* t) {
        return with_type(dP->type, [&](auto* o) {
            return sum_entries<std::remove_pointer_t<decltype(t)>, std::remove_pointer_t<decltype(o)>, true>(j, s, which, pieces, st);
        });
    });
    CU(nullptr, launched);
    return MASCOT_OK;
}

}  // extern "C"
