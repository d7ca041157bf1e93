// Sums by row: the gradient of a row lookup, and the gradients of the preference loss in both factor tables.
//
// Both are  out[r] = scale * sum over the entries e of row r of value(e),  where an entry is a place that looked a row up, and
// a value a row of its own: a gradient row (lookup), or c * (Q[i] - Q[j]) for the user and +-c * P[u] for the two items of a
// pair.  Atomic additions would settle the order of a sum by chance; here the entries are sorted by row, stably, and then
// summed in that order, in fp32:
//
//   sort     least significant digit first, on (row, entry) pairs of 32 bits each.  All entries of both tables are sorted at once,
//            the items' rows counted behind the users'.  Up to kSmall entries one cluster of blocks does all passes;
//            more take count / scan / scatter kernels for each digit.
//   reduce   the sorted entries are cut into chunks of equal length, a team of lanes for each, so that a popular row is
//            shared by many teams and many unpopular ones by one.  A row that ends less than a quarter of a chunk behind a chunk's
//            end is finished by that chunk's team; of one that goes on further, each chunk's part is left in the workspace.
//   combine  adds these parts up in the order of the chunks, and clears rows that no entry names.
#include <cooperative_groups.h>

#include <algorithm>
#include <initializer_list>

#include "row_ops.h"

namespace mascot {
namespace {

namespace cg = cooperative_groups;

constexpr int kSortBlock = 512, kSortWarps = kSortBlock / 32;
constexpr int kFewItems = 4, kManyItems = 16;   // entries of a thread of the sort: a tile is 2048 or 8192
constexpr uint32_t kManyFrom = 1u << 20;        // entries from which tiles are large: there are enough of them for all SMs then
constexpr int kMaxBins = 1024;                  // digits of 8 or 10 bits
constexpr uint32_t kScanTiles = 16;             // up to so many tiles the scatter kernel adds their counts up itself
constexpr int kSmallBlock = 512, kSmallItems = 8, kSmallWarps = kSmallBlock / 32, kSmallBits = 8, kSmallBins = 1 << kSmallBits;
constexpr uint32_t kSmallCluster = 8, kSmall = kSmallBlock * kSmallItems * kSmallCluster;
constexpr int kReduceBlock = 256, kCombineBlock = 512;

// What is summed: where entries come from and what their values are.
struct Job {
    Ids ids[3];                                 // lookup: one; pairs: users, preferred, other
    uint32_t kinds;                             // 1: lookup, 3: pairs; entry e of pairs is id e / 3 of kind e % 3, so that a tile of entries is one of pairs
    uint32_t n;                                 // entries: kinds * ids of one kind
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
    uint2* owners;                              // (chunk, row) where a row begins whose parts are added up
    uint32_t* n_owners;
    uint8_t* touched;                           // a byte per row
    uint32_t pitch, chunks, tiles;
};

// For kernels that launch_behind launches, and those before them: the next kernel's blocks may be brought up; the kernel before has ended.
// What one kernel of a call leaves for the next is read with plain loads, since it changes while the next one's blocks are already there.
__device__ __forceinline__ void follow() {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
}

// ---- sort --------------------------------------------------------------------------------------------------

// Rows, or `total`, of COUNT entries `step` apart, as far as there are so many; all loads are under way at once.  Pairs: the entry of the
// user also leaves the pair where the sums find it.
template <int COUNT>
__device__ __forceinline__ void entry_keys(const Job& j, const Space& s, uint32_t first, uint32_t step, uint32_t (&key)[COUNT], bool& bad) {
    uint32_t at[COUNT];
#pragma unroll
    for (int k = 0; k < COUNT; k++) at[k] = min(first + k * step, j.n - 1) / j.kinds;
    if (j.kinds == 1) {
        RawId id[COUNT];
        load_ids<COUNT>(j.ids[0], at, id);
#pragma unroll
        for (int k = 0; k < COUNT; k++) {
            const uint32_t r = row_of(id[k], j.ids[0], j.rows[0], bad);
            key[k] = r == kNoRow ? j.total : r;
        }
        return;
    }
    RawId u[COUNT], p[COUNT], o[COUNT];
    load_ids<COUNT>(j.ids[0], at, u);
    load_ids<COUNT>(j.ids[1], at, p);
    load_ids<COUNT>(j.ids[2], at, o);
#pragma unroll
    for (int k = 0; k < COUNT; k++) {
        const uint32_t e = first + k * step, b = e / 3, kind = e - 3 * b;
        const uint32_t ur = row_of(u[k], j.ids[0], j.rows[0], bad), pr = row_of(p[k], j.ids[1], j.rows[1], bad), orow = row_of(o[k], j.ids[2], j.rows[1], bad);
        if (e < j.n && kind == 0) s.pair[b] = make_uint4(ur, pr, orow, __float_as_uint(__ldg(j.coef + b)));
        key[k] = ur == kNoRow || pr == kNoRow || orow == kNoRow ? j.total : kind == 0 ? ur : j.rows[0] + (kind == 1 ? pr : orow);
    }
}

// Stable ranks of a warp's keys among the keys with the same digit that the warp has met so far; `count` is the
// warp's own row of counters, zero at first.
template <int BITS> __device__ __forceinline__ uint32_t warp_rank(uint32_t digit, bool there, uint16_t* count, uint32_t lane) {
    uint32_t peers = __ballot_sync(0xffffffffu, there);
#pragma unroll
    for (int b = 0; b < BITS; b++) {
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
    uint32_t sum = 0;                                           // two halves that never carry: a tile has at most 8192 entries
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

__device__ __forceinline__ void begin_sums(const Job& j, const Space& s, size_t first, size_t step) {
    if (first == 0) *s.n_owners = 0;
    if (!j.accumulate) for (size_t w = first; w < ((size_t)j.total + 15) / 16; w += step) reinterpret_cast<uint4*>(s.touched)[w] = make_uint4(0, 0, 0, 0);
}

// One cluster of eight blocks (one block for the fewest entries), a tile of entries each, that tell one another their counts through distributed shared memory and
// meet twice a pass: 12,288 entries in two passes take 14 us; kernels of their own for each pass took 32.
__global__ void __launch_bounds__(kSmallBlock) small_sort_kernel(const Job j, const Space s, int passes) {
    __shared__ uint2 at[kSmallBlock * kSmallItems];
    __shared__ __align__(16) uint16_t count[kSmallWarps * kSmallBins];
    __shared__ uint32_t counts[kSmallBins], start[kSmallBins], base[kSmallBins], warp_sums[32];
    follow();
    cg::cluster_group cluster = cg::this_cluster();
    const uint32_t blocks = cluster.num_blocks(), block = cluster.block_rank();
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
    begin_sums(j, s, block * kSmallBlock + t, blocks * kSmallBlock);
    const uint32_t rounds = (j.n + blocks * kSmallBlock - 1) / (blocks * kSmallBlock), tile0 = block * rounds * kSmallBlock;
    const uint32_t here = j.n > tile0 ? min(rounds * kSmallBlock, j.n - tile0) : 0, mine0 = warp * rounds * 32 + lane;      // a warp's entries, in order
    uint32_t key[kSmallItems], val[kSmallItems];
    bool bad = false;
    entry_keys<kSmallItems>(j, s, tile0 + mine0, 32, key, bad);
#pragma unroll
    for (int k = 0; k < kSmallItems; k++) val[k] = tile0 + mine0 + k * 32;
    if (bad && j.flags) atomicOr(j.flags, (uint32_t)MASCOT_FLAG_BAD_ID);
    uint16_t* const mine = count + warp * kSmallBins;
    for (int p = 0; p < passes; p++) {
        const int shift = p * kSmallBits;
        reinterpret_cast<uint4*>(mine)[lane] = make_uint4(0, 0, 0, 0);
        __syncwarp();
        uint32_t rank[kSmallItems];
#pragma unroll
        for (int k = 0; k < kSmallItems; k++)
            if (k < rounds) rank[k] = warp_rank<kSmallBits>(key[k] >> shift & (kSmallBins - 1), mine0 + k * 32 < here, mine, lane);
        __syncthreads();
        if (t < kSmallBins / 2) {
            const uint32_t sums = warp_offsets(count, kSmallWarps, kSmallBins, t);
            counts[2 * t] = start[2 * t] = sums & 0xffff;
            counts[2 * t + 1] = start[2 * t + 1] = sums >> 16;
        }
        cluster.sync();
        uint32_t within = 0;                                    // entries of the bin in the tiles before
        if (t < kSmallBins) {
            uint32_t of[kSmallCluster], sum = 0;
#pragma unroll
            for (uint32_t b = 0; b < kSmallCluster; b++) of[b] = b < blocks ? *cluster.map_shared_rank(&counts[t], b) : 0u;
#pragma unroll
            for (uint32_t b = 0; b < kSmallCluster; b++) { if (b == block) within = sum; sum += of[b]; }
            base[t] = sum;
        }
        __syncthreads();
        block_scan(start, kSmallBins, warp_sums);
        block_scan(base, kSmallBins, warp_sums);
        if (t < kSmallBins) base[t] += within - start[t];
#pragma unroll
        for (int k = 0; k < kSmallItems; k++)
            if (k < rounds && mine0 + k * 32 < here) { const uint32_t d = key[k] >> shift & (kSmallBins - 1); at[start[d] + mine[d] + rank[k]] = make_uint2(key[k], val[k]); }
        __syncthreads();
        uint2* const to = s.entry[p & 1];
        for (uint32_t i = t; i < here; i += kSmallBlock) { const uint2 x = at[i]; to[i + base[x.x >> shift & (kSmallBins - 1)]] = x; }
        cluster.sync();                                         // also before a block leaves whose counts another one may read
        if (p + 1 < passes) {
#pragma unroll
            for (int k = 0; k < kSmallItems; k++)
                if (k < rounds && mine0 + k * 32 < here) { const uint2 x = __ldcg(to + tile0 + mine0 + k * 32); key[k] = x.x; val[k] = x.y; }
        }
    }
}

// Counts of the digits of a tile, [tile][bin].  The first pass makes the keys, and keeps them.
template <bool FIRST, int ITEMS>
__global__ void __launch_bounds__(kSortBlock) count_kernel(const Job j, const Space s, const uint2* entry, int shift, int bits) {
    __shared__ uint32_t hist[kMaxBins];
    follow();
    const int bins = 1 << bits;
    for (int b = threadIdx.x; b < bins; b += kSortBlock) hist[b] = 0;
    if (FIRST) begin_sums(j, s, (size_t)blockIdx.x * kSortBlock + threadIdx.x, (size_t)gridDim.x * kSortBlock);
    const uint32_t first = blockIdx.x * (ITEMS * kSortBlock) + threadIdx.x;
    uint32_t key[ITEMS];
    if (FIRST) {
        bool bad = false;
#pragma unroll
        for (int k = 0; k < ITEMS; k += 4) {
            uint32_t four[4];
            entry_keys<4>(j, s, first + k * kSortBlock, kSortBlock, four, bad);
#pragma unroll
            for (int q = 0; q < 4; q++) key[k + q] = four[q];
        }
        if (bad && j.flags) atomicOr(j.flags, (uint32_t)MASCOT_FLAG_BAD_ID);
    } else {
#pragma unroll
        for (int k = 0; k < ITEMS; k++) key[k] = entry[min(first + k * kSortBlock, j.n - 1)].x;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < ITEMS; k++) {
        const uint32_t e = first + k * kSortBlock;
        if (e < j.n) {
            if (FIRST) s.key[e] = key[k];
            atomicAdd(&hist[key[k] >> shift & (bins - 1)], 1u);
        }
    }
    __syncthreads();
    for (int b = threadIdx.x; b < bins; b += kSortBlock) s.counts[(size_t)blockIdx.x * bins + b] = hist[b];
}

// A block for 32 bins of 256 or 1024, a warp for a run of tiles: counts of the tiles become offsets within the bin, the sums go to totals.
__global__ void __launch_bounds__(1024) scan_kernel(const Space s, int bins) {
    __shared__ uint32_t sums[32][32];
    follow();
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5, bin = blockIdx.x * 32 + lane;
    const uint32_t per = (s.tiles + 31) / 32, t0 = min(s.tiles, warp * per), t1 = min(s.tiles, t0 + per);
    uint32_t sum = 0;
#pragma unroll 8
    for (uint32_t t = t0; t < t1; t++) sum += s.counts[(size_t)t * bins + bin];
    sums[warp][lane] = sum;
    __syncthreads();
    uint32_t run = 0;
    for (uint32_t w = 0; w < warp; w++) run += sums[w][lane];
#pragma unroll 8
    for (uint32_t t = t0; t < t1; t++) {
        const uint32_t x = s.counts[(size_t)t * bins + bin];
        s.counts[(size_t)t * bins + bin] = run;
        run += x;
    }
    if (warp == 31) s.totals[bin] = run;
}

// Moves a tile's entries to their places: ranked by warps in the order of the entries, put in order in shared memory, and written from
// there, so that the entries of a bin leave as one run (4M entries: 40 us a digit, 80 when they left one by one).  Bound by the
// instructions of the ranking: a vote for each bit of the digit.
template <bool FIRST, int ITEMS, int BITS>
__global__ void __launch_bounds__(kSortBlock, 2) scatter_kernel(const Space s, uint32_t n, const uint2* from, uint2* to, int shift, bool scanned) {
    extern __shared__ uint2 at[];                               // entries in their order; the warps' counters; the bins' offsets
    __shared__ uint32_t warp_sums[32];
    follow();
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
    constexpr int bins = 1 << BITS, kTile = ITEMS * kSortBlock, kPer = (bins + kSortBlock - 1) / kSortBlock;
    uint16_t* const count = reinterpret_cast<uint16_t*>(at + kTile), *const mine = count + (warp << BITS);
    uint32_t* const start = reinterpret_cast<uint32_t*>(count + (kSortWarps << BITS)), *const base = start + bins;
    for (int b = lane; b < bins / 2; b += 32) reinterpret_cast<uint32_t*>(mine)[b] = 0;
    const uint32_t first = blockIdx.x * kTile + warp * (32 * ITEMS) + lane;
    uint32_t key[ITEMS];
#pragma unroll
    for (int k = 0; k < ITEMS; k++) { const uint32_t i = min(first + k * 32, n - 1); key[k] = FIRST ? s.key[i] : from[i].x; }
    uint32_t within[kPer];                     // entries of the bin in the tiles before
#pragma unroll
    for (int k = 0; k < kPer; k++) {
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
    uint32_t rank[ITEMS / 2];                              // two to a word
#pragma unroll
    for (int k = 0; k < ITEMS; k++) {
        const uint32_t r = warp_rank<BITS>(key[k] >> shift & (bins - 1), first + k * 32 < n, mine, lane);
        if (k % 2 == 0) rank[k / 2] = r; else rank[k / 2] |= r << 16;
    }
    __syncthreads();
    for (int b = t; b < bins / 2; b += kSortBlock) {
        const uint32_t sums = warp_offsets(count, kSortWarps, bins, b);
        start[2 * b] = sums & 0xffff;
        start[2 * b + 1] = sums >> 16;
    }
    block_scan(base, bins, warp_sums);
    block_scan(start, bins, warp_sums);
#pragma unroll
    for (int k = 0; k < kPer; k++) { const int b = t + k * kSortBlock; if (b < bins) base[b] += within[k] - start[b]; }
#pragma unroll
    for (int k = 0; k < ITEMS; k++) {
        const uint32_t i = first + k * 32, d = key[k] >> shift & (bins - 1);
        if (i < n) at[start[d] + mine[d] + (rank[k / 2] >> 16 * (k % 2) & 0xffff)] = make_uint2(key[k], FIRST ? i : from[i].y);
    }
    __syncthreads();
    const uint32_t here = min((uint32_t)kTile, n - blockIdx.x * kTile);
#pragma unroll 4
    for (uint32_t i = t; i < here; i += kSortBlock) { const uint2 x = at[i]; to[i + base[x.x >> shift & (bins - 1)]] = x; }
}

// ---- sums --------------------------------------------------------------------------------------------------

// N columns of a row: ALIGNED ones from `col` on as one piece, else those `gap` apart, as far as the row goes.
template <typename Out, int N, bool ALIGNED>
__device__ __forceinline__ void write_row(const Job& j, uint32_t row, uint32_t col, uint32_t gap, const float (&sum)[N]) {
    const bool second = row >= j.rows[0];
    Out* const at = static_cast<Out*>(second ? j.out[1] : j.out[0]) + (size_t)(second ? row - j.rows[0] : row) * (second ? j.out_stride[1] : j.out_stride[0]) + col;
    const auto value = [&](float x, Out was) { return from_float<Out>(j.accumulate ? fmaf(x, j.scale, as_float(was)) : x * j.scale); };
    if constexpr (ALIGNED) {
        Piece<Out, N> r = {};
        if (j.accumulate) r = *reinterpret_cast<const Piece<Out, N>*>(at);
#pragma unroll
        for (int k = 0; k < N; k++) r.v[k] = value(sum[k], r.v[k]);
        store_piece<Out, N>(at, r);
    } else {
#pragma unroll
        for (int k = 0; k < N; k++)
            if (col + k * gap < j.width) at[k * gap] = value(sum[k], j.accumulate ? at[k * gap] : from_float<Out>(0.f));
    }
}

// What an entry adds: c * (row a - row b), as far as it has these rows.
struct Term { uint32_t key, a, b; float c; bool has_a, has_b; };
template <bool PAIRS> __device__ __forceinline__ Term term_of(const Job& j, uint2 entry, uint4 pair) {
    Term t{entry.x, entry.y, 0, 1.f, entry.x < j.total, false};
    if (PAIRS) {
        const uint32_t kind = entry.y % 3;
        t.a = kind ? pair.x : pair.y;
        t.b = pair.z;
        t.c = kind == 2 ? -__uint_as_float(pair.w) : __uint_as_float(pair.w);
        t.has_a = t.has_a && t.c != 0.f;                        // coef 0: whatever the rows hold
        t.has_b = t.has_a && kind == 0;
    }
    if (!t.has_a) { t.a = 0; t.c = 0.f; }
    if (!t.has_b) t.b = 0;
    return t;
}

// 8 or 16 bytes on their way to shared memory.  16 go past L1 (with it, pairs on a popular law take 6 % longer); for 8 there is only the form through it.
// Zeros instead where it is not there: nothing is read then.
template <int BYTES> __device__ __forceinline__ void fetch_piece(uint32_t to, const void* from, bool there) {
    if constexpr (BYTES == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(there ? 16 : 0) : "memory");
    else asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(to), "l"(from), "r"(there ? 8 : 0) : "memory");
}

// A team's lanes take a group of entries each and hand their rows round; what a lane can work out for a group (where rows begin, which
// entries add nothing) it does, and the team reads it off ballots.  What bounds it is the rows, random ones from HBM or
// L2, so AHEAD of them are under way for each team: every lane copies its pieces into shared memory of its own, which needs
// no registers and no meeting of threads.  4M rows of 256 bytes into 480k of 512: 213 us for 1.29 GB, 6.1 TB/s (286 with four rows in
// flight in registers).  The gradients of 1M pairs, binary16 rows of 128: 235 us, bound by instructions and by the latency of L2.
// Rows that cannot be moved in pieces are loaded where they are added, element by element, four for each lane a team's width apart
// (20,000 rows of 333 binary16 numbers into as many: 43 us on the GPU in all; 91 with one for each lane).
template <typename T, int N, bool PAIRS, bool ALIGNED> struct Ring {
    static constexpr int piece = sizeof(T) * N, ahead = PAIRS ? 8 : 16, sides = PAIRS ? 2 : 1;      // rows of an entry
    static constexpr size_t smem = ALIGNED ? (size_t)ahead * sides * kReduceBlock * piece : 0;
};

template <typename T, typename Out, int N, bool PAIRS, bool ALIGNED>
__global__ void __launch_bounds__(kReduceBlock, PAIRS && N == 8 ? 2 : 3) reduce_kernel(const Job j, const Space s, const uint2* entry, int team_log2) {
    using R = Ring<T, N, PAIRS, ALIGNED>;
    constexpr int BATCH = 4, kSlot = R::sides * kReduceBlock * R::piece;
    extern __shared__ __align__(16) uint8_t ring[];             // [ahead][sides][threads]
    follow();
    const uint32_t team = 1u << team_log2, lane = threadIdx.x & 31, tl = lane & (team - 1), team_at = lane & ~(team - 1), ahead = min(team, (uint32_t)R::ahead);
    const uint32_t team_mask = (team == 32 ? 0xffffffffu : (1u << team) - 1) << team_at;
    const uint32_t chunk = (blockIdx.x * kReduceBlock + threadIdx.x) >> team_log2, gap = ALIGNED ? 1 : team;
    const uint32_t col = (blockIdx.y << team_log2) * N + tl * (ALIGNED ? N : 1);      // this lane's first column; the others are `gap` apart
    const uint32_t size = 1u << j.chunk_log2, over = size / 4;
    const uint32_t begin = min(j.n, chunk << j.chunk_log2), end = min(j.n, begin + size);
    const bool writes = chunk < s.chunks && col < j.width;
    // rows across the chunk's ends: finished by the chunk before where they end within `over` entries, else in parts
    const auto row_at = [&](uint32_t i) { return i < j.n ? entry[i].x : kNoRow; };
    const uint32_t before = chunk < s.chunks && begin ? row_at(begin - 1) : kNoRow, last = end > begin ? row_at(end - 1) : kNoRow;
    const bool in_parts = before != kNoRow && row_at(begin + over) == before, on_in_parts = end < j.n && row_at(end + over) == last;
    const uint32_t until = on_in_parts || end == begin ? end : min(j.n, end + over);
    const T* const src0 = static_cast<const T*>(j.src[0]) + col, *const src1 = static_cast<const T*>(j.src[1]) + col;
    const size_t stride0 = j.src_stride[0], stride1 = j.src_stride[1];
    const uint8_t* const mine_at = ring + threadIdx.x * R::piece;
    const uint32_t mine_to = (uint32_t)__cvta_generic_to_shared(mine_at);
    uint32_t row = j.total;
    float sum[N] = {};
    const auto flush = [&]() {
        if (row >= j.total || !writes) return;
        const bool from_before = in_parts && row == before;
        if (from_before || (on_in_parts && row == last)) {
            float* const part = (from_before ? s.head : s.tail) + (size_t)chunk * s.pitch + col;
#pragma unroll
            for (int k = 0; k < N; k++) if (ALIGNED || col + k * gap < j.width) part[k * gap] = sum[k];
            if (!from_before && col == 0) s.owners[atomicAdd(s.n_owners, 1u)] = make_uint2(chunk, row);
        } else write_row<Out, N, ALIGNED>(j, row, col, gap, sum);
        if (!from_before && !j.accumulate && col == 0) s.touched[row] = 1;
    };
    const auto entry_at = [&](uint32_t i) {
        uint2 e = make_uint2(j.total, 0);
        if (i < until) e = entry[i];
        if (i >= end ? e.x != last : !in_parts && e.x == before) e.x = j.total;
        return e;
    };
    const auto pair_of = [&](uint2 e) { return PAIRS && e.x < j.total ? s.pair[e.y / 3] : make_uint4(0, 0, 0, 0); };
    const auto ballot = [&](bool b) { return __ballot_sync(0xffffffffu, b) >> team_at; };
    // rows of the entries k .. k + 3 of a group; `some`: a team of the warp has second rows
    const auto fetch = [&](const Term& t, uint32_t adds, uint32_t twos, bool some, uint32_t k0) {
        const uint32_t to = mine_to + (k0 & (ahead - 1)) * kSlot, ones = writes ? adds >> k0 : 0u, pairs = writes ? twos >> k0 : 0u;
        if (PAIRS && some) {
#pragma unroll
            for (int k = 0; k < BATCH; k++) {
                const uint32_t ra = __shfl_sync(0xffffffffu, t.a, k0 + k, team), rb = __shfl_sync(0xffffffffu, t.b, k0 + k, team);
                const bool two = pairs >> k & 1;
                fetch_piece<R::piece>(to + k * kSlot, two ? src1 + ra * stride1 : src0 + ra * stride0, ones >> k & 1);
                fetch_piece<R::piece>(to + k * kSlot + kReduceBlock * R::piece, src1 + rb * stride1, two);
            }
        } else {
#pragma unroll
            for (int k = 0; k < BATCH; k++) fetch_piece<R::piece>(to + k * kSlot, src0 + __shfl_sync(0xffffffffu, t.a, k0 + k, team) * stride0, ones >> k & 1);
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    uint2 after = entry_at(begin + 2 * team + tl);
    const uint2 e0 = entry_at(begin + tl), e1 = entry_at(begin + team + tl);
    Term now = term_of<PAIRS>(j, e0, pair_of(e0)), next = term_of<PAIRS>(j, e1, pair_of(e1));
    uint4 pair = pair_of(after);
    const auto any = [](uint32_t mask) { return __any_sync(0xffffffffu, mask != 0); };
    uint32_t adds = ballot(now.has_a), twos = PAIRS ? ballot(now.has_b) : 0u;
    bool some = PAIRS && any(twos);                             // seldom both: users' rows are sorted before items'
    if constexpr (ALIGNED) for (uint32_t k0 = 0; k0 < ahead; k0 += BATCH) fetch(now, adds, twos, some, k0);
    for (uint32_t g = begin; __any_sync(0xffffffffu, g < until); g += team) {
        const uint32_t left = __shfl_up_sync(0xffffffffu, now.key, 1, team), begins = ballot(now.key != (tl ? left : row));
        const uint32_t next_adds = ballot(next.has_a), next_twos = PAIRS ? ballot(next.has_b) : 0u;
        const bool next_some = PAIRS && any(next_twos);
        for (uint32_t k0 = 0; k0 < team; k0 += BATCH) {
            if (!__any_sync(0xffffffffu, g + k0 < until)) break;
            Piece<T, N> a[BATCH], b[PAIRS ? BATCH : 1];
            float c[BATCH];
            if constexpr (ALIGNED) {
                if (ahead == 16) asm volatile("cp.async.wait_group 3;" ::: "memory");
                else asm volatile("cp.async.wait_group 1;" ::: "memory");
            }
#pragma unroll
            for (int k = 0; k < BATCH; k++) {
                c[k] = PAIRS ? __shfl_sync(0xffffffffu, now.c, k0 + k, team) : 1.f;
                if constexpr (ALIGNED) {
                    const uint8_t* const at = mine_at + (k0 & (ahead - 1)) * kSlot + k * kSlot;
                    a[k] = shared_piece<T, N>(at);
                    if (PAIRS && some) b[k] = shared_piece<T, N>(at + kReduceBlock * R::piece);
                } else {
                    const uint32_t ra = __shfl_sync(0xffffffffu, now.a, k0 + k, team), rb = PAIRS ? __shfl_sync(0xffffffffu, now.b, k0 + k, team) : 0u;
                    const bool one = (adds >> (k0 + k) & 1) && writes, two = PAIRS && (twos >> (k0 + k) & 1);
                    const T* const from_a = two ? src1 + ra * stride1 : src0 + ra * stride0, *const from_b = src1 + rb * stride1;
#pragma unroll
                    for (int x = 0; x < N; x++) {
                        const bool there = col + x * gap < j.width;
                        a[k].v[x] = from_float<T>(0.f);
                        if (one && there) a[k].v[x] = load_piece<T, 1>(from_a + x * gap).v[0];
                        if (PAIRS) {
                            b[k].v[x] = from_float<T>(0.f);
                            if (two && writes && there) b[k].v[x] = load_piece<T, 1>(from_b + x * gap).v[0];
                        }
                    }
                }
            }
#pragma unroll
            for (int k = 0; k < BATCH; k++) {
                if (begins >> (k0 + k) & 1) {
                    flush();
                    row = __shfl_sync(team_mask, now.key, k0 + k, team);
#pragma unroll
                    for (int x = 0; x < N; x++) sum[x] = 0.f;
                }
                if (!PAIRS) {
#pragma unroll
                    for (int x = 0; x < N; x++) sum[x] += as_float(a[k].v[x]);
                } else if (some) {
#pragma unroll
                    for (int x = 0; x < N; x++) sum[x] = fmaf(c[k], as_float(a[k].v[x]) - as_float(b[k].v[x]), sum[x]);
                } else {
#pragma unroll
                    for (int x = 0; x < N; x++) sum[x] = fmaf(c[k], as_float(a[k].v[x]), sum[x]);
                }
            }
            __syncwarp();
            if constexpr (ALIGNED) {                              // into the places that have just been read
                const uint32_t k1 = k0 + ahead;
                if (k1 < team) fetch(now, adds, twos, some, k1);
                else fetch(next, next_adds, next_twos, next_some, k1 - team);
            }
        }
        now = next;
        adds = next_adds;
        twos = next_twos;
        some = next_some;
        next = term_of<PAIRS>(j, after, pair);
        after = entry_at(g + 3 * team + tl);
        pair = pair_of(after);
    }
    if constexpr (ALIGNED) asm volatile("cp.async.wait_all;" ::: "memory");      // zeros behind the last entry: none is written after the block has ended
    flush();
}

// The first position behind the entries of `row`, searched by a warp from `at`, which is one of them: 32 places at a time.
__device__ __forceinline__ uint32_t row_end(const uint2* entry, uint32_t at, uint32_t n, uint32_t row, uint32_t lane) {
    uint32_t lo = at, hi = n;                                   // the entry at lo is one, that at hi is none
    while (hi - lo > 1) {
        const uint32_t step = (hi - lo + 31) / 32, mid = lo + lane * step;      // lane 0: lo
        const uint32_t in = __popc(__ballot_sync(0xffffffffu, mid < hi && entry[mid].x == row));      // the first `in` places
        hi = min(hi, lo + in * step);
        lo += (in - 1) * step;
    }
    return hi;
}

// Blocks below `combine_blocks` add up the parts of the rows that the owners name: a warp each, and all warps of the block a slice
// each where a row has more parts than the block has warps (200,000 binary16 rows of 336 into 30: 68 us on the GPU in all, some 230 when neighbouring owners
// shared a block).  The other blocks clear the rows that no entry names, a warp for 32 of them.
template <int N> __device__ __forceinline__ void add_parts(const Space& s, uint32_t first, uint32_t end, uint32_t col, float (&sum)[N]) {
#pragma unroll 16
    for (uint32_t q = first; q < end; q++) {
        const Piece<float, N> part = *reinterpret_cast<const Piece<float, N>*>(s.head + (size_t)q * s.pitch + col);
#pragma unroll
        for (int k = 0; k < N; k++) sum[k] += part.v[k];
    }
}

template <typename Out, bool ALIGNED>
__global__ void __launch_bounds__(kCombineBlock, 2) combine_kernel(const Job j, const Space s, const uint2* entry, uint32_t combine_blocks) {
    constexpr uint32_t kWarps = kCombineBlock / 32;
    constexpr int N = 4;                                        // parts lie in rows of whole pieces, whatever the output's do
    follow();
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    if (blockIdx.x >= combine_blocks) {
        const uint32_t row0 = (blockIdx.x - combine_blocks) * kCombineBlock + warp * 32;
        const bool clear = row0 + lane < j.total && (j.n == 0 || s.touched[row0 + lane] == 0);
        uint32_t todo = __ballot_sync(0xffffffffu, clear);
        while (todo) {
            const uint32_t r = row0 + __ffs(todo) - 1;
            todo &= todo - 1;
            const bool second = r >= j.rows[0];
            Out* const at = static_cast<Out*>(second ? j.out[1] : j.out[0]) + (size_t)(second ? r - j.rows[0] : r) * (second ? j.out_stride[1] : j.out_stride[0]);
            constexpr int kZeros = ALIGNED ? N : 1;
            for (uint32_t c = lane * kZeros; c < j.width; c += 32 * kZeros) {
                Piece<Out, kZeros> zero;
#pragma unroll
                for (int k = 0; k < kZeros; k++) zero.v[k] = from_float<Out>(0.f);
                store_piece<Out, kZeros>(at + c, zero);
            }
        }
        return;
    }
    __shared__ float slice[kWarps][32 * N];
    __shared__ uint32_t long_chunk[kWarps], long_count[kWarps], long_row[kWarps], n_long;
    const uint32_t owners = *s.n_owners, size = 1u << j.chunk_log2;
    for (uint32_t o0 = blockIdx.x; o0 < owners; o0 += combine_blocks * kWarps) {      // a block's warps take owners far apart: few owners, a block each
        const uint32_t o = o0 + warp * combine_blocks;
        if (threadIdx.x == 0) n_long = 0;
        __syncthreads();
        if (o < owners) {
            const uint2 owner = s.owners[o];
            const uint32_t chunk = owner.x, row = owner.y, first = (chunk + 1) << j.chunk_log2;
            // Chunks that follow with a part of the row.  Most rows end soon: lane q looks whether the row goes on in parts behind q chunks more.
            const uint64_t at = (uint64_t)first + (uint64_t)lane * size + size / 4;
            const uint32_t through = __ballot_sync(0xffffffffu, at < j.n && entry[at].x == row);
            uint32_t count = __popc(through);
            if (through == 0xffffffffu) {                       // all but one where it ends within a quarter of a chunk: those entries are in the part before
                const uint32_t stop = row_end(entry, first, j.n, row, lane), whole = (stop - first) >> j.chunk_log2;
                count = whole + (stop - first - whole * size > size / 4 ? 1 : 0);
            }
            if (count > kWarps) {
                if (lane == 0) { const uint32_t at_long = atomicAdd(&n_long, 1u); long_chunk[at_long] = chunk; long_count[at_long] = count; long_row[at_long] = row; }
            } else {
                for (uint32_t c = lane * N; c < j.width; c += 32 * N) {
                    float sum[N];
#pragma unroll
                    for (int k = 0; k < N; k++) sum[k] = s.tail[(size_t)chunk * s.pitch + c + k];
                    add_parts<N>(s, chunk + 1, chunk + 1 + count, c, sum);
                    write_row<Out, N, ALIGNED>(j, row, c, 1, sum);
                }
            }
        }
        __syncthreads();
        for (uint32_t l = 0; l < n_long; l++) {
            const uint32_t chunk = long_chunk[l], count = long_count[l], per = (count + kWarps - 1) / kWarps, q0 = min(count, warp * per), q1 = min(count, q0 + per);
            for (uint32_t c0 = 0; c0 < j.width; c0 += 32 * N) {
                const uint32_t c = c0 + lane * N;
                float sum[N] = {};
                if (c < j.width) {
                    if (warp == 0) {
#pragma unroll
                        for (int k = 0; k < N; k++) sum[k] = s.tail[(size_t)chunk * s.pitch + c + k];
                    }
                    add_parts<N>(s, chunk + 1 + q0, chunk + 1 + q1, c, sum);
                }
#pragma unroll
                for (int k = 0; k < N; k++) slice[warp][lane * N + k] = sum[k];
                __syncthreads();
                if (warp == 0 && c < j.width) {
#pragma unroll
                    for (int w = 1; w < (int)kWarps; w++)
#pragma unroll
                        for (int k = 0; k < N; k++) sum[k] += slice[w][lane * N + k];
                    write_row<Out, N, ALIGNED>(j, long_row[l], c, 1, sum);
                }
                __syncthreads();
            }
        }
        __syncthreads();
    }
}

// ---- host ---------------------------------------------------------------------------------------------------

// Entries of a chunk: enough chunks to fill the GPU, and no more parts than that needs (4M entries: 128, 364 us in all; 256, 377 us;
// 64, 385 us.  12,288 entries, of 4,096 pairs: 8, 31 us with the loss; 16, 34 us; 32, 40 us).
int chunk_log2(uint64_t n) { return n < (1u << 14) ? 3 : n < (1u << 17) ? 4 : n < (1u << 19) ? 5 : n < (1u << 21) ? 6 : 7; }
int bits_for(uint64_t keys) { int b = 1; while (b < 32 && (1ull << b) < keys) b++; return b; }      // of the largest key, keys - 1

size_t carve(uint64_t n, uint64_t total, uint32_t width, bool pairs, char* base, Space* s) {
    size_t at = 0;
    const auto take = [&](size_t bytes) { char* const p = base ? base + at : nullptr; at += (bytes + 255) / 256 * 256; return p; };
    Space sp = {};
    if (n) {
        const uint32_t tile = kSortBlock * (n < kManyFrom ? kFewItems : kManyItems);
        sp.tiles = (uint32_t)((n + tile - 1) / tile);
        sp.chunks = (uint32_t)((n + (1u << chunk_log2(n)) - 1) >> chunk_log2(n));
        sp.pitch = (width + 3) / 4 * 4;
        const bool small = n <= kSmall;
        sp.entry[0] = reinterpret_cast<uint2*>(take(8 * n));
        sp.entry[1] = reinterpret_cast<uint2*>(take(8 * n));
        sp.key = reinterpret_cast<uint32_t*>(take(small ? 0 : 4 * n));
        sp.counts = reinterpret_cast<uint32_t*>(take(small ? 0 : 4 * (size_t)sp.tiles * kMaxBins));
        sp.totals = reinterpret_cast<uint32_t*>(take(small ? 0 : 4 * kMaxBins));
        sp.pair = reinterpret_cast<uint4*>(take(pairs ? 16 * (n / 3) : 0));
        sp.head = reinterpret_cast<float*>(take(4 * (size_t)sp.chunks * sp.pitch));
        sp.tail = reinterpret_cast<float*>(take(4 * (size_t)sp.chunks * sp.pitch));
        sp.owners = reinterpret_cast<uint2*>(take(8 * (size_t)sp.chunks));
        sp.n_owners = reinterpret_cast<uint32_t*>(take(4));
        sp.touched = reinterpret_cast<uint8_t*>(take(total));
    }
    if (s) *s = sp;
    return at;
}

// Launches a kernel behind the first of a call: its blocks are brought up while the kernel before still runs, and wait for its end and
// its results in follow(), the first thing that they do.  A launch less to wait for is 1 to 1.5 us.
template <class Kernel, class... Args>
cudaError_t launch_behind(Kernel kernel, dim3 grid, unsigned block, size_t smem, cudaStream_t st, Args... args) {
    cudaLaunchConfig_t config = {};
    config.gridDim = grid;
    config.blockDim = dim3(block);
    config.dynamicSmemBytes = smem;
    config.stream = st;
    cudaLaunchAttribute behind[1];
    behind[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    behind[0].val.programmaticStreamSerializationAllowed = 1;
    config.attrs = behind;
    config.numAttrs = 1;
    return reported(cudaLaunchKernelEx(&config, kernel, args...));
}

// One digit of BITS bits: the first pass takes its entries from `key`.
template <int ITEMS, int BITS>
cudaError_t sort_digit(const Job& j, const Space& s, int pass, cudaStream_t st) {
    static LaunchCache first_cache, next_cache;
    constexpr int bins = 1 << BITS;
    constexpr size_t smem = 8 * (size_t)ITEMS * kSortBlock + 2 * (size_t)bins * kSortWarps + 8 * (size_t)bins;
    cudaError_t e = allow_smem(scatter_kernel<true, ITEMS, BITS>, smem, first_cache);
    if (e == cudaSuccess) e = allow_smem(scatter_kernel<false, ITEMS, BITS>, smem, next_cache);
    if (e != cudaSuccess) return e;
    const bool scanned = s.tiles > kScanTiles;
    uint2* const from = s.entry[pass & 1], *const to = s.entry[~pass & 1];
    const uint2* const none = nullptr;
    if (pass == 0) e = launch(count_kernel<true, ITEMS>, s.tiles, kSortBlock, 0, st, j, s, none, 0, BITS);
    else e = launch_behind(count_kernel<false, ITEMS>, s.tiles, kSortBlock, 0, st, j, s, (const uint2*)from, pass * BITS, BITS);
    if (e == cudaSuccess && scanned) e = launch_behind(scan_kernel, bins / 32, 1024, 0, st, s, bins);
    if (e == cudaSuccess && pass == 0) e = launch_behind(scatter_kernel<true, ITEMS, BITS>, s.tiles, kSortBlock, smem, st, s, j.n, none, to, 0, scanned);
    else if (e == cudaSuccess) e = launch_behind(scatter_kernel<false, ITEMS, BITS>, s.tiles, kSortBlock, smem, st, s, j.n, (const uint2*)from, to, pass * BITS, scanned);
    return e;
}

// Sorts the entries; *which tells which of the two buffers holds them.
cudaError_t sort_entries(const Job& j, const Space& s, int* which, cudaStream_t st) {
    const int key_bits = bits_for((uint64_t)j.total + 1);
    if (j.n <= kSmall) {
        const int passes = (key_bits + kSmallBits - 1) / kSmallBits;
        const uint32_t blocks = j.n > kSmallBlock ? kSmallCluster : 1;
        cudaLaunchConfig_t config = {};
        config.gridDim = dim3(blocks);
        config.blockDim = dim3(kSmallBlock);
        config.stream = st;
        cudaLaunchAttribute cluster[1];
        cluster[0].id = cudaLaunchAttributeClusterDimension;
        cluster[0].val.clusterDim.x = blocks;
        cluster[0].val.clusterDim.y = cluster[0].val.clusterDim.z = 1;
        config.attrs = cluster;
        config.numAttrs = 1;
        *which = (passes - 1) & 1;
        return reported(cudaLaunchKernelEx(&config, small_sort_kernel, j, s, passes));
    }
    const bool ten = (key_bits + 9) / 10 < (key_bits + 7) / 8, many = j.n >= kManyFrom;      // wider digits where they save a pass
    const int passes = ten ? (key_bits + 9) / 10 : (key_bits + 7) / 8;
    for (int p = 0; p < passes; p++) {
        const cudaError_t e = many ? (ten ? sort_digit<kManyItems, 10>(j, s, p, st) : sort_digit<kManyItems, 8>(j, s, p, st))
                                   : (ten ? sort_digit<kFewItems, 10>(j, s, p, st) : sort_digit<kFewItems, 8>(j, s, p, st));
        if (e != cudaSuccess) return e;
    }
    *which = passes & 1;
    return cudaSuccess;
}

template <typename T, typename Out, int N, bool PAIRS, bool ALIGNED>
cudaError_t sum_pieces(const Job& j, const Space& s, int which, cudaStream_t st) {
    const uint32_t pieces = (j.width + N - 1) / N;
    int log2 = 3;
    while (log2 < 5 && (1u << log2) < pieces) log2++;
    const uint32_t teams_per_block = kReduceBlock >> log2;
    const dim3 grid((s.chunks + teams_per_block - 1) / teams_per_block, (pieces + (1u << log2) - 1) >> log2);
    const uint32_t combine_blocks = s.chunks > 1 ? std::min<uint32_t>(s.chunks - 1, 2 * current_sms()) : 0;
    const uint32_t clear_blocks = j.accumulate ? 0 : (uint32_t)(((uint64_t)j.total + kCombineBlock - 1) / kCombineBlock);
    if (j.n) {
        static LaunchCache cache;
        constexpr size_t smem = Ring<T, N, PAIRS, ALIGNED>::smem;
        cudaError_t e = allow_smem(reduce_kernel<T, Out, N, PAIRS, ALIGNED>, smem, cache);
        if (e != cudaSuccess) return e;
        e = launch_behind(reduce_kernel<T, Out, N, PAIRS, ALIGNED>, grid, kReduceBlock, smem, st, j, s, (const uint2*)s.entry[which], log2);
        if (e == cudaSuccess && combine_blocks + clear_blocks)
            e = launch_behind(combine_kernel<Out, ALIGNED>, combine_blocks + clear_blocks, kCombineBlock, 0, st, j, s, (const uint2*)s.entry[which], combine_blocks);
        return e;
    }
    return clear_blocks ? launch(combine_kernel<Out, ALIGNED>, clear_blocks, kCombineBlock, 0, st, j, s, static_cast<const uint2*>(nullptr), 0u) : cudaSuccess;
}

// `pieces`: elements that all rows may be moved in.
template <typename T, typename Out, bool PAIRS>
cudaError_t sum_entries(const Job& j, const Space& s, int which, uint32_t pieces, cudaStream_t st) {
    if (sizeof(T) == 2 && pieces == 8) return sum_pieces<T, Out, (sizeof(T) == 2 ? 8 : 4), PAIRS, true>(j, s, which, st);
    return pieces >= 4 ? sum_pieces<T, Out, 4, PAIRS, true>(j, s, which, st) : sum_pieces<T, Out, 4, PAIRS, false>(j, s, which, st);
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

int mascot_rows_gradient_workspace(uint64_t count, uint64_t rows, uint32_t width, uint64_t* bytes) try {
    if (!bytes || count >= kMaxRows || rows >= kMaxRows || width == 0 || width > kMaxWidth) return fail(nullptr, MASCOT_ERR_BAD_ARG, "null pointer or size out of range");
    *bytes = carve(count, rows, width, false, nullptr, nullptr);
    return MASCOT_OK;
} ROW_CATCH

int mascot_pair_gradient_workspace(uint64_t count, uint64_t n_users, uint64_t n_items, uint32_t width, uint64_t* bytes) try {
    if (!bytes || count >= kMaxRows || n_users >= kMaxRows || n_items >= kMaxRows || width == 0 || width > kMaxWidth || 3 * count >= kMaxRows || n_users + n_items >= kMaxRows)
        return fail(nullptr, MASCOT_ERR_BAD_ARG, "null pointer or size out of range");
    *bytes = carve(3 * count, n_users + n_items, width, true, nullptr, nullptr);
    return MASCOT_OK;
} ROW_CATCH

int mascot_rows_gradient(const mascot_rows* grad, const mascot_ids* ids, float scale, const mascot_rows* out, int accumulate, void* workspace,
                         uint64_t workspace_bytes, uint32_t* flags, void* stream) try {
    ROW_CHECK(check_rows("grad", grad, false));
    ROW_CHECK(check_ids("ids", ids));
    ROW_CHECK(check_rows("out", out, false));
    if (grad->width != out->width) return fail(nullptr, MASCOT_ERR_BAD_ARG, "out: width is not the gradient's");
    ROW_CHECK(check_words("flags", flags));
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
    int device = 0;
    ROW_CHECK(check_device(&device));
    if (ids->count) {
        ROW_CHECK(check_memory("grad", grad->data, device));
        ROW_CHECK(check_memory("ids", ids->data, device));
        ROW_CHECK(check_memory("workspace", workspace, device));
    }
    if (out->rows) ROW_CHECK(check_memory("out", out->data, device));
    ROW_CHECK(check_memory("flags", flags, device));
    Job j = {};
    j.ids[0] = ids_of(*ids);
    j.n = (uint32_t)ids->count;
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
} ROW_CATCH

int mascot_pair_gradient(const mascot_rows* P, const mascot_rows* Q, const mascot_ids* users, const mascot_ids* preferred, const mascot_ids* other,
                         const float* coef, float scale, const mascot_rows* dP, const mascot_rows* dQ, int accumulate, void* workspace,
                         uint64_t workspace_bytes, uint32_t* flags, void* stream) try {
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
    ROW_CHECK(check_words("coef", coef));
    ROW_CHECK(check_words("flags", flags));
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
    int device = 0;
    ROW_CHECK(check_device(&device));
    for (const auto& m : mats) if (m.m->rows) ROW_CHECK(check_memory(m.what, m.m->data, device));
    if (n) {
        for (const auto& x : idss) ROW_CHECK(check_memory(x.what, x.ids->data, device));
        ROW_CHECK(check_memory("coef", coef, device));
        ROW_CHECK(check_memory("workspace", workspace, device));
    }
    ROW_CHECK(check_memory("flags", flags, device));
    Job j = {};
    j.ids[0] = ids_of(*users); j.ids[1] = ids_of(*preferred); j.ids[2] = ids_of(*other);
    j.kinds = 3; j.n = (uint32_t)(3 * n);
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
} ROW_CATCH

}  // extern "C"
