// Scores of every row of one e4m3 matrix against every row of another, with a scale for each block of 128 columns.
//
// out[m][n] = sum over column blocks c of a_scale[c][m] * b_scale[c][n] * <a[m], b[n]> within c.  Each block of 128 columns is one
// accumulation of four tcgen05.mma of kind f8f6f4 (a block is 128 bytes of a row, one line of the 128-byte swizzle); its sum is read
// back from tensor memory, scaled and added in fp32 registers while the tensor cores work on the next one in another part of it.
//
// A block of threads is persistent and takes every gridDim.x-th tile of 128 lanes x CN columns of an accumulator.  One warp fetches
// operands by TMA, one issues the matrix instructions, one fetches scales, one looks whether they are in a safe range, the others read back, scale and store: warp w the
// lanes 32 (w % 4) on, and columns of the group w / 4.  Rows of a (users) are the inner index of the tiles, so that rows
// of b (items) are fetched from HBM once and from L2 after that.  What differs is which side the lanes are (Mode):
//   ONE     rows of 128 columns and less: items.  What is written bounds it.  Four warps read 16 columns of all lanes at a time, meet
//           over shared memory and store whole rows of 128 scores, in pieces as wide as the row's address allows (32 scores a
//           warp, straight from the accumulator, took 1.4 times as long; that is how up to 16 users are stored).  Nothing is summed up, so registers allow 16 such warps.
//   ROWS    longer rows, a scale for each row of b, or few users: items too.  A column's scale is a broadcast from shared memory,
//           whose 128 bytes to a warp bound the step at 4 CN cycles, twice what the matrix instructions take (4,096 x 17,770 x 4,096
//           to bf16: 460 us a call, 409 in a burst too short for the power limit).
//   SQUARE  longer rows, a scale for 128 rows of b: users.  The scale of a lane and half of the columns is one number, kept in a
//           register; scores go through shared memory to be stored along the rows of `out` (the same sizes: 353 us a call,
//           1.69 PFLOP/s, and 301 us in a short burst; the tensor cores are busy half of the time, the rest they wait for accumulators to be read back).
#include <cuda.h>

#include <algorithm>

#include "reader.h"
#include "row_ops.h"

namespace mascot {
namespace {

enum Mode { ONE, ROWS, SQUARE };
constexpr int kLanes = 128;                          // lanes of tensor memory
constexpr int kLaneTileBytes = kLanes * kScaleBlock;
constexpr int kScaleSteps = 8;                       // steps whose scales are under way or in use: a step may be shorter than a fetch from HBM
constexpr int kStagePitch = 80;                      // bytes of a row's piece of 64 on its way through shared memory (SQUARE)
constexpr uint32_t kNap = 1'000'000;                 // ns
constexpr long long kPatience = 1ll << 33;           // cycles: more than four seconds

template <int CN, Mode MODE> struct Shape {
    static constexpr int stages = CN == 256 ? (MODE == ONE ? 3 : 4) : CN == 128 ? (MODE == ONE ? 4 : 6) : MODE == ONE && CN == 64 ? 6 : 8;
    static constexpr int buffers = CN == 256 ? 2 : 4;                        // accumulators in tensor memory
    static constexpr int tmem_columns = CN * buffers;                        // powers of two, 64 to 512
    static constexpr int groups = MODE == ONE && CN >= 64 ? 4 : 2;           // of four warps that read back, CN / groups columns each
    static constexpr int readers = 4 * groups, threads = 32 * readers + 128;
    static constexpr int stage_bytes = kLaneTileBytes + CN * kScaleBlock;
    static constexpr int step_scales = kLanes + (MODE == SQUARE ? 4 : CN);
    static constexpr int transit = MODE == SQUARE ? readers * 32 * kStagePitch : MODE == ONE && CN > 16 ? groups * 2 * 16 * kLanes * 4 : 0;
    static constexpr size_t smem = 1024 + (size_t)stages * stage_bytes + transit + kScaleSteps * step_scales * 4 + 8 * (2 * stages + 2 * buffers + 3 * kScaleSteps) + 16;
    static_assert(smem <= 227 * 1024, "shared memory of a block");
};

// One side of the product: the lanes' or the columns' rows.
struct Side {
    const float* scale;
    uint32_t rows, scales, shift;                    // scales of a column block, rows to a scale (log2)
    const uint8_t* row_data;
    size_t stride;                                   // bytes
    __device__ float of(uint32_t block, uint32_t row) const { return __ldg(scale + (size_t)block * scales + (row >> shift)); }
};
struct ProductArgs {
    Side lane, col;
    void* out;
    size_t lane_step, col_step;                      // elements of `out` from one row of a side to the next
    uint32_t blocks, user_tiles, tiles;              // blocks of 128 columns
    uint32_t width;                                  // columns
    uint32_t* flags;
};

__device__ __forceinline__ uint32_t smem_at(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }

__device__ __forceinline__ void barrier_init(uint64_t* b, uint32_t count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_at(b)), "r"(count) : "memory");
}
__device__ __forceinline__ void barrier_arrive(uint64_t* b) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_at(b)) : "memory");
}
__device__ __forceinline__ void barrier_expect(uint64_t* b, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_at(b)), "r"(bytes) : "memory");
}
// Waits for the phase of that parity to end, but not for ever: each try sleeps up to kNap ns, and what has not come kPatience cycles
// after the first few gives up.
__device__ __forceinline__ bool barrier_wait(uint64_t* b, uint32_t parity) {
    constexpr uint32_t kFew = 64;
    const uint32_t at = smem_at(b);
    long long begin = 0;
#pragma unroll 1
    for (uint32_t tries = 0;; tries++) {
        uint32_t done;
        asm volatile("{ .reg .pred p; mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3; selp.u32 %0, 1, 0, p; }" : "=r"(done) : "r"(at), "r"(parity), "r"(kNap) : "memory");
        if (done) return true;
        if (tries < kFew) begin = clock64();
        else if (clock64() - begin > kPatience) return false;
    }
}

// True in one lane of a converged warp, always the same one.  The compiler knows that it is one, and keeps what tcgen05 and TMA
// instructions take in uniform registers; behind `lane == 0` each of them is wrapped into a loop over lanes.
__device__ __forceinline__ bool elect_one() {
    uint32_t one;
    asm volatile("{ .reg .pred p; elect.sync _|p, 0xffffffff; selp.u32 %0, 1, 0, p; }" : "=r"(one));
    return one;
}

// Box of 128 columns by the map's rows at (column, row) into shared memory; what lies outside the matrix is zero.
__device__ __forceinline__ void fetch_tile(const CUtensorMap* map, void* to, uint64_t* bar, int col, int row) {
    asm volatile("cp.async.bulk.tensor.2d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(smem_at(to)),
                 "l"(map), "r"(col), "r"(row), "r"(smem_at(bar)) : "memory");
}

// A word on its way to shared memory, zero instead where it is not there.
__device__ __forceinline__ void fetch_word(float* to, const float* from, bool there) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(smem_at(to)), "l"(from), "r"(there ? 4 : 0) : "memory");
}

// Operand in shared memory, K-major rows of 128 bytes in the 128-byte swizzle, eight rows (1024 bytes) to a group.
__device__ __forceinline__ uint64_t operand_desc(const void* tile) {
    return (uint64_t)((smem_at(tile) & 0x3ffffu) >> 4) | 1ull << 16 | (uint64_t)(1024 >> 4) << 32 | 1ull << 46 | 2ull << 61;
}
__device__ __forceinline__ void multiply(uint32_t tmem, uint64_t items, uint64_t users, uint32_t idesc, bool add) {
    asm volatile("{ .reg .pred p; setp.ne.b32 p, %4, 0; tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p; }" ::"r"(tmem), "l"(items), "l"(users), "r"(idesc),
                 "r"((uint32_t)add) : "memory");
}
__device__ __forceinline__ void commit(uint64_t* bar) {        // arrives when the matrix instructions so far are done
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_at(bar)) : "memory");
}
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }

// Sixteen or eight consecutive columns of the warp's 32 lanes, under way until wait_columns.
template <int N> __device__ __forceinline__ void read_columns(uint32_t tmem, uint32_t (&r)[N]) {
    static_assert(N == 8 || N == 16, "");
    if constexpr (N == 16)
        asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
            : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]) : "r"(tmem));
    else
        asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
            : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]) : "r"(tmem));
}
// The registers are operands, so that nothing that uses them is moved before the wait.
template <int N> __device__ __forceinline__ void wait_columns(uint32_t (&r)[N]) {
    if constexpr (N == 16)
        asm volatile("tcgen05.wait::ld.sync.aligned;" : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]),
            "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]) :: "memory");
    else
        asm volatile("tcgen05.wait::ld.sync.aligned;" : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]) :: "memory");
}

// Two products, two sums at once.
__device__ __forceinline__ uint64_t pair_of(float x, float y) { return (uint64_t)__float_as_uint(y) << 32 | __float_as_uint(x); }
__device__ __forceinline__ uint64_t pair_of(uint32_t x, uint32_t y) { return (uint64_t)y << 32 | x; }
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) { uint64_t d; asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b)); return d; }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) { uint64_t d; asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c)); return d; }

__device__ __forceinline__ float half_of(uint64_t pair, int which) { return __uint_as_float((uint32_t)(pair >> 32 * which)); }

// Scales may be any numbers of fp32, and a step on the way may leave its range where the score does not.  A block's sum x is 0 or between 2^-18
// and 2^25 in magnitude (128 products of e4m3 values, multiples of 2^-9 and at most 448): times a scale of 2^-100 to 2^100 it is a normal
// number, and times the other scale it is the block's part of the score.  So the first factor decides: the lane's scale, or in SQUARE the
// product of both.  Where it is a far one the score is worked out a second time, from its rows.
__device__ __forceinline__ bool is_far(float lane_scale) {
    const uint32_t m = __float_as_uint(lane_scale) & 0x7fffffffu;
    return m != 0 && m - (27u << 23) > (200u << 23);
}
__device__ __forceinline__ bool is_far(float lane_scale, float col_scale) {
    const uint32_t m = __float_as_uint(lane_scale * col_scale) & 0x7fffffffu;
    return m - (1u << 23) >= (254u << 23) && lane_scale != 0.f && col_scale != 0.f;
}

// One score with its scales applied in fp64, from rows that start on 16 bytes.
__device__ __forceinline__ float exact_score(const ProductArgs& p, uint32_t l, uint32_t c) {
    const uint8_t* const x = p.lane.row_data + l * p.lane.stride, *const y = p.col.row_data + c * p.col.stride;
    float sum = 0.f;
#pragma unroll 1
    for (uint32_t b = 0; b < p.blocks; b++) {
        const uint32_t end = min(p.width, (b + 1) * kScaleBlock);
        float dot = 0.f;
        uint32_t k = b * kScaleBlock;
#pragma unroll 1
        for (; k + 16 <= end; k += 16) {
            const Piece<E4m3, 16> u = load_piece<E4m3, 16>(reinterpret_cast<const E4m3*>(x + k)), v = load_piece<E4m3, 16>(reinterpret_cast<const E4m3*>(y + k));
#pragma unroll
            for (int i = 0; i < 16; i++) dot = fmaf(as_float(u.v[i]), as_float(v.v[i]), dot);
        }
#pragma unroll 1
        for (; k < end; k++) dot = fmaf(as_float(load_piece<E4m3, 1>(reinterpret_cast<const E4m3*>(x + k)).v[0]), as_float(load_piece<E4m3, 1>(reinterpret_cast<const E4m3*>(y + k)).v[0]), dot);
        sum += __double2float_rn((double)dot * p.lane.of(b, l) * p.col.of(b, c));
    }
    return sum;
}

// Stores N columns of the warp's lanes, two to an element of v, at the offsets `at` from an address that is the same for the warp.
template <typename Out, int N>
__device__ __forceinline__ void store_columns(uint8_t* base, const uint32_t* at, const uint64_t* v, bool there, int cols) {
    if (cols >= N) {
#pragma unroll
        for (int k = 0; k < N; k++) if (there) *reinterpret_cast<Out*>(base + at[k]) = from_float<Out>(half_of(v[k / 2], k & 1));
    } else {
#pragma unroll
        for (int k = 0; k < N; k++) if (there && k < cols) *reinterpret_cast<Out*>(base + at[k]) = from_float<Out>(half_of(v[k / 2], k & 1));
    }
}

// Stores R rows of 128 scores, fp32 in shared memory, each times its scale: a warp, WIDE neighbours a lane.
template <typename Out, int R, int WIDE>
__device__ __forceinline__ void store_whole(uint8_t* to, size_t pitch, const float* from, const float (&s)[R], int lane) {
#pragma unroll
    for (int r = 0; r < R; r++, to += pitch) {
#pragma unroll
        for (int k = 0; k < 4 / WIDE; k++) {
            const Piece<float, WIDE> x = reinterpret_cast<const Piece<float, WIDE>*>(from + r * kLanes)[lane + 32 * k];
            Piece<Out, WIDE> y;
#pragma unroll
            for (int i = 0; i < WIDE; i++) y.v[i] = from_float<Out>(x.v[i] * s[r]);
            reinterpret_cast<Piece<Out, WIDE>*>(to)[lane + 32 * k] = y;
        }
    }
}

// Stores the warp's 32 rows of NC scores, two to an element of v, along the rows: 64 bytes of each row at a time go through `transit`.
// `out`: the first row's first score; rows and cols: how many there are of them.
template <typename Out, int NC>
__device__ __forceinline__ void store_rows(const uint64_t (&v)[NC / 2], uint8_t* transit, Out* out, size_t stride, int rows, int cols, int lane) {
    constexpr int kPiece = 64 / sizeof(Out);                    // scores of a row's piece
    const uint32_t odd = (uint32_t)(reinterpret_cast<uintptr_t>(out) | stride * sizeof(Out));
#pragma unroll
    for (int c0 = 0; c0 < NC; c0 += kPiece) {
        Out mine[kPiece];
#pragma unroll
        for (int k = 0; k < kPiece; k++) mine[k] = from_float<Out>(half_of(v[(c0 + k) / 2], k & 1));
        __syncwarp();
#pragma unroll
        for (int k = 0; k < 4; k++) reinterpret_cast<uint4*>(transit + lane * kStagePitch)[k] = reinterpret_cast<const uint4*>(mine)[k];
        __syncwarp();
        if (odd % 16 == 0 && c0 + kPiece <= cols) {             // 16 bytes a lane, eight rows at once
#pragma unroll
            for (int r0 = 0; r0 < 32; r0 += 8) {
                const int r = r0 + lane / 4;
                const uint4 x = *reinterpret_cast<const uint4*>(transit + r * kStagePitch + lane % 4 * 16);
                if (r < rows) *reinterpret_cast<uint4*>(out + r * stride + c0 + lane % 4 * (16 / sizeof(Out))) = x;
            }
        } else if (odd % 4 == 0 && c0 + kPiece <= cols) {       // 4 bytes a lane, two rows at once
#pragma unroll 4
            for (int r0 = 0; r0 < 32; r0 += 2) {
                const int r = r0 + lane / 16;
                const uint32_t x = *reinterpret_cast<const uint32_t*>(transit + r * kStagePitch + lane % 16 * 4);
                if (r < rows) *reinterpret_cast<uint32_t*>(out + r * stride + c0 + lane % 16 * (4 / sizeof(Out))) = x;
            }
        } else {
            for (int r = 0; r < rows; r++)
                if (lane < kPiece && c0 + lane < cols) out[r * stride + c0 + lane] = reinterpret_cast<const Out*>(transit + r * kStagePitch)[lane];
        }
    }
}

template <int CN, typename Out, Mode MODE>
__global__ void __launch_bounds__(Shape<CN, MODE>::threads, 1) product_kernel(const __grid_constant__ CUtensorMap lane_map, const __grid_constant__ CUtensorMap col_map, const ProductArgs p) {
    using S = Shape<CN, MODE>;
    constexpr int kStages = S::stages, kBuffers = S::buffers, kGroup = CN / S::groups, kRead = kGroup < 16 ? 8 : 16;
    extern __shared__ uint8_t raw[];
    uint8_t* const stages = raw + (1024 - smem_at(raw) % 1024) % 1024;                                               // the swizzle's period
    uint8_t* const transit = stages + kStages * S::stage_bytes;
    float* const scales = reinterpret_cast<float*>(transit + S::transit);                                            // [kScaleSteps][columns', lanes']
    uint64_t* const full = reinterpret_cast<uint64_t*>(scales + kScaleSteps * S::step_scales), *const empty = full + kStages;
    uint64_t* const ready = empty + kStages, *const spare = ready + kBuffers;                                        // accumulators: summed, read back
    uint64_t* const fetched = spare + kBuffers, *const judged = fetched + kScaleSteps, *const used = judged + kScaleSteps;      // scales: there, looked at, used
    uint32_t* const tmem_slot = reinterpret_cast<uint32_t*>(used + kScaleSteps), *const any_far = tmem_slot + 1;
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;     // the same for the warp, and known to be
    if (threadIdx.x == 0) {
        for (int s = 0; s < kStages; s++) { barrier_init(full + s, 1); barrier_init(empty + s, 1); }
        for (int b = 0; b < kBuffers; b++) { barrier_init(ready + b, 1); barrier_init(spare + b, S::readers); }
        for (int s = 0; s < kScaleSteps; s++) { barrier_init(fetched + s, 32); barrier_init(judged + s, 1); barrier_init(used + s, S::readers); }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 0) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_at(tmem_slot)), "n"(S::tmem_columns) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = *tmem_slot;
    // first rows of tile t
    const auto user_of = [&](uint32_t t) { return t % p.user_tiles * (MODE == SQUARE ? kLanes : CN); };
    const auto item_of = [&](uint32_t t) { return t / p.user_tiles * (MODE == SQUARE ? CN : kLanes); };
    const auto lane_of = [&](uint32_t t) { return MODE == SQUARE ? user_of(t) : item_of(t); };
    const auto col_of = [&](uint32_t t) { return MODE == SQUARE ? item_of(t) : user_of(t); };
    const auto scores_stored = [&]() { asm volatile("bar.sync %0, %1;" ::"n"(1 + S::groups), "n"(S::threads) : "memory"); };      // the whole block meets, from both branches
    if (warp >= S::readers) {
        // Where sums take registers, 384 threads are launched with 168 each; those that hold sums take what the others leave: 128 * 56 + 256 * 224
        if (MODE != ONE) asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
        uint32_t step = 0;
        bool ok = true;
        const auto wait = [&](uint64_t* bar, uint32_t parity) { return __all_sync(0xffffffffu, barrier_wait(bar, parity)); };
        if (warp == S::readers) {                               // operands
            for (uint32_t t = blockIdx.x; ok && t < p.tiles; t += gridDim.x) {
                const int lane0 = (int)lane_of(t), col0 = (int)col_of(t);
                for (uint32_t c = 0; c < p.blocks; c++, step++) {
                    const int s = step % kStages;
                    if (step >= kStages && !(ok = wait(empty + s, (step / kStages + 1) & 1))) break;
                    if (elect_one()) {
                        barrier_expect(full + s, S::stage_bytes);
                        fetch_tile(&lane_map, stages + s * S::stage_bytes, full + s, (int)(c * kScaleBlock), lane0);
                        fetch_tile(&col_map, stages + s * S::stage_bytes + kLaneTileBytes, full + s, (int)(c * kScaleBlock), col0);
                    }
                    __syncwarp();
                }
            }
            // copies in flight end before the block does
            for (uint32_t q = step > kStages ? step - kStages : 0; q < step; q++) ok &= wait(full + q % kStages, q / kStages & 1);
        }
        if (warp == S::readers + 1) {                           // matrix instructions
            // accumulators fp32 (1 << 4), both operands e4m3 (0) and K-major (0), N / 8, M / 16
            constexpr uint32_t idesc = 1u << 4 | (uint32_t)(CN / 8) << 17 | (uint32_t)(kLanes / 16) << 24;
            for (uint32_t t = blockIdx.x; ok && t < p.tiles; t += gridDim.x)
                for (uint32_t c = 0; c < p.blocks; c++, step++) {
                    const int s = step % kStages, b = step % kBuffers;
                    if (step >= kBuffers && !(ok = wait(spare + b, (step / kBuffers + 1) & 1))) break;
                    if (!(ok = wait(full + s, step / kStages & 1))) break;
                    fence_after();
                    const uint64_t lanes = operand_desc(stages + s * S::stage_bytes), cols = operand_desc(stages + s * S::stage_bytes + kLaneTileBytes);
                    if (elect_one()) {
#pragma unroll
                        for (int k = 0; k < 4; k++) multiply(tmem + b * CN, lanes + 2 * k, cols + 2 * k, idesc, k > 0);      // 32 columns each
                        commit(empty + s);
                        commit(ready + b);
                    }
                    __syncwarp();
                }
        }
        if (warp == S::readers + 2) {                           // scales, 0 for rows that are not there
            for (uint32_t t = blockIdx.x; ok && t < p.tiles; t += gridDim.x) {
                const uint32_t lane0 = lane_of(t), col0 = col_of(t);
                for (uint32_t c = 0; c < p.blocks; c++, step++) {
                    const int q = step % kScaleSteps;
                    if (step >= kScaleSteps && !(ok = wait(used + q, (step / kScaleSteps + 1) & 1))) break;
                    float* const to = scales + q * S::step_scales;
                    const float* const of_lanes = p.lane.scale + (size_t)c * p.lane.scales, *const of_cols = p.col.scale + (size_t)c * p.col.scales;
                    const auto fetch = [&](float* at, const float* from, const Side& side, uint32_t row) {
                        fetch_word(at, from + (min(row, side.rows - 1) >> side.shift), row < side.rows);
                    };
                    if (MODE == SQUARE) { if (lane < S::groups) fetch(to + lane, of_cols, p.col, col0 + lane * kGroup); }
                    else {
#pragma unroll
                        for (int k = lane; k < CN; k += 32) fetch(to + k, of_cols, p.col, col0 + k);
                    }
#pragma unroll
                    for (int k = lane; k < kLanes; k += 32) fetch(to + S::step_scales - kLanes + k, of_lanes, p.lane, lane0 + k);
                    asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_at(fetched + q)) : "memory");
                }
            }
            asm volatile("cp.async.wait_all;" ::: "memory");
        }
        if (warp == S::readers + 3) {                           // looks for far scales ahead of the readers, whom a look and a branch of their own cost a quarter
            bool far = false;                                   // of any step
            for (uint32_t t = blockIdx.x; ok && t < p.tiles; t += gridDim.x)
                for (uint32_t c = 0; c < p.blocks; c++, step++) {
                    const int q = step % kScaleSteps;
                    if (!(ok = wait(fetched + q, step / kScaleSteps & 1))) break;
                    const float* const of_cols = scales + q * S::step_scales, *const of_lanes = of_cols + S::step_scales - kLanes;
#pragma unroll
                    for (int k = lane; k < kLanes; k += 32) {
                        if (MODE == SQUARE) {
#pragma unroll
                            for (int g = 0; g < S::groups; g++) far |= is_far(of_lanes[k], of_cols[g]);
                        } else far |= is_far(of_lanes[k]);
                    }
                    __syncwarp();
                    if (lane == 0) barrier_arrive(judged + q);
                }
            far = __any_sync(0xffffffffu, far);
            if (lane == 0) *any_far = far;
        }
        if (!ok && lane == 0 && p.flags) atomicOr(p.flags, (uint32_t)MASCOT_FLAG_GAVE_UP);
        scores_stored();
        if (*any_far)
            for (uint32_t t = blockIdx.x; t < p.tiles; t += gridDim.x)
                for (uint32_t i = threadIdx.x - 32 * S::readers; i < kLanes * CN; i += S::threads - 32 * S::readers) {
                    const uint32_t l = lane_of(t) + i % kLanes, c = col_of(t) + i / kLanes;
                    bool far = false;
                    if (l < p.lane.rows && c < p.col.rows)
                        for (uint32_t b = 0; b < p.blocks && !far; b++) far = MODE == SQUARE ? is_far(p.lane.of(b, l), p.col.of(b, c)) : is_far(p.lane.of(b, l));
                    if (far) static_cast<Out*>(p.out)[l * p.lane_step + c * p.col_step] = from_float<Out>(exact_score(p, l, c));
                }
    } else {                                                    // sums and scores
        if (MODE != ONE) asm volatile("setmaxnreg.inc.sync.aligned.u32 224;");
        const int group = warp / 4;
        const uint32_t lanes = (uint32_t)(warp % 4) * 32;
        // where a lane's scores of kRead columns go, from the first one: bytes below 2^32, since steps are below 2^26 elements
        uint32_t at[MODE == ROWS ? kRead : 1];
        if (MODE == ROWS) {
#pragma unroll
            for (int k = 0; k < kRead; k++) at[k] = (uint32_t)((lane + k * p.col_step) * sizeof(Out));
        }
        // ONE: the chunk's half of the group's part of `transit`, and neighbours that a store may take at once
        const size_t pitch = p.col_step * sizeof(Out);
        const uint32_t odd = (uint32_t)(reinterpret_cast<uintptr_t>(p.out) | pitch) % 16;
        const int wide = odd % (4 * sizeof(Out)) == 0 ? 4 : odd % (2 * sizeof(Out)) == 0 ? 2 : 1;
        float* chunk = reinterpret_cast<float*>(transit) + group * 2 * kRead * kLanes;
        bool turn = false;
        uint32_t step = 0;
        Reader reader;
        for (uint32_t t = blockIdx.x; t < p.tiles; t += gridDim.x) {
            const uint32_t l = lane_of(t) + lanes, c0 = col_of(t) + group * kGroup;      // the warp's first lane and column
            uint8_t* const out = static_cast<uint8_t*>(p.out) + (l * p.lane_step + c0 * p.col_step) * sizeof(Out);
            const int rows = l < p.lane.rows ? (int)min(p.lane.rows - l, 32u) : 0, cols = c0 < p.col.rows ? (int)min(p.col.rows - c0, (uint32_t)kGroup) : 0;
            uint64_t sum[MODE == ONE ? 1 : kGroup / 2] = {};    // two columns each
            for (uint32_t c = 0; c < p.blocks; c++, step++) {
                const int b = step % kBuffers, q = step % kScaleSteps;
                const float* const scale = scales + q * S::step_scales;
                const uint32_t from = tmem + (lanes << 16) + b * CN + group * kGroup;
                reader.waited(__all_sync(0xffffffffu, reader.ok() && barrier_wait(judged + q, step / kScaleSteps & 1) && barrier_wait(ready + b, step / kBuffers & 1)));
                fence_after();
                float lane_scale = scale[S::step_scales - kLanes + lanes + lane];
                if (MODE == SQUARE) lane_scale *= scale[group];
                lane_scale = reader.factor(lane_scale);
                const uint64_t lane_scales = pair_of(lane_scale, lane_scale);
                const auto release = [&]() {                    // the accumulator has been read
                    fence_before();
                    __syncwarp();
                    if (lane == 0) reader.hand_back([&] { barrier_arrive(spare + b); });
                };
                if constexpr (MODE == ONE && CN == 16) {        // few users: a store of 32 scores for each, and no meeting
                    if (cols > 0) {
                        uint32_t part[kRead];
                        read_columns<kRead>(from, part);
                        wait_columns<kRead>(part);
                        release();
#pragma unroll
                        for (int k = 0; k < kRead; k++)
                            if (k < cols && lane < rows) reinterpret_cast<Out*>(out + k * pitch)[lane] = from_float<Out>(__uint_as_float(part[k]) * lane_scale * scale[group * kGroup + k]);
                    } else release();
                } else if constexpr (MODE == ONE) {
                    constexpr int kRows = kRead / 4;            // of a chunk, for each of the four warps
                    const int items = (int)min(p.lane.rows - (l - lanes), (uint32_t)kLanes), row0 = warp % 4 * kRows;
                    uint8_t* row = out - lanes * sizeof(Out) + row0 * pitch;
                    const float* of_rows = scale + group * kGroup + row0;
                    uint32_t part[kRead];
                    read_columns<kRead>(from, part);
#pragma unroll 1
                    for (int left = cols - row0, k0 = 0; k0 < kGroup; k0 += kRead, left -= kRead, row += kRead * pitch, of_rows += kRead) {
                        float* const to = chunk + lanes + lane;
                        wait_columns<kRead>(part);
#pragma unroll
                        for (int k = 0; k < kRead; k += 2) {
                            const uint64_t x = mul2(pair_of(part[k], part[k + 1]), lane_scales);
                            to[k * kLanes] = half_of(x, 0);
                            to[(k + 1) * kLanes] = half_of(x, 1);
                        }
                        if (k0 + kRead < kGroup) read_columns<kRead>(from + k0 + kRead, part);
                        else release();
                        asm volatile("bar.sync %0, 128;" ::"r"(1 + group) : "memory");     // one a chunk: its half of `transit` is written again two chunks on
                        const float* const rows_at = chunk + row0 * kLanes;
                        float s[kRows];
#pragma unroll
                        for (int r = 0; r < kRows; r++) s[r] = reader.factor(of_rows[r]);
                        if (items == kLanes && left >= kRows) {
                            if (wide == 4) store_whole<Out, kRows, 4>(row, pitch, rows_at, s, lane);
                            else if (sizeof(Out) == 2 && wide == 2) store_whole<Out, kRows, 2>(row, pitch, rows_at, s, lane);
                            else store_whole<Out, kRows, 1>(row, pitch, rows_at, s, lane);
                        } else {
#pragma unroll
                            for (int r = 0; r < kRows; r++) {
                                if (r >= left) break;
                                for (int i = lane; i < items; i += 32) reinterpret_cast<Out*>(row + r * pitch)[i] = from_float<Out>(rows_at[r * kLanes + i] * s[r]);
                            }
                        }
                        chunk = turn ? chunk - kRead * kLanes : chunk + kRead * kLanes;
                        turn = !turn;
                    }
                } else {
                    uint32_t part[2][kRead];
                    read_columns<kRead>(from, part[0]);
#pragma unroll
                    for (int k0 = 0; k0 < kGroup; k0 += kRead) {
                        uint32_t (&now)[kRead] = part[k0 / kRead & 1];
                        wait_columns<kRead>(now);
                        if (k0 + kRead < kGroup) read_columns<kRead>(from + k0 + kRead, part[(k0 / kRead + 1) & 1]);
                        else release();
#pragma unroll
                        for (int k = 0; k < kRead; k += 4) {
                            const uint64_t x[2] = {pair_of(now[k], now[k + 1]), pair_of(now[k + 2], now[k + 3])};
                            if constexpr (MODE == SQUARE) {
                                sum[(k0 + k) / 2] = fma2(x[0], lane_scales, sum[(k0 + k) / 2]);
                                sum[(k0 + k) / 2 + 1] = fma2(x[1], lane_scales, sum[(k0 + k) / 2 + 1]);
                            } else {
                                const ulonglong2 s = *reinterpret_cast<const ulonglong2*>(scale + group * kGroup + k0 + k);
                                sum[(k0 + k) / 2] = fma2(mul2(x[0], lane_scales), s.x, sum[(k0 + k) / 2]);
                                sum[(k0 + k) / 2 + 1] = fma2(mul2(x[1], lane_scales), s.y, sum[(k0 + k) / 2 + 1]);
                            }
                        }
                    }
                }
                __syncwarp();
                if (lane == 0) reader.hand_back([&] { barrier_arrive(used + q); });
            }
            if constexpr (MODE == ROWS) {
#pragma unroll
                for (int k = 0; k < kGroup; k += 4) {
                    const uint64_t y[2] = {sum[k / 2], sum[k / 2 + 1]};
                    store_columns<Out, 4>(out + k / kRead * kRead * p.col_step * sizeof(Out), at + k % kRead, y, lane < rows, cols - k);
                }
            }
            if constexpr (MODE == SQUARE) store_rows<Out, kGroup>(sum, transit + warp * 32 * kStagePitch, reinterpret_cast<Out*>(out), p.lane_step, rows, cols, lane);
        }
        if (!reader.ok() && lane == 0 && p.flags) atomicOr(p.flags, (uint32_t)MASCOT_FLAG_GAVE_UP);
        scores_stored();
        fence_before();
    }
    __syncthreads();
    if (warp == 0) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(S::tmem_columns) : "memory");
}

using EncodeTiled = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*, const cuuint32_t*,
                                 CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeTiled encode_tiled() {
    static const EncodeTiled f = [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult found;
        return cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &found) == cudaSuccess && found == cudaDriverEntryPointSuccess ? reinterpret_cast<EncodeTiled>(p) : nullptr;
    }();
    return f;
}
// Boxes of 128 columns by `box_rows` rows.
bool tile_map(CUtensorMap* map, const mascot_rows& m, uint32_t box_rows) {
    const cuuint64_t dims[2] = {m.width, m.rows}, strides[1] = {m.rows > 1 ? m.stride : (m.stride + 15) / 16 * 16};
    const cuuint32_t box[2] = {kScaleBlock, box_rows}, steps[2] = {1, 1};
    return encode_tiled()(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, m.data, dims, strides, box, steps, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                          CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int CN, typename Out, Mode MODE>
cudaError_t launch_product(const mascot_rows& a, const mascot_rows& b, const ProductArgs& given, int sms, cudaStream_t st) {
    using S = Shape<CN, MODE>;
    ProductArgs p = given;                                      // lane side: items, column side: users
    const uint32_t users = MODE == SQUARE ? kLanes : CN, items = MODE == SQUARE ? CN : kLanes;
    if (MODE == SQUARE) { std::swap(p.lane, p.col); std::swap(p.lane_step, p.col_step); }
    CUtensorMap lane_map, col_map;
    if (!tile_map(&lane_map, MODE == SQUARE ? a : b, kLanes) || !tile_map(&col_map, MODE == SQUARE ? b : a, CN)) return cudaErrorInvalidValue;
    p.user_tiles = (uint32_t)((a.rows + users - 1) / users);
    p.tiles = p.user_tiles * (uint32_t)((b.rows + items - 1) / items);
    static LaunchCache cache;
    const cudaError_t e = allow_smem(product_kernel<CN, Out, MODE>, S::smem, cache);
    if (e != cudaSuccess) return e;
    return launch(product_kernel<CN, Out, MODE>, std::min<uint32_t>(p.tiles, sms), S::threads, S::smem, st, lane_map, col_map, p);
}

// Users of a tile: as many as there are, up to 256, but fewer where that leaves SMs without a tile.
int users_of_tile(uint64_t m, uint64_t n, int sms) {
    int users = 16;
    while (users < 256 && (uint64_t)users < m) users *= 2;
    while (users > 32 && (n + kLanes - 1) / kLanes * ((m + users - 1) / users) < (uint64_t)sms) users /= 2;
    return users;
}

template <typename Out, Mode MODE>
cudaError_t launch_users(const mascot_rows& a, const mascot_rows& b, const ProductArgs& p, int sms, cudaStream_t st) {
    switch (users_of_tile(a.rows, b.rows, sms)) {
        case 16: return launch_product<16, Out, MODE>(a, b, p, sms, st);
        case 32: return launch_product<32, Out, MODE>(a, b, p, sms, st);
        case 64: return launch_product<64, Out, MODE>(a, b, p, sms, st);
        case 128: return launch_product<128, Out, MODE>(a, b, p, sms, st);
        default: return launch_product<256, Out, MODE>(a, b, p, sms, st);
    }
}

template <typename Out>
cudaError_t launch_tiles(const mascot_rows& a, const mascot_rows& b, const ProductArgs& p, cudaStream_t st) {
    const int sms = current_sms();
    if (p.blocks == 1) return launch_users<Out, ONE>(a, b, p, sms, st);
    // lanes for users pay where there are enough for all of them; half a tile of items where whole ones leave SMs without a tile
    if (p.lane.shift && a.rows > kLanes)
        return (a.rows + kLanes - 1) / kLanes * ((b.rows + 255) / 256) >= (uint64_t)sms ? launch_product<256, Out, SQUARE>(a, b, p, sms, st) : launch_product<128, Out, SQUARE>(a, b, p, sms, st);
    return launch_users<Out, ROWS>(a, b, p, sms, st);
}

}  // namespace
}  // namespace mascot

using namespace mascot;

extern "C" int mascot_rows_product(const mascot_rows* a, const float* a_scale, const mascot_rows* b, const float* b_scale, uint32_t b_block_rows,
                                   const mascot_rows* out, uint32_t* flags, void* stream) try {
    ROW_CHECK(check_rows("a", a, true));
    ROW_CHECK(check_rows("b", b, true));
    if (((a->rows + 15) / 16) * ((b->rows + kLanes - 1) / kLanes) > 0x3fffffffull) return fail(nullptr, MASCOT_ERR_UNSUPPORTED, "too many scores for one call: split a or b");
    if (!out) return fail(nullptr, MASCOT_ERR_BAD_ARG, "out: null pointer");
    if (out->rows != a->rows || out->width != b->rows) return fail(nullptr, MASCOT_ERR_BAD_ARG, "out: must have a row for each of a, and a column for each of b");
    if (a->width != b->width) return fail(nullptr, MASCOT_ERR_BAD_ARG, "a and b must have one width");
    if (b_block_rows != 1 && b_block_rows != kScaleBlock) return fail(nullptr, MASCOT_ERR_BAD_ARG, "b_block_rows must be 1 or 128");
    if (is_empty(*a) || is_empty(*b)) return MASCOT_OK;
    if (out->type > MASCOT_BF16) return fail(nullptr, MASCOT_ERR_BAD_ARG, "out: must be MASCOT_F32, MASCOT_F16 or MASCOT_BF16");
    if (out->stride < out->width || out->stride >= (1ull << 26)) return fail(nullptr, MASCOT_ERR_BAD_ARG, "out: stride must be from the width to 2^26");
    if (!out->data || !a_scale || !b_scale) return fail(nullptr, MASCOT_ERR_BAD_ARG, "null pointer");
    if (reinterpret_cast<uintptr_t>(out->data) % type_bytes(out->type)) return fail(nullptr, MASCOT_ERR_BAD_ARG, "out: address is not a multiple of the element's size");
    ROW_CHECK(check_words("a_scale", a_scale));
    ROW_CHECK(check_words("b_scale", b_scale));
    ROW_CHECK(check_words("flags", flags));
    for (const auto* m : {a, b})
        if ((m->rows > 1 && m->stride % 16) || reinterpret_cast<uintptr_t>(m->data) % 16) return fail(nullptr, MASCOT_ERR_BAD_ARG, "a and b: base and stride must be multiples of 16 bytes");
    const uint32_t col_blocks = (a->width + kScaleBlock - 1) / kScaleBlock, n_scales = (uint32_t)((b->rows + b_block_rows - 1) / b_block_rows);
    ROW_CHECK(check_distinct("a", a, "out", out));
    ROW_CHECK(check_distinct("b", b, "out", out));
    ROW_CHECK(check_distinct("a_scale", a_scale, 4 * (size_t)col_blocks * a->rows, "out", out));
    ROW_CHECK(check_distinct("b_scale", b_scale, 4 * (size_t)col_blocks * n_scales, "out", out));
    ROW_CHECK(check_distinct("flags", flags, 4, "out", out));
    int device = 0;
    ROW_CHECK(check_device(&device));
    ROW_CHECK(check_memory("a", a->data, device));
    ROW_CHECK(check_memory("b", b->data, device));
    ROW_CHECK(check_memory("a_scale", a_scale, device));
    ROW_CHECK(check_memory("b_scale", b_scale, device));
    ROW_CHECK(check_memory("out", out->data, device));
    ROW_CHECK(check_memory("flags", flags, device));
    if (!encode_tiled()) return fail(nullptr, MASCOT_ERR_UNSUPPORTED, "the driver has no cuTensorMapEncodeTiled");
    ProductArgs p = {};
    p.lane = Side{b_scale, (uint32_t)b->rows, n_scales, b_block_rows == 1 ? 0u : 7u, static_cast<const uint8_t*>(b->data), b->stride};
    p.col = Side{a_scale, (uint32_t)a->rows, (uint32_t)a->rows, 0, static_cast<const uint8_t*>(a->data), a->stride};
    p.out = out->data; p.lane_step = 1; p.col_step = out->stride;
    p.width = a->width; p.blocks = col_blocks;
    p.flags = flags;
    const cudaError_t launched = with_type(out->type, [&](auto* o) { return launch_tiles<std::remove_pointer_t<decltype(o)>>(*a, *b, p, static_cast<cudaStream_t>(stream)); });
    CU(nullptr, launched);
    return MASCOT_OK;
} ROW_CATCH
