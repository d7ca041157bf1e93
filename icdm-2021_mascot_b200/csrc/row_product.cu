// Scores of every row of one e4m3 matrix against every row of another, with a scale for each block of 128 columns.
//
// out[m][n] = sum over column blocks c of a_scale[c][m] * b_scale[c][n] * <a[m], b[n]> within c.  Rows of b (items) are the 128 lanes of
// an accumulator in tensor memory and rows of a (users) its columns: what a warp reads back of one column is 32 consecutive
// scores of one row of `out`, stored as they come, whatever the alignment of `out`.  Each block of 128 columns is one
// accumulation of four tcgen05.mma of kind f8f6f4 (a block is 128 bytes of a row, one line of the 128-byte swizzle); its sum is read
// back, scaled and added in fp32 registers while the tensor cores work on the next one in another part of tensor memory.
//
// A block of threads is persistent and takes every gridDim.x-th tile of 128 items x UN users: one warp fetches operands by TMA, one
// issues the matrix instructions, eight read back, scale and store: warps w and w + 4 the lanes 32 (w % 4) on, half of the users
// each.  Users are the inner index of the tiles, so that an item tile is fetched from HBM once and from L2 after that.
#include <cuda.h>

#include <algorithm>

#include "row_ops.h"

namespace mascot {
namespace {

constexpr int kItems = 128;                          // items of a tile: lanes of tensor memory
constexpr int kEpilogueThreads = 256, kProductThreads = kEpilogueThreads + 128;      // three warpgroups
constexpr int kItemTileBytes = kItems * kScaleBlock;
constexpr long long kPatience = 1ll << 33;           // cycles (four seconds) that a wait may take

__host__ __device__ constexpr int stages_for(int users) { return users == 256 ? 4 : users == 128 ? 6 : 8; }
__host__ __device__ constexpr int buffers_for(int users) { return users == 256 ? 2 : 4; }      // accumulators in tensor memory
__host__ __device__ constexpr int columns_for(int users) { return users * buffers_for(users); }    // powers of two, 64 to 512
__host__ __device__ constexpr size_t smem_for(int users) {
    return 1024 + (size_t)stages_for(users) * (kItemTileBytes + users * kScaleBlock) + 2 * users * 4 + 8 * (2 * stages_for(users) + 2 * buffers_for(users)) + 16;
}

struct ProductArgs {
    const float *a_scale, *b_scale;
    void* out;
    size_t out_stride;
    uint32_t m, n, col_blocks, n_scales, user_tiles, tiles;      // n_scales: scales of b in a column block
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
// Waits for the phase of that parity to end, but not for ever.
__device__ __forceinline__ bool barrier_wait(uint64_t* b, uint32_t parity) {
    const uint32_t at = smem_at(b);
    long long begin = 0;
    for (int round = 0;; round++) {
        uint32_t done;
        asm volatile("{ .reg .pred p; mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2; selp.u32 %0, 1, 0, p; }" : "=r"(done) : "r"(at), "r"(parity) : "memory");
        if (done) return true;
        if (round == 0) begin = clock64();
        else if (clock64() - begin > kPatience) return false;
    }
}

// Box of 128 columns by the map's rows at (column, row) into shared memory; what lies outside the matrix is zero.
__device__ __forceinline__ void fetch_tile(const CUtensorMap* map, void* to, uint64_t* bar, int col, int row) {
    asm volatile("cp.async.bulk.tensor.2d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(smem_at(to)),
                 "l"(map), "r"(col), "r"(row), "r"(smem_at(bar)) : "memory");
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

// N consecutive columns of the warp's 32 lanes.
template <int N> __device__ __forceinline__ void read_columns(uint32_t tmem, float (&v)[N]) {
    static_assert(N == 8 || N == 16 || N == 32, "");
    uint32_t r[N];
    if constexpr (N == 32)
        asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
            : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
              "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31]) : "r"(tmem));
    else if constexpr (N == 16)
        asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
            : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]) : "r"(tmem));
    else
        asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
            : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]) : "r"(tmem));
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
    for (int k = 0; k < N; k++) v[k] = __uint_as_float(r[k]);
}

template <int UN, typename Out, bool SQUARE>
__global__ void __launch_bounds__(kProductThreads, 1) product_kernel(const __grid_constant__ CUtensorMap item_map, const __grid_constant__ CUtensorMap user_map, const ProductArgs p) {
    constexpr int kStages = stages_for(UN), kBuffers = buffers_for(UN), kStageBytes = kItemTileBytes + UN * kScaleBlock, kHalf = UN / 2, kRead = kHalf < 32 ? kHalf : 32;
    extern __shared__ uint8_t raw[];
    uint8_t* const tiles = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) / 1024 * 1024);      // the swizzle's period
    float* const user_scale = reinterpret_cast<float*>(tiles + kStages * kStageBytes);                               // [2][UN]
    uint64_t* const full = reinterpret_cast<uint64_t*>(user_scale + 2 * UN), *const empty = full + kStages;
    uint64_t* const ready = empty + kStages, *const spare = ready + kBuffers;                                        // accumulators: summed, read back
    uint32_t* const tmem_slot = reinterpret_cast<uint32_t*>(spare + kBuffers);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int s = 0; s < kStages; s++) { barrier_init(full + s, 1); barrier_init(empty + s, 1); }
        for (int b = 0; b < kBuffers; b++) { barrier_init(ready + b, 1); barrier_init(spare + b, kEpilogueThreads / 32); }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 0) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_at(tmem_slot)), "n"(columns_for(UN)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = *tmem_slot;

    // 384 threads are launched with 168 registers each; those that hold sums take what the others leave: 128 * 56 + 256 * 224
    if (warp >= kEpilogueThreads / 32) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
        if (warp == kEpilogueThreads / 32 && lane == 0) {       // operands
            uint32_t step = 0;
            bool ok = true;
            for (uint32_t t = blockIdx.x; ok && t < p.tiles; t += gridDim.x) {
                const int item0 = (int)(t / p.user_tiles) * kItems, user0 = (int)(t % p.user_tiles) * UN;
                for (uint32_t c = 0; c < p.col_blocks; c++, step++) {
                    const int s = step % kStages;
                    if (step >= kStages && !(ok = barrier_wait(empty + s, (step / kStages + 1) & 1))) break;
                    barrier_expect(full + s, kStageBytes);
                    fetch_tile(&item_map, tiles + s * kStageBytes, full + s, (int)(c * kScaleBlock), item0);
                    fetch_tile(&user_map, tiles + s * kStageBytes + kItemTileBytes, full + s, (int)(c * kScaleBlock), user0);
                }
            }
            // copies in flight end before the block does
            for (uint32_t q = step > kStages ? step - kStages : 0; q < step; q++) ok &= barrier_wait(full + q % kStages, q / kStages & 1);
            if (!ok && p.flags) atomicOr(p.flags, (uint32_t)MASCOT_FLAG_GAVE_UP);
        }
        if (warp == kEpilogueThreads / 32 + 1 && lane == 0) {   // matrix instructions
            // accumulators fp32 (1 << 4), both operands e4m3 (0) and K-major (0), N / 8, M / 16
            constexpr uint32_t idesc = 1u << 4 | (uint32_t)(UN / 8) << 17 | (uint32_t)(kItems / 16) << 24;
            uint32_t step = 0;
            bool ok = true;
            for (uint32_t t = blockIdx.x; ok && t < p.tiles; t += gridDim.x)
                for (uint32_t c = 0; c < p.col_blocks; c++, step++) {
                    const int s = step % kStages, b = step % kBuffers;
                    if (step >= kBuffers && !(ok = barrier_wait(spare + b, (step / kBuffers + 1) & 1))) break;
                    if (!(ok = barrier_wait(full + s, step / kStages & 1))) break;
                    fence_after();
                    const uint64_t items = operand_desc(tiles + s * kStageBytes), users = operand_desc(tiles + s * kStageBytes + kItemTileBytes);
#pragma unroll
                    for (int k = 0; k < 4; k++) multiply(tmem + b * UN, items + 2 * k, users + 2 * k, idesc, k > 0);     // 32 columns each
                    commit(empty + s);
                    commit(ready + b);
                }
            if (!ok && p.flags) atomicOr(p.flags, (uint32_t)MASCOT_FLAG_GAVE_UP);
        }
    } else {                                                    // scales, sums, scores
        asm volatile("setmaxnreg.inc.sync.aligned.u32 224;");
        const int half = warp / 4;
        const uint32_t lanes = (uint32_t)(warp % 4) * 32;
        const auto scales_of = [&](uint32_t t, uint32_t c, float& user, float& item) {      // this thread's share of a step's scales
            user = item = 0.f;
            if (t >= p.tiles) return;
            const uint32_t item0 = t / p.user_tiles * kItems, u = t % p.user_tiles * UN + threadIdx.x, i = item0 + lanes + lane;
            if (threadIdx.x < UN && u < p.m) user = __ldg(p.a_scale + (size_t)c * p.m + u);
            if (SQUARE) item = __ldg(p.b_scale + (size_t)c * p.n_scales + item0 / kScaleBlock);
            else if (i < p.n) item = __ldg(p.b_scale + (size_t)c * p.n_scales + i);
        };
        uint32_t step = 0;
        bool ok = true;
        float next_user, next_item;
        scales_of(blockIdx.x, 0, next_user, next_item);
        for (uint32_t t = blockIdx.x; t < p.tiles; t += gridDim.x) {
            float sum[kHalf] = {};
            for (uint32_t c = 0; c < p.col_blocks; c++, step++) {
                const int b = step % kBuffers;
                const float item_scale = next_item;
                float* const scale = user_scale + (step & 1) * UN;
                if (threadIdx.x < UN) scale[threadIdx.x] = next_user;
                if (c + 1 < p.col_blocks) scales_of(t, c + 1, next_user, next_item);
                else scales_of(t + gridDim.x, 0, next_user, next_item);
                asm volatile("bar.sync 1, %0;" ::"n"(kEpilogueThreads) : "memory");      // one a step: its buffer is used again two steps on
                ok = __all_sync(0xffffffffu, ok && barrier_wait(ready + b, step / kBuffers & 1));
                fence_after();
#pragma unroll
                for (int k0 = 0; k0 < kHalf; k0 += kRead) {
                    float part[kRead];
                    read_columns<kRead>(tmem + (lanes << 16) + b * UN + half * kHalf + k0, part);
                    if (k0 + kRead == kHalf) {
                        fence_before();
                        __syncwarp();
                        if (lane == 0) barrier_arrive(spare + b);
                    }
#pragma unroll
                    for (int k = 0; k < kRead; k += 4) {
                        const float4 s = *reinterpret_cast<const float4*>(scale + half * kHalf + k0 + k);
                        sum[k0 + k] = fmaf(part[k] * item_scale, s.x, sum[k0 + k]);
                        sum[k0 + k + 1] = fmaf(part[k + 1] * item_scale, s.y, sum[k0 + k + 1]);
                        sum[k0 + k + 2] = fmaf(part[k + 2] * item_scale, s.z, sum[k0 + k + 2]);
                        sum[k0 + k + 3] = fmaf(part[k + 3] * item_scale, s.w, sum[k0 + k + 3]);
                    }
                }
            }
            const uint32_t i = t / p.user_tiles * kItems + lanes + lane, u0 = t % p.user_tiles * UN + half * kHalf;
            if (i < p.n) {
                Out* out = static_cast<Out*>(p.out) + (size_t)u0 * p.out_stride + i;
                const int users = u0 < p.m ? (int)min(p.m - u0, (uint32_t)kHalf) : 0;
#pragma unroll
                for (int k = 0; k < kHalf; k++, out += p.out_stride)
                    if (k < users) *out = from_float<Out>(ok ? sum[k] : __int_as_float(0x7fffffff));
            }
        }
        if (!ok && lane == 0 && p.flags) atomicOr(p.flags, (uint32_t)MASCOT_FLAG_GAVE_UP);
        fence_before();
    }
    __syncthreads();
    if (warp == 0) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(columns_for(UN)) : "memory");
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

int sm_count() {
    int dev = 0, n = 0;
    return cudaGetDevice(&dev) == cudaSuccess && cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) == cudaSuccess ? n : 1;
}

template <int UN, typename Out, bool SQUARE>
cudaError_t launch_product(const mascot_rows& a, const mascot_rows& b, ProductArgs p, int sms, cudaStream_t st) {
    CUtensorMap items, users;
    if (!tile_map(&items, b, kItems) || !tile_map(&users, a, UN)) return cudaErrorInvalidValue;
    p.user_tiles = (p.m + UN - 1) / UN;
    p.tiles = p.user_tiles * ((p.n + kItems - 1) / kItems);
    const cudaError_t e = cudaFuncSetAttribute(product_kernel<UN, Out, SQUARE>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem_for(UN));
    if (e != cudaSuccess) return e;
    product_kernel<UN, Out, SQUARE><<<std::min<uint32_t>(p.tiles, sms), kProductThreads, smem_for(UN), st>>>(items, users, p);
    return cudaGetLastError();
}

// Users of a tile: as many as there are, up to 256, but fewer where that leaves SMs without a tile.
int users_of_tile(uint32_t m, uint32_t n, int sms) {
    int users = 16;
    while (users < 256 && (uint32_t)users < m) users *= 2;
    const uint32_t item_tiles = (n + kItems - 1) / kItems;
    while (users > 32 && (uint64_t)item_tiles * ((m + users - 1) / users) < (uint32_t)sms) users /= 2;
    return users;
}

template <typename Out, bool SQUARE>
cudaError_t launch_tiles(const mascot_rows& a, const mascot_rows& b, const ProductArgs& p, cudaStream_t st) {
    const int sms = sm_count();
    switch (users_of_tile(p.m, p.n, sms)) {
        case 16: return launch_product<16, Out, SQUARE>(a, b, p, sms, st);
        case 32: return launch_product<32, Out, SQUARE>(a, b, p, sms, st);
        case 64: return launch_product<64, Out, SQUARE>(a, b, p, sms, st);
        case 128: return launch_product<128, Out, SQUARE>(a, b, p, sms, st);
        default: return launch_product<256, Out, SQUARE>(a, b, p, sms, st);
    }
}

}  // namespace
}  // namespace mascot

using namespace mascot;

extern "C" int mascot_rows_product(const mascot_rows* a, const float* a_scale, const mascot_rows* b, const float* b_scale, uint32_t b_block_rows,
                                   const mascot_rows* out, uint32_t* flags, void* stream) {
    ROW_CHECK(check_rows("a", a, true));
    ROW_CHECK(check_rows("b", b, true));
    if (((a->rows + 15) / 16) * ((b->rows + kItems - 1) / kItems) > 0x3fffffffull) return fail(nullptr, MASCOT_ERR_UNSUPPORTED, "too many scores for one call: split a or b");
    if (!out) return fail(nullptr, MASCOT_ERR_BAD_ARG, "out: null pointer");
    if (out->rows != a->rows || out->width != b->rows) return fail(nullptr, MASCOT_ERR_BAD_ARG, "out: must have a row for each of a, and a column for each of b");
    if (a->width != b->width) return fail(nullptr, MASCOT_ERR_BAD_ARG, "a and b must have one width");
    if (b_block_rows != 1 && b_block_rows != kScaleBlock) return fail(nullptr, MASCOT_ERR_BAD_ARG, "b_block_rows must be 1 or 128");
    if (is_empty(*a) || is_empty(*b)) return MASCOT_OK;
    if (out->type > MASCOT_BF16) return fail(nullptr, MASCOT_ERR_BAD_ARG, "out: must be MASCOT_F32, MASCOT_F16 or MASCOT_BF16");
    if (out->stride < out->width || out->stride > (1ull << 31)) return fail(nullptr, MASCOT_ERR_BAD_ARG, "out: stride must be from the width to 2^31");
    if (!out->data || !a_scale || !b_scale) return fail(nullptr, MASCOT_ERR_BAD_ARG, "null pointer");
    if (reinterpret_cast<uintptr_t>(out->data) % type_bytes(out->type) || reinterpret_cast<uintptr_t>(a_scale) % 4 || reinterpret_cast<uintptr_t>(b_scale) % 4)
        return fail(nullptr, MASCOT_ERR_BAD_ARG, "an address is not a multiple of the element's size");
    for (const auto* m : {a, b})
        if ((m->rows > 1 && m->stride % 16) || reinterpret_cast<uintptr_t>(m->data) % 16) return fail(nullptr, MASCOT_ERR_BAD_ARG, "a and b: base and stride must be multiples of 16 bytes");
    const uint32_t col_blocks = (a->width + kScaleBlock - 1) / kScaleBlock, n_scales = (uint32_t)((b->rows + b_block_rows - 1) / b_block_rows);
    ROW_CHECK(check_distinct("a", a, "out", out));
    ROW_CHECK(check_distinct("b", b, "out", out));
    ROW_CHECK(check_distinct("a_scale", a_scale, 4 * (size_t)col_blocks * a->rows, "out", out));
    ROW_CHECK(check_distinct("b_scale", b_scale, 4 * (size_t)col_blocks * n_scales, "out", out));
    ROW_CHECK(check_distinct("flags", flags, 4, "out", out));
    ROW_CHECK(check_device());
    ROW_CHECK(check_memory("a", a->data));
    ROW_CHECK(check_memory("b", b->data));
    ROW_CHECK(check_memory("a_scale", a_scale));
    ROW_CHECK(check_memory("b_scale", b_scale));
    ROW_CHECK(check_memory("out", out->data));
    ROW_CHECK(check_memory("flags", flags));
    if (!encode_tiled()) return fail(nullptr, MASCOT_ERR_UNSUPPORTED, "the driver has no cuTensorMapEncodeTiled");
    const ProductArgs p{a_scale, b_scale, out->data, out->stride, (uint32_t)a->rows, (uint32_t)b->rows, col_blocks, n_scales, 0, 0, flags};
    const cudaError_t e = with_type(out->type, [&](auto* o) {
        using Out = std::remove_pointer_t<decltype(o)>;
        return b_block_rows == 1 ? launch_tiles<Out, false>(*a, *b, p, static_cast<cudaStream_t>(stream)) : launch_tiles<Out, true>(*a, *b, p, static_cast<cudaStream_t>(stream));
    });
    CU(nullptr, e);
    return MASCOT_OK;
}
