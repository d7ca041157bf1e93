// Scores of every row of one e4m3 matrix against every row of another, with a scale for each block of 128 columns.
#include "row_ops.h"

namespace mascot {
namespace {

constexpr int kTileM = 64, kTileN = 64, kProductBlock = 256;

struct ProductArgs {
    const uint8_t *a, *b;
    const float *a_scale, *b_scale;
    void* out;
    size_t a_stride, b_stride, out_stride;
    uint32_t m, n, width, n_scales, b_shift;        // n_scales: scales of b in a column block
};

// A block per 64 x 64 scores, a thread per 4 x 4.
template <typename Out>
__global__ void __launch_bounds__(kProductBlock) product_kernel(const ProductArgs p) {
    __shared__ float sa[32][kTileM + 1], sb[32][kTileN + 1];
    const uint32_t m0 = blockIdx.y * kTileM, n0 = blockIdx.x * kTileN, tx = threadIdx.x % 16, ty = threadIdx.x / 16;
    float acc[4][4] = {};
    for (uint32_t c0 = 0; c0 < p.width; c0 += kScaleBlock) {
        float part[4][4] = {};
        for (uint32_t c1 = c0; c1 < min(p.width, c0 + kScaleBlock); c1 += 32) {
            __syncthreads();
            for (int t = threadIdx.x; t < 32 * 64; t += kProductBlock) {
                const uint32_t c = c1 + t % 32, r = t / 32;
                sa[t % 32][r] = c < p.width && m0 + r < p.m ? as_float(E4m3{p.a[(m0 + r) * p.a_stride + c]}) : 0.f;
                sb[t % 32][r] = c < p.width && n0 + r < p.n ? as_float(E4m3{p.b[(n0 + r) * p.b_stride + c]}) : 0.f;
            }
            __syncthreads();
            for (int c = 0; c < 32; c++)
#pragma unroll
                for (int i = 0; i < 4; i++)
#pragma unroll
                    for (int k = 0; k < 4; k++) part[i][k] = fmaf(sa[c][ty * 4 + i], sb[c][tx * 4 + k], part[i][k]);
        }
        const uint32_t cb = c0 / kScaleBlock;
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
            for (int k = 0; k < 4; k++) {
                const uint32_t m = m0 + ty * 4 + i, n = n0 + tx * 4 + k;
                if (m < p.m && n < p.n) acc[i][k] = fmaf(part[i][k], p.a_scale[(size_t)cb * p.m + m] * p.b_scale[(size_t)cb * p.n_scales + (n >> p.b_shift)], acc[i][k]);
            }
    }
#pragma unroll
    for (int i = 0; i < 4; i++)
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const uint32_t m = m0 + ty * 4 + i, n = n0 + tx * 4 + k;
            if (m < p.m && n < p.n) static_cast<Out*>(p.out)[m * p.out_stride + n] = from_float<Out>(acc[i][k]);
        }
}

}  // namespace
}  // namespace mascot

using namespace mascot;

extern "C" int mascot_rows_product(const mascot_rows* a, const float* a_scale, const mascot_rows* b, const float* b_scale, uint32_t b_block_rows,
                                   const mascot_rows* out, uint32_t* flags, void* stream) {
    ROW_CHECK(check_rows("a", a, true));
    ROW_CHECK(check_rows("b", b, true));
    if (b->rows > kMaxWidth * 128ull) return fail(nullptr, MASCOT_ERR_BAD_ARG, "b: rows must be at most 2^23");
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
        if (m->stride % 16 || reinterpret_cast<uintptr_t>(m->data) % 16) return fail(nullptr, MASCOT_ERR_BAD_ARG, "a and b: base and stride must be multiples of 16 bytes");
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
    const ProductArgs p{static_cast<const uint8_t*>(a->data), static_cast<const uint8_t*>(b->data), a_scale, b_scale, out->data, a->stride, b->stride, out->stride,
                        (uint32_t)a->rows, (uint32_t)b->rows, a->width, n_scales, b_block_rows == 1 ? 0u : 7u};
    const dim3 grid((p.n + kTileN - 1) / kTileN, (p.m + kTileM - 1) / kTileM);
    if (grid.y > 65535) return fail(nullptr, MASCOT_ERR_UNSUPPORTED, "a: too many rows");
    const cudaError_t e = with_type(out->type, [&](auto* o) {
        product_kernel<std::remove_pointer_t<decltype(o)>><<<grid, kProductBlock, 0, static_cast<cudaStream_t>(stream)>>>(p);
        return cudaGetLastError();
    });
    CU(nullptr, e);
    return MASCOT_OK;
}
