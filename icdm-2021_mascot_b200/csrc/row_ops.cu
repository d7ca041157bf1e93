// Operators on factor rows that the caller keeps in device memory: lookup by id, the preference loss, quantisation in
// blocks, and the checks of arguments that they share with row_gradient.cu and row_product.cu.
#include <algorithm>
#include <cmath>
#include <cstdio>

#include "row_ops.h"

namespace mascot {

// ---- arguments ---------------------------------------------------------------------------------------------
namespace {

int refuse(int code, const char* what, const char* why) {
    char msg[256];
    snprintf(msg, sizeof msg, "%s: %s", what, why);
    return fail(nullptr, code, msg);
}

struct Span { uintptr_t begin, end; size_t stride, row; };     // bytes
Span span_of(const mascot_rows& m) {
    const size_t el = type_bytes(m.type), row = m.width * el;
    const uintptr_t at = reinterpret_cast<uintptr_t>(m.data);
    return {at, at + (m.rows ? (m.rows - 1) * m.stride * el + row : 0), m.stride * el, row};
}
bool apart(const Span& a, const Span& b) {
    if (a.begin >= b.end || b.begin >= a.end) return true;
    if (a.stride != b.stride) return false;                    // rows of unlike strides that interleave: not told apart
    const size_t d = b.begin >= a.begin ? (b.begin - a.begin) % a.stride : (a.stride - (a.begin - b.begin) % a.stride) % a.stride;
    return d >= a.row && d + b.row <= a.stride;                // columns of one wider matrix
}

}  // namespace

int check_rows(const char* what, const mascot_rows* m, bool e4m3) {
    if (!m) return refuse(MASCOT_ERR_BAD_ARG, what, "null pointer");
    if (e4m3 ? m->type != MASCOT_E4M3 : m->type > MASCOT_BF16)
        return refuse(MASCOT_ERR_BAD_ARG, what, e4m3 ? "must be MASCOT_E4M3" : "must be MASCOT_F32, MASCOT_F16 or MASCOT_BF16");
    if (m->width == 0 || m->width > kMaxWidth) return refuse(MASCOT_ERR_BAD_ARG, what, "width must be 1 to 65536");
    if (m->rows >= kMaxRows) return refuse(MASCOT_ERR_BAD_ARG, what, "rows must be below 2^31 - 1");
    if (m->stride < m->width) return refuse(MASCOT_ERR_BAD_ARG, what, "stride is less than the width");
    if (m->stride > (1ull << 31)) return refuse(MASCOT_ERR_BAD_ARG, what, "stride must be at most 2^31");
    if (m->rows && !m->data) return refuse(MASCOT_ERR_BAD_ARG, what, "null pointer");
    if (reinterpret_cast<uintptr_t>(m->data) % type_bytes(m->type)) return refuse(MASCOT_ERR_BAD_ARG, what, "address is not a multiple of the element's size");
    return MASCOT_OK;
}

int check_ids(const char* what, const mascot_ids* ids) {
    if (!ids) return refuse(MASCOT_ERR_BAD_ARG, what, "null pointer");
    if (ids->bits != 32 && ids->bits != 64) return refuse(MASCOT_ERR_BAD_ARG, what, "bits must be 32 or 64");
    if (ids->reserved) return refuse(MASCOT_ERR_BAD_ARG, what, "reserved must be 0");
    if (ids->count >= kMaxRows) return refuse(MASCOT_ERR_BAD_ARG, what, "count must be below 2^31 - 1");
    if (ids->count && !ids->data) return refuse(MASCOT_ERR_BAD_ARG, what, "null pointer");
    if (reinterpret_cast<uintptr_t>(ids->data) % (ids->bits / 8)) return refuse(MASCOT_ERR_BAD_ARG, what, "address is not a multiple of the element's size");
    return MASCOT_OK;
}

int check_distinct(const char* what_a, const mascot_rows* a, const char* what_b, const mascot_rows* b) {
    if (apart(span_of(*a), span_of(*b))) return MASCOT_OK;
    char msg[128];
    snprintf(msg, sizeof msg, "%s and %s overlap", what_a, what_b);
    return fail(nullptr, MASCOT_ERR_BAD_ARG, msg);
}
int check_distinct(const char* what_a, const void* a, size_t bytes_a, const char* what_b, const void* b, size_t bytes_b) {
    const uintptr_t pa = reinterpret_cast<uintptr_t>(a), pb = reinterpret_cast<uintptr_t>(b);
    if (!a || !b || !bytes_a || !bytes_b || pa >= pb + bytes_b || pb >= pa + bytes_a) return MASCOT_OK;
    char msg[128];
    snprintf(msg, sizeof msg, "%s and %s overlap", what_a, what_b);
    return fail(nullptr, MASCOT_ERR_BAD_ARG, msg);
}
int check_distinct(const char* what_a, const void* a, size_t bytes_a, const char* what_b, const mascot_rows* b) {
    const Span s = span_of(*b);
    return check_distinct(what_a, a, bytes_a, what_b, b->data, s.end - s.begin);
}

int check_words(const char* what, const void* p) {
    return reinterpret_cast<uintptr_t>(p) % 4 ? refuse(MASCOT_ERR_BAD_ARG, what, "address is not a multiple of the element's size") : MASCOT_OK;
}

int check_device(int* device) {
    if (cudaGetDevice(device) == cudaSuccess) return MASCOT_OK;
    cudaGetLastError();
    return fail(nullptr, MASCOT_ERR_NO_DEVICE, "no usable CUDA device; libmascot has no CPU path");
}

int current_sms() {
    int dev = 0, n = 0;
    return cudaGetDevice(&dev) == cudaSuccess && cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) == cudaSuccess ? n : 1;
}

int check_memory(const char* what, const void* p, int device) {
    if (!p) return MASCOT_OK;
    cudaPointerAttributes at;
    if (cudaPointerGetAttributes(&at, p) != cudaSuccess) {
        cudaGetLastError();
        return fail(nullptr, MASCOT_ERR_NO_DEVICE, "no usable CUDA device; libmascot has no CPU path");
    }
    if (at.type == cudaMemoryTypeManaged || (at.type == cudaMemoryTypeDevice && at.device == device)) return MASCOT_OK;
    return refuse(MASCOT_ERR_BAD_ARG, what, "not memory of the current device");
}

namespace {

// ---- lookup ------------------------------------------------------------------------------------------------
// What bounds it: the rows written, and those read where they are not in L2.  Lanes of a row write 16 bytes each next
// to one another, and a team has the loads of kLookupRows rows in flight before its first store.  2M rows of 128 elements, binary16
// into fp32, from a table of a million: 206 us, 6.2 TB/s of what has to move (a copy: 6.55).
constexpr int kLookupBlock = 256, kLookupRows = 4;

struct LookupArgs {
    const void* table; const float* table_scale; void* out;
    size_t table_stride, out_stride, n;
    Ids ids;
    uint32_t rows, width, scale_rows, block_shift;     // scale_rows: row blocks of a column block
    float scale;
    uint32_t* flags;
};

template <typename In, typename Out, int N>
__global__ void __launch_bounds__(kLookupBlock) lookup_kernel(const LookupArgs a, int team_log2) {
    const int tl = threadIdx.x & ((1 << team_log2) - 1);
    const size_t first = (((size_t)blockIdx.x * kLookupBlock + threadIdx.x) >> team_log2) * kLookupRows;
    if (first >= a.n) return;
    uint32_t at[kLookupRows], row[kLookupRows];
    RawId id[kLookupRows];
    bool bad = false;
#pragma unroll
    for (int k = 0; k < kLookupRows; k++) at[k] = (uint32_t)min(first + k, a.n - 1);
    load_ids<kLookupRows>(a.ids, at, id);
#pragma unroll
    for (int k = 0; k < kLookupRows; k++) row[k] = row_of(id[k], a.ids, a.rows, bad);
    if (bad && tl == 0 && a.flags) atomicOr(a.flags, (uint32_t)MASCOT_FLAG_BAD_ID);
    for (uint32_t c = tl * N; c < a.width; c += N << team_log2) {
        Piece<In, N> in[kLookupRows];
        float s[kLookupRows];
#pragma unroll
        for (int k = 0; k < kLookupRows; k++) {
            s[k] = a.scale;
            if (row[k] != kNoRow) {
                in[k] = load_piece<In, N>(static_cast<const In*>(a.table) + row[k] * a.table_stride + c);
                if (sizeof(In) == 1) s[k] = __ldg(a.table_scale + (size_t)(c / kScaleBlock) * a.scale_rows + (row[k] >> a.block_shift));
            }
        }
#pragma unroll
        for (int k = 0; k < kLookupRows; k++) {
            if (first + k >= a.n) break;
            Piece<Out, N> out;
#pragma unroll
            for (int i = 0; i < N; i++) {
                float x = row[k] == kNoRow ? 0.f : as_float(in[k].v[i]) * s[k];
                if (sizeof(In) == 1) x = row[k] == kNoRow ? 0.f : x * a.scale;
                out.v[i] = from_float<Out>(x);
            }
            store_piece<Out, N>(static_cast<Out*>(a.out) + (first + k) * a.out_stride + c, out);
        }
    }
}

template <typename In, typename Out>
cudaError_t launch_lookup(const LookupArgs& a, bool aligned, cudaStream_t st) {
    constexpr int N = 16 / sizeof(Out);
    const uint32_t pieces = aligned ? a.width / N : a.width;
    int log2 = 0;
    while (log2 < 5 && (1u << log2) < pieces) log2++;
    const size_t teams = (a.n + kLookupRows - 1) / kLookupRows;
    const unsigned grid = (unsigned)((teams + (kLookupBlock >> log2) - 1) / (kLookupBlock >> log2));
    return aligned ? launch(lookup_kernel<In, Out, N>, grid, kLookupBlock, 0, st, a, log2) : launch(lookup_kernel<In, Out, 1>, grid, kLookupBlock, 0, st, a, log2);
}

// ---- preference loss -------------------------------------------------------------------------------------------
// A pair is three rows and a dot product: bound by fetching rows, and by the instructions around them.  A team of lanes takes a
// run of pairs: each lane finds the rows of one of them and hands them round, the rows of kPairs pairs are in flight at once, and
// in the end each lane works out the loss of its own pair.  1M pairs of binary16 rows of 128: 105 us, 7.3 TB/s from L2 and HBM
// together; 180 us while all lanes of a team looked at the ids of every pair.
constexpr int kPairBlock = 256, kPairs = 4;

struct PairArgs {
    const void *P, *Q;
    size_t p_stride, q_stride, n;
    Ids u, i, j;
    uint32_t n_users, n_items, width;
    float beta, smoothing;
    const float *reference, *weight;
    float *loss, *margin, *coef;
    uint32_t* flags;
};

template <typename T, int N>
__global__ void __launch_bounds__(kPairBlock, 2) pair_loss_kernel(const PairArgs a, int team_log2, uint32_t run) {
    const uint32_t team = 1u << team_log2, lane = threadIdx.x & 31, tl = lane & (team - 1);
    const size_t first = (((size_t)blockIdx.x * kPairBlock + threadIdx.x) >> team_log2) * run, at = first + tl;      // this lane's pair
    const bool in_run = tl < run && at < a.n;
    uint32_t u = kNoRow, i = kNoRow, j = kNoRow;
    bool bad = false;
    if (in_run) {
        u = row_of(a.u, (uint32_t)at, a.n_users, bad);
        i = row_of(a.i, (uint32_t)at, a.n_items, bad);
        j = row_of(a.j, (uint32_t)at, a.n_items, bad);
        if (i == kNoRow || j == kNoRow) u = kNoRow;
    }
    if (bad && a.flags) atomicOr(a.flags, (uint32_t)MASCOT_FLAG_BAD_ID);
    const float reference = in_run && a.reference ? __ldg(a.reference + at) : 0.f, w = in_run && a.weight ? __ldg(a.weight + at) : 1.f;
    const uint32_t there = __ballot_sync(0xffffffffu, u != kNoRow) >> (lane & ~(team - 1));
    const T* const P = static_cast<const T*>(a.P), *const Q = static_cast<const T*>(a.Q);
    float margin = 0.f;
    for (uint32_t k0 = 0; k0 < run; k0 += kPairs) {
        float m[kPairs] = {};
        uint32_t uk[kPairs], ik[kPairs], jk[kPairs];
#pragma unroll
        for (int k = 0; k < kPairs; k++) {
            uk[k] = __shfl_sync(0xffffffffu, u, k0 + k, team);
            ik[k] = __shfl_sync(0xffffffffu, i, k0 + k, team);
            jk[k] = __shfl_sync(0xffffffffu, j, k0 + k, team);
        }
        for (uint32_t c = tl * N; c < a.width; c += N << team_log2) {
            Piece<T, N> p[kPairs], qi[kPairs], qj[kPairs];
#pragma unroll
            for (int k = 0; k < kPairs; k++)
                if (k0 + k < team && (there >> (k0 + k) & 1)) {
                    p[k] = load_piece<T, N>(P + uk[k] * a.p_stride + c);
                    qi[k] = load_piece<T, N>(Q + ik[k] * a.q_stride + c);
                    qj[k] = load_piece<T, N>(Q + jk[k] * a.q_stride + c);
                }
#pragma unroll
            for (int k = 0; k < kPairs; k++)
                if (k0 + k < team && (there >> (k0 + k) & 1)) {
#pragma unroll
                    for (int x = 0; x < N; x++) m[k] = fmaf(as_float(p[k].v[x]), as_float(qi[k].v[x]) - as_float(qj[k].v[x]), m[k]);
                }
        }
        for (uint32_t d = team >> 1; d >= 1; d >>= 1) {
#pragma unroll
            for (int k = 0; k < kPairs; k++) m[k] += __shfl_xor_sync(0xffffffffu, m[k], d);
        }
#pragma unroll
        for (int k = 0; k < kPairs; k++) margin = tl == k0 + k ? m[k] : margin;
    }
    if (!in_run) return;
    float loss = 0.f, coef = 0.f;
    if (u != kNoRow && w != 0.f) {
        // log(1 + exp(x)) = max(x, 0) + log(1 + exp(-|x|)); 1 - sigmoid(|z|) = e / (1 + e) keeps its digits where sigmoid is near 1
        const float z = a.beta * (margin - reference), e = expf(-fabsf(z)), soft = log1pf(e), tail = e / (1.f + e), eps = a.smoothing, part = z >= 0.f ? eps : 1.f - eps;
        loss = w * (part == 0.f ? soft : fmaf(part, fabsf(z), soft));      // no 0 * infinity
        coef = w * a.beta * (z >= 0.f ? eps - tail : tail - (1.f - eps));
    }
    if (a.margin) a.margin[at] = margin;
    if (a.loss) a.loss[at] = loss;
    if (a.coef) a.coef[at] = coef;
}

template <typename T>
cudaError_t launch_pair_loss(const PairArgs& a, bool aligned, cudaStream_t st) {
    constexpr int N = 16 / sizeof(T);
    const uint32_t pieces = aligned ? a.width / N : a.width;
    int log2 = 2;
    while (log2 < 5 && (1u << log2) < pieces) log2++;
    // pairs of a team: as many as it has lanes where there are enough of them, one batch where there are few
    const size_t teams = (size_t)current_sms() * 2 * (kPairBlock >> log2);
    const uint32_t run = (uint32_t)std::min<size_t>(1u << log2, std::max<size_t>(kPairs, a.n / teams / kPairs * kPairs));
    const size_t runs = (a.n + run - 1) / run;
    const unsigned grid = (unsigned)((runs + (kPairBlock >> log2) - 1) / (kPairBlock >> log2));
    return aligned ? launch(pair_loss_kernel<T, N>, grid, kPairBlock, 0, st, a, log2, run) : launch(pair_loss_kernel<T, 1>, grid, kPairBlock, 0, st, a, log2, run);
}

// ---- quantisation ------------------------------------------------------------------------------------------
// One pass over the rows: a block stays in registers between its maximum and its rounding.  A power of two as the scale
// makes x / s exact, so that the only rounding is the one to four significant bits, and costs no precision: what
// the larger scale takes from the range is at its lower end, below 2^-14 of the block's maximum.  What bounds it is the
// rows; a warp has those of four blocks (eight of a square) under way at once: 625k rows of 128 floats, 402 MB, take 60 us
// (6.7 TB/s), and took 107 with one block a warp and values converted one by one.
constexpr int kQuantBlock = 256, kQuantWarps = kQuantBlock / 32, kQuantRows = 4, kSquareBlock = 512, kSquareWarps = kSquareBlock / 32;

// The scale of a block from the bits of its largest finite magnitude: 448 = 1.75 * 2^8.
__device__ __forceinline__ float scale_of(uint32_t top) {
    if (top == 0) return 1.f;
    const int e = (int)(top >> 23) - 127 - 8 + ((top & 0x7fffffu) > 0x600000u ? 1 : 0);
    return __uint_as_float((uint32_t)(max(e, -126) + 127) << 23);
}
constexpr uint32_t kInfinity = 0x7f800000u;
__device__ __forceinline__ uint32_t magnitude(float x) { return __float_as_uint(x) & 0x7fffffffu; }

struct QuantArgs {
    const void* x; uint8_t* q; float* scale;
    size_t x_stride, q_stride;
    uint32_t rows, width, row_blocks;
};

// Four elements of a row from column c on, zeros behind its end.
template <typename T, bool ALIGNED> __device__ __forceinline__ Piece<T, 4> load_four(const T* x, uint32_t c, uint32_t width) {
    Piece<T, 4> in;
#pragma unroll
    for (int k = 0; k < 4; k++) in.v[k] = from_float<T>(0.f);
    if (ALIGNED) { if (c < width) in = load_piece<T, 4>(x + c); }
    else {
#pragma unroll
        for (int k = 0; k < 4; k++) if (c + k < width) in.v[k] = load_piece<T, 1>(x + c + k).v[0];
    }
    return in;
}
template <typename T> __device__ __forceinline__ float4 values(const Piece<T, 4>& p) { return make_float4(as_float(p.v[0]), as_float(p.v[1]), as_float(p.v[2]), as_float(p.v[3])); }
// The largest magnitude among them, and `odd` set where one of them is no number or infinite (such ones do not count).
__device__ __forceinline__ uint32_t largest(const float4& v, bool& odd) {
    uint32_t top = max(max(magnitude(v.x), magnitude(v.y)), max(magnitude(v.z), magnitude(v.w)));
    if (top >= kInfinity) {
        odd = true;
        const auto finite = [](float x) { const uint32_t b = magnitude(x); return b < kInfinity ? b : 0u; };
        top = max(max(finite(v.x), finite(v.y)), max(finite(v.z), finite(v.w)));
    }
    return top;
}
template <bool ALIGNED> __device__ __forceinline__ void store_four(uint8_t* q, uint32_t c, uint32_t width, const float4& v, float s, bool odd) {
    const float inverse = __uint_as_float(0x7f000000u - __float_as_uint(s));
    uint32_t out = __nv_cvt_float2_to_fp8x2(make_float2(v.x * inverse, v.y * inverse), __NV_SATFINITE, __NV_E4M3) |
                   (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(v.z * inverse, v.w * inverse), __NV_SATFINITE, __NV_E4M3) << 16;
    if (odd) {                                      // infinities as NaN
        if (magnitude(v.x) >= kInfinity) out |= 0x7fu;
        if (magnitude(v.y) >= kInfinity) out |= 0x7fu << 8;
        if (magnitude(v.z) >= kInfinity) out |= 0x7fu << 16;
        if (magnitude(v.w) >= kInfinity) out |= 0x7fu << 24;
    }
    if (ALIGNED) { if (c < width) *reinterpret_cast<uint32_t*>(q + c) = out; }
    else {
#pragma unroll
        for (int k = 0; k < 4; k++) if (c + k < width) q[c + k] = (uint8_t)(out >> 8 * k);
    }
}

// A warp for kQuantRows rows of a column block, four elements a lane.
template <typename T, bool ALIGNED>
__global__ void __launch_bounds__(kQuantBlock) quantize_rows_kernel(const QuantArgs a) {
    const uint32_t lane = threadIdx.x & 31, cb = blockIdx.y, c = cb * kScaleBlock + lane * 4;
    const uint32_t row0 = (blockIdx.x * kQuantWarps + (threadIdx.x >> 5)) * kQuantRows;
    if (row0 >= a.rows) return;
    Piece<T, 4> v[kQuantRows];
#pragma unroll
    for (int r = 0; r < kQuantRows; r++)
        v[r] = load_four<T, ALIGNED>(static_cast<const T*>(a.x) + min(row0 + r, a.rows - 1) * a.x_stride, c, a.width);
#pragma unroll
    for (int r = 0; r < kQuantRows; r++) {
        if (row0 + r >= a.rows) break;
        bool odd = false;
        const float s = scale_of(__reduce_max_sync(0xffffffffu, largest(values(v[r]), odd)));
        store_four<ALIGNED>(a.q + (row0 + r) * a.q_stride, c, a.width, values(v[r]), s, odd);
        if (lane == 0) a.scale[(size_t)cb * a.row_blocks + row0 + r] = s;
    }
}

// A block of threads per 128 x 128 square, a warp for 8 rows of it.
template <typename T, bool ALIGNED>
__global__ void __launch_bounds__(kSquareBlock) quantize_square_kernel(const QuantArgs a) {
    constexpr int kRows = kScaleBlock / kSquareWarps;
    __shared__ uint32_t tops[kSquareWarps];
    const uint32_t rb = blockIdx.x, cb = blockIdx.y, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const uint32_t c = cb * kScaleBlock + lane * 4, row0 = rb * kScaleBlock + warp * kRows;
    Piece<T, 4> v[kRows];
#pragma unroll
    for (int r = 0; r < kRows; r++) v[r] = load_four<T, ALIGNED>(static_cast<const T*>(a.x) + min(row0 + r, a.rows - 1) * a.x_stride, c, a.width);     // the last row again does not matter
    uint32_t top = 0;
    bool odd = false;
#pragma unroll
    for (int r = 0; r < kRows; r++) top = max(top, largest(values(v[r]), odd));
    top = __reduce_max_sync(0xffffffffu, top);
    if (lane == 0) tops[warp] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kSquareWarps; w++) top = max(top, tops[w]);
    const float s = scale_of(top);
#pragma unroll
    for (int r = 0; r < kRows; r++)
        if (row0 + r < a.rows) store_four<ALIGNED>(a.q + (row0 + r) * a.q_stride, c, a.width, values(v[r]), s, odd);
    if (threadIdx.x == 0) a.scale[(size_t)cb * a.row_blocks + rb] = s;
}

}  // namespace
}  // namespace mascot

using namespace mascot;

extern "C" {

int mascot_rows_lookup(const mascot_rows* table, const float* table_scale, uint32_t block_rows, const mascot_ids* ids, float scale,
                       const mascot_rows* out, uint32_t* flags, void* stream) try {
    const bool e4m3 = table && table->type == MASCOT_E4M3;
    ROW_CHECK(check_rows("table", table, e4m3));
    ROW_CHECK(check_ids("ids", ids));
    ROW_CHECK(check_rows("out", out, false));
    if (out->width != table->width) return fail(nullptr, MASCOT_ERR_BAD_ARG, "out: width is not the table's");
    if (out->rows != ids->count) return fail(nullptr, MASCOT_ERR_BAD_ARG, "out: must have a row for each id");
    if (e4m3 && (block_rows != 1 && block_rows != kScaleBlock)) return fail(nullptr, MASCOT_ERR_BAD_ARG, "block_rows must be 1 or 128");
    if (e4m3 && !table_scale && table->rows) return fail(nullptr, MASCOT_ERR_BAD_ARG, "table_scale: null pointer");
    if (!e4m3 && (table_scale || block_rows)) return fail(nullptr, MASCOT_ERR_BAD_ARG, "table_scale and block_rows belong to a table of MASCOT_E4M3");
    ROW_CHECK(check_words("table_scale", table_scale));
    ROW_CHECK(check_words("flags", flags));
    const uint64_t row_blocks = e4m3 ? (table->rows + block_rows - 1) / block_rows : 0;
    ROW_CHECK(check_distinct("table", table, "out", out));
    ROW_CHECK(check_distinct("ids", ids->data, ids->count * ids->bits / 8, "out", out));
    ROW_CHECK(check_distinct("table_scale", table_scale, row_blocks * ((table->width + kScaleBlock - 1) / kScaleBlock) * 4, "out", out));
    ROW_CHECK(check_distinct("flags", flags, 4, "out", out));
    if (is_empty(*out)) return MASCOT_OK;
    int device = 0;
    ROW_CHECK(check_device(&device));
    if (table->rows) ROW_CHECK(check_memory("table", table->data, device));
    ROW_CHECK(check_memory("table_scale", table_scale, device));
    ROW_CHECK(check_memory("ids", ids->data, device));
    ROW_CHECK(check_memory("out", out->data, device));
    ROW_CHECK(check_memory("flags", flags, device));
    LookupArgs a{table->data, table_scale, out->data, table->stride, out->stride, ids->count, ids_of(*ids), (uint32_t)table->rows, table->width,
                 (uint32_t)row_blocks, block_rows == kScaleBlock ? 7u : 0u, scale, flags};
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    const cudaError_t launched = with_type(out->type, [&](auto* o) {
        using Out = std::remove_pointer_t<decltype(o)>;
        const bool aligned = aligned_rows(*table, 16 / sizeof(Out)) && aligned_rows(*out, 16 / sizeof(Out));
        if (e4m3) return launch_lookup<E4m3, Out>(a, aligned, st);
        return with_type(table->type, [&](auto* t) { return launch_lookup<std::remove_pointer_t<decltype(t)>, Out>(a, aligned, st); });
    });
    CU(nullptr, launched);
    return MASCOT_OK;
} ROW_CATCH

int mascot_pair_loss(const mascot_rows* P, const mascot_rows* Q, const mascot_ids* users, const mascot_ids* preferred, const mascot_ids* other,
                     float beta, float smoothing, const float* reference, const float* weight, float* loss, float* margin, float* coef,
                     uint32_t* flags, void* stream) try {
    ROW_CHECK(check_rows("P", P, false));
    ROW_CHECK(check_rows("Q", Q, false));
    ROW_CHECK(check_ids("users", users));
    ROW_CHECK(check_ids("preferred", preferred));
    ROW_CHECK(check_ids("other", other));
    if (P->width != Q->width || P->type != Q->type) return fail(nullptr, MASCOT_ERR_BAD_ARG, "P and Q must have one width and one type");
    if (users->count != preferred->count || users->count != other->count) return fail(nullptr, MASCOT_ERR_BAD_ARG, "users, preferred and other must have one count");
    if (!(smoothing >= 0.f && smoothing <= 1.f)) return fail(nullptr, MASCOT_ERR_BAD_ARG, "smoothing must be 0 to 1");
    if (!std::isfinite(beta)) return fail(nullptr, MASCOT_ERR_BAD_ARG, "beta must be finite");
    if (!loss && !margin && !coef && users->count) return fail(nullptr, MASCOT_ERR_BAD_ARG, "no output is asked for");
    const size_t n = users->count, vector = n * sizeof(float);
    struct { const char* what; const void* p; size_t bytes; } in[] = {{"users", users->data, n * users->bits / 8}, {"preferred", preferred->data, n * preferred->bits / 8},
        {"other", other->data, n * other->bits / 8}, {"reference", reference, vector}, {"weight", weight, vector}, {"flags", flags, 4}},
        out[] = {{"loss", loss, vector}, {"margin", margin, vector}, {"coef", coef, vector}};
    ROW_CHECK(check_words("reference", reference));
    ROW_CHECK(check_words("weight", weight));
    ROW_CHECK(check_words("flags", flags));
    for (int o = 0; o < 3; o++) {
        ROW_CHECK(check_words(out[o].what, out[o].p));
        for (const auto& x : in) ROW_CHECK(check_distinct(x.what, x.p, x.bytes, out[o].what, out[o].p, vector));
        for (int q = 0; q < o; q++) ROW_CHECK(check_distinct(out[q].what, out[q].p, vector, out[o].what, out[o].p, vector));
        if (out[o].p) {
            ROW_CHECK(check_distinct(out[o].what, out[o].p, vector, "P", P));
            ROW_CHECK(check_distinct(out[o].what, out[o].p, vector, "Q", Q));
        }
    }
    if (n == 0) return MASCOT_OK;
    int device = 0;
    ROW_CHECK(check_device(&device));
    if (P->rows) ROW_CHECK(check_memory("P", P->data, device));
    if (Q->rows) ROW_CHECK(check_memory("Q", Q->data, device));
    for (const auto& x : in) ROW_CHECK(check_memory(x.what, x.p, device));
    for (const auto& x : out) ROW_CHECK(check_memory(x.what, x.p, device));
    const PairArgs a{P->data, Q->data, P->stride, Q->stride, n, ids_of(*users), ids_of(*preferred), ids_of(*other), (uint32_t)P->rows, (uint32_t)Q->rows,
                     P->width, beta, smoothing, reference, weight, loss, margin, coef, flags};
    const cudaError_t launched = with_type(P->type, [&](auto* t) {
        using T = std::remove_pointer_t<decltype(t)>;
        return launch_pair_loss<T>(a, aligned_rows(*P, 16 / sizeof(T)) && aligned_rows(*Q, 16 / sizeof(T)), static_cast<cudaStream_t>(stream));
    });
    CU(nullptr, launched);
    return MASCOT_OK;
} ROW_CATCH

int mascot_rows_quantize(const mascot_rows* x, uint32_t block_rows, const mascot_rows* q, float* scale, void* stream) try {
    ROW_CHECK(check_rows("x", x, false));
    ROW_CHECK(check_rows("q", q, true));
    if (q->rows != x->rows || q->width != x->width) return fail(nullptr, MASCOT_ERR_BAD_ARG, "q: must have the shape of x");
    if (block_rows != 1 && block_rows != kScaleBlock) return fail(nullptr, MASCOT_ERR_BAD_ARG, "block_rows must be 1 or 128");
    if (is_empty(*x)) return MASCOT_OK;
    if (!scale) return fail(nullptr, MASCOT_ERR_BAD_ARG, "scale: null pointer");
    ROW_CHECK(check_words("scale", scale));
    const uint32_t col_blocks = (x->width + kScaleBlock - 1) / kScaleBlock, row_blocks = (uint32_t)((x->rows + block_rows - 1) / block_rows);
    const size_t scale_bytes = (size_t)col_blocks * row_blocks * 4;
    ROW_CHECK(check_distinct("x", x, "q", q));
    ROW_CHECK(check_distinct("scale", scale, scale_bytes, "q", q));
    ROW_CHECK(check_distinct("scale", scale, scale_bytes, "x", x));
    int device = 0;
    ROW_CHECK(check_device(&device));
    ROW_CHECK(check_memory("x", x->data, device));
    ROW_CHECK(check_memory("q", q->data, device));
    ROW_CHECK(check_memory("scale", scale, device));
    const QuantArgs a{x->data, static_cast<uint8_t*>(q->data), scale, x->stride, q->stride, (uint32_t)x->rows, x->width, row_blocks};
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    const bool aligned = aligned_rows(*x, 4) && aligned_rows(*q, 4);
    const cudaError_t launched = with_type(x->type, [&](auto* t) {
        using T = std::remove_pointer_t<decltype(t)>;
        const dim3 grid(block_rows == 1 ? (a.rows + kQuantWarps * kQuantRows - 1) / (kQuantWarps * kQuantRows) : row_blocks, col_blocks);
        if (block_rows == 1) return launch(aligned ? quantize_rows_kernel<T, true> : quantize_rows_kernel<T, false>, grid, kQuantBlock, 0, st, a);
        return launch(aligned ? quantize_square_kernel<T, true> : quantize_square_kernel<T, false>, grid, kSquareBlock, 0, st, a);
    });
    CU(nullptr, launched);
    return MASCOT_OK;
} ROW_CATCH

}  // extern "C"
