// What the operators on factor rows share (row_ops.cu: lookup, preference loss, quantisation; row_gradient.cu: sums by row;
// row_product.cu: scores): checks of their arguments, and elements of the three float types as fp32.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>

#include <cstdint>
#include <new>

#include "handle.h"
#include "launch_cache.h"

namespace mascot {

constexpr uint32_t kScaleBlock = 128;          // columns (and, for square blocks, rows) that share a scale
constexpr uint32_t kMaxWidth = 65536;
constexpr uint64_t kMaxRows = 0x7fffffffull;   // rows and ids are counted in 31 bits

inline size_t type_bytes(uint32_t type) { return type == MASCOT_F32 ? 4 : type == MASCOT_E4M3 ? 1 : 2; }

// Each returns MASCOT_OK or leaves the reason as the last error.
int check_rows(const char* what, const mascot_rows* m, bool e4m3);       // e4m3: that type, else one of the float types
int check_ids(const char* what, const mascot_ids* ids);
int check_distinct(const char* what_a, const mascot_rows* a, const char* what_b, const mascot_rows* b);   // no element in common
int check_distinct(const char* what_a, const void* a, size_t bytes_a, const char* what_b, const mascot_rows* b);
int check_distinct(const char* what_a, const void* a, size_t bytes_a, const char* what_b, const void* b, size_t bytes_b);
int check_words(const char* what, const void* p);                        // an address of 4-byte elements, or null
int check_device(int* device);                                           // the current one (a launch refuses a stream of another one itself)
int check_memory(const char* what, const void* p, int device);           // device memory of that device, or null
int current_sms();                                                          // of the current device

#define ROW_CHECK(call) do { const int rc_ = (call); if (rc_ != MASCOT_OK) return rc_; } while (0)

// Nothing leaves a C entry as an exception: behind the body of one that begins with `try`.
#define ROW_CATCH catch (const std::bad_alloc&) { return MASCOT_ERR_OOM; } catch (...) { return MASCOT_ERR_CUDA; }

inline bool is_empty(const mascot_rows& m) { return m.rows == 0; }
// Whether rows of `m` can be moved in pieces of `elements` aligned elements.
inline bool aligned_rows(const mascot_rows& m, uint32_t elements) {
    return m.width % elements == 0 && m.stride % elements == 0 && reinterpret_cast<uintptr_t>(m.data) % (elements * type_bytes(m.type)) == 0;
}

struct Ids {
    const void* data;
    bool wide;
};
inline Ids ids_of(const mascot_ids& ids) { return Ids{ids.data, ids.bits == 64}; }

// Hands on what a CUDA call returned.  An error that is reported that way does not stay behind as the thread's last one as well, where the
// next check of somebody else would find it.
inline cudaError_t reported(cudaError_t e) {
    if (e != cudaSuccess) cudaGetLastError();
    return e;
}

#ifdef __CUDACC__
// A launch with its own status: the thread's last error may be an old one of the caller's, which is not ours to report or to take away.
template <class Kernel, class... Args>
cudaError_t launch(Kernel kernel, dim3 grid, unsigned block, size_t smem, cudaStream_t st, Args... args) {
    cudaLaunchConfig_t config = {};
    config.gridDim = grid;
    config.blockDim = dim3(block);
    config.dynamicSmemBytes = smem;
    config.stream = st;
    return reported(cudaLaunchKernelEx(&config, kernel, args...));
}

// Raises a kernel's limit of dynamic shared memory, once for a device.
template <class Kernel>
cudaError_t allow_smem(Kernel kernel, size_t bytes, LaunchCache& cache) {
    int dev = 0, fit = 0;
    const cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return reported(e);
    return (cudaError_t)cache.lookup(dev, 0, 0, bytes, [&](size_t most) { return (int)reported(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)most)); },
                                     [](int, size_t, int*) { return 0; }, &fit);
}

constexpr uint32_t kNoRow = 0xffffffffu;

// Ids as they come, COUNT of them at once: all loads are under way together, whatever the ids' width.
struct RawId { uint32_t low, high; };
template <int COUNT> __device__ __forceinline__ void load_ids(const Ids& ids, const uint32_t (&at)[COUNT], RawId (&id)[COUNT]) {
    if (ids.wide) {
#pragma unroll
        for (int k = 0; k < COUNT; k++) { const uint2 w = __ldg(static_cast<const uint2*>(ids.data) + at[k]); id[k] = {w.x, w.y}; }
    } else {
#pragma unroll
        for (int k = 0; k < COUNT; k++) id[k] = {__ldg(static_cast<const uint32_t*>(ids.data) + at[k]), 0xffffffffu};
    }
}
// The row that it names in a table of `rows` rows, or kNoRow; `bad` collects ids that are neither rows nor -1.
__device__ __forceinline__ uint32_t row_of(RawId id, const Ids& ids, uint32_t rows, bool& bad) {
    if (id.low < rows && (!ids.wide || id.high == 0)) return id.low;
    bad |= (id.low & id.high) != 0xffffffffu;
    return kNoRow;
}
__device__ __forceinline__ uint32_t row_of(const Ids& ids, uint32_t at, uint32_t rows, bool& bad) {
    const uint32_t one[1] = {at};
    RawId id[1];
    load_ids<1>(ids, one, id);
    return row_of(id[0], ids, rows, bad);
}

template <typename T> __device__ __forceinline__ float as_float(T x);
template <> __device__ __forceinline__ float as_float(float x) { return x; }
template <> __device__ __forceinline__ float as_float(__half x) { return __half2float(x); }
template <> __device__ __forceinline__ float as_float(__nv_bfloat16 x) { return __bfloat162float(x); }
struct E4m3 { uint8_t bits; };
template <> __device__ __forceinline__ float as_float(E4m3 x) { return __half2float(__half(__nv_cvt_fp8_to_halfraw(x.bits, __NV_E4M3))); }
template <typename T> __device__ __forceinline__ T from_float(float x);       // to nearest even; too large for binary16: infinity
template <> __device__ __forceinline__ float from_float(float x) { return x; }
template <> __device__ __forceinline__ __half from_float(float x) { return __float2half_rn(x); }
template <> __device__ __forceinline__ __nv_bfloat16 from_float(float x) { return __float2bfloat16_rn(x); }

// N consecutive elements as they are loaded and stored: one piece where N > 1, whose address must be a multiple of its size.
template <typename T, int N> struct alignas(sizeof(T) * N <= 16 ? sizeof(T) * N : 16) Piece { T v[N]; };
template <typename T, int N> __device__ __forceinline__ Piece<T, N> load_piece(const T* p) {
    Piece<T, N> r;
    constexpr int bytes = sizeof(T) * N;
    if constexpr (bytes % 16 == 0) {
#pragma unroll
        for (int i = 0; i < bytes / 16; i++) reinterpret_cast<uint4*>(&r)[i] = __ldg(reinterpret_cast<const uint4*>(p) + i);
    } else if constexpr (bytes == 8) *reinterpret_cast<uint2*>(&r) = __ldg(reinterpret_cast<const uint2*>(p));
    else if constexpr (bytes == 4) *reinterpret_cast<uint32_t*>(&r) = __ldg(reinterpret_cast<const uint32_t*>(p));
    else if constexpr (bytes == 2) *reinterpret_cast<uint16_t*>(&r) = __ldg(reinterpret_cast<const uint16_t*>(p));
    else *reinterpret_cast<uint8_t*>(&r) = __ldg(reinterpret_cast<const uint8_t*>(p));
    return r;
}
// The same from shared memory.
template <typename T, int N> __device__ __forceinline__ Piece<T, N> shared_piece(const uint8_t* p) {
    Piece<T, N> r;
    constexpr int bytes = sizeof(T) * N;
    if constexpr (bytes % 16 == 0) {
#pragma unroll
        for (int i = 0; i < bytes / 16; i++) reinterpret_cast<uint4*>(&r)[i] = reinterpret_cast<const uint4*>(p)[i];
    } else if constexpr (bytes == 8) *reinterpret_cast<uint2*>(&r) = *reinterpret_cast<const uint2*>(p);
    else r = *reinterpret_cast<const Piece<T, N>*>(p);
    return r;
}
template <typename T, int N> __device__ __forceinline__ void store_piece(T* p, const Piece<T, N>& r) { *reinterpret_cast<Piece<T, N>*>(p) = r; }
#endif

// Calls f with a null pointer of the float type `type`, for templates over it.
template <class F> auto with_type(uint32_t type, F f) {
    switch (type) {
        case MASCOT_F16: return f(static_cast<__half*>(nullptr));
        case MASCOT_BF16: return f(static_cast<__nv_bfloat16*>(nullptr));
        default: return f(static_cast<float*>(nullptr));
    }
}

}  // namespace mascot
