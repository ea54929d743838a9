// enc_common.cuh -- what the encoder's kernels share: programmatic dependent launch, TMA tensor
// maps, 16-bit vectors of either floating type, activations.
#pragma once
#include <cuda.h>
#include <cuda_bf16.h>

#include <atomic>
#include <type_traits>
#include <utility>

#include "common.cuh"

namespace ragrt {

// Programmatic dependent launch: every encoder kernel is launched so that it may start while
// its predecessor in the stream drains; it does its own set-up, then waits for the
// predecessor's results (griddepcontrol.wait returns at once for a normal launch) and lets
// its own successor start early.
__device__ __forceinline__ void pdl_wait_then_release() {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

// Launch with programmatic stream serialisation (see pdl_wait_then_release).
template <typename... KArgs, typename... Args>
int enc_launch(void (*kern)(KArgs...), dim3 grid, dim3 block, size_t smem, cudaStream_t stream, Args&&... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, std::forward<Args>(args)...);
    if (e != cudaSuccess) {
        cudaGetLastError();
        return fail(RAGRT_ERR_CUDA, "encoder kernel launch: %s", cudaGetErrorString(e));
    }
    count_launch();
    return RAGRT_OK;
}

typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                  const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                  CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

inline EncodeTiledFn enc_encode_fn() {
    static std::atomic<EncodeTiledFn> fn{nullptr};          // two threads' first calls may meet here
    if (!fn.load()) {
        void* f = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) == cudaSuccess &&
            q == cudaDriverEntryPointSuccess)
            fn.store((EncodeTiledFn)f);
    }
    return fn.load();
}

// 16-bit [rows, cols] matrix whose rows lie `stride` elements apart (a multiple of 8), box
// [box_rows x 64 cols], 128-byte swizzle; what lies outside reads 0.
inline int enc_map_2d(CUtensorMap* m, int dtype, const void* base, int64_t rows, int64_t cols, int64_t stride,
                      int box_rows) {
    EncodeTiledFn fn = enc_encode_fn();
    if (!fn) return fail(RAGRT_ERR_CUDA, "cuTensorMapEncodeTiled is not available from the driver");
    const cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
    const cuuint64_t strides[1] = {(cuuint64_t)stride * 2};
    const cuuint32_t box[2] = {64u, (cuuint32_t)box_rows};
    const cuuint32_t estr[2] = {1, 1};
    CUresult r = fn(m, dtype == RAGRT_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2,
                    const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                    CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                    CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return fail(RAGRT_ERR_CUDA, "cuTensorMapEncodeTiled failed (%d)", (int)r);
    return RAGRT_OK;
}

// f32 [rows, cols] matrix (cols a multiple of 4), box [32 rows x 32 cols], 128-byte swizzle, for stores.
inline int enc_map_f32(CUtensorMap* m, const void* base, int64_t rows, int64_t cols) {
    EncodeTiledFn fn = enc_encode_fn();
    if (!fn) return fail(RAGRT_ERR_CUDA, "cuTensorMapEncodeTiled is not available from the driver");
    const cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
    const cuuint64_t strides[1] = {(cuuint64_t)cols * 4};
    const cuuint32_t box[2] = {32u, 32u};
    const cuuint32_t estr[2] = {1, 1};
    CUresult r = fn(m, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 2, const_cast<void*>(base), dims, strides, box, estr,
                    CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_NONE,
                    CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return fail(RAGRT_ERR_CUDA, "cuTensorMapEncodeTiled failed (%d)", (int)r);
    return RAGRT_OK;
}

// 16-bit [rows, heads, dim] tensor, rows `stride` elements apart, box [box_rows x 1 x 64]: one head's
// columns of box_rows rows; columns behind dim and rows behind the last read 0.
inline int enc_map_heads(CUtensorMap* m, int dtype, const void* base, int64_t rows, int heads, int dim, int64_t stride,
                         int box_rows) {
    EncodeTiledFn fn = enc_encode_fn();
    if (!fn) return fail(RAGRT_ERR_CUDA, "cuTensorMapEncodeTiled is not available from the driver");
    const cuuint64_t dims[3] = {(cuuint64_t)dim, (cuuint64_t)heads, (cuuint64_t)rows};
    const cuuint64_t strides[2] = {(cuuint64_t)dim * 2, (cuuint64_t)stride * 2};
    const cuuint32_t box[3] = {64u, 1u, (cuuint32_t)box_rows};
    const cuuint32_t estr[3] = {1, 1, 1};
    CUresult r = fn(m, dtype == RAGRT_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3,
                    const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                    CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                    CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return fail(RAGRT_ERR_CUDA, "cuTensorMapEncodeTiled failed (%d)", (int)r);
    return RAGRT_OK;
}

// The shared-memory attribute of a kernel is per device: set once for each device used.
template <typename K>
int enc_allow_smem(K kern, int bytes, std::atomic<uint64_t>& done) {
    int dev = 0;
    RAGRT_CUDA_TRY(cudaGetDevice(&dev));
    const uint64_t bit = 1ull << (dev & 63);
    if (!(done.load() & bit)) {
        RAGRT_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
        done.fetch_or(bit);
    }
    return RAGRT_OK;
}

// tcgen05 instruction-descriptor bits of an operand pair of type T (0 = fp16, 1 = bf16)
template <typename T>
__host__ __device__ constexpr uint32_t idesc_type() {
    return std::is_same<T, __nv_bfloat16>::value ? (1u << 7) | (1u << 10) : 0u;
}
constexpr uint32_t kIdescAMn = 1u << 15, kIdescBMn = 1u << 16;      // operand is MN-major

// ------------------------------------------------------------------ 16-bit vectors
template <typename T>
struct Pair16;
template <>
struct Pair16<__half> {
    typedef __half2 type;
    static __device__ __forceinline__ float2 up(__half2 v) { return __half22float2(v); }
    static __device__ __forceinline__ __half2 down(float a, float b) { return __floats2half2_rn(a, b); }
};
template <>
struct Pair16<__nv_bfloat16> {
    typedef __nv_bfloat162 type;
    static __device__ __forceinline__ float2 up(__nv_bfloat162 v) { return __bfloat1622float2(v); }
    static __device__ __forceinline__ __nv_bfloat162 down(float a, float b) { return __floats2bfloat162_rn(a, b); }
};

// 8 values of 16 bits <-> 8 floats
template <typename T>
__device__ __forceinline__ void up8(const uint4& u, float (&f)[8]) {
    const typename Pair16<T>::type* h = reinterpret_cast<const typename Pair16<T>::type*>(&u);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 v = Pair16<T>::up(h[i]);
        f[2 * i] = v.x;
        f[2 * i + 1] = v.y;
    }
}
template <typename T>
__device__ __forceinline__ uint4 down8(const float (&f)[8]) {
    uint4 u;
    typename Pair16<T>::type* h = reinterpret_cast<typename Pair16<T>::type*>(&u);
#pragma unroll
    for (int i = 0; i < 4; ++i) h[i] = Pair16<T>::down(f[2 * i], f[2 * i + 1]);
    return u;
}

// 32 bytes at once, a whole sector (address a multiple of 32)
__device__ __forceinline__ void store32(void* p, const uint4& a, const uint4& b) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(a.x), "r"(a.y), "r"(a.z),
                 "r"(a.w), "r"(b.x), "r"(b.y), "r"(b.z), "r"(b.w)
                 : "memory");
}

// ------------------------------------------------------------------ fp32 pairs
// two fp32 values side by side, one instruction for both
__device__ __forceinline__ uint64_t pack2(float a, float b) {
    uint64_t v;
    asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(a), "f"(b));
    return v;
}
__device__ __forceinline__ void unpack2(uint64_t v, float& a, float& b) {
    asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v));
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t v;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(v) : "l"(a), "l"(b), "l"(c));
    return v;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t v;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(v) : "l"(a), "l"(b));
    return v;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
    uint64_t v;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(v) : "l"(a), "l"(b));
    return v;
}

// ------------------------------------------------------------------ activations
__device__ __forceinline__ float gelu_erf(float x) { return 0.5f * x * (1.0f + erff(x * 0.70710678118654752f)); }
__device__ __forceinline__ float gelu_tanh(float x) {
    const float u = 0.7978845608028654f * (x + 0.044715f * x * x * x);
    return 0.5f * x * (1.0f + tanhf(u));
}

}  // namespace ragrt
