// enc_ffn.cu -- the gated feed-forward product of a transformer layer and its backward pass.
//
//   forward    g = x Wg^T, u = x Wu^T, h = act(g) * u                 x [M, K], Wg, Wu [F, K]
//   backward   dg = dh * u * act'(g), du = dh * act(g)
//              dx = dg Wg + du Wu, dWg = dg^T x, dWu = du^T x
//
//   ffn_mma<T, kGated>  both projections of a 128-row tile in one accumulator (columns 0-127 gate,
//                       128-255 up), so that one pass over x feeds both and the activation and the
//                       product are done on the accumulator.  Keeps g and u for the backward pass
//                       when asked to.
//   ffn_mma<T, kDx>     one product over the 2 F columns of [dg | du] and the rows of [Wg ; Wu]:
//                       the two halves add up in the accumulator.
//   ffn_mma<T, kDw>     both weight gradients in one launch, contracted over the rows of x.
//   ffn_act_backward    dg and du, elementwise.
//
// The weight matrices and x are read as they lie: an operand whose contraction index is the row of
// its matrix is fed to the tensor cores MN-major.  Accumulators are fp32; g and u are rounded once
// where they are kept, dg and du where they become operands, results at the end.
#include <algorithm>
#include <atomic>
#include <type_traits>

#include "enc_common.cuh"
#include "tc.cuh"

namespace ragrt {

namespace {

constexpr int kFM = 128;                       // rows per tile
constexpr int kFN = 256;                       // accumulator columns
constexpr int kFK = 64;                        // contraction values per stage (one swizzle atom)
constexpr int kFTileA = kFM * kFK * 2;
constexpr int kFTileB = kFN * kFK * 2;
constexpr int kFStages = 4;
constexpr int kFSmem = 1024 + kFStages * (kFTileA + kFTileB) + 256;
constexpr int kFThreads = 320;                 // TMA warp, MMA warp, 8 epilogue warps
constexpr uint32_t kFWaitLimit = 1u << 26;

enum FfnMode : int { kGated = 0, kDx = 1, kDw = 2 };
enum FfnAct : int { kSilu = 0, kGelu = 1, kGeluTanh = 2 };

struct FfnMaps {
    CUtensorMap a[2], b[2];
};

struct FfnParams {
    int rows, cols;            // of one output matrix
    int depth;                 // length of one contraction
    int act;
    void* out[2];              // kGated: h; kDx: dx; kDw: dWg, dWu
    void* gate;                // kGated: g and u are kept where not null
    void* up;
    int* err;
};

__device__ __forceinline__ float sigmoid(float x) { return __fdividef(1.0f, 1.0f + __expf(-x)); }

// act(x); gelu's tanh form is x * sigmoid(2 u)
__device__ __forceinline__ float ffn_act(float x, int act) {
    if (act == kSilu) return x * sigmoid(x);
    if (act == kGelu) return gelu_erf(x);
    return x * sigmoid(1.5957691216057308f * (x + 0.044715f * x * x * x));
}
// act(x) and act'(x)
__device__ __forceinline__ void ffn_act_grad(float x, int act, float& a, float& d) {
    if (act == kSilu) {
        const float s = sigmoid(x);
        a = x * s;
        d = s * (1.0f + x * (1.0f - s));
    } else if (act == kGelu) {
        const float cdf = 0.5f * (1.0f + erff(x * 0.70710678118654752f));
        a = x * cdf;
        d = fmaf(x * 0.3989422804014327f, __expf(-0.5f * x * x), cdf);
    } else {
        const float s = sigmoid(1.5957691216057308f * (x + 0.044715f * x * x * x));
        a = x * s;
        d = s + x * s * (1.0f - s) * (1.5957691216057308f * (1.0f + 0.134145f * x * x));
    }
}

template <typename T, int kMode>
__global__ void __launch_bounds__(kFThreads, 1) ffn_mma(const __grid_constant__ FfnMaps maps, const FfnParams p) {
    constexpr bool kAMn = kMode == kDw, kBMn = kMode != kGated;
    constexpr int kOutCols = kMode == kGated ? kFN / 2 : kFN;
    extern __shared__ uint8_t ffn_raw[];
    uint8_t* sm = (uint8_t*)(((uintptr_t)ffn_raw + 1023) & ~(uintptr_t)1023);
    uint8_t* sA = sm;
    uint8_t* sB = sm + kFStages * kFTileA;
    uint64_t* full = reinterpret_cast<uint64_t*>(sB + kFStages * kFTileB);
    uint64_t* empty = full + kFStages;
    uint64_t* accf = empty + kFStages;
    uint64_t* acce = accf + 2;
    uint32_t* tslot = reinterpret_cast<uint32_t*>(acce + 2);
    volatile int* abort = reinterpret_cast<volatile int*>(tslot + 1);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int chunks = (p.depth + kFK - 1) / kFK;
    const int nk = kMode == kDx ? 2 * chunks : chunks;
    const int tiles_n = (p.cols + kOutCols - 1) / kOutCols;
    const int tiles_m = (p.rows + kFM - 1) / kFM;
    const int per_out = tiles_n * tiles_m;
    const int tiles = kMode == kDw ? 2 * per_out : per_out;

    if (threadIdx.x == 0) {
        for (int s = 0; s < kFStages; ++s) {
            tc::mbar_init(full + s, 1);
            tc::mbar_init(empty + s, 1);
        }
        for (int b = 0; b < 2; ++b) {
            tc::mbar_init(accf + b, 1);
            tc::mbar_init(acce + b, 8);
        }
        *abort = 0;
        tc::mbar_fence_init();
    }
    if (warp == 1) {
        tc::tmem_alloc(tslot, 512);
        tc::tmem_relinquish();
    }
    tc::fence_before();
    __syncthreads();
    tc::fence_after();
    const uint32_t tbase = *tslot;
    bool failed = false;
    pdl_wait_then_release();

    if (warp == 0) {
        // ------------------------------------------------------------ TMA producer
        if (lane == 0) {
            int g = 0;
            for (int t = blockIdx.x; t < tiles && !failed; t += gridDim.x) {
                const int o = kMode == kDw ? t / per_out : 0, tt = kMode == kDw ? t % per_out : t;
                const int m0 = (tt / tiles_n) * kFM, n0 = (tt % tiles_n) * kOutCols;
                for (int i = 0; i < nk; ++i, ++g) {
                    const int s = g % kFStages;
                    if (g >= kFStages && !tc::mbar_wait_or_abort(empty + s, ((g / kFStages) - 1) & 1, abort, kFWaitLimit)) {
                        failed = true;
                        break;
                    }
                    const int set = kMode == kDx ? (i >= chunks) : o;
                    const int k = (kMode == kDx && i >= chunks ? i - chunks : i) * kFK;
                    uint8_t* da = sA + s * kFTileA;
                    uint8_t* db = sB + s * kFTileB;
                    tc::mbar_arrive_expect_tx(full + s, kFTileA + kFTileB);
                    if (kAMn) {
#pragma unroll
                        for (int j = 0; j < kFM / 64; ++j)
                            tc::tma_load_2d(da + j * 8192, &maps.a[set], m0 + 64 * j, k, full + s);
                    } else {
                        tc::tma_load_2d(da, &maps.a[set], k, m0, full + s);
                    }
                    if (kMode == kGated) {
                        tc::tma_load_2d(db, &maps.b[0], k, n0, full + s);
                        tc::tma_load_2d(db + kFTileB / 2, &maps.b[1], k, n0, full + s);
                    } else {
#pragma unroll
                        for (int j = 0; j < kFN / 64; ++j)
                            tc::tma_load_2d(db + j * 8192, &maps.b[kMode == kDx ? set : 0], n0 + 64 * j, k, full + s);
                    }
                }
            }
        }
    } else if (warp == 1) {
        // ------------------------------------------------------------ MMA issuer
        if (lane == 0) {
            constexpr uint32_t fmt = std::is_same<T, __nv_bfloat16>::value ? (1u << 7) | (1u << 10) : 0u;
            constexpr uint32_t idesc = tc::idesc_f16_f32(kFM, kFN) | fmt | (kAMn ? 1u << 15 : 0u) | (kBMn ? 1u << 16 : 0u);
            int g = 0, j = 0, issued_g = -1;
            for (int t = blockIdx.x; t < tiles && !failed; t += gridDim.x, ++j) {
                const int b = j & 1;
                if (j >= 2 && !tc::mbar_wait_or_abort(acce + b, ((j >> 1) - 1) & 1, abort, kFWaitLimit)) {
                    failed = true;
                    break;
                }
                tc::fence_after();
                const uint32_t d = tbase + (uint32_t)(b * kFN);
                for (int i = 0; i < nk; ++i, ++g) {
                    const int s = g % kFStages;
                    if (!tc::mbar_wait_or_abort(full + s, (g / kFStages) & 1, abort, kFWaitLimit)) {
                        failed = true;
                        break;
                    }
                    tc::fence_after();
                    const uint32_t a = tc::smem_u32(sA + s * kFTileA), bb = tc::smem_u32(sB + s * kFTileB);
#pragma unroll
                    for (int k = 0; k < kFK / 16; ++k)
                        tc::mma_ss(d, kAMn ? tc::sw128_mnmajor_desc(a + 2048 * k, 8192) : tc::sw128_kmajor_desc(a + 32 * k),
                                   kBMn ? tc::sw128_mnmajor_desc(bb + 2048 * k, 8192) : tc::sw128_kmajor_desc(bb + 32 * k),
                                   idesc, (i | k) != 0 ? 1u : 0u);
                    tc::mma_commit(empty + s);
                    issued_g = g;
                }
                if (!failed) tc::mma_commit(accf + b);
            }
            if (failed && issued_g >= 0)   // the last MMAs read shared memory: let them finish
                (void)tc::mbar_wait_bounded(empty + issued_g % kFStages, (issued_g / kFStages) & 1, kFWaitLimit);
        }
    } else {
        // ------------------------------------------------------------ epilogue
        const int quad = warp & 3;                  // tensor-memory lane quadrant of this warp
        const int half = (warp - 2) >> 2;           // which half of the tile's columns
        constexpr int kPer = kOutCols / 64;         // 32-column steps of a half
        int j = 0;
        for (int t = blockIdx.x; t < tiles; t += gridDim.x, ++j) {
            const int o = kMode == kDw ? t / per_out : 0, tt = kMode == kDw ? t % per_out : t;
            const int b = j & 1;
            const int m0 = (tt / tiles_n) * kFM, n0 = (tt % tiles_n) * kOutCols;
            const int row = m0 + quad * 32 + lane;
            const bool ok = tc::mbar_wait_or_abort(accf + b, (j >> 1) & 1, abort, kFWaitLimit);
            if (!__all_sync(0xFFFFFFFFu, ok)) {
                failed = true;
                break;
            }
            tc::fence_after();
            const uint32_t taddr = tbase + ((uint32_t)(quad * 32) << 16) + (uint32_t)(b * kFN);
#pragma unroll 1
            for (int c = half * kPer; c < (half + 1) * kPer; ++c) {
                uint32_t r[32], u[32];
                __syncwarp();
                tc::ld32x32(taddr + 32 * c, r);
                if (kMode == kGated) tc::ld32x32(taddr + kFN / 2 + 32 * c, u);
                tc::wait_ld();
                if (row < p.rows) {
                    const int64_t at = (int64_t)row * p.cols + n0 + 32 * c;
#pragma unroll
                    for (int q = 0; q < 32; q += 8) {
                        if (n0 + 32 * c + q < p.cols) {          // cols is a multiple of 8
                            float f[8];
#pragma unroll
                            for (int e = 0; e < 8; ++e) f[e] = __uint_as_float(r[q + e]);
                            if (kMode == kGated) {
                                float v[8];
#pragma unroll
                                for (int e = 0; e < 8; ++e) v[e] = __uint_as_float(u[q + e]);
                                if (p.gate) {
                                    *reinterpret_cast<uint4*>(static_cast<T*>(p.gate) + at + q) = down8<T>(f);
                                    *reinterpret_cast<uint4*>(static_cast<T*>(p.up) + at + q) = down8<T>(v);
                                }
#pragma unroll
                                for (int e = 0; e < 8; ++e) f[e] = ffn_act(f[e], p.act) * v[e];
                            }
                            *reinterpret_cast<uint4*>(static_cast<T*>(p.out[o]) + at + q) = down8<T>(f);
                        }
                    }
                }
            }
            tc::fence_before();
            __syncwarp();
            if (lane == 0) tc::mbar_arrive(acce + b);
        }
    }
    if (failed && lane == 0) atomicExch(p.err, 1);
    tc::fence_before();
    __syncthreads();
    if (warp == 1) {
        tc::fence_after();
        tc::tmem_dealloc(tbase, 512);
    }
}

// dg = dh * u * act'(g), du = dh * act(g); a thread per 8 values
template <typename T>
__global__ void __launch_bounds__(256) ffn_act_backward(const T* __restrict__ dh, const T* __restrict__ gate,
                                                        const T* __restrict__ up, T* __restrict__ dg,
                                                        T* __restrict__ du, int64_t n8, int act) {
    pdl_wait_then_release();
    for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < n8; i += (int64_t)gridDim.x * blockDim.x) {
        float d[8], g[8], u[8], x[8], y[8];
        up8<T>(reinterpret_cast<const uint4*>(dh)[i], d);
        up8<T>(reinterpret_cast<const uint4*>(gate)[i], g);
        up8<T>(reinterpret_cast<const uint4*>(up)[i], u);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            float a, da;
            ffn_act_grad(g[e], act, a, da);
            x[e] = d[e] * u[e] * da;
            y[e] = d[e] * a;
        }
        reinterpret_cast<uint4*>(dg)[i] = down8<T>(x);
        reinterpret_cast<uint4*>(du)[i] = down8<T>(y);
    }
}

template <typename T, int kMode>
int ffn_launch(const FfnMaps& maps, const FfnParams& p, cudaStream_t stream) {
    // the shared-memory attribute is per device: set it once for each device used
    static std::atomic<uint64_t> attr_set{0};
    int dev = 0;
    RAGRT_CUDA_TRY(cudaGetDevice(&dev));
    const uint64_t bit = 1ull << (dev & 63);
    if (!(attr_set.load() & bit)) {
        RAGRT_CUDA_TRY(cudaFuncSetAttribute(ffn_mma<T, kMode>, cudaFuncAttributeMaxDynamicSharedMemorySize, kFSmem));
        attr_set.fetch_or(bit);
    }
    const int out_cols = kMode == kGated ? kFN / 2 : kFN;
    const int64_t tiles = ceil_div(p.rows, kFM) * ceil_div(p.cols, out_cols) * (kMode == kDw ? 2 : 1);
    return enc_launch(ffn_mma<T, kMode>, dim3((unsigned)std::min<int64_t>(tiles, num_sms())), dim3(kFThreads), kFSmem,
                      stream, maps, p);
}

template <int kMode>
int ffn_launch_typed(int dtype, const FfnMaps& maps, const FfnParams& p, cudaStream_t stream) {
    return dtype == RAGRT_BF16 ? ffn_launch<__nv_bfloat16, kMode>(maps, p, stream)
                               : ffn_launch<__half, kMode>(maps, p, stream);
}

int ffn_check(int32_t M, int32_t F, int32_t K, int32_t act, int32_t dtype) {
    RAGRT_REQUIRE(dtype == RAGRT_F16 || dtype == RAGRT_BF16, "dtype must be RAGRT_F16 or RAGRT_BF16; got %d",
                  (int)dtype);
    RAGRT_REQUIRE(act >= kSilu && act <= kGeluTanh, "unknown activation %d", (int)act);
    RAGRT_REQUIRE(M >= 0 && F >= 8 && F % 8 == 0 && K >= 8 && K % 8 == 0,
                  "gated_ffn needs M >= 0 and F, K multiples of 8 (M=%d F=%d K=%d)", (int)M, (int)F, (int)K);
    return RAGRT_OK;
}

}  // namespace
}  // namespace ragrt

using namespace ragrt;

extern "C" int ragrt_enc_gated_ffn(const void* d_x, const void* d_w_gate, const void* d_w_up, void* d_h, void* d_gate,
                                   void* d_up, int32_t M, int32_t F, int32_t K, int32_t act, int32_t dtype,
                                   void* stream_) {
    int rc = ffn_check(M, F, K, act, dtype);
    if (rc) return rc;
    RAGRT_REQUIRE(!d_gate == !d_up, "d_gate and d_up are kept together or not at all");
    if (M == 0) return RAGRT_OK;
    RAGRT_REQUIRE(d_x && d_w_gate && d_w_up && d_h, "null argument");
    RAGRT_REQUIRE((((uintptr_t)d_x | (uintptr_t)d_w_gate | (uintptr_t)d_w_up | (uintptr_t)d_h | (uintptr_t)d_gate |
                    (uintptr_t)d_up) & 15) == 0,
                  "gated_ffn operands must be 16-byte aligned");
    int* err = device_error_flag();
    if (!err) return fail(RAGRT_ERR_CUDA, "device error flag unavailable");
    FfnMaps m;
    if ((rc = enc_map_2d(&m.a[0], dtype, d_x, M, K, K, kFM)) ||
        (rc = enc_map_2d(&m.b[0], dtype, d_w_gate, F, K, K, kFN / 2)) ||
        (rc = enc_map_2d(&m.b[1], dtype, d_w_up, F, K, K, kFN / 2)))
        return rc;
    m.a[1] = m.a[0];
    FfnParams p{M, F, K, act, {d_h, nullptr}, d_gate, d_up, err};
    return ffn_launch_typed<kGated>(dtype, m, p, (cudaStream_t)stream_);
}

extern "C" int ragrt_enc_gated_ffn_backward(const void* d_dh, const void* d_x, const void* d_w_gate,
                                            const void* d_w_up, const void* d_gate, const void* d_up, void* d_dgate,
                                            void* d_dup, void* d_dx, void* d_dw_gate, void* d_dw_up, int32_t M,
                                            int32_t F, int32_t K, int32_t act, int32_t dtype, void* stream_) {
    int rc = ffn_check(M, F, K, act, dtype);
    if (rc) return rc;
    cudaStream_t stream = (cudaStream_t)stream_;
    RAGRT_REQUIRE(!d_dw_gate == !d_dw_up, "d_dw_gate and d_dw_up are computed together or not at all");
    if (M == 0) {
        if (d_dw_gate) {
            RAGRT_CUDA_TRY(cudaMemsetAsync(d_dw_gate, 0, (size_t)F * K * 2, stream));
            RAGRT_CUDA_TRY(cudaMemsetAsync(d_dw_up, 0, (size_t)F * K * 2, stream));
        }
        return RAGRT_OK;
    }
    RAGRT_REQUIRE(d_dh && d_gate && d_up && d_dgate && d_dup, "null argument");
    RAGRT_REQUIRE(!d_dx || (d_w_gate && d_w_up), "dx needs the weights");
    RAGRT_REQUIRE(!d_dw_gate || d_x, "the weight gradients need x");
    RAGRT_REQUIRE((((uintptr_t)d_dh | (uintptr_t)d_x | (uintptr_t)d_w_gate | (uintptr_t)d_w_up | (uintptr_t)d_gate |
                    (uintptr_t)d_up | (uintptr_t)d_dgate | (uintptr_t)d_dup | (uintptr_t)d_dx | (uintptr_t)d_dw_gate |
                    (uintptr_t)d_dw_up) & 15) == 0,
                  "gated_ffn_backward operands must be 16-byte aligned");
    int* err = device_error_flag();
    if (!err) return fail(RAGRT_ERR_CUDA, "device error flag unavailable");
    const int64_t n8 = (int64_t)M * F / 8;
    const unsigned blocks = (unsigned)std::min<int64_t>(ceil_div(n8, 256), (int64_t)num_sms() * 16);
    rc = dtype == RAGRT_BF16
             ? enc_launch(ffn_act_backward<__nv_bfloat16>, dim3(blocks), dim3(256), 0, stream,
                          (const __nv_bfloat16*)d_dh, (const __nv_bfloat16*)d_gate, (const __nv_bfloat16*)d_up,
                          (__nv_bfloat16*)d_dgate, (__nv_bfloat16*)d_dup, n8, (int)act)
             : enc_launch(ffn_act_backward<__half>, dim3(blocks), dim3(256), 0, stream, (const __half*)d_dh,
                          (const __half*)d_gate, (const __half*)d_up, (__half*)d_dgate, (__half*)d_dup, n8, (int)act);
    if (rc) return rc;
    FfnMaps m;
    if (d_dx) {
        if ((rc = enc_map_2d(&m.a[0], dtype, d_dgate, M, F, F, kFM)) ||
            (rc = enc_map_2d(&m.a[1], dtype, d_dup, M, F, F, kFM)) ||
            (rc = enc_map_2d(&m.b[0], dtype, d_w_gate, F, K, K, kFK)) ||
            (rc = enc_map_2d(&m.b[1], dtype, d_w_up, F, K, K, kFK)))
            return rc;
        FfnParams p{M, K, F, act, {d_dx, nullptr}, nullptr, nullptr, err};
        if ((rc = ffn_launch_typed<kDx>(dtype, m, p, stream))) return rc;
    }
    if (d_dw_gate) {
        if ((rc = enc_map_2d(&m.a[0], dtype, d_dgate, M, F, F, kFK)) ||
            (rc = enc_map_2d(&m.a[1], dtype, d_dup, M, F, F, kFK)) ||
            (rc = enc_map_2d(&m.b[0], dtype, d_x, M, K, K, kFK)))
            return rc;
        m.b[1] = m.b[0];
        FfnParams p{F, K, M, act, {d_dw_gate, d_dw_up}, nullptr, nullptr, err};
        if ((rc = ffn_launch_typed<kDw>(dtype, m, p, stream))) return rc;
    }
    return RAGRT_OK;
}
