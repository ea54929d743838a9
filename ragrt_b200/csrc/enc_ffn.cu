// enc_ffn.cu -- the gated feed-forward product of a transformer layer and its backward pass.
//
//   forward    g = x Wg^T, u = x Wu^T, h = act(g) * u                 x [M, K], Wg, Wu [F, K]
//   backward   dg = dh * u * act'(g), du = dh * act(g)
//              dx = dg Wg + du Wu, dWg = dg^T x, dWu = du^T x
//
// ffn_mma is persistent: pairs of CTAs (cta_group::2) walk 256 x 256 accumulator tiles, each CTA loading
// and draining its half.
//
//   ffn_mma<T, kGated>  both projections of a 256-row tile in one accumulator (columns 0-127 gate,
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

constexpr int kFM = 256;                       // rows per tile, half of them in each CTA of a pair
constexpr int kFN = 256;                       // accumulator columns
constexpr int kFK = 64;                        // contraction values per stage (one swizzle atom)
constexpr int kFTileA = kFM / 2 * kFK * 2;     // bytes of a CTA's half of an operand
constexpr int kFTileB = kFN / 2 * kFK * 2;
constexpr int kFStages = 6;
constexpr int kFOut = 32 * 64 * 2;             // an epilogue warp's 32 rows x 64 columns on their way out
constexpr int kFSmem = 1024 + kFStages * (kFTileA + kFTileB) + 8 * kFOut + 256;
constexpr int kFThreads = 320;                 // TMA warp, MMA warp, 8 epilogue warps
constexpr uint32_t kFWaitLimit = 1u << 26;

enum FfnMode : int { kGated = 0, kDx = 1, kDw = 2 };
enum FfnAct : int { kSilu = 0, kGelu = 1, kGeluTanh = 2 };

struct FfnMaps {
    CUtensorMap a[2], b[2];
    CUtensorMap out[3];        // kGated: h, g, u; kDx: dx; kDw: dWg, dWu
};

struct FfnParams {
    int rows, cols;            // of one output matrix
    int depth;                 // length of one contraction
    int act;
    int keep;                  // kGated: g and u are written too
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

// Tile t of an output of tiles_m x tiles_n tiles, eight tile rows at a time, so that the tiles in flight
// together read few distinct rows and columns.
__device__ __forceinline__ void ffn_place(int t, int tiles_m, int tiles_n, int& m, int& n) {
    const int band = t / (8 * tiles_n), in = t % (8 * tiles_n);
    const int high = min(8, tiles_m - 8 * band);
    m = 8 * band + in % high;
    n = in / high;
}

template <typename T, int kMode>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kFThreads, 1)
ffn_mma(const __grid_constant__ FfnMaps maps, const FfnParams p) {
    constexpr bool kAMn = kMode == kDw, kBMn = kMode != kGated;
    constexpr int kOutCols = kMode == kGated ? kFN / 2 : kFN;
    extern __shared__ uint8_t ffn_raw[];
    uint8_t* sm = (uint8_t*)(((uintptr_t)ffn_raw + 1023) & ~(uintptr_t)1023);
    uint8_t* sA = sm;
    uint8_t* sB = sm + kFStages * kFTileA;
    uint8_t* sO = sB + kFStages * kFTileB;
    uint64_t* full = reinterpret_cast<uint64_t*>(sO + 8 * kFOut);     // [rank 0] both CTAs' halves are there
    uint64_t* empty = full + kFStages;
    uint64_t* accf = empty + kFStages;       // [2] accumulator ready (MMA -> epilogue)
    uint64_t* acce = accf + 2;               // [2] [rank 0] accumulator drained (both epilogues -> MMA)
    uint64_t* drain = acce + 2;
    uint32_t* tslot = reinterpret_cast<uint32_t*>(drain + 1);
    volatile int* abort = reinterpret_cast<volatile int*>(tslot + 1);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = (int)tc::cluster_rank(), pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
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
            tc::mbar_init(acce + b, 16);
        }
        tc::mbar_init(drain, 1);
        *abort = 0;
        tc::mbar_fence_init();
    }
    if (warp == 1) {
        tc::tmem_alloc2(tslot, 512);
        tc::tmem_relinquish2();
    }
    tc::fence_before();
    __syncthreads();
    tc::cluster_sync();                      // the other CTA's barriers are there before anything arrives on them
    tc::fence_after();
    const uint32_t tbase = *tslot;
    bool failed = false;
    pdl_wait_then_release();

    if (warp == 0) {
        // ------------------------------------------------------------ TMA producer
        if (lane == 0) {
            int g = 0;
            for (int t = pair; t < tiles && !failed; t += pairs) {
                const int o = kMode == kDw ? t / per_out : 0;
                int m, n;
                ffn_place(kMode == kDw ? t % per_out : t, tiles_m, tiles_n, m, n);
                const int m0 = m * kFM + rank * (kFM / 2);
                const int n0 = n * kOutCols + (kMode == kGated ? 0 : rank * (kFN / 2));
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
                    const uint32_t bar = tc::cluster_addr(full + s, 0);
                    if (rank == 0) tc::mbar_arrive_expect_tx(full + s, 2 * (kFTileA + kFTileB));
                    if (kAMn) {
#pragma unroll
                        for (int j = 0; j < kFM / 128; ++j)
                            tc::tma_load_2d_pair(da + j * 8192, &maps.a[set], m0 + 64 * j, k, bar);
                    } else {
                        tc::tma_load_2d_pair(da, &maps.a[set], k, m0, bar);
                    }
                    if (kMode == kGated) {           // rank 0: the gate's half of the columns, rank 1: the other
                        tc::tma_load_2d_pair(db, &maps.b[rank], k, n0, bar);
                    } else {
#pragma unroll
                        for (int j = 0; j < kFN / 128; ++j)
                            tc::tma_load_2d_pair(db + j * 8192, &maps.b[kMode == kDx ? set : 0], n0 + 64 * j, k, bar);
                    }
                }
            }
            if (failed && rank == 0)         // copies in flight end before the CTA does
                for (int i = max(0, g - kFStages); i < g; ++i)
                    (void)tc::mbar_wait_bounded(full + i % kFStages, (i / kFStages) & 1, 1u << 16);
        }
    } else if (warp == 1) {
        // ------------------------------------------------------------ MMA issuer, one lane of rank 0's warp
        if (rank == 0) {
            constexpr uint32_t idesc = tc::idesc_f16_f32(kFM, kFN) | idesc_type<T>() | (kAMn ? kIdescAMn : 0u) |
                                       (kBMn ? kIdescBMn : 0u);
            const uint32_t lead = tc::elect_one();
            int g = 0, j = 0;
            for (int t = pair; t < tiles && !failed; t += pairs, ++j) {
                const int b = j & 1;
                bool ok = j < 2 || tc::mbar_wait_or_abort(acce + b, ((j >> 1) - 1) & 1, abort, kFWaitLimit);
                failed = !__all_sync(0xFFFFFFFFu, ok);
                if (failed) break;
                tc::fence_after();
                const uint32_t d = tbase + (uint32_t)(b * kFN);
                for (int i = 0; i < nk; ++i, ++g) {
                    const int s = g % kFStages;
                    ok = tc::mbar_wait_or_abort(full + s, (g / kFStages) & 1, abort, kFWaitLimit);
                    failed = !__all_sync(0xFFFFFFFFu, ok);
                    if (failed) break;
                    tc::fence_after();
                    const uint32_t a = tc::smem_u32(sA + s * kFTileA), bb = tc::smem_u32(sB + s * kFTileB);
#pragma unroll
                    for (int k = 0; k < kFK / 16; ++k)
                        tc::mma_ss2_if(lead, d,
                                       kAMn ? tc::sw128_mnmajor_desc(a + 2048 * k, 8192) : tc::sw128_kmajor_desc(a + 32 * k),
                                       kBMn ? tc::sw128_mnmajor_desc(bb + 2048 * k, 8192) : tc::sw128_kmajor_desc(bb + 32 * k),
                                       idesc, (i | k) != 0 ? 1u : 0u);
                    tc::mma_commit2_if(lead, empty + s);
                }
                if (!failed) tc::mma_commit2_if(lead, accf + b);
            }
            if (failed) {                    // the last products read shared memory: let them finish
                tc::mma_commit2_if(lead, drain);
                (void)tc::mbar_wait_bounded(drain, 0, 1u << 16);
            }
        }
    } else {
        // ------------------------------------------------------------ epilogue
        const int quad = warp & 3;                  // tensor-memory lane quadrant of this warp
        const int half = (warp - 2) >> 2;           // which half of the tile's columns
        constexpr int kBoxes = kOutCols / 128;      // 64-column boxes of a half
        uint8_t* out = sO + (warp - 2) * kFOut;
        const uint32_t drained[2] = {tc::cluster_addr(acce, 0), tc::cluster_addr(acce + 1, 0)};
        // 32 rows x 32 columns of the box: into shared memory, swizzled like the map
        auto put = [&](int c, const float (&f)[32]) {
#pragma unroll
            for (int q = 0; q < 32; q += 8)
                *reinterpret_cast<uint4*>(out + lane * 128 + ((((c & 1) * 4 + q / 8) ^ (lane & 7)) << 4)) =
                    down8<T>(*reinterpret_cast<const float(*)[8]>(f + q));
        };
        auto send = [&](const CUtensorMap* map, int x, int y) {
            tc::fence_proxy_async();
            __syncwarp();
            if (lane == 0) {
                tc::tma_store_2d(map, x, y, out);
                tc::bulk_commit();
                tc::bulk_wait_read();
            }
            __syncwarp();
        };
        int j = 0;
        for (int t = pair; t < tiles; t += pairs, ++j) {
            const int o = kMode == kDw ? t / per_out : 0, b = j & 1;
            int m, n;
            ffn_place(kMode == kDw ? t % per_out : t, tiles_m, tiles_n, m, n);
            const int y = m * kFM + rank * (kFM / 2) + quad * 32;
            const bool ok = tc::mbar_wait_or_abort(accf + b, (j >> 1) & 1, abort, kFWaitLimit);
            if (!__all_sync(0xFFFFFFFFu, ok)) {
                failed = true;
                break;
            }
            tc::fence_after();
            const uint32_t taddr = tbase + ((uint32_t)(quad * 32) << 16) + (uint32_t)(b * kFN);
            const bool rows = y < p.rows;           // of this warp
#pragma unroll 1
            for (int x = 0; x < kBoxes; ++x) {
                const int c0 = (half * kBoxes + x) * 64, at = n * kOutCols + c0;
                if (!rows || at >= p.cols) break;
                if (kMode == kGated && p.keep) {
#pragma unroll 1
                    for (int w = 0; w < 2; ++w) {
#pragma unroll
                        for (int c = 0; c < 2; ++c) {
                            float f[32];
                            tc::ld32x32(taddr + w * (kFN / 2) + c0 + 32 * c, *reinterpret_cast<uint32_t(*)[32]>(f));
                            tc::wait_ld();
                            put(c, f);
                        }
                        send(&maps.out[1 + w], at, y);
                    }
                }
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    float f[32];
                    tc::ld32x32(taddr + c0 + 32 * c, *reinterpret_cast<uint32_t(*)[32]>(f));
                    if (kMode == kGated) {
                        float v[32];
                        tc::ld32x32(taddr + kFN / 2 + c0 + 32 * c, *reinterpret_cast<uint32_t(*)[32]>(v));
                        tc::wait_ld();
                        if (p.act == kSilu) {
#pragma unroll
                            for (int e = 0; e < 32; ++e) f[e] = ffn_act(f[e], kSilu) * v[e];
                        } else if (p.act == kGelu) {
#pragma unroll
                            for (int e = 0; e < 32; ++e) f[e] = ffn_act(f[e], kGelu) * v[e];
                        } else {
#pragma unroll
                            for (int e = 0; e < 32; ++e) f[e] = ffn_act(f[e], kGeluTanh) * v[e];
                        }
                    } else {
                        tc::wait_ld();
                    }
                    put(c, f);
                }
                if (x == kBoxes - 1) {              // all of the accumulator is in registers
                    tc::fence_before();
                    __syncwarp();
                    if (lane == 0) tc::mbar_arrive_cluster(drained[b]);
                }
                send(&maps.out[kMode == kDw ? o : 0], at, y);
            }
            if (!rows || n * kOutCols + (half * kBoxes + kBoxes - 1) * 64 >= p.cols) {
                tc::fence_before();
                __syncwarp();
                if (lane == 0) tc::mbar_arrive_cluster(drained[b]);
            }
        }
        if (lane == 0) tc::bulk_wait();
    }
    if (failed && lane == 0) atomicExch(p.err, 1);
    tc::fence_before();
    __syncthreads();
    tc::cluster_sync();                      // neither CTA's memory goes while the other may still reach it
    if (warp == 1) {
        tc::fence_after();
        tc::tmem_dealloc2(tbase, 512);
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
    static std::atomic<uint64_t> done{0};
    int rc = enc_allow_smem(ffn_mma<T, kMode>, kFSmem, done);
    if (rc) return rc;
    const int out_cols = kMode == kGated ? kFN / 2 : kFN;
    const int64_t tiles = ceil_div(p.rows, kFM) * ceil_div(p.cols, out_cols) * (kMode == kDw ? 2 : 1);
    if (tiles > 0x3FFFFFFF) return fail(RAGRT_ERR_CAPACITY, "too many tiles");
    return enc_launch(ffn_mma<T, kMode>, dim3((unsigned)(2 * std::min<int64_t>(tiles, num_sms() / 2))), dim3(kFThreads),
                      kFSmem, stream, maps, p);
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
    if ((rc = enc_map_2d(&m.a[0], dtype, d_x, M, K, K, kFM / 2)) ||
        (rc = enc_map_2d(&m.b[0], dtype, d_w_gate, F, K, K, kFN / 2)) ||
        (rc = enc_map_2d(&m.b[1], dtype, d_w_up, F, K, K, kFN / 2)) ||
        (rc = enc_map_2d(&m.out[0], dtype, d_h, M, F, F, 32)) ||
        (rc = enc_map_2d(&m.out[1], dtype, d_gate ? d_gate : d_h, M, F, F, 32)) ||
        (rc = enc_map_2d(&m.out[2], dtype, d_up ? d_up : d_h, M, F, F, 32)))
        return rc;
    m.a[1] = m.a[0];
    FfnParams p{M, F, K, act, d_gate != nullptr, err};
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
        if ((rc = enc_map_2d(&m.a[0], dtype, d_dgate, M, F, F, kFM / 2)) ||
            (rc = enc_map_2d(&m.a[1], dtype, d_dup, M, F, F, kFM / 2)) ||
            (rc = enc_map_2d(&m.b[0], dtype, d_w_gate, F, K, K, kFK)) ||
            (rc = enc_map_2d(&m.b[1], dtype, d_w_up, F, K, K, kFK)) ||
            (rc = enc_map_2d(&m.out[0], dtype, d_dx, M, K, K, 32)))
            return rc;
        m.out[1] = m.out[2] = m.out[0];
        FfnParams p{M, K, F, act, 0, err};
        if ((rc = ffn_launch_typed<kDx>(dtype, m, p, stream))) return rc;
    }
    if (d_dw_gate) {
        if ((rc = enc_map_2d(&m.a[0], dtype, d_dgate, M, F, F, kFK)) ||
            (rc = enc_map_2d(&m.a[1], dtype, d_dup, M, F, F, kFK)) ||
            (rc = enc_map_2d(&m.b[0], dtype, d_x, M, K, K, kFK)) ||
            (rc = enc_map_2d(&m.out[0], dtype, d_dw_gate, F, K, K, 32)) ||
            (rc = enc_map_2d(&m.out[1], dtype, d_dw_up, F, K, K, 32)))
            return rc;
        m.b[1] = m.b[0];
        m.out[2] = m.out[1];
        FfnParams p{F, K, M, act, 0, err};
        if ((rc = ffn_launch_typed<kDw>(dtype, m, p, stream))) return rc;
    }
    return RAGRT_OK;
}
