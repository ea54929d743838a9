// enc_ffn.cu -- the gated feed-forward product of a transformer layer and its backward pass.
//
//   forward    g = x Wg^T, u = x Wu^T, h = act(g) * u                 x [M, K], Wg, Wu [F, K]
//   backward   dg = dh * u * act'(g), du = dh * act(g)
//              dx = dg Wg + du Wu, dWg = dg^T x, dWu = du^T x
//
//   ffn_pair<T, kForward>   both projections in one accumulator (half of its columns gate, half up), so that
//                           one pass over x feeds both and the activation and the product are done on
//                           the accumulator.  Keeps g and u for the backward pass when asked to.
//   ffn_pair<T, kBackward>  dx, one product over the 2 F columns of [dg | du] and the rows of [Wg ; Wu] (the
//                           halves add up in the accumulator), and both weight gradients, contracted
//                           over the rows of x: one list of tiles.  Persistent pairs of CTAs
//                           (cta_group::2) on 256 x 256 accumulators, each CTA loading and draining its half.
//   ffn_small<T, ...>       the same on accumulators of 128 x 64, or 128 for the gradients, two single CTAs per
//                           SM: more and shorter tiles where the large ones would leave SMs without work,
//                           and contractions cut into parts where even these are few.
//   ffn_join                those parts' sums, in fp32 and in their order.
//   ffn_rows                forward of up to four rows: a warp per pair of weight rows, fp32 on the CUDA
//                           cores, bound by the weights' bytes.
//   ffn_act_backward        dg and du, elementwise; at memory speed (8192 x 5504: 97 us, 6.5 TB/s).
//
// Measured: 16384 x 2048 -> 8192 forward 688 us in a burst (1,600 TFLOP/s, the tensor pipe at work 98 % of its
// cycles; 805 us, 1,370 TFLOP/s, under the power cap); a training step of 8192 x 2048 -> 5504 236 us forward, 36 more
// for keeping g and u, 645 backward, 99 of them elementwise, the tensor pipe at work 87 % of the rest (cuBLAS for the
// three products alone: 248, 202 and 226 us; one behind the other for longer, at the power cap, 301, 286 and 306, and
// the backward pass here 694).
//
// The weight matrices and x are read as they lie: an operand whose contraction index is the row of
// its matrix is fed to the tensor cores MN-major.  Accumulators are fp32.  g and u are kept in fp32: in 16
// bits their rounding would add as much to the gradients' error as the results' own does (bf16: 3.1e-3 of
// the gradients' norm instead of 2.4e-3, for 360 MB less to move in a step of 8192 x 2048 -> 5504).  dg and du
// are rounded where they become operands, results at the end.
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
// Chunks of a contraction at most: at a microsecond each, far more than any takes, half of what a wait allows.
constexpr int64_t kFLongest = 1 << 20;

enum FfnMode : int { kForward = 0, kBackward = 1 };
enum FfnAct : int { kSilu = 0, kGelu = 1, kGeluTanh = 2 };

struct FfnMaps {
    // kForward: a[0] = x, b[0], b[1] = Wg, Wu, out = h, g, u
    // kBackward: dx: a[0], a[1] = dg, du, b[0], b[1] = Wg, Wu, out[0] = dx
    //            dWg, dWu: a[2], a[3] = dg, du, b[2] = x, out[1], out[2]
    CUtensorMap a[4], b[3], out[3];
};

struct FfnParams {
    int M, F, K;
    int act;
    int keep;                  // kForward: g and u are written too
    int dx, dw;                // kBackward: which gradients
    int a_rows;                // ffn_small: rows of x, dg, du that a load brings
    int split, split_dw;       // ffn_small: parts of dx's and the weight gradients' contraction, each an entry
    float4* partial;           // their sums, [entry][quad of columns][row], what a warp's stores fill whole
    void* out[3];              // as in FfnMaps
    int* err;
};

// A tile of one of the products: output `out` (0, or 1 and 2 for the weight gradients), its rows x cols,
// the tile's first row and column, the length of the contraction in chunks of kFK (dx: of each half), and
// the chunks [i0, i1) to take (dx: those of du and Wu follow those of dg and Wg).
struct FfnTile {
    int out, rows, cols, m0, n0, chunks, i0, i1;
};

// Tile t of the list: dx first, the longest contraction, then dWg, dWu.  Within an output eight tile
// rows at a time, so that the tiles in flight together read few distinct rows and columns.
template <int kMode, int kTileM, int kTileN>
struct FfnList {
    int tn, first, per, total;               // tiles of dx (or h) per tile row, of dx, of dWg, in all
    __device__ __forceinline__ FfnList(const FfnParams& p) {
        const int cols = kMode == kForward ? p.F : p.K;
        tn = (cols + kTileN - 1) / kTileN;
        first = kMode == kForward || p.dx ? tn * ((p.M + kTileM - 1) / kTileM) * p.split : 0;
        per = kMode == kBackward && p.dw ? tn * ((p.F + kTileM - 1) / kTileM) * p.split_dw : 0;
        total = first + 2 * per;
    }
    __device__ __forceinline__ FfnTile get(const FfnParams& p, int t) const {
        FfnTile r;
        const bool dw = t >= first;
        r.out = 0;
        if (dw) {
            t -= first;
            r.out = 1 + (t >= per);
            if (t >= per) t -= per;
        }
        r.rows = dw ? p.F : p.M;
        r.cols = kMode == kForward ? p.F : p.K;
        r.chunks = ((kMode == kForward ? p.K : dw ? p.M : p.F) + kFK - 1) / kFK;
        const int nk = kMode == kBackward && !dw ? 2 * r.chunks : r.chunks;
        r.i0 = 0;
        r.i1 = nk;
        const int split = dw ? p.split_dw : p.split;
        if (kMode == kBackward && split > 1) {
            const int part = t % split;
            t /= split;
            r.i0 = (int)((int64_t)nk * part / split);
            r.i1 = (int)((int64_t)nk * (part + 1) / split);
        }
        const int tm = (r.rows + kTileM - 1) / kTileM;
        const int band = t / (8 * tn), in = t % (8 * tn), high = min(8, tm - 8 * band);
        r.m0 = (8 * band + in % high) * kTileM;
        r.n0 = in / high * kTileN;
        return r;
    }
};

__device__ __forceinline__ float sigmoid(float x) { return __fdividef(1.0f, 1.0f + __expf(-x)); }

// act(x); gelu's tanh form is x * sigmoid(2 u)
__device__ __forceinline__ float ffn_act(float x, int act) {
    if (act == kSilu) return x * sigmoid(x);
    if (act == kGelu) return gelu_erf(x);
    return x * sigmoid(1.5957691216057308f * (x + 0.044715f * x * x * x));
}
// f = act(f) * v
__device__ __forceinline__ void ffn_gate(float (&f)[32], const float (&v)[32], int act) {
    if (act == kSilu) {
#pragma unroll
        for (int e = 0; e < 32; ++e) f[e] = ffn_act(f[e], kSilu) * v[e];
    } else if (act == kGelu) {
#pragma unroll
        for (int e = 0; e < 32; ++e) f[e] = ffn_act(f[e], kGelu) * v[e];
    } else {
#pragma unroll
        for (int e = 0; e < 32; ++e) f[e] = ffn_act(f[e], kGeluTanh) * v[e];
    }
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
        const float y = fminf(fabsf(x), 1e4f);       // the square of more could be infinite, where 1 - s or s is 0
        d = s + x * s * (1.0f - s) * (1.5957691216057308f * (1.0f + 0.134145f * y * y));
    }
}

template <typename T, int kMode>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kFThreads, 1)
ffn_pair(const __grid_constant__ FfnMaps maps, const __grid_constant__ FfnParams p) {
    constexpr int kOutCols = kMode == kForward ? kFN / 2 : kFN;
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
    const FfnList<kMode, kFM, kOutCols> list(p);
    // The tiles are dealt out in turn, those of the last round, which does not reach all pairs, from the last pair on:
    // the first ones hold one tile of dx more, and those are longer.
    const int last = list.total / pairs * pairs;
    auto after = [&](int t) { return t + pairs < last ? t + pairs : t < last ? last + pairs - 1 - pair : list.total; };

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
            for (int t = pair; t < list.total && !failed; t = after(t)) {
                const FfnTile tile = list.get(p, t);
                const bool dw = kMode == kBackward && tile.out > 0;
                const int m0 = tile.m0 + rank * (kFM / 2);
                const int n0 = tile.n0 + (kMode == kForward ? 0 : rank * (kFN / 2));
                for (int i = tile.i0; i < tile.i1; ++i, ++g) {
                    const int s = g % kFStages;
                    if (g >= kFStages && !tc::mbar_wait_or_abort(empty + s, ((g / kFStages) - 1) & 1, abort, kFWaitLimit)) {
                        failed = true;
                        break;
                    }
                    const bool second = i >= tile.chunks;        // dx: the half of du and Wu
                    const int k = (second ? i - tile.chunks : i) * kFK;
                    uint8_t* da = sA + s * kFTileA;
                    uint8_t* db = sB + s * kFTileB;
                    const uint32_t bar = tc::cluster_addr(full + s, 0);
                    if (rank == 0) tc::mbar_arrive_expect_tx(full + s, 2 * (kFTileA + kFTileB));
                    if (dw) {
#pragma unroll
                        for (int j = 0; j < kFM / 128; ++j)
                            tc::tma_load_2d_pair(da + j * 8192, &maps.a[1 + tile.out], m0 + 64 * j, k, bar);
                    } else {
                        tc::tma_load_2d_pair(da, &maps.a[second], k, m0, bar);
                    }
                    if (kMode == kForward) {         // rank 0: the gate's half of the columns, rank 1: the other
                        tc::tma_load_2d_pair(db, &maps.b[rank], k, n0, bar);
                    } else {
#pragma unroll
                        for (int j = 0; j < kFN / 128; ++j)
                            tc::tma_load_2d_pair(db + j * 8192, &maps.b[dw ? 2 : (int)second], n0 + 64 * j, k, bar);
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
            const uint32_t lead = tc::elect_one();
            int g = 0, j = 0;
            for (int t = pair; t < list.total && !failed; t = after(t), ++j) {
                const FfnTile tile = list.get(p, t);
                const bool dw = kMode == kBackward && tile.out > 0;
                const uint32_t idesc = tc::idesc_f16_f32(kFM, kFN) | idesc_type<T>() | (dw ? kIdescAMn : 0u) |
                                       (kMode == kBackward ? kIdescBMn : 0u);
                const uint32_t step = dw ? 2048 : 32;
                const int b = j & 1;
                bool ok = j < 2 || tc::mbar_wait_or_abort(acce + b, ((j >> 1) - 1) & 1, abort, kFWaitLimit);
                failed = !__all_sync(0xFFFFFFFFu, ok);
                if (failed) break;
                tc::fence_after();
                const uint32_t d = tbase + (uint32_t)(b * kFN);
                for (int i = tile.i0; i < tile.i1; ++i, ++g) {
                    const int s = g % kFStages;
                    ok = tc::mbar_wait_or_abort(full + s, (g / kFStages) & 1, abort, kFWaitLimit);
                    failed = !__all_sync(0xFFFFFFFFu, ok);
                    if (failed) break;
                    tc::fence_after();
                    // the leading byte offset, which only an MN-major operand has, is there for both
                    const uint32_t a = tc::smem_u32(sA + s * kFTileA), bb = tc::smem_u32(sB + s * kFTileB);
#pragma unroll
                    for (int k = 0; k < kFK / 16; ++k)
                        tc::mma_ss2_if(lead, d, tc::sw128_mnmajor_desc(a + step * k, 8192),
                                       kMode == kBackward ? tc::sw128_mnmajor_desc(bb + 2048 * k, 8192)
                                                          : tc::sw128_kmajor_desc(bb + 32 * k),
                                       idesc, i != tile.i0 || k != 0 ? 1u : 0u);
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
        for (int t = pair; t < list.total; t = after(t), ++j) {
            const FfnTile tile = list.get(p, t);
            const int b = j & 1;
            const int y = tile.m0 + rank * (kFM / 2) + quad * 32;
            const bool ok = tc::mbar_wait_or_abort(accf + b, (j >> 1) & 1, abort, kFWaitLimit);
            if (!__all_sync(0xFFFFFFFFu, ok)) {
                failed = true;
                break;
            }
            tc::fence_after();
            const uint32_t taddr = tbase + ((uint32_t)(quad * 32) << 16) + (uint32_t)(b * kFN);
            const bool rows = y < tile.rows;        // of this warp
#pragma unroll 1
            for (int x = 0; x < kBoxes; ++x) {
                const int c0 = (half * kBoxes + x) * 64, at = tile.n0 + c0;
                if (!rows || at >= tile.cols) break;
                if (kMode == kForward && p.keep) {
#pragma unroll 1
                    for (int w = 0; w < 4; ++w) {       // g and u, 32 columns at a time
                        float f[32];
                        tc::ld32x32(taddr + (w >> 1) * (kFN / 2) + c0 + 32 * (w & 1), *reinterpret_cast<uint32_t(*)[32]>(f));
                        tc::wait_ld();
#pragma unroll
                        for (int q = 0; q < 32; q += 4)
                            *reinterpret_cast<float4*>(out + lane * 128 + (((q / 4) ^ (lane & 7)) << 4)) =
                                make_float4(f[q], f[q + 1], f[q + 2], f[q + 3]);
                        if (at + 32 * (w & 1) < tile.cols) send(&maps.out[1 + (w >> 1)], at + 32 * (w & 1), y);
                    }
                }
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    float f[32];
                    tc::ld32x32(taddr + c0 + 32 * c, *reinterpret_cast<uint32_t(*)[32]>(f));
                    if (kMode == kForward) {
                        float v[32];
                        tc::ld32x32(taddr + kFN / 2 + c0 + 32 * c, *reinterpret_cast<uint32_t(*)[32]>(v));
                        tc::wait_ld();
                        ffn_gate(f, v, p.act);
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
                send(&maps.out[kMode == kForward ? 0 : tile.out], at, y);
            }
            if (!rows || tile.n0 + (half * kBoxes + kBoxes - 1) * 64 >= tile.cols) {
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

// ------------------------------------------------------------------ 128-row tiles of one CTA, two to an SM
constexpr int kSTileA = kFM / 2 * kFK * 2;
template <int kMode, int kN_>
struct SmallCfg {
    static constexpr int kN = kN_;                               // accumulator columns
    static constexpr int kOutCols = kMode == kForward ? kN / 2 : kN;
    static constexpr int kTileB = kN * kFK * 2;
    static constexpr int kStages = kN == 64 ? 4 : 3;
    static constexpr int kSmem = 1024 + kStages * (kSTileA + kTileB) + 256;
};
constexpr int kFewRows = 4;                    // rows that ffn_rows takes at most
constexpr int kSThreads = 192;                 // TMA warp, MMA warp, 4 epilogue warps

template <typename T, int kMode, int kN>
__global__ void __launch_bounds__(kSThreads, 2)
ffn_small(const __grid_constant__ FfnMaps maps, const __grid_constant__ FfnParams p) {
    typedef SmallCfg<kMode, kN> Cfg;
    constexpr int kOutCols = Cfg::kOutCols, kSStages = Cfg::kStages, kSTileB = Cfg::kTileB;
    extern __shared__ uint8_t ffn_raw[];
    uint8_t* sm = (uint8_t*)(((uintptr_t)ffn_raw + 1023) & ~(uintptr_t)1023);
    uint8_t* sA = sm;
    uint8_t* sB = sm + kSStages * kSTileA;
    uint64_t* full = reinterpret_cast<uint64_t*>(sB + kSStages * kSTileB);
    uint64_t* empty = full + kSStages;
    uint64_t* accf = empty + kSStages;
    uint64_t* acce = accf + 2;
    uint64_t* drain = acce + 2;
    uint32_t* tslot = reinterpret_cast<uint32_t*>(drain + 1);
    volatile int* abort = reinterpret_cast<volatile int*>(tslot + 1);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const FfnList<kMode, kFM / 2, kOutCols> list(p);
    if (threadIdx.x == 0) {
        for (int s = 0; s < kSStages; ++s) {
            tc::mbar_init(full + s, 1);
            tc::mbar_init(empty + s, 1);
        }
        for (int b = 0; b < 2; ++b) {
            tc::mbar_init(accf + b, 1);
            tc::mbar_init(acce + b, 4);
        }
        tc::mbar_init(drain, 1);
        *abort = 0;
        tc::mbar_fence_init();
    }
    if (warp == 1) {
        tc::tmem_alloc(tslot, 2 * kN);
        tc::tmem_relinquish();
    }
    tc::fence_before();
    __syncthreads();
    tc::fence_after();
    const uint32_t tbase = *tslot;
    bool failed = false;
    pdl_wait_then_release();

    if (warp == 0) {
        if (lane == 0) {
            int g = 0;
            for (int t = blockIdx.x; t < list.total && !failed; t += gridDim.x) {
                const FfnTile tile = list.get(p, t);
                const bool dw = kMode == kBackward && tile.out > 0;
                for (int i = tile.i0; i < tile.i1; ++i, ++g) {
                    const int s = g % kSStages;
                    if (g >= kSStages && !tc::mbar_wait_or_abort(empty + s, ((g / kSStages) - 1) & 1, abort, kFWaitLimit)) {
                        failed = true;
                        break;
                    }
                    const bool second = i >= tile.chunks;
                    const int k = (second ? i - tile.chunks : i) * kFK;
                    uint8_t* da = sA + s * kSTileA;
                    uint8_t* db = sB + s * kSTileB;
                    tc::mbar_arrive_expect_tx(full + s, (dw ? kSTileA : p.a_rows * kFK * 2) + kSTileB);
                    if (dw) {
                        tc::tma_load_2d(da, &maps.a[1 + tile.out], tile.m0, k, full + s);
                        tc::tma_load_2d(da + 8192, &maps.a[1 + tile.out], tile.m0 + 64, k, full + s);
                    } else {
                        tc::tma_load_2d(da, &maps.a[second], k, tile.m0, full + s);
                    }
                    if (kMode == kForward) {
                        tc::tma_load_2d(db, &maps.b[0], k, tile.n0, full + s);
                        tc::tma_load_2d(db + kSTileB / 2, &maps.b[1], k, tile.n0, full + s);
                    } else {
                        for (int c = 0; c < kN / 64; ++c)
                            tc::tma_load_2d(db + 8192 * c, &maps.b[dw ? 2 : (int)second], tile.n0 + 64 * c, k, full + s);
                    }
                }
            }
            if (failed)                      // copies in flight end before the CTA does
                for (int i = max(0, g - kSStages); i < g; ++i)
                    (void)tc::mbar_wait_bounded(full + i % kSStages, (i / kSStages) & 1, 1u << 16);
        }
    } else if (warp == 1) {
        const uint32_t lead = tc::elect_one();
        int g = 0, j = 0;
        for (int t = blockIdx.x; t < list.total && !failed; t += gridDim.x, ++j) {
            const FfnTile tile = list.get(p, t);
            const bool dw = kMode == kBackward && tile.out > 0;
            const uint32_t idesc = tc::idesc_f16_f32(kFM / 2, kN) | idesc_type<T>() | (dw ? kIdescAMn : 0u) |
                                   (kMode == kBackward ? kIdescBMn : 0u);
            const uint32_t step = dw ? 2048 : 32;
            const int b = j & 1;
            bool ok = j < 2 || tc::mbar_wait_or_abort(acce + b, ((j >> 1) - 1) & 1, abort, kFWaitLimit);
            failed = !__all_sync(0xFFFFFFFFu, ok);
            if (failed) break;
            tc::fence_after();
            for (int i = tile.i0; i < tile.i1; ++i, ++g) {
                const int s = g % kSStages;
                ok = tc::mbar_wait_or_abort(full + s, (g / kSStages) & 1, abort, kFWaitLimit);
                failed = !__all_sync(0xFFFFFFFFu, ok);
                if (failed) break;
                tc::fence_after();
                const uint32_t a = tc::smem_u32(sA + s * kSTileA), bb = tc::smem_u32(sB + s * kSTileB);
#pragma unroll
                for (int k = 0; k < kFK / 16; ++k)
                    tc::mma_ss_if(lead, tbase + (uint32_t)(b * kN), tc::sw128_mnmajor_desc(a + step * k, 8192),
                                  kMode == kBackward ? tc::sw128_mnmajor_desc(bb + 2048 * k, 8192)
                                                     : tc::sw128_kmajor_desc(bb + 32 * k),
                                  idesc, i != tile.i0 || k != 0 ? 1u : 0u);
                tc::mma_commit_if(lead, empty + s);
            }
            if (!failed) tc::mma_commit_if(lead, accf + b);
        }
        if (failed) {                        // the last products read shared memory: let them finish
            tc::mma_commit_if(lead, drain);
            (void)tc::mbar_wait_bounded(drain, 0, 1u << 16);
        }
    } else {
        const int quad = warp & 3;
        int j = 0;
        for (int t = blockIdx.x; t < list.total; t += gridDim.x, ++j) {
            const FfnTile tile = list.get(p, t);
            const int b = j & 1, row = tile.m0 + quad * 32 + lane;
            const bool ok = tc::mbar_wait_or_abort(accf + b, (j >> 1) & 1, abort, kFWaitLimit);
            if (!__all_sync(0xFFFFFFFFu, ok)) {
                failed = true;
                break;
            }
            tc::fence_after();
            const uint32_t taddr = tbase + ((uint32_t)(quad * 32) << 16) + (uint32_t)(b * kN);
#pragma unroll 1
            for (int c0 = 0; c0 < kN; c0 += 64) {
                float f[32], v[32];
                tc::ld32x32(taddr + c0, *reinterpret_cast<uint32_t(*)[32]>(f));
                tc::ld32x32(taddr + c0 + 32, *reinterpret_cast<uint32_t(*)[32]>(v));
                tc::wait_ld();
                if (c0 + 64 == kN) {
                    tc::fence_before();
                    __syncwarp();
                    if (lane == 0) tc::mbar_arrive(acce + b);
                }
                if (kMode == kBackward && (tile.out == 0 ? p.split : p.split_dw) > 1) {
                    const int entry = p.split > 1 ? t : t - list.first;
                    float4* to = p.partial + ((int64_t)entry * (kN / 4) + c0 / 4) * (kFM / 2) + quad * 32 + lane;
#pragma unroll
                    for (int q = 0; q < 8; ++q) {
                        to[q * (kFM / 2)] = make_float4(f[4 * q], f[4 * q + 1], f[4 * q + 2], f[4 * q + 3]);
                        to[(8 + q) * (kFM / 2)] = make_float4(v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]);
                    }
                } else if (row < tile.rows) {
                    const int64_t at = (int64_t)row * tile.cols + tile.n0;
                    auto put = [&](void* base, int off, const float (&x)[32]) {
                        T* dst = static_cast<T*>(base) + at + off;
                        if (tile.cols % 16 == 0 && ((uintptr_t)base & 31) == 0) {       // whole sectors
#pragma unroll
                            for (int q = 0; q < 32; q += 16)
                                if (tile.n0 + off + q < tile.cols)
                                    store32(dst + q, down8<T>(*reinterpret_cast<const float(*)[8]>(x + q)),
                                            down8<T>(*reinterpret_cast<const float(*)[8]>(x + q + 8)));
                        } else {
#pragma unroll
                            for (int q = 0; q < 32; q += 8)
                                if (tile.n0 + off + q < tile.cols)       // cols is a multiple of 8
                                    *reinterpret_cast<uint4*>(dst + q) =
                                        down8<T>(*reinterpret_cast<const float(*)[8]>(x + q));
                        }
                    };
                    auto keep = [&](void* base, const float (&x)[32]) {
#pragma unroll
                        for (int q = 0; q < 32; q += 4)
                            if (tile.n0 + q < tile.cols)
                                *reinterpret_cast<float4*>(static_cast<float*>(base) + at + q) =
                                    make_float4(x[q], x[q + 1], x[q + 2], x[q + 3]);
                    };
                    if (kMode == kForward) {
                        if (p.keep) {
                            keep(p.out[1], f);
                            keep(p.out[2], v);
                        }
                        ffn_gate(f, v, p.act);
                        put(p.out[0], 0, f);
                    } else {
                        put(p.out[tile.out], c0, f);
                        put(p.out[tile.out], c0 + 32, v);
                    }
                }
            }
        }
    }
    if (failed && lane == 0) atomicExch(p.err, 1);
    tc::fence_before();
    __syncthreads();
    if (warp == 1) {
        tc::fence_after();
        tc::tmem_dealloc(tbase, 2 * kN);
    }
}

// Gradients from their parts' sums, in the parts' order; a thread per 8 values, the tiles of what is not split left out.
template <typename T, int kN>
__global__ void __launch_bounds__(256) ffn_join(const __grid_constant__ FfnParams p) {
    pdl_wait_then_release();
    const int i = blockIdx.x * 256 + threadIdx.x;
    const int r = i % (kFM / 2), c = i / (kFM / 2) % (kN / 8) * 8;
    FfnParams whole = p;
    if (p.split == 1) whole.dx = 0;
    if (p.split_dw == 1) whole.dw = 0;
    whole.split = whole.split_dw = 1;
    const FfnList<kBackward, kFM / 2, kN> list(whole);
    const int t = i / (kFM / 2 * kN / 8);
    if (t >= list.total) return;
    const FfnTile tile = list.get(whole, t);
    const int row = tile.m0 + r, col = tile.n0 + c;
    if (row >= tile.rows || col >= tile.cols) return;
    const int parts = tile.out == 0 ? p.split : p.split_dw;
    const int entry = tile.out == 0 ? t * p.split : list.first * p.split + (t - list.first) * p.split_dw;
    float sum[8] = {};
    const float4* from = p.partial + (int64_t)entry * (kN / 4 * kFM / 2) + c / 4 * (kFM / 2) + r;
#pragma unroll 4
    for (int s = 0; s < parts; ++s, from += kN / 4 * kFM / 2) {
        const float4 a = __ldcs(from), b = __ldcs(from + kFM / 2);
        sum[0] += a.x; sum[1] += a.y; sum[2] += a.z; sum[3] += a.w;
        sum[4] += b.x; sum[5] += b.y; sum[6] += b.z; sum[7] += b.w;
    }
    *reinterpret_cast<uint4*>(static_cast<T*>(p.out[tile.out]) + (int64_t)row * tile.cols + col) = down8<T>(sum);
}

// ------------------------------------------------------------------ few rows
// A warp per kCols output columns: it reads their rows of Wg and Wu, 8 values a lane and step, against the
// same values of up to kRows rows of x.
template <typename T, int kRows, int kCols>
__global__ void __launch_bounds__(256) ffn_rows(const T* __restrict__ x, const T* __restrict__ wg,
                                                const T* __restrict__ wu, const __grid_constant__ FfnParams p) {
    const int f0 = (int)(blockIdx.x * 8 + (threadIdx.x >> 5)) * kCols, lane = threadIdx.x & 31;
    pdl_wait_then_release();
    if (f0 >= p.F) return;                           // F is a multiple of 8
    const T* w[2] = {wg + (int64_t)f0 * p.K, wu + (int64_t)f0 * p.K};
    uint64_t sum[kRows][2][kCols] = {};
    const uint4 zero = make_uint4(0u, 0u, 0u, 0u);
    constexpr int kAhead = 4 / kCols;                // steps whose weights are in flight together
    for (int k0 = lane * 8; k0 < p.K + lane * 8; k0 += 256 * kAhead) {
        uint4 a[kAhead][2][kCols], xr[kAhead][kRows];
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            const bool in = k0 + 256 * i < p.K;
#pragma unroll
            for (int m = 0; m < 2; ++m)
#pragma unroll
                for (int c = 0; c < kCols; ++c)
                    a[i][m][c] = in ? __ldg(reinterpret_cast<const uint4*>(w[m] + (int64_t)c * p.K + k0 + 256 * i)) : zero;
#pragma unroll
            for (int r = 0; r < kRows; ++r)
                xr[i][r] = in && r < p.M ? __ldg(reinterpret_cast<const uint4*>(x + (int64_t)r * p.K + k0 + 256 * i)) : zero;
        }
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            if (k0 + 256 * i >= p.K) break;          // a row of x behind M adds nothing, weights of no value could
            float fx[kRows][8];
#pragma unroll
            for (int r = 0; r < kRows; ++r) up8<T>(xr[i][r], fx[r]);
#pragma unroll
            for (int m = 0; m < 2; ++m)
#pragma unroll
                for (int c = 0; c < kCols; ++c) {
                    float fw[8];
                    up8<T>(a[i][m][c], fw);
#pragma unroll
                    for (int r = 0; r < kRows; ++r)
#pragma unroll
                        for (int e = 0; e < 8; e += 2)
                            sum[r][m][c] = fma2(pack2(fw[e], fw[e + 1]), pack2(fx[r][e], fx[r][e + 1]), sum[r][m][c]);
                }
        }
    }
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
        if (r >= p.M) break;
#pragma unroll
        for (int c = 0; c < kCols; ++c) {
            float v[2];
#pragma unroll
            for (int m = 0; m < 2; ++m) {
                float a, b;
                unpack2(sum[r][m][c], a, b);
                v[m] = a + b;
#pragma unroll
                for (int o = 16; o; o >>= 1) v[m] += __shfl_xor_sync(0xFFFFFFFFu, v[m], o);
            }
            if (lane == 0) {
                const int64_t at = (int64_t)r * p.F + f0 + c;
                if (p.keep) {
                    static_cast<float*>(p.out[1])[at] = v[0];
                    static_cast<float*>(p.out[2])[at] = v[1];
                }
                static_cast<T*>(p.out[0])[at] = (T)(ffn_act(v[0], p.act) * v[1]);
            }
        }
    }
}

template <typename T>
int ffn_rows_launch(const void* x, const void* wg, const void* wu, const FfnParams& p, cudaStream_t stream) {
    if (p.M == 1)
        return enc_launch(ffn_rows<T, 1, 1>, dim3((unsigned)ceil_div(p.F, 8)), dim3(256), 0, stream, (const T*)x,
                          (const T*)wg, (const T*)wu, p);
    return enc_launch(ffn_rows<T, kFewRows, 2>, dim3((unsigned)ceil_div(p.F, 16)), dim3(256), 0, stream, (const T*)x,
                      (const T*)wg, (const T*)wu, p);
}

// dg = dh * u * act'(g), du = dh * act(g); a thread per 8 values
template <typename T>
__global__ void __launch_bounds__(256) ffn_act_backward(const T* __restrict__ dh, const float* __restrict__ gate,
                                                        const float* __restrict__ up, T* __restrict__ dg,
                                                        T* __restrict__ du, int64_t n8, int act) {
    pdl_wait_then_release();
    for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < n8; i += (int64_t)gridDim.x * blockDim.x) {
        float d[8], g[8], u[8], x[8], y[8];
        up8<T>(reinterpret_cast<const uint4*>(dh)[i], d);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            *reinterpret_cast<float4*>(g + 4 * h) = __ldcs(reinterpret_cast<const float4*>(gate) + 2 * i + h);
            *reinterpret_cast<float4*>(u + 4 * h) = __ldcs(reinterpret_cast<const float4*>(up) + 2 * i + h);
        }
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

// The operands' maps differ in their boxes between the two kernels.
int ffn_maps(FfnMaps& m, int mode, bool pair, int dtype, const FfnParams& p, const void* x, const void* wg, const void* wu,
             const void* dg, const void* du) {
    int rc;
    if (mode == kForward) {
        const int wrows = pair ? kFN / 2 : SmallCfg<kForward, 64>::kOutCols;
        if ((rc = enc_map_2d(&m.a[0], dtype, x, p.M, p.K, p.K, pair ? kFM / 2 : p.a_rows)) ||
            (rc = enc_map_2d(&m.b[0], dtype, wg, p.F, p.K, p.K, wrows)) ||
            (rc = enc_map_2d(&m.b[1], dtype, wu, p.F, p.K, p.K, wrows)))
            return rc;
        if (pair && ((rc = enc_map_2d(&m.out[0], dtype, p.out[0], p.M, p.F, p.F, 32)) ||
                     (p.keep && ((rc = enc_map_f32(&m.out[1], p.out[1], p.M, p.F)) ||
                                 (rc = enc_map_f32(&m.out[2], p.out[2], p.M, p.F))))))
            return rc;
        return RAGRT_OK;
    }
    if (p.dx && ((rc = enc_map_2d(&m.a[0], dtype, dg, p.M, p.F, p.F, pair ? kFM / 2 : p.a_rows)) ||
                 (rc = enc_map_2d(&m.a[1], dtype, du, p.M, p.F, p.F, pair ? kFM / 2 : p.a_rows)) ||
                 (rc = enc_map_2d(&m.b[0], dtype, wg, p.F, p.K, p.K, kFK)) ||
                 (rc = enc_map_2d(&m.b[1], dtype, wu, p.F, p.K, p.K, kFK)) ||
                 (pair && (rc = enc_map_2d(&m.out[0], dtype, p.out[0], p.M, p.K, p.K, 32)))))
        return rc;
    if (p.dw && ((rc = enc_map_2d(&m.a[2], dtype, dg, p.M, p.F, p.F, kFK)) ||
                 (rc = enc_map_2d(&m.a[3], dtype, du, p.M, p.F, p.F, kFK)) ||
                 (rc = enc_map_2d(&m.b[2], dtype, x, p.M, p.K, p.K, kFK)) ||
                 (pair && ((rc = enc_map_2d(&m.out[1], dtype, p.out[1], p.F, p.K, p.K, 32)) ||
                           (rc = enc_map_2d(&m.out[2], dtype, p.out[2], p.F, p.K, p.K, 32))))))
        return rc;
    return RAGRT_OK;
}

int64_t ffn_tiles(int mode, const FfnParams& p, int tile_m, int tile_n) {
    if (mode == kForward) return ceil_div(p.M, tile_m) * ceil_div(p.F, tile_n);
    return ((p.dx ? ceil_div(p.M, tile_m) : 0) + (p.dw ? 2 * ceil_div(p.F, tile_m) : 0)) * ceil_div(p.K, tile_n);
}

// How the gradients run on 128-row tiles: their width, the parts that the contraction of dx and of the weight gradients
// is cut into (1: whole), and whether dx has a launch of its own (apart).
struct FfnPlan {
    int width, split, split_dw;
    bool apart;
};

int64_t ffn_dx_tiles(int M, int K, int width) { return ceil_div(M, kFM / 2) * ceil_div(K, width); }
int64_t ffn_dw_tiles(int F, int K, int width) { return 2 * ceil_div(F, kFM / 2) * ceil_div(K, width); }
int64_t ffn_part_bytes(int width) { return (int64_t)(kFM / 2) * width * 4; }

// The parts of least time, as the longest share of a CTA in chunks of the contraction: dx's parts and then `per` tiles
// of of_dw chunks, dealt out to two CTAs per SM in turn.  A tile of the weight gradients takes 16 chunks at least, its
// epilogue; a part 4 more; every entry of the list costs the SM 2; the joining kernel 8 and one per 64 parts.  Parts of
// 8 chunks or more, at most two per SM in all (and 16 of a tile).  Against all counts, measured for 20 shapes from 25 x
// 768 -> 2048 to 256 x 4096 -> 8192 with the same inputs again and again (in L2, but for the largest): within 5 % of
// the best for dx, 13 % for all gradients.
int ffn_parts(int tiles, int nk, int per, int of_dw) {
    const int sms = num_sms(), ctas = 2 * sms;
    int best = 1, least = 0;
    for (int s = 1; s <= 16 && (s == 1 || (s <= nk / 8 && s * tiles <= ctas)); ++s) {
        // a CTA's first entry is one of dx, its own number if it has one; then come the others in turn
        const int parts = tiles * s, part = (nk + s - 1) / s + 4;
        auto share = [&](int c) {
            const int n = (std::max(parts + per - c, 0) + ctas - 1) / ctas, dx = c < parts ? 1 : 0;
            return dx * part + (n - dx) * std::max(of_dw, 16);
        };
        const int time = std::max(share(0), share(parts % ctas)) + (s > 1 ? 8 + parts / 64 : 0) + 2 * (parts + per) / sms;
        if (s == 1 || time < least) {
            best = s;
            least = time;
        }
    }
    return best;
}

// Whether the weight gradients' contraction, over the rows, is cut: where many rows meet small matrices, so that even
// the 128 x 128 tiles are no more than the SMs.  An SM takes 0.41 us for a chunk of those, a pair as long for one of 256 x
// 256 (so twice the rate); the former are spread evenly by the cut and pay 8 us for it, the latter's longest share counts.
// All gradients whole and cut, inputs from memory: 16000 rows 256 -> 256 94 and 30 us, 16384 rows 384 -> 1536 190 and
// 150, 4000 rows 512 -> 512 32 and 25; not cut by this rule: 8192 rows 512 -> 2048 129, 3000 rows 512 -> 1024 30.
bool ffn_cut_dw(int M, int F, int K, bool dx) {
    const int64_t sms = num_sms(), pairs = sms / 2, nk = 2 * ceil_div(F, kFK), of_dw = ceil_div(M, kFK);
    const int64_t per = ffn_dw_tiles(F, K, 128);
    if (per > sms || of_dw < 32) return false;
    const int64_t n_dx = dx ? ceil_div(M, kFM) * ceil_div(K, kFN) : 0, n_dw = 2 * ceil_div(F, kFM) * ceil_div(K, kFN);
    auto share = [&](int64_t c) {
        const int64_t n = ceil_div(std::max<int64_t>(n_dx + n_dw - c, 0), pairs);
        const int64_t d = ceil_div(std::max<int64_t>(n_dx - c, 0), pairs);
        return d * nk + (n - d) * of_dw;
    };
    const int64_t large = std::max(share(0), share(n_dx % pairs));
    const int64_t small = ((dx ? ffn_dx_tiles(M, K, 128) * nk : 0) + per * of_dw) / sms + 20;
    return 10 * small < 9 * large;
}

// dx is cut where it has fewer tiles than there are SMs: its time is that of the 2 F steps of one tile then, 0.3 us
// a chunk.  Not under 32 chunks (60 rows 512 -> 512 in two parts 10.1 us, whole 8.2).  The weight gradients join its
// launch while they are 27 chunks per SM or fewer; else dx runs apart if its chain shrinks by 64 chunks, or is left
// whole (1500 rows 768 -> 2048: large tiles for all 36 us, dx apart 40).  With their elementwise kernel, inputs from
// memory, whole and in parts, dx / all gradients: 25 rows 768 -> 2048 24 / 26 and 10.9 / 14.4 us, 128 rows 2048 -> 5504
// 59 / 72 and 21 / 35, 300 rows 65 / 78 and 32 / 55, 25 rows 4096 -> 8192 87 / 123 and 34 / 76, 1000 rows 768 -> 2048
// 29 / 33 and 23 / 30 (cuBLAS's dx, operands in L2: 9.3, 17, 18.5, 26, 10.7; here then 9.5, 17, 30, 33, 20).
// Tiles of 64 columns where those are one round of CTAs and 64 chunks per SM; else of 128, whose products take no
// longer (100 cycles: the 128-row operand comes from shared memory at that rate).  In L2: all gradients of 1000 rows 768 ->
// 2048 by 64 27.8 us, by 128 24.4; 128 rows 2048 -> 5504 39.2 and 32.0; 1200 rows 384 -> 1536 17.4 and 18.9; dx alone
// of 25 rows 768 -> 2048 9.9 and 10.4, of 256 rows 4096 -> 8192 60 and 52.
FfnPlan ffn_plan(int M, int F, int K, bool dx, bool dw) {
    const int64_t sms = num_sms(), nk = 2 * ceil_div(F, kFK), of_dw = ceil_div(M, kFK);
    FfnPlan plan{64, 1, 1, false};
    if (dw && ffn_cut_dw(M, F, K, dx)) {
        const int64_t tiles = dx ? ffn_dx_tiles(M, K, 128) : 0, per = ffn_dw_tiles(F, K, 128);
        plan.width = 128;
        plan.split_dw = (int)std::min({(int64_t)16, of_dw / 8, 2 * sms / per});
        if (tiles > 0 && tiles <= sms) plan.split = (int)std::max<int64_t>(1, std::min({(int64_t)16, nk / 16, sms / tiles}));
        return plan;
    }
    for (const int width : {64, 128}) {
        const int64_t tiles = dx ? ffn_dx_tiles(M, K, width) : 0, per = dw ? ffn_dw_tiles(F, K, width) : 0;
        plan = FfnPlan{width, 1, 1, false};
        if (tiles > 0 && tiles <= sms && nk >= 32) {
            plan.apart = dw && per * of_dw * width / 128 > 27 * sms;
            plan.split = ffn_parts((int)tiles, (int)nk, plan.apart ? 0 : (int)per, (int)of_dw);
            if (plan.apart && nk - nk / plan.split < 64) plan.split = 1;
        }
        if (plan.split == 1) plan.apart = false;
        const int64_t rest = plan.apart ? 0 : per;
        if (tiles * plan.split + rest <= 2 * sms && tiles * nk + rest * of_dw <= 64 * sms) break;
    }
    return plan;
}

template <typename T, int kMode, int kN>
int ffn_launch_small(const FfnMaps& m, const FfnParams& p, int64_t entries, cudaStream_t stream) {
    typedef SmallCfg<kMode, kN> Cfg;
    static std::atomic<uint64_t> done{0};
    const int rc = enc_allow_smem(ffn_small<T, kMode, kN>, Cfg::kSmem, done);
    if (rc) return rc;
    return enc_launch(ffn_small<T, kMode, kN>, dim3((unsigned)std::min<int64_t>(entries, 2 * num_sms())),
                      dim3(kSThreads), Cfg::kSmem, stream, m, p);
}

template <typename T, int kMode>
int ffn_launch(int dtype, FfnParams p, int width, const void* x, const void* wg, const void* wu, const void* dg,
               const void* du, cudaStream_t stream) {
    FfnMaps m = {};
    int rc;
    const int64_t sms = num_sms(), pairs = sms / 2;
    const int64_t large = ffn_tiles(kMode, p, kFM, kMode == kForward ? kFN / 2 : kFN);
    int64_t small = ffn_tiles(kMode, p, kFM / 2, kMode == kForward ? width / 2 : width);
    if (p.dx) small += (p.split - 1) * ffn_dx_tiles(p.M, p.K, width);
    if (p.dw) small += (p.split_dw - 1) * ffn_dw_tiles(p.F, p.K, width);
    bool pair;
    if (kMode == kForward) {
        // small tiles while they are one round of two CTAs per SM.  Weights from memory: 128 rows 2048 -> 5504 (172
        // tiles) 15.6 us against 17.6, 512 rows 768 -> 2048 (256) 7.7 against 10.4; 256 rows 2048 -> 5504 (344) 23.9
        // against 18.2, 1000 rows 768 -> 2048 (512) 11.9 against 11.0
        pair = small > 2 * sms;
    } else {
        // small tiles where the large ones' longest contraction is far above their average per pair of SMs
        // (five times).  Calls that got no scratch, inputs in L2: all gradients of 512 rows 768 -> 2048 (6.4 times)
        // 27.4 us against 28.7; 1000 rows (3.1) 30.3 against 31.4, 256 rows 2048 -> 5504 (4.6) 93.9 against 74.2.
        // From memory the large tiles gain: 36.0 against 30.7, 37.6 and 33.5, 95.4 and 74.9.
        const int64_t of_dx = 2 * ceil_div(p.F, kFK), of_dw = ceil_div(p.M, kFK);
        const int64_t n_dx = p.dx ? ceil_div(p.M, kFM) * ceil_div(p.K, kFN) : 0;
        const int64_t sum = n_dx * of_dx + (large - n_dx) * of_dw;
        pair = p.split == 1 && p.split_dw == 1 && 5 * sum >= pairs * std::max(p.dx ? of_dx : 0, p.dw ? of_dw : 0);
    }
    if (std::max(large, small) > 0x3FFFFFFF) return fail(RAGRT_ERR_CAPACITY, "too many tiles");
    const int64_t longest = kMode == kForward ? ceil_div(p.K, kFK)
                                              : std::max(p.dx ? 2 * ceil_div(p.F, kFK) / p.split : 0,
                                                         p.dw ? ceil_div(p.M, kFK) / p.split_dw : 0);
    if (longest > kFLongest)
        return fail(RAGRT_ERR_CAPACITY, "gated_ffn: a sum over %lld values is too long", (long long)longest * kFK);
    // few rows: a load brings no more of them than there are (one row of 2048 -> 5504, weights in L2, 11.2 us; with
    // 128-row boxes, most of them outside the tensor, 30)
    p.a_rows = std::min(kFM / 2, (int)ceil_div(p.M, 8) * 8);
    if ((rc = ffn_maps(m, kMode, pair, dtype, p, x, wg, wu, dg, du))) return rc;
    if (pair) {
        static std::atomic<uint64_t> done{0};
        if ((rc = enc_allow_smem(ffn_pair<T, kMode>, kFSmem, done))) return rc;
        return enc_launch(ffn_pair<T, kMode>, dim3((unsigned)(2 * std::min(large, pairs))), dim3(kFThreads), kFSmem,
                          stream, m, p);
    }
    if constexpr (kMode == kBackward)
        if (width == 128) return ffn_launch_small<T, kMode, 128>(m, p, small, stream);
    return ffn_launch_small<T, kMode, 64>(m, p, small, stream);
}

template <typename T>
int ffn_backward(int dtype, FfnParams p, const void* x, const void* wg, const void* wu, const void* dg, const void* du,
                 void* ws, int64_t ws_bytes, cudaStream_t stream) {
    const FfnPlan plan = ffn_plan(p.M, p.F, p.K, p.dx != 0, p.dw != 0);
    const int64_t tiles = p.dx ? ffn_dx_tiles(p.M, p.K, plan.width) : 0;
    const int64_t per = p.dw ? ffn_dw_tiles(p.F, p.K, plan.width) : 0;
    int64_t room = ws ? ws_bytes / ffn_part_bytes(plan.width) : 0;           // parts
    if (tiles) p.split = (int)std::max<int64_t>(1, std::min<int64_t>(plan.split, room / tiles));
    if (p.split > 1) room -= tiles * p.split;
    if (per) p.split_dw = (int)std::max<int64_t>(1, std::min<int64_t>(plan.split_dw, room / per));
    if (p.split == 1 && p.split_dw == 1) return ffn_launch<T, kBackward>(dtype, p, plan.width, x, wg, wu, dg, du, stream);
    FfnParams d = p;
    if (plan.apart) d.dw = 0;
    d.partial = (float4*)ws;
    int rc = ffn_launch<T, kBackward>(dtype, d, plan.width, x, wg, wu, dg, du, stream);
    if (rc) return rc;
    const int64_t joined = (p.split > 1 ? tiles : 0) + (p.split_dw > 1 ? per : 0);
    const dim3 blocks((unsigned)(joined * (kFM / 2) * plan.width / 8 / 256));
    rc = plan.width == 64 ? enc_launch(ffn_join<T, 64>, blocks, dim3(256), 0, stream, d)
                          : enc_launch(ffn_join<T, 128>, blocks, dim3(256), 0, stream, d);
    if (rc || d.dw == p.dw) return rc;
    p.dx = 0;
    p.split = 1;
    return ffn_launch<T, kBackward>(dtype, p, plan.width, x, wg, wu, dg, du, stream);
}

int ffn_check(int32_t M, int32_t F, int32_t K, int32_t act, int32_t dtype) {
    RAGRT_REQUIRE(dtype == RAGRT_F16 || dtype == RAGRT_BF16, "dtype must be RAGRT_F16 or RAGRT_BF16; got %d",
                  (int)dtype);
    RAGRT_REQUIRE(act >= kSilu && act <= kGeluTanh, "unknown activation %d", (int)act);
    RAGRT_REQUIRE(M >= 0 && F >= 8 && F % 8 == 0 && K >= 8 && K % 8 == 0,
                  "gated_ffn needs M >= 0 and F, K multiples of 8 (M=%d F=%d K=%d)", (int)M, (int)F, (int)K);
    RAGRT_REQUIRE(std::max({M, F, K}) <= 0x7FFFFFFF - 4096, "gated_ffn: sizes up to 2^31 - 4097 (M=%d F=%d K=%d)",
                  (int)M, (int)F, (int)K);          // positions past the last tile stay in 32 bits
    return RAGRT_OK;
}

}  // namespace
}  // namespace ragrt

using namespace ragrt;

extern "C" int ragrt_enc_gated_ffn(const void* d_x, const void* d_w_gate, const void* d_w_up, void* d_h, float* d_gate,
                                   float* d_up, int32_t M, int32_t F, int32_t K, int32_t act, int32_t dtype,
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
    cudaStream_t stream = (cudaStream_t)stream_;
    FfnParams p{M, F, K, act, d_gate != nullptr, 0, 0, 0, 1, 1, nullptr, {d_h, d_gate, d_up}, err};
    // One row at any size: 2048 -> 5504 9.2 us with the weights from memory, 6.9 us of bytes, on the tensor cores 14.4.
    // Up to four where the weights are few: 4 rows 768 -> 2048 5.7 us against 6.5, 2048 -> 4096 12.6 against 13.3; 2 rows
    // 2048 -> 5504 17.4 against 14.5.
    if (M == 1 || (M <= kFewRows && (int64_t)F * K <= (1 << 23))) {
        return dtype == RAGRT_BF16 ? ffn_rows_launch<__nv_bfloat16>(d_x, d_w_gate, d_w_up, p, stream)
                                   : ffn_rows_launch<__half>(d_x, d_w_gate, d_w_up, p, stream);
    }
    return dtype == RAGRT_BF16
               ? ffn_launch<__nv_bfloat16, kForward>(dtype, p, 64, d_x, d_w_gate, d_w_up, nullptr, nullptr, stream)
               : ffn_launch<__half, kForward>(dtype, p, 64, d_x, d_w_gate, d_w_up, nullptr, nullptr, stream);
}

extern "C" int ragrt_enc_gated_ffn_backward(const void* d_dh, const void* d_x, const void* d_w_gate,
                                            const void* d_w_up, const float* d_gate, const float* d_up, void* d_dgate,
                                            void* d_dup, void* d_dx, void* d_dw_gate, void* d_dw_up, int32_t M,
                                            int32_t F, int32_t K, int32_t act, int32_t dtype, void* d_ws,
                                            int64_t ws_bytes, void* stream_) {
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
                    (uintptr_t)d_dw_up | (uintptr_t)d_ws) & 15) == 0,
                  "gated_ffn_backward operands must be 16-byte aligned");
    int* err = device_error_flag();
    if (!err) return fail(RAGRT_ERR_CUDA, "device error flag unavailable");
    const int64_t n8 = (int64_t)M * F / 8;
    const unsigned blocks = (unsigned)std::min<int64_t>(ceil_div(n8, 256), (int64_t)num_sms() * 16);
    rc = dtype == RAGRT_BF16
             ? enc_launch(ffn_act_backward<__nv_bfloat16>, dim3(blocks), dim3(256), 0, stream,
                          (const __nv_bfloat16*)d_dh, d_gate, d_up,
                          (__nv_bfloat16*)d_dgate, (__nv_bfloat16*)d_dup, n8, (int)act)
             : enc_launch(ffn_act_backward<__half>, dim3(blocks), dim3(256), 0, stream, (const __half*)d_dh,
                          d_gate, d_up, (__half*)d_dgate, (__half*)d_dup, n8, (int)act);
    if (rc) return rc;
    if (!d_dx && !d_dw_gate) return RAGRT_OK;
    FfnParams p{M, F, K, act, 0, d_dx != nullptr, d_dw_gate != nullptr, 0, 1, 1, nullptr, {d_dx, d_dw_gate, d_dw_up}, err};
    return dtype == RAGRT_BF16
               ? ffn_backward<__nv_bfloat16>(dtype, p, d_x, d_w_gate, d_w_up, d_dgate, d_dup, d_ws, ws_bytes, stream)
               : ffn_backward<__half>(dtype, p, d_x, d_w_gate, d_w_up, d_dgate, d_dup, d_ws, ws_bytes, stream);
}

extern "C" int64_t ragrt_enc_gated_ffn_workspace(int32_t M, int32_t F, int32_t K, int32_t dx, int32_t dw) {
    if (M < 1 || F < 8 || K < 8) return 0;
    const FfnPlan plan = ffn_plan(M, F, K, dx != 0, dw != 0);
    const int64_t parts = (dx && plan.split > 1 ? ffn_dx_tiles(M, K, plan.width) * plan.split : 0) +
                          (dw && plan.split_dw > 1 ? ffn_dw_tiles(F, K, plan.width) * plan.split_dw : 0);
    return parts * ffn_part_bytes(plan.width);
}
