// enc_attn.cu -- attention over packed sequences, with grouped heads, full or causal.
//
//   o[t, h] = sum_j p_j v[j, g(h)],  p = softmax_j(scale q[t, h] . k[j, g(h)]),  g(h) = h / (heads / kv_heads)
//
// over the keys j of t's own sequence (with causal set: those up to t).  The sequences lie one behind
// the other in the rows of q, k, v; cu_seqlens names where each begins.
//
//   packed_attn_mma    a CTA per 256 packed rows (two tiles of 128) and head.  The tiles run over the rows
//                      as they lie, whatever sequences they belong to: a tile walks the keys of the
//                      sequences that it touches, and each row masks what is not its own.  Short sequences
//                      thus share a tile, and no tile is padded but the last.  Warp 0 streams Q and the
//                      128-key blocks of K and V by TMA, warp 1 issues the products (S = Q K^T and
//                      O += P V, P from tensor memory), and per tile four warps run the softmax, a
//                      thread per row.
//   attn_row           one row of one head by a warp, in fp32.  A weight of zero does not keep a NaN or
//                      an infinity in a masked row of V out of a matrix product: rows that come out
//                      of it not finite are computed once more by this, over their own keys alone.
#include <algorithm>

#include "enc_common.cuh"
#include "tc.cuh"

namespace ragrt {

namespace {

struct AttnParams {
    const void* q;
    const void* k;
    const void* v;
    void* out;
    const int32_t* cu;
    int64_t q_stride, k_stride, v_stride, out_stride;
    int T, B, heads, kv_heads, dim, causal, per_cta;
    float scale;
    int* err;
};

// The keys [lo, hi) that row t sees; empty for rows outside every sequence.  The last begin <= t is
// found by bisection; what a table that is not ascending names outside [0, T] gives an empty range.
__device__ __forceinline__ void attn_range(const AttnParams& p, int t, int& lo, int& hi) {
    lo = hi = 0;
    if (t >= p.T) return;
    int a = 0, b = p.B;                              // cu[a] <= t (or a == 0), cu[b] > t (or b == B)
    while (b - a > 1) {
        const int m = (a + b) >> 1;
        if (__ldg(p.cu + m) <= t) a = m; else b = m;
    }
    const int begin = __ldg(p.cu + a), end = __ldg(p.cu + a + 1);
    if (begin < 0 || end > p.T) return;              // a bad table
    if (t < begin || t >= end) return;               // before the first or behind the last sequence
    lo = begin;
    hi = p.causal ? t + 1 : end;
}

// Every entry of the table is looked at by one thread of the grid: bisection alone does not see them all.
__device__ __forceinline__ void attn_check_table(const AttnParams& p) {
    for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < p.B; i += (int64_t)gridDim.x * blockDim.x) {
        const int begin = __ldg(p.cu + i), end = __ldg(p.cu + i + 1);
        if (begin < 0 || end < begin || end > p.T) atomicExch(p.err, 6);
    }
}

// One row of one head by one warp.
template <typename T>
__device__ void attn_row(const AttnParams& p, int t, int h, int lo, int hi) {
    const int lane = threadIdx.x & 31;
    const int g = h / (p.heads / p.kv_heads);
    const T* q = static_cast<const T*>(p.q) + t * p.q_stride + (int64_t)h * p.dim;
    const T* k = static_cast<const T*>(p.k) + (int64_t)g * p.dim;
    const T* v = static_cast<const T*>(p.v) + (int64_t)g * p.dim;
    float m = -INFINITY, l = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};         // dims lane, lane + 32, ...
    for (int base = lo; base < hi; base += 32) {
        const int j = base + lane;
        float s = -INFINITY;
        if (j < hi) {
            const T* kr = k + j * p.k_stride;
            s = 0.f;
            for (int c = 0; c < p.dim; c += 8) {
                float f[8], a[8];
                up8<T>(__ldg(reinterpret_cast<const uint4*>(kr + c)), f);
                up8<T>(__ldg(reinterpret_cast<const uint4*>(q + c)), a);
#pragma unroll
                for (int e = 0; e < 8; ++e) s = fmaf(f[e], a[e], s);
            }
            s *= p.scale;
        }
        float mx = s;
#pragma unroll
        for (int x = 16; x; x >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xFFFFFFFFu, mx, x));
        mx = fmaxf(mx, m);
        const float ref = mx == -INFINITY ? 0.f : mx;
        const float e = __expf(s - ref), alpha = __expf(m - ref);
        float sum = e;
#pragma unroll
        for (int x = 16; x; x >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, x);
        l = l * alpha + sum;
        m = mx;
#pragma unroll
        for (int i = 0; i < 4; ++i) o[i] *= alpha;
        const int n = min(32, hi - base);
        for (int i = 0; i < n; ++i) {
            const float pj = __shfl_sync(0xFFFFFFFFu, e, i);
            const T* vr = v + (int64_t)(base + i) * p.v_stride;
#pragma unroll
            for (int c = 0; c < 4; ++c)
                if (lane + 32 * c < p.dim) o[c] = fmaf(pj, (float)vr[lane + 32 * c], o[c]);
        }
    }
    T* dst = static_cast<T*>(p.out) + t * p.out_stride + (int64_t)h * p.dim;
#pragma unroll
    for (int c = 0; c < 4; ++c)
        if (lane + 32 * c < p.dim) dst[lane + 32 * c] = (T)(o[c] / l);
}

constexpr int kAM = 128;                       // rows per tile, keys per block
constexpr int kATiles = 2;
constexpr int kAFirst = 4;                    // first softmax warp: TMA, MMA and two idle warps before them
constexpr int kAThreads = 32 * (kAFirst + 4 * kATiles);
// The launch's 384 x 168 registers, dealt out anew: a softmax thread holds its row of 128 scores.
constexpr int kARegsFew = 88, kARegsMany = 208;
static_assert(128 * kARegsFew + 256 * kARegsMany <= kAThreads * 168, "more registers than the launch holds");
constexpr uint32_t kAWaitLimit = 1u << 26;
// The reference maximum of a row moves only when it is exceeded by 2^8: until then the weights are
// at most 256, well inside either type, and the accumulator is not rescaled.
constexpr float kARescale = 8.0f;

template <int DP>
struct AttnCfg {
    static constexpr int kTile = kAM * DP * 2;                    // bytes of a Q tile, a K or a V block
    static constexpr int kQ = DP == 128 ? 1 : 2;                  // heads whose Q is in shared memory
    static constexpr int kStages = DP == 128 ? 4 : 8;             // K and V blocks in flight
    static constexpr int kSmem = 1024 + (kQ * kATiles + kStages) * kTile + 512;
    static constexpr uint32_t kO = kATiles * kAM;                 // first accumulator column: S and P lie before
};

struct AttnMaps {
    CUtensorMap q, k, v;
};

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float y;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
    return y;
}
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

template <typename T, int DP>
__global__ void __launch_bounds__(kAThreads, 1) packed_attn_mma(const __grid_constant__ AttnMaps maps, const AttnParams p) {
    using Cfg = AttnCfg<DP>;
    constexpr int S = Cfg::kStages, NQ = Cfg::kQ;
    extern __shared__ uint8_t attn_raw[];
    uint8_t* sm = (uint8_t*)(((uintptr_t)attn_raw + 1023) & ~(uintptr_t)1023);
    uint8_t* sQ = sm;
    uint8_t* sKV = sm + NQ * kATiles * Cfg::kTile;
    uint64_t* full = reinterpret_cast<uint64_t*>(sKV + S * Cfg::kTile);
    uint64_t* empty = full + S;
    uint64_t* qfull = empty + S;
    uint64_t* qempty = qfull + NQ;           // both tiles' last scores of a head are done
    uint64_t* sfull = qempty + NQ;           // [2] scores ready (MMA -> softmax)
    uint64_t* pready = sfull + kATiles;      // [2] weights written (softmax -> MMA)
    uint64_t* ofull = pready + kATiles;      // [2] last product of a head done
    uint64_t* drain = ofull + kATiles;
    uint32_t* tslot = reinterpret_cast<uint32_t*>(drain + 1);
    volatile int* abort = reinterpret_cast<volatile int*>(tslot + 1);
    int* swlo = reinterpret_cast<int*>(tslot + 2);                // [8] key range of each softmax warp's rows
    int* swhi = swlo + 4 * kATiles;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    // a CTA takes per_cta heads of its rows, one behind the other
    const int shares = (p.heads + p.per_cta - 1) / p.per_cta;
    const int h0 = (int)(blockIdx.x % shares) * p.per_cta, nh = min(p.per_cta, p.heads - h0);
    // the tiles of a causal sequence grow along it: the longest go first
    const int tiles = (p.T + kATiles * kAM - 1) / (kATiles * kAM);
    const int row0 = (tiles - 1 - (int)(blockIdx.x / shares)) * kATiles * kAM;

    if (threadIdx.x == 0) {
        for (int s = 0; s < S; ++s) {
            tc::mbar_init(full + s, 1);
            tc::mbar_init(empty + s, 1);
        }
        for (int s = 0; s < NQ; ++s) {
            tc::mbar_init(qfull + s, 1);
            tc::mbar_init(qempty + s, 1);
        }
        tc::mbar_init(drain, 1);
        for (int t = 0; t < kATiles; ++t) {
            tc::mbar_init(sfull + t, 1);
            tc::mbar_init(pready + t, 4);
            tc::mbar_init(ofull + t, 1);
        }
        *abort = 0;
        tc::mbar_fence_init();
    }
    if (warp == 1) {
        tc::tmem_alloc(tslot, 512);
        tc::tmem_relinquish();
    }
    pdl_wait_then_release();
    attn_check_table(p);
    const int tile = (warp - kAFirst) >> 2, quad = warp & 3;
    int lo = 0, hi = 0, wlo = 0, whi = 0;                         // this row's keys, and its warp's
    const int row = row0 + tile * kAM + quad * 32 + lane;         // of a softmax thread
    if (warp >= kAFirst) {
        attn_range(p, row, lo, hi);
        wlo = __reduce_min_sync(0xFFFFFFFFu, lo < hi ? lo : 0x7FFFFFFF);
        whi = __reduce_max_sync(0xFFFFFFFFu, hi);
        if (lane == 0) {
            swlo[warp - kAFirst] = wlo;
            swhi[warp - kAFirst] = whi;
        }
    }
    tc::fence_before();
    __syncthreads();
    tc::fence_after();
    const uint32_t tbase = *tslot;
    // the keys that each tile walks, in blocks of 128 from the first key of either
    int kv0 = 0x7FFFFFFF, jb[kATiles], je[kATiles];
#pragma unroll
    for (int t = 0; t < kATiles; ++t) {
        jb[t] = 0x7FFFFFFF;
        je[t] = 0;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            jb[t] = min(jb[t], swlo[4 * t + w]);
            je[t] = max(je[t], swhi[4 * t + w]);
        }
        kv0 = min(kv0, jb[t]);
    }
#pragma unroll
    for (int t = 0; t < kATiles; ++t) {
        const bool any = je[t] > 0;
        jb[t] = any ? (jb[t] - kv0) / kAM : 0;
        je[t] = any ? (je[t] - kv0 + kAM - 1) / kAM : 0;
    }
    const int n = max(je[0], je[1]);                              // blocks per head
    bool failed = false;

    if (warp < kAFirst) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kARegsFew));
    if (warp == 0) {
        // ------------------------------------------------------------ TMA producer
        if (lane == 0 && n > 0) {
            const int per = p.heads / p.kv_heads;
            int i = 0, hh = 0;
            for (; hh < nh && !failed; ++hh) {
                const int b = hh % NQ;
                if (hh >= NQ && !tc::mbar_wait_or_abort(qempty + b, (hh / NQ - 1) & 1, abort, kAWaitLimit)) {
                    failed = true;
                    break;
                }
                tc::mbar_arrive_expect_tx(qfull + b, kATiles * Cfg::kTile);
                for (int t = 0; t < kATiles; ++t)
                    for (int c = 0; c < DP / 64; ++c)
                        tc::tma_load_3d(sQ + (b * kATiles + t) * Cfg::kTile + c * kAM * 128, &maps.q, 64 * c, h0 + hh,
                                        row0 + t * kAM, qfull + b);
                const int g = (h0 + hh) / per;
                for (int k = 0; k < 2 * n; ++k, ++i) {            // K0, V0, K1, V1, ...
                    const int s = i % S;
                    if (i >= S && !tc::mbar_wait_or_abort(empty + s, ((i / S) - 1) & 1, abort, kAWaitLimit)) {
                        failed = true;
                        break;
                    }
                    tc::mbar_arrive_expect_tx(full + s, Cfg::kTile);
                    for (int c = 0; c < DP / 64; ++c)
                        tc::tma_load_3d(sKV + s * Cfg::kTile + c * kAM * 128, k & 1 ? &maps.v : &maps.k, 64 * c, g,
                                        kv0 + (k >> 1) * kAM, full + s);
                }
            }
            if (failed) {                                         // copies in flight end before the CTA does
                for (int k = max(0, hh - NQ); k < min(hh + 1, nh); ++k)
                    (void)tc::mbar_wait_bounded(qfull + k % NQ, (k / NQ) & 1, 1u << 16);
                for (int k = max(0, i - S); k < i; ++k)
                    (void)tc::mbar_wait_bounded(full + k % S, (k / S) & 1, 1u << 16);
            }
        }
    } else if (warp == 1) {
        // ------------------------------------------------------------ MMA issuer
        if (lane == 0 && n > 0) {
            constexpr uint32_t idS = tc::idesc_f16_f32(kAM, kAM) | idesc_type<T>();
            constexpr uint32_t idO = tc::idesc_f16_f32(kAM, DP) | idesc_type<T>() | kIdescBMn;
            // step u: the product with V of block u, and the scores of block u + 1, over all heads' blocks
            const int total = nh * n;
            uint32_t pph[kATiles] = {0u, 0u};                     // pready phases used
            int j = -1;                                           // u % n
            for (int u = -1, hq = 0; u < total && !failed; ++u) {
                const int vi = 2 * u + 1, ki = 2 * u + 2;
                const int jn = j + 1 == n ? 0 : j + 1;            // block of u + 1, and
                const bool next = u + 1 < total;                  // whether there is one
                if (u >= 0) failed = !tc::mbar_wait_or_abort(full + vi % S, (vi / S) & 1, abort, kAWaitLimit);
                if (!failed && next) failed = !tc::mbar_wait_or_abort(full + ki % S, (ki / S) & 1, abort, kAWaitLimit);
                if (!failed && next && jn == 0) {                 // u + 1 begins head hq
                    failed = !tc::mbar_wait_or_abort(qfull + hq % NQ, (hq / NQ) & 1, abort, kAWaitLimit);
                    ++hq;
                }
                if (failed) break;
                tc::fence_after();
                const uint32_t v = tc::smem_u32(sKV + (vi % S) * Cfg::kTile), k = tc::smem_u32(sKV + (ki % S) * Cfg::kTile);
#pragma unroll
                for (int t = 0; t < kATiles; ++t) {
                    if (u >= 0 && j >= jb[t] && j < je[t]) {
                        if (!tc::mbar_wait_or_abort(pready + t, pph[t] & 1, abort, kAWaitLimit)) {
                            failed = true;
                            break;
                        }
                        ++pph[t];
                        tc::fence_after();
#pragma unroll
                        for (int c = 0; c < kAM / 16; ++c)
                            tc::mma_ts(tbase + Cfg::kO + t * DP, tbase + t * kAM + 8 * c,
                                       tc::sw128_mnmajor_desc(v + 2048 * c, kAM * 128), idO, j > jb[t] || c > 0);
                        if (j == je[t] - 1) tc::mma_commit(ofull + t);
                    }
                    if (next && jn >= jb[t] && jn < je[t]) {
                        // S takes the columns of the P that the product just issued reads: the tensor
                        // pipe runs them one behind the other
                        const uint32_t q = tc::smem_u32(sQ + (((hq - 1) % NQ) * kATiles + t) * Cfg::kTile);
#pragma unroll
                        for (int c = 0; c < DP / 16; ++c) {
                            const uint32_t at = (c >> 2) * kAM * 128 + (c & 3) * 32;
                            tc::mma_ss(tbase + t * kAM, tc::sw128_kmajor_desc(q + at), tc::sw128_kmajor_desc(k + at), idS,
                                       c > 0);
                        }
                        tc::mma_commit(sfull + t);
                    }
                }
                if (failed) break;
                if (u >= 0) tc::mma_commit(empty + vi % S);
                if (next) {
                    tc::mma_commit(empty + ki % S);
                    if (jn == n - 1) tc::mma_commit(qempty + (hq - 1) % NQ);
                }
                j = jn;
            }
            if (failed) {                                         // the last products read shared memory
                tc::mma_commit(drain);
                (void)tc::mbar_wait_bounded(drain, 0, 1u << 16);
            }
        }
    }
    } else {
        // ------------------------------------------------------------ softmax, a thread per row
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kARegsMany));
        const uint32_t lanes = (uint32_t)(quad * 32) << 16;
        const uint32_t ts = tbase + lanes + (uint32_t)(tile * kAM), to = tbase + lanes + Cfg::kO + (uint32_t)(tile * DP);
        const float scale2 = p.scale * 1.4426950408889634f;       // weights are powers of two
        const uint64_t scale22 = pack2(scale2, scale2);
        const int b0 = tile == 0 ? jb[0] : jb[1], b1 = tile == 0 ? je[0] : je[1];
        uint32_t sph = 0;
        for (int hh = 0; hh < nh && b0 < b1 && !failed; ++hh) {
            float m = -INFINITY, l = 0.f;
            for (int j = b0; j < b1; ++j, ++sph) {
                const bool ok = tc::mbar_wait_or_abort(sfull + tile, sph & 1, abort, kAWaitLimit);
                if (!__all_sync(0xFFFFFFFFu, ok)) {
                    failed = true;
                    break;
                }
                tc::fence_after();
                const int first = kv0 + j * kAM;
                // most blocks lie inside every row's range; in the others, 32-key steps that no row of
                // the warp sees are left out
                const bool whole = __all_sync(0xFFFFFFFFu, lo <= first && first + kAM <= hi);
                float s[128];
                if (whole) {
#pragma unroll
                    for (int c = 0; c < 4; ++c) tc::ld32x32(ts + 32 * c, *reinterpret_cast<uint32_t(*)[32]>(s + 32 * c));
                    tc::wait_ld();
                } else {
                    const int c0 = lo - first, c1 = hi - first;
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        if (first + 32 * c < whi && first + 32 * c + 32 > wlo) {
                            tc::ld32x32(ts + 32 * c, *reinterpret_cast<uint32_t(*)[32]>(s + 32 * c));
                            tc::wait_ld();
#pragma unroll
                            for (int q = 32 * c; q < 32 * c + 32; ++q) s[q] = q >= c0 && q < c1 ? s[q] : -INFINITY;
                        } else {
#pragma unroll
                            for (int q = 32 * c; q < 32 * c + 32; ++q) s[q] = -INFINITY;
                        }
                    }
                }
                float mx[4];
#pragma unroll
                for (int c = 0; c < 4; ++c) mx[c] = fmaxf(s[c], s[c + 4]);
#pragma unroll
                for (int c = 8; c < 128; c += 8)
#pragma unroll
                    for (int e = 0; e < 4; ++e) mx[e] = max3(mx[e], s[c + e], s[c + e + 4]);
                const float bm = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * scale2;
                if (__any_sync(0xFFFFFFFFu, bm > m + kARescale)) {
                    // the scores of this block came behind the product with the last weights, so the
                    // accumulator is at rest
                    const float mn = fmaxf(m, bm);
                    const float alpha = m == -INFINITY ? 0.f : ex2(m - mn);
                    l *= alpha;
                    m = mn;
                    if (j > b0) {
#pragma unroll 1
                        for (int c = 0; c < DP / 32; ++c) {
                            uint32_t r[32];
                            tc::ld32x32(to + 32 * c, r);
                            tc::wait_ld();
#pragma unroll
                            for (int q = 0; q < 32; ++q) r[q] = __float_as_uint(__uint_as_float(r[q]) * alpha);
                            tc::st32x32(to + 32 * c, r);
                        }
                    }
                }
                const float ref = m == -INFINITY ? 0.f : m;
                const uint64_t ref2 = pack2(-ref, -ref);
                uint64_t sum[2] = {0ull, 0ull};
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    uint32_t w[16];
                    if (whole || (first + 32 * c < whi && first + 32 * c + 32 > wlo)) {
#pragma unroll
                        for (int q = 0; q < 16; ++q) {
                            float a, b;
                            unpack2(fma2(pack2(s[32 * c + 2 * q], s[32 * c + 2 * q + 1]), scale22, ref2), a, b);
                            a = ex2(a);
                            b = ex2(b);
                            sum[q & 1] = add2(sum[q & 1], pack2(a, b));
                            const typename Pair16<T>::type ab = Pair16<T>::down(a, b);
                            w[q] = *reinterpret_cast<const uint32_t*>(&ab);
                        }
                    } else {
#pragma unroll
                        for (int q = 0; q < 16; ++q) w[q] = 0u;
                    }
                    tc::st32x16(ts + 16 * c, w);
                }
                float sa, sb;
                unpack2(add2(sum[0], sum[1]), sa, sb);
                l += sa + sb;
                tc::wait_st();
                tc::fence_before();
                __syncwarp();
                if (lane == 0) tc::mbar_arrive(pready + tile);
            }
            if (!failed) {
                const bool ok = tc::mbar_wait_or_abort(ofull + tile, hh & 1, abort, kAWaitLimit);
                failed = !__all_sync(0xFFFFFFFFu, ok);
            }
            if (failed) break;
            tc::fence_after();
            // The next head's weights are announced behind these loads, so that its first product finds
            // the accumulator read.
            const float inv = 1.0f / l;
            const int h = h0 + hh;
            const bool mine = lo < hi;
            T* dst = static_cast<T*>(p.out) + row * p.out_stride + (int64_t)h * p.dim;
            float odd = 0.f;
            float o[DP];
#pragma unroll
            for (int c = 0; c < DP / 32; ++c) tc::ld32x32(to + 32 * c, *reinterpret_cast<uint32_t(*)[32]>(o + 32 * c));
            tc::wait_ld();
#pragma unroll
            for (int c = 0; c < DP; ++c) {
                o[c] *= inv;
                odd = fmaf(o[c], 0.f, odd);                       // NaN as soon as one is not finite
            }
            const bool bad = mine && !(odd == 0.f);
            if (mine && !bad) {
#pragma unroll
                for (int c = 0; c < DP; c += 8)
                    if (c < p.dim) *reinterpret_cast<uint4*>(dst + c) = down8<T>(*reinterpret_cast<float(*)[8]>(o + c));
            }
            for (unsigned left = __ballot_sync(0xFFFFFFFFu, bad); left; left &= left - 1) {
                const int src = __ffs(left) - 1;
                attn_row<T>(p, __shfl_sync(0xFFFFFFFFu, row, src), h, __shfl_sync(0xFFFFFFFFu, lo, src),
                            __shfl_sync(0xFFFFFFFFu, hi, src));
            }
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

template <typename T, int DP>
int attn_launch(int dtype, AttnParams p, cudaStream_t stream) {
    static std::atomic<uint64_t> done{0};
    int rc = enc_allow_smem(packed_attn_mma<T, DP>, AttnCfg<DP>::kSmem, done);
    if (rc) return rc;
    AttnMaps m;
    if ((rc = enc_map_heads(&m.q, dtype, p.q, p.T, p.heads, p.dim, p.q_stride, kAM)) ||
        (rc = enc_map_heads(&m.k, dtype, p.k, p.T, p.kv_heads, p.dim, p.k_stride, kAM)) ||
        (rc = enc_map_heads(&m.v, dtype, p.v, p.T, p.kv_heads, p.dim, p.v_stride, kAM)))
        return rc;
    // Several heads per CTA save its set-up (barriers, tensor memory, the bisection of the table), as
    // long as eight CTAs remain for each SM to even out their lengths.
    const int64_t pairs = ceil_div(p.T, kATiles * kAM);
    p.per_cta = (int)std::max<int64_t>(1, std::min<int64_t>(p.heads, pairs * p.heads / (8 * (int64_t)num_sms())));
    const int64_t blocks = pairs * ceil_div(p.heads, p.per_cta);
    if (blocks > 0x7FFFFFFF) return fail(RAGRT_ERR_CAPACITY, "too many rows x heads");
    return enc_launch(packed_attn_mma<T, DP>, dim3((unsigned)blocks), dim3(kAThreads), AttnCfg<DP>::kSmem, stream, m, p);
}

}  // namespace
}  // namespace ragrt

using namespace ragrt;

extern "C" int ragrt_enc_packed_attention(const void* d_q, const void* d_k, const void* d_v,
                                          const int32_t* d_cu_seqlens, void* d_out, int32_t T, int32_t B,
                                          int32_t heads, int32_t kv_heads, int32_t head_dim, int64_t q_stride,
                                          int64_t k_stride, int64_t v_stride, int64_t out_stride, float scale,
                                          int32_t causal, int32_t dtype, void* stream_) {
    RAGRT_REQUIRE(dtype == RAGRT_F16 || dtype == RAGRT_BF16, "dtype must be RAGRT_F16 or RAGRT_BF16; got %d",
                  (int)dtype);
    RAGRT_REQUIRE(T >= 0 && B >= 0, "T and B must be >= 0");
    RAGRT_REQUIRE(heads >= 1 && heads <= 65535 && kv_heads >= 1 && heads % kv_heads == 0,
                  "heads must be in [1, 65535] and a multiple of kv_heads (heads=%d kv_heads=%d)", (int)heads,
                  (int)kv_heads);
    RAGRT_REQUIRE(head_dim >= 8 && head_dim <= 128 && head_dim % 8 == 0,
                  "packed_attention needs head_dim a multiple of 8 in [8, 128]; got %d", (int)head_dim);
    const int64_t qw = (int64_t)heads * head_dim, kw = (int64_t)kv_heads * head_dim;
    RAGRT_REQUIRE(q_stride >= qw && out_stride >= qw && k_stride >= kw && v_stride >= kw &&
                      (q_stride | k_stride | v_stride | out_stride) % 8 == 0,
                  "row strides must hold all heads and be multiples of 8 elements");
    RAGRT_REQUIRE(scale > 0.f && scale <= 3.0e38f, "scale must be positive and finite");
    if (T == 0 || B == 0) return RAGRT_OK;
    RAGRT_REQUIRE(d_q && d_k && d_v && d_cu_seqlens && d_out, "null argument");
    RAGRT_REQUIRE((((uintptr_t)d_q | (uintptr_t)d_k | (uintptr_t)d_v | (uintptr_t)d_out) & 15) == 0 &&
                      ((uintptr_t)d_cu_seqlens & 3) == 0,
                  "packed_attention operands must be 16-byte aligned");
    int* err = device_error_flag();
    if (!err) return fail(RAGRT_ERR_CUDA, "device error flag unavailable");
    AttnParams p{d_q, d_k, d_v, d_out, d_cu_seqlens, q_stride, k_stride, v_stride, out_stride, T, B, heads, kv_heads,
                 head_dim, causal != 0, 1, scale, err};
    cudaStream_t stream = (cudaStream_t)stream_;
    if (dtype == RAGRT_BF16)
        return head_dim <= 64 ? attn_launch<__nv_bfloat16, 64>(dtype, p, stream)
                              : attn_launch<__nv_bfloat16, 128>(dtype, p, stream);
    return head_dim <= 64 ? attn_launch<__half, 64>(dtype, p, stream) : attn_launch<__half, 128>(dtype, p, stream);
}
