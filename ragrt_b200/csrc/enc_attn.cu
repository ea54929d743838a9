// enc_attn.cu -- attention over packed sequences, with grouped heads, full or causal.
//
//   o[t, h] = sum_j p_j v[j, g(h)],  p = softmax_j(scale q[t, h] . k[j, g(h)]),  g(h) = h / (heads / kv_heads)
//
// over the keys j of t's own sequence (with causal set: those up to t).  The sequences lie one behind
// the other in the rows of q, k, v; cu_seqlens names where each begins.
//
//   packed_attn_mma    persistent; an item is 256 packed rows (two tiles of 128) of one head.  The tiles run
//                      over the rows as they lie, whatever sequences they belong to: a tile walks the
//                      keys of the sequences that it touches, and each row masks what is not its own.
//                      Short sequences thus share a tile, and no tile is padded but the last.  Warp 0
//                      streams Q and the 64-key blocks of K and V by TMA, warps 1 and 3 issue a tile's
//                      products each (S = Q K^T and O += P V, P from tensor memory), warp 2 finds the
//                      coming items' key ranges, and per tile four warps run the softmax, a thread per row.
//                      Each tile has two score buffers, so that the scores of the block after next are
//                      computed while a block's weights are: no role waits for a whole turn of another.
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
    int T, B, heads, kv_heads, dim, causal, items;
    float scale;
    int* err;
};

// The keys [lo, hi) that rows t, t + 32, ... see; empty for rows outside every sequence.  The last begin
// <= t is found by bisection, for N rows side by side; what a table that is not ascending names outside
// [0, T] gives an empty range.
template <int N>
__device__ __forceinline__ void attn_ranges(const AttnParams& p, int t, int (&lo)[N], int (&hi)[N]) {
    int a[N], b[N];                                  // cu[a] <= t (or a == 0), cu[b] > t (or b == B)
#pragma unroll
    for (int i = 0; i < N; ++i) {
        a[i] = 0;
        b[i] = p.B;
    }
    for (int size = p.B; size > 1; size = (size + 1) >> 1) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int m = (a[i] + b[i]) >> 1;
            if (b[i] - a[i] > 1) {
                if (__ldg(p.cu + m) <= t + 32 * i) a[i] = m; else b[i] = m;
            }
        }
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const int row = t + 32 * i, begin = __ldg(p.cu + a[i]), end = __ldg(p.cu + a[i] + 1);
        // behind T, a bad table, before the first or behind the last sequence
        const bool none = row >= p.T || begin < 0 || end > p.T || row < begin || row >= end;
        lo[i] = none ? 0 : begin;
        hi[i] = none ? 0 : p.causal ? row + 1 : end;
    }
}

// Every entry of the table is looked at by one thread of the grid: bisection alone does not see them all.
__device__ __forceinline__ void attn_check_table(const AttnParams& p, int lane) {
    for (int64_t i = (int64_t)blockIdx.x * 32 + lane; i < p.B; i += (int64_t)gridDim.x * 32) {
        const int begin = __ldg(p.cu + i), end = __ldg(p.cu + i + 1);
        if (begin < 0 || end < begin || end > p.T) atomicExch(p.err, 6);
    }
}

// bits below n of a word, n of any size
__device__ __forceinline__ uint32_t low_bits(int n) { return n <= 0 ? 0u : n >= 32 ? 0xFFFFFFFFu : (1u << n) - 1u; }

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

constexpr int kAM = 128;                       // rows per tile
constexpr int kAN = 64;                        // keys per block
constexpr int kATiles = 2;
constexpr int kAFirst = 4;                     // first softmax warp: TMA, two MMA and the range warp before them
constexpr int kAThreads = 32 * (kAFirst + 4 * kATiles);
constexpr int kARanges = 4;                    // items whose key ranges are in shared memory
constexpr uint32_t kAWaitLimit = 1u << 26;
// The launch's 384 x 168 registers, dealt out anew: a softmax thread holds its row of scores.
constexpr int kARegsFew = 88, kARegsMany = 208;
static_assert(128 * kARegsFew + 256 * kARegsMany <= kAThreads * 168, "more registers than the launch holds");
// The reference maximum of a row moves only when it is exceeded by 2^8: until then the weights are
// at most 256, well inside either type, and the accumulator is not rescaled.
constexpr float kARescale = 8.0f;

template <int DP>
struct AttnCfg {
    static constexpr int kTileQ = kAM * DP * 2;                   // bytes of a Q tile
    static constexpr int kTileK = kAN * DP * 2;                   // bytes of a K or a V block
    static constexpr int kQ = DP == 128 ? 1 : 2;                  // items whose Q is in shared memory
    static constexpr int kStage = 2 * kTileK;                     // the V of a block, the K of the one after next
    static constexpr int kStages = DP == 128 ? 4 : 6;
    static constexpr int kShared = kARanges * 8 * kATiles * kAM + 1024;      // at least sizeof(AttnShared)
    static constexpr int kSmem = 1024 + kQ * kATiles * kTileQ + kStages * kStage + kShared;
    static constexpr uint32_t kO = 2 * kATiles * kAN;             // first accumulator column: S and P lie before
};

struct AttnMaps {
    CUtensorMap q, k, v;
};

// What the roles hand one another, behind the tiles in shared memory.
template <int DP>
struct AttnShared {
    int lo[kARanges][kATiles * kAM], hi[kARanges][kATiles * kAM];     // keys [lo, hi) of each row
    int tlo[kARanges][kATiles], thi[kARanges][kATiles];               // of each tile; [1, 0) where it has none
    int row0[kARanges], head[kARanges];                               // row0 < 0: no more items
    uint64_t full[AttnCfg<DP>::kStages], empty[AttnCfg<DP>::kStages];
    uint64_t qfull[AttnCfg<DP>::kQ], qempty[AttnCfg<DP>::kQ];
    uint64_t rfull[kARanges], rempty[kARanges];
    uint64_t sfull[kATiles][2];              // scores ready (MMA -> softmax)
    uint64_t pready[kATiles][2];             // weights written (softmax -> MMA)
    uint64_t odone[kATiles][2];              // product with V done, even and odd blocks
    uint64_t drain[kATiles];
    uint32_t tmem;
    int abort;
};

// The blocks of an item: 64-key blocks 0 .. n - 1 from key kv0 on, tile t takes [jb[t], je[t]) of them.
struct AttnBlocks {
    int row0 = -1, head, kv0, n = 0, jb[kATiles], je[kATiles];
    __device__ __forceinline__ int lo(int t) const { return t == 0 ? jb[0] : jb[1]; }
    __device__ __forceinline__ int hi(int t) const { return t == 0 ? je[0] : je[1]; }
    template <int DP>
    __device__ __forceinline__ void get(const AttnShared<DP>* sh, int r) {
        row0 = sh->row0[r];
        head = sh->head[r];
        kv0 = 0x7FFFFFFF;
        n = 0;
#pragma unroll
        for (int t = 0; t < kATiles; ++t)
            if (sh->thi[r][t] > 0) kv0 = min(kv0, sh->tlo[r][t]);
#pragma unroll
        for (int t = 0; t < kATiles; ++t) {
            const bool any = sh->thi[r][t] > 0;
            jb[t] = any ? (sh->tlo[r][t] - kv0) / kAN : 0;
            je[t] = any ? (sh->thi[r][t] - kv0 + kAN - 1) / kAN : 0;
            n = max(n, je[t]);
        }
    }
};

// A walk of a thread or a whole warp over the blocks of its CTA's items.  The last of a role's walks
// gives the items' ranges back behind itself (by the lane with `lead` set).
template <int DP, bool kRelease>
struct AttnWalk {
    AttnBlocks b;
    int rec = -1, j = 0;
    bool lead = true;
    // On to the next block; 1: there is one, 0: no more, -1: gave up waiting.
    __device__ __forceinline__ int next(AttnShared<DP>* sh) {
        if (j + 1 < b.n) {
            ++j;
            return 1;
        }
        if (kRelease && rec >= 0 && lead) tc::mbar_arrive(&sh->rempty[rec % kARanges]);
        ++rec;
        if (!tc::mbar_wait_or_abort(&sh->rfull[rec % kARanges], (rec / kARanges) & 1, &sh->abort, kAWaitLimit)) return -1;
        b.get(sh, rec % kARanges);
        j = 0;
        return b.row0 >= 0;
    }
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
    uint8_t* sKV = sm + NQ * kATiles * Cfg::kTileQ;
    AttnShared<DP>* sh = reinterpret_cast<AttnShared<DP>*>(sKV + S * Cfg::kStage);
    static_assert(sizeof(AttnShared<DP>) <= Cfg::kShared, "shared memory of the roles");
    volatile int* abort = &sh->abort;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int s = 0; s < S; ++s) {
            tc::mbar_init(&sh->full[s], 1);
            tc::mbar_init(&sh->empty[s], kATiles);
        }
        for (int s = 0; s < NQ; ++s) {
            tc::mbar_init(&sh->qfull[s], 1);
            tc::mbar_init(&sh->qempty[s], kATiles);
        }
        for (int r = 0; r < kARanges; ++r) {
            tc::mbar_init(&sh->rfull[r], 1);
            tc::mbar_init(&sh->rempty[r], 1 + 5 * kATiles);       // TMA, MMA and softmax warps
        }
        for (int t = 0; t < kATiles; ++t) {
            tc::mbar_init(&sh->drain[t], 1);
            for (int b = 0; b < 2; ++b) {
                tc::mbar_init(&sh->sfull[t][b], 1);
                tc::mbar_init(&sh->pready[t][b], 4);
                tc::mbar_init(&sh->odone[t][b], 1);
            }
        }
        sh->abort = 0;
        tc::mbar_fence_init();
    }
    if (warp == 1) {
        tc::tmem_alloc(&sh->tmem, 512);
        tc::tmem_relinquish();
    }
    tc::fence_before();
    __syncthreads();
    tc::fence_after();
    const uint32_t tbase = sh->tmem;
    bool failed = false;
    pdl_wait_then_release();

    if (warp < kAFirst) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kARegsFew));
        if (warp == 0 && lane == 0) {
            // -------------------------------------------------------- TMA producer
            // stage 0: K0; stage 1: K1; stage u + 2: the V of block u and the K of block u + 2, over all
            // items' blocks
            const int per = p.heads / p.kv_heads;
            AttnWalk<DP, false> kw;
            AttnWalk<DP, true> vw;
            int pos = 0, nq = 0;
            auto load = [&](const AttnBlocks& b, int j, const CUtensorMap* map, uint8_t* to, uint64_t* bar) {
                for (int c = 0; c < DP / 64; ++c)
                    tc::tma_load_3d(to + c * kAN * 128, map, 64 * c, b.head / per, b.kv0 + j * kAN, bar);
            };
            int k = 1;
            for (; !failed; ++pos) {
                if (k > 0) k = kw.next(sh);
                const int v = pos < 2 ? 0 : vw.next(sh);
                if (k < 0 || v < 0) failed = true;
                if (failed || (pos >= 2 && v == 0)) break;
                if (k == 0 && v == 0) {                           // fewer than two blocks in all: nothing to load
                    if (pos == 0) break;
                    continue;
                }
                const int s = pos % S;
                if (pos >= S && !tc::mbar_wait_or_abort(&sh->empty[s], (pos / S - 1) & 1, abort, kAWaitLimit)) {
                    failed = true;
                    break;
                }
                uint8_t* at = sKV + s * Cfg::kStage;
                tc::mbar_arrive_expect_tx(&sh->full[s], ((k > 0) + (v > 0)) * Cfg::kTileK);
                if (v > 0) load(vw.b, vw.j, &maps.v, at + Cfg::kTileK, &sh->full[s]);
                if (k > 0) load(kw.b, kw.j, &maps.k, at, &sh->full[s]);
                if (k > 0 && kw.j == 0) {                         // a new item: its Q
                    const int b = nq % NQ;
                    if (nq >= NQ && !tc::mbar_wait_or_abort(&sh->qempty[b], (nq / NQ - 1) & 1, abort, kAWaitLimit)) {
                        failed = true;
                        break;
                    }
                    tc::mbar_arrive_expect_tx(&sh->qfull[b], kATiles * Cfg::kTileQ);
                    for (int t = 0; t < kATiles; ++t)
                        for (int c = 0; c < DP / 64; ++c)
                            tc::tma_load_3d(sQ + (b * kATiles + t) * Cfg::kTileQ + c * kAM * 128, &maps.q, 64 * c,
                                            kw.b.head, kw.b.row0 + t * kAM, &sh->qfull[b]);
                    ++nq;
                }
            }
            if (failed) {                                         // copies in flight end before the CTA does
                for (int i = max(0, nq - NQ); i < nq; ++i)
                    (void)tc::mbar_wait_bounded(&sh->qfull[i % NQ], (i / NQ) & 1, 1u << 16);
                for (int i = max(0, pos - S); i <= pos; ++i)
                    (void)tc::mbar_wait_bounded(&sh->full[i % S], (i / S) & 1, 1u << 16);
            }
        } else if (warp == 1 || warp == 3) {
            // -------------------------------------------------------- a tile's MMA issuer, one lane of a warp in step
            constexpr uint32_t idS = tc::idesc_f16_f32(kAM, kAN) | idesc_type<T>();
            constexpr uint32_t idO = tc::idesc_f16_f32(kAM, DP) | idesc_type<T>() | kIdescBMn;
            const int t = warp >> 1;
            const uint32_t lead = tc::elect_one();
            AttnWalk<DP, false> sw;                               // scores run two blocks ahead of
            AttnWalk<DP, true> vw;                                // the products with V
            vw.lead = lead != 0;
            uint32_t ns = 0, nv = 0;                              // the tile's blocks begun
            int nq = 0, more = 1;
            for (int pos = 0;; ++pos) {
                const int there = pos < 2 ? 0 : vw.next(sh);
                if (more > 0) more = sw.next(sh);
                if (!__all_sync(0xFFFFFFFFu, there >= 0 && more >= 0)) {
                    failed = true;
                    break;
                }
                if (there == 0 && (pos >= 2 || more == 0)) {
                    if (pos >= 2 || pos == 0) break;
                    continue;
                }
                const int stage = pos % S;
                bool ok = tc::mbar_wait_or_abort(&sh->full[stage], (pos / S) & 1, abort, kAWaitLimit);
                if (!__all_sync(0xFFFFFFFFu, ok)) {
                    failed = true;
                    break;
                }
                tc::fence_after();
                const uint32_t k = tc::smem_u32(sKV + stage * Cfg::kStage), v = k + Cfg::kTileK;
                if (there > 0 && vw.j >= vw.b.lo(t) && vw.j < vw.b.hi(t)) {
                    const uint32_t b = nv & 1u;
                    ok = tc::mbar_wait_or_abort(&sh->pready[t][b], (nv >> 1) & 1, abort, kAWaitLimit);
                    if (!__all_sync(0xFFFFFFFFu, ok)) {
                        failed = true;
                        break;
                    }
                    ++nv;
                    tc::fence_after();
#pragma unroll
                    for (int c = 0; c < kAN / 16; ++c)
                        tc::mma_ts_if(lead, tbase + Cfg::kO + t * DP, tbase + (2 * t + b) * kAN + 8 * c,
                                      tc::sw128_mnmajor_desc(v + 2048 * c, kAN * 128), idO, vw.j > vw.b.lo(t) || c > 0);
                    tc::mma_commit_if(lead, &sh->odone[t][b]);
                }
                if (more > 0) {
                    if (sw.j == 0) {
                        ok = tc::mbar_wait_or_abort(&sh->qfull[nq % NQ], (nq / NQ) & 1, abort, kAWaitLimit);
                        if (!__all_sync(0xFFFFFFFFu, ok)) {
                            failed = true;
                            break;
                        }
                        tc::fence_after();
                    }
                    if (sw.j >= sw.b.lo(t) && sw.j < sw.b.hi(t)) {
                        // S takes the buffer whose weights the product just issued (or an earlier one)
                        // reads: the tensor pipe runs them one behind the other
                        const uint32_t q = tc::smem_u32(sQ + ((nq % NQ) * kATiles + t) * Cfg::kTileQ);
                        const uint32_t b = ns & 1u;
                        ++ns;
#pragma unroll
                        for (int c = 0; c < DP / 16; ++c)
                            tc::mma_ss_if(lead, tbase + (2 * t + b) * kAN,
                                          tc::sw128_kmajor_desc(q + (c >> 2) * kAM * 128 + (c & 3) * 32),
                                          tc::sw128_kmajor_desc(k + (c >> 2) * kAN * 128 + (c & 3) * 32), idS, c > 0);
                        tc::mma_commit_if(lead, &sh->sfull[t][b]);
                    }
                    if (sw.j == sw.b.n - 1) {
                        tc::mma_commit_if(lead, &sh->qempty[nq % NQ]);
                        ++nq;
                    }
                }
                tc::mma_commit_if(lead, &sh->empty[stage]);
            }
            if (failed) {                                         // the last products read shared memory
                tc::mma_commit_if(lead, &sh->drain[t]);
                (void)tc::mbar_wait_bounded(&sh->drain[t], 0, 1u << 16);
            }
        } else if (warp == 2) {
            // -------------------------------------------------------- the items' key ranges, 8 rows a lane
            // This CTA's items: blockIdx.x, blockIdx.x + gridDim.x, ...; heads fastest, and the last rows
            // first: the tiles of a causal sequence grow along it.  Items without a key are passed over.
            constexpr int kRows = kATiles * kAM / 32;
            const int pairs = (p.T + kATiles * kAM - 1) / (kATiles * kAM);
            int lo[kRows], hi[kRows], tlo[kATiles], thi[kATiles], row0 = -1, rec = 0;
            for (int64_t i = blockIdx.x; !failed; i += gridDim.x) {
                const bool end = i >= p.items;
                if (!end) {
                    const int r0 = (pairs - 1 - (int)(i / p.heads)) * kATiles * kAM;
                    if (r0 != row0) {
                        row0 = r0;
                        attn_ranges<kRows>(p, r0 + lane, lo, hi);
#pragma unroll
                        for (int t = 0; t < kATiles; ++t) {
                            tlo[t] = 0x7FFFFFFF;
                            thi[t] = 0;
#pragma unroll
                            for (int x = t * kRows / kATiles; x < (t + 1) * kRows / kATiles; ++x) {
                                if (lo[x] < hi[x]) tlo[t] = min(tlo[t], lo[x]);
                                thi[t] = max(thi[t], hi[x]);
                            }
                            tlo[t] = __reduce_min_sync(0xFFFFFFFFu, tlo[t]);
                            thi[t] = __reduce_max_sync(0xFFFFFFFFu, thi[t]);
                        }
                    }
                    if (max(thi[0], thi[1]) == 0) continue;
                }
                const int r = rec % kARanges;
                const bool ok = rec < kARanges ||
                                tc::mbar_wait_or_abort(&sh->rempty[r], (rec / kARanges - 1) & 1, abort, kAWaitLimit);
                if (!__all_sync(0xFFFFFFFFu, ok)) {
                    failed = true;
                    break;
                }
                if (!end) {
#pragma unroll
                    for (int x = 0; x < kRows; ++x) {
                        sh->lo[r][lane + 32 * x] = lo[x];
                        sh->hi[r][lane + 32 * x] = hi[x];
                    }
                }
                if (lane < kATiles) {
                    sh->tlo[r][lane] = lane == 0 ? tlo[0] : tlo[1];
                    sh->thi[r][lane] = end ? 0 : lane == 0 ? thi[0] : thi[1];
                }
                if (lane == 0) {
                    sh->row0[r] = end ? -1 : row0;
                    sh->head[r] = (int)(i % p.heads);
                }
                __syncwarp();
                if (lane == 0) tc::mbar_arrive(&sh->rfull[r]);
                ++rec;
                if (end) break;
            }
            attn_check_table(p, lane);
        }
    } else {
        // ------------------------------------------------------------ softmax, a thread per row
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kARegsMany));
        const int tile = (warp - kAFirst) >> 2, quad = warp & 3;
        const uint32_t lanes = (uint32_t)(quad * 32) << 16;
        const uint32_t ts = tbase + lanes + (uint32_t)(2 * tile * kAN), to = tbase + lanes + Cfg::kO + (uint32_t)(tile * DP);
        const float scale2 = p.scale * 1.4426950408889634f;       // weights are powers of two
        const uint64_t scale22 = pack2(scale2, scale2);
        const int in_item = tile * kAM + quad * 32 + lane;
        uint32_t blk = 0;                                         // blocks of this tile, over all items
        for (int rec = 0; !failed; ++rec) {
            const int r = rec % kARanges;
            bool ok = tc::mbar_wait_or_abort(&sh->rfull[r], (rec / kARanges) & 1, abort, kAWaitLimit);
            if (!__all_sync(0xFFFFFFFFu, ok)) {
                failed = true;
                break;
            }
            AttnBlocks b;
            b.get(sh, r);
            const int lo = sh->lo[r][in_item], hi = sh->hi[r][in_item];
            __syncwarp();
            if (lane == 0) tc::mbar_arrive(&sh->rempty[r]);
            if (b.row0 < 0) break;
            const int b0 = b.lo(tile), b1 = b.hi(tile);
            if (b0 >= b1) continue;
            const int wlo = __reduce_min_sync(0xFFFFFFFFu, lo < hi ? lo : 0x7FFFFFFF);
            const int whi = __reduce_max_sync(0xFFFFFFFFu, hi);
            float m = -INFINITY, l = 0.f;
            for (int j = b0; j < b1; ++j, ++blk) {
                ok = tc::mbar_wait_or_abort(&sh->sfull[tile][blk & 1], (blk >> 1) & 1, abort, kAWaitLimit);
                if (!__all_sync(0xFFFFFFFFu, ok)) {
                    failed = true;
                    break;
                }
                tc::fence_after();
                const uint32_t tb = ts + (blk & 1) * kAN;
                const int first = b.kv0 + j * kAN;
                // most blocks lie inside every row's range; in the others, 32-key steps that no row of
                // the warp sees are left out
                const bool whole = __all_sync(0xFFFFFFFFu, lo <= first && first + kAN <= hi);
                bool seen[2];
#pragma unroll
                for (int c = 0; c < 2; ++c) seen[c] = whole || (first + 32 * c < whi && first + 32 * c + 32 > wlo);
                float s[kAN];
#pragma unroll
                for (int c = 0; c < 2; ++c)
                    if (seen[c]) tc::ld32x32(tb + 32 * c, *reinterpret_cast<uint32_t(*)[32]>(s + 32 * c));
                tc::wait_ld();
                float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
                if (!whole) {
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        const uint32_t see = low_bits(hi - first - 32 * c) & ~low_bits(lo - first - 32 * c);
#pragma unroll
                        for (int q = 0; q < 32; ++q) s[32 * c + q] = (see >> q) & 1u ? s[32 * c + q] : -INFINITY;
                    }
                }
#pragma unroll
                for (int c = 0; c < kAN; c += 8)
#pragma unroll
                    for (int e = 0; e < 4; ++e) mx[e] = max3(mx[e], s[c + e], s[c + e + 4]);
                const float bm = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * scale2;
                if (__any_sync(0xFFFFFFFFu, bm > m + kARescale)) {
                    const float mn = fmaxf(m, bm);
                    const float alpha = m == -INFINITY ? 0.f : ex2(m - mn);
                    l *= alpha;
                    m = mn;
                    if (j > b0) {                                 // behind the product with the last weights
                        ok = tc::mbar_wait_or_abort(&sh->odone[tile][(blk - 1) & 1], ((blk - 1) >> 1) & 1, abort, kAWaitLimit);
                        if (!__all_sync(0xFFFFFFFFu, ok)) {
                            failed = true;
                            break;
                        }
                        tc::fence_after();
#pragma unroll 1
                        for (int c = 0; c < DP / 32; ++c) {
                            uint32_t r32[32];
                            tc::ld32x32(to + 32 * c, r32);
                            tc::wait_ld();
#pragma unroll
                            for (int q = 0; q < 32; ++q) r32[q] = __float_as_uint(__uint_as_float(r32[q]) * alpha);
                            tc::st32x32(to + 32 * c, r32);
                        }
                    }
                }
                const float ref = m == -INFINITY ? 0.f : m;
                const uint64_t ref2 = pack2(-ref, -ref);
                uint64_t sum[2] = {0ull, 0ull};
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    uint32_t w[16];
                    if (seen[c]) {
#pragma unroll
                        for (int q = 0; q < 16; ++q) {
                            float x, y;
                            unpack2(fma2(pack2(s[32 * c + 2 * q], s[32 * c + 2 * q + 1]), scale22, ref2), x, y);
                            x = ex2(x);
                            y = ex2(y);
                            sum[q & 1] = add2(sum[q & 1], pack2(x, y));
                            const typename Pair16<T>::type xy = Pair16<T>::down(x, y);
                            w[q] = *reinterpret_cast<const uint32_t*>(&xy);
                        }
                    } else {
#pragma unroll
                        for (int q = 0; q < 16; ++q) w[q] = 0u;
                    }
                    tc::st32x16(tb + 16 * c, w);
                }
                float sx, sy;
                unpack2(add2(sum[0], sum[1]), sx, sy);
                l += sx + sy;
                tc::wait_st();
                tc::fence_before();
                __syncwarp();
                if (lane == 0) tc::mbar_arrive(&sh->pready[tile][blk & 1]);
            }
            if (failed) break;
            // the last product; the one two blocks before it came before this block's scores, so that the
            // parity names it
            ok = tc::mbar_wait_or_abort(&sh->odone[tile][(blk - 1) & 1], ((blk - 1) >> 1) & 1, abort, kAWaitLimit);
            if (!__all_sync(0xFFFFFFFFu, ok)) {
                failed = true;
                break;
            }
            tc::fence_after();
            // The next item's weights are announced behind these loads, so that its first product finds
            // the accumulator read.
            const float inv = 1.0f / l;
            const bool mine = lo < hi;
            const int row = b.row0 + in_item;
            T* dst = static_cast<T*>(p.out) + row * p.out_stride + (int64_t)b.head * p.dim;
            float odd = 0.f, o[DP];
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
                attn_row<T>(p, __shfl_sync(0xFFFFFFFFu, row, src), b.head, __shfl_sync(0xFFFFFFFFu, lo, src),
                            __shfl_sync(0xFFFFFFFFu, hi, src));
            }
        }
    }
    if (failed) atomicExch(p.err, 1);
    tc::fence_before();
    __syncthreads();
    if (warp == 1) {
        tc::fence_after();
        tc::tmem_dealloc(tbase, 512);
    }
}

template <typename T, int DP>
int attn_launch(int dtype, const AttnParams& p, cudaStream_t stream) {
    static std::atomic<uint64_t> done{0};
    int rc = enc_allow_smem(packed_attn_mma<T, DP>, AttnCfg<DP>::kSmem, done);
    if (rc) return rc;
    AttnMaps m;
    if ((rc = enc_map_heads(&m.q, dtype, p.q, p.T, p.heads, p.dim, p.q_stride, kAM)) ||
        (rc = enc_map_heads(&m.k, dtype, p.k, p.T, p.kv_heads, p.dim, p.k_stride, kAN)) ||
        (rc = enc_map_heads(&m.v, dtype, p.v, p.T, p.kv_heads, p.dim, p.v_stride, kAN)))
        return rc;
    return enc_launch(packed_attn_mma<T, DP>, dim3((unsigned)std::min(p.items, num_sms())), dim3(kAThreads),
                      AttnCfg<DP>::kSmem, stream, m, p);
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
    RAGRT_REQUIRE(T <= 0x7FFFFFFF - 1024, "too many rows");          // row numbers past the last tile stay in 32 bits
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
    const int64_t items = ceil_div(T, kATiles * kAM) * heads;
    if (items > 0x7FFFFFFF) return fail(RAGRT_ERR_CAPACITY, "too many rows x heads");
    AttnParams p{d_q, d_k, d_v, d_out, d_cu_seqlens, q_stride, k_stride, v_stride, out_stride, T, B, heads, kv_heads,
                 head_dim, causal != 0, (int)items, scale, err};
    cudaStream_t stream = (cudaStream_t)stream_;
    if (dtype == RAGRT_BF16)
        return head_dim <= 64 ? attn_launch<__nv_bfloat16, 64>(dtype, p, stream)
                              : attn_launch<__nv_bfloat16, 128>(dtype, p, stream);
    return head_dim <= 64 ? attn_launch<__half, 64>(dtype, p, stream) : attn_launch<__half, 128>(dtype, p, stream);
}
