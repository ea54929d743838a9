// enc_attn.cu -- attention over packed sequences, with grouped heads, full or causal.
//
//   o[t, h] = sum_j p_j v[j, g(h)],  p = softmax_j(scale q[t, h] . k[j, g(h)]),  g(h) = h / (heads / kv_heads)
//
// over the keys j of t's own sequence (with causal set: those up to t).  The sequences lie one behind
// the other in the rows of q, k, v; cu_seqlens names where each begins.
//
//   packed_attn_mma    persistent; an item is one or two tiles of 128 rows of a head, each tile of one sequence.
//                      Warp 0 streams Q and the blocks of K and V by TMA, warp 1 issues the products
//                      (S = Q K^T and O += P V, P from tensor memory), warp 2 finds the coming items'
//                      sequences, and per tile four warps run the softmax, a thread per row.
//                      CTAs of two tiles are bound by the turn of a tile: per 128 keys about 2,300 cycles of
//                      softmax (two warps share an exponential unit that needs 1,024 for each), then P V and
//                      the next Q K^T (16 products of about 95 cycles; a 128-row operand from shared memory
//                      takes that long whatever the width of the other).  One sequence of 16,384 rows, 16
//                      heads of 128, causal: 1.03 ms, 1,070 TFLOP/s, the tensor pipe at work 57 % of its
//                      cycles (12 prompts of 1-4,096, 46 %: the turns end with each item).  CTAs of one tile, for
//                      short sequences, wait: an item is one chain of load, product, softmax, product, store, and
//                      of the 17 warps that share an issued instruction 6.6 wait for memory or tensor memory, with
//                      47 % of the issue slots, 19 % of the tensor pipe and 36 % of the memory's rate used.  1,024
//                      passages of 20-180 rows, 12 heads: 195 us, 3.2 TB/s (218 in a long run).  Tried and
//                      dropped: tiles over the rows as they lie, several sequences in one (masks cost more than
//                      the rows saved: 263 us); 64-key blocks with two score buffers for wide heads
//                      (1.59 ms for the long sequence: twice the products at the same 95 cycles); a quarter of
//                      the exponentials as polynomials on the FMA units (0.97 ms, no gain); two tiles of one
//                      CTA with an issuing warp each (1.20 ms: they fall into step and want the same units at
//                      the same time).
//   attn_odd_rows      A weight of zero does not keep a NaN or an infinity in a masked row of V out of a
//                      matrix product.  Of the rows that come out of it not finite this finds those that
//                      are so by the formula, and what they are;
//   attn_rows          computes the others once more, over their own keys alone: a few rows of one head at
//                      a time by a warp, in fp32.
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

constexpr int kAM = 128;                       // rows per tile

// Where the tiles lie: sequence b has the slots floor(cu[b] / 128) + b on, one for each 128 of its rows.
// A sequence's slots end where the next one's begin or one before, so that no sums over the sequences'
// lengths are needed: a slot's sequence is the last one that begins at or before it.
__device__ __forceinline__ int64_t attn_slot(int begin, int b) { return (int64_t)(begin >> 7) + b; }

// The rows [row0, row0 + rows) of a slot and the keys [lo, hi) they see (the last row's, if causal); rows
// = 0 for a slot without any.  By a whole warp: 32 entries of the table are looked at a time.  What a
// table that is not ascending names outside [0, T] counts as none.
struct AttnTile {
    int row0, rows, lo, hi;
};
__device__ __forceinline__ AttnTile attn_tile(const AttnParams& p, int64_t slot, int lane) {
    int b = 0, n = p.B;                              // the sequence is among b .. b + n - 1
    bool any = true;
#pragma unroll 1
    while (n > 1 && any) {
        const int step = (n + 31) >> 5;
        const int i = b + min(lane * step, n - 1);
        const bool before = lane * step < n && attn_slot(__ldg(p.cu + i), i) <= slot;
        const int k = __popc(__ballot_sync(0xFFFFFFFFu, before));
        any = k > 0;
        b += max(k - 1, 0) * step;
        n = min(step, n - max(k - 1, 0) * step);
    }
    const int begin = __ldg(p.cu + b), end = __ldg(p.cu + b + 1);
    const int64_t first = begin + (slot - attn_slot(begin, b)) * kAM;
    AttnTile t{0, 0, 0, 0};
    if (any && begin >= 0 && end <= p.T && first >= begin && first < end) {
        t.row0 = (int)first;
        t.rows = min(kAM, end - t.row0);
        t.lo = begin;
        t.hi = p.causal ? t.row0 + t.rows : end;
    }
    return t;
}

// bits below n of a word, n of any size
__device__ __forceinline__ uint32_t low_bits(int n) { return n <= 0 ? 0u : n >= 32 ? 0xFFFFFFFFu : (1u << n) - 1u; }

// The first R of a warp's rows of one head (bit i of `rows`: row row0 + i, with the keys [lo, end), causal
// [lo, row0 + i]), by the warp: a lane per key for the scores, per four columns for the sums.  Returns the other rows.
// They share what is loaded of K and V, kScores and kSums loads ahead: it is their latency that counts.  8192 rows,
// 8 heads of 128, causal, with a NaN in V in the middle (84 rows before it in its tile): 5.8 ms in all, a row by itself
// and load by load 38; two full sequences of 8000 and 192 rows, V of the second NaN, so that all of the first is
// computed again: 29 ms (165), 0.27 where all is finite.  Tried and dropped: zeros over the rest of the last block of V
// in shared memory before the products read it: 0.36 ms for that call, but 1024 passages 195 -> 229 us.
template <typename T, int R, int kScores, int kSums>
__device__ __noinline__ unsigned attn_rows(const AttnParams& p, int h, int row0, unsigned rows, int lo, int end) {
    const int lane = threadIdx.x & 31, g = h / (p.heads / p.kv_heads);
    const T* q = static_cast<const T*>(p.q) + (int64_t)h * p.dim;
    const T* k = static_cast<const T*>(p.k) + (int64_t)g * p.dim;
    const bool there = 4 * lane < p.dim;
    const T* v = static_cast<const T*>(p.v) + (int64_t)g * p.dim + (there ? 4 * lane : 0);
    int row[R], n = 0, last = end;                   // behind the last one: the first again, not stored
    float m[R], l[R], o[R][4];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        row[r] = rows ? row0 + __ffs(rows) - 1 : row[0];
        if (p.causal && rows) last = row[r] + 1;
        n += rows ? 1 : 0;
        rows &= rows - 1;
        m[r] = -INFINITY;
        l[r] = o[r][0] = o[r][1] = o[r][2] = o[r][3] = 0.f;
    }
#pragma unroll 1
    for (int base = lo; base < last; base += 32) {
        const int j = base + lane;
        float s[R] = {};
        const T* kr = k + min(j, last - 1) * p.k_stride;
#pragma unroll kScores
        for (int c = 0; c < p.dim; c += 8) {
            float f[8], a[8];
            up8<T>(__ldg(reinterpret_cast<const uint4*>(kr + c)), f);
#pragma unroll
            for (int r = 0; r < R; ++r) {
                up8<T>(__ldg(reinterpret_cast<const uint4*>(q + row[r] * p.q_stride + c)), a);
#pragma unroll
                for (int e = 0; e < 8; ++e) s[r] = fmaf(f[e], a[e], s[r]);
            }
        }
#pragma unroll
        for (int r = 0; r < R; ++r) {
            s[r] = j < (p.causal ? row[r] + 1 : end) ? s[r] * p.scale : -INFINITY;
            float mx = s[r];
#pragma unroll
            for (int x = 16; x; x >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xFFFFFFFFu, mx, x));
            mx = fmaxf(mx, m[r]);
            const float ref = mx == -INFINITY ? 0.f : mx, alpha = __expf(m[r] - ref);
            s[r] = __expf(s[r] - ref);               // the weight
            float sum = s[r];
#pragma unroll
            for (int x = 16; x; x >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, x);
            l[r] = l[r] * alpha + sum;
            m[r] = mx;
#pragma unroll
            for (int c = 0; c < 4; ++c) o[r][c] *= alpha;
        }
        const int keys = min(32, last - base);
#pragma unroll kSums
        for (int i = 0; i < keys; ++i) {
            const uint2 u = __ldg(reinterpret_cast<const uint2*>(v + (base + i) * p.v_stride));
            const float2 f = Pair16<T>::up(*reinterpret_cast<const typename Pair16<T>::type*>(&u.x));
            const float2 e = Pair16<T>::up(*reinterpret_cast<const typename Pair16<T>::type*>(&u.y));
#pragma unroll
            for (int r = 0; r < R; ++r) {
                const float w = __shfl_sync(0xFFFFFFFFu, s[r], i);
                const bool sees = base + i < (p.causal ? row[r] + 1 : end);      // not a matter of its weight: V may be NaN
                o[r][0] = sees ? fmaf(w, f.x, o[r][0]) : o[r][0];
                o[r][1] = sees ? fmaf(w, f.y, o[r][1]) : o[r][1];
                o[r][2] = sees ? fmaf(w, e.x, o[r][2]) : o[r][2];
                o[r][3] = sees ? fmaf(w, e.y, o[r][3]) : o[r][3];
            }
        }
    }
#pragma unroll
    for (int r = 0; r < R; ++r) {
        if (r >= n || !there) break;
        typename Pair16<T>::type y[2] = {Pair16<T>::down(o[r][0] / l[r], o[r][1] / l[r]),
                                         Pair16<T>::down(o[r][2] / l[r], o[r][3] / l[r])};
        *reinterpret_cast<uint2*>(static_cast<T*>(p.out) + row[r] * p.out_stride + (int64_t)h * p.dim + 4 * lane) =
            *reinterpret_cast<const uint2*>(y);
    }
    return rows;
}

// Rows of one head, of a warp, whose output is not finite although the sum of their weights is: bit i of `rows` is
// row row0 + i, which sees the keys [lo, end) (causal: [lo, row0 + i]).  A column in which a row of V that is seen is
// not finite is NaN, or the infinity that all such rows agree on, by the formula.  A column without any has it from
// a row of V that may not be seen, through a weight of zero: the rows returned, which are to be computed again.  A
// row of V that is not finite does that to the rows before it in its tile alone, and there only in columns in which
// no row before it was: few rows of a causal sequence.  It does it to all rows of a full sequence that ends less than
// a block of keys before it (attn_rows has what that costs).  The warp looks at each seen row of V once.  8192 rows, 8 heads of 128, causal, 0.19 ms
// when all is finite: one NaN in an early row of V 0.69 ms, the later half of V NaN 0.89 (all such rows computed
// again: 105 and 81).  No branch but the whole warp's and no vote: those made the kernel hold a convergence barrier's
// state in memory across the call (1024 passages 194 -> 203 us).
template <typename T>
__device__ __noinline__ unsigned attn_odd_rows(const AttnParams& p, int h, int row0, unsigned rows, int lo, int end) {
    constexpr uint32_t kExp = std::is_same_v<T, __half> ? 0x7C00u : 0x7F80u, kStep = kExp & (0u - kExp);
    const int lane = threadIdx.x & 31, vec = lane & 15;                           // 8 values of every other row
    const bool there = vec < p.dim / 8;
    const T* v = static_cast<const T*>(p.v) + (int64_t)(h / (p.heads / p.kv_heads)) * p.dim + (there ? 8 * vec : 0);
    const uint4 zero = make_uint4(0u, 0u, 0u, 0u);
    uint32_t up = 0, down = 0, nan = 0;               // bit e: a seen row's value e is +inf, -inf, NaN
    auto halves = [&](const uint4& u, auto f) {
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int e = 0; e < 8; ++e) f(e, (w[e >> 1] >> (16 * (e & 1))) & 0xFFFFu);
    };
    auto odd = [&](uint32_t w) { return (w & (kExp * 0x10001u)) + kStep * 0x10001u; };         // its top bits: not finite
    int done = lo;
    unsigned again = 0;
    for (; rows; rows &= rows - 1) {                  // the branches are the whole warp's throughout
        const int row = row0 + __ffs(rows) - 1, hi = p.causal ? row + 1 : end;
#pragma unroll 1
        for (; done < hi; done += 8) {
            uint4 u[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int j = done + 2 * i + (lane >> 4);
                u[i] = there && j < hi ? __ldg(reinterpret_cast<const uint4*>(v + j * p.v_stride)) : zero;
            }
            uint32_t any = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) any |= odd(u[i].x) | odd(u[i].y) | odd(u[i].z) | odd(u[i].w);
            if (__reduce_or_sync(0xFFFFFFFFu, any & 0x80008000u) == 0) continue;
#pragma unroll
            for (int i = 0; i < 4; ++i)
                halves(u[i], [&](int e, uint32_t x) {
                    const uint32_t is = (x & kExp) == kExp ? 1u << e : 0u, not_inf = (x & 0x7FFFu & ~kExp) ? is : 0u;
                    nan |= not_inf;
                    down |= (x >> 15) ? is & ~not_inf : 0u;
                    up |= (x >> 15) ? 0u : is & ~not_inf;
                });
        }
        done = hi;
        up |= __shfl_xor_sync(0xFFFFFFFFu, up, 16);
        down |= __shfl_xor_sync(0xFFFFFFFFu, down, 16);
        nan |= __shfl_xor_sync(0xFFFFFFFFu, nan, 16);
        uint4* dst = reinterpret_cast<uint4*>(static_cast<T*>(p.out) + row * p.out_stride + (int64_t)h * p.dim) + vec;
        const uint32_t all = up | down | nan;
        const uint4 was = there ? *dst : zero;
        uint32_t w[4] = {}, left = 0;                 // left: not finite, and none of the seen rows is
        halves(was, [&](int e, uint32_t x) {
            const bool known = (all >> e) & 1u, is_nan = ((nan | (up & down)) >> e) & 1u;
            left |= (x & kExp) == kExp && !known ? 1u : 0u;
            x = !known ? x : is_nan ? 0x7FFFu : (down >> e) & 1u ? kExp | 0x8000u : kExp;
            w[e >> 1] |= x << (16 * (e & 1));
        });
        if (__reduce_or_sync(0xFFFFFFFFu, left)) again |= rows & (0u - rows);
        else if (there && lane < 16) *dst = make_uint4(w[0], w[1], w[2], w[3]);
    }
    return again;
}

constexpr int kAFirst = 4;                     // first softmax warp: TMA, MMA and search warp before them, one idle
constexpr int kAItems = 2;                     // items whose tiles are in shared memory
// The reference maximum of a row moves only when it is exceeded by a factor of 2^8: until then the weights are
// at most 256, well inside either type, and the accumulator is not rescaled.  It is a whole number at or below a
// maximum of the row: the row's largest weight is at least 1, and what fp16 rounds off the smallest ones at most
// 2^-25 of it.
constexpr float kARescale = 8.0f;

// CTAs of one tile, several to an SM, so that the many short steps of short sequences (loads, products,
// weights, stores) of one run while another's wait; and for long sequences CTAs of two tiles that share
// K and V and take turns, one's products running while the other's weights are computed.
template <int DP_, int kTiles_>
struct AttnCfg {
    static constexpr int DP = DP_, kTiles = kTiles_;              // columns of a head, tiles
    static constexpr int kCtas = kTiles == 2 ? 1 : DP == 128 ? 2 : 4;        // per SM
    static constexpr int kThreads = 32 * (kAFirst + 4 * kTiles);
    static constexpr int kN = kTiles == 2 ? 128 : 64;             // keys per block
    static constexpr int kHalves = kN / 64;                       // a block's weights are announced 64 at a time
    static constexpr bool kSteps = kTiles == 1;                   // a row's scores are held 32 at a time, not a block's
    static constexpr int kTileQ = kAM * DP * 2;                   // bytes of a Q tile
    static constexpr int kTileK = kN * DP * 2;                    // bytes of a K or a V block
    static constexpr int kStages = 2;                             // K blocks, and V blocks, in flight
    static constexpr int kSmem = 1024 + kTiles * kTileQ + 2 * kStages * kTileK + 1024;
    static constexpr uint32_t kO = kTiles * kN;                   // first accumulator column: S and P lie before
    static constexpr uint32_t kCols = 512 / kCtas;                // tensor-memory columns: a power of two
    static_assert(kO + kTiles * DP <= kCols, "tensor memory");
    // The launch's registers, dealt out anew: a softmax thread holds its row of scores.
    static constexpr int kRegs = kTiles == 2 ? 168 : DP == 128 ? 128 : 64;
    static constexpr int kRegsFew = kTiles == 2 ? 88 : DP == 128 ? 80 : 40;
    static constexpr int kRegsMany = kTiles == 2 ? 208 : DP == 128 ? 176 : 88;
    // rows at a time, and loads ahead, that attn_rows has the registers for
    static constexpr int kAgain = kTiles == 2 || DP == 128 ? 4 : 2, kAgainAhead = kAgain == 4 ? 8 : 2;
    static_assert(128 * kRegsFew + (kThreads - 128) * kRegsMany <= kThreads * kRegs, "more registers than the launch holds");
};

struct AttnMaps {
    CUtensorMap q, k, v;
};

// Bounded wait: 2 s, not counting the time that a warp of the CTA spends in attn_odd_rows and attn_rows (abort[1]:
// how many do), or until another role gave up (abort[0]).  In few instructions: the roles' code shares the
// instruction cache, and this is in it some twenty times.
__device__ __forceinline__ bool attn_wait(uint64_t* m, uint32_t parity, volatile int* abort) {
    if (tc::mbar_try_wait_hint(m, parity, tc::kWaitHintNs)) return true;
    uint32_t since, now;
    asm volatile("mov.u32 %0, %%globaltimer_lo;" : "=r"(since));
    for (uint32_t i = 0; i < (1u << 30); ++i) {
        if (tc::mbar_try_wait_hint(m, parity, tc::kWaitHintNs)) return true;
        if (abort[0]) return false;
        asm volatile("mov.u32 %0, %%globaltimer_lo;" : "=r"(now));
        if (abort[1]) since = now;
        if (now - since > (uint32_t)tc::kWaitDeadlineNs) break;
    }
    abort[0] = 1;
    return false;
}

// What the roles hand one another, behind the tiles in shared memory.
template <class Cfg>
struct AttnShared {
    static constexpr int kTiles = Cfg::kTiles, kStages = Cfg::kStages;
    AttnTile tile[kAItems][kTiles];
    uint4 answer;                            // to a request for the next item
    int head[kAItems], group[kAItems];       // query and key head; head < 0: no more items
    uint64_t kfull[kStages], kempty[kStages], vfull[kStages], vempty[kStages];
    uint64_t qfull, qempty;
    uint64_t ifull[kAItems], iempty[kAItems];
    uint64_t sfull[kTiles];                  // scores ready (MMA -> softmax)
    uint64_t pready[kTiles][Cfg::kHalves];       // weights written (softmax -> MMA)
    uint64_t odone[kTiles];                  // product with V done
    uint64_t drain, taken;
    uint32_t tmem;
    int abort[2];                            // given up; warps that mend rows
};

// The blocks of an item: blocks 0 .. n - 1 from key kv0 on, tile t takes [jb[t], je[t]) of them.
template <class Cfg>
struct AttnBlocks {
    int head = -1, group, kv0, n = 0, jb[Cfg::kTiles], je[Cfg::kTiles];
    __device__ __forceinline__ void get(const AttnShared<Cfg>* sh, int r) {
        head = sh->head[r];
        group = sh->group[r];
        kv0 = 0x7FFFFFFF;
        n = 0;
#pragma unroll
        for (int t = 0; t < Cfg::kTiles; ++t)
            if (sh->tile[r][t].rows > 0) kv0 = min(kv0, sh->tile[r][t].lo);
#pragma unroll
        for (int t = 0; t < Cfg::kTiles; ++t) {
            const bool any = sh->tile[r][t].rows > 0;
            jb[t] = any ? (unsigned)(sh->tile[r][t].lo - kv0) / Cfg::kN : 0;
            je[t] = any ? (unsigned)(sh->tile[r][t].hi - kv0 + Cfg::kN - 1) / Cfg::kN : 0;
            n = max(n, je[t]);
        }
    }
};

// A walk of a thread or a whole warp over the blocks of its CTA's items; gives the items' records back
// behind itself (by the lane with `lead` set).
template <class Cfg>
struct AttnWalk {
    AttnBlocks<Cfg> b;
    int rec = -1, j = 0;
    bool lead = true;
    // On to the next block; 1: there is one, 0: no more, -1: gave up waiting.
    __device__ __forceinline__ int next(AttnShared<Cfg>* sh) {
        if (j + 1 < b.n) {
            ++j;
            return 1;
        }
        if (rec >= 0 && lead) tc::mbar_arrive(&sh->iempty[rec % kAItems]);
        ++rec;
        if (!attn_wait(&sh->ifull[rec % kAItems], (rec / kAItems) & 1, sh->abort)) return -1;
        b.get(sh, rec % kAItems);
        j = 0;
        return b.head >= 0;
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
// A pair of 16-bit values added to two fp32 sums.
template <typename T>
__device__ __forceinline__ void add_pair(uint32_t w, float& a, float& b) {
    if constexpr (std::is_same_v<T, __half>)
        asm("{.reg .b16 x, y;\n mov.b32 {x, y}, %2;\n add.rn.f32.f16 %0, x, %0;\n add.rn.f32.f16 %1, y, %1;\n}"
            : "+f"(a), "+f"(b) : "r"(w));
    else
        asm("{.reg .b16 x, y;\n mov.b32 {x, y}, %2;\n add.rn.f32.bf16 %0, x, %0;\n add.rn.f32.bf16 %1, y, %1;\n}"
            : "+f"(a), "+f"(b) : "r"(w));
}
// w = 2^(s scale + ref) of 32 scores, rounded and packed in pairs; returns their sum.  Summing the rounded weights
// (kRounded) makes the division take out the rounding of a weight that dominates its row: a row of one key is that
// key's v exactly, and the error of 8 to 64 keys is 1.25 to 1.37 times that of the output's own rounding
// instead of 1.42.  It costs one more instruction per pair (1024 passages 193 -> 195 us).  Blocks of 128 keys that all
// rows see sum the weights as they come: rounded, 16384 tokens 1,040 -> 1,070 us, 12 prompts 850 -> 935.
template <typename T, bool kRounded>
__device__ __forceinline__ float attn_weights(const float* s, uint64_t scale, uint64_t ref, uint32_t* w) {
    float sum[4] = {};
    uint64_t sum2[2] = {0ull, 0ull};
#pragma unroll
    for (int q = 0; q < 16; ++q) {
        float x, y;
        unpack2(fma2(pack2(s[2 * q], s[2 * q + 1]), scale, ref), x, y);
        x = ex2(x);
        y = ex2(y);
        const typename Pair16<T>::type xy = Pair16<T>::down(x, y);
        w[q] = *reinterpret_cast<const uint32_t*>(&xy);
        if constexpr (kRounded) add_pair<T>(w[q], sum[q & 1], sum[2 + (q & 1)]);
        else sum2[q & 1] = add2(sum2[q & 1], pack2(x, y));
    }
    if constexpr (!kRounded) unpack2(add2(sum2[0], sum2[1]), sum[0], sum[1]);
    return (sum[0] + sum[1]) + (sum[2] + sum[3]);
}

template <typename T, class Cfg>
__global__ void __launch_bounds__(Cfg::kThreads, Cfg::kCtas)
packed_attn_mma(const __grid_constant__ AttnMaps maps, const __grid_constant__ AttnParams p) {
    constexpr int S = Cfg::kStages, N = Cfg::kN, kTiles = Cfg::kTiles, DP = Cfg::DP;
    extern __shared__ uint8_t attn_raw[];
    uint8_t* sm = (uint8_t*)(((uintptr_t)attn_raw + 1023) & ~(uintptr_t)1023);
    uint8_t* sQ = sm;
    uint8_t* sK = sm + kTiles * Cfg::kTileQ;
    uint8_t* sV = sK + S * Cfg::kTileK;
    AttnShared<Cfg>* sh = reinterpret_cast<AttnShared<Cfg>*>(sV + S * Cfg::kTileK);
    static_assert(sizeof(AttnShared<Cfg>) <= 1024, "shared memory of the roles");
    volatile int* abort = sh->abort;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int s = 0; s < S; ++s) {
            tc::mbar_init(&sh->kfull[s], 1);
            tc::mbar_init(&sh->vfull[s], 1);
            tc::mbar_init(&sh->kempty[s], 1);
            tc::mbar_init(&sh->vempty[s], 1);
        }
        tc::mbar_init(&sh->qfull, 1);
        tc::mbar_init(&sh->qempty, 1);
        for (int r = 0; r < kAItems; ++r) {
            tc::mbar_init(&sh->ifull[r], 1);
            tc::mbar_init(&sh->iempty[r], 2 + 4 * kTiles);        // TMA, MMA and softmax warps
        }
        for (int t = 0; t < kTiles; ++t) {
            tc::mbar_init(&sh->sfull[t], 1);
            for (int x = 0; x < Cfg::kHalves; ++x) tc::mbar_init(&sh->pready[t][x], 4);
            tc::mbar_init(&sh->odone[t], 1);
        }
        tc::mbar_init(&sh->drain, 1);
        tc::mbar_init(&sh->taken, 1);
        sh->abort[0] = sh->abort[1] = 0;
        tc::mbar_fence_init();
    }
    if (warp == 1) {
        tc::tmem_alloc(&sh->tmem, Cfg::kCols);
        tc::tmem_relinquish();
    }
    tc::fence_before();
    __syncthreads();
    tc::fence_after();
    const uint32_t tbase = sh->tmem;
    bool failed = false;
    pdl_wait_then_release();

    if (warp < kAFirst) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(Cfg::kRegsFew));
        if (warp == 0 && lane == 0) {
            // -------------------------------------------------------- TMA producer
            AttnWalk<Cfg> walk;
            int n = 0, nq = 0;                                    // blocks and items
            auto slot = [&](uint64_t* full, uint64_t* empty) {
                if (n >= S && !attn_wait(empty + n % S, (n / S - 1) & 1, abort)) return false;
                tc::mbar_arrive_expect_tx(full + n % S, Cfg::kTileK);
                return true;
            };
            auto load = [&](const CUtensorMap* map, uint8_t* ring, uint64_t* full) {
                for (int c = 0; c < DP / 64; ++c)
                    tc::tma_load_3d(ring + (n % S) * Cfg::kTileK + c * N * 128, map, 64 * c, walk.b.group,
                                    walk.b.kv0 + walk.j * N, full + n % S);
            };
            for (;; ++n) {
                const int there = walk.next(sh);
                if (there <= 0) {
                    failed = there < 0;
                    break;
                }
                if (!slot(sh->kfull, sh->kempty)) {
                    failed = true;
                    break;
                }
                load(&maps.k, sK, sh->kfull);
                if (walk.j == 0) {                                // a new item: its Q
                    if (nq > 0 && !attn_wait(&sh->qempty, (nq - 1) & 1, abort)) {
                        failed = true;
                        break;
                    }
                    // rows of a tile behind its sequence are another's: read along and not used
                    tc::mbar_arrive_expect_tx(&sh->qfull, kTiles * Cfg::kTileQ);
                    for (int t = 0; t < kTiles; ++t)
                        for (int c = 0; c < DP / 64; ++c)
                            tc::tma_load_3d(sQ + t * Cfg::kTileQ + c * kAM * 128, &maps.q, 64 * c, walk.b.head,
                                            sh->tile[walk.rec % kAItems][t].row0, &sh->qfull);
                    ++nq;
                }
                if (!slot(sh->vfull, sh->vempty)) {
                    failed = true;
                    break;
                }
                load(&maps.v, sV, sh->vfull);
            }
            if (failed) {                                         // copies in flight end before the CTA does
                if (nq > 0) (void)tc::mbar_wait_bounded(&sh->qfull, (nq - 1) & 1, 1u << 16);
#pragma unroll 1
                for (int i = max(0, n - S); i <= n; ++i) {
                    (void)tc::mbar_wait_bounded(&sh->kfull[i % S], (i / S) & 1, 1u << 16);
                    (void)tc::mbar_wait_bounded(&sh->vfull[i % S], (i / S) & 1, 1u << 16);
                }
            }
        } else if (warp == 1) {
            // -------------------------------------------------------- MMA issuer, one lane of a warp in step
            constexpr uint32_t idS = tc::idesc_f16_f32(kAM, N) | idesc_type<T>();
            constexpr uint32_t idO = tc::idesc_f16_f32(kAM, DP) | idesc_type<T>() | kIdescBMn;
            const uint32_t lead = tc::elect_one();
            AttnWalk<Cfg> walk;                                    // of the scores; the products with V are
            int vj = 0, vjb[kTiles] = {}, vje[kTiles] = {};                 // one block behind it, at vj
            walk.lead = lead != 0;
            uint32_t np[kTiles] = {};                             // products of each tile
            int nk = 0, nv = 0, nq = 0;
            auto scores = [&](int t) {
                if (walk.j < walk.b.jb[t] || walk.j >= walk.b.je[t]) return;
                // S takes the columns of the weights that the product just issued reads: the tensor pipe
                // runs them one behind the other
                const uint32_t q = tc::smem_u32(sQ + t * Cfg::kTileQ), k = tc::smem_u32(sK + (nk % S) * Cfg::kTileK);
#pragma unroll
                for (int c = 0; c < DP / 16; ++c)
                    tc::mma_ss_if(lead, tbase + t * N, tc::sw128_kmajor_desc(q + (c >> 2) * kAM * 128 + (c & 3) * 32),
                                  tc::sw128_kmajor_desc(k + (c >> 2) * N * 128 + (c & 3) * 32), idS, c > 0);
                tc::mma_commit_if(lead, &sh->sfull[t]);
            };
            auto product = [&](int t) {
                if (vj < vjb[t] || vj >= vje[t]) return true;
                const uint32_t v = tc::smem_u32(sV + (nv % S) * Cfg::kTileK);
                const bool begun = vj > vjb[t];
#pragma unroll
                for (int x = 0; x < Cfg::kHalves; ++x) {
                    const bool ok = attn_wait(&sh->pready[t][x], np[t] & 1, abort);
                    if (!__all_sync(0xFFFFFFFFu, ok)) return false;
                    tc::fence_after();
#pragma unroll
                    for (int c = 4 * x; c < 4 * x + 4; ++c)
                        tc::mma_ts_if(lead, tbase + Cfg::kO + t * DP, tbase + t * N + 8 * c,
                                      tc::sw128_mnmajor_desc(v + 2048 * c, N * 128), idO, begun || c > 0);
                }
                ++np[t];
                if (vj == vje[t] - 1) tc::mma_commit_if(lead, &sh->odone[t]);
                return true;
            };
            auto k_arrived = [&] {
                const bool ok = attn_wait(&sh->kfull[nk % S], (nk / S) & 1, abort) &&
                                (walk.j != 0 || attn_wait(&sh->qfull, nq & 1, abort));
                if (!__all_sync(0xFFFFFFFFu, ok)) return false;
                tc::fence_after();
                return true;
            };
            // Within an item two tiles take turns, each one's scores behind its product: its products run
            // while the other's weights are computed.  At an item's end, and with one tile, all products
            // come first: the next item's record, K and Q may still be on their way.
            bool first = true;
            for (;;) {
                const bool follow = kTiles > 1 && !first && walk.j + 1 < walk.b.n;
                if (!first) {
                    vj = walk.j;
#pragma unroll
                    for (int t = 0; t < kTiles; ++t) {
                        vjb[t] = walk.b.jb[t];
                        vje[t] = walk.b.je[t];
                    }
                    if (follow) ++walk.j;
                    const bool ok = attn_wait(&sh->vfull[nv % S], (nv / S) & 1, abort);
                    failed = !__all_sync(0xFFFFFFFFu, ok) || (follow && !k_arrived());
                    if (failed) break;
                    tc::fence_after();
#pragma unroll
                    for (int t = 0; t < kTiles; ++t) {
                        failed = failed || !product(t);
                        if (kTiles > 1 && !failed && follow) scores(t);
                    }
                    if (failed) break;
                    tc::mma_commit_if(lead, &sh->vempty[nv % S]);
                    ++nv;
                }
                first = false;
                if (!follow) {
                    const int more = walk.next(sh);
                    failed = !__all_sync(0xFFFFFFFFu, more >= 0) || (more > 0 && !k_arrived());
                    if (failed || more == 0) break;
#pragma unroll
                    for (int t = 0; t < kTiles; ++t) scores(t);
                }
                tc::mma_commit_if(lead, &sh->kempty[nk % S]);
                ++nk;
                if (walk.j == walk.b.n - 1) {
                    tc::mma_commit_if(lead, &sh->qempty);
                    ++nq;
                }
            }
            if (failed) {                                         // the last products read shared memory
                tc::mma_commit_if(lead, &sh->drain);
                (void)tc::mbar_wait_bounded(&sh->drain, 0, 1u << 16);
            }
        } else if (warp == 2) {
            // -------------------------------------------------------- the coming items
            // The grid has a CTA for each item: heads fastest, and the last rows first, since the tiles of a
            // causal sequence grow along it.  The CTAs that are running take over those that are not, one
            // at a time, so that none is left with more than its share of long ones.  Items without a row
            // are passed over.
            const uint32_t heads = p.heads, per = heads / p.kv_heads, groups = p.items / heads;
            uint32_t rec = 0, asked = 0, group = 0xFFFFFFFFu;
            AttnTile tile[kTiles];
            bool any = false;
            int64_t item = blockIdx.x;
            for (;;) {
                const bool end = item < 0;
                if (!end) {
                    if (lane == 0) {
                        tc::fence_proxy_async();                  // behind the reading of the answer before
                        tc::take_ask(&sh->answer, &sh->taken);
                    }
                    // an entry of the table for each lane and item: that is all of them, which bisection
                    // alone does not see
                    const int64_t e = item * 32 + lane;
                    if (e < p.B) {
                        const int begin = __ldg(p.cu + e), stop = __ldg(p.cu + e + 1);
                        if (begin < 0 || stop < begin || stop > p.T) atomicExch(p.err, 6);
                    }
                    const uint32_t g = groups - 1 - (uint32_t)item / heads;
                    if (g != group) {
                        group = g;
                        any = false;
#pragma unroll
                        for (int t = 0; t < kTiles; ++t) {
                            tile[t] = attn_tile(p, (int64_t)g * kTiles + t, lane);
                            any = any || tile[t].rows > 0;
                        }
                    }
                }
                if (end || any) {
                    const uint32_t r = rec % kAItems;
                    const bool ok = rec < (uint32_t)kAItems || attn_wait(&sh->iempty[r], (rec / kAItems - 1) & 1, abort);
                    failed = !__all_sync(0xFFFFFFFFu, ok);
                    if (lane == 0 && !failed) {
#pragma unroll
                        for (int t = 0; t < kTiles; ++t) sh->tile[r][t] = end ? AttnTile{0, 0, 0, 0} : tile[t];
                        sh->head[r] = end ? -1 : (int)((uint32_t)item % heads);
                        sh->group[r] = end ? 0 : (int)((uint32_t)item % heads / per);
                        tc::mbar_arrive(&sh->ifull[r]);
                    }
                    ++rec;
                }
                if (end) break;
                // also behind a failure: the answer must have come before the CTA goes
                const bool ok = attn_wait(&sh->taken, asked++ & 1, abort) ||
                                tc::mbar_wait_bounded(&sh->taken, (asked - 1) & 1, 1u << 20);
                failed = failed || !__all_sync(0xFFFFFFFFu, ok);
                if (failed) break;
                item = tc::take_answer(&sh->answer);
                __syncwarp();
            }
        }
    } else {
        // ------------------------------------------------------------ softmax, a thread per row
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(Cfg::kRegsMany));
        const int tile = (warp - kAFirst) >> 2, quad = warp & 3;
        const uint32_t lanes = (uint32_t)(quad * 32) << 16;
        const uint32_t ts = tbase + lanes + (uint32_t)(tile * N), to = tbase + lanes + Cfg::kO + (uint32_t)(tile * DP);
        const float scale2 = p.scale * 1.4426950408889634f;       // weights are powers of two
        const uint64_t scale22 = pack2(scale2, scale2);
        uint32_t blk = 0, outs = 0;                               // blocks and items of this tile
        for (int rec = 0; !failed; ++rec) {
            const int r = rec % kAItems;
            bool ok = attn_wait(&sh->ifull[r], (rec / kAItems) & 1, abort);
            if (!__all_sync(0xFFFFFFFFu, ok)) {
                failed = true;
                break;
            }
            AttnBlocks<Cfg> b;
            b.get(sh, r);
            const AttnTile own = sh->tile[r][tile];
            __syncwarp();
            if (lane == 0) tc::mbar_arrive(&sh->iempty[r]);
            if (b.head < 0) break;
            if (own.rows == 0) continue;
            const int in_tile = quad * 32 + lane, row = own.row0 + in_tile;
            const bool mine = in_tile < own.rows, idle = quad * 32 >= own.rows;      // idle: no row of the warp
            const int hi = p.causal ? min(row + 1, own.hi) : own.hi;
            const int wlast = p.causal ? min(own.row0 + quad * 32 + 32, own.hi) : own.hi;      // keys some row sees
            const int wall = p.causal ? min(own.row0 + quad * 32 + 1, own.hi) : own.hi;        // keys all rows see
            float m = -INFINITY, l = 0.f;
            const int b0 = tile == 0 ? b.jb[0] : b.jb[kTiles - 1], b1 = tile == 0 ? b.je[0] : b.je[kTiles - 1];
            for (int j = b0; j < b1; ++j, ++blk) {
                ok = attn_wait(&sh->sfull[tile], blk & 1, abort);
                if (!__all_sync(0xFFFFFFFFu, ok)) {
                    failed = true;
                    break;
                }
                tc::fence_after();
                const int first = b.kv0 + j * N;
                // 32-key steps: all rows see all of it, some see some of it, or none sees any (left out)
                auto seen = [&](int c) { return !idle && first + 32 * c + 32 > own.lo && first + 32 * c < wlast; };
                auto load = [&](int c, float* v) {
                    tc::ld32x32(ts + 32 * c, *reinterpret_cast<uint32_t(*)[32]>(v));
                    tc::wait_ld();
                    if (first + 32 * c < own.lo || first + 32 * c + 32 > wall) {
                        const uint32_t see = low_bits(hi - first - 32 * c) & ~low_bits(own.lo - first - 32 * c);
#pragma unroll
                        for (int q = 0; q < 32; ++q) v[q] = (see >> q) & 1u ? v[q] : -INFINITY;
                    }
                };
                auto maxima = [&](const float* v, float (&mx)[4]) {
#pragma unroll
                    for (int q = 0; q < 32; q += 8)
#pragma unroll
                        for (int e = 0; e < 4; ++e) mx[e] = max3(mx[e], v[q + e], v[q + e + 4]);
                };
                // Moves the row's reference maximum where scores pass it by too much; returns what earlier
                // weights are to be multiplied with.  The reference is a whole number: the factor is a
                // power of two and rounds nothing.
                auto refer = [&](const float (&mx)[4]) {
                    const float bm = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * scale2;
                    float alpha = 1.0f;
                    if (__any_sync(0xFFFFFFFFu, bm > m + kARescale)) {
                        const float mn = fmaxf(m, floorf(bm));
                        alpha = m == -INFINITY ? 0.f : ex2(m - mn);
                        l *= alpha;
                        m = mn;
                        if (j > b0) {   // these scores came behind the last product: the accumulator is at rest
#pragma unroll 1
                            for (int c = 0; c < DP / 16; ++c) {
                                uint32_t r16[16];
                                tc::ld32x16(to + 16 * c, r16);
                                tc::wait_ld();
#pragma unroll
                                for (int q = 0; q < 16; ++q) r16[q] = __float_as_uint(__uint_as_float(r16[q]) * alpha);
                                tc::st32x16(to + 16 * c, r16);
                            }
                            tc::wait_st();      // the next step of 32 keys may read it again, to move it once more
                        }
                    }
                    return alpha;
                };
                auto announce = [&](int x) {
                    tc::wait_st();
                    tc::fence_before();
                    __syncwarp();
                    if (lane == 0) tc::mbar_arrive(&sh->pready[tile][x]);
                };
                float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
                if constexpr (Cfg::kSteps) {
                    // 32 keys at a time, each step with a maximum of its own
                    uint32_t w[N / 2] = {};
#pragma unroll
                    for (int c = 0; c < N / 32; ++c) {
                        if (seen(c)) {
                            float s[32];
                            load(c, s);
                            mx[0] = mx[1] = mx[2] = mx[3] = -INFINITY;
                            maxima(s, mx);
                            const float alpha = refer(mx);
                            if (c > 0 && __any_sync(0xFFFFFFFFu, alpha != 1.0f)) {
#pragma unroll
                                for (int q = 0; q < 16 * c; ++q) {
                                    const float2 f = Pair16<T>::up(*reinterpret_cast<typename Pair16<T>::type*>(w + q));
                                    const typename Pair16<T>::type h = Pair16<T>::down(f.x * alpha, f.y * alpha);
                                    w[q] = *reinterpret_cast<const uint32_t*>(&h);
                                }
                            }
                            const float ref = m == -INFINITY ? 0.f : m;
                            l += attn_weights<T, true>(s, scale22, pack2(-ref, -ref), w + 16 * c);
                        }
                    }
                    tc::st32x32(ts, w);
                    announce(0);
                } else {
                    float s[N];
                    const bool all = !idle && first >= own.lo && first + N <= wall;
                    if (all) {
#pragma unroll
                        for (int c = 0; c < N / 32; ++c)
                            tc::ld32x32(ts + 32 * c, *reinterpret_cast<uint32_t(*)[32]>(s + 32 * c));
                        tc::wait_ld();
                    } else {
#pragma unroll
                        for (int c = 0; c < N / 32; ++c) {
                            if (seen(c)) {
                                load(c, s + 32 * c);
                            } else {
#pragma unroll
                                for (int q = 0; q < 32; ++q) s[32 * c + q] = -INFINITY;
                            }
                        }
                    }
#pragma unroll
                    for (int c = 0; c < N / 32; ++c) maxima(s + 32 * c, mx);
                    (void)refer(mx);
                    const float ref = m == -INFINITY ? 0.f : m;
                    const uint64_t ref2 = pack2(-ref, -ref);
                    if (all) {                                    // straight code: no step waits for a branch
#pragma unroll
                        for (int c = 0; c < N / 32; ++c) {
                            uint32_t w[16];
                            l += attn_weights<T, false>(s + 32 * c, scale22, ref2, w);
                            tc::st32x16(ts + 16 * c, w);
                            if (c & 1) announce(c / 2);
                        }
                    } else {
#pragma unroll
                        for (int c = 0; c < N / 32; ++c) {
                            uint32_t w[16] = {};
                            if (seen(c)) l += attn_weights<T, true>(s + 32 * c, scale22, ref2, w);
                            tc::st32x16(ts + 16 * c, w);
                            if (c & 1) announce(c / 2);
                        }
                    }
                }
            }
            if (failed) break;
            ok = attn_wait(&sh->odone[tile], outs++ & 1, abort);
            if (!__all_sync(0xFFFFFFFFu, ok)) {
                failed = true;
                break;
            }
            if (idle) continue;
            tc::fence_after();
            // The next item's weights are announced behind these loads, so that its first product finds
            // the accumulator read.
            const float inv = 1.0f / l;
            T* dst = static_cast<T*>(p.out) + row * p.out_stride + (int64_t)b.head * p.dim;
            // whole sectors where the rows allow it: half as many stores, each to 32 rows
            const bool sectors = ((uintptr_t)p.out & 31) == 0 && p.out_stride % 16 == 0 && p.dim % 16 == 0;
            bool bad = false;
#pragma unroll 1
            for (int c = 0; c < DP; c += 32) {
                float o[32], odd = 0.f;
                tc::ld32x32(to + c, *reinterpret_cast<uint32_t(*)[32]>(o));
                tc::wait_ld();
#pragma unroll
                for (int q = 0; q < 32; ++q) {
                    o[q] *= inv;
                    odd = fmaf(o[q], 0.f, odd);                   // NaN as soon as one is not finite
                }
                bad = bad || (mine && !(odd == 0.f));
                if (mine && sectors) {
#pragma unroll
                    for (int q = 0; q < 32; q += 16)
                        if (c + q < p.dim)
                            store32(dst + c + q, down8<T>(*reinterpret_cast<float(*)[8]>(o + q)),
                                    down8<T>(*reinterpret_cast<float(*)[8]>(o + q + 8)));
                } else if (mine) {
#pragma unroll
                    for (int q = 0; q < 32; q += 8)
                        if (c + q < p.dim) *reinterpret_cast<uint4*>(dst + c + q) = down8<T>(*reinterpret_cast<float(*)[8]>(o + q));
                }
            }
            __syncwarp();                                         // the rows' values above come before what mends them
            // A sum of weights that is NaN or 0 (a score is NaN or infinite, or all are -inf) makes all of the row NaN
            // by the formula, as it is already.
            unsigned left = __ballot_sync(0xFFFFFFFFu, bad && inv < INFINITY);
            if (left) {
                if (lane == 0) atomicAdd(&sh->abort[1], 1);
                left = attn_odd_rows<T>(p, b.head, row - lane, left, own.lo, hi);
                while (left)
                    left = attn_rows<T, Cfg::kAgain, Cfg::kAgainAhead, 2 * Cfg::kAgainAhead>(p, b.head, row - lane, left, own.lo, hi);
                if (lane == 0) atomicAdd(&sh->abort[1], -1);
            }
        }
    }
    if (failed) atomicExch(p.err, 1);
    tc::fence_before();
    __syncthreads();
    if (warp == 1) {
        tc::fence_after();
        tc::tmem_dealloc(tbase, Cfg::kCols);
    }
}

template <typename T, class Cfg>
int attn_launch(int dtype, AttnParams p, cudaStream_t stream) {
    static std::atomic<uint64_t> done{0};
    int rc = enc_allow_smem(packed_attn_mma<T, Cfg>, Cfg::kSmem, done);
    if (rc) return rc;
    AttnMaps m;
    if ((rc = enc_map_heads(&m.q, dtype, p.q, p.T, p.heads, p.dim, p.q_stride, kAM)) ||
        (rc = enc_map_heads(&m.k, dtype, p.k, p.T, p.kv_heads, p.dim, p.k_stride, Cfg::kN)) ||
        (rc = enc_map_heads(&m.v, dtype, p.v, p.T, p.kv_heads, p.dim, p.v_stride, Cfg::kN)))
        return rc;
    const int64_t groups = ceil_div(p.T / kAM + (int64_t)p.B, Cfg::kTiles);
    if (groups * p.heads > 0x7FFFFFFF) return fail(RAGRT_ERR_CAPACITY, "too many rows x heads");
    p.items = (int)(groups * p.heads);
    return enc_launch(packed_attn_mma<T, Cfg>, dim3((unsigned)p.items), dim3(Cfg::kThreads), Cfg::kSmem, stream, m, p);
}

template <typename T>
int attn_launch_sized(int dtype, const AttnParams& p, cudaStream_t stream) {
    // Two tiles where a row sees many keys: as far as the host knows, the mean length (half of it, causal).
    // 65536 rows of 16 heads, one tile / two: heads of 128, full, length 100 226 / 345 us, 512 536 / 543, 768
    // 733 / 640, 2048 1761 / 1214; causal, 1024 596 / 619, 2048 1026 / 828; heads of 64, full, 100 151 / 321,
    // 1024 602 / 641, 2048 1114 / 1042; causal, 2048 668 / 729, 8192 (half the rows) 1124 / 881.
    const bool wide = p.dim > 64, two = p.T / p.B / (p.causal ? 2 : 1) >= (wide ? 544 : 1536);
    if (wide) return two ? attn_launch<T, AttnCfg<128, 2>>(dtype, p, stream) : attn_launch<T, AttnCfg<128, 1>>(dtype, p, stream);
    return two ? attn_launch<T, AttnCfg<64, 2>>(dtype, p, stream) : attn_launch<T, AttnCfg<64, 1>>(dtype, p, stream);
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
    // the kernel's scores are powers of two: scale times log2 e is finite too
    RAGRT_REQUIRE(scale > 0.f && scale <= 2.3e38f, "scale must be positive and at most 2.3e38");
    if (T == 0 || B == 0) return RAGRT_OK;
    RAGRT_REQUIRE(d_q && d_k && d_v && d_cu_seqlens && d_out, "null argument");
    RAGRT_REQUIRE((((uintptr_t)d_q | (uintptr_t)d_k | (uintptr_t)d_v | (uintptr_t)d_out) & 15) == 0 &&
                      ((uintptr_t)d_cu_seqlens & 3) == 0,
                  "packed_attention operands must be 16-byte aligned");
    int* err = device_error_flag();
    if (!err) return fail(RAGRT_ERR_CUDA, "device error flag unavailable");
    AttnParams p{d_q, d_k, d_v, d_out, d_cu_seqlens, q_stride, k_stride, v_stride, out_stride, T, B, heads, kv_heads,
                 head_dim, causal != 0, 0, scale, err};
    cudaStream_t stream = (cudaStream_t)stream_;
    return dtype == RAGRT_BF16 ? attn_launch_sized<__nv_bfloat16>(dtype, p, stream) : attn_launch_sized<__half>(dtype, p, stream);
}
