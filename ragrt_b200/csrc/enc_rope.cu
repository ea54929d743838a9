// enc_rope.cu -- per-head RMS norm of queries and keys with the rotary positions in the same pass.
//
//   n_i = x_i / sqrt(mean_j x_j^2 + eps) * w_i            (no weight: n = x)
//   y_i = n_i cos - n_i' sin,  y_i' = n_i' cos + n_i sin  for the pairs (i, i') of the first rot_dim
//         values, i' = i + rot_dim / 2 or (interleaved) i' = i + 1; the values behind them stay n
//
// The pass is bound by memory (each value is read once and written once).  A lane holds two 8-value
// chunks of a head that rotate with one another, so that a head is ceil(dim / 16) lanes, the
// rotation needs no exchange, the mean a few shuffles, and a lane's cos / sin stay in registers
// while its warp walks the heads of one token.  Measured: 102,411 tokens of 24 heads of 64 (32 values
// turned) 127 us in a burst, 137 in a long run, 4.6 TB/s; 32,768 tokens of 40 heads of 128 133 us, 5.2 TB/s.
// What is left of the way to a copy's 6.5 is latency: 64 to 66 % of the issue slots are used (about 230
// instructions per warp for 512 values) and 53 to 60 % of the memory's rate, by 5.5 warps of a scheduler's 16, each
// of which loads, computes, stores and ends with nothing of the next token in flight.
#include <algorithm>

#include "enc_common.cuh"

namespace ragrt {

namespace {

struct RopeParams {
    const void* q;
    const void* k;
    const void* qw;
    const void* kw;
    const float* cos;
    const float* sin;
    const void* pos;
    void* qo;
    void* ko;
    int64_t q_stride, k_stride, qo_stride, ko_stride;
    int T, heads, kv_heads, dim, rot, max_pos, pos64, interleaved, slabs;
    float eps;
    int* err;
};


constexpr int kRopeWarps = 2;                    // small CTAs: a place is free again as soon as two tokens are done

// 8 values of 16 bits <-> 4 fp32 pairs
template <typename T>
__device__ __forceinline__ void up8x2(const uint4& u, uint64_t (&f)[4]) {
    const typename Pair16<T>::type* h = reinterpret_cast<const typename Pair16<T>::type*>(&u);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 v = Pair16<T>::up(h[i]);
        f[i] = pack2(v.x, v.y);
    }
}
template <typename T>
__device__ __forceinline__ uint4 down8x2(const uint64_t (&f)[4]) {
    uint4 u;
    typename Pair16<T>::type* h = reinterpret_cast<typename Pair16<T>::type*>(&u);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        float a, b;
        unpack2(f[i], a, b);
        h[i] = Pair16<T>::down(a, b);
    }
    return u;
}
// A warp takes one token and one of `slabs` shares of its heads, kBatch of a lane's heads in flight at a
// time.
template <typename T, bool kNeighbours, int kBatch>
__global__ void __launch_bounds__(32 * kRopeWarps, 24 / kRopeWarps) enc_qk_norm_rope(const RopeParams p, const int group) {
    pdl_wait_then_release();
    const int64_t unit = ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) >> 5;
    if (unit >= (int64_t)p.T * p.slabs) return;
    const int64_t t = p.slabs == 1 ? unit : unit / p.slabs;
    const int slab = (int)(unit - t * p.slabs);
    const int lane = threadIdx.x & 31, l = lane & (group - 1), sub = lane / group, per = 32 / group;
    int64_t pos = p.pos64 ? static_cast<const int64_t*>(p.pos)[t] : (int64_t) static_cast<const int32_t*>(p.pos)[t];
    // the lane's two chunks: first value of each, and whether they are there
    const int pairs = p.rot / 16;
    const bool turn = l < pairs;
    int a, b;
    if (turn) {
        a = kNeighbours ? 16 * l : 8 * l;
        b = kNeighbours ? 16 * l + 8 : 8 * l + p.rot / 2;
    } else {
        a = p.rot + 16 * (l - pairs);
        b = a + 8;
    }
    const bool has_a = a < p.dim, has_b = b < p.dim;
    const T* q = static_cast<const T*>(p.q) + t * p.q_stride;
    const T* k = static_cast<const T*>(p.k) + t * p.k_stride - p.heads * p.dim;
    T* qo = static_cast<T*>(p.qo) + t * p.qo_stride;
    T* ko = static_cast<T*>(p.ko) + t * p.ko_stride - p.heads * p.dim;
    const int all = p.heads + p.kv_heads;
    const int rounds = (all + per - 1) / per;               // heads in steps of a warp's worth
    // of a token with a million heads the product passes 32 bits
    const int r0 = (int)((int64_t)rounds * slab / p.slabs), r1 = (int)((int64_t)rounds * (slab + 1) / p.slabs);
    const float inv_dim = 1.0f / (float)p.dim;
    const uint4 zero = make_uint4(0u, 0u, 0u, 0u);
    float c[8], s[8];
    for (int r = r0; r < r1; r += kBatch) {
        uint4 ua[kBatch], ub[kBatch];
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
            const int h = (r + i) * per + sub;
            const bool on = r + i < r1 && h < all;
            const T* src = (h < p.heads ? q : k) + h * p.dim;
            ua[i] = on && has_a ? __ldcs(reinterpret_cast<const uint4*>(src + a)) : zero;
            ub[i] = on && has_b ? __ldcs(reinterpret_cast<const uint4*>(src + b)) : zero;
        }
        if (r == r0) {                                      // the angles, behind the first heads' loads
            if (pos < 0 || pos >= p.max_pos) {
                if (lane == 0) atomicExch(p.err, 5);
                pos = 0;
            }
            if (turn) {
                const float4* cp = reinterpret_cast<const float4*>(p.cos + pos * (p.rot / 2) + 8 * l);
                const float4* sp = reinterpret_cast<const float4*>(p.sin + pos * (p.rot / 2) + 8 * l);
                *reinterpret_cast<float4*>(c) = __ldg(cp);
                *reinterpret_cast<float4*>(c + 4) = __ldg(cp + 1);
                *reinterpret_cast<float4*>(s) = __ldg(sp);
                *reinterpret_cast<float4*>(s + 4) = __ldg(sp + 1);
            }
        }
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
            const int h = (r + i) * per + sub;
            const bool on = r + i < r1 && h < all, is_q = h < p.heads;
            if (r + i >= r1) break;
            uint64_t x[4], y[4];
            up8x2<T>(ua[i], x);
            up8x2<T>(ub[i], y);
            const T* w = static_cast<const T*>(is_q ? p.qw : p.kw);
            uint64_t ss2 = 0ull;
#pragma unroll
            for (int e = 0; e < 4; ++e) ss2 = fma2(x[e], x[e], fma2(y[e], y[e], ss2));
            float ss, sb;
            unpack2(ss2, ss, sb);
            ss += sb;
            for (int o = group >> 1; o; o >>= 1) ss += __shfl_xor_sync(0xFFFFFFFFu, ss, o);
            if (w) {
                const float rstd = rsqrtf(ss * inv_dim + p.eps);
                const uint64_t rstd2 = pack2(rstd, rstd);
                uint64_t wa[4], wb[4];
                up8x2<T>(has_a ? __ldg(reinterpret_cast<const uint4*>(w + a)) : zero, wa);
                up8x2<T>(has_b ? __ldg(reinterpret_cast<const uint4*>(w + b)) : zero, wb);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    x[e] = mul2(mul2(x[e], rstd2), wa[e]);
                    y[e] = mul2(mul2(y[e], rstd2), wb[e]);
                }
            }
            if (turn) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    float x0, x1, y0, y1;
                    unpack2(x[e], x0, x1);
                    unpack2(y[e], y0, y1);
                    if (kNeighbours) {
                        x[e] = pack2(fmaf(x0, c[e], -x1 * s[e]), fmaf(x1, c[e], x0 * s[e]));
                        y[e] = pack2(fmaf(y0, c[e + 4], -y1 * s[e + 4]), fmaf(y1, c[e + 4], y0 * s[e + 4]));
                    } else {
                        x[e] = pack2(fmaf(x0, c[2 * e], -y0 * s[2 * e]), fmaf(x1, c[2 * e + 1], -y1 * s[2 * e + 1]));
                        y[e] = pack2(fmaf(y0, c[2 * e], x0 * s[2 * e]), fmaf(y1, c[2 * e + 1], x1 * s[2 * e + 1]));
                    }
                }
            }
            if (on) {
                T* dst = (is_q ? qo : ko) + h * p.dim;
                if (has_a) __stcs(reinterpret_cast<uint4*>(dst + a), down8x2<T>(x));
                if (has_b) __stcs(reinterpret_cast<uint4*>(dst + b), down8x2<T>(y));
            }
        }
    }
}

template <typename T, bool kNeighbours>
int rope_launch(const RopeParams& p, int group, int batch, cudaStream_t stream) {
    const int64_t blocks = ceil_div((int64_t)p.T * p.slabs, kRopeWarps);
    return batch == 3 ? enc_launch(enc_qk_norm_rope<T, kNeighbours, 3>, dim3((unsigned)blocks), dim3(32 * kRopeWarps), 0, stream, p, group)
                      : enc_launch(enc_qk_norm_rope<T, kNeighbours, 2>, dim3((unsigned)blocks), dim3(32 * kRopeWarps), 0, stream, p, group);
}

}  // namespace
}  // namespace ragrt

using namespace ragrt;

extern "C" int ragrt_enc_qk_norm_rope(const void* d_q, const void* d_k, const void* d_q_weight, const void* d_k_weight,
                                      const float* d_cos, const float* d_sin, const void* d_pos, int32_t pos_bytes,
                                      void* d_q_out, void* d_k_out, int32_t T, int32_t heads, int32_t kv_heads,
                                      int32_t head_dim, int32_t rot_dim, int32_t max_pos, int64_t q_stride,
                                      int64_t k_stride, int64_t q_out_stride, int64_t k_out_stride, float eps,
                                      int32_t interleaved, int32_t dtype, void* stream_) {
    RAGRT_REQUIRE(dtype == RAGRT_F16 || dtype == RAGRT_BF16, "dtype must be RAGRT_F16 or RAGRT_BF16; got %d",
                  (int)dtype);
    RAGRT_REQUIRE(T >= 0 && heads >= 1 && kv_heads >= 0, "T >= 0, heads >= 1, kv_heads >= 0 required");
    RAGRT_REQUIRE(head_dim >= 16 && head_dim <= 256 && head_dim % 8 == 0,
                  "enc_qk_norm_rope needs head_dim a multiple of 8 in [16, 256]; got %d", (int)head_dim);
    RAGRT_REQUIRE(rot_dim >= 16 && rot_dim <= head_dim && rot_dim % 16 == 0,
                  "rot_dim must be a multiple of 16 in [16, head_dim]; got %d", (int)rot_dim);
    RAGRT_REQUIRE(max_pos >= 1, "max_pos must be >= 1");
    RAGRT_REQUIRE(pos_bytes == 4 || pos_bytes == 8, "positions are 4 or 8 bytes wide; got %d", (int)pos_bytes);
    RAGRT_REQUIRE(heads <= (1 << 20) && kv_heads <= (1 << 20), "too many heads");
    const int64_t qw = (int64_t)heads * head_dim, kw = (int64_t)kv_heads * head_dim;
    RAGRT_REQUIRE(q_stride >= qw && q_out_stride >= qw && k_stride >= kw && k_out_stride >= kw &&
                      (q_stride | k_stride | q_out_stride | k_out_stride) % 8 == 0,
                  "row strides must hold all heads and be multiples of 8 elements");
    if (T == 0) return RAGRT_OK;
    RAGRT_REQUIRE(d_q && d_q_out && d_cos && d_sin && d_pos && (kv_heads == 0 || (d_k && d_k_out)), "null argument");
    RAGRT_REQUIRE((((uintptr_t)d_q | (uintptr_t)d_k | (uintptr_t)d_q_weight | (uintptr_t)d_k_weight |
                    (uintptr_t)d_cos | (uintptr_t)d_sin | (uintptr_t)d_q_out | (uintptr_t)d_k_out) & 15) == 0 &&
                      ((uintptr_t)d_pos & (uintptr_t)(pos_bytes - 1)) == 0,
                  "enc_qk_norm_rope operands must be 16-byte aligned");
    int* err = device_error_flag();
    if (!err) return fail(RAGRT_ERR_CUDA, "device error flag unavailable");
    int group = 1;
    while (group * 16 < head_dim) group *= 2;
    const int rounds = (int)ceil_div(heads + kv_heads, 32 / group);
    // Two or three steps of heads at a time, whichever leaves fewer of a warp's steps empty: 102411 tokens
    // of 24 heads of 64 (3 steps) take 135 us by three and 149 us by two, 32768 tokens of 40 heads of 128
    // (10 steps) 146 and 131 us.
    const int batch = ceil_div(rounds, 3) * 3 <= ceil_div(rounds, 2) * 2 ? 3 : 2;
    // Few tokens: a warp per batch of heads, so that they run side by side; many tokens: a warp per
    // token, which loads its angles once.
    const int warps = num_sms() * 16;
    const int slabs = (int)std::min<int64_t>(ceil_div(rounds, batch), std::max<int64_t>(1, warps / T));
    RAGRT_REQUIRE(ceil_div((int64_t)T * slabs, kRopeWarps) <= 0x7FFFFFFF, "too many tokens");
    RopeParams p{d_q, d_k, d_q_weight, d_k_weight, d_cos, d_sin, d_pos, d_q_out, d_k_out, q_stride, k_stride,
                 q_out_stride, k_out_stride, T, heads, kv_heads, head_dim, rot_dim, max_pos, pos_bytes == 8,
                 interleaved != 0, slabs, eps, err};
    cudaStream_t stream = (cudaStream_t)stream_;
    if (dtype == RAGRT_BF16)
        return p.interleaved ? rope_launch<__nv_bfloat16, true>(p, group, batch, stream)
                             : rope_launch<__nv_bfloat16, false>(p, group, batch, stream);
    return p.interleaved ? rope_launch<__half, true>(p, group, batch, stream)
                         : rope_launch<__half, false>(p, group, batch, stream);
}
