// enc_attn.cu -- attention over packed sequences, with grouped heads, full or causal.
//
//   o[t, h] = sum_j p_j v[j, g(h)],  p = softmax_j(scale q[t, h] . k[j, g(h)]),  g(h) = h / (heads / kv_heads)
//
// over the keys j of t's own sequence (with causal set: those up to t).  The sequences lie one behind
// the other in the rows of q, k, v; cu_seqlens names where each begins.
//
//   packed_attn_simt   a warp per (row, head): 32 keys per step, scores, running maximum and sum in fp32.
#include <algorithm>

#include "enc_common.cuh"

namespace ragrt {

namespace {

struct AttnParams {
    const void* q;
    const void* k;
    const void* v;
    void* out;
    const int32_t* cu;
    int64_t q_stride, k_stride, v_stride, out_stride;
    int T, B, heads, kv_heads, dim, causal;
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

// One row of one head by one warp.  sq: dim floats of shared memory of this warp's own.
template <typename T>
__device__ void attn_row(const AttnParams& p, int t, int h, int lo, int hi, float* sq) {
    const int lane = threadIdx.x & 31;
    const int g = h / (p.heads / p.kv_heads);
    const T* q = static_cast<const T*>(p.q) + t * p.q_stride + (int64_t)h * p.dim;
    const T* k = static_cast<const T*>(p.k) + (int64_t)g * p.dim;
    const T* v = static_cast<const T*>(p.v) + (int64_t)g * p.dim;
    __syncwarp();
    for (int d = lane; d < p.dim; d += 32) sq[d] = (float)q[d] * p.scale;
    __syncwarp();
    float m = -INFINITY, l = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};         // dims lane, lane + 32, ...
    for (int base = lo; base < hi; base += 32) {
        const int j = base + lane;
        float s = -INFINITY;
        if (j < hi) {
            const uint4* kr = reinterpret_cast<const uint4*>(k + j * p.k_stride);
            s = 0.f;
            for (int c = 0; c < p.dim / 8; ++c) {
                float f[8];
                up8<T>(__ldg(kr + c), f);
#pragma unroll
                for (int e = 0; e < 8; ++e) s = fmaf(f[e], sq[8 * c + e], s);
            }
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

template <typename T>
__global__ void __launch_bounds__(256) packed_attn_simt(const AttnParams p) {
    __shared__ float sq[8][128];
    pdl_wait_then_release();
    attn_check_table(p);
    const int warp = threadIdx.x >> 5;
    const int64_t unit = (int64_t)blockIdx.x * 8 + warp;
    if (unit >= (int64_t)p.T * p.heads) return;
    const int t = (int)(unit / p.heads), h = (int)(unit % p.heads);
    int lo, hi;
    attn_range(p, t, lo, hi);
    if (lo < hi) attn_row<T>(p, t, h, lo, hi, sq[warp]);
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
                 head_dim, causal != 0, scale, err};
    const int64_t blocks = ceil_div((int64_t)T * heads, 8);
    RAGRT_REQUIRE(blocks <= 0x7FFFFFFF, "too many rows x heads");
    return dtype == RAGRT_BF16 ? enc_launch(packed_attn_simt<__nv_bfloat16>, dim3((unsigned)blocks), dim3(256), 0,
                                            (cudaStream_t)stream_, p)
                               : enc_launch(packed_attn_simt<__half>, dim3((unsigned)blocks), dim3(256), 0,
                                            (cudaStream_t)stream_, p);
}
