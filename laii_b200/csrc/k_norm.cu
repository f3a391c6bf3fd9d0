/*
 * Residual addition, RMSNorm and block_q8_K rows in one pass.
 *
 *   y = x + delta,  n = y * (1 / sqrt(mean(y^2) + eps)) * w,
 *   per 256 values: m = max|n|, d = m / 127, q = rne(n * (127 / m)), 16 sums of 16 codes.
 *
 * One block a row, one warp a 256-value Q8_K block: a lane holds values
 * 4 l .. 4 l + 3 and 128 + 4 l .. of its block in registers from the load to
 * the codes, so every tensor is touched once and the row's only exchange is
 * the sum of squares (warp shuffles, then the warps' sums in order: the same
 * result on every run).
 *
 * Floor: x, delta and the outputs once, 13.1 bytes a value with an fp32 delta:
 * bound by HBM.  4096 rows of 2048 values, 110 MB, call after call (some of it
 * then comes from L2): 16.0 us, 6.9 TB/s; the rows read back as bf16 values (26
 * MB, 4.1 us at a copy's rate) 5.2 more.  1021 rows of 5120 with bf16 rows as
 * well, 69 MB: 10.6 us.  64 rows of 2048: 1.7 us, a launch and a chain of loads,
 * sum and maximum.
 */
#include "attn_device.cuh"

namespace {

constexpr uint32_t kMaxWarps = 32; /* D <= 8192 */

template <class T>
__device__ __forceinline__ void add_row(const T *p, float (&v)[8]) {
    float a[4], b[4];
    lfm_load<4>(p, a);
    lfm_load<4>(p + 128, b);
#pragma unroll
    for (int i = 0; i < 4; ++i) { v[i] = v[i] + a[i]; v[4 + i] = v[4 + i] + b[i]; }
}

template <class T>
__device__ __forceinline__ void store_row(T *p, const float (&v)[8]) {
    const float a[4] = {v[0], v[1], v[2], v[3]}, b[4] = {v[4], v[5], v[6], v[7]};
    lfm_store<4>(p, a);
    lfm_store<4>(p + 128, b);
}

__device__ __forceinline__ uint32_t code4(const int (&q)[4]) {
    uint32_t w = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) w |= (uint32_t)(uint8_t)(int8_t)max(-128, min(127, q[i])) << (8 * i);
    return w;
}

template <int kDelta> /* 0: none, 1: fp32, 2: fp16, 3: bf16 */
__global__ void __launch_bounds__(1024) k_add_rmsnorm(const float *x, const void *delta, uint32_t D, const float *weight,
                                                      float eps, float *x_out, void *xb, uint32_t xb_type, uint8_t *q8) {
    __shared__ float s_sum[kMaxWarps];
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31, nw = blockDim.x >> 5;
    const size_t col = 256u * warp + 4u * lane, at = (size_t)blockIdx.x * D + col;
    float w[8] = {1.f, 1.f, 1.f, 1.f, 1.f, 1.f, 1.f, 1.f}, v[8];
    lfm_pdl_wait();
    lfm_pdl_launch_dependents();
    {
        float a[4], b[4];
        lfm_load<4>(x + at, a);
        lfm_load<4>(x + at + 128, b);
#pragma unroll
        for (int i = 0; i < 4; ++i) { v[i] = a[i]; v[4 + i] = b[i]; }
    }
    if constexpr (kDelta == 1) add_row(static_cast<const float *>(delta) + at, v);
    if constexpr (kDelta == 2) add_row(static_cast<const __half *>(delta) + at, v);
    if constexpr (kDelta == 3) add_row(static_cast<const __nv_bfloat16 *>(delta) + at, v);
    if (weight) {
        float a[4], b[4];
        lfm_load<4>(weight + col, a);
        lfm_load<4>(weight + col + 128, b);
#pragma unroll
        for (int i = 0; i < 4; ++i) { w[i] = a[i]; w[4 + i] = b[i]; }
    }
    if (x_out) store_row(x_out + at, v);
    if (!xb && !q8) return;
    float ss = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) ss = __fmaf_rn(v[i], v[i], ss);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(LFM_FULL_MASK, ss, o);
    if (lane == 0) s_sum[warp] = ss;
    __syncthreads();
    ss = 0.0f;
    for (uint32_t i = 0; i < nw; ++i) ss += s_sum[i];
    const float r = 1.0f / sqrtf(ss / (float)D + eps);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = v[i] * r * w[i];
    if (xb) {
        if (xb_type == 0) store_row(static_cast<float *>(xb) + at, v);
        else if (xb_type == 1) store_row(static_cast<__half *>(xb) + at, v);
        else store_row(static_cast<__nv_bfloat16 *>(xb) + at, v);
    }
    if (!q8) return;
    /* magnitudes as integers, where NaN is above infinity above the rest: a block that holds one gets the scale NaN, so
     * that its values read as such (codes alone cannot say it) */
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(v[i]) & 0x7FFFFFFFu);
    const float m = __uint_as_float(__reduce_max_sync(LFM_FULL_MASK, top));
    const float sc = m != 0.0f ? 127.0f / m : 0.0f;
    int a[4], b[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) { a[i] = __float2int_rn(v[i] * sc); b[i] = __float2int_rn(v[4 + i] * sc); }
    uint8_t *blk = q8 + ((size_t)blockIdx.x * nw + warp) * LFM_Q8K_BYTES; /* d, 256 codes, 16 sums */
    uint32_t *codes = reinterpret_cast<uint32_t *>(blk + 4);
    codes[lane] = code4(a);
    codes[32 + lane] = code4(b);
    int sa = a[0] + a[1] + a[2] + a[3], sb = b[0] + b[1] + b[2] + b[3];
#pragma unroll
    for (int o = 1; o <= 2; o <<= 1) {
        sa += __shfl_xor_sync(LFM_FULL_MASK, sa, o);
        sb += __shfl_xor_sync(LFM_FULL_MASK, sb, o);
    }
    int16_t *sums = reinterpret_cast<int16_t *>(blk + 260);
    if ((lane & 3) == 0) {
        sums[lane >> 2] = (int16_t)sa;
        sums[8 + (lane >> 2)] = (int16_t)sb;
    }
    if (lane == 0) *reinterpret_cast<float *>(blk) = m / 127.0f;
}

/* A warp a block: the values d * q. */
__global__ void __launch_bounds__(256) k_q8k_read(const uint8_t *q8, size_t n_blocks, uint32_t type, void *out) {
    lfm_pdl_wait();
    lfm_pdl_launch_dependents();
    const size_t b = (size_t)blockIdx.x * 8 + (threadIdx.x >> 5);
    const uint32_t lane = threadIdx.x & 31;
    if (b >= n_blocks) return;
    const uint8_t *blk = q8 + b * LFM_Q8K_BYTES;
    const float d = *reinterpret_cast<const float *>(blk);
    const uint32_t *codes = reinterpret_cast<const uint32_t *>(blk + 4);
    const uint32_t c[2] = {codes[lane], codes[32 + lane]};
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = d * (float)(int8_t)(uint8_t)(c[i >> 2] >> (8 * (i & 3)));
    const size_t at = b * 256 + 4 * lane;
    if (type == 0) store_row(static_cast<float *>(out) + at, v);
    else if (type == 1) store_row(static_cast<__half *>(out) + at, v);
    else store_row(static_cast<__nv_bfloat16 *>(out) + at, v);
}

}  // namespace

cudaError_t lfm_launch_add_rmsnorm(const float *x, const void *delta, uint32_t delta_type, uint32_t T, uint32_t D,
                                   const float *weight, float eps, float *x_out, void *xb, uint32_t xb_type,
                                   uint8_t *q8, cudaStream_t s, bool pdl) {
    auto fn = !delta ? k_add_rmsnorm<0> : delta_type == 0 ? k_add_rmsnorm<1> : delta_type == 1 ? k_add_rmsnorm<2>
                                                                                               : k_add_rmsnorm<3>;
    return lfm_launch_pdl(fn, dim3(T), dim3(D / 8), 0, s, pdl, x, delta, D, weight, eps, x_out, xb, xb_type, q8);
}

cudaError_t lfm_launch_q8k_read(const uint8_t *q8, uint32_t rows, uint32_t D, uint32_t type, void *out, cudaStream_t s,
                                bool pdl) {
    const size_t n = (size_t)rows * (D / 256);
    return lfm_launch_pdl(k_q8k_read, dim3((uint32_t)((n + 7) / 8)), dim3(256), 0, s, pdl, q8, n, type, out);
}
