/*
 * Grouped-query attention over the paged 4-bit cache, one block a (row, head):
 * tiles of 128 keys, a thread a key for the scores, a thread a value (and a
 * part of the keys) for the sum, running maximum and sum in fp32.
 */
#include "attn_device.cuh"

namespace {

constexpr int kThreads = 128;

__device__ __forceinline__ float read_row(const void *p, uint32_t type, size_t at) {
    return type == 0 ? static_cast<const float *>(p)[at]
         : type == 1 ? __half2float(static_cast<const __half *>(p)[at])
                     : __bfloat162float(static_cast<const __nv_bfloat16 *>(p)[at]);
}
__device__ __forceinline__ void write_row(void *p, uint32_t type, size_t at, float v) {
    if (type == 0) static_cast<float *>(p)[at] = v;
    else if (type == 1) static_cast<__half *>(p)[at] = __float2half_rn(v);
    else static_cast<__nv_bfloat16 *>(p)[at] = __float2bfloat16_rn(v);
}

/* Value i of a token's head: its word and nibble in the codes. */
__device__ __forceinline__ float cached(const uint8_t *half, uint32_t codes, uint32_t in, uint32_t D, uint32_t i) {
    const uint32_t w = reinterpret_cast<const uint32_t *>(half + (size_t)in * (D / 2) + 32 * (i >> 6))[(i & 31) >> 2];
    const float d = __half2float(reinterpret_cast<const __half *>(half + codes)[in * (D / 32) + (i >> 5)]);
    return d * (float)((int)(w >> (4 * ((i >> 5 & 1) * 4 + (i & 3))) & 15u) - 8);
}

template <int D>
__global__ void __launch_bounds__(kThreads) k_attn(AttnArgs A) {
    __shared__ int s_seq;
    __shared__ float s_q[D], s_p[kThreads], s_red[4], s_o[kThreads];
    lfm_pdl_wait();
    const uint32_t tok = blockIdx.x, head = blockIdx.y, kvh = head / A.group;
    const int b = lfm_find_seq(A.bt, tok, &s_seq);
    if (b < 0) return;
    const int tid = threadIdx.x;
    const int64_t q0 = A.bt.q_start[b], q1 = A.bt.q_start[b + 1], len = A.bt.kv_len[b];
    const int64_t pos = len - (q1 - q0) + ((int64_t)tok - q0);
    int64_t lo = 0, hi = A.causal ? pos + 1 : len;
    if (A.window && hi - (int64_t)A.window > 0) lo = hi - A.window;
    if (tid < D) s_q[tid] = read_row(A.q, A.type, (size_t)tok * A.q_stride + (size_t)head * D + tid);
    __syncthreads();
    float m = -INFINITY, l = 0.0f, o = 0.0f;
    const int d = tid % D, part = tid / D;
    for (int64_t j0 = lo; j0 < hi; j0 += kThreads) {
        const int64_t j = j0 + tid;
        float z = -INFINITY;
        if (j < hi) {
            const uint8_t *page = lfm_page(A.kv, A.bt, b, j, kvh, A.err);
            if (page) {
                z = 0.0f;
                for (int i = 0; i < D; ++i)
                    z = __fmaf_rn(s_q[i], cached(page, A.kv.codes, (uint32_t)j & (A.kv.page_tokens - 1), D, i), z);
                z *= A.scale;
                if (A.softcap > 0.0f) z = A.softcap * tanhf(z / A.softcap);
            }
        }
        float t = lfm_warp_max(z);
        if ((tid & 31) == 0) s_red[tid >> 5] = t;
        __syncthreads();
        t = fmaxf(fmaxf(s_red[0], s_red[1]), fmaxf(s_red[2], s_red[3]));
        const float mn = fmaxf(m, t), p = z == -INFINITY ? 0.0f : expf(z - mn);
        const float c = m == -INFINITY ? 0.0f : expf(m - mn);
        s_p[tid] = p;
        m = mn;
        __syncthreads();
        l *= c;
        o *= c;
        for (int i = 0; i < kThreads; ++i) l += s_p[i];
        for (int i = part; i < kThreads && j0 + i < hi; i += kThreads / D) {
            if (s_p[i] == 0.0f) continue;
            const uint8_t *page = lfm_page(A.kv, A.bt, b, j0 + i, kvh, A.err);
            o = __fmaf_rn(s_p[i], cached(page + A.kv.half, A.kv.codes, (uint32_t)(j0 + i) & (A.kv.page_tokens - 1), D, d), o);
        }
        __syncthreads();
    }
    s_o[tid] = o;
    __syncthreads();
    if (tid < D) {
        for (int i = 1; i < kThreads / D; ++i) o += s_o[tid + i * D];
        write_row(A.out, A.type, (size_t)tok * A.out_stride + (size_t)head * D + tid, l > 0.0f ? o / l : 0.0f);
    }
}

}  // namespace

cudaError_t lfm_launch_attn(const AttnArgs &a, uint32_t head_dim, cudaStream_t s, bool pdl) {
    return lfm_launch_pdl(head_dim == 64 ? k_attn<64> : k_attn<128>, dim3(a.bt.n_tokens, a.n_heads), dim3(kThreads), 0, s,
                          pdl, a);
}
