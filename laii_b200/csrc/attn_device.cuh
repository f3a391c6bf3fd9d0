/*
 * Device helpers shared by the attention-side kernels: typed loads and stores,
 * the sequence that a row belongs to, and pages.
 */
#ifndef LFM_ATTN_DEVICE_CUH
#define LFM_ATTN_DEVICE_CUH

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include "attn_internal.h"
#include "moe_device.cuh"

/* Programmatic launches: every kernel here waits for its predecessor before it
 * reads or writes memory that the stream's earlier work may touch. */
template <class... A>
inline cudaError_t lfm_launch_pdl(void (*fn)(A...), dim3 grid, dim3 block, size_t smem, cudaStream_t s, bool pdl,
                                  A... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = pdl ? 1 : 0;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, fn, args...);
}

/* N (4 or 8) consecutive values as fp32. */
template <int N>
__device__ __forceinline__ void lfm_load(const float *p, float (&v)[N]) {
#pragma unroll
    for (int i = 0; i < N; i += 4) {
        const float4 f = *reinterpret_cast<const float4 *>(p + i);
        v[i] = f.x; v[i + 1] = f.y; v[i + 2] = f.z; v[i + 3] = f.w;
    }
}
template <int N, class T2, class T>
__device__ __forceinline__ void lfm_load16(const T *p, float (&v)[N], float2 (*cv)(T2)) {
    uint32_t w[N / 2];
    if constexpr (N == 8) {
        const uint4 u = *reinterpret_cast<const uint4 *>(p);
        w[0] = u.x; w[1] = u.y; w[2] = u.z; w[3] = u.w;
    } else {
        const uint2 u = *reinterpret_cast<const uint2 *>(p);
        w[0] = u.x; w[1] = u.y;
    }
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
        const float2 f = cv(*reinterpret_cast<T2 *>(&w[i]));
        v[2 * i] = f.x; v[2 * i + 1] = f.y;
    }
}
__device__ __forceinline__ float2 lfm_h2_f2(__half2 h) { return __half22float2(h); }
__device__ __forceinline__ float2 lfm_b2_f2(__nv_bfloat162 h) { return __bfloat1622float2(h); }
template <int N>
__device__ __forceinline__ void lfm_load(const __half *p, float (&v)[N]) { lfm_load16<N, __half2>(p, v, lfm_h2_f2); }
template <int N>
__device__ __forceinline__ void lfm_load(const __nv_bfloat16 *p, float (&v)[N]) {
    lfm_load16<N, __nv_bfloat162>(p, v, lfm_b2_f2);
}

template <int N>
__device__ __forceinline__ void lfm_store(float *p, const float (&v)[N]) {
#pragma unroll
    for (int i = 0; i < N; i += 4) *reinterpret_cast<float4 *>(p + i) = make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
}
__device__ __forceinline__ uint32_t lfm_pack2(float a, float b, __half) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
}
__device__ __forceinline__ uint32_t lfm_pack2(float a, float b, __nv_bfloat16) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
}
template <int N, class T>
__device__ __forceinline__ void lfm_store(T *p, const float (&v)[N]) {
    uint32_t w[N / 2];
#pragma unroll
    for (int i = 0; i < N / 2; ++i) w[i] = lfm_pack2(v[2 * i], v[2 * i + 1], T());
    if constexpr (N == 8) *reinterpret_cast<uint4 *>(p) = make_uint4(w[0], w[1], w[2], w[3]);
    else *reinterpret_cast<uint2 *>(p) = make_uint2(w[0], w[1]);
}

/* The whole block: the sequence that owns row `tok`, or -1 (padding, or
 * offsets that do not contain it).  s_seq: one shared int. */
__device__ __forceinline__ int lfm_find_seq(const BatchDev &bt, uint32_t tok, int *s_seq) {
    if (threadIdx.x == 0) *s_seq = -1;
    __syncthreads();
    for (uint32_t b = threadIdx.x; b < bt.n_seqs; b += blockDim.x)
        if ((int64_t)bt.q_start[b] <= (int64_t)tok && (int64_t)tok < (int64_t)bt.q_start[b + 1]) *s_seq = (int)b;
    __syncthreads();
    return *s_seq;
}

/* Start of kv head `head` in the page of token `pos` of sequence b; nullptr
 * (and the error bit) where the table or the pool does not reach. */
__device__ __forceinline__ uint8_t *lfm_page(const KvDev &kv, const BatchDev &bt, int b, int64_t pos, uint32_t head,
                                             uint32_t *err) {
    const int64_t at = pos >> kv.page_shift;
    if (pos >= 0 && at < (int64_t)bt.table_stride) {
        const uint32_t id = (uint32_t)bt.page_table[(size_t)b * bt.table_stride + (size_t)at];
        if (id < kv.n_pages) return kv.pages + (size_t)id * kv.page_bytes + (size_t)head * kv.head_bytes;
    }
    atomicOr(err, LFM_DEVERR_PAGE);
    return nullptr;
}

#endif /* LFM_ATTN_DEVICE_CUH */
