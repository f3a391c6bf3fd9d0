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

/* Rows q0 .. q0 + n of a call of n_tokens. */
__device__ __forceinline__ bool lfm_sane(const BatchDev &bt, int64_t q0, int64_t n) {
    return q0 >= 0 && n >= 0 && q0 + n <= (int64_t)bt.n_tokens;
}

/* Reports sequences whose rows are out of order or beyond the call's: the thread looks at sequences at, at + step, ... */
__device__ __forceinline__ void lfm_check_batch(const BatchDev &bt, uint32_t at, uint32_t step, uint32_t *err) {
    bool sane = true;
#pragma unroll 1
    for (uint32_t b = at; b < bt.n_seqs; b += step) {
        const uint32_t q = (uint32_t)bt.q_start[b], end = (uint32_t)bt.q_start[b + 1]; /* negative: above n_tokens */
        sane &= q <= end && end <= bt.n_tokens;
    }
    if (!sane) atomicOr(err, LFM_DEVERR_PAGE);
}

/* A length that the page table has room for; attention's walk over a sequence is bounded by that. */
__device__ __forceinline__ bool lfm_sane_len(const BatchDev &bt, int64_t len) { return (uint32_t)len <= bt.span; }

/* One warp: the want-th tile of `per` rows (token, head of a group of G) over the sequences of more than `above` rows:
 * (sequence, tile) into out, or a sequence of -1.  Returns the tiles looked through: all where there is no such. */
__device__ __forceinline__ uint64_t lfm_find_tile(const BatchDev &bt, uint32_t G, uint32_t per, uint64_t above, uint64_t want,
                                                  int *out) {
    const uint32_t lane = threadIdx.x & 31;
    uint64_t before = 0;
    for (uint32_t b0 = 0; b0 < bt.n_seqs; b0 += 32) {
        uint64_t n = 0;
        if (b0 + lane < bt.n_seqs) {
            const int64_t q = bt.q_start[b0 + lane], q_n = (int64_t)bt.q_start[b0 + lane + 1] - q;
            const uint64_t rows = q_n > 0 && lfm_sane(bt, q, q_n) ? (uint64_t)q_n * G : 0;
            if (rows > above) n = (rows - 1) / per + 1;
        }
        uint64_t sum = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint64_t v = __shfl_up_sync(LFM_FULL_MASK, sum, o);
            if (lane >= (uint32_t)o) sum += v;
        }
        const bool here = want >= before + sum - n && want < before + sum;
        if (here) {
            out[0] = (int)(b0 + lane);
            out[1] = (int)(want - (before + sum - n));
        }
        before += __shfl_sync(LFM_FULL_MASK, sum, 31);
        if (__any_sync(LFM_FULL_MASK, here)) return before;
    }
    if (lane == 0) out[0] = -1;
    __syncwarp(); /* before another call's writer */
    return before;
}

/* Codes to fp16: a nibble in an fp16 exponent, bits 0-3 of a half as 1024 + c, bits 4-7 as 64 + c. */
#define LFM_NIB0_OFF 0x64086408u /* 1032, 1032: the exponent's offset and the code's own 8 */
#define LFM_NIB1_OFF 0x54805480u /*   72,   72 */
struct LfmNib {
    uint32_t e0, e1;
    /* the exponents stay in registers: as two immediates the compiler spends two instructions a pair */
    __device__ __forceinline__ LfmNib() {
        asm volatile("mov.b32 %0, 0x64006400;" : "=r"(e0));
        asm volatile("mov.b32 %0, 0x54005400;" : "=r"(e1));
    }
    __device__ __forceinline__ uint32_t lo(uint32_t x) const {
        uint32_t r;
        asm("lop3.b32 %0, %1, 0x000F000F, %2, 0xEA;" : "=r"(r) : "r"(x), "r"(e0));
        return r;
    }
    __device__ __forceinline__ uint32_t hi(uint32_t x) const {
        uint32_t r;
        asm("lop3.b32 %0, %1, 0x00F000F0, %2, 0xEA;" : "=r"(r) : "r"(x), "r"(e1));
        return r;
    }
};
__device__ __forceinline__ uint32_t lfm_hsub2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("sub.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
__device__ __forceinline__ uint32_t lfm_hmul2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("mul.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
__device__ __forceinline__ float lfm_ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float lfm_rcp(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

/* tanh(x) for capped scores, e2 = 2 x / ln 2, as 1 - 2 / (1 + e^2x): within 2^-22 of the truth, so a score is off by
 * softcap 2^-22.  That is well under what rounding the probabilities to fp16 costs up to LFM_PLAIN_CAP; beyond, where the
 * error would grow with the cap, small arguments take the series x - x^3 / 3 + 2 x^5 / 15 - 17 x^7 / 315 (relative error
 * below 62 / 2835 4^-8 = 2^-21 up to 1/4), and the score is off by 2^-20 of itself whatever the cap. */
#define LFM_PLAIN_CAP 128.0f
__device__ __forceinline__ float lfm_tanh(float e2) { return __fmaf_rn(-2.0f, lfm_rcp(1.0f + lfm_ex2(e2)), 1.0f); }
__device__ __forceinline__ float lfm_tanh_any(float e2) {
    const float x = e2 * 0.34657359f, y = x * x;
    const float p = __fmaf_rn(y, __fmaf_rn(y, -17.0f / 315.0f, 2.0f / 15.0f), -1.0f / 3.0f);
    return fabsf(x) < 0.25f ? __fmaf_rn(x * y, p, x) : lfm_tanh(e2);
}
/* 2 / ln 2 times what takes a product to tanh's argument: finite, so that a product of zero stays one. */
__device__ __forceinline__ float lfm_cap_scale(float scale, float softcap) { return fminf(fabsf(scale) * 2.88539008f / softcap, 3e38f); }

/* The running reference m of a row, in powers of two: p = 2^(z - m) is held in fp16.  It is set LFM_REF_LOW below a score,
 * so that keys far below a row's largest one keep their part of the product as they do of the sum (fp16 ends 2^-31 below
 * the largest; set at the score itself it was 2^-24, and 131072 keys 17.4 nats below one lost 0.4% of the output), and
 * moves when a score passes it by LFM_REF_MOVE: p <= 2^15, within fp16. */
#define LFM_REF_LOW 7.0f
#define LFM_REF_MOVE 15.0f
#define LFM_NO_KEY -1e30f /* of a row that has seen no key */

/* Eight values of q within fp16's finite range (NaN stays), negated for a negative scale. */
__device__ __forceinline__ void lfm_fit_q(bool neg, float (&v)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float x = neg ? -v[i] : v[i];
        v[i] = x > 65504.0f ? 65504.0f : x < -65504.0f ? -65504.0f : x;
    }
}
/* Keys [lo, hi) that row r (token, head of the group) of a sequence of n_q tokens behind len cached ones sees. */
__device__ __forceinline__ void lfm_visible(const AttnArgs &A, int64_t n_q, int64_t len, uint32_t r, int64_t &lo,
                                            int64_t &hi) {
    hi = A.causal ? len - n_q + (int64_t)(r / A.group) + 1 : len;
    if (hi < 0) hi = 0;
    lo = A.window && hi > (int64_t)A.window ? hi - A.window : 0;
}

#endif /* LFM_ATTN_DEVICE_CUH */
