/*
 * Keys and values into the paged 4-bit cache (with q's and k's per-head
 * RMSNorm and rotation on the way), and back out as values.
 *
 * Append: one block a token.  head_dim / 8 lanes hold a head, eight values
 * each, from the load to the codes: the norm's sum of squares, the rotation's
 * partner values and the extremes of a 32-value block come by shuffles.  A
 * 32-bit word of codes holds four values of each 32-value block of a 64-wide
 * span, so the two lanes that hold them swap halves and each writes one word.
 * Bound by HBM for prompts and by launch and load latency for single tokens.
 */
#include "attn_device.cuh"

namespace {

/* Values of the rotation's partners: lane `src` (of the warp) holds them. */
__device__ __forceinline__ void partner(const float (&v)[8], float (&o)[8], int src) {
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = __shfl_sync(LFM_FULL_MASK, v[i], src);
}

/* Every lane of the warp runs this (the shuffles need them all); w: the lane's
 * norm weights or nullptr. */
template <int D>
__device__ __forceinline__ void norm_rotate(float (&v)[8], const float *w, const RopeDev &rp, int64_t pos, uint32_t sub) {
    constexpr int kL = D / 8;
    if (rp.q_norm || rp.k_norm) {
        float ss = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) ss = __fmaf_rn(v[i], v[i], ss);
#pragma unroll
        for (int o = kL / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(LFM_FULL_MASK, ss, o);
        if (w) {
            float g[8];
            const float r = 1.0f / sqrtf(ss / (float)D + rp.eps);
            lfm_load<8>(w + 8 * sub, g);
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = v[i] * r * g[i];
        }
    }
    const uint32_t half = rp.rot_dim / 2, e = 8 * sub;
    if (half == 0) return;
    if (rp.pairs) {
        if (e >= rp.rot_dim) return;
        float c[4], s[4];
        lfm_load<4>(rp.cos + (size_t)pos * half + e / 2, c);
        lfm_load<4>(rp.sin + (size_t)pos * half + e / 2, s);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float a = v[2 * i], b = v[2 * i + 1];
            v[2 * i] = a * c[i] - b * s[i];
            v[2 * i + 1] = b * c[i] + a * s[i];
        }
        return;
    }
    const int lane = threadIdx.x & 31;
    const bool first = e < half, in = e < rp.rot_dim;
    float o[8];
    partner(v, o, in ? (first ? lane + (int)(half / 8) : lane - (int)(half / 8)) : lane);
    if (!in) return;
    float c[8], s[8];
    const size_t at = (size_t)pos * half + (first ? e : e - half);
    lfm_load<8>(rp.cos + at, c);
    lfm_load<8>(rp.sin + at, s);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = first ? v[i] * c[i] - o[i] * s[i] : v[i] * c[i] + o[i] * s[i];
}

/* A head's eight values of this lane -> codes and scales at `codes` / `scales`. */
__device__ __forceinline__ void quant_store(float (&v)[8], uint32_t sub, uint8_t *codes, __half *scales, bool write) {
    float hi = -65504.0f, lo = 65504.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        /* the cache holds finite numbers only */
        v[i] = v[i] != v[i] ? 0.0f : fminf(fmaxf(v[i], -65504.0f), 65504.0f);
        hi = fmaxf(hi, v[i]);
        lo = fminf(lo, v[i]);
    }
#pragma unroll
    for (int o = 1; o <= 2; o <<= 1) {
        hi = fmaxf(hi, __shfl_xor_sync(LFM_FULL_MASK, hi, o));
        lo = fminf(lo, __shfl_xor_sync(LFM_FULL_MASK, lo, o));
    }
    const __half d = __float2half_rn((hi >= -lo ? hi : lo) * -0.125f);
    const float f = __half2float(d), inv = f != 0.0f ? 1.0f / f : 0.0f;
    uint32_t mine[2] = {0, 0};
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int c = min(15, max(0, __float2int_rd(v[i] * inv + 8.5f)));
        mine[i >> 2] |= (uint32_t)c << (4 * (i & 3));
    }
    /* lanes sub and sub ^ 4 hold the two 32-value blocks of a 64-wide span */
    const uint32_t g = (sub >> 2) & 1;
    const uint32_t got = __shfl_xor_sync(LFM_FULL_MASK, g ? mine[0] : mine[1], 4);
    const uint32_t word = g ? got | mine[1] << 16 : mine[0] | got << 16;
    if (!write) return;
    *reinterpret_cast<uint32_t *>(codes + 32 * (sub >> 3) + 4 * (2 * (sub & 3) + g)) = word;
    if ((sub & 3) == 0) scales[sub >> 2] = d;
}

template <class T, int D>
__global__ void __launch_bounds__(512) k_kv_append(AppendArgs A) {
    constexpr uint32_t kL = D / 8;
    __shared__ int s_seq;
    lfm_pdl_wait();
    const uint32_t tok = blockIdx.x;
    const int b = lfm_find_seq(A.bt, tok, &s_seq);
    if (b < 0) return;
    const int64_t q0 = A.bt.q_start[b], q1 = A.bt.q_start[b + 1];
    const int64_t pos = (int64_t)A.bt.kv_len[b] - (q1 - q0) + ((int64_t)tok - q0);
    if (pos < 0 || (A.rp.rot_dim && pos >= (int64_t)A.rp.n_pos)) {
        if (threadIdx.x == 0) atomicOr(A.err, LFM_DEVERR_PAGE);
        return;
    }
    const uint32_t hkv = A.k ? A.kv.hkv : 0, heads = A.n_heads + 2 * hkv, sub = threadIdx.x % kL;
    /* whole warps run every pass: the shuffles need them */
    for (uint32_t i0 = 0; i0 < heads; i0 += blockDim.x / kL) {
        const uint32_t i = i0 + threadIdx.x / kL;
        const bool on = i < heads;
        const bool isq = i < A.n_heads, isk = !isq && i < A.n_heads + hkv;
        const uint32_t head = isq ? i : isk ? i - A.n_heads : i - A.n_heads - hkv;
        float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        if (on) {
            const T *src = isq ? static_cast<const T *>(A.q) + (size_t)tok * A.q_stride
                         : isk ? static_cast<const T *>(A.k) + (size_t)tok * A.k_stride
                               : static_cast<const T *>(A.v) + (size_t)tok * A.v_stride;
            lfm_load<8>(src + (size_t)head * D + 8 * sub, v);
        }
        if (__any_sync(LFM_FULL_MASK, isq || isk)) { /* a warp may hold values too: they stay as they are */
            float r[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) r[j] = v[j];
            norm_rotate<D>(r, isq ? A.rp.q_norm : isk ? A.rp.k_norm : nullptr, A.rp, pos, sub);
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = isq || isk ? r[j] : v[j];
        }
        if (isq) lfm_store<8>(static_cast<T *>(A.q_out) + (size_t)tok * A.q_out_stride + (size_t)head * D + 8 * sub, v);
        if (!__any_sync(LFM_FULL_MASK, on && !isq)) continue;
        uint8_t *page = on && !isq ? lfm_page(A.kv, A.bt, b, pos, head, A.err) : nullptr;
        const uint32_t in = (uint32_t)pos & (A.kv.page_tokens - 1);
        uint8_t *half = page ? page + (isk ? 0 : A.kv.half) : nullptr;
        quant_store(v, sub, half + (size_t)in * (D / 2),
                    reinterpret_cast<__half *>(half + A.kv.codes) + (size_t)in * (D / 32), page != nullptr);
    }
}

template <class T, int D>
__global__ void __launch_bounds__(256) k_kv_read(ReadArgs A) {
    constexpr uint32_t kL = D / 8;
    __shared__ int s_seq;
    lfm_pdl_wait();
    const uint32_t tok = blockIdx.x;
    const int b = lfm_find_seq(A.bt, tok, &s_seq);
    if (b < 0) return;
    const int64_t q0 = A.bt.q_start[b], q1 = A.bt.q_start[b + 1];
    const int64_t pos = (int64_t)A.bt.kv_len[b] - (q1 - q0) + ((int64_t)tok - q0);
    for (uint32_t u = threadIdx.x; u < 2 * A.kv.hkv * kL; u += blockDim.x) {
        const uint32_t sub = u % kL, isv = u / kL & 1, head = u / kL / 2;
        const uint8_t *page = lfm_page(A.kv, A.bt, b, pos, head, A.err);
        if (!page) continue;
        const uint32_t in = (uint32_t)pos & (A.kv.page_tokens - 1);
        const uint8_t *half = page + (isv ? A.kv.half : 0);
        /* values 8 sub ..: four nibbles of each of two neighbouring words */
        const uint32_t g = (sub >> 2) & 1;
        const uint2 w = *reinterpret_cast<const uint2 *>(half + (size_t)in * (D / 2) + 32 * (sub >> 3) + 8 * (sub & 3));
        const float d = __half2float(reinterpret_cast<const __half *>(half + A.kv.codes)[(size_t)in * (D / 32) + (sub >> 2)]);
        const uint32_t c[2] = {w.x >> (16 * g), w.y >> (16 * g)};
        float v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = d * (float)((int)(c[i >> 2] >> (4 * (i & 3)) & 15u) - 8);
        T *out = static_cast<T *>(isv ? A.v_out : A.k_out);
        lfm_store<8>(out + ((size_t)tok * A.kv.hkv + head) * D + 8 * sub, v);
    }
}

}  // namespace

cudaError_t lfm_launch_kv_append(const AppendArgs &a, uint32_t head_dim, uint32_t type, cudaStream_t s, bool pdl) {
    void (*fn)(AppendArgs);
    if (head_dim == 64) fn = type == 0 ? k_kv_append<float, 64> : type == 1 ? k_kv_append<__half, 64> : k_kv_append<__nv_bfloat16, 64>;
    else fn = type == 0 ? k_kv_append<float, 128> : type == 1 ? k_kv_append<__half, 128> : k_kv_append<__nv_bfloat16, 128>;
    uint32_t threads = ((a.n_heads + (a.k ? 2 * a.kv.hkv : 0)) * (head_dim / 8) + 31) / 32 * 32;
    if (threads > 512) threads = 512;
    return lfm_launch_pdl(fn, dim3(a.bt.n_tokens), dim3(threads), 0, s, pdl, a);
}

cudaError_t lfm_launch_kv_read(const ReadArgs &a, uint32_t head_dim, uint32_t type, cudaStream_t s, bool pdl) {
    void (*fn)(ReadArgs);
    if (head_dim == 64) fn = type == 0 ? k_kv_read<float, 64> : type == 1 ? k_kv_read<__half, 64> : k_kv_read<__nv_bfloat16, 64>;
    else fn = type == 0 ? k_kv_read<float, 128> : type == 1 ? k_kv_read<__half, 128> : k_kv_read<__nv_bfloat16, 128>;
    uint32_t threads = (2 * a.kv.hkv * (head_dim / 8) + 31) / 32 * 32;
    if (threads > 256) threads = 256;
    return lfm_launch_pdl(fn, dim3(a.bt.n_tokens), dim3(threads), 0, s, pdl, a);
}
