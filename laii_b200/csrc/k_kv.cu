/*
 * Keys and values into the paged 4-bit cache (with q's and k's per-head
 * RMSNorm and rotation on the way), and back out as values.
 *
 * head_dim / 8 lanes hold a head, eight values each, from the load to the
 * codes: the norm's sum of squares, the rotation's partner values and the
 * extremes of a 32-value block come by shuffles.  A 32-bit word of codes holds
 * four values of each 32-value block of a 64-wide span, so the two lanes that
 * hold them swap halves and each writes one word.  A warp takes some steps of
 * 32 lanes of one token by itself -- its sequence, position, angles and page
 * found once, a step's loads under way while the one before computes, no
 * block-wide barrier: one step for a few tokens (latency), more for prompts.
 * d and the codes are formed in fp32 from the rounded fp16 d, so that reading
 * back and attending see the d that the code was chosen for.
 *
 * Floor: the rows of q, k and v read, q and the codes written.  5307 tokens of
 * 32 / 8 heads of 128 values, 116 MB: 30.1 us, 3.9 TB/s, read back (28 MB, 4.3 us
 * at a copy's rate) 8.8 us.  Neither pipe is full (issue 62%, HBM 30%): with 24
 * warps an SM and two loads of each under way, of the 9.1 cycles between a warp's
 * instructions 3.2 wait for memory, 1.6 for the instruction before, 1.6 for their
 * turn; the reading kernel is one such chain a warp.  A block of threads for each
 * token, its steps between barriers: 74 us for both, 42 so.  64 tokens, 64-value
 * heads: 3.1 us, a launch and a chain of loads.
 */
#include "attn_device.cuh"

namespace {

/* The cosines and sines of this lane's values (of its four pairs, where the pairs are neighbours), read once for all
 * heads of a token. */
struct Angles {
    float c[8], s[8];
    __device__ __forceinline__ Angles(const RopeDev &rp, int64_t pos, uint32_t sub) {
        const uint32_t half = rp.rot_dim / 2, e = 8 * sub;
#pragma unroll
        for (int i = 0; i < 8; ++i) c[i] = s[i] = 0.0f;
        if (e >= rp.rot_dim) return;
        if (rp.pairs) {
            float a[4], b[4];
            lfm_load<4>(rp.cos + (size_t)pos * half + e / 2, a);
            lfm_load<4>(rp.sin + (size_t)pos * half + e / 2, b);
#pragma unroll
            for (int i = 0; i < 4; ++i) { c[i] = a[i]; s[i] = b[i]; }
        } else {
            const size_t at = (size_t)pos * half + (e < half ? e : e - half);
            lfm_load<8>(rp.cos + at, c);
            lfm_load<8>(rp.sin + at, s);
        }
    }
};

/* Every lane of the warp runs this (the shuffles need them all); w: the norm's
 * weights or nullptr. */
template <int D>
__device__ __forceinline__ void norm_rotate(float (&v)[8], const float *w, const RopeDev &rp, const Angles &g, uint32_t sub) {
    constexpr int kL = D / 8;
    if (w) {
        float ss = 0.0f, x[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) ss = __fmaf_rn(v[i], v[i], ss);
#pragma unroll
        for (int o = kL / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(LFM_FULL_MASK, ss, o);
        const float r = 1.0f / sqrtf(ss / (float)D + rp.eps);
        lfm_load<8>(w + 8 * sub, x);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = v[i] * r * x[i];
    }
    const uint32_t half = rp.rot_dim / 2, e = 8 * sub;
    if (half == 0) return;
    if (rp.pairs) {
        if (e >= rp.rot_dim) return;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float a = v[2 * i], b = v[2 * i + 1];
            v[2 * i] = a * g.c[i] - b * g.s[i];
            v[2 * i + 1] = b * g.c[i] + a * g.s[i];
        }
        return;
    }
    const int lane = threadIdx.x & 31;
    const bool first = e < half, in = e < rp.rot_dim;
    const int src = in ? (first ? lane + (int)(half / 8) : lane - (int)(half / 8)) : lane;
    float o[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = __shfl_sync(LFM_FULL_MASK, v[i], src); /* the partners */
    if (!in) return;
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = first ? v[i] * g.c[i] - o[i] * g.s[i] : v[i] * g.c[i] + o[i] * g.s[i];
}

/* A head's eight values of this lane -> codes and scales at `codes` / `scales`. */
__device__ __forceinline__ void quant_store(float (&v)[8], uint32_t sub, uint8_t *codes, __half *scales, bool write) {
    /* magnitudes as integers, where NaN is above infinity above the rest; the largest value beside them for the sign */
    uint32_t a;
    float hi;
    auto extremes = [&]() {
        a = 0;
        hi = -65504.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            a = max(a, __float_as_uint(v[i]) & 0x7FFFFFFFu);
            hi = fmaxf(hi, v[i]);
        }
    };
    extremes();
    if (__any_sync(LFM_FULL_MASK, a > 0x477FE000u)) { /* above 65504: the cache holds finite numbers only */
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = v[i] != v[i] ? 0.0f : fminf(fmaxf(v[i], -65504.0f), 65504.0f);
        extremes();
    }
#pragma unroll
    for (int o = 1; o <= 2; o <<= 1) {
        a = max(a, __shfl_xor_sync(LFM_FULL_MASK, a, o));
        hi = fmaxf(hi, __shfl_xor_sync(LFM_FULL_MASK, hi, o));
    }
    const float m = __uint_as_float(a);
    const __half d = __float2half_rn((hi == m ? m : -m) * -0.125f);
    const float f = __half2float(d), inv = f != 0.0f ? 1.0f / f : 0.0f;
    uint32_t mine[2] = {0, 0};
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        /* floor by an addition of 2^23 that rounds down: the code is in the low bits, 0x4B000000 above it */
        const float t = __fadd_rd(fminf(fmaxf(v[i] * inv + 8.5f, 0.0f), 15.0f), 8388608.0f);
        mine[i >> 2] += __float_as_uint(t) << (4 * (i & 3));
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) mine[i] &= 0xFFFFu;
    /* lanes sub and sub ^ 4 hold the two 32-value blocks of a 64-wide span */
    const uint32_t g = (sub >> 2) & 1;
    const uint32_t got = __shfl_xor_sync(LFM_FULL_MASK, g ? mine[0] : mine[1], 4);
    const uint32_t word = g ? got | mine[1] << 16 : mine[0] | got << 16;
    if (!write) return;
    *reinterpret_cast<uint32_t *>(codes + 32 * (sub >> 3) + 4 * (2 * (sub & 3) + g)) = word;
    if ((sub & 3) == 0) scales[sub >> 2] = d;
}

/* Eight values in memory. */
template <class T>
struct alignas(16) Eight {
    uint32_t w[sizeof(T) * 2] = {};
};

/* One warp: the sequence that owns row `tok` (-1: none) and the token's position.  A sequence whose rows are out of order
 * or beyond the call's owns none. */
__device__ __forceinline__ int locate(const BatchDev &bt, uint32_t tok, int64_t &pos) {
    const uint32_t lane = threadIdx.x & 31;
    for (uint32_t b0 = 0; b0 < bt.n_seqs; b0 += 32) {
        const uint32_t b = b0 + lane;
        int64_t q0 = 0, q1 = 0, len = 0;
        if (b < bt.n_seqs) {
            q0 = bt.q_start[b];
            q1 = bt.q_start[b + 1];
            len = bt.kv_len[b];
        }
        const uint32_t who = __ballot_sync(LFM_FULL_MASK, q0 >= 0 && q0 <= (int64_t)tok && (int64_t)tok < q1 && q1 <= (int64_t)bt.n_tokens);
        if (who) {
            const int src = __ffs(who) - 1;
            pos = __shfl_sync(LFM_FULL_MASK, len - (q1 - q0) + ((int64_t)tok - q0), src);
            return (int)b0 + src;
        }
    }
    return -1;
}

template <class T, int D>
__global__ void __launch_bounds__(256, 4) k_kv_append(AppendArgs A, uint32_t per_token, uint32_t steps) {
    constexpr uint32_t kL = D / 8, kHeads = 32 / kL; /* lanes of a head, heads of a step */
    lfm_pdl_wait();
    lfm_pdl_launch_dependents();
    if (blockIdx.x == 0) lfm_check_batch(A.bt, threadIdx.x, blockDim.x, A.err);
    const uint32_t task = blockIdx.x * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31, sub = lane % kL;
    const uint32_t tok = task / per_token, own = lane / kL;
    if (tok >= A.bt.n_tokens) return;
    /* a step is all q, all k or all v */
    const uint32_t hkv = A.k ? A.kv.hkv : 0, nq = (A.n_heads + kHeads - 1) / kHeads, nk = (hkv + kHeads - 1) / kHeads;
    const uint32_t first = task % per_token * steps, end = min(nq + 2 * nk, first + steps);
    int64_t pos = 0;
    const int b = locate(A.bt, tok, pos);
    if (b < 0) return;
    if (pos < 0 || (A.rp.rot_dim && pos >= (int64_t)A.rp.n_pos)) {
        if (lane == 0) atomicOr(A.err, LFM_DEVERR_PAGE);
        return;
    }
    /* the token's page, where this warp holds keys or values */
    uint8_t *page = end > nq ? lfm_page(A.kv, A.bt, b, pos, 0, A.err) : nullptr;
    const uint32_t in = (uint32_t)pos & (A.kv.page_tokens - 1);
    const Angles ang(A.rp, pos, sub);
    /* the steps [lo, hi) of one kind, two steps' values under way */
    auto walk = [&](const T *src, uint32_t lo, uint32_t hi, uint32_t n_heads, auto &&each) {
        using Raw = Eight<T>;
        uint32_t head = lo * kHeads + own;
        src += (size_t)head * D + 8 * sub;
        Raw x0{}, x1{};
        if (lo < hi && head < n_heads) x0 = *reinterpret_cast<const Raw *>(src);
        if (lo + 1 < hi && head + kHeads < n_heads) x1 = *reinterpret_cast<const Raw *>(src + kHeads * D);
#pragma unroll 1
        for (uint32_t st = lo; st < hi; ++st) {
            float v[8];
            lfm_load<8>(reinterpret_cast<const T *>(&x0), v);
            x0 = x1;
            src += kHeads * D;
            if (st + 2 < hi && head + 2 * kHeads < n_heads) x1 = *reinterpret_cast<const Raw *>(src + kHeads * D);
            each(v, head);
            head += kHeads;
        }
    };
    if (first < nq) {
        T *out = static_cast<T *>(A.q_out) + (size_t)tok * A.q_out_stride + 8 * sub;
        walk(static_cast<const T *>(A.q) + (size_t)tok * A.q_stride, first, min(end, nq), A.n_heads, [&](float (&v)[8], uint32_t head) {
            norm_rotate<D>(v, A.rp.q_norm, A.rp, ang, sub);
            if (head < A.n_heads) lfm_store<8>(out + head * D, v);
        });
    }
    if (end <= nq) return;
    uint8_t *codes = page + (size_t)in * (D / 2);
    __half *scales = reinterpret_cast<__half *>(page + A.kv.codes) + (size_t)in * (D / 32);
    const uint32_t hb = (uint32_t)A.kv.head_bytes; /* of one page: below 2^16 */
    const bool held = page != nullptr;
    if (first < nq + nk)
        walk(static_cast<const T *>(A.k) + (size_t)tok * A.k_stride, first > nq ? first - nq : 0, min(end - nq, nk), hkv,
             [&](float (&v)[8], uint32_t head) {
                 norm_rotate<D>(v, A.rp.k_norm, A.rp, ang, sub);
                 quant_store(v, sub, codes + head * hb, scales + head * (hb / 2), held && head < hkv);
             });
    if (end > nq + nk)
        walk(static_cast<const T *>(A.v) + (size_t)tok * A.v_stride, first > nq + nk ? first - nq - nk : 0, end - nq - nk, hkv,
             [&](float (&v)[8], uint32_t head) {
                 quant_store(v, sub, codes + head * hb + A.kv.half, scales + head * (hb / 2) + A.kv.half / 2, held && head < hkv);
             });
}

template <class T, int D, int kPass>
__global__ void __launch_bounds__(256) k_kv_read(ReadArgs A, uint32_t per_token) {
    constexpr uint32_t kL = D / 8, kHeads = 32 / kL;
    lfm_pdl_wait();
    lfm_pdl_launch_dependents();
    if (blockIdx.x == 0) lfm_check_batch(A.bt, threadIdx.x, blockDim.x, A.err);
    const uint32_t task = blockIdx.x * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31, sub = lane % kL;
    const uint32_t tok = task / per_token, first = task % per_token * kPass * kHeads + lane / kL;
    if (tok >= A.bt.n_tokens) return;
    int64_t pos = 0;
    const int b = locate(A.bt, tok, pos);
    if (b < 0) return;
    const uint8_t *page = lfm_page(A.kv, A.bt, b, pos, 0, A.err);
    if (!page) return;
    const uint32_t in = (uint32_t)pos & (A.kv.page_tokens - 1), g = (sub >> 2) & 1;
    uint2 w[kPass];
    float d[kPass];
#pragma unroll
    for (int p = 0; p < kPass; ++p) {
        const uint32_t i = first + p * kHeads; /* keys of all heads, then values */
        if (i < 2 * A.kv.hkv) {
            const uint32_t isv = i >= A.kv.hkv;
            const uint8_t *half = page + (size_t)(i - isv * A.kv.hkv) * A.kv.head_bytes + (isv ? A.kv.half : 0);
            /* values 8 sub ..: four nibbles of each of two neighbouring words */
            w[p] = *reinterpret_cast<const uint2 *>(half + (size_t)in * (D / 2) + 32 * (sub >> 3) + 8 * (sub & 3));
            d[p] = __half2float(reinterpret_cast<const __half *>(half + A.kv.codes)[(size_t)in * (D / 32) + (sub >> 2)]);
        }
    }
#pragma unroll
    for (int p = 0; p < kPass; ++p) {
        const uint32_t i = first + p * kHeads;
        if (i < 2 * A.kv.hkv) {
            const uint32_t isv = i >= A.kv.hkv, c[2] = {w[p].x >> (16 * g), w[p].y >> (16 * g)};
            float v[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) v[k] = d[p] * (float)((int)(c[k >> 2] >> (4 * (k & 3)) & 15u) - 8);
            T *out = static_cast<T *>(isv ? A.v_out : A.k_out);
            lfm_store<8>(out + ((size_t)tok * A.kv.hkv + (i - isv * A.kv.hkv)) * D + 8 * sub, v);
        }
    }
}

/* Steps a warp takes: one where that leaves the GPU unfilled, eight beyond.  Tokens of 32 / 8 heads of 64 values, append
 * and read back, one step / eight: 64 tokens 5.0 / 8.8 us, 512: 7.5 / 9.1, 1024: 10.6 / 9.9, 4096: 28.8 / 19.0; of 128
 * values: 256: 7.4 / 11.0, 768: 12.5 / 12.0, 4096: 53.9 / 32.0.  The sides meet at 900 and 700 tokens, 11 and 17
 * thousand steps; 96 warps an SM, 14 thousand, lie between. */
constexpr uint64_t kManySteps = 148 * 96;

template <class T, int D>
cudaError_t launch_append(const AppendArgs &a, cudaStream_t s, bool pdl) {
    constexpr uint32_t kHeads = 256 / D;
    const uint32_t steps = (a.n_heads + kHeads - 1) / kHeads + (a.k ? 2 * ((a.kv.hkv + kHeads - 1) / kHeads) : 0);
    const uint32_t pass = (uint64_t)steps * a.bt.n_tokens > kManySteps ? 8 : 1, per = (steps + pass - 1) / pass;
    const uint64_t blocks = ((uint64_t)per * a.bt.n_tokens + 7) / 8;
    if (blocks > 0x7FFFFFFFull) return cudaErrorInvalidConfiguration;
    return lfm_launch_pdl(k_kv_append<T, D>, dim3((uint32_t)blocks), dim3(256), 0, s, pdl, a, per, pass);
}
template <class T, int D>
cudaError_t launch_read(const ReadArgs &a, cudaStream_t s, bool pdl) {
    const uint32_t steps = (2 * a.kv.hkv * (D / 8) + 31) / 32;
    const uint32_t pass = (uint64_t)steps * a.bt.n_tokens > kManySteps ? 8 : 1, per = (steps + pass - 1) / pass;
    const uint64_t blocks = ((uint64_t)per * a.bt.n_tokens + 7) / 8;
    if (blocks > 0x7FFFFFFFull) return cudaErrorInvalidConfiguration;
    return lfm_launch_pdl(pass == 8 ? k_kv_read<T, D, 8> : k_kv_read<T, D, 1>, dim3((uint32_t)blocks), dim3(256), 0, s, pdl, a, per);
}

}  // namespace

cudaError_t lfm_launch_kv_append(const AppendArgs &a, uint32_t head_dim, uint32_t type, cudaStream_t s, bool pdl) {
    if (head_dim == 64)
        return type == 0 ? launch_append<float, 64>(a, s, pdl) : type == 1 ? launch_append<__half, 64>(a, s, pdl)
                                                                           : launch_append<__nv_bfloat16, 64>(a, s, pdl);
    return type == 0 ? launch_append<float, 128>(a, s, pdl) : type == 1 ? launch_append<__half, 128>(a, s, pdl)
                                                                        : launch_append<__nv_bfloat16, 128>(a, s, pdl);
}

cudaError_t lfm_launch_kv_read(const ReadArgs &a, uint32_t head_dim, uint32_t type, cudaStream_t s, bool pdl) {
    if (head_dim == 64)
        return type == 0 ? launch_read<float, 64>(a, s, pdl) : type == 1 ? launch_read<__half, 64>(a, s, pdl)
                                                                         : launch_read<__nv_bfloat16, 64>(a, s, pdl);
    return type == 0 ? launch_read<float, 128>(a, s, pdl) : type == 1 ? launch_read<__half, 128>(a, s, pdl)
                                                                      : launch_read<__nv_bfloat16, 128>(a, s, pdl);
}
