/*
 * C-ABI implementation of include/lfm_gpu_attn.h: argument checks, device
 * views and launches.  Nothing is computed here and nothing falls back to the
 * CPU: every failure is returned as a status.
 */
#include <cuda_runtime.h>
#include <math.h>

#include <type_traits>

#include "attn_internal.h"
#include "lfm_gpu_attn.h"

#define LFM_API extern "C" __attribute__((visibility("default")))

namespace {

/* The handle's device for the duration of a call (one runtime call where it is current already). */
struct OnDevice {
    int prev = -1;
    explicit OnDevice(int dev) {
        if (cudaGetDevice(&prev) != cudaSuccess) prev = -1;
        if (prev == dev) prev = -1;
        else cudaSetDevice(dev);
    }
    ~OnDevice() {
        if (prev >= 0) cudaSetDevice(prev);
    }
};

bool type_ok(uint32_t t) { return t == LFM_GPU_TYPE_F32 || t == LFM_GPU_TYPE_F16 || t == LFM_GPU_TYPE_BF16; }
uint32_t type_bytes(uint32_t t) { return t == LFM_GPU_TYPE_F32 ? 4 : 2; }
bool misaligned(const void *p, size_t a = 16) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) != 0; }

#define FAIL(...) return lfm_host_fail(h, LFM_GPU_ERR_INVALID_ARG, __VA_ARGS__)
#define UNSUPPORTED(...) return lfm_host_fail(h, LFM_GPU_ERR_UNSUPPORTED, __VA_ARGS__)

/* Rows of `what`: aligned, of a stride that covers them. */
lfm_gpu_status_t check_rows(lfm_gpu_moe_t *h, const char *what, const void *p, size_t stride, uint32_t type,
                            size_t values) {
    if (!p) FAIL("%s is null", what);
    if (misaligned(p) || stride * type_bytes(type) % 16)
        FAIL("%s: rows must start on 16-byte boundaries (pointer %p, token stride %zu)", what, p, stride);
    if (stride < values || stride > ((size_t)1 << 40)) FAIL("%s: token stride %zu for rows of %zu values", what, stride, values);
    return LFM_GPU_OK;
}

lfm_gpu_status_t view_cache(lfm_gpu_moe_t *h, const lfm_gpu_kv_t *kv, const lfm_gpu_kv_batch_t *bt, KvDev *k,
                            BatchDev *b) {
    if (!kv || !bt) FAIL("null cache or batch descriptor");
    const size_t page = lfm_gpu_kv_page_bytes(kv->page_tokens, kv->n_kv_heads, kv->head_dim);
    if (!page)
        UNSUPPORTED("cache of %u-token pages, %u kv heads of %u values (pages of 16, 32, 64 or 128 tokens, 1..1024 "
                    "heads of 64 or 128 values)", kv->page_tokens, kv->n_kv_heads, kv->head_dim);
    if (!kv->pages || misaligned(kv->pages) || kv->n_pages == 0 || kv->n_pages > 0x7FFFFFFFu)
        FAIL("cache pool %p of %u pages (16-byte aligned, at least one page)", kv->pages, kv->n_pages);
    if (bt->n_seqs > (1u << 20) || bt->n_tokens > (1u << 24))
        FAIL("batch of %u sequences, %u tokens (at most 2^20 and 2^24)", bt->n_seqs, bt->n_tokens);
    if (bt->n_seqs && bt->n_tokens) {
        if (!bt->q_start || !bt->kv_len || !bt->page_table || bt->table_stride == 0)
            FAIL("batch offsets, lengths and page table must be given");
        if (misaligned(bt->q_start, 4) || misaligned(bt->kv_len, 4) || misaligned(bt->page_table, 4))
            FAIL("batch offsets, lengths and page table must be 4-byte aligned");
        if ((uint64_t)bt->table_stride * kv->page_tokens > 0x7FFFFFFFull)
            FAIL("page table of %u entries a sequence: more than 2^31 tokens", bt->table_stride);
    }
    k->pages = static_cast<uint8_t *>(kv->pages);
    k->n_pages = kv->n_pages;
    k->page_tokens = kv->page_tokens;
    k->page_shift = kv->page_tokens == 16 ? 4 : kv->page_tokens == 32 ? 5 : kv->page_tokens == 64 ? 6 : 7;
    k->hkv = kv->n_kv_heads;
    k->page_bytes = page;
    k->head_bytes = page / kv->n_kv_heads;
    k->codes = kv->page_tokens * (kv->head_dim / 2);
    k->half = (uint32_t)(k->head_bytes / 2);
    *b = BatchDev{bt->n_seqs, bt->n_tokens, bt->table_stride, bt->table_stride * kv->page_tokens, bt->q_start, bt->kv_len, bt->page_table};
    return LFM_GPU_OK;
}

template <class F>
lfm_gpu_status_t launch(lfm_gpu_moe_t *h, const HostView &v, AttnKernelId id, const char *what, cudaStream_t s,
                        F &&fn) {
    OnDevice g(v.device);
    const cudaError_t e = lfm_host_timed(
        h, id, s, [](void *f) -> cudaError_t { return (*static_cast<std::remove_reference_t<F> *>(f))(); }, &fn);
    return e == cudaSuccess ? LFM_GPU_OK : lfm_host_cuda_fail(h, e, what);
}

}  // namespace

LFM_API size_t lfm_gpu_kv_page_bytes(uint32_t page_tokens, uint32_t n_kv_heads, uint32_t head_dim) {
    if ((head_dim != 64 && head_dim != 128) || n_kv_heads == 0 || n_kv_heads > 1024) return 0;
    if (page_tokens != 16 && page_tokens != 32 && page_tokens != 64 && page_tokens != 128) return 0;
    return (size_t)n_kv_heads * 2 * page_tokens * (head_dim / 2 + head_dim / 16);
}

LFM_API lfm_gpu_status_t lfm_gpu_add_rmsnorm(lfm_gpu_moe_t *h, const float *x, const void *delta, uint32_t delta_type,
                                             uint32_t T, uint32_t D, const float *weight, float eps, float *x_out,
                                             void *xb, uint32_t xb_type, void *q8, void *stream) {
    if (!h) return LFM_GPU_ERR_INVALID_ARG;
    if (D == 0 || D % 256 || D > 8192) UNSUPPORTED("D=%u must be a multiple of 256 up to 8192", D);
    if (T > (1u << 24)) FAIL("T=%u above 2^24 rows", T);
    if ((delta && !type_ok(delta_type)) || (xb && !type_ok(xb_type)))
        UNSUPPORTED("types %u and %u (F32=0, F16=1, BF16=30)", delta_type, xb_type);
    if (!(eps >= 0.0f) || isinf(eps)) FAIL("eps=%g", (double)eps);
    if (T == 0) return LFM_GPU_OK; /* empty tensors have null pointers */
    if (!x_out && !xb && !q8) FAIL("no output asked for");
    if (!x) FAIL("x is null");
    if (misaligned(x) || misaligned(delta) || misaligned(weight) || misaligned(x_out) || misaligned(xb) || misaligned(q8, 4))
        FAIL("x, delta, weight, x_out and xb must be 16-byte aligned, q8 4-byte aligned");
    const HostView v = lfm_host_view(h);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    return launch(h, v, AK_NORM, "add_rmsnorm", s, [&] {
        return lfm_launch_add_rmsnorm(x, delta, delta_type, T, D, weight, eps, x_out, xb, xb_type,
                                      static_cast<uint8_t *>(q8), s, v.pdl);
    });
}

LFM_API lfm_gpu_status_t lfm_gpu_q8k_read(lfm_gpu_moe_t *h, const void *q8, uint32_t rows, uint32_t D, uint32_t type,
                                          void *out, void *stream) {
    if (!h) return LFM_GPU_ERR_INVALID_ARG;
    if (D == 0 || D % 256 || D > 8192) UNSUPPORTED("D=%u must be a multiple of 256 up to 8192", D);
    if (!type_ok(type)) UNSUPPORTED("type %u (F32=0, F16=1, BF16=30)", type);
    if (rows > (1u << 24)) FAIL("%u rows: above 2^24", rows);
    if (rows == 0) return LFM_GPU_OK;
    if (!q8 || !out || misaligned(q8, 4) || misaligned(out)) FAIL("q8 (4-byte aligned) and out (16-byte aligned) must be given");
    const HostView v = lfm_host_view(h);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    return launch(h, v, AK_Q8K_READ, "q8k_read", s, [&] {
        return lfm_launch_q8k_read(static_cast<const uint8_t *>(q8), rows, D, type, out, s, v.pdl);
    });
}

LFM_API lfm_gpu_status_t lfm_gpu_kv_append(lfm_gpu_moe_t *h, const lfm_gpu_kv_t *kv, const lfm_gpu_kv_batch_t *batch,
                                           const lfm_gpu_rope_t *rope, uint32_t type, uint32_t n_heads, const void *q,
                                           size_t q_stride, void *q_out, size_t q_out_stride, const void *k,
                                           size_t k_stride, const void *v, size_t v_stride, void *stream) {
    if (!h) return LFM_GPU_ERR_INVALID_ARG;
    AppendArgs a{};
    lfm_gpu_status_t st = view_cache(h, kv, batch, &a.kv, &a.bt);
    if (st != LFM_GPU_OK) return st;
    if (!type_ok(type)) UNSUPPORTED("type %u (F32=0, F16=1, BF16=30)", type);
    if (!q && !k && !v) FAIL("neither q nor k and v given");
    if (!k != !v) FAIL("k and v come together");
    if (q && (n_heads == 0 || n_heads > 65535)) FAIL("n_heads=%u", n_heads);
    if (rope) {
        if (rope->rot_dim % 16 || rope->rot_dim > kv->head_dim)
            UNSUPPORTED("rot_dim=%u must be a multiple of 16 up to head_dim=%u", rope->rot_dim, kv->head_dim);
        if (rope->rot_dim && (!rope->cos || !rope->sin || rope->n_pos == 0)) FAIL("rotation without its tables");
        if (misaligned(rope->cos) || misaligned(rope->sin) || misaligned(rope->q_norm) || misaligned(rope->k_norm))
            FAIL("cos, sin, q_norm and k_norm must be 16-byte aligned");
        if ((rope->q_norm || rope->k_norm) && (!(rope->eps >= 0.0f) || isinf(rope->eps))) FAIL("eps=%g", (double)rope->eps);
        a.rp = RopeDev{rope->cos, rope->sin, rope->q_norm, rope->k_norm, rope->n_pos, rope->rot_dim, rope->pairs != 0, rope->eps};
    }
    if (batch->n_seqs == 0 || batch->n_tokens == 0) return LFM_GPU_OK;
    if (q) {
        st = check_rows(h, "q", q, q_stride, type, (size_t)n_heads * kv->head_dim);
        if (st == LFM_GPU_OK) st = check_rows(h, "q_out", q_out, q_out_stride, type, (size_t)n_heads * kv->head_dim);
        if (st != LFM_GPU_OK) return st;
    }
    if (k) {
        st = check_rows(h, "k", k, k_stride, type, (size_t)kv->n_kv_heads * kv->head_dim);
        if (st == LFM_GPU_OK) st = check_rows(h, "v", v, v_stride, type, (size_t)kv->n_kv_heads * kv->head_dim);
        if (st != LFM_GPU_OK) return st;
    }
    const HostView hv = lfm_host_view(h);
    a.n_heads = q ? n_heads : 0;
    a.q = q; a.k = k; a.v = v; a.q_out = q_out;
    a.q_stride = q_stride; a.q_out_stride = q_out_stride; a.k_stride = k_stride; a.v_stride = v_stride;
    a.err = hv.err;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    return launch(h, hv, AK_APPEND, "kv_append", s,
                  [&] { return lfm_launch_kv_append(a, kv->head_dim, type, s, hv.pdl); });
}

LFM_API lfm_gpu_status_t lfm_gpu_kv_read(lfm_gpu_moe_t *h, const lfm_gpu_kv_t *kv, const lfm_gpu_kv_batch_t *batch,
                                         uint32_t type, void *k_out, void *v_out, void *stream) {
    if (!h) return LFM_GPU_ERR_INVALID_ARG;
    ReadArgs a{};
    lfm_gpu_status_t st = view_cache(h, kv, batch, &a.kv, &a.bt);
    if (st != LFM_GPU_OK) return st;
    if (!type_ok(type)) UNSUPPORTED("type %u (F32=0, F16=1, BF16=30)", type);
    if (batch->n_seqs == 0 || batch->n_tokens == 0) return LFM_GPU_OK;
    if (!k_out || !v_out || misaligned(k_out) || misaligned(v_out)) FAIL("k_out and v_out must be given, 16-byte aligned");
    const HostView hv = lfm_host_view(h);
    a.k_out = k_out; a.v_out = v_out;
    a.err = hv.err;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    return launch(h, hv, AK_KV_READ, "kv_read", s,
                  [&] { return lfm_launch_kv_read(a, kv->head_dim, type, s, hv.pdl); });
}

LFM_API lfm_gpu_status_t lfm_gpu_attn_forward(lfm_gpu_moe_t *h, const lfm_gpu_kv_t *kv, const lfm_gpu_kv_batch_t *batch,
                                              uint32_t n_heads, float scale, int causal, uint32_t window, float softcap,
                                              uint32_t type, const void *q, size_t q_stride, void *out,
                                              size_t out_stride, void *stream) {
    if (!h) return LFM_GPU_ERR_INVALID_ARG;
    AttnArgs a{};
    lfm_gpu_status_t st = view_cache(h, kv, batch, &a.kv, &a.bt);
    if (st != LFM_GPU_OK) return st;
    if (!type_ok(type)) UNSUPPORTED("type %u (F32=0, F16=1, BF16=30)", type);
    if (n_heads == 0 || n_heads > 65535 || n_heads % kv->n_kv_heads)
        FAIL("n_heads=%u is not a multiple of the cache's %u", n_heads, kv->n_kv_heads);
    if ((uint64_t)batch->n_tokens * n_heads > 0x7FFFFFFFull) FAIL("%u tokens of %u heads: above 2^31 rows", batch->n_tokens, n_heads);
    if (!isfinite(scale)) FAIL("scale=%g", (double)scale);
    if (!(softcap >= 0.0f) || isinf(softcap)) FAIL("softcap=%g", (double)softcap);
    if (window && !causal) FAIL("a window needs causal attention");
    if (batch->n_seqs == 0 || batch->n_tokens == 0) return LFM_GPU_OK;
    st = check_rows(h, "q", q, q_stride, type, (size_t)n_heads * kv->head_dim);
    if (st == LFM_GPU_OK) st = check_rows(h, "out", out, out_stride, type, (size_t)n_heads * kv->head_dim);
    if (st != LFM_GPU_OK) return st;
    const HostView hv = lfm_host_view(h);
    a.n_heads = n_heads;
    a.group = n_heads / kv->n_kv_heads;
    a.scale = scale;
    /* a product is at most 65504^2 head_dim: above this cap the argument of tanh is below 2^-12, and tanh itself in fp32 */
    a.softcap = softcap > fabs((double)scale) * 4096.0 * 65504.0 * 65504.0 * kv->head_dim ? 0.0f : softcap;
    a.causal = causal != 0;
    a.window = window;
    a.type = type;
    a.q = q; a.out = out;
    a.q_stride = q_stride; a.out_stride = out_stride;
    a.err = hv.err;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    OnDevice g(hv.device);
    void *scratch = nullptr;
    st = lfm_host_scratch(h, s, &scratch);
    if (st != LFM_GPU_OK) return st;
    const uint32_t span = a.bt.span;
    const uint32_t hint = batch->max_kv_len && batch->max_kv_len < span ? batch->max_kv_len : span;
    st = launch(h, hv, AK_ATTN, "attn_forward", s,
                [&] { return lfm_launch_attn(a, kv->head_dim, hint, hv.sm_count, scratch, s, hv.pdl); });
    return st == LFM_GPU_OK ? lfm_host_scratch_used(h, s) : st;
}

LFM_API lfm_gpu_status_t lfm_gpu_attn_reserve(lfm_gpu_moe_t *h) {
    if (!h) return LFM_GPU_ERR_INVALID_ARG;
    OnDevice g(lfm_host_view(h).device);
    void *scratch = nullptr;
    return lfm_host_scratch(h, nullptr, &scratch);
}
