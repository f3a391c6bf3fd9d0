/*
 * Internal (non-exported) interfaces of the attention side of
 * liblfm_gpu_moe.so (include/lfm_gpu_attn.h): device views of the caller's
 * descriptors, the kernel launchers and what the entry points use of a handle.
 */
#ifndef LFM_ATTN_INTERNAL_H
#define LFM_ATTN_INTERNAL_H

#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "lfm_gpu_moe.h"

/* Device error word bit: a page id, position or batch offset out of range. */
#define LFM_DEVERR_PAGE 0x8u

struct KvDev {
    uint8_t *pages;
    uint32_t n_pages, page_tokens, page_shift, hkv;
    size_t page_bytes, head_bytes; /* head_bytes: one kv head of one page, K and V */
    uint32_t codes, half;          /* bytes of K codes; bytes of K codes and scales (V starts there) */
};

struct BatchDev {
    uint32_t n_seqs, n_tokens, table_stride, span; /* span: tokens that a sequence's entries hold, below 2^31 */
    const int32_t *q_start, *kv_len, *page_table;
};

struct RopeDev {
    const float *cos, *sin, *q_norm, *k_norm;
    uint32_t n_pos, rot_dim;
    int pairs;
    float eps;
};

struct AppendArgs {
    KvDev kv;
    BatchDev bt;
    RopeDev rp;
    uint32_t n_heads; /* of q; 0: keys and values only */
    const void *q, *k, *v;
    void *q_out;
    size_t q_stride, q_out_stride, k_stride, v_stride;
    uint32_t *err;
};

struct ReadArgs {
    KvDev kv;
    BatchDev bt;
    void *k_out, *v_out;
    uint32_t *err;
};

struct AttnArgs {
    KvDev kv;
    BatchDev bt;
    uint32_t n_heads, group;
    float scale, softcap;
    int causal;
    uint32_t window, type;
    const void *q;
    void *out;
    size_t q_stride, out_stride;
    uint32_t *err;
};

cudaError_t lfm_launch_add_rmsnorm(const float *x, const void *delta, uint32_t delta_type, uint32_t T, uint32_t D,
                                   const float *weight, float eps, float *x_out, void *xb, uint32_t xb_type,
                                   uint8_t *q8, cudaStream_t s, bool pdl);
cudaError_t lfm_launch_q8k_read(const uint8_t *q8, uint32_t rows, uint32_t D, uint32_t type, void *out, cudaStream_t s,
                                bool pdl);
cudaError_t lfm_launch_kv_append(const AppendArgs &a, uint32_t head_dim, uint32_t type, cudaStream_t s, bool pdl);
cudaError_t lfm_launch_kv_read(const ReadArgs &a, uint32_t head_dim, uint32_t type, cudaStream_t s, bool pdl);
/* max_kv_len bounds the blocks launched, scratch holds the parts of split sequences (LFM_ATTN_SCRATCH_BYTES, the leading
 * LFM_ATTN_COUNTS words zero; the kernels leave them zero). */
cudaError_t lfm_launch_attn(const AttnArgs &a, uint32_t head_dim, uint32_t max_kv_len, int sm_count, void *scratch,
                            cudaStream_t s, bool pdl);
/* The tensor-core kernel for the sequences of more than `above` rows (token, head of a group). */
struct TilePlan {
    uint64_t above;
    uint64_t blocks;               /* of keys, in the longest walk by max_kv_len (what a row sees at most) */
    uint64_t cost;                 /* blocks that the busiest SM walks */
    uint32_t tiles, parts;         /* tiles of rows of one kv head, at most; most parts of one */
    uint32_t *counts;              /* zero before and after */
    float *part;
};
TilePlan lfm_attn_tile_plan(const AttnArgs &a, uint32_t head_dim, uint64_t above, uint32_t max_kv_len, int sm_count);
cudaError_t lfm_launch_attn_tile(const AttnArgs &a, uint32_t head_dim, const TilePlan &plan, int sm_count, void *scratch,
                                 cudaStream_t s, bool pdl);
#define LFM_ATTN_COUNTS 4096u /* words */
#define LFM_ATTN_BLOCKS 1022u /* most blocks of the few-row kernel: two parts each, 32 x (64 + 2) or 16 x (128 + 2) floats */
#define LFM_ATTN_TILES 592u   /* most parts of split tiles: 256 x (128 + 2) floats, more than the former */
#define LFM_ATTN_SCRATCH_BYTES (LFM_ATTN_COUNTS * sizeof(uint32_t) + (size_t)LFM_ATTN_TILES * 256 * 130 * 4)

/* ---- the handle, as lfm_gpu_moe.cu keeps it ------------------------------ */
enum AttnKernelId { AK_NORM, AK_Q8K_READ, AK_APPEND, AK_KV_READ, AK_ATTN };
struct HostView {
    int device, sm_count;
    bool pdl;
    uint32_t *err;
};
HostView lfm_host_view(lfm_gpu_moe_t *h);
lfm_gpu_status_t lfm_host_fail(lfm_gpu_moe_t *h, lfm_gpu_status_t st, const char *fmt, ...);
lfm_gpu_status_t lfm_host_cuda_fail(lfm_gpu_moe_t *h, cudaError_t e, const char *what);
/* fn(ctx), the launch, between the profile's events where profiling is on.
 * (The launch statistics of a handle stay those of its last MoE forward.) */
cudaError_t lfm_host_timed(lfm_gpu_moe_t *h, AttnKernelId id, cudaStream_t s, cudaError_t (*fn)(void *), void *ctx);

/* The handle's attention scratch for work on `s`, allocated on first use (not
 * while `s` captures); work that other streams still do on it comes first. */
lfm_gpu_status_t lfm_host_scratch(lfm_gpu_moe_t *h, cudaStream_t s, void **out);
/* ... and after that work's launch. */
lfm_gpu_status_t lfm_host_scratch_used(lfm_gpu_moe_t *h, cudaStream_t s);

#endif /* LFM_ATTN_INTERNAL_H */
