/*
 * lfm_gpu_attn.h -- C-ABI of the attention side of an lfm2moe layer on B200
 * (sm_100a): what a layer does before its MoE FFN (lfm_gpu_moe.h).
 *
 *   lfm_gpu_add_rmsnorm   residual addition, RMSNorm and block_q8_K output
 *   lfm_gpu_kv_append     per-head RMSNorm and rotation of q and k, keys and
 *                         values into a paged cache of 4-bit codes
 *   lfm_gpu_attn_forward  grouped-query attention over that cache: single
 *                         tokens, verify batches, prompts and chunks
 *   lfm_gpu_q8k_read, lfm_gpu_kv_read   the values that 8- and 4-bit data stand for
 *
 * Conventions are those of lfm_gpu_moe.h: the same handle (its device, its
 * error text, its device error word, its scratch), the same status codes, no
 * CPU fallback, one host thread per handle, `stream` a cudaStream_t as void*
 * (NULL = the CUDA default stream).  Further:
 *  - every pointer is device memory of the handle's device; the caller owns
 *    it, and the library keeps no address after a call returns;
 *  - every call is asynchronous on `stream` and may be captured into a CUDA
 *    graph (lfm_gpu_attn_forward: after lfm_gpu_attn_reserve);
 *  - rows are [tokens][heads][head_dim] with a token stride in elements, so q,
 *    k and v may be slices of one projection's output; a row starts on a
 *    16-byte boundary (checked);
 *  - `type` is the GGML type of the 16- or 32-bit tensors: 0 (F32), 1 (F16)
 *    or 30 (BF16);
 *  - a bad page id, a position outside the page table or the rotation table,
 *    offsets out of order or range and, for attention, a length that the page
 *    table has no room for are found on the device: the access is skipped, the
 *    sequence of bad offsets or length is passed over (its rows are left
 *    alone), and the next lfm_gpu_moe_sync returns LFM_GPU_ERR_DEVICE_CHECK.
 */
#ifndef LFM_GPU_ATTN_H
#define LFM_GPU_ATTN_H

#include "lfm_gpu_moe.h"

#ifdef __cplusplus
extern "C" {
#endif

#define LFM_GPU_TYPE_F32 0u
#define LFM_GPU_TYPE_F16 1u
#define LFM_GPU_TYPE_BF16 30u

/* One layer's pool of cache pages, 16-byte aligned: page p starts at
 * pages + p * lfm_gpu_kv_page_bytes(...) and holds, for each kv head in turn,
 *   K codes  [page_tokens][head_dim / 2] bytes
 *   K scales [page_tokens][head_dim / 32] fp16
 *   V codes and V scales, the same.
 * A head's vector is quantised in blocks of 32 values: value = d * (code - 8)
 * with the fp16 scale d = m / -8, m the value of largest magnitude in the
 * block (the positive one on a tie), code = floor(value / d + 8.5) within
 * 0..15 -- the arithmetic of GGUF's Q4_0, 4.5 bits a value.  Values outside
 * fp16's finite range are stored as +-65504 and NaN as 0, so a cache never
 * holds a non-finite number.  The codes of each 64-wide span of a head lie in
 * eight little-endian 32-bit words: nibble n of word w is value
 * 32 * (n / 4) + 4 * w + n % 4 of the span.
 * head_dim 64 or 128; page_tokens 16, 32, 64 or 128. */
typedef struct {
    void *pages;
    uint32_t n_pages, page_tokens, n_kv_heads, head_dim;
} lfm_gpu_kv_t;

/* Bytes of a page; 0 for a shape that is not supported.  Host only. */
size_t lfm_gpu_kv_page_bytes(uint32_t page_tokens, uint32_t n_kv_heads, uint32_t head_dim);

/* A ragged batch.  Sequence b owns the q rows q_start[b] .. q_start[b + 1] of
 * the call (none is fine); kv_len[b] tokens of it are in the cache, those rows'
 * tokens last, so its row i is at position kv_len[b] - rows + i; token j lies
 * in page page_table[b * table_stride + j / page_tokens].  Rows outside every
 * sequence (padding) are left alone.  Entries past a sequence's last page are
 * not read, nor by attention with a window those of pages that end before the
 * first token that a row of the sequence sees: such pages may be given back. */
typedef struct {
    uint32_t n_seqs;
    uint32_t n_tokens;      /* rows of q (an upper bound of q_start[n_seqs])          */
    uint32_t table_stride;  /* page table entries a sequence                          */
    uint32_t max_kv_len;    /* plans the work, any value is safe; 0: the table's span */
    const int32_t *q_start;     /* [n_seqs + 1] */
    const int32_t *kv_len;      /* [n_seqs]     */
    const int32_t *page_table;  /* [n_seqs][table_stride] */
} lfm_gpu_kv_batch_t;

/* What happens to q and k before the cache.  q_norm / k_norm: fp32 [head_dim]
 * weights of a per-head RMSNorm, or NULL for none.  Rotation: the first
 * rot_dim values of a head (a multiple of 16, 0: none) by the angles whose
 * cosines and sines are cos / sin, fp32 [n_pos][rot_dim / 2], row = position:
 * (a, b) -> (a cos - b sin, b cos + a sin) on the pairs (i, i + rot_dim / 2),
 * or with `pairs` on neighbours (2i, 2i + 1). */
typedef struct {
    const float *cos, *sin;
    uint32_t n_pos, rot_dim;
    int pairs;
    float eps;
    const float *q_norm, *k_norm;
} lfm_gpu_rope_t;

/* y = x + delta (delta NULL: y = x); x_out = y;  n = y / sqrt(mean(y^2) + eps)
 * * weight;  xb = n as xb_type, q8 = n as block_q8_K [T][D / 256] (292 bytes
 * each, 4-byte aligned).  x and x_out fp32 [T][D] (may be the same memory),
 * delta of delta_type, weight fp32 [D] (NULL: ones); x_out, xb and q8 may each
 * be NULL.  D a multiple of 256, at most 8192.  A block of q8 with a NaN or an
 * infinity in it has that scale and codes of 0: its values read as NaN.  The
 * batched, stand-alone counterpart of lfm2_rmsnorm_quantize_q8_K
 * (tools/lfm2_decode_1x4.c:93-196) with the residual's addition in front; its
 * sums run in another order. */
lfm_gpu_status_t lfm_gpu_add_rmsnorm(lfm_gpu_moe_t *h, const float *x, const void *delta, uint32_t delta_type,
                                     uint32_t T, uint32_t D, const float *weight, float eps, float *x_out, void *xb,
                                     uint32_t xb_type, void *q8, void *stream);

/* out [rows][D] of `type` = the values d * q of block_q8_K rows. */
lfm_gpu_status_t lfm_gpu_q8k_read(lfm_gpu_moe_t *h, const void *q8, uint32_t rows, uint32_t D, uint32_t type,
                                  void *out, void *stream);

/* Rows of q [n_tokens][n_heads][head_dim] normalised and rotated into q_out
 * (may be q); k and v [n_tokens][n_kv_heads][head_dim], k normalised and
 * rotated, into the cache at their positions.  q == NULL: keys and values
 * only.  k == v == NULL: q only.  The strides are in elements. */
lfm_gpu_status_t lfm_gpu_kv_append(lfm_gpu_moe_t *h, const lfm_gpu_kv_t *kv, const lfm_gpu_kv_batch_t *batch,
                                   const lfm_gpu_rope_t *rope, uint32_t type, uint32_t n_heads, const void *q,
                                   size_t q_stride, void *q_out, size_t q_out_stride, const void *k, size_t k_stride,
                                   const void *v, size_t v_stride, void *stream);

/* The values that the cache holds for the batch's rows, [n_tokens][n_kv_heads][head_dim]
 * of `type`, dense (a batch whose rows are whole sequences reads them back whole). */
lfm_gpu_status_t lfm_gpu_kv_read(lfm_gpu_moe_t *h, const lfm_gpu_kv_t *kv, const lfm_gpu_kv_batch_t *batch,
                                 uint32_t type, void *k_out, void *v_out, void *stream);

/* out = softmax(z) V per row and head, z = scale * q . k, or with softcap > 0
 * softcap * tanh(scale * q . k / softcap), within 2^-20 of the score or 2^-15
 * for any cap.  Head h reads kv head h / (n_heads / n_kv_heads).  causal != 0:
 * the row at position p sees the keys j <= p, with window > 0 only those with
 * j > p - window; causal == 0: every key (window must be 0).  A row that sees
 * no key is 0, one whose q holds a NaN is NaN.  q and out
 * [n_tokens][n_heads][head_dim] of `type`, strides in elements.  For the tensor
 * cores q is rounded to fp16 whatever its type (beyond its range +-65504, below
 * 2^-14 to multiples of 2^-24), the cache's values and the probabilities too;
 * products and sums are fp32. */
lfm_gpu_status_t lfm_gpu_attn_forward(lfm_gpu_moe_t *h, const lfm_gpu_kv_t *kv, const lfm_gpu_kv_batch_t *batch,
                                      uint32_t n_heads, float scale, int causal, uint32_t window, float softcap,
                                      uint32_t type, const void *q, size_t q_stride, void *out, size_t out_stride,
                                      void *stream);

/* Allocate the scratch in which lfm_gpu_attn_forward joins the parts of long
 * sequences (79 MB per handle, whatever is asked later).  The first forward does it otherwise,
 * which a stream capture does not allow.  Calls on several streams (per-thread
 * default streams of several threads among them) are ordered among each other
 * where they share the scratch.  Captured calls are not: keep those of one
 * capture on one stream, or order them, and replay one graph at a time per
 * handle, with no call beside it. */
lfm_gpu_status_t lfm_gpu_attn_reserve(lfm_gpu_moe_t *h);

#ifdef __cplusplus
}
#endif

#endif /* LFM_GPU_ATTN_H */
