/*
 * Grouped-query attention over the paged 4-bit cache for few query rows a
 * sequence: single tokens, verify batches, short chunks.
 *
 *   z_j = scale q . k_j,  m = max z,  out = sum e^(z_j - m) v_j / sum e^(z_j - m)
 *
 * One pass over the keys with a running reference m and sum.  The products run
 * on mma.sync m16n8k16 with the KEYS as the M dimension: S^T = K Q^T and
 * O^T = V^T P^T, so one token's few heads fill the 8 columns of N, and the
 * 4-bit operand is the A fragment, built in registers from the codes:
 *   - a nibble c OR-ed into an fp16 exponent is 1024 + c (bits 0-3) or 64 + c
 *     (bits 4-7): one logic instruction for two codes, a shift for four;
 *   - K: the offsets (1032 and 72 with the code's own 8) are taken off through
 *     the accumulator's start value, -sum of offset * q, and a block's scale is
 *     multiplied into its 32-value partial sum in fp32: K enters exact;
 *   - V: offset subtracted and scale multiplied in fp16 pairs (the product is
 *     rounded to fp16: 2^-12 relative, under the output's rounding);
 *   - P: e^(z - m) in fp16 as the B fragment, transposed by movmatrix.  m only
 *     moves when a score passes it by 2^8, so p <= 256, and the sum is fp32.
 * A warp takes 4608-byte blocks of keys and values (64 keys of 64 values, 32 of
 * 128) through its own ring of bulk copies; the eight warps of a block split
 * the keys and are joined in shared memory, blocks that split a long sequence
 * through scratch: the last to finish joins the parts in their order (the same
 * bits on every run).
 */
#include "attn_device.cuh"

namespace {

constexpr int kWarps = 8, kThreads = kWarps * 32, kStages = 3;

template <int D>
struct Cfg {
    static constexpr int kKeys = D == 64 ? 64 : 32;         /* keys of a block      */
    static constexpr int kBytes = kKeys * (D + D / 8);      /* 4608                 */
    static constexpr int kSpans = D / 64;
    static constexpr int kRing = kWarps * kStages * kBytes; /* shared memory        */
};

__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
__device__ __forceinline__ uint2 lds64(uint32_t a) {
    uint2 v;
    asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(a));
    return v;
}
__device__ __forceinline__ uint32_t lds32(uint32_t a) {
    uint32_t v;
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(a));
    return v;
}
/* The D / 32 scales of a key. */
template <int N>
__device__ __forceinline__ void lds_scales(uint32_t a, uint32_t (&v)[N]) {
    if constexpr (N == 2) {
        const uint2 u = lds64(a);
        v[0] = u.x; v[1] = u.y;
    } else {
        v[0] = lds32(a);
    }
}
__device__ __forceinline__ float2 half2_of(uint32_t u) { return __half22float2(*reinterpret_cast<const __half2 *>(&u)); }
__device__ __forceinline__ void store4(void *p, uint32_t type, size_t at, const float (&v)[4]) {
    if (type == 0) lfm_store<4>(static_cast<float *>(p) + at, v);
    else if (type == 1) lfm_store<4>(static_cast<__half *>(p) + at, v);
    else lfm_store<4>(static_cast<__nv_bfloat16 *>(p) + at, v);
}

struct RowsPlan {
    uint32_t n_splits, chunk; /* blocks of keys a split takes (the last takes what is left) */
    uint32_t extra;           /* blocks past n_seqs that walk the further column tiles       */
    uint64_t most;            /* rows of the longest sequence that is this kernel's          */
    uint64_t tiles;           /* n_seqs and the most further tiles that there can be         */
    uint64_t units;           /* (tile, head) units that the scratch has room for            */
    float *parts;             /* [units * n_splits][cols][D + 2]                             */
    uint32_t *counts;         /* [units], zero between calls                                 */
};

/* A warp's issue and wait state over its blocks first, first + kWarps, ... */
template <int D>
struct Ring {
    const AttnArgs &A;
    int b;
    uint32_t kvh, smem, n;   /* n: blocks of this warp */
    int64_t first, end;      /* first block; keys that exist */
    uint64_t *bars;
    uint32_t id, next;       /* page ids of 8 blocks, four pieces each, a lane a piece */

    /* Page of piece lane % 4 of block i8 + lane / 4. */
    __device__ __forceinline__ uint32_t lookup(uint32_t i8) {
        constexpr int kK = Cfg<D>::kKeys;
        const uint32_t lane = threadIdx.x & 31, i = i8 + lane / 4, j = lane & 3, P = A.kv.page_tokens;
        const int64_t key = (first + (int64_t)i * kWarps) * kK + (P < kK ? j * P : 0);
        if (i >= n || key >= end || (P < kK && j * P >= kK) || (P == kK && j)) return ~0u - 1; /* nothing to copy */
        const int64_t at = key >> A.kv.page_shift;
        uint32_t page = ~0u;
        if (at < (int64_t)A.bt.table_stride) page = (uint32_t)A.bt.page_table[(size_t)b * A.bt.table_stride + (size_t)at];
        if (page >= A.kv.n_pages) {
            atomicOr(A.err, LFM_DEVERR_PAGE);
            return ~0u;
        }
        return page;
    }

    /* Copies of block i into its stage: pages of up to a block whole, a longer page's four parts. */
    __device__ __forceinline__ void issue(uint32_t i) {
        constexpr uint32_t kK = Cfg<D>::kKeys;
        if ((i & 7) == 0 && i) id = next;
        const uint32_t lane = threadIdx.x & 31, j = lane & 3, P = A.kv.page_tokens;
        if (lane / 4 == (i & 7)) {
            uint64_t *bar = bars + i % kStages;
            if (id < A.kv.n_pages) {
                const uint8_t *page = A.kv.pages + (size_t)id * A.kv.page_bytes + (size_t)kvh * A.kv.head_bytes;
                uint32_t to = smem + i % kStages * Cfg<D>::kBytes, bytes;
                if (P <= kK) {
                    bytes = P * (D + D / 8);
                    to += j * bytes;
                } else {
                    const uint32_t in = (uint32_t)((first + (int64_t)i * kWarps) * kK) & (P - 1);
                    bytes = (j & 1) ? kK * (D / 16) : kK * (D / 2);
                    page += (j & 2 ? A.kv.half : 0) + ((j & 1) ? A.kv.codes + in * (D / 16) : in * (D / 2));
                    to += (j & 2 ? kK * (D / 2 + D / 16) : 0) + ((j & 1) ? kK * (D / 2) : 0);
                }
                lfm_mbar_arrive_tx(bar, bytes);
                asm volatile(
                    "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(to),
                    "l"(page), "r"(bytes), "r"(lfm_smem_u32(bar))
                    : "memory");
            } else {
                lfm_mbar_arrive(bar);
            }
        }
        if ((i & 7) == 4) next = lookup((i & ~7u) + 8);
    }
};

template <int D, int NT, bool kCap>
__global__ void __launch_bounds__(kThreads, D * NT <= 128 ? 2 : 1) k_attn_rows(AttnArgs A, RowsPlan P) {
    using C = Cfg<D>;
    constexpr int kCols = 8 * NT, kS = C::kSpans, kPitch = D + 4;
    static_assert(kWarps * kCols * kPitch * 4 <= C::kRing, "the join fits the ring");
    extern __shared__ __align__(128) uint8_t ring[];
    __shared__ uint64_t s_bar[kWarps][kStages];
    __shared__ float s_m[kWarps][kCols], s_l[kWarps][kCols];
    __shared__ int64_t s_hi[kCols], s_lo[kCols];
    __shared__ int s_tile[2], s_last;
    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const uint32_t kvh = blockIdx.y, split = blockIdx.z, G = A.group;
    if (lane < kStages) lfm_mbar_init(&s_bar[warp][lane], 4);
    lfm_fence_mbar_init();
    __syncwarp();
    uint32_t phases = 0; /* parity of each stage's next wait */
    lfm_pdl_wait();
    const float sc = kCap ? A.softcap * 1.44269504f : fmaxf(fabsf(A.scale) * 1.44269504f, 1e-30f);

    for (uint64_t z = blockIdx.x; z < P.tiles; z += P.extra) {
        /* ---- the tile: its sequence and columns ---- */
        int b = (int)z;
        uint32_t ct = 0;
        if (z >= A.bt.n_seqs) {
            /* the (z - n_seqs)-th of the tiles behind each sequence's first, in order */
            __syncthreads();
            if (warp == 0) lfm_find_tile(A.bt, G, kCols, 1, 0, P.most, z - A.bt.n_seqs, s_tile);
            __syncthreads();
            b = s_tile[0];
            if (b < 0) return;
            ct = (uint32_t)s_tile[1];
        }
        const int64_t q0 = A.bt.q_start[b], n_q = (int64_t)A.bt.q_start[b + 1] - q0, len = A.bt.kv_len[b];
        const bool good = lfm_sane(A.bt, q0, n_q) && len >= 0;
        if (!good && tid == 0) atomicOr(A.err, LFM_DEVERR_PAGE);
        const uint32_t row0 = ct * kCols; /* rows of a sequence: (token, head of the group), below 2^31 */
        const int64_t rows = n_q * G - row0;
        if (!good || rows <= 0 || (uint64_t)n_q * G > P.most) {
            if (z < A.bt.n_seqs) return;
            continue;
        }
        const uint32_t last = (uint32_t)(rows < kCols ? rows : kCols) - 1;
        /* what a row sees grows over the tile */
        int64_t lo0, hi0, lo1, hi1;
        lfm_visible(A, n_q, len, row0, lo0, hi0);
        lfm_visible(A, n_q, len, row0 + last, lo1, hi1);
        if (tid < kCols) {
            int64_t lo = 0, hi = 0;
            if (tid <= last) lfm_visible(A, n_q, len, row0 + tid, lo, hi);
            s_lo[tid] = lo;
            s_hi[tid] = hi;
        }
        const int64_t blk0 = lo0 / C::kKeys, blk1 = (hi1 + C::kKeys - 1) / C::kKeys;
        const int64_t n_blk = blk1 - blk0;
        /* splits that have blocks; a tile without any is split 0's */
        const uint64_t unit = z * gridDim.y + kvh;
        const uint32_t n_act = n_blk <= 0 || unit >= P.units ? 1u
                             : (uint32_t)min((int64_t)P.n_splits, (n_blk + P.chunk - 1) / P.chunk);
        if (split >= n_act) {
            if (z < A.bt.n_seqs) return;
            continue;
        }
        const int64_t from = blk0 + (int64_t)split * P.chunk;
        const int64_t to = split + 1 == n_act ? blk1 : from + P.chunk;
        const int64_t mine = to - from - warp;
        Ring<D> rg{A, b, kvh, lfm_smem_u32(ring) + warp * kStages * C::kBytes,
                   mine > 0 ? (uint32_t)((mine + kWarps - 1) / kWarps) : 0u, from + warp, len, s_bar[warp], 0, 0};
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncthreads(); /* s_lo, s_hi; the ring is free of an earlier tile's join, for the copies too */
        rg.id = rg.lookup(0);
#pragma unroll
        for (uint32_t i = 0; i < kStages; ++i)
            if (i < rg.n) rg.issue(i);

        /* ---- Q as B fragments: column g, values 64 s + 32 c + 8 t .. of the head ---- */
        uint32_t qf[NT][kS][2][4];
        float corr[NT][kS][2][2];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const uint32_t r = row0 + n * 8 + g;
            const bool on = n * 8 + g <= last;
            const size_t at = on ? (size_t)(q0 + r / G) * A.q_stride + ((size_t)kvh * G + r % G) * D : 0;
#pragma unroll
            for (int s = 0; s < kS; ++s)
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
                    if (on) lfm_load_q(A, at + 64 * s + 32 * c + 8 * t, A.scale < 0.0f && !kCap, v);
                    float h[8], sum = 0.0f;
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        h[i] = __half2float(__float2half_rn(v[i]));
                        sum = __fmaf_rn(h[i], (i & 1) ? 72.0f : 1032.0f, sum);
                    }
#pragma unroll
                    for (int i = 0; i < 4; ++i) qf[n][s][c][i] = lfm_pack2(h[i], h[4 + i], __half());
                    sum += __shfl_xor_sync(LFM_FULL_MASK, sum, 1);
                    sum += __shfl_xor_sync(LFM_FULL_MASK, sum, 2);
                    corr[n][s][c][0] = -__shfl_sync(LFM_FULL_MASK, sum, 8 * t);
                    corr[n][s][c][1] = -__shfl_sync(LFM_FULL_MASK, sum, 8 * t + 4);
                }
        }

        /* ---- the keys ---- */
        float o[NT][kS][2][2][4], m[NT][2], l[NT][2];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            m[n][0] = m[n][1] = LFM_NO_KEY;
            l[n][0] = l[n][1] = 0.0f;
#pragma unroll
            for (int s = 0; s < kS; ++s)
#pragma unroll
                for (int c = 0; c < 2; ++c)
#pragma unroll
                    for (int i = 0; i < 2; ++i) o[n][s][c][i][0] = o[n][s][c][i][1] = o[n][s][c][i][2] = o[n][s][c][i][3] = 0.0f;
        }
        const uint32_t sub = min(A.kv.page_tokens, (uint32_t)C::kKeys); /* keys of a contiguous piece */
        const uint32_t rk = g ^ (g >> 2);                     /* key of A row g (rows 8.. : + 8)            */
        const uint32_t ve = 2 * t ^ (t >> 1), vo = ve ^ 1;    /* keys of A columns 2 t and 2 t + 1 for V    */
        const float capz = kCap ? A.scale * 2.88539008f / A.softcap : 0.0f;
        bool ok = true;
        for (uint32_t i = 0; i < rg.n; ++i) {
            const uint32_t st = i % kStages;
            ok = __all_sync(LFM_FULL_MASK, lfm_mbar_wait(&s_bar[warp][st], (phases >> st) & 1, A.err));
            phases ^= 1u << st;
            if (!ok) break;
            const uint32_t buf = rg.smem + st * C::kBytes;
            const int64_t key0 = (rg.first + (int64_t)i * kWarps) * C::kKeys;
            const bool whole = key0 >= lo1 && key0 + C::kKeys <= hi0; /* every row sees every key */
            const bool tail = key0 + C::kKeys > len;                  /* slots that hold no token */
#pragma unroll 1
            for (uint32_t s16 = 0; s16 < C::kKeys; s16 += 16) {
                if (tail && key0 + s16 >= len) break;
                const uint32_t in = s16 & (sub - 1), base = buf + (s16 - in) * (D + D / 8);
                const uint32_t kc = base + in * (D / 2), ks = base + sub * (D / 2) + in * (D / 16);
                const uint32_t vc = kc + sub * (D / 2 + D / 16), vs = ks + sub * (D / 2 + D / 16);
                /* S^T: rows rk and rk + 8, columns 2 t and 2 t + 1 */
                float z4[NT][4];
                {
                    uint32_t d0[kS], d1[kS];
                    lds_scales<kS>(ks + rk * (D / 16), d0);
                    lds_scales<kS>(ks + (rk + 8) * (D / 16), d1);
#pragma unroll
                    for (int s = 0; s < kS; ++s) {
                        const uint2 x0 = lds64(kc + rk * (D / 2) + 32 * s + 8 * t);
                        const uint2 x1 = lds64(kc + (rk + 8) * (D / 2) + 32 * s + 8 * t);
                        const float2 e0 = half2_of(d0[s]), e1 = half2_of(d1[s]);
#pragma unroll
                        for (int c = 0; c < 2; ++c) {
                            const uint32_t u = __byte_perm(x0.x, x0.y, c ? 0x7632 : 0x5410);
                            const uint32_t w = __byte_perm(x1.x, x1.y, c ? 0x7632 : 0x5410);
                            const uint32_t a0[4] = {lfm_nib0(u), lfm_nib0(w), lfm_nib1(u), lfm_nib1(w)};
                            const uint32_t a1[4] = {lfm_nib0(u >> 8), lfm_nib0(w >> 8), lfm_nib1(u >> 8), lfm_nib1(w >> 8)};
                            const float f0 = c ? e0.y : e0.x, f1 = c ? e1.y : e1.x;
#pragma unroll
                            for (int n = 0; n < NT; ++n) {
                                float acc[4] = {corr[n][s][c][0], corr[n][s][c][1], corr[n][s][c][0], corr[n][s][c][1]};
                                mma16816(acc, a0, qf[n][s][c][0], qf[n][s][c][1]);
                                mma16816(acc, a1, qf[n][s][c][2], qf[n][s][c][3]);
                                if (s == 0 && c == 0) {
                                    z4[n][0] = acc[0] * f0; z4[n][1] = acc[1] * f0;
                                    z4[n][2] = acc[2] * f1; z4[n][3] = acc[3] * f1;
                                } else {
                                    z4[n][0] = __fmaf_rn(acc[0], f0, z4[n][0]); z4[n][1] = __fmaf_rn(acc[1], f0, z4[n][1]);
                                    z4[n][2] = __fmaf_rn(acc[2], f1, z4[n][2]); z4[n][3] = __fmaf_rn(acc[3], f1, z4[n][3]);
                                }
                            }
                        }
                    }
                }
                if (kCap) { /* tanh(x) = 1 - 2 / (1 + e^2x) */
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int j = 0; j < 4; ++j) z4[n][j] = __fmaf_rn(-2.0f, lfm_rcp(1.0f + lfm_ex2(z4[n][j] * capz)), 1.0f);
                }
                if (!whole) {
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const int64_t key = key0 + s16 + rk + (j >= 2 ? 8 : 0);
                            const uint32_t col = n * 8 + 2 * t + (j & 1);
                            if (key < s_lo[col] || key >= s_hi[col]) z4[n][j] = -INFINITY;
                        }
                }
                bool grow = false;
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int e = 0; e < 2; ++e)
                        grow |= __fmaf_rn(fmaxf(z4[n][e], z4[n][2 + e]), sc, -m[n][e]) > 8.0f;
                if (__any_sync(LFM_FULL_MASK, grow)) {
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            float x = fmaxf(z4[n][e], z4[n][2 + e]);
#pragma unroll
                            for (int k = 4; k < 32; k <<= 1) x = fmaxf(x, __shfl_xor_sync(LFM_FULL_MASK, x, k));
                            const float nm = fmaxf(m[n][e], x * sc), f = lfm_ex2(m[n][e] - nm);
                            m[n][e] = nm;
                            l[n][e] *= f;
#pragma unroll
                            for (int s = 0; s < kS; ++s)
#pragma unroll
                                for (int c = 0; c < 2; ++c)
#pragma unroll
                                    for (int k = 0; k < 2; ++k) {
                                        o[n][s][c][k][e] *= f;
                                        o[n][s][c][k][2 + e] *= f;
                                    }
                        }
                }
                uint32_t pf[NT][2];
#pragma unroll
                for (int n = 0; n < NT; ++n) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) z4[n][j] = lfm_ex2(__fmaf_rn(z4[n][j], sc, -m[n][j & 1]));
                    l[n][0] += z4[n][0] + z4[n][2];
                    l[n][1] += z4[n][1] + z4[n][3];
                    pf[n][0] = transpose8(lfm_pack2(z4[n][0], z4[n][1], __half()));
                    pf[n][1] = transpose8(lfm_pack2(z4[n][2], z4[n][3], __half()));
                }
                /* O^T: rows are values 64 s + 32 c + 4 g + i of the head */
                uint32_t dv[4][kS];
                lds_scales<kS>(vs + ve * (D / 16), dv[0]);
                lds_scales<kS>(vs + vo * (D / 16), dv[1]);
                lds_scales<kS>(vs + (ve + 8) * (D / 16), dv[2]);
                lds_scales<kS>(vs + (vo + 8) * (D / 16), dv[3]);
                if (tail) { /* what no token holds may be anything */
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        if (key0 + s16 + (k & 1 ? vo : ve) + (k & 2 ? 8 : 0) >= len) {
#pragma unroll
                            for (int s = 0; s < kS; ++s) dv[k][s] = 0;
                        }
                }
#pragma unroll
                for (int s = 0; s < kS; ++s) {
                    const uint32_t at = vc + 32 * s + 4 * g;
                    const uint32_t x0 = lds32(at + ve * (D / 2)), x1 = lds32(at + vo * (D / 2));
                    const uint32_t x2 = lds32(at + (ve + 8) * (D / 2)), x3 = lds32(at + (vo + 8) * (D / 2));
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        const uint32_t sel = c ? 0x7632 : 0x5410;
                        const uint32_t u = __byte_perm(x0, x1, sel), w = __byte_perm(x2, x3, sel);
                        const uint32_t du = __byte_perm(dv[0][s], dv[1][s], sel), dw = __byte_perm(dv[2][s], dv[3][s], sel);
#pragma unroll
                        for (int k = 0; k < 2; ++k) {
                            const uint32_t uu = k ? u >> 8 : u, ww = k ? w >> 8 : w;
                            const uint32_t a[4] = {lfm_hmul2(lfm_hsub2(lfm_nib0(uu), LFM_NIB0_OFF), du), lfm_hmul2(lfm_hsub2(lfm_nib1(uu), LFM_NIB1_OFF), du),
                                                   lfm_hmul2(lfm_hsub2(lfm_nib0(ww), LFM_NIB0_OFF), dw), lfm_hmul2(lfm_hsub2(lfm_nib1(ww), LFM_NIB1_OFF), dw)};
#pragma unroll
                            for (int n = 0; n < NT; ++n) mma16816(o[n][s][c][k], a, pf[n][0], pf[n][1]);
                        }
                    }
                }
            }
            __syncwarp();
            if (i + kStages < rg.n) rg.issue(i + kStages);
        }
        if (!ok) { /* a copy never came: wait (bounded) for those still under way before the ring is used again */
            for (uint32_t st = 0; st < kStages; ++st) lfm_mbar_wait(&s_bar[warp][st], (phases >> st) & 1, A.err);
            return;
        }

        /* ---- the warps' parts ---- */
        __syncthreads();
        float *so = reinterpret_cast<float *>(ring);
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                float x = l[n][e];
#pragma unroll
                for (int k = 4; k < 32; k <<= 1) x += __shfl_xor_sync(LFM_FULL_MASK, x, k);
                const uint32_t col = n * 8 + 2 * t + e;
                if (g == 0) { s_m[warp][col] = m[n][e]; s_l[warp][col] = x; }
#pragma unroll
                for (int s = 0; s < kS; ++s)
#pragma unroll
                    for (int c = 0; c < 2; ++c)
                        *reinterpret_cast<float4 *>(so + (size_t)(warp * kCols + col) * kPitch + 64 * s + 32 * c + 4 * g) =
                            make_float4(o[n][s][c][0][e], o[n][s][c][0][2 + e], o[n][s][c][1][e], o[n][s][c][1][2 + e]);
            }
        __syncthreads();
        float *part = n_act > 1 ? P.parts + (unit * P.n_splits + split) * kCols * (D + 2) : nullptr;
        auto write = [&](uint32_t col, uint32_t d, float (&v)[4], float sum) {
            const float inv = sum > 0.0f ? 1.0f / sum : 0.0f;
#pragma unroll
            for (int k = 0; k < 4; ++k) v[k] = sum == sum ? v[k] * inv : sum; /* a NaN row stays one */
            const uint32_t r = row0 + col;
            store4(A.out, A.type, (size_t)(q0 + r / G) * A.out_stride + ((size_t)kvh * G + r % G) * D + d, v);
        };
        for (uint32_t i = tid; i < (last + 1) * (D / 4); i += kThreads) {
            const uint32_t col = i / (D / 4), d = i % (D / 4) * 4;
            float mx = s_m[0][col], v[4] = {0.f, 0.f, 0.f, 0.f}, sum = 0.0f;
#pragma unroll
            for (int w = 1; w < kWarps; ++w) mx = fmaxf(mx, s_m[w][col]);
#pragma unroll
            for (int w = 0; w < kWarps; ++w) {
                const float f = lfm_ex2(s_m[w][col] - mx);
                const float4 x = *reinterpret_cast<const float4 *>(so + (size_t)(w * kCols + col) * kPitch + d);
                v[0] = __fmaf_rn(f, x.x, v[0]); v[1] = __fmaf_rn(f, x.y, v[1]);
                v[2] = __fmaf_rn(f, x.z, v[2]); v[3] = __fmaf_rn(f, x.w, v[3]);
                sum = __fmaf_rn(f, s_l[w][col], sum);
            }
            if (!part) {
                write(col, d, v, sum);
            } else {
                float *p = part + (size_t)col * (D + 2);
                *reinterpret_cast<float2 *>(p + 2 + d) = make_float2(v[0], v[1]);
                *reinterpret_cast<float2 *>(p + 4 + d) = make_float2(v[2], v[3]);
                if (d == 0) *reinterpret_cast<float2 *>(p) = make_float2(mx, sum);
            }
        }
        if (part) {
            /* the last split to arrive joins them all, in their order */
            __threadfence();
            __syncthreads();
            if (tid == 0) {
                s_last = atomicAdd(P.counts + unit, 1u) + 1 == n_act;
                if (s_last) P.counts[unit] = 0;
            }
            __syncthreads();
            if (s_last) {
                __threadfence();
                const float *all = P.parts + unit * P.n_splits * kCols * (D + 2);
                for (uint32_t i = tid; i < (last + 1) * (D / 4); i += kThreads) {
                    const uint32_t col = i / (D / 4), d = i % (D / 4) * 4;
                    float mx = LFM_NO_KEY, v[4] = {0.f, 0.f, 0.f, 0.f}, sum = 0.0f;
                    for (uint32_t k = 0; k < n_act; ++k) mx = fmaxf(mx, __ldcg(all + (size_t)(k * kCols + col) * (D + 2)));
                    for (uint32_t k = 0; k < n_act; ++k) {
                        const float2 *p = reinterpret_cast<const float2 *>(all + (size_t)(k * kCols + col) * (D + 2));
                        const float2 ml = __ldcg(p), x = __ldcg(p + 1 + d / 2), y = __ldcg(p + 2 + d / 2);
                        const float f = lfm_ex2(ml.x - mx);
                        v[0] = __fmaf_rn(f, x.x, v[0]); v[1] = __fmaf_rn(f, x.y, v[1]);
                        v[2] = __fmaf_rn(f, y.x, v[2]); v[3] = __fmaf_rn(f, y.y, v[3]);
                        sum = __fmaf_rn(f, ml.y, sum);
                    }
                    write(col, d, v, sum);
                }
            }
        }
        if (z < A.bt.n_seqs) return;
    }
}

template <int D, int NT>
cudaError_t launch_rows(const AttnArgs &a, const RowsPlan &p, dim3 grid, cudaStream_t s, bool pdl) {
    static size_t set[2][16];
    auto fn = a.softcap > 0.0f ? k_attn_rows<D, NT, true> : k_attn_rows<D, NT, false>;
    const cudaError_t e = lfm_smem_attr((const void *)fn, Cfg<D>::kRing, set[a.softcap > 0.0f]);
    return e != cudaSuccess ? e : lfm_launch_pdl(fn, grid, dim3(kThreads), Cfg<D>::kRing, s, pdl, a, p);
}

}  // namespace

/* Rows of a sequence up to which it is this file's: measured, see launch below. */
constexpr uint64_t kFewRows = 64;

static cudaError_t lfm_launch_attn_rows(const AttnArgs &a, uint32_t head_dim, uint64_t few, uint32_t max_kv_len, int sm_count, void *scratch,
                            bool *used, cudaStream_t s, bool pdl) {
    const uint32_t T = a.bt.n_tokens, B = a.bt.n_seqs, G = a.group, keys = head_dim == 64 ? 64 : 32;
    /* columns of a tile: what an average sequence fills, as far as registers go */
    const uint64_t per = ((uint64_t)T + B - 1) / B * G;
    const uint32_t nt = per <= 8 ? 1 : per <= 16 || head_dim == 128 ? 2 : 4, cols = 8 * nt;
    /* tiles beyond each sequence's first: at most T G / cols.  As many tokens as sequences are taken for a step
     * of single tokens, and one block in z walks what further tiles there are */
    const uint64_t bound = (uint64_t)T * G / cols;
    RowsPlan p{};
    p.most = few;
    p.extra = bound == 0 ? 0 : T == B ? 1 : (uint32_t)(bound < 4096 ? bound : 4096);
    p.tiles = B + bound;
    uint64_t span = a.window && a.window < max_kv_len ? (uint64_t)a.window + T + keys : max_kv_len;
    if (span > max_kv_len) span = max_kv_len;
    const uint64_t blocks = span ? (span + keys - 1) / keys : 1;
    /* splits: enough blocks to fill the GPU a few times over where there are few units, none of them under a
     * block of keys a warp */
    const uint64_t want = 4ull * 2 * sm_count, live = (uint64_t)B * a.kv.hkv, most = (blocks + kWarps - 1) / kWarps;
    uint64_t n = (want + live - 1) / live;
    if (n > most) n = most;
    p.units = p.tiles * a.kv.hkv;
    const size_t part = (size_t)cols * (head_dim + 2) * sizeof(float);
    if (p.units > LFM_ATTN_COUNTS) p.units = LFM_ATTN_COUNTS;
    if (n > LFM_ATTN_PARTS_BYTES / part / p.units) n = LFM_ATTN_PARTS_BYTES / part / p.units;
    if (n < 1) n = 1;
    p.chunk = (uint32_t)((blocks + n - 1) / n);
    p.n_splits = (uint32_t)((blocks + p.chunk - 1) / p.chunk);
    *used = p.n_splits > 1;
    p.counts = static_cast<uint32_t *>(scratch);
    p.parts = reinterpret_cast<float *>(static_cast<uint8_t *>(scratch) + LFM_ATTN_COUNTS * sizeof(uint32_t));
    const dim3 grid(B + p.extra, a.kv.hkv, p.n_splits);
    if (head_dim == 64)
        return nt == 1 ? launch_rows<64, 1>(a, p, grid, s, pdl) : nt == 2 ? launch_rows<64, 2>(a, p, grid, s, pdl)
                                                                          : launch_rows<64, 4>(a, p, grid, s, pdl);
    return nt == 1 ? launch_rows<128, 1>(a, p, grid, s, pdl) : launch_rows<128, 2>(a, p, grid, s, pdl);
}

cudaError_t lfm_launch_attn(const AttnArgs &a, uint32_t head_dim, uint32_t max_kv_len, int sm_count, void *scratch,
                            bool *used, cudaStream_t s, bool pdl) {
    const uint64_t T = a.bt.n_tokens, B = a.bt.n_seqs, rows = T * a.group;
    *used = false;
    /* one sequence, or at most as many tokens as make few rows: one kernel takes all.  As many tokens as sequences
     * are a step of single tokens, whatever the odd sequence holds.  Otherwise each takes its sequences */
    if (rows <= kFewRows || T == B) return lfm_launch_attn_rows(a, head_dim, ~0ull, max_kv_len, sm_count, scratch, used, s, pdl);
    if (B == 1) return lfm_launch_attn_tile(a, head_dim, 0, s, pdl);
    const cudaError_t e = lfm_launch_attn_tile(a, head_dim, kFewRows, s, pdl);
    return e != cudaSuccess ? e : lfm_launch_attn_rows(a, head_dim, kFewRows, max_kv_len, sm_count, scratch, used, s, pdl);
}
