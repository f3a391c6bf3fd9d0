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
 *   - P: e^(z - m) in fp16 as the B fragment, transposed by movmatrix.  m lies
 *     2^7 below a score and only moves when one passes it by 2^15, so p <= 2^15,
 *     and the sum is fp32.
 * A warp takes 4608-byte blocks of keys and values (64 keys of 64 values, 32 of
 * 128) through its own ring of bulk copies.  All (tile of columns, kv head)
 * units' blocks of keys lie in a row that is cut into equal parts, one for each
 * block that the GPU holds at once, whatever the lengths; its four warps take
 * the part's key blocks in turn and are joined in shared memory, the parts of a
 * unit through scratch: the last to finish joins them in their order (the same
 * bits on every run).  A block for each unit and a ring through its keys, which
 * leaves the longest sequence to one SM, took 92 us where equal parts take 73
 * (64 sequences of up to 8192 keys).
 *
 * Where the time goes: 32 / 8 heads of 64 values, 64 tokens on ragged sequences
 * of up to 8192 keys take 62 us for 186 MB, 3.0 TB/s (46% of a copy's rate).  No
 * pipe is full: issue 57%, tensor pipe 17%.  A step of 16 keys is some 220
 * instructions of a warp, unpacking above all, for 1152 bytes, in one chain of
 * dependent ones, and an SM holds 16 warps: of the 6.1 cycles between a warp's
 * instructions 1.4 pass in the fixed latency of the one before, 1.0 until its
 * turn, 0.7 for a busy arithmetic pipe, 0.7 for memory, 0.6 at the join's barriers
 * and fences.  128-value heads, two sequences of 131072 keys: 83 us, 302 MB, 3.6
 * TB/s (56%), the same picture.  One token on 1024 keys: 9.0 us, a chain of table,
 * copy, products and join.  72 tokens of 16 sequences (2 to 7 each) of up to 8192
 * keys: 46 us, two warps a scheduler with wide tiles half empty, issue 27%.
 */
#include <type_traits>

#include "attn_device.cuh"

namespace {

constexpr int kWarps = 4, kThreads = kWarps * 32, kStages = 3;

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
/* d = A B + c; c in registers of its own, so that a start value is not copied first. */
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1, const float (&c)[4]) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(c[0]), "f"(c[1]), "f"(c[2]), "f"(c[3]));
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
/* N words. */
template <int N>
__device__ __forceinline__ void lds(uint32_t a, uint32_t (&v)[N]) {
    if constexpr (N == 4) {
        asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]) : "r"(a));
    } else if constexpr (N == 2) {
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
    uint64_t most;    /* rows of the longest sequence that is this kernel's */
    float *parts;     /* [blocks][2][cols][D + 2]                           */
    uint32_t *counts; /* [blocks], zero between calls                       */
};

/* A sequence's share of the work: its tiles of kCols rows, on every kv head, over its blocks of keys. */
struct Seq {
    int64_t q0, n_q, len, blk0, blk1;
    uint64_t tiles, weight;
    bool sane;
};

/* Words of a stage that no copy fills.  Not inlined: in the kernel it changes the key loop's registers (64 sequences:
 * 62.0 -> 62.7 us; a test of each key pair beside the one for `held` 62.9). */
__device__ __noinline__ void zero_shared(uint32_t to, uint32_t bytes) {
    for (uint32_t i = 0; i < bytes; i += 4) asm volatile("st.shared.u32 [%0], %1;" ::"r"(to + i), "r"(0u) : "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); /* before a later copy into the stage */
}

/* A warp's copies of its blocks of keys first, first + kWarps, ... of a unit. */
template <int D>
struct Ring {
    static constexpr uint32_t kK = Cfg<D>::kKeys;
    const KvDev &kv;
    const BatchDev &bt;
    uint32_t *err;
    uint64_t *bars;
    uint32_t lane, to, bytes, per; /* this lane's part of a page: where it goes, its bytes, and bytes a token */
    const int32_t *row;            /* the sequence's page table */
    const uint8_t *from;           /* the part in page 0 */
    uint32_t n;                    /* blocks of this warp */
    int64_t first, end;            /* first block; keys that exist */
    uint32_t id, next;             /* pages of two blocks, 16 lanes each: a lane a part of a page */

    /* Lane l: part l % 4 (K codes, K scales, V codes, V scales) of piece l / 4 % 4 of a block; a stage is
     * [K codes][K scales][V codes][V scales] of its keys whatever the page's size. */
    __device__ __forceinline__ Ring(const AttnArgs &A, uint64_t *bars, uint32_t smem)
        : kv(A.kv), bt(A.bt), err(A.err), bars(bars), lane(threadIdx.x & 31) {
        const uint32_t part = lane & 3, j = (lane >> 2) & 3, P = kv.page_tokens;
        per = (part & 1) ? D / 16 : D / 2;
        bytes = min(P, kK) * per;
        to = smem + (part & 2 ? Cfg<D>::kBytes / 2 : 0) + ((part & 1) ? kK * (D / 2) : 0) + j * bytes;
    }
    __device__ __forceinline__ void unit(uint32_t b, uint32_t kvh, int64_t first_, uint32_t n_, int64_t lo, int64_t end_) {
        row = bt.page_table + (size_t)b * bt.table_stride;
        from = kv.pages + (size_t)kvh * kv.head_bytes + (lane & 2 ? kv.half : 0) + (lane & 1 ? kv.codes : 0);
        first = first_;
        n = n_;
        end = end_;
        /* only a unit's first block begins below lo.  A page of it that ends there may be gone: it is not copied, and its
         * slots' values get scales of zero (their scores are masked) */
        bool gone = false;
        next = lookup(0, [&](int64_t key) { return gone = key + min(kv.page_tokens, kK) <= lo; });
        if (gone && (lane & 3) == 3) zero_shared(to, bytes);
    }
    /* This lane's page in block i2 + lane / 16, but for keys that no row sees. */
    template <class Unseen>
    __device__ __forceinline__ uint32_t lookup(uint32_t i2, Unseen &&unseen) {
        const uint32_t i = i2 + lane / 16, at = ((lane >> 2) & 3) * kv.page_tokens;
        const int64_t key = (first + (int64_t)i * kWarps) * kK + at;
        if (i >= n || key >= end || (at && at >= kK) || unseen(key)) return ~0u; /* nothing to copy */
        const int64_t place = key >> kv.page_shift;
        uint32_t page = ~0u;
        if (place < (int64_t)bt.table_stride) page = (uint32_t)row[place];
        if (page >= kv.n_pages) atomicOr(err, LFM_DEVERR_PAGE);
        return page;
    }
    /* Block i into stage st. */
    __device__ __forceinline__ void issue(uint32_t i, uint32_t st) {
        if ((i & 1) == 0) {
            id = next;
            next = lookup(i + 2, [](int64_t) { return false; });
        }
        const bool on = (lane >> 4) == (i & 1) && id < kv.n_pages;
        const uint32_t all = __reduce_add_sync(LFM_FULL_MASK, on ? bytes : 0u);
        if (lane == 0) lfm_mbar_arrive_tx(bars + st, all);
        __syncwarp();
        if (on) {
            /* a page longer than a block: the block's keys in it */
            const uint32_t in = ((uint32_t)(first + (int64_t)i * kWarps) * kK) & (kv.page_tokens - 1);
            asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                             to + st * Cfg<D>::kBytes),
                         "l"(from + (size_t)id * kv.page_bytes + in * per), "r"(bytes), "r"(lfm_smem_u32(bars + st))
                         : "memory");
        }
    }
};

template <int D, int NT, bool kCap>
__global__ void __launch_bounds__(kThreads, D * NT < 128 ? 4 : D * NT == 128 ? 3 : 2) k_attn_rows(AttnArgs A, RowsPlan P) {
    using C = Cfg<D>;
    constexpr int kCols = 8 * NT, kS = C::kSpans, kPitch = D + 4;
    static_assert(kWarps * kCols * kPitch * 4 <= C::kRing, "the join fits the ring");
    extern __shared__ __align__(128) uint8_t ring[];
    __shared__ uint64_t s_bar[kWarps][kStages];
    __shared__ float s_m[kWarps][kCols], s_l[kWarps][kCols];
    __shared__ int64_t s_hi[kCols], s_lo[kCols];
    __shared__ uint64_t s_sum[kWarps], s_first;
    __shared__ int s_seq, s_last;
    __shared__ uint32_t s_units[kWarps];
    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const uint32_t G = A.group;
    if (lane < kStages) lfm_mbar_init(&s_bar[warp][lane], 1);
    lfm_fence_mbar_init();
    __syncwarp();
    uint32_t phases = 0; /* parity of each stage's next wait */
    lfm_pdl_wait();
    lfm_pdl_launch_dependents();
    const float sc = fmaxf((kCap ? A.softcap : fabsf(A.scale)) * 1.44269504f, 1e-30f); /* not 0: times -inf */

    /* ---- this block's share: all (tile, head) units' key blocks in a row, cut into equal parts ---- */
    auto sequence = [&](uint32_t b) {
        Seq q{};
        q.q0 = A.bt.q_start[b];
        q.n_q = (int64_t)A.bt.q_start[b + 1] - q.q0;
        q.len = A.bt.kv_len[b];
        q.sane = lfm_sane(A.bt, q.q0, q.n_q) && (q.n_q == 0 || lfm_sane_len(A.bt, q.len));
        const uint64_t rows = q.sane ? (uint64_t)q.n_q * G : 0;
        if (rows == 0 || rows > P.most) return q;
        int64_t lo, hi, unused;
        lfm_visible(A, q.n_q, q.len, 0, lo, unused);
        lfm_visible(A, q.n_q, q.len, (uint32_t)rows - 1, unused, hi);
        q.blk0 = lo / C::kKeys;
        q.blk1 = max(q.blk0 + 1, (hi + C::kKeys - 1) / C::kKeys); /* one where there is no key: rows of zeros */
        q.tiles = (rows + kCols - 1) / kCols;
        q.weight = q.tiles * A.kv.hkv * (uint64_t)(q.blk1 - q.blk0);
        return q;
    };
    auto warp_scan = [&](uint64_t v) {
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint64_t u = __shfl_up_sync(LFM_FULL_MASK, v, o);
            if (lane >= (uint32_t)o) v += u;
        }
        return v;
    };
    uint64_t w = 0; /* this thread's sequence of the last kThreads looked at */
    {
        uint64_t sum = 0;
        uint32_t units = 0;
        for (uint32_t b0 = 0; b0 < A.bt.n_seqs; b0 += kThreads) {
            w = 0;
            if (b0 + tid < A.bt.n_seqs) {
                const Seq q = sequence(b0 + tid);
                if (!q.sane && blockIdx.x == 0) atomicOr(A.err, LFM_DEVERR_PAGE);
                w = q.weight;
                units += (uint32_t)min(q.tiles * A.kv.hkv, (uint64_t)(1u << 20));
                units = min(units, 1u << 20);
            }
            sum += w;
        }
        sum = warp_scan(sum);
        if (lane == 31) s_sum[warp] = sum;
        units = __reduce_add_sync(LFM_FULL_MASK, min(units, 1u << 20)); /* beyond the blocks it makes no difference */
        if (lane == 0) s_units[warp] = units;
    }
    __syncthreads();
    uint64_t total = 0;
    uint32_t units = 0;
#pragma unroll
    for (int i = 0; i < kWarps; ++i) {
        total += s_sum[i];
        units += s_units[i];
    }
    /* blocks at work: a block of keys for each warp, or one for each unit where units are shorter */
    uint64_t n_cta = min((uint64_t)gridDim.x, max((total + kWarps - 1) / kWarps, (uint64_t)units));
    /* units that are all alike: cuts that fall between them, where that leaves few blocks idle.  A block that ends one
     * unit and begins another loads q and joins twice (256 rows on 2048 keys, 8 kv heads: 31 us, 21 so) */
    if (units && units <= n_cta && total % units == 0 && 4 * (n_cta / units * units) >= 3 * n_cta) n_cta = n_cta / units * units;
    if (blockIdx.x >= n_cta) return;
    uint64_t x = total * blockIdx.x / n_cta;
    const uint64_t x1 = total * (blockIdx.x + 1) / n_cta;
    /* the part that holds place u */
    auto owner = [&](uint64_t u) { return (uint32_t)(((u + 1) * n_cta + total - 1) / total - 1); };
    /* the whole block: the sequence that holds place u, and its first place */
    auto locate = [&](uint64_t u) {
        uint64_t before = 0;
        for (uint32_t b0 = 0; b0 < A.bt.n_seqs; b0 += kThreads) {
            if (A.bt.n_seqs > kThreads) w = b0 + tid < A.bt.n_seqs ? sequence(b0 + tid).weight : 0;
            uint64_t sum = warp_scan(w);
            __syncthreads();
            if (lane == 31) s_sum[warp] = sum;
            __syncthreads();
            sum += before;
            for (uint32_t i = 0; i < kWarps; ++i) {
                if (i < warp) sum += s_sum[i];
                before += s_sum[i];
            }
            if (u >= sum - w && u < sum) {
                s_seq = (int)(b0 + tid);
                s_first = sum - w;
            }
            if (u < before) break;
        }
        __syncthreads();
    };
    locate(x);
    uint32_t b = (uint32_t)s_seq;
    uint64_t first = s_first; /* place of the sequence's first unit */
    Seq seq = sequence(b);
    uint64_t n_blk = (uint64_t)(seq.blk1 - seq.blk0), u0 = (x - first) / n_blk; /* blocks of a unit, place of ours */
    uint32_t kvh = (uint32_t)(u0 % A.kv.hkv), ct = (uint32_t)(u0 / A.kv.hkv);
    u0 = first + u0 * n_blk;
    Ring<D> rg(A, s_bar[warp], lfm_smem_u32(ring) + warp * kStages * C::kBytes);

    while (x < x1) {
        if (x >= first + seq.weight) { /* the next sequence that has work */
            first += seq.weight;
            ++b;
            seq = sequence(b);
            if (seq.weight == 0) {
                locate(x);
                b = (uint32_t)s_seq;
                seq = sequence(b);
            }
            n_blk = (uint64_t)(seq.blk1 - seq.blk0);
            u0 = first;
            kvh = ct = 0;
        }
        const int64_t q0 = seq.q0, n_q = seq.n_q, len = seq.len;
        const uint64_t seg = min(x1, u0 + n_blk) - x; /* key blocks of this unit that are ours */
        /* the blocks that share the unit */
        const uint32_t own0 = x == u0 ? blockIdx.x : owner(u0);
        const uint32_t own1 = x + seg == u0 + n_blk ? blockIdx.x : owner(u0 + n_blk - 1);
        const uint32_t row0 = ct * kCols; /* rows of a sequence: (token, head of the group), below 2^31 */
        const int64_t rows = n_q * G - row0;
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
        const int64_t at0 = seq.blk0 + (int64_t)(x - u0), at1 = at0 + (int64_t)seg;
        const int64_t from = max(at0, lo0 / C::kKeys), to = min(at1, (hi1 + C::kKeys - 1) / C::kKeys);
        const int64_t mine = to - from - warp;
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncthreads(); /* s_lo, s_hi; the ring is free of an earlier unit's join, for the copies too */
        rg.unit(b, kvh, from + warp, mine > 0 ? (uint32_t)((mine + kWarps - 1) / kWarps) : 0u, lo0, len);
#pragma unroll
        for (uint32_t i = 0; i < kStages; ++i)
            if (i < rg.n) rg.issue(i, i);

        /* ---- Q as B fragments: column g, values 64 s + 32 c + 8 t .. of the head ---- */
        uint32_t qf[NT][kS][2][4];
        float corr[NT][kS][2][4]; /* start values of the scores: minus the codes' offsets times q */
        auto load = [&](const auto *q) { /* the type is told apart once, so the loads are under way together */
            float v[NT][kS][2][8];
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                const uint32_t r = row0 + n * 8 + g;
                const bool on = n * 8 + g <= last;
                const size_t at = on ? (size_t)(q0 + r / G) * A.q_stride + ((size_t)kvh * G + r % G) * D : 0;
#pragma unroll
                for (int s = 0; s < kS; ++s)
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
#pragma unroll
                        for (int i = 0; i < 8; ++i) v[n][s][c][i] = 0.0f;
                        if (on) lfm_load<8>(q + at + 64 * s + 32 * c + 8 * t, v[n][s][c]);
                    }
            }
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int s = 0; s < kS; ++s)
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        lfm_fit_q(A.scale < 0.0f, v[n][s][c]);
                        float h[8], sum = 0.0f;
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            h[i] = __half2float(__float2half_rn(v[n][s][c][i]));
                            sum = __fmaf_rn(h[i], (i & 1) ? 72.0f : 1032.0f, sum);
                        }
#pragma unroll
                        for (int i = 0; i < 4; ++i) qf[n][s][c][i] = lfm_pack2(h[i], h[4 + i], __half());
                        sum += __shfl_xor_sync(LFM_FULL_MASK, sum, 1);
                        sum += __shfl_xor_sync(LFM_FULL_MASK, sum, 2);
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            corr[n][s][c][i] = -__shfl_sync(LFM_FULL_MASK, sum, 8 * t + 4 * (i & 1));
                            asm volatile("" : "+f"(corr[n][s][c][i])); /* four registers, not two */
                        }
                    }
        };
        if (A.type == 0) load(static_cast<const float *>(A.q));
        else if (A.type == 1) load(static_cast<const __half *>(A.q));
        else load(static_cast<const __nv_bfloat16 *>(A.q));

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
        const uint32_t rk = g ^ (g >> 2);                     /* key of A row g (rows 8.. : + 8)            */
        const uint32_t ve = 2 * t ^ (t >> 1), vo = ve ^ 1;    /* keys of A columns 2 t and 2 t + 1 for V    */
        const uint32_t sel0 = t < 2 ? 0x5410 : 0x1054, sel1 = t < 2 ? 0x7632 : 0x3276; /* scales of ve, vo  */
        constexpr uint32_t kKs = C::kKeys * (D / 2), kV = C::kBytes / 2;
        const uint32_t atk = rk * (D / 2) + 8 * t, atks = kKs + rk * (D / 16);
        const uint32_t atve = kV + ve * (D / 2) + 4 * g, atvo = kV + vo * (D / 2) + 4 * g;
        const uint32_t atvs = kV + kKs + (ve & ~1u) * (D / 16);
        const float capz = kCap ? lfm_cap_scale(A.scale, A.softcap) : 0.0f;
        constexpr int kPair = NT == 1 ? 2 : 1; /* steps of 16 keys whose scores are looked at together */
        const LfmNib nib;
        bool ok = true;
        /* a block of keys: every row sees all of it (inside), or masks, and `held` slots that hold a token */
        auto block = [&](auto inside, uint32_t buf, int64_t key0) {
            const int held = (int)min((int64_t)C::kKeys, len - key0);
            constexpr bool kWhole = decltype(inside)::value;
#pragma unroll(kWhole ? C::kKeys / 16 / kPair : 1)
            for (int s16 = 0; s16 < C::kKeys; s16 += 16 * kPair) {
                /* S^T: rows rk and rk + 8, columns 2 t and 2 t + 1 */
                float z4[kPair][NT][4];
#pragma unroll
                for (int q = 0; q < kPair; ++q) {
                    const uint32_t kc = buf + atk + (s16 + 16 * q) * (D / 2), ks = buf + atks + (s16 + 16 * q) * (D / 16);
                    uint32_t d0[kS], d1[kS];
                    lds(ks, d0);
                    lds(ks + 8 * (D / 16), d1);
#pragma unroll
                    for (int s = 0; s < kS; ++s) {
                        const uint2 x0 = lds64(kc + 32 * s), x1 = lds64(kc + 8 * (D / 2) + 32 * s);
                        const float2 e0 = half2_of(d0[s]), e1 = half2_of(d1[s]);
#pragma unroll
                        for (int c = 0; c < 2; ++c) {
                            const uint32_t u = __byte_perm(x0.x, x0.y, c ? 0x7632 : 0x5410);
                            const uint32_t w = __byte_perm(x1.x, x1.y, c ? 0x7632 : 0x5410);
                            const uint32_t a0[4] = {nib.lo(u), nib.lo(w), nib.hi(u), nib.hi(w)};
                            const uint32_t a1[4] = {nib.lo(u >> 8), nib.lo(w >> 8), nib.hi(u >> 8), nib.hi(w >> 8)};
                            const float f0 = c ? e0.y : e0.x, f1 = c ? e1.y : e1.x;
#pragma unroll
                            for (int n = 0; n < NT; ++n) {
                                float acc[4];
                                float(&z)[4] = z4[q][n];
                                mma16816(acc, a0, qf[n][s][c][0], qf[n][s][c][1], corr[n][s][c]);
                                mma16816(acc, a1, qf[n][s][c][2], qf[n][s][c][3]);
                                if (s == 0 && c == 0) {
                                    z[0] = acc[0] * f0; z[1] = acc[1] * f0;
                                    z[2] = acc[2] * f1; z[3] = acc[3] * f1;
                                } else {
                                    z[0] = __fmaf_rn(acc[0], f0, z[0]); z[1] = __fmaf_rn(acc[1], f0, z[1]);
                                    z[2] = __fmaf_rn(acc[2], f1, z[2]); z[3] = __fmaf_rn(acc[3], f1, z[3]);
                                }
                            }
                        }
                    }
                }
                if (kCap) {
                    auto cap = [&](auto &&tanh_of) {
#pragma unroll
                        for (int q = 0; q < kPair; ++q)
#pragma unroll
                            for (int n = 0; n < NT; ++n)
#pragma unroll
                                for (int j = 0; j < 4; ++j) z4[q][n][j] = tanh_of(z4[q][n][j] * capz);
                    };
                    if (A.softcap <= LFM_PLAIN_CAP) cap([](float x) { return lfm_tanh(x); });
                    else cap([](float x) { return lfm_tanh_any(x); });
                }
                if (!kWhole) {
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            const int64_t lo = s_lo[n * 8 + 2 * t + e] - key0, hi = s_hi[n * 8 + 2 * t + e] - key0;
#pragma unroll
                            for (int k = 0; k < 2 * kPair; ++k) {
                                const int64_t key = s16 + 8 * k + (int)rk;
                                if (key < lo || key >= hi) z4[k >> 1][n][2 * (k & 1) + e] = -INFINITY;
                            }
                        }
                }
                float top[NT][2];
                bool grow = false;
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        float x = fmaxf(z4[0][n][e], z4[0][n][2 + e]);
                        if (kPair == 2) x = fmaxf(x, fmaxf(z4[kPair - 1][n][e], z4[kPair - 1][n][2 + e]));
                        top[n][e] = x;
                        grow |= __fmaf_rn(x, sc, -m[n][e]) > LFM_REF_MOVE;
                    }
                if (__any_sync(LFM_FULL_MASK, grow)) {
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            float x = top[n][e];
#pragma unroll
                            for (int k = 4; k < 32; k <<= 1) x = fmaxf(x, __shfl_xor_sync(LFM_FULL_MASK, x, k));
                            const float nm = fmaxf(m[n][e], __fmaf_rn(x, sc, -LFM_REF_LOW)), f = lfm_ex2(m[n][e] - nm);
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
#pragma unroll
                for (int q = 0; q < kPair; ++q) {
                    uint32_t pf[NT][2];
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        float(&z)[4] = z4[q][n];
#pragma unroll
                        for (int j = 0; j < 4; ++j) z[j] = lfm_ex2(__fmaf_rn(z[j], sc, -m[n][j & 1]));
                        l[n][0] += z[0] + z[2];
                        l[n][1] += z[1] + z[3];
                        pf[n][0] = transpose8(lfm_pack2(z[0], z[1], __half()));
                        pf[n][1] = transpose8(lfm_pack2(z[2], z[3], __half()));
                    }
                    /* O^T: rows are values 64 s + 32 c + 4 g + i of the head */
                    const int k16 = s16 + 16 * q;
                    uint32_t dv[2][2 * kS]; /* scales of a pair of keys, and of the pair eight further */
                    lds(buf + atvs + k16 * (D / 16), dv[0]);
                    lds(buf + atvs + (k16 + 8) * (D / 16), dv[1]);
                    if (!kWhole) { /* what no token holds may be anything */
#pragma unroll
                        for (int k = 0; k < 4; ++k)
                            if (k16 + (int)(ve & ~1u) + (k & 1) + (k & 2 ? 8 : 0) >= held) {
#pragma unroll
                                for (int s = 0; s < kS; ++s) dv[k >> 1][(k & 1) * kS + s] = 0;
                            }
                    }
#pragma unroll
                    for (int s = 0; s < kS; ++s) {
                        const uint32_t e = buf + atve + k16 * (D / 2) + 32 * s, o1 = buf + atvo + k16 * (D / 2) + 32 * s;
                        const uint32_t x0 = lds32(e), x1 = lds32(o1), x2 = lds32(e + 8 * (D / 2)), x3 = lds32(o1 + 8 * (D / 2));
#pragma unroll
                        for (int c = 0; c < 2; ++c) {
                            const uint32_t u = __byte_perm(x0, x1, c ? 0x7632 : 0x5410), w = __byte_perm(x2, x3, c ? 0x7632 : 0x5410);
                            const uint32_t du = __byte_perm(dv[0][s], dv[0][kS + s], c ? sel1 : sel0);
                            const uint32_t dw = __byte_perm(dv[1][s], dv[1][kS + s], c ? sel1 : sel0);
#pragma unroll
                            for (int k = 0; k < 2; ++k) {
                                const uint32_t uu = k ? u >> 8 : u, ww = k ? w >> 8 : w;
                                const uint32_t a[4] = {lfm_hmul2(lfm_hsub2(nib.lo(uu), LFM_NIB0_OFF), du),
                                                       lfm_hmul2(lfm_hsub2(nib.hi(uu), LFM_NIB1_OFF), du),
                                                       lfm_hmul2(lfm_hsub2(nib.lo(ww), LFM_NIB0_OFF), dw),
                                                       lfm_hmul2(lfm_hsub2(nib.hi(ww), LFM_NIB1_OFF), dw)};
#pragma unroll
                                for (int n = 0; n < NT; ++n) mma16816(o[n][s][c][k], a, pf[n][0], pf[n][1]);
                            }
                        }
                    }
                }
            }
        };
        for (uint32_t i = 0, st = 0; i < rg.n; ++i, st = st + 1 == kStages ? 0 : st + 1) {
            ok = __all_sync(LFM_FULL_MASK, lfm_mbar_wait(&s_bar[warp][st], (phases >> st) & 1, A.err));
            phases ^= 1u << st;
            if (!ok) break;
            const uint32_t buf = lfm_smem_u32(ring) + (warp * kStages + st) * C::kBytes;
            const int64_t key0 = (rg.first + (int64_t)i * kWarps) * C::kKeys;
            const bool whole = key0 >= lo1 && key0 + C::kKeys <= hi0; /* every row sees every key */
            if (whole) block(std::true_type(), buf, key0);
            else block(std::false_type(), buf, key0);
            __syncwarp();
            if (i + kStages < rg.n) rg.issue(i + kStages, st);
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
        const uint32_t n_parts = own1 - own0 + 1;
        auto part_of = [&](uint32_t c) { return P.parts + ((size_t)c * 2 + (c == own0)) * kCols * (D + 2); };
        float *part = n_parts > 1 ? part_of(blockIdx.x) : nullptr;
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
            /* the last part to arrive joins them all, in their order */
            __threadfence();
            __syncthreads();
            if (tid == 0) {
                s_last = atomicAdd(P.counts + own0, 1u) + 1 == n_parts;
                if (s_last) P.counts[own0] = 0;
            }
            __syncthreads();
            if (s_last) {
                __threadfence();
                for (uint32_t i = tid; i < (last + 1) * (D / 4); i += kThreads) {
                    const uint32_t col = i / (D / 4), d = i % (D / 4) * 4;
                    float mx = LFM_NO_KEY, v[4] = {0.f, 0.f, 0.f, 0.f}, sum = 0.0f;
                    for (uint32_t c0 = own0; c0 <= own1; c0 += 8) { /* eight parts' loads under way together */
                        float2 ml[8], a[8], b[8];
#pragma unroll
                        for (uint32_t k = 0; k < 8; ++k) {
                            ml[k] = make_float2(LFM_NO_KEY, 0.0f);
                            a[k] = b[k] = make_float2(0.0f, 0.0f);
                            if (c0 + k <= own1) {
                                const float2 *p = reinterpret_cast<const float2 *>(part_of(c0 + k) + (size_t)col * (D + 2));
                                ml[k] = __ldcg(p);
                                a[k] = __ldcg(p + 1 + d / 2);
                                b[k] = __ldcg(p + 2 + d / 2);
                            }
                        }
                        float top = mx;
#pragma unroll
                        for (int k = 0; k < 8; ++k) top = fmaxf(top, ml[k].x);
                        const float old = lfm_ex2(mx - top);
                        mx = top;
                        sum *= old;
#pragma unroll
                        for (int k = 0; k < 4; ++k) v[k] *= old;
#pragma unroll
                        for (int k = 0; k < 8; ++k) {
                            const float f = lfm_ex2(ml[k].x - mx);
                            v[0] = __fmaf_rn(f, a[k].x, v[0]); v[1] = __fmaf_rn(f, a[k].y, v[1]);
                            v[2] = __fmaf_rn(f, b[k].x, v[2]); v[3] = __fmaf_rn(f, b[k].y, v[3]);
                            sum = __fmaf_rn(f, ml[k].y, sum);
                        }
                    }
                    write(col, d, v, sum);
                }
            }
        }
        x += seg;
        u0 += n_blk;
        if (++kvh == A.kv.hkv) {
            kvh = 0;
            ++ct;
        }
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

static cudaError_t lfm_launch_attn_rows(const AttnArgs &a, uint32_t head_dim, uint64_t few, uint32_t max_kv_len,
                                        int sm_count, void *scratch, cudaStream_t s, bool pdl) {
    const uint64_t T = a.bt.n_tokens, B = a.bt.n_seqs, G = a.group, keys = head_dim == 64 ? 64 : 32;
    /* columns of a tile: what an average sequence fills, as far as registers go, but narrow ones where the work is little:
     * more warps run at once, and each block has less to load, join and write.  By the keys that a warp would walk with
     * tiles of 8, 16 or 12 warps an SM: up to 256, tiles of 8; up to 1024, of 16 if tiles of 32 are so few that their
     * keys are split (otherwise each costs its loads and its join).  64-value heads, 8 kv heads, tiles of 8 / 16 / 32
     * columns, rows of a sequence:
     *   1 sequence of 2048 keys     32 rows 11.0, 12.6, 16.9 us
     *   1 sequence of 16384 keys    16 rows 17.8, 23.6, 23.8;  32: 20.8, 22.0, 30.9;  64: 28.8, 25.3, 31.4
     *   16 sequences of 1000 keys   32 rows 16.9, 23.4, 20.6;  64: 34.8, 33.6, 21.6
     *   16 sequences of 8192 keys   4 rows 29, 37, 55;  12: 49, 39, 59;  24: 67, 65, 60;  64: 155, 116, 101
     * 128-value heads, 8 / 16:
     *   1 sequence of 16384 keys    16 rows 23.5, 31.1;  32: 30.2, 31.8;  64: 49.8, 40.6
     *   16 sequences of 1000 keys   8 rows 15.4, 18.1;  16: 24.6, 19.8 (the wrong side)
     *   16 sequences of 8192 keys   4 rows 50, 66;  12: 84, 68;  64: 292, 216 */
    const uint64_t per = (T + B - 1) / B * G, span = ((uint64_t)max_kv_len + keys - 1) / keys;
    const uint64_t walk = B * ((per + 7) / 8) * a.kv.hkv * span * keys / ((uint64_t)sm_count * (head_dim == 64 ? 16 : 12));
    const bool split = B * ((per + 31) / 32) * a.kv.hkv < (uint64_t)sm_count / 2;
    const uint32_t nt = per <= 8 || walk <= 256 ? 1 : per <= 16 || head_dim == 128 || (walk <= 1024 && split) ? 2 : 4;
    /* blocks: as many as run at once by their registers (some instances spill 20 to 136 bytes at that; more blocks, with
     * fewer registers and more spills, ran slower), fewer where there are not enough blocks of keys by the hint */
    uint64_t grid = (uint64_t)sm_count * (head_dim * nt < 128 ? 4 : head_dim * nt == 128 ? 3 : 2);
    const uint64_t units = (B + T * G / (8 * nt)) * a.kv.hkv, work = units * (span + 1);
    const uint64_t most = work / kWarps > units ? work / kWarps : units;
    if (grid > most) grid = most;
    if (grid > LFM_ATTN_BLOCKS) grid = LFM_ATTN_BLOCKS;
    RowsPlan p{few, reinterpret_cast<float *>(static_cast<uint8_t *>(scratch) + LFM_ATTN_COUNTS * sizeof(uint32_t)),
               static_cast<uint32_t *>(scratch)};
    const dim3 g((uint32_t)grid);
    if (head_dim == 64)
        return nt == 1 ? launch_rows<64, 1>(a, p, g, s, pdl) : nt == 2 ? launch_rows<64, 2>(a, p, g, s, pdl)
                                                                       : launch_rows<64, 4>(a, p, g, s, pdl);
    return nt == 1 ? launch_rows<128, 1>(a, p, g, s, pdl) : launch_rows<128, 2>(a, p, g, s, pdl);
}

/* Which kernel takes a sequence.  Per SM, 32 rows against 64 keys take this file's kernel 0.44 us (64-value heads;
 * 128: 0.98), and 256 rows, however few of them there are, the tile kernel 0.99 us (1.18): about 2 to 5 and 6 to 7.
 * This one spreads any work over all SMs, the tile kernel whole rounds of tiles or of their parts; a call for both pays
 * for two launches.  So both sides are estimated, in blocks of keys, and the shorter taken.  Measured, 32 / 8 heads, rows of a sequence
 * (token, head of the group), this kernel and the other:
 *   32 sequences of 4096 keys, 64-value heads   64 rows: 110 us, 115;  128: 201, 174;  256: 376, 140
 *                              128-value heads  32 rows: 122, 136;  64: 225, 216;  128: 428, 213
 *   8 sequences of 4096 keys, 64-value heads    64 rows: 37, 43;  128: 55, 78;  256: 107, 72
 *   1 sequence of 16384 keys, 64-value heads    128 rows: 39, 48;  256: 59, 45;  512: 104, 50
 *   1 sequence of 2048 keys, 64-value heads     256 rows: 19, 23;  512: 26, 25;  1024: 33, 26
 * In a batch for both, sequences of up to 64 rows (128-value heads: 32) are this kernel's. */
cudaError_t lfm_launch_attn(const AttnArgs &a, uint32_t head_dim, uint32_t max_kv_len, int sm_count, void *scratch,
                            cudaStream_t s, bool pdl) {
    /* what a row, or the rows of a tile, can see */
    if (a.window && max_kv_len > (uint64_t)a.window + 256) max_kv_len = a.window + 256;
    const uint64_t T = a.bt.n_tokens, B = a.bt.n_seqs, rows = T * a.group, few = B == 1 ? 0 : head_dim == 64 ? 64 : 32;
    const TilePlan p = lfm_attn_tile_plan(a, head_dim, few, max_kv_len, sm_count);
    const uint64_t here = (rows + 16 * B) / 32 * a.kv.hkv * (p.blocks + 12);   /* 12: a unit's cost beside its blocks, by the pairs above */
    const uint64_t there = (p.cost + (B == 1 ? 3 : 10)) * (uint64_t)sm_count;  /* 10: the second launch */
    /* sequences of few rows by their average, and of no odd one that could be long: a step of single tokens (64
     * sequences of 8192 keys: 86 us, 92 with an idle launch of the other kernel), a batch to verify (16 sequences of
     * 8 tokens and 8192 keys: 63, 70) */
    const bool short_ones = T <= B || (rows <= few * B && (T - B + 1) * a.group <= 1024);
    if (short_ones || (head_dim == 64 ? here * 2 < there * 5 : here * 6 < there * 7))
        return lfm_launch_attn_rows(a, head_dim, ~0ull, max_kv_len, sm_count, scratch, s, pdl);
    const cudaError_t e = lfm_launch_attn_tile(a, head_dim, p, sm_count, scratch, s, pdl);
    return e != cudaSuccess || B == 1 ? e : lfm_launch_attn_rows(a, head_dim, few, max_kv_len, sm_count, scratch, s, pdl);
}
