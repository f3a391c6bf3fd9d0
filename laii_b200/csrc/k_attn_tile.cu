/*
 * Grouped-query attention over the paged 4-bit cache for many query rows a
 * sequence (prompts, chunks), on the 5th-generation tensor cores.
 *
 * A block takes 256 rows (token, head of the group) of one kv head as two
 * tiles of M = 128 and walks their keys 64 at a time, once:
 *   loader    bulk copies of a key block's codes and scales, K and V apart
 *   4 warps   codes -> fp16 values, two threads a key, into the operand layout of
 *             the MMA (no swizzle: 8 x 16-byte core matrices).  The layout's
 *             order of a head's values is that of the codes' words -- values
 *             4 w + i and 32 + 4 w + i side by side, so a word gives its eight
 *             with one shift and four pairs of one logic instruction, and the
 *             two scales of a span are the pair that multiplies them.  q is
 *             laid out in the same order and the output read back from it
 *   MMA       one thread: S = Q_h K^T (fp32, TMEM), O_h += P V with P, fp16,
 *             read from the TMEM columns of its S.  S has as many buffers as
 *             TMEM leaves beside O (6 of 64 columns for 64-value heads, 4 for
 *             128), taken in turn by (key block, tile), so the scores of a
 *             tile's next block are there when its softmax ends
 *   2 x 4 warps  softmax, a thread a row: no exchange between threads.  The
 *             running reference m lies 2^7 below a score and only moves when one
 *             passes it by 2^15 (p <= 2^15 in fp16); then the thread scales its
 *             row of O in TMEM
 * The blocks are persistent, one an SM, and take the tiles from a counter, the
 * longest first: loader and dequantisation run ahead into the next tile while
 * the softmax warps finish one.  Few tiles of long walks have their keys split
 * into parts, tickets of their own, which leave O unscaled, m and the sum in
 * scratch; for each 32 rows the last warp to arrive joins them in their order,
 * the same bits on every run.
 * O in TMEM is scaled by 1 / sum at the end.  Rows that end early in a block
 * and slots that hold no token are masked in S; values of such slots are zero.
 *
 * Keys and values enter as fp16 products d * (code - 8), rounded once (2^-12
 * relative, under the output's rounding and q's own); scores, m, the sum and O
 * are fp32, p is fp16 <= 2^15.
 *
 * 32 / 8 heads.  4096 tokens from the beginning, 64-value heads: 128 us, 537
 * TFLOP/s; 42 us of tensor work, 60 of exponentials (one a score, 16 a clock and
 * SM).  2048 tokens behind 14336, 128-value heads: 525 us call after call, 560 to
 * 575 with other work between, some 900 TFLOP/s; 314 of tensor work.  12 ragged
 * chunks, 3891 tokens in all, window 1024, capped: 128 us, 53 of them the three
 * operations of the exponential unit for each score.  No pipe is full: for the
 * prompt tensor 25%, exponential unit 51%, issue 46% (chunk: 51, 51, 50; capped:
 * 11, 68, 38).  Of the 8.3 cycles between a warp's instructions 2.1 wait for tensor
 * memory and barriers, 2.1 for the instruction before (capped: 3.4 and 2.2 of 10):
 * the hand-over from role to role for each block, with two softmax warps a
 * scheduler.  Without the softmax's arithmetic the same barriers take 91 and 344 us.
 * The few-row kernel's fragments in registers took 696 and 3469 us, a block's
 * barriers for 128 keys at a time 141 and 646 when 64 took 138 and 595.  512 rows on 16384 keys: 50 us, in one part 245.
 */
#include <type_traits>

#include "attn_device.cuh"

namespace {

constexpr int kM = 128, kRows = 2 * kM, kKeys = 64, kThreads = 512;
constexpr uint32_t kChunkQ = kM * 16, kChunk = kKeys * 16; /* bytes between the 8-value chunks of a row */

/* Key blocks that a part of a split tile has at least; what a tile costs beside its blocks, in blocks.  64-value heads,
 * one tile an SM of 8, 32, 128 key blocks: 17.5, 43.0, 136 us, each further one 12.9, 38.4, 132: 0.99 us a block and 5 us;
 * 128-value heads 24.3, 52.7, 164 and 20.0, 48.3, 161: 1.18 us and 10.5, nine blocks. */
constexpr uint32_t kPartBlocks = 8, kJobBlocks = 6;

template <int D>
struct Cfg {
    static constexpr int kQ = kM * D * 2, kOp = kKeys * D * 2; /* a tile of q; of keys or values */
    static constexpr int kRaw = kKeys * (D / 2 + D / 16);      /* its codes and scales           */
    static constexpr int kOps = D == 64 ? 12 : 8, kRaws = D == 64 ? 12 : 6;
    static constexpr uint32_t kBufs = D == 64 ? 6 : 4, kColO = kBufs * kKeys; /* of S, before O in TMEM */
    static constexpr int kOffOp = 2 * kQ, kOffRaw = kOffOp + kOps * kOp, kSmem = kOffRaw + kRaws * kRaw;
    static_assert(kSmem <= 226 * 1024, "shared memory");
};

constexpr uint32_t kTmemCols = 512, kColS = kKeys;
/* kind::f16, A and B fp16, D fp32 (bit 4), M / 16 at bit 24, N / 8 at 17; B transposed (N contiguous) at 16 */
constexpr uint32_t kIdescQK = (1u << 4) | ((uint32_t)(kM >> 4) << 24) | ((uint32_t)(kKeys >> 3) << 17);
template <int D>
constexpr uint32_t kIdescPV = (1u << 4) | ((uint32_t)(kM >> 4) << 24) | ((uint32_t)(D >> 3) << 17) | (1u << 16);

/* 256 rows of a kv head: rows row0 .. of sequence b, key blocks blk0 .. + n, of them the keys from lo on; part `part` of
 * `parts` of tile `tile`. */
struct Job {
    int64_t q0, n_q, len, blk0, lo;
    uint32_t row0, rows, kvh, n, tile, part, parts;
    int b; /* -1: no more */
};
struct Bars {
    uint64_t raw_full[12], raw_empty[12], op_full[12], op_empty[12], s_full[6], p_full[6], o_full[2][2];
    uint64_t q_full[2], job_full[2], job_empty[2];
    uint32_t tmem;
    int abort, tile[2];
    Job job[2]; /* the one at work and the next */
};

/* No swizzle, version 1: start, leading and stride byte offsets. */
__device__ __forceinline__ uint64_t sdesc(uint32_t saddr, uint32_t lbo, uint32_t sbo) {
    return (uint64_t)((saddr >> 4) & 0x3FFFu) | ((uint64_t)(lbo >> 4) << 16) | ((uint64_t)(sbo >> 4) << 32) | (1ull << 46);
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d), "l"(a), "l"(b), "r"(idesc),
        "r"((uint32_t)acc)
        : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}\n" ::"r"(d), "r"(a), "l"(b), "r"(idesc),
        "r"((uint32_t)acc)
        : "memory");
}
__device__ __forceinline__ void commit(uint64_t *bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(lfm_smem_u32(bar))
                 : "memory");
}
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

#define R8(v, i) "r"(v[i]), "r"(v[i + 1]), "r"(v[i + 2]), "r"(v[i + 3]), "r"(v[i + 4]), "r"(v[i + 5]), "r"(v[i + 6]), "r"(v[i + 7])
#define W8(v, i) "=r"(v[i]), "=r"(v[i + 1]), "=r"(v[i + 2]), "=r"(v[i + 3]), "=r"(v[i + 4]), "=r"(v[i + 5]), "=r"(v[i + 6]), "=r"(v[i + 7])
#define X8(v, i) "+r"(v[i]), "+r"(v[i + 1]), "+r"(v[i + 2]), "+r"(v[i + 3]), "+r"(v[i + 4]), "+r"(v[i + 5]), "+r"(v[i + 6]), "+r"(v[i + 7])
/* 32 consecutive 32-bit columns of this thread's TMEM lane. */
__device__ __forceinline__ void ld32(uint32_t t, uint32_t *v) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,"
        "%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : W8(v, 0), W8(v, 8), W8(v, 16), W8(v, 24)
        : "r"(t));
}
__device__ __forceinline__ void st32(uint32_t t, const uint32_t *v) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,"
        "%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(t),
        R8(v, 0), R8(v, 8), R8(v, 16), R8(v, 24)
        : "memory");
}
__device__ __forceinline__ void max3(float &m, uint32_t a, uint32_t b) {
    asm("max.f32 %0, %0, %1, %2;" : "+f"(m) : "f"(__uint_as_float(a)), "f"(__uint_as_float(b)));
}
/* Keeps the uses of loaded registers behind the wait. */
__device__ __forceinline__ void tie32(uint32_t *v) { asm volatile("" : X8(v, 0), X8(v, 8), X8(v, 16), X8(v, 24)::"memory"); }

__device__ __forceinline__ uint64_t pk2(uint32_t x, uint32_t y) { return (uint64_t)x | ((uint64_t)y << 32); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.ftz.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("mul.rn.ftz.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.ftz.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}

/* One thread of the warp, all of which run this. */
__device__ __forceinline__ bool elect() {
    uint32_t p;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xFFFFFFFF;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
    return p != 0;
}

/* Bounded wait that also gives up once another role has. */
__device__ __forceinline__ bool wait(uint64_t *bar, uint32_t parity, volatile int *abort, uint32_t *err) {
    if (lfm_mbar_try_wait(bar, parity)) return true;
    const uint64_t t0 = lfm_globaltimer();
    while (!lfm_mbar_try_wait_sleep(bar, parity, LFM_WAIT_SLEEP_NS)) {
        if (*abort) return false;
        if (lfm_globaltimer() - t0 > LFM_WAIT_LIMIT_NS) {
            atomicOr(err, LFM_DEVERR_TIMEOUT);
            *abort = 1;
            return false;
        }
    }
    return true;
}

/* A test that does not wait.  Its answer comes through the queue that the softmax warps' exponentials fill, some
 * hundred cycles later: asked for ahead of other work, it costs nothing. */
__device__ __forceinline__ bool test(uint64_t *bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(lfm_smem_u32(bar)), "r"(parity)
        : "memory");
    return ok != 0;
}

/* kSplit: tiles in parts (an instance of its own: with the join's code in it the other one is 2% slower: prompt 132 us,
 * 130). */
template <int D, bool kCap, bool kSplit>
__global__ void __launch_bounds__(kThreads, 1) k_attn_tile(AttnArgs A, TilePlan plan) {
    using C = Cfg<D>;
    uint32_t *const ticket = plan.counts + LFM_ATTN_COUNTS - 2;
    extern __shared__ __align__(1024) uint8_t sm[];
    __shared__ Bars bars;
    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, G = A.group;
    volatile int *abort = &bars.abort;
    if (tid == 0) {
        for (int i = 0; i < C::kRaws; ++i) {
            lfm_mbar_init(&bars.raw_full[i], 1);
            lfm_mbar_init(&bars.raw_empty[i], 4);
        }
        for (int i = 0; i < C::kOps; ++i) {
            lfm_mbar_init(&bars.op_full[i], 4);
            lfm_mbar_init(&bars.op_empty[i], 2);
        }
        for (uint32_t i = 0; i < C::kBufs; ++i) {
            lfm_mbar_init(&bars.s_full[i], 1);
            lfm_mbar_init(&bars.p_full[i], 4);
        }
        for (int i = 0; i < 4; ++i) lfm_mbar_init(&bars.o_full[i >> 1][i & 1], 1);
        for (int i = 0; i < 2; ++i) {
            lfm_mbar_init(&bars.q_full[i], 4);
            lfm_mbar_init(&bars.job_full[i], 1);
            lfm_mbar_init(&bars.job_empty[i], 14); /* softmax, dequantisation and MMA warps */
        }
        bars.abort = 0;
        lfm_fence_mbar_init();
    }
    if (warp == 12) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(lfm_smem_u32(&bars.tmem)),
                     "r"(kTmemCols)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
        fence_before();
    }
    __syncthreads();
    fence_after();
    lfm_pdl_wait();
    const uint32_t smem = lfm_smem_u32(sm);
    bool ok = true;
    /* job `it`, for all roles but the loader; false at the end */
    auto take = [&](uint32_t it) {
        ok = __all_sync(LFM_FULL_MASK, wait(&bars.job_full[it & 1], (it >> 1) & 1, abort, A.err));
        return ok && bars.job[it & 1].b >= 0;
    };
    auto drop = [&](uint32_t it) {
        __syncwarp();
        if (lane == 0) lfm_mbar_arrive(&bars.job_empty[it & 1]);
    };
    uint32_t base = 0; /* key blocks of the jobs before: ring slots and phases go on from job to job */

    if (warp < 8) {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 152;"); /* 256 x 152 + 256 x 104 = 512 x 128 */
        const uint32_t h = warp >> 2, r = h * kM + (warp & 3) * 32 + lane, tmem = bars.tmem;
        for (uint32_t it = 0; take(it); ++it) {
            const Job &jb = bars.job[it & 1];
            const uint32_t n = jb.n;
            /* this thread's row of q or out */
            auto row_at = [&](size_t stride) {
                const uint32_t row = jb.row0 + r;
                return (size_t)(jb.q0 + row / G) * stride + ((size_t)jb.kvh * G + row % G) * D;
            };
            if (n == 0) { /* no key for any row */
                if (r < jb.rows) {
                    const float z[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
                    const size_t at = row_at(A.out_stride);
                    for (int c = 0; c < D; c += 8) {
                        if (A.type == 0) lfm_store<8>(static_cast<float *>(A.out) + at + c, z);
                        else if (A.type == 1) lfm_store<8>(static_cast<__half *>(A.out) + at + c, z);
                        else lfm_store<8>(static_cast<__nv_bfloat16 *>(A.out) + at + c, z);
                    }
                }
                drop(it);
                continue;
            }
            {
                /* values 8 v .. + 7 and 32 + 8 v .. + 7 of a span make chunks 2 v and 2 v + 1; the last job's products,
                 * waited for below, are done with the space */
                const bool on = r < jb.rows;
                const size_t at = on ? row_at(A.q_stride) : 0;
                uint8_t *to = sm + h * C::kQ + (r % kM) * 16;
                const bool neg = A.scale < 0.0f;
                auto load = [&](const auto *q) { /* the type is told apart once, so the loads are under way together */
#pragma unroll
                    for (int c = 0; c < D / 16; ++c) {
                        float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f}, y[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
                        if (on) {
                            lfm_load<8>(q + at + 64 * (c >> 2) + 8 * (c & 3), x);
                            lfm_load<8>(q + at + 64 * (c >> 2) + 8 * (c & 3) + 32, y);
                        }
                        lfm_fit_q(neg, x);
                        lfm_fit_q(neg, y);
#pragma unroll
                        for (int k = 0; k < 2; ++k)
                            *reinterpret_cast<uint4 *>(to + (2 * c + k) * kChunkQ) =
                                make_uint4(lfm_pack2(x[4 * k], y[4 * k], __half()),
                                           lfm_pack2(x[4 * k + 1], y[4 * k + 1], __half()),
                                           lfm_pack2(x[4 * k + 2], y[4 * k + 2], __half()),
                                           lfm_pack2(x[4 * k + 3], y[4 * k + 3], __half()));
                    }
                };
                if (A.type == 0) load(static_cast<const float *>(A.q));
                else if (A.type == 1) load(static_cast<const __half *>(A.q));
                else load(static_cast<const __nv_bfloat16 *>(A.q));
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0) lfm_mbar_arrive(&bars.q_full[h]);
            }
            const uint32_t tO = tmem + C::kColO + h * D + ((warp & 3) << 21);
            const float sc = fmaxf((kCap ? A.softcap : fabsf(A.scale)) * 1.44269504f, 1e-30f); /* not 0: times -inf */
            const float capz = kCap ? lfm_cap_scale(A.scale, A.softcap) : 0.0f;
            /* what the row sees, in keys from the first block; the blocks [inside0, inside1) every row of the tile sees
             * whole */
            int lo = 0, hi = 0, inside0 = 0, inside1 = 0;
            {
                int64_t a = 0, e = 0, a_all = 0, e_all = 0, unused;
                if (r < jb.rows) lfm_visible(A, jb.n_q, jb.len, jb.row0 + r, a, e);
                if (h * kM < jb.rows) {
                    lfm_visible(A, jb.n_q, jb.len, jb.row0 + h * kM, unused, e_all);
                    lfm_visible(A, jb.n_q, jb.len, jb.row0 + min(jb.rows, (h + 1) * kM) - 1, a_all, unused);
                }
                const int64_t key0 = jb.blk0 * kKeys; /* positions are below 2^31 */
                lo = (int)max((int64_t)0, a - key0);
                hi = (int)max((int64_t)0, e - key0);
                inside0 = (int)((max((int64_t)0, a_all - key0) + kKeys - 1) / kKeys);
                inside1 = (int)(max((int64_t)0, e_all - key0) / kKeys);
            }
            const uint64_t sc2 = pk2(__float_as_uint(sc), __float_as_uint(sc));
            /* O holds the products of block j.  A barrier's parity tells two phases apart: with the scores of block
             * j + 1 the products of j - 2 are done (kBufs <= 6), so those of j and j - 1 take a barrier each, in turn */
            auto products = [&](uint32_t j) {
                return __all_sync(LFM_FULL_MASK, wait(&bars.o_full[h][(base + j) & 1], ((base + j) >> 1) & 1, abort, A.err));
            };
            float m = LFM_NO_KEY;
            uint64_t l2 = 0;
            for (uint32_t j = 0; j < n; ++j) {
                const uint32_t q = 2 * (base + j) + h, buf = q % C::kBufs;
                const uint32_t tS = tmem + buf * kColS + ((warp & 3) << 21);
                ok = __all_sync(LFM_FULL_MASK, wait(&bars.s_full[buf], (q / C::kBufs) & 1, abort, A.err));
                if (!ok) break;
                fence_after();
                const bool masked = (int)j < inside0 || (int)j >= inside1;
                const int from = lo - (int)j * kKeys, to = hi - (int)j * kKeys;
                uint32_t x[kKeys];
                float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
                ld32(tS, x);
                ld32(tS + 32, x + 32);
                wait_ld();
                tie32(x);
                tie32(x + 32);
                if (kCap) {
                    if (A.softcap <= LFM_PLAIN_CAP) {
#pragma unroll
                        for (int i = 0; i < kKeys; ++i) x[i] = __float_as_uint(lfm_tanh(__uint_as_float(x[i]) * capz));
                    } else {
#pragma unroll
                        for (int i = 0; i < kKeys; ++i) x[i] = __float_as_uint(lfm_tanh_any(__uint_as_float(x[i]) * capz));
                    }
                }
                if (masked) {
#pragma unroll
                    for (int i = 0; i < kKeys; ++i)
                        if (i < from || i >= to) x[i] = 0xFF800000u;
                }
#pragma unroll
                for (int i = 0; i < kKeys; i += 8) {
                    max3(mx[0], x[i], x[i + 1]);
                    max3(mx[1], x[i + 2], x[i + 3]);
                    max3(mx[2], x[i + 4], x[i + 5]);
                    max3(mx[3], x[i + 6], x[i + 7]);
                }
                const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
                if (__any_sync(LFM_FULL_MASK, __fmaf_rn(top, sc, -m) > LFM_REF_MOVE)) {
                    const float nm = fmaxf(m, __fmaf_rn(top, sc, -LFM_REF_LOW)), f = lfm_ex2(m - nm);
                    const uint64_t f2 = pk2(__float_as_uint(f), __float_as_uint(f));
                    m = nm;
                    l2 = mul2(l2, f2);
                    if (j) { /* the products of the block before are in O first */
                        ok = products(j - 1);
                        if (!ok) break;
                        fence_after();
#pragma unroll
                        for (int c = 0; c < D; c += 32) {
                            uint32_t o[32];
                            ld32(tO + c, o);
                            wait_ld();
                            tie32(o);
#pragma unroll
                            for (int i = 0; i < 32; i += 2) {
                                const uint64_t x = mul2(pk2(o[i], o[i + 1]), f2);
                                o[i] = (uint32_t)x;
                                o[i + 1] = (uint32_t)(x >> 32);
                            }
                            st32(tO + c, o);
                        }
                    }
                }
                const uint64_t nm2 = pk2(__float_as_uint(-m), __float_as_uint(-m));
                uint64_t la = 0;
                /* each operation on all before the next one: the exponentials' latency hides behind one another */
#pragma unroll
                for (int i = 0; i < kKeys; i += 2) {
                    const uint64_t z = fma2(pk2(x[i], x[i + 1]), sc2, nm2);
                    x[i] = (uint32_t)z;
                    x[i + 1] = (uint32_t)(z >> 32);
                }
#pragma unroll
                for (int i = 0; i < kKeys; ++i) asm volatile("ex2.approx.ftz.f32 %0, %0;" : "+r"(x[i]));
#pragma unroll
                for (int i = 0; i < kKeys; i += 2) {
                    if (i & 2) la = add2(la, pk2(x[i], x[i + 1]));
                    else l2 = add2(l2, pk2(x[i], x[i + 1]));
                    x[i / 2] = lfm_pack2(__uint_as_float(x[i]), __uint_as_float(x[i + 1]), __half());
                }
                l2 = add2(l2, la);
                st32(tS, x);
                wait_st();
                fence_before();
                __syncwarp();
                if (lane == 0) lfm_mbar_arrive(&bars.p_full[buf]);
            }
            /* the barrier of the last products may still be two of its phases back: the one before goes first */
            if (ok && n > 1) ok = products(n - 2);
            if (ok) ok = products(n - 1);
            if (!ok) break;
            {
                fence_after();
                const float l = __uint_as_float((uint32_t)l2) + __uint_as_float((uint32_t)(l2 >> 32));
                const bool on = r < jb.rows;
                const size_t at = on ? row_at(A.out_stride) : 0;
                /* columns 32 c ..: values 16 k .. + 15 of the span in the even ones, 32 + 16 k .. in the odd ones */
                auto write = [&](int c, const float *o, float inv) {
                    if (!on) return;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        float v[8];
#pragma unroll
                        for (int i = 0; i < 8; ++i) v[i] = o[2 * (8 * (e & 1) + i) + (e >> 1)] * inv;
                        const size_t to = at + 64 * (c >> 1) + 16 * (c & 1) + 8 * (e & 1) + 32 * (e >> 1);
                        if (A.type == 0) lfm_store<8>(static_cast<float *>(A.out) + to, v);
                        else if (A.type == 1) lfm_store<8>(static_cast<__half *>(A.out) + to, v);
                        else lfm_store<8>(static_cast<__nv_bfloat16 *>(A.out) + to, v);
                    }
                };
                /* a part: [value / 4][row] of 16 bytes, then the rows' m and sum */
                auto part_of = [&](uint32_t s) { return plan.part + ((size_t)jb.tile * plan.parts + s) * kRows * (D + 2); };
                float *const mine = kSplit && jb.parts > 1 ? part_of(jb.part) : nullptr;
#pragma unroll
                for (int c = 0; c < D / 32; ++c) {
                    uint32_t u[32];
                    float o[32];
                    ld32(tO + 32 * c, u);
                    wait_ld();
                    tie32(u);
#pragma unroll
                    for (int i = 0; i < 32; ++i) o[i] = __uint_as_float(u[i]);
                    if (!kSplit || !mine) {
                        write(c, o, l > 0.0f ? 1.0f / l : 0.0f);
                    } else {
#pragma unroll
                        for (int k = 0; k < 8; ++k)
                            __stcg(reinterpret_cast<float4 *>(mine) + (size_t)(8 * c + k) * kRows + r,
                                   make_float4(o[4 * k], o[4 * k + 1], o[4 * k + 2], o[4 * k + 3]));
                    }
                }
                if (kSplit && mine) {
                    /* the last warp to arrive with a part of these 32 rows joins them all, in their order */
                    __stcg(reinterpret_cast<float2 *>(mine + kRows * D) + r, make_float2(m, l));
                    __threadfence();
                    __syncwarp();
                    uint32_t *const arrived = plan.counts + jb.tile * 8 + warp;
                    uint32_t before = 0;
                    if (lane == 0) before = atomicAdd(arrived, 1u);
                    if (__shfl_sync(LFM_FULL_MASK, before, 0) + 1 == jb.parts) {
                        __threadfence();
                        if (lane == 0) *arrived = 0;
                        auto ml = [&](uint32_t s) {
                            return __ldcg(reinterpret_cast<const float2 *>(part_of(s) + kRows * D) + r);
                        };
                        float top = LFM_NO_KEY, sum = 0.0f;
#pragma unroll 4
                        for (uint32_t s = 0; s < jb.parts; ++s) top = fmaxf(top, ml(s).x);
#pragma unroll 1
                        for (int c = 0; c < D / 32; ++c) {
                            float o[32];
#pragma unroll
                            for (int i = 0; i < 32; ++i) o[i] = 0.0f;
                            sum = 0.0f;
#pragma unroll 2
                            for (uint32_t s = 0; s < jb.parts; ++s) {
                                const float2 x = ml(s);
                                const float f = lfm_ex2(x.x - top);
                                sum = __fmaf_rn(f, x.y, sum);
#pragma unroll
                                for (int k = 0; k < 8; ++k) {
                                    const float4 y = __ldcg(reinterpret_cast<const float4 *>(part_of(s)) +
                                                            (size_t)(8 * c + k) * kRows + r);
                                    o[4 * k] = __fmaf_rn(f, y.x, o[4 * k]);
                                    o[4 * k + 1] = __fmaf_rn(f, y.y, o[4 * k + 1]);
                                    o[4 * k + 2] = __fmaf_rn(f, y.z, o[4 * k + 2]);
                                    o[4 * k + 3] = __fmaf_rn(f, y.w, o[4 * k + 3]);
                                }
                            }
                            write(c, o, sum > 0.0f ? 1.0f / sum : 0.0f);
                        }
                    }
                }
            }
            base += n;
            drop(it);
        }
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 104;");
        if (warp < 12) {
            /* codes -> values */
            const LfmNib nib;
            /* two threads a key: halves of its words */
            const uint32_t key = (warp & 1) * 32 + lane, half = (warp >> 1) & 1;
            const uint32_t codes = key * (D / 2) + half * (D / 4);
            const uint32_t scales = kKeys * (D / 2) + key * (D / 16) + (D == 64 ? 0 : 4 * half);
            for (uint32_t it = 0; take(it); ++it) {
                const uint32_t n = bars.job[it & 1].n;
                /* slots that hold a token that a row sees, counted from the first block: from `lo` on, `held` of them */
                const int64_t key0 = bars.job[it & 1].blk0 * kKeys;
                const uint32_t lo = (uint32_t)max((int64_t)0, bars.job[it & 1].lo - key0), held = (uint32_t)(bars.job[it & 1].len - key0) - lo;
                for (uint32_t u = 2 * base; u < 2 * (base + n); ++u) {
                    const uint32_t rs = u % C::kRaws, os = u % C::kOps;
                    bool w = wait(&bars.raw_full[rs], (u / C::kRaws) & 1, abort, A.err);
                    if (u >= (uint32_t)C::kOps) w = w && wait(&bars.op_empty[os], ((u / C::kOps) & 1) ^ 1, abort, A.err);
                    ok = __all_sync(LFM_FULL_MASK, w);
                    if (!ok) break;
                    const uint8_t *raw = sm + C::kOffRaw + rs * C::kRaw;
                    uint8_t *to = sm + C::kOffOp + os * C::kOp + key * 16 + half * (D / 16) * kChunk;
                    /* a slot that holds no token, or none that a row sees, may hold anything: zero, for V */
                    const uint32_t at = ((u >> 1) - base) * kKeys + key - lo;
                    const uint32_t d = at < held ? *reinterpret_cast<const uint32_t *>(raw + scales) : 0u;
#pragma unroll
                    for (int c = 0; c < D / 64; ++c) {
                        const uint4 a = *reinterpret_cast<const uint4 *>(raw + codes + 16 * c);
                        const uint32_t x[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            const uint32_t y = x[k] >> 8;
                            *reinterpret_cast<uint4 *>(to + (4 * c + k) * kChunk) =
                                make_uint4(lfm_hmul2(lfm_hsub2(nib.lo(x[k]), LFM_NIB0_OFF), d),
                                           lfm_hmul2(lfm_hsub2(nib.hi(x[k]), LFM_NIB1_OFF), d),
                                           lfm_hmul2(lfm_hsub2(nib.lo(y), LFM_NIB0_OFF), d),
                                           lfm_hmul2(lfm_hsub2(nib.hi(y), LFM_NIB1_OFF), d));
                        }
                    }
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    __syncwarp();
                    if (lane == 0) {
                        lfm_mbar_arrive(&bars.op_full[os]);
                        lfm_mbar_arrive(&bars.raw_empty[rs]);
                    }
                }
                if (!ok) break;
                base += n;
                drop(it);
            }
        } else if (warp == 12 || warp == 14) {
            /* A warp a tile: what one spends on barriers between its MMAs is the other's tensor time.  The whole warp
             * walks the loop and one thread issues: descriptors and TMEM addresses (base 0: all columns are ours) then
             * stay in uniform registers.  From a branch of lane 0 alone they take moves through the pipe that the
             * softmax warps' exponentials fill, and an MMA waits 350 cycles for its turn */
            auto full = [&](uint32_t u) {
                const bool w = __all_sync(LFM_FULL_MASK, wait(&bars.op_full[u % C::kOps], (u / C::kOps) & 1, abort, A.err));
                fence_after();
                return w;
            };
            const uint64_t kd0 = sdesc(smem + C::kOffOp, kChunk, 128), vd0 = sdesc(smem + C::kOffOp, 128, kChunk);
            auto walk = [&](auto tile) {
                constexpr uint32_t h = decltype(tile)::value;
                const uint64_t qd = sdesc(smem + h * C::kQ, kChunkQ, 128);
                /* keys of block j are operand 2 j, its values 2 j + 1 */
                auto qk = [&](uint32_t j) {
                    const uint32_t buf = (2 * j + h) % C::kBufs, slot = 2 * j % C::kOps;
                    const uint64_t kd = kd0 + slot * (C::kOp >> 4);
#pragma unroll
                    for (int k = 0; k < D / 16; ++k)
                        mma_ss(buf * kColS, qd + k * (2 * kChunkQ >> 4), kd + k * (2 * kChunk >> 4), kIdescQK, k > 0);
                    commit(&bars.s_full[buf]);
                    commit(&bars.op_empty[slot]);
                };
                auto pv = [&](uint32_t j, bool first) {
                    const uint32_t buf = (2 * j + h) % C::kBufs, slot = (2 * j + 1) % C::kOps;
                    const uint64_t vd = vd0 + slot * (C::kOp >> 4);
#pragma unroll
                    for (int k = 0; k < kKeys / 16; ++k)
                        mma_ts(C::kColO + h * D, buf * kColS + 8 * k, vd + k * (256 >> 4), kIdescPV<D>, !first || k > 0);
                    commit(&bars.o_full[h][j & 1]);
                    commit(&bars.op_empty[slot]);
                };
                constexpr uint32_t kAhead = C::kBufs / 2; /* blocks whose scores are asked for ahead */
                ok = bars.tmem == 0;
                for (uint32_t it = 0, jobs = 0; ok && take(it); ++it) {
                    const uint32_t end = base + bars.job[it & 1].n;
                    if (end > base) {
                        ok = __all_sync(LFM_FULL_MASK, wait(&bars.q_full[h], jobs & 1, abort, A.err));
                        ++jobs;
                    }
                    for (uint32_t j = base; j < base + kAhead && j < end && ok; ++j) {
                        ok = full(2 * j);
                        if (ok && elect()) qk(j);
                    }
                    bool ready = false; /* block j's keys (those asked for ahead), values and probabilities */
                    for (uint32_t j = base; j < end && ok; ++j) {
                        const uint32_t q = 2 * j + h;
                        const bool more = j + kAhead < end;
                        if (!__all_sync(LFM_FULL_MASK, ready))
                            ok = full(2 * j + 1) && (!more || full(2 * (j + kAhead))) &&
                                 __all_sync(LFM_FULL_MASK, wait(&bars.p_full[q % C::kBufs], (q / C::kBufs) & 1, abort, A.err));
                        if (!ok) break;
                        fence_after();
                        const uint32_t u = 2 * j + 3, v = 2 * (j + 1 + kAhead), q1 = q + 2;
                        const bool a = test(&bars.op_full[u % C::kOps], (u / C::kOps) & 1);
                        const bool b = test(&bars.op_full[v % C::kOps], (v / C::kOps) & 1);
                        const bool c = test(&bars.p_full[q1 % C::kBufs], (q1 / C::kBufs) & 1);
                        if (elect()) {
                            pv(j, j == base);
                            if (more) qk(j + kAhead);
                        }
                        ready = j + 1 < end && a && (b || j + 1 + kAhead >= end) && c;
                    }
                    if (!ok) break;
                    base = end;
                    drop(it);
                }
            };
            if (warp == 12) walk(std::integral_constant<uint32_t, 0>());
            else walk(std::integral_constant<uint32_t, 1>());
        } else if (warp == 13) {
            /* a lane the codes or the scales of a page's tokens in the block, K then V: [codes][scales] of all keys */
            const uint32_t P = A.kv.page_tokens, sub = min(P, (uint32_t)kKeys), piece = lane >> 1, part = lane & 1;
            const uint32_t per = part ? D / 16 : D / 2, bytes = sub * per;
            const uint32_t to = C::kOffRaw + (part ? kKeys * (D / 2) : 0) + piece * bytes;
            uint32_t w = blockIdx.x;
            const uint32_t parts = kSplit ? plan.parts : 1;
            /* parts are few rounds of the blocks: no ticket goes to a tile that is not there */
            uint32_t tiles = plan.tiles;
            if (kSplit) tiles = (uint32_t)min((uint64_t)tiles, lfm_find_tile(A.bt, G, kRows, plan.above, ~0ull, bars.tile));
            for (uint32_t it = 0; ok; ++it) {
                /* the next job: the longest walks first (tiles from the last), all heads of one side by side */
                Job jb;
                jb.b = -1;
                jb.n = 0;
                for (; w < tiles * A.kv.hkv * parts; w = gridDim.x + __shfl_sync(LFM_FULL_MASK, w, 0)) {
                    const uint32_t tile = w / (A.kv.hkv * parts);
                    lfm_find_tile(A.bt, G, kRows, plan.above, tiles - 1 - tile, bars.tile);
                    __syncwarp();
                    const int b = *(volatile int *)&bars.tile[0];
                    jb.row0 = (uint32_t)*(volatile int *)&bars.tile[1] * kRows;
                    jb.kvh = w % A.kv.hkv;
                    const uint32_t part = w / A.kv.hkv % parts;
                    __syncwarp();
                    if (lane == 0) w = atomicAdd(ticket, 1u); /* of the one after */
                    if (b < 0) continue;
                    jb.q0 = A.bt.q_start[b];
                    jb.n_q = (int64_t)A.bt.q_start[b + 1] - jb.q0;
                    jb.len = A.bt.kv_len[b];
                    if (!lfm_sane_len(A.bt, jb.len)) {
                        if (lane == 0) atomicOr(A.err, LFM_DEVERR_PAGE);
                        continue;
                    }
                    jb.rows = (uint32_t)min((int64_t)kRows, jb.n_q * (int64_t)G - jb.row0); /* at least 1 */
                    int64_t lo0, hi0, lo1, hi1;
                    lfm_visible(A, jb.n_q, jb.len, jb.row0, lo0, hi0);
                    lfm_visible(A, jb.n_q, jb.len, jb.row0 + jb.rows - 1, lo1, hi1);
                    jb.lo = lo0;
                    jb.blk0 = lo0 / kKeys;
                    jb.n = hi1 > lo0 ? (uint32_t)((hi1 + kKeys - 1) / kKeys - jb.blk0) : 0;
                    if (kSplit) {
                        jb.tile = tile * A.kv.hkv + jb.kvh;
                        jb.part = part;
                        jb.parts = min(parts, max(1u, jb.n / kPartBlocks));
                        if (part >= jb.parts) continue;
                        const uint32_t at = (uint32_t)((uint64_t)jb.n * part / jb.parts);
                        jb.n = (uint32_t)((uint64_t)jb.n * (part + 1) / jb.parts) - at;
                        jb.blk0 += at;
                    }
                    jb.b = b;
                    break;
                }
                if (jb.b >= 0) w = gridDim.x + __shfl_sync(LFM_FULL_MASK, w, 0);
                if (it > 1) ok = __all_sync(LFM_FULL_MASK, wait(&bars.job_empty[it & 1], ((it >> 1) & 1) ^ 1, abort, A.err));
                if (!ok) break;
                if (lane == 0) {
                    bars.job[it & 1] = jb;
                    lfm_mbar_arrive(&bars.job_full[it & 1]);
                }
                if (jb.b < 0) break;
                const uint32_t n = jb.n;
                for (uint32_t j = 0; j < n; ++j) {
                    const int64_t key = (jb.blk0 + j) * kKeys + (int64_t)piece * sub;
                    const uint8_t *page = nullptr; /* one below the window may be gone */
                    if (piece * sub < kKeys && key < jb.len && key + sub > jb.lo) page = lfm_page(A.kv, A.bt, jb.b, key, jb.kvh, A.err);
                    const uint32_t all = __reduce_add_sync(LFM_FULL_MASK, page ? bytes : 0u);
                    const uint32_t in = ((uint32_t)key & (P - 1)) * per + (part ? A.kv.codes : 0);
#pragma unroll
                    for (uint32_t k = 0; k < 2; ++k) {
                        const uint32_t u = 2 * (base + j) + k, rs = u % C::kRaws;
                        ok = ok && (u < (uint32_t)C::kRaws || wait(&bars.raw_empty[rs], ((u / C::kRaws) & 1) ^ 1, abort, A.err));
                        ok = __all_sync(LFM_FULL_MASK, ok);
                        if (!ok) break;
                        if (lane == 0) lfm_mbar_arrive_tx(&bars.raw_full[rs], all);
                        __syncwarp();
                        if (page)
                            lfm_bulk_g2s_plain(sm + to + rs * C::kRaw, page + in + (k ? A.kv.half : 0), bytes,
                                               &bars.raw_full[rs]);
                    }
                    if (!ok) break;
                }
                base += n;
            }
            /* the last block to come here leaves the counters zero */
            if (lane == 0 && atomicAdd(ticket + 1, 1u) == gridDim.x - 1) {
                ticket[0] = 0;
                ticket[1] = 0;
            }
        }
    }
    /* the loader passes bad sequences over.  Warp 15, which has no other part, reports them, from behind the roles: beside
     * them the check made prompts 2% slower */
    if (blockIdx.x == 0 && warp == 15) lfm_check_batch(A.bt, lane, 32, A.err);
    if (!ok) *abort = 1;
    fence_before();
    __syncthreads();
    if (*abort) {
        /* copies and MMAs already issued end within microseconds: let them land */
        const uint64_t t0 = lfm_globaltimer();
        while (lfm_globaltimer() - t0 < 2000000ull) {
        }
    }
    if (warp == 12) {
        __syncwarp();
        fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(bars.tmem), "r"(kTmemCols));
    }
}

template <int D>
cudaError_t launch_tile(const AttnArgs &a, const TilePlan &p, dim3 grid, cudaStream_t s, bool pdl) {
    static size_t set[4][16];
    const bool cap = a.softcap > 0.0f, split = p.parts > 1;
    auto fn = split ? (cap ? k_attn_tile<D, true, true> : k_attn_tile<D, false, true>)
                    : (cap ? k_attn_tile<D, true, false> : k_attn_tile<D, false, false>);
    const cudaError_t e = lfm_smem_attr((const void *)fn, Cfg<D>::kSmem, set[2 * split + cap]);
    return e != cudaSuccess ? e : lfm_launch_pdl(fn, grid, dim3(kThreads), Cfg<D>::kSmem, s, pdl, a, p);
}

}  // namespace

TilePlan lfm_attn_tile_plan(const AttnArgs &a, uint32_t head_dim, uint64_t above, uint32_t max_kv_len, int sm_count) {
    /* a tile for every started kRows rows of a sequence of more than `above`: at most this many */
    const uint64_t rows = (uint64_t)a.bt.n_tokens * a.group, most = rows / (above + 1), sms = (uint64_t)sm_count;
    TilePlan p{};
    p.above = above;
    p.tiles = (uint32_t)((rows + (kRows - 1) * (most < a.bt.n_seqs ? most : a.bt.n_seqs)) / kRows);
    const uint64_t jobs = (uint64_t)p.tiles * a.kv.hkv;
    const uint64_t blocks = max_kv_len / kKeys + 1;
    /* parts: as many as make the busiest SM's walk shortest.  One of more than a part pays for what it writes, and the
     * last one joins n (a part of 128 values is as many bytes as a block takes time) */
    const uint64_t bound = blocks / kPartBlocks < LFM_ATTN_TILES ? blocks / kPartBlocks : LFM_ATTN_TILES;
    for (uint64_t n = 1; n == 1 || (n <= bound && jobs * n <= LFM_ATTN_TILES && jobs * 8 <= LFM_ATTN_COUNTS - 2); ++n) {
        const uint64_t rounds = (jobs * n + sms - 1) / sms, walk = (blocks + n - 1) / n + kJobBlocks + (n > 1);
        const uint64_t cost = rounds * walk + (n > 1 ? n * head_dim / 128 : 0);
        if (n == 1 || cost < p.cost) {
            p.cost = cost;
            p.parts = (uint32_t)n;
        }
    }
    p.blocks = blocks;
    return p;
}

cudaError_t lfm_launch_attn_tile(const AttnArgs &a, uint32_t head_dim, const TilePlan &plan, int sm_count, void *scratch,
                                 cudaStream_t s, bool pdl) {
    TilePlan p = plan;
    const uint64_t jobs = (uint64_t)p.tiles * a.kv.hkv * p.parts;
    if (jobs == 0) return cudaSuccess;
    if (jobs > 0x7FFFFFFFull) return cudaErrorInvalidConfiguration;
    p.counts = static_cast<uint32_t *>(scratch);
    p.part = reinterpret_cast<float *>(p.counts + LFM_ATTN_COUNTS);
    const dim3 grid((uint32_t)(jobs < (uint64_t)sm_count ? jobs : (uint64_t)sm_count));
    return head_dim == 64 ? launch_tile<64>(a, p, grid, s, pdl) : launch_tile<128>(a, p, grid, s, pdl);
}
