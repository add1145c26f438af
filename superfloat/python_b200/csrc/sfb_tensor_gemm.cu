// The matrix products of the tensor-core linear on tcgen05, with their epilogues.
//
//   forward   z = (x code^T) s[n] 2^-(bits-1) + b[n],  y = act(z) + r
//   x grad    dx = (dz s) code          contraction over the channels n
//   w grad    dW = dz^T x               contraction over the rows m
//
// sf4..sf8 codes are integers of at most 7 bits, exact in bf16 and fp16, so the
// operands of the forward product are exact; the sums are held in float32 in
// TMEM and rounded once, when they are stored.
//
// One CTA per SM walks output tiles; warp 0 lane 0 issues the TMA loads (64
// elements of the contraction a stage, 128-byte swizzle), warp 1 lane 0 the MMAs,
// warps 2..9 read the accumulator out of TMEM, two warps to each group of 32
// lanes, each half of the columns.  Two accumulators (2 BN TMEM columns) let a
// tile's epilogue run under the next tile's products.
// CTAS = 2: a pair of SMs shares a tile of 256 x BN.  Each holds 128 rows of A,
// half of B's columns and the sums of its own rows; the first one's thread issues
// the products of both (cta_group::2).  B crosses into shared memory once for
// the pair, which a single SM's tile of 128 x 256 has to load and read twice.
// CTAS = 1: tiles of 128 x BN, for problems with too few tiles for the pairs.
// An operand whose contraction index is contiguous in memory is loaded K-major
// (rows of 64); one whose row index is contiguous MN-major (64 rows wide, 64
// deep), so that no operand of the backward products is transposed beforehand.
//
// Every wait is bounded; one that runs out is counted in g_failures, the CTA's
// remaining outputs are written as NaN, and the CTA waits for its copies and
// products in flight before it frees its TMEM.
#include <cuda.h>

#include <algorithm>
#include <mutex>

#include "sfb_tensor.cuh"

namespace sfb {

unsigned wait_polls();                        // the calling thread's sfb_wide_wait_limit
int wait_stall();

namespace {

constexpr int BM = 128, BK = 64, THREADS = 320, EPI_WARPS = 8;
constexpr unsigned kSpinLimit = 1u << 26;     // polls of one wait, some seconds
constexpr int SMEM_OPERANDS = 196608;         // of the stages
constexpr int GROUP_ROWS = 1024;              // rows that sweep the columns together, for L2

__device__ unsigned long long g_failures;

// --- PTX -----------------------------------------------------------------------------------------------------

__device__ __forceinline__ uint32_t smem_u32(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }

__device__ __forceinline__ void mbar_init(uint32_t bar, uint32_t count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}

__device__ __forceinline__ void mbar_expect_tx(uint32_t bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}

__device__ __forceinline__ void mbar_arrive(uint32_t bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}

// one lane of the warp, the same each time.  The warps that issue copies and
// products run their loops as a whole and only the issue is one lane's: descriptors
// and addresses then stay in uniform registers.  With the loops inside `if
// (threadIdx.x == 32)` a stage of 4 products took 750 cycles to issue, whatever
// their size (timestamps around the issue; 128 x 128 and 256 x 256 tiles alike).
__device__ __forceinline__ bool elected() {
    uint32_t p;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "elect.sync _|p, 0xffffffff;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(p));
    return p != 0;
}

// the same barrier of the pair's first CTA
__device__ __forceinline__ uint32_t of_leader(uint32_t bar) {
    uint32_t r;
    asm("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(r) : "r"(bar));
    return r;
}

__device__ __forceinline__ void mbar_arrive_cluster(uint32_t bar) {
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}

__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// false once `limit` polls have not seen the phase of this parity end
__device__ __forceinline__ bool mbar_wait(uint32_t bar, uint32_t parity, unsigned limit) {
    for (unsigned i = 0; i < limit; i++) {
        uint32_t ok;
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
            "selp.u32 %0, 1, 0, p;\n\t}"
            : "=r"(ok)
            : "r"(bar), "r"(parity)
            : "memory");
        if (ok) return true;
    }
    return false;
}

// the same wait by all lanes of a warp, with one answer
__device__ __forceinline__ bool all_wait(uint32_t bar, uint32_t parity, unsigned limit) {
    return __all_sync(0xffffffffu, mbar_wait(bar, parity, limit));
}

// into this CTA's shared memory; the barrier is the pair's first CTA's with CTAS = 2
template <int CTAS>
__device__ __forceinline__ void tma_load_2d(uint32_t dst, const CUtensorMap *map, int c0, int c1, uint32_t bar) {
    if constexpr (CTAS == 2)
        asm volatile(
            "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, "
            "{%2, %3}], [%4];" ::"r"(dst),
            "l"(map), "r"(c0), "r"(c1), "r"(bar)
            : "memory");
    else
        asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], "
        "[%4];" ::"r"(dst),
        "l"(map), "r"(c0), "r"(c1), "r"(bar)
        : "memory");
}

__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// Shared-memory descriptor, 128-byte swizzle.  K-major: rows of 128 bytes, groups
// of 8 rows 1024 bytes apart (the stride offset; the leading one is unused).
// MN-major: 64 rows of the operand by 64 k, each k a line of 128 bytes; groups of
// 8 k are 1024 bytes apart, the next 64 rows 8192 (the leading offset).
template <bool MN>
__device__ __forceinline__ uint64_t smem_desc(uint32_t addr) {
    uint64_t d = 0;
    d |= (uint64_t)((addr >> 4) & 0x3FFF);
    d |= (uint64_t)(MN ? 8192 >> 4 : 1) << 16;
    d |= (uint64_t)(1024 >> 4) << 32;
    d |= (uint64_t)1 << 46;                 // descriptor version for sm_100
    d |= (uint64_t)2 << 61;                 // SWIZZLE_128B
    return d;
}

template <typename T> struct Kind;
template <> struct Kind<__half> { static constexpr uint32_t id = 0; };
template <> struct Kind<__nv_bfloat16> { static constexpr uint32_t id = 1; };

// kind::f16: float32 accumulator, both operands of type T, M = 128 CTAS, N = BN
template <typename T, bool A_MN, bool B_MN, int BN, int CTAS>
__host__ __device__ constexpr uint32_t instruction() {
    return (1u << 4) | (Kind<T>::id << 7) | (Kind<T>::id << 10) | ((uint32_t)A_MN << 15) | ((uint32_t)B_MN << 16) |
           ((uint32_t)(BN >> 3) << 17) | ((uint32_t)(CTAS * BM >> 4) << 24);
}

template <int CTAS>
__device__ __forceinline__ void mma(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc,
                                    uint32_t accumulate) {
    if constexpr (CTAS == 2)
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "setp.ne.b32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(tmem_d),
            "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
            : "memory");
    else
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "setp.ne.b32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(tmem_d),
            "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
            : "memory");
}

// arrives on this CTA's barrier once the products issued so far are done
template <int CTAS>
__device__ __forceinline__ void mma_commit(uint32_t bar) {
    if constexpr (CTAS == 2)
        asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
    else
        asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}

// on that barrier of both CTAs of a pair
template <int CTAS>
__device__ __forceinline__ void mma_commit_all(uint32_t bar) {
    if constexpr (CTAS == 2)
        asm volatile(
            "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar),
            "h"((uint16_t)3)
            : "memory");
    else
        mma_commit<1>(bar);
}

__device__ __forceinline__ void tmem_ld32(uint32_t taddr, float (&v)[32]) {
    uint32_t r[32];
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,"
        "%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
          "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
          "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr));
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
    for (int i = 0; i < 32; i++) v[i] = __uint_as_float(r[i]);
}

// --- the epilogue --------------------------------------------------------------------------------------------

struct Epilogue {
    const float *scale;          // per column (forward), or null
    const void *bias;            // per column, or null
    const void *residual;        // of the operands' type, or null
    const float *alpha;          // one factor for all, in device memory, or null
    __half *z;                   // the pre-activation for the backward pass, or null
    void *y;
    float unit;                  // 2^-(bits-1) where a scale or alpha stands for codes, else 1
    int bias_dtype, y_dtype;
    int64_t ldr, ldz, ldy;
    bool vec;                    // rows of y, r and z are aligned to 16 bytes
};

template <typename Y>
__device__ __forceinline__ void put8(Y *to, const float *v) {
    Vec<Y, 8> q;
#pragma unroll
    for (int j = 0; j < 8; j++) q.v[j] = from_f<Y>(v[j]);
    *reinterpret_cast<Vec<Y, 8> *>(to) = q;
}

// 8 columns n .. n + 7 of one row
template <typename T, int ACT>
__device__ __forceinline__ void finish8(const Epilogue &e, float (&v)[8], const float *scale, const float *bias,
                                        int64_t m, int64_t n, int64_t N) {
#pragma unroll
    for (int j = 0; j < 8; j++) v[j] = fmaf(v[j], scale[j], bias[j]);
    const bool vec = e.vec && n + 8 <= N;
    if (e.z) {
        __half *to = e.z + m * e.ldz + n;
        if (vec) {
            Vec<__half, 8> q;
#pragma unroll
            for (int j = 0; j < 8; j++) q.v[j] = kept(v[j]);
            *reinterpret_cast<Vec<__half, 8> *>(to) = q;
        } else {
#pragma unroll
            for (int j = 0; j < 8; j++)
                if (n + j < N) to[j] = kept(v[j]);
        }
    }
#pragma unroll
    for (int j = 0; j < 8; j++) v[j] = activate<ACT>(v[j]);
    if (e.residual) {
        const T *from = static_cast<const T *>(e.residual) + m * e.ldr + n;
        if (vec) {
            const Vec<T, 8> q = *reinterpret_cast<const Vec<T, 8> *>(from);
#pragma unroll
            for (int j = 0; j < 8; j++) v[j] += to_f(q.v[j]);
        } else {
#pragma unroll
            for (int j = 0; j < 8; j++)
                if (n + j < N) v[j] += to_f(from[j]);
        }
    }
    const int64_t at = m * e.ldy + n;
    if (vec) {
        if (e.y_dtype == SFB_F32) put8(static_cast<float *>(e.y) + at, v);
        else if (e.y_dtype == SFB_BF16) put8(static_cast<__nv_bfloat16 *>(e.y) + at, v);
        else put8(static_cast<__half *>(e.y) + at, v);
    } else {
#pragma unroll
        for (int j = 0; j < 8; j++)
            if (n + j < N) store_as(e.y, at + j, e.y_dtype, v[j]);
    }
}

struct Tiles {
    int mt, nt, total;
};

template <int CTAS>
__device__ __forceinline__ void tile_of(const Tiles &t, int i, int &tm, int &tn) {
    constexpr int GROUP_M = GROUP_ROWS / (CTAS * BM);
    const int gsize = GROUP_M * t.nt, g = i / gsize, m0 = g * GROUP_M;
    const int gm = min(GROUP_M, t.mt - m0), r = i - g * gsize;
    tm = m0 + r % gm;
    tn = r / gm;
}

template <int BN, int CTAS>
struct Shape {
    static constexpr int BNL = BN / CTAS;                            // columns of B that a CTA loads
    static constexpr int A = BM * BK * 2, B = BNL * BK * 2, STAGE = A + B, STAGES = SMEM_OPERANDS / STAGE;
    static constexpr int COLS = 2 * BN;                              // TMEM columns
    static constexpr int FACTORS = EPI_WARPS * 2 * (BN / 2) * 4;     // each warp's scales and biases
    static constexpr int SMEM = STAGES * STAGE + FACTORS + 512 + 1024;
};

template <typename T, bool A_MN, bool B_MN, int BN, int CTAS, int ACT>
__global__ void __launch_bounds__(THREADS, 1)
gemm_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB, int nkb, int64_t M,
            int64_t N, Tiles tiles, const __grid_constant__ Epilogue e, unsigned spin, int stall) {
    using S = Shape<BN, CTAS>;
    constexpr int STAGES = S::STAGES;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    float *factors = reinterpret_cast<float *>(smem + STAGES * S::STAGE);
    uint64_t *bars = reinterpret_cast<uint64_t *>(smem + STAGES * S::STAGE + S::FACTORS);
    // full [0, S), empty [S, 2 S), accumulator full 2 S + {0, 1}, accumulator empty 2 S + {2, 3}, all done 2 S + 4,
    // and one that nothing arrives on (the tests' stall).  Of a pair, the first CTA's full, accumulator empty and
    // done barriers serve both; each has its own empty and accumulator full ones.
    auto full = [&](int s) { return smem_u32(&bars[s]); };
    auto empty = [&](int s) { return smem_u32(&bars[STAGES + s]); };
    auto acc_full = [&](int a) { return smem_u32(&bars[2 * STAGES + a]); };
    auto acc_empty = [&](int a) { return smem_u32(&bars[2 * STAGES + 2 + a]); };
    const uint32_t done = smem_u32(&bars[2 * STAGES + 4]), never = smem_u32(&bars[2 * STAGES + 5]);
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(bars + 2 * STAGES + 6);
    __shared__ int s_fail;
    volatile int *failed = &s_fail;

    const int warp = __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
    const int rank = CTAS == 2 ? (int)(blockIdx.x & 1) : 0, first = blockIdx.x / CTAS, step = gridDim.x / CTAS;
    if (threadIdx.x == 0) {
        s_fail = 0;
        for (int s = 0; s < STAGES; s++) {
            mbar_init(full(s), 1);
            mbar_init(empty(s), 1);
        }
        for (int a = 0; a < 2; a++) {
            mbar_init(acc_full(a), 1);
            mbar_init(acc_empty(a), CTAS * EPI_WARPS);
        }
        mbar_init(done, 1);
        mbar_init(never, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 0) {
        if constexpr (CTAS == 2) {
            asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                         "n"(S::COLS)
                         : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
        } else {
            asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                         "n"(S::COLS)
                         : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
        }
    }
    tc_fence_before();
    __syncthreads();
    if constexpr (CTAS == 2) cluster_sync();           // the barriers of both are set
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;

    int issued = 0;
    if (warp == 0) {
        for (int t = first; t < tiles.total; t += step) {
            int tm, tn;
            tile_of<CTAS>(tiles, t, tm, tn);
            const int m0 = (tm * CTAS + rank) * BM, n0 = tn * BN + rank * S::BNL;
            for (int kb = 0; kb < nkb; kb++, issued++) {
                const int s = issued % STAGES, round = issued / STAGES;
                if (round > 0 && !all_wait(empty(s), (round - 1) & 1, spin)) {
                    *failed = 1;
                    break;
                }
                if (__any_sync(0xffffffffu, *failed)) break;
                const uint32_t a = smem_u32(smem + s * S::STAGE), b = a + S::A;
                const uint32_t bar = CTAS == 2 ? of_leader(full(s)) : full(s);
                if (elected()) {
                    if (rank == 0) mbar_expect_tx(full(s), CTAS * S::STAGE);
                    if constexpr (A_MN) {
#pragma unroll
                        for (int i = 0; i < BM / 64; i++) tma_load_2d<CTAS>(a + i * 8192, &tmA, m0 + i * 64, kb * BK, bar);
                    } else {
                        tma_load_2d<CTAS>(a, &tmA, kb * BK, m0, bar);
                    }
                    if constexpr (B_MN) {
#pragma unroll
                        for (int i = 0; i < S::BNL / 64; i++)
                            tma_load_2d<CTAS>(b + i * 8192, &tmB, n0 + i * 64, kb * BK, bar);
                    } else {
                        tma_load_2d<CTAS>(b, &tmB, kb * BK, n0, bar);
                    }
                }
                __syncwarp();
            }
            if (__any_sync(0xffffffffu, *failed)) break;
        }
    } else if (warp == 1 && rank == 0) {
        constexpr uint32_t id = instruction<T, A_MN, B_MN, BN, CTAS>();
        bool ok = !(stall && !all_wait(never, 0, spin));
        int it = 0, i = 0;
        for (int t = first; t < tiles.total && ok; t += step, i++) {
            const int acc = i & 1;
            if (i >= 2 && !all_wait(acc_empty(acc), ((i >> 1) - 1) & 1, spin)) {
                ok = false;
                break;
            }
            tc_fence_after();
            for (int kb = 0; kb < nkb; kb++, it++) {
                const int s = it % STAGES;
                if (!all_wait(full(s), (it / STAGES) & 1, spin) || __any_sync(0xffffffffu, *failed)) {
                    ok = false;
                    break;
                }
                tc_fence_after();
                const uint32_t a = smem_u32(smem + s * S::STAGE), b = a + S::A;
                if (elected()) {
#pragma unroll
                    for (int kk = 0; kk < BK / 16; kk++)
                        mma<CTAS>(tmem + acc * BN, smem_desc<A_MN>(a + kk * (A_MN ? 2048 : 32)),
                                  smem_desc<B_MN>(b + kk * (B_MN ? 2048 : 32)), id, kb == 0 && kk == 0 ? 0u : 1u);
                    mma_commit_all<CTAS>(empty(s));
                }
                __syncwarp();
            }
            if (ok && elected()) mma_commit_all<CTAS>(acc_full(acc));
            __syncwarp();
        }
        if (!ok) *failed = 1;
        if (elected()) {
            if (!ok) {
                // release this CTA's epilogue, which sees that the CTA failed; the other CTA's waits run out by themselves
                mma_commit<CTAS>(acc_full(0));
                mma_commit<CTAS>(acc_full(1));
            }
            mma_commit<CTAS>(done);
        }
    } else if (warp >= 2) {
        const int half = (warp - 2) >> 2, quad = warp & 3;        // a warp reaches the TMEM lanes 32 (warp % 4) ..
        const uint32_t lanes = (uint32_t)(32 * quad) << 16;
        float *scale = factors + (warp - 2) * BN, *bias = scale + BN / 2;
        const float alpha = e.alpha ? *e.alpha * e.unit : e.unit;
        int i = 0;
        for (int t = first; t < tiles.total; t += step, i++) {
            int tm, tn;
            tile_of<CTAS>(tiles, t, tm, tn);
            const int acc = i & 1;
            const int64_t n0 = (int64_t)tn * BN + half * (BN / 2);
            __syncwarp();
            for (int c = lane; c < BN / 2; c += 32) {
                scale[c] = n0 + c < N && e.scale ? e.scale[n0 + c] * alpha : alpha;
                bias[c] = n0 + c < N && e.bias ? load_as(e.bias, n0 + c, e.bias_dtype) : 0.0f;
            }
            // one lane polls: 256 of them would crowd the copies' and products' issue out of the memory pipe
            int fine = 0;
            if (lane == 0) fine = !*failed && mbar_wait(acc_full(acc), (i >> 1) & 1, spin) && !*failed;
            fine = __shfl_sync(0xffffffffu, fine, 0);    // TMEM loads are the whole warp's
            if (!fine) *failed = 1;
            tc_fence_after();
            const int64_t m = (int64_t)(tm * CTAS + rank) * BM + quad * 32 + lane;
            for (int c = 0; c < BN / 2; c += 32) {
                if (n0 + c >= N) break;
                float v[32];
                if (fine) {
                    tmem_ld32(tmem + lanes + acc * BN + half * (BN / 2) + c, v);
                } else {
#pragma unroll
                    for (int j = 0; j < 32; j++) v[j] = __int_as_float(0x7FC00000);
                }
                if (m < M) {
#pragma unroll
                    for (int j = 0; j < 32; j += 8)
                        if (n0 + c + j < N)
                            finish8<T, ACT>(e, *reinterpret_cast<float(*)[8]>(v + j), scale + c + j, bias + c + j, m,
                                            n0 + c + j, N);
                }
                __syncwarp();
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) {
                if constexpr (CTAS == 2) mbar_arrive_cluster(of_leader(acc_empty(acc)));
                else mbar_arrive(acc_empty(acc));
            }
        }
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if (s_fail && threadIdx.x == 0) {
        atomicAdd(&g_failures, 1ull);
        // the copies land before their shared memory is released (a pair's complete on the first CTA's barriers; the
        // other CTA waits for it below), the products (the commit on `done` follows them) end before TMEM is freed:
        // full-length waits, whatever `spin` was
        if (rank == 0) {
            for (int it = issued > STAGES ? issued - STAGES : 0; it < issued; it++)
                (void)mbar_wait(full(it % STAGES), (it / STAGES) & 1, kSpinLimit);
            (void)mbar_wait(done, 0, kSpinLimit);
        }
    }
    tc_fence_before();
    __syncthreads();
    if constexpr (CTAS == 2) cluster_sync();           // neither leaves while the other's copies or arrivals may come
    tc_fence_after();
    if (warp == 0) {
        if constexpr (CTAS == 2)
            asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(S::COLS) : "memory");
        else
            asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(S::COLS) : "memory");
    }
}

// --- launches ------------------------------------------------------------------------------------------------

typedef CUresult (*EncodeTiled)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *,
                                const cuuint64_t *, const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave,
                                CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiled encoder() {
    static EncodeTiled fn = nullptr;
    static std::once_flag once;
    std::call_once(once, [] {
        void *p = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
            q == cudaDriverEntryPointSuccess)
            fn = reinterpret_cast<EncodeTiled>(p);
    });
    return fn;
}

// a matrix of `rows` lines of `cols` elements, ld apart, read in boxes of 64 columns
int make_map(CUtensorMap *map, const void *base, int dtype, int64_t rows, int64_t cols, int64_t ld, int box_rows) {
    EncodeTiled enc = encoder();
    if (!enc) return set_error(SFB_ECUDA, "sf tensor linear: cuTensorMapEncodeTiled is unavailable");
    const cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
    const cuuint64_t strides[1] = {(cuuint64_t)ld * 2};
    const cuuint32_t box[2] = {64, (cuuint32_t)box_rows};
    const cuuint32_t estr[2] = {1, 1};
    const CUresult r = enc(map, dtype == SFB_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16,
                           2, const_cast<void *>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                           CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                           CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return set_error(SFB_ECUDA, "sf tensor linear: tensor map encoding failed (%d)", (int)r);
    return SFB_OK;
}

struct Problem {
    const void *A, *B;
    int64_t lda, ldb, M, N, K;
    int dtype;
};

template <typename T, bool A_MN, bool B_MN, int BN, int CTAS, int ACT>
int launch(const Problem &p, const Epilogue &e, cudaStream_t st) {
    using S = Shape<BN, CTAS>;
    auto *kernel = gemm_kernel<T, A_MN, B_MN, BN, CTAS, ACT>;
    static std::mutex lock;
    static unsigned long long ready[64] = {};          // the CUDA context whose attribute is set, per device
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64)
        return set_error(SFB_ECUDA, "sf tensor linear: no current CUDA device");
    {
        std::lock_guard<std::mutex> g(lock);
        const unsigned long long ctx = context_id();
        if (ctx == 0 || ready[dev] != ctx) {
            if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, S::SMEM) != cudaSuccess)
                return check_launch("sf tensor linear (attributes)");
            ready[dev] = context_id();
        }
    }
    CUtensorMap tmA, tmB;
    int rc = A_MN ? make_map(&tmA, p.A, p.dtype, p.K, p.M, p.lda, BK) : make_map(&tmA, p.A, p.dtype, p.M, p.K, p.lda, BM);
    if (rc) return rc;
    rc = B_MN ? make_map(&tmB, p.B, p.dtype, p.K, p.N, p.ldb, BK) : make_map(&tmB, p.B, p.dtype, p.N, p.K, p.ldb, S::BNL);
    if (rc) return rc;
    Tiles t;
    t.mt = (int)((p.M + CTAS * BM - 1) / (CTAS * BM));
    t.nt = (int)((p.N + BN - 1) / BN);
    t.total = t.mt * t.nt;
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute pair;
    pair.id = cudaLaunchAttributeClusterDimension;
    pair.val.clusterDim.x = CTAS;
    pair.val.clusterDim.y = pair.val.clusterDim.z = 1;
    cfg.gridDim = dim3((unsigned)(CTAS * std::min(t.total, sm_count() / CTAS)));
    cfg.blockDim = dim3(THREADS);
    cfg.dynamicSmemBytes = S::SMEM;
    cfg.stream = st;
    cfg.attrs = &pair;
    cfg.numAttrs = CTAS > 1 ? 1 : 0;
    const unsigned spin = wait_polls() ? wait_polls() : kSpinLimit;
    if (cudaLaunchKernelEx(&cfg, kernel, tmA, tmB, (int)((p.K + BK - 1) / BK), p.M, p.N, t, e, spin, wait_stall()) !=
        cudaSuccess)
        return check_launch("sf tensor linear");
    return check_launch("sf tensor linear");
}

// The tile: passes over the SMs times what a pass costs.  A pair's tile of 256 x
// 256 keeps its two SMs as busy as 128 x 128 keeps one for 0.6 of that time.
bool pairs(int64_t M, int64_t N) {
    const int64_t sms = sm_count(), two = ((M + 255) / 256) * ((N + 255) / 256),
                  one = ((M + BM - 1) / BM) * ((N + 127) / 128);
    return (double)((two + sms / 2 - 1) / (sms / 2)) <= 0.6 * (double)((one + sms - 1) / sms);
}

int check(const Problem &p, const char *what) {
    if (p.dtype != SFB_BF16 && p.dtype != SFB_F16) return set_error(SFB_EINVAL, "%s: element type %d", what, p.dtype);
    if (p.M < 0 || p.N < 0 || p.K < 1) return set_error(SFB_EINVAL, "%s: bad shape", what);
    if (p.M >= (1ll << 31) || p.N >= (1ll << 31) || p.K >= (1ll << 31) || p.lda >= (1ll << 36) || p.ldb >= (1ll << 36) ||
        ((p.M + BM - 1) / BM) * ((p.N + 127) / 128) >= (1ll << 31))
        return set_error(SFB_ERANGE, "%s: a size of %lld x %lld x %lld", what, (long long)p.M, (long long)p.N,
                         (long long)p.K);
    if (p.M == 0 || p.N == 0) return SFB_OK;
    if (!p.A || !p.B) return set_error(SFB_EINVAL, "%s: null pointer", what);
    if (((reinterpret_cast<uintptr_t>(p.A) | reinterpret_cast<uintptr_t>(p.B)) & 15) || p.lda % 8 || p.ldb % 8)
        return set_error(SFB_EINVAL, "%s: operands and their rows must be aligned to 16 bytes", what);
    return SFB_OK;
}

bool aligned16(const void *p, int64_t ld, int size) {
    return p == nullptr || ((reinterpret_cast<uintptr_t>(p) & 15) == 0 && (ld * size) % 16 == 0);
}

template <bool A_MN, bool B_MN, int ACT>
int launch_typed(const Problem &p, const Epilogue &e, cudaStream_t st) {
    const bool two = pairs(p.M, p.N);
    if (p.dtype == SFB_BF16)
        return two ? launch<__nv_bfloat16, A_MN, B_MN, 256, 2, ACT>(p, e, st)
                   : launch<__nv_bfloat16, A_MN, B_MN, 128, 1, ACT>(p, e, st);
    return two ? launch<__half, A_MN, B_MN, 256, 2, ACT>(p, e, st) : launch<__half, A_MN, B_MN, 128, 1, ACT>(p, e, st);
}

}  // namespace
}  // namespace sfb

extern "C" int sfb_tensor_linear(int dtype, const void *x, int64_t ldx, const void *codes, int64_t ldw,
                                 const float *scale, int bits, const void *bias, int bias_dtype, int act,
                                 const void *residual, int64_t ldr, void *y, int64_t ldy, void *z, int64_t ldz,
                                 int64_t M, int64_t N, int64_t K, sfb_stream stream) {
    using namespace sfb;
    const Problem p{x, codes, ldx, ldw, M, N, K, dtype};
    const int rc = check(p, "sfb_tensor_linear");
    if (rc) return rc;
    if (bits < 4 || bits > 8) return set_error(SFB_EINVAL, "sfb_tensor_linear: width %d is not in 4..8", bits);
    if (ldx < K || ldw < K || ldy < N || (residual && ldr < N) || (z && ldz < N))
        return set_error(SFB_EINVAL, "sfb_tensor_linear: a row stride is shorter than its row");
    if (bias && bias_dtype != SFB_F32 && bias_dtype != SFB_BF16 && bias_dtype != SFB_F16)
        return set_error(SFB_EINVAL, "sfb_tensor_linear: bias type %d", bias_dtype);
    if (M == 0 || N == 0) return SFB_OK;
    if (!scale || !y) return set_error(SFB_EINVAL, "sfb_tensor_linear: null pointer");
    Epilogue e{};
    e.scale = scale;
    e.bias = bias;
    e.residual = residual;
    e.z = static_cast<__half *>(z);
    e.y = y;
    e.unit = 1.0f / (float)(1 << (bits - 1));
    e.bias_dtype = bias_dtype;
    e.y_dtype = dtype;
    e.ldr = ldr;
    e.ldz = ldz;
    e.ldy = ldy;
    e.vec = aligned16(y, ldy, 2) && aligned16(residual, ldr, 2) && aligned16(z, ldz, 2);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    return with_activation(act, [&](auto a) { return launch_typed<false, false, decltype(a)::value>(p, e, st); });
}

extern "C" int sfb_tensor_grad_x(int dtype, const void *dzs, int64_t ldd, const void *codes, int64_t ldw,
                                 const float *top, int bits, void *dx, int64_t ldy, int64_t M, int64_t N, int64_t K,
                                 sfb_stream stream) {
    using namespace sfb;
    if (N < 1) return set_error(SFB_EINVAL, "sfb_tensor_grad_x: no channels");
    const Problem p{dzs, codes, ldd, ldw, M, K, N, dtype};
    const int rc = check(p, "sfb_tensor_grad_x");
    if (rc) return rc;
    if (bits < 4 || bits > 8) return set_error(SFB_EINVAL, "sfb_tensor_grad_x: width %d is not in 4..8", bits);
    if (ldd < N || ldw < K || ldy < K) return set_error(SFB_EINVAL, "sfb_tensor_grad_x: a row stride is shorter than its row");
    if (M == 0 || K == 0) return SFB_OK;
    if (!dx) return set_error(SFB_EINVAL, "sfb_tensor_grad_x: null pointer");
    Epilogue e{};
    e.alpha = top;
    e.y = dx;
    e.unit = top ? 1.0f / (float)(1 << (bits - 1)) : 1.0f;
    e.y_dtype = dtype;
    e.ldy = ldy;
    e.vec = aligned16(dx, ldy, 2);
    return launch_typed<false, true, SFB_ACT_NONE>(p, e, static_cast<cudaStream_t>(stream));
}

extern "C" int sfb_tensor_grad_w(int dtype, const void *dz, int64_t ldd, const void *x, int64_t ldx, void *dw,
                                 int dw_dtype, int64_t ldy, int64_t M, int64_t N, int64_t K, sfb_stream stream) {
    using namespace sfb;
    if (M < 1) return set_error(SFB_EINVAL, "sfb_tensor_grad_w: no rows");
    const Problem p{dz, x, ldd, ldx, N, K, M, dtype};
    const int rc = check(p, "sfb_tensor_grad_w");
    if (rc) return rc;
    if (dw_dtype != SFB_F32 && dw_dtype != SFB_BF16 && dw_dtype != SFB_F16)
        return set_error(SFB_EINVAL, "sfb_tensor_grad_w: weight type %d", dw_dtype);
    if (ldd < N || ldx < K || ldy < K) return set_error(SFB_EINVAL, "sfb_tensor_grad_w: a row stride is shorter than its row");
    if (N == 0 || K == 0) return SFB_OK;
    if (!dw) return set_error(SFB_EINVAL, "sfb_tensor_grad_w: null pointer");
    Epilogue e{};
    e.y = dw;
    e.unit = 1.0f;
    e.y_dtype = dw_dtype;
    e.ldy = ldy;
    e.vec = aligned16(dw, ldy, dw_dtype == SFB_F32 ? 4 : 2);
    return launch_typed<true, true, SFB_ACT_NONE>(p, e, static_cast<cudaStream_t>(stream));
}

extern "C" int sfb_tensor_failures(int64_t *count) {
    using namespace sfb;
    unsigned long long n = 0;
    if (!count) return set_error(SFB_EINVAL, "sfb_tensor_failures: null pointer");
    if (cudaMemcpyFromSymbol(&n, g_failures, sizeof n) != cudaSuccess) return check_launch("sfb_tensor_failures");
    *count = (int64_t)n;
    return SFB_OK;
}
