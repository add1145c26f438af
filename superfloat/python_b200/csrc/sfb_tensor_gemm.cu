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
// A tile's rows (TMEM lanes) run along the result's contiguous index, its columns
// along the other: operand A is the codes (forward), the codes again (x grad) or x
// (w grad).  A lane then has one channel, with its scale and bias in registers.
// (With a row of the result to a lane they came from shared memory, 16 wide loads
// a lane for 32 columns, and a tile's epilogue took 7500 cycles where K = 768 gives
// its products 6100.)  A store of two bytes a lane costs the memory pipe as much as
// one of 16 (about 8 cycles), so 32 x 32 values are packed and turned around in
// shared memory, written a channel to a lane and read by ldmatrix with its rows
// chosen so that a lane gets 8 neighbouring channels of one column.
// A pair of SMs (a cluster of two CTAs) shares an output tile of 256 x BN: each
// holds 128 rows of A, half of B's columns and the sums of its own rows, and the
// first one's warp 1 issues the products of both (cta_group::2; the other's adds up
// the bias's gradient).  4096 x 4096 x 8192 of bf16: 181 us, the tensor pipe busy for
// 91 % of them (1520 TFLOP/s).  Products read their operands from shared memory at the
// rate at which copies write them, and that is what bounds a smaller tile: 256 x 256 of
// bf16 moves 64 KB an SM and stage of 64 against 512 cycles of products, at the 128
// bytes a cycle that it has; 128 x 128 on one SM needs 64 KB for 256 cycles (577 were
// measured).
// Warp 0 issues the TMA loads (128-byte swizzle), warps 2..9 are the epilogue, two
// to each group of 32 rows, each half of the columns, 32 at a time, the next ones'
// TMEM load and residual in flight.  Two accumulators (2 BN TMEM columns) let a
// tile's epilogue run under the next tile's products.
// An operand whose contraction index is contiguous in memory is loaded K-major
// (lines of 64), one whose row index is contiguous MN-major (64 rows wide, 64
// deep), so that no operand of the backward products is transposed beforehand.
//
// Every wait is bounded; one that runs out is counted in g_failures, the CTA's
// remaining outputs are written as NaN, and the CTA waits for its copies and
// products in flight before it frees its TMEM.
#include <cuda.h>

#include <algorithm>
#include <mutex>

#include "sfb_tensor_parts.cuh"

namespace sfb {

unsigned wait_polls();                        // the calling thread's sfb_wide_wait_limit
int wait_stall();

namespace {

constexpr int BM = 128, THREADS = 320, EPI_WARPS = 8;
constexpr unsigned kSpinLimit = 1u << 26;     // polls of one wait, some seconds
constexpr int SMEM_OPERANDS = 196608;         // of the stages: what hides a copy's 1500 cycles or so under load
constexpr int SMEM_BOXES = EPI_WARPS * 2048;  // of the epilogue
constexpr int GROUP = 4;                      // row tiles that sweep the columns together, for L2

__device__ unsigned long long g_failures;

// --- PTX -----------------------------------------------------------------------------------------------------

__device__ __forceinline__ uint32_t smem_u32(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }

__device__ __forceinline__ void mbar_init(uint32_t bar, uint32_t count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}

__device__ __forceinline__ void mbar_expect_tx(uint32_t bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
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
    asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}

__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

__device__ __forceinline__ bool mbar_try(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(bar), "r"(parity)
        : "memory");
    return ok != 0;
}

// the same without a wait: try_wait may hold the thread some microseconds
__device__ __forceinline__ bool mbar_test(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(bar), "r"(parity)
        : "memory");
    return ok != 0;
}

// false once `limit` polls have not seen the phase of this parity end
__device__ __forceinline__ bool mbar_wait(uint32_t bar, uint32_t parity, unsigned limit) {
    for (unsigned i = 0; i < limit; i++)
        if (mbar_try(bar, parity)) return true;
    return false;
}

// the same wait by all lanes of a warp, with one answer
__device__ __forceinline__ bool all_wait(uint32_t bar, uint32_t parity, unsigned limit) {
    return __all_sync(0xffffffffu, mbar_wait(bar, parity, limit));
}

// an operand's box into this CTA's shared memory; the barrier is the pair's first CTA's
__device__ __forceinline__ void tma_load_operand(uint32_t dst, const CUtensorMap *map, int c0, int c1, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, "
        "{%2, %3}], [%4];" ::"r"(dst),
        "l"(map), "r"(c0), "r"(c1), "r"(bar)
        : "memory");
}

// 128 rows of two operands, 16 of the one and 16 of the other in turn: coordinates k and the first group of 16
__device__ __forceinline__ void tma_load_gated(uint32_t dst, const CUtensorMap *map, int c0, int group, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.4d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, "
        "{%2, %3, %3, %4}], [%5];" ::"r"(dst),
        "l"(map), "r"(c0), "r"(0), "r"(group), "r"(bar)
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

// kind::f16: float32 accumulator, both operands of type T, M = 256, N = BN
template <typename T, bool A_MN, bool B_MN, int BN>
__host__ __device__ constexpr uint32_t instruction() {
    return (1u << 4) | (Kind<T>::id << 7) | (Kind<T>::id << 10) | ((uint32_t)A_MN << 15) | ((uint32_t)B_MN << 16) |
           ((uint32_t)(BN >> 3) << 17) | ((uint32_t)(2 * BM >> 4) << 24);
}

__device__ __forceinline__ void mma(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc,
                                    uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(tmem_d),
        "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
        : "memory");
}

// arrives on this CTA's barrier once the products issued so far are done
__device__ __forceinline__ void mma_commit(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}

// on that barrier of both CTAs of the pair
__device__ __forceinline__ void mma_commit_both(uint32_t bar) {
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar),
        "h"((uint16_t)3)
        : "memory");
}

// 32 columns of this lane's row: in flight until tmem_landed
__device__ __forceinline__ void tmem_load(uint32_t taddr, uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,"
        "%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
          "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
          "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr));
}

// waits for the loads; the registers pass through, so that nothing reads them before
__device__ __forceinline__ void tmem_landed(uint32_t (&r)[32]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                   "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]),
                   "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]),
                   "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]),
                   "+r"(r[30]), "+r"(r[31])::"memory");
}

// --- the epilogue --------------------------------------------------------------------------------------------

struct Epilogue {
    const float *scale;          // per row of the tile, a channel (forward), or null
    const void *bias;            // likewise
    const void *residual;        // of the operands' type, or null
    const float *alpha;          // one factor for all, in device memory, or null
    __half *z;                   // the pre-activation for the backward pass, or null
    void *y;
    float unit;                  // 2^-(bits-1) where a scale or alpha stands for codes, else 1
    int bias_dtype, y_dtype;
    int64_t ldr, ldz, ldy;
    // of a gated product: the up half's scales, bias and columns of z (float32), Np after the gate's
    const void *bias2;
    int bias2_dtype;
    int64_t half;
    float *zf;
    Sums sums;                   // the bias's gradient, for the warp that has nothing to issue in the second CTA
    bool vec;                    // y (of 16 bits), z and r start on 16 bytes, and so do their rows
};

template <typename E> __device__ __forceinline__ void unpack2(uint32_t w, float &a, float &b);
template <> __device__ __forceinline__ void unpack2<__nv_bfloat16>(uint32_t w, float &a, float &b) {
    a = __uint_as_float(w << 16);
    b = __uint_as_float(w & 0xFFFF0000u);
}
template <> __device__ __forceinline__ void unpack2<__half>(uint32_t w, float &a, float &b) {
    const float2 f = __half22float2(reinterpret_cast<__half2 &>(w));
    a = f.x;
    b = f.y;
}

// two values in 16 bits each
template <typename E> __device__ __forceinline__ uint32_t pack2(float a, float b);
template <> __device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b) {
    __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return reinterpret_cast<uint32_t &>(h);
}
template <> __device__ __forceinline__ uint32_t pack2<__half>(float a, float b) {
    __half2 h = __floats2half2_rn(a, b);
    return reinterpret_cast<uint32_t &>(h);
}

// A box: 32 channels (rows of 64 bytes) by 32 columns of 16 bits.  A row's four
// pieces of 16 bytes change places so that neither 8 neighbouring rows (a channel
// to a lane) nor the rows 2 i, 2 i + 1 and those 8, 16 and 24 on (ldmatrix below)
// meet in a bank.
__device__ __forceinline__ uint32_t box_at(int row, int piece) {
    return row * 64 + (((piece ^ (row >> 1) ^ (row >> 3)) & 3) << 4);
}

__device__ __forceinline__ void box_put(uint32_t box, int row, const uint32_t (&w)[16]) {
#pragma unroll
    for (int i = 0; i < 4; i++)
        asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(box + box_at(row, i)), "r"(w[4 * i]),
                     "r"(w[4 * i + 1]), "r"(w[4 * i + 2]), "r"(w[4 * i + 3])
                     : "memory");
}

__device__ __forceinline__ void box_get(uint32_t box, int row, uint32_t (&w)[16]) {
#pragma unroll
    for (int i = 0; i < 4; i++)
        asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                     : "=r"(w[4 * i]), "=r"(w[4 * i + 1]), "=r"(w[4 * i + 2]), "=r"(w[4 * i + 3])
                     : "r"(box + box_at(row, i))
                     : "memory");
}

// Columns 8 p .. 8 p + 7 turned around: lane l has channels 8 (l mod 4) .. + 7 of
// column 8 p + l / 4.  Matrix i's line q is the channel 8 (q / 2) + 2 i + q mod 2,
// of which a lane gets lines 2 (l mod 4) and one on.
__device__ __forceinline__ uint32_t turn_at(uint32_t box, int p, int lane) {
    const int i = lane >> 3, q = lane & 7;
    return box + box_at(8 * (q >> 1) + 2 * i + (q & 1), p);
}

__device__ __forceinline__ uint4 box_turn(uint32_t box, int p, int lane) {
    uint4 o;
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(o.x), "=r"(o.y), "=r"(o.z), "=r"(o.w)
                 : "r"(turn_at(box, p, lane))
                 : "memory");
    return o;
}

__device__ __forceinline__ void box_turn_in(uint32_t box, int p, int lane, uint4 o) {
    asm volatile("stmatrix.sync.aligned.m8n8.x4.trans.shared.b16 [%0], {%1, %2, %3, %4};" ::"r"(turn_at(box, p, lane)),
                 "r"(o.x), "r"(o.y), "r"(o.z), "r"(o.w)
                 : "memory");
}

// 8 channels of a column, those past `left` not the matrix's
__device__ __forceinline__ void store8(uint16_t *to, uint4 o, int left) {
    if (left >= 8) {
        *reinterpret_cast<uint4 *>(to) = o;
    } else {
        const uint32_t w[4] = {o.x, o.y, o.z, o.w};
#pragma unroll
        for (int j = 0; j < 8; j++)
            if (j < left) to[j] = (uint16_t)(w[j / 2] >> (16 * (j & 1)));
    }
}

__device__ __forceinline__ uint4 load8(const uint16_t *from, int left) {
    if (left >= 8) return __ldg(reinterpret_cast<const uint4 *>(from));
    uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
    for (int j = 0; j < 8; j++)
        if (j < left) w[j / 2] |= (uint32_t)from[j] << (16 * (j & 1));
    return make_uint4(w[0], w[1], w[2], w[3]);
}

// A box of 16-bit values to memory.  `to` is the warp's first channel in the box's
// first column; `cols` and `chans` are what the matrix has from there on.
__device__ __forceinline__ void box_out(uint32_t box, const uint32_t (&w)[16], uint16_t *to, int64_t ld, int cols,
                                        int chans, bool vec, int lane) {
    if (vec) {
        box_put(box, lane, w);
        __syncwarp();
        const int part = 8 * (lane & 3), c = lane >> 2;
#pragma unroll
        for (int p = 0; p < 4; p++) {
            const uint4 o = box_turn(box, p, lane);
            if (8 * p + c < cols) store8(to + (8 * p + c) * ld + part, o, chans - part);
        }
        __syncwarp();
    } else if (lane < chans) {
        to += lane;
#pragma unroll
        for (int j = 0; j < 32; j++, to += ld)
            if (j < cols) *to = (uint16_t)(w[j / 2] >> (16 * (j & 1)));
    }
}

// A gated box: 16 channels by 32 columns.  A lane has the channel lane mod 16 in the 16 columns 16 (lane / 16) ..; turned
// around, lane l has the channels 8 (l mod 2) .. + 7 of column 8 (2 h + l / 2 mod 2) + l / 4, for h of 0 and 1.
__device__ __forceinline__ uint32_t gated_at(int row, int piece) {
    return row * 64 + (((piece ^ (row >> 1) ^ (row >> 3 << 1)) & 3) << 4);
}

__device__ __forceinline__ void gated_out(uint32_t box, const uint32_t (&w)[8], uint16_t *to, int64_t ld, int cols, int chans,
                                          bool vec, int lane) {
    const int row = lane & 15, side = lane >> 4;
    if (vec) {
#pragma unroll
        for (int i = 0; i < 2; i++)
            asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(box + gated_at(row, 2 * side + i)), "r"(w[4 * i]),
                         "r"(w[4 * i + 1]), "r"(w[4 * i + 2]), "r"(w[4 * i + 3])
                         : "memory");
        __syncwarp();
        const int i = lane >> 3, q = lane & 7, part = 8 * (lane & 1);
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const uint32_t from = box + gated_at(8 * (q >> 1 & 1) + 2 * i + (q & 1), 2 * h + (q >> 2));
            uint4 o;
            asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                         : "=r"(o.x), "=r"(o.y), "=r"(o.z), "=r"(o.w)
                         : "r"(from)
                         : "memory");
            const int c = 8 * (2 * h + (lane >> 1 & 1)) + (lane >> 2);
            if (c < cols) store8(to + c * ld + part, o, chans - part);
        }
        __syncwarp();
    } else if (row < chans) {
        to += row;
#pragma unroll
        for (int j = 0; j < 16; j++)
            if (16 * side + j < cols) to[(16 * side + j) * ld] = (uint16_t)(w[j / 2] >> (16 * (j & 1)));
    }
}

struct Tiles {
    int rt, ct, total;               // of rows, of columns
};

__device__ __forceinline__ void tile_of(const Tiles &t, int i, int &tr, int &tc) {
    const int gsize = GROUP * t.ct, g = i / gsize, r0 = g * GROUP;
    const int gr = min(GROUP, t.rt - r0), r = i - g * gsize;
    tr = r0 + r % gr;
    tc = r / gr;
}

template <int BN>
struct Shape {
    static constexpr int BNL = BN / 2;                               // columns of B that a CTA loads
    static constexpr int BK = BN == 256 ? 64 : 128;                  // of the contraction, a stage
    static constexpr int A = BM * BK * 2, B = BNL * BK * 2, STAGE = A + B, STAGES = SMEM_OPERANDS / STAGE;
    static constexpr int COLS = 2 * BN;                              // TMEM columns
    static constexpr int SMEM = STAGES * STAGE + SMEM_BOXES + 512 + 1024;
};

// GATED: operand A is two of N rows, 16 channels of the one and 16 of the other in turn, so that a warp's 32 TMEM lanes hold
// both products of 16 channels and two exchanges of a register join them
template <typename T, bool A_MN, bool B_MN, int BN, int ACT, bool GATED>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(THREADS, 1)
gemm_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB, int nkb, int64_t R,
            int64_t C, Tiles tiles, const __grid_constant__ Epilogue e, unsigned spin, int stall) {
    using S = Shape<BN>;
    constexpr int STAGES = S::STAGES, BK = S::BK;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    uint64_t *bars = reinterpret_cast<uint64_t *>(smem + STAGES * S::STAGE + SMEM_BOXES);
    // full [0, S), empty [S, 2 S), accumulator full 2 S + {0, 1}, accumulator empty 2 S + {2, 3}, all done 2 S + 4,
    // and one that nothing arrives on (the tests' stall).  The first CTA's full, accumulator empty and done barriers
    // serve both; each has its own empty and accumulator full ones.
    auto full = [&](int s) { return smem_u32(&bars[s]); };
    auto empty = [&](int s) { return smem_u32(&bars[STAGES + s]); };
    auto acc_full = [&](int a) { return smem_u32(&bars[2 * STAGES + a]); };
    auto acc_empty = [&](int a) { return smem_u32(&bars[2 * STAGES + 2 + a]); };
    const uint32_t done = smem_u32(&bars[2 * STAGES + 4]), never = smem_u32(&bars[2 * STAGES + 5]);
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(bars + 2 * STAGES + 6);
    __shared__ int s_fail;
    volatile int *failed = &s_fail;

    const int warp = __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
    const int rank = (int)(blockIdx.x & 1), first = blockIdx.x / 2, step = gridDim.x / 2;
    if (threadIdx.x == 0) {
        s_fail = 0;
        for (int s = 0; s < STAGES; s++) {
            mbar_init(full(s), 1);
            mbar_init(empty(s), 1);
        }
        for (int a = 0; a < 2; a++) {
            mbar_init(acc_full(a), 1);
            mbar_init(acc_empty(a), 2 * EPI_WARPS);
        }
        mbar_init(done, 1);
        mbar_init(never, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 0) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                     "n"(S::COLS)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    cluster_sync();                                    // the barriers of both are set
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;

    int issued = 0;
    if (warp == 0) {
        for (int t = first; t < tiles.total; t += step) {
            int tr, tc;
            tile_of(tiles, t, tr, tc);
            const int r0 = (tr * 2 + rank) * BM, c0 = tc * BN + rank * S::BNL;
            for (int kb = 0; kb < nkb; kb++, issued++) {
                const int s = issued % STAGES, round = issued / STAGES;
                if (round > 0 && !all_wait(empty(s), (round - 1) & 1, spin)) {
                    *failed = 1;
                    break;
                }
                const uint32_t a = smem_u32(smem + s * S::STAGE), b = a + S::A, bar = of_leader(full(s));
                if (elected()) {
                    if (rank == 0) mbar_expect_tx(full(s), 2 * S::STAGE);
#pragma unroll
                    for (int h = 0; h < BK / 64; h++) {              // 64 of the contraction at a time
                        const int k = kb * BK + h * 64;
                        const uint32_t ah = a + h * (BM * 128), bh = b + h * (S::BNL * 128);
                        if constexpr (A_MN) {
#pragma unroll
                            for (int i = 0; i < BM / 64; i++) tma_load_operand(ah + i * 8192, &tmA, r0 + i * 64, k, bar);
                        } else if constexpr (GATED) {
                            tma_load_gated(ah, &tmA, k, r0 / 32, bar);
                        } else {
                            tma_load_operand(ah, &tmA, k, r0, bar);
                        }
                        if constexpr (B_MN) {
#pragma unroll
                            for (int i = 0; i < S::BNL / 64; i++)
                                tma_load_operand(bh + i * 8192, &tmB, c0 + i * 64, k, bar);
                        } else {
                            tma_load_operand(bh, &tmB, k, c0, bar);
                        }
                    }
                }
                __syncwarp();
            }
            if (__any_sync(0xffffffffu, *failed)) break;
        }
        // The last stages' commits still have to arrive here, the second CTA's from the first one's products: neither
        // CTA may end before its own have come.  They do under the last tile's epilogue.
        for (int it = issued > STAGES ? issued - STAGES : 0; it < issued; it++)
            if (__any_sync(0xffffffffu, *failed) || !all_wait(empty(it % STAGES), (it / STAGES) & 1, spin)) {
                *failed = 1;
                break;
            }
    } else if (warp == 1 && rank == 0) {
        constexpr uint32_t id = instruction<T, A_MN, B_MN, BN>();
        bool ok = !(stall && !all_wait(never, 0, spin));
        // The next stage's barrier is tested under this one's products, and nothing else is asked in the loop: a stage
        // took 480 cycles to issue (115 the wait on a barrier that was ready, 150 a look at s_fail and a fence, 190
        // the products and their commit), as long as 256 columns' products take and twice as long as 128's.
        int s = 0, parity = 0, i = 0;
        bool ready = mbar_test(full(0), 0);
        for (int t = first; t < tiles.total && ok; t += step, i++) {
            const int acc = i & 1;
            if (i >= 2 && !all_wait(acc_empty(acc), ((i >> 1) - 1) & 1, spin)) {
                ok = false;
                break;
            }
            tc_fence_after();
            for (int kb = 0; kb < nkb; kb++) {
                if (!__all_sync(0xffffffffu, ready) && !all_wait(full(s), parity, spin)) {
                    ok = false;
                    break;
                }
                const uint32_t a = smem_u32(smem + s * S::STAGE), b = a + S::A, free = empty(s);
                if (++s == STAGES) s = 0, parity ^= 1;
                ready = mbar_test(full(s), parity);
                if (elected()) {
#pragma unroll
                    for (int kk = 0; kk < BK / 16; kk++) {
                        const int h = kk / 4, q = kk % 4;
                        const uint64_t da = smem_desc<A_MN>(a + h * (BM * 128)), db = smem_desc<B_MN>(b + h * (S::BNL * 128));
                        mma(tmem + acc * BN, da + q * (A_MN ? 128 : 2), db + q * (B_MN ? 128 : 2), id,
                            kb == 0 && kk == 0 ? 0u : 1u);
                    }
                    mma_commit_both(free);
                }
                __syncwarp();
            }
            if (ok && elected()) mma_commit_both(acc_full(acc));
            __syncwarp();
        }
        if (!ok) *failed = 1;
        if (elected()) {
            if (!ok) {
                // release this CTA's epilogue, which sees that the CTA failed; the other CTA's waits run out by themselves
                mma_commit(acc_full(0));
                mma_commit(acc_full(1));
            }
            mma_commit(done);
        }
        __syncwarp();
        if (ok && !all_wait(done, 0, spin)) *failed = 1;
    } else if (warp == 1) {
        if (e.sums.parts)
            for (int64_t n = (int64_t)first * 32 + lane; n < e.sums.N; n += (int64_t)step * 32)
                store_sum(e.sums, n, column_sum(e.sums, n));
    } else if (warp >= 2) {
        const int half = (warp - 2) >> 2, quad = warp & 3;   // a warp reaches the TMEM lanes 32 (warp % 4) ..
        const uint32_t lanes = (uint32_t)(32 * quad) << 16, box = smem_u32(smem + STAGES * S::STAGE) + (warp - 2) * 2048;
        const float alpha = e.alpha ? *e.alpha * e.unit : e.unit;
        const uint16_t *res = static_cast<const uint16_t *>(e.residual);
        uint16_t *z = reinterpret_cast<uint16_t *>(e.z);
        int i = 0;
        for (int t = first; t < tiles.total; t += step, i++) {
            int tr, tc;
            tile_of(tiles, t, tr, tc);
            const int acc = i & 1;
            const int64_t rows = (int64_t)(tr * 2 + rank) * BM + quad * 32, c0 = (int64_t)tc * BN + half * (BN / 2);
            // the warp's first channel, how many it has (GATED: R counts channels, two rows of the tile each)
            const int64_t r0 = GATED ? rows / 2 : rows;
            const int chans = (int)min((int64_t)(GATED ? 16 : 32), R - r0), cols = (int)min((int64_t)(BN / 2), C - c0);
            const int count = chans > 0 && cols > 0 ? (cols + 31) / 32 : 0;
            const int chan = GATED ? lane & 15 : lane;
            const bool mine = chan < chans, up = GATED && lane >= 16;
            const float scale = mine && e.scale ? e.scale[r0 + chan + (up ? e.half : 0)] * alpha : alpha;
            const void *const offset = up ? e.bias2 : e.bias;
            const float bias = mine && offset ? load_as(offset, r0 + chan, up ? e.bias2_dtype : e.bias_dtype) : 0.0f;
            // the residual of box b: as box_turn has it or, unaligned, the lane's channel in 32 columns
            uint32_t rnext[16];
            auto fetch = [&](int b) {
                const int left = cols - 32 * b;
                const uint16_t *from = res + (c0 + 32 * b) * e.ldr + r0;
                if (e.vec) {
                    const int part = 8 * (lane & 3), c = lane >> 2;
#pragma unroll
                    for (int p = 0; p < 4; p++) {
                        uint4 q = make_uint4(0, 0, 0, 0);
                        if (8 * p + c < left) q = load8(from + (8 * p + c) * e.ldr + part, chans - part);
                        rnext[4 * p] = q.x, rnext[4 * p + 1] = q.y, rnext[4 * p + 2] = q.z, rnext[4 * p + 3] = q.w;
                    }
                } else {
                    from += lane;
#pragma unroll
                    for (int j = 0; j < 32; j += 2, from += 2 * e.ldr) {
                        const uint32_t lo = mine && j < left ? __ldg(from) : 0;
                        const uint32_t hi = mine && j + 1 < left ? __ldg(from + e.ldr) : 0;
                        rnext[j / 2] = lo | hi << 16;
                    }
                }
            };
            if (res && count) fetch(0);
            // one lane polls: 256 of them would crowd the memory pipe
            int fine = 0;
            if (lane == 0) fine = !*failed && mbar_wait(acc_full(acc), (i >> 1) & 1, spin) && !*failed;
            fine = __shfl_sync(0xffffffffu, fine, 0);    // TMEM loads are the whole warp's
            if (!fine) *failed = 1;
            tc_fence_after();
            const uint32_t from = tmem + lanes + acc * BN + half * (BN / 2);
            uint32_t next[32];
            if (fine && count) tmem_load(from, next);
            for (int b = 0; b < count; b++) {
                float v[32];
                uint32_t w[16], rr[16];
                if (fine) tmem_landed(next);
#pragma unroll
                for (int j = 0; j < 32; j++) v[j] = fine ? __uint_as_float(next[j]) : __int_as_float(0x7FC00000);
#pragma unroll
                for (int j = 0; j < 16; j++) rr[j] = rnext[j];
                const int left = cols - 32 * b;
                const int64_t c = c0 + 32 * b;
                if (b + 1 < count) {
                    if (fine) tmem_load(from + 32 * (b + 1), next);
                    if (res) fetch(b + 1);
                } else {
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive_cluster(of_leader(acc_empty(acc)));
                }
#pragma unroll
                for (int j = 0; j < 32; j++) v[j] = fmaf(v[j], scale, bias);
                if constexpr (GATED) {
                    if (e.zf && mine) {
                        float *to = e.zf + c * e.ldz + r0 + chan + (up ? e.half : 0);
#pragma unroll
                        for (int j = 0; j < 32; j++, to += e.ldz)
                            if (j < left) *to = v[j];
                    }
                    // a lane of the gate's joins the first 16 columns, one of the other's the last
                    float h[16];
#pragma unroll
                    for (int j = 0; j < 16; j++) {
                        const float got = __shfl_xor_sync(0xffffffffu, up ? v[j] : v[16 + j], 16);
                        h[j] = activate<ACT>(up ? got : v[j]) * (up ? v[16 + j] : got);
                    }
                    uint32_t q[8];
#pragma unroll
                    for (int j = 0; j < 8; j++) q[j] = pack2<T>(h[2 * j], h[2 * j + 1]);
                    gated_out(box, q, static_cast<uint16_t *>(e.y) + c * e.ldy + r0, e.ldy, left, chans, e.vec, lane);
                    continue;
                }
                if (z) {
#pragma unroll
                    for (int j = 0; j < 16; j++) w[j] = kept2<ACT>(v[2 * j], v[2 * j + 1]);
                    box_out(box, w, z + c * e.ldz + r0, e.ldz, left, chans, e.vec, lane);
                }
#pragma unroll
                for (int j = 0; j < 32; j++) v[j] = activate<ACT>(v[j]);
                if (res) {
                    if (e.vec) {
#pragma unroll
                        for (int p = 0; p < 4; p++)
                            box_turn_in(box, p, lane, make_uint4(rr[4 * p], rr[4 * p + 1], rr[4 * p + 2], rr[4 * p + 3]));
                        __syncwarp();
                        box_get(box, lane, rr);
                        __syncwarp();
                    }
#pragma unroll
                    for (int j = 0; j < 16; j++) {
                        float lo, hi;
                        unpack2<T>(rr[j], lo, hi);
                        v[2 * j] += lo;
                        v[2 * j + 1] += hi;
                    }
                }
                if (e.y_dtype == SFB_F32) {
                    float *y = static_cast<float *>(e.y) + c * e.ldy + r0 + lane;
                    if (mine)
#pragma unroll
                        for (int j = 0; j < 32; j++, y += e.ldy)
                            if (j < left) *y = v[j];
                } else {
                    if (e.y_dtype == SFB_BF16) {
#pragma unroll
                        for (int j = 0; j < 16; j++) w[j] = pack2<__nv_bfloat16>(v[2 * j], v[2 * j + 1]);
                    } else {
#pragma unroll
                        for (int j = 0; j < 16; j++) w[j] = pack2<__half>(v[2 * j], v[2 * j + 1]);
                    }
                    box_out(box, w, static_cast<uint16_t *>(e.y) + c * e.ldy + r0, e.ldy, left, chans, e.vec, lane);
                }
            }
            if (count == 0) {
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive_cluster(of_leader(acc_empty(acc)));
            }
        }
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if (s_fail && threadIdx.x == 0) {
        atomicAdd(&g_failures, 1ull);
        // the copies land before their shared memory is released (both CTAs' complete on the first one's barriers; the
        // other waits for it below), the products (the commit on `done` follows them) end before TMEM is freed:
        // full-length waits, whatever `spin` was
        if (rank == 0) {
            for (int it = issued > STAGES ? issued - STAGES : 0; it < issued; it++)
                (void)mbar_wait(full(it % STAGES), (it / STAGES) & 1, kSpinLimit);
            (void)mbar_wait(done, 0, kSpinLimit);
        }
    }
    tc_fence_before();
    __syncthreads();
    cluster_sync();                                    // neither leaves while the other's copies or arrivals may come
    tc_fence_after();
    if (warp == 0)
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(S::COLS) : "memory");
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

// rows of A, columns (rows of B in memory where it is K-major), contraction
struct Problem {
    const void *A, *B;
    int64_t lda, ldb, R, C, K;
    int dtype;
};

// an operand, `rows` lines of `cols` elements, ld apart, read in boxes of 64 columns
int operand_map(CUtensorMap *map, const void *base, int dtype, int64_t rows, int64_t cols, int64_t ld, int box_rows) {
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

// whether a matrix of 16-bit elements and its rows start on 16 bytes
bool rows_on16(const void *p, int64_t ld) {
    return p == nullptr || (reinterpret_cast<uintptr_t>(p) % 16 == 0 && ld % 8 == 0);
}

// The two operands of a gated product, N rows each (Np apart, a multiple of 16), as one of four dimensions: a box has 64 of
// the contraction, 16 rows, both operands, 4 groups of 16 rows.  The rows' order in shared memory is that of the box.
int gated_map(CUtensorMap *map, const void *base, int dtype, int64_t Np, int64_t cols, int64_t ld) {
    EncodeTiled enc = encoder();
    if (!enc) return set_error(SFB_ECUDA, "sf gated product: cuTensorMapEncodeTiled is unavailable");
    const cuuint64_t dims[4] = {(cuuint64_t)cols, 16, 2, (cuuint64_t)(Np / 16)};
    const cuuint64_t strides[3] = {(cuuint64_t)ld * 2, (cuuint64_t)(Np * ld) * 2, (cuuint64_t)ld * 32};
    const cuuint32_t box[4] = {64, 16, 2, 4};
    const cuuint32_t estr[4] = {1, 1, 1, 1};
    const CUresult r = enc(map, dtype == SFB_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16,
                           4, const_cast<void *>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                           CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                           CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return set_error(SFB_ECUDA, "sf gated product: tensor map encoding failed (%d)", (int)r);
    return SFB_OK;
}

template <typename T, bool A_MN, bool B_MN, int BN, int ACT, bool GATED>
int launch(const Problem &p, Epilogue e, cudaStream_t st) {
    using S = Shape<BN>;
    auto *kernel = gemm_kernel<T, A_MN, B_MN, BN, ACT, GATED>;
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
    e.vec = (e.y_dtype == SFB_F32 || rows_on16(e.y, e.ldy)) && rows_on16(e.z, e.ldz) && rows_on16(e.residual, e.ldr);
    CUtensorMap tmA, tmB;
    int rc = GATED  ? gated_map(&tmA, p.A, p.dtype, e.half, p.K, p.lda)
             : A_MN ? operand_map(&tmA, p.A, p.dtype, p.K, p.R, p.lda, 64)
                    : operand_map(&tmA, p.A, p.dtype, p.R, p.K, p.lda, BM);
    if (!rc)
        rc = B_MN ? operand_map(&tmB, p.B, p.dtype, p.K, p.C, p.ldb, 64)
                  : operand_map(&tmB, p.B, p.dtype, p.C, p.K, p.ldb, S::BNL);
    if (rc) return rc;
    Tiles t;
    const int64_t lines = GATED ? 2 * e.half : p.R;                    // rows of operand A
    t.rt = (int)((lines + 2 * BM - 1) / (2 * BM));
    t.ct = (int)((p.C + BN - 1) / BN);
    t.total = t.rt * t.ct;
    kernel<<<2 * std::min(t.total, sm_count() / 2), THREADS, S::SMEM, st>>>(
        tmA, tmB, (int)((p.K + S::BK - 1) / S::BK), p.R, p.C, t, e, wait_polls() ? wait_polls() : kSpinLimit,
        wait_stall());
    return check_launch("sf tensor linear");
}

// Columns of a tile.  A stage of 256 columns takes its 512 cycles of products, one
// of 128 about 390 (48 KB of shared memory's traffic against 256 cycles of products),
// so the wider tile wins unless it leaves pairs without one.  Measured, 256 and 128
// columns: 4096 x 4096 x 8192 forward 199 and 246 us, 8192 x 4096 x 4096 w grad 254 and
// 262; 4096 x 768 x 2304 w grad 25.1 and 16.0, 128 x 4096 x 4096 x grad 24.0 and 14.7.
// With 768 deep, where a tile's epilogue is as long as its products, the rule still
// holds for the forward product (z kept, gelu_tanh; 4096 and 8192 rows of 2304
// channels: 23.6 and 25.3, 39.1 and 43.7) and x's gradient of 4096 x 768 (19.7 and
// 19.8), but takes the slower side for that of 8192 x 768 (30.5 and 27.1).
int columns(int64_t R, int64_t C) {
    const int64_t rt = (R + 2 * BM - 1) / (2 * BM), n = sm_count() / 2;
    const int64_t wide = (rt * ((C + 255) / 256) + n - 1) / n, narrow = (rt * ((C + 127) / 128) + n - 1) / n;
    return 512 * wide <= 390 * narrow ? 256 : 128;
}

template <bool A_MN, bool B_MN, int ACT, bool GATED = false>
int launch_typed(const Problem &p, const Epilogue &e, cudaStream_t st) {
    const bool wide = columns(GATED ? 2 * e.half : p.R, p.C) == 256;
    if (p.dtype == SFB_BF16)
        return wide ? launch<__nv_bfloat16, A_MN, B_MN, 256, ACT, GATED>(p, e, st)
                    : launch<__nv_bfloat16, A_MN, B_MN, 128, ACT, GATED>(p, e, st);
    return wide ? launch<__half, A_MN, B_MN, 256, ACT, GATED>(p, e, st) : launch<__half, A_MN, B_MN, 128, ACT, GATED>(p, e, st);
}

}  // namespace

int tensor_product(int dtype, const void *x, int64_t ldx, const void *codes, int64_t ldw, const float *scale, int bits,
                   const void *bias, int bias_dtype, int act, const void *residual, int64_t ldr, void *y, int64_t ldy,
                   void *z, int64_t ldz, int64_t M, int64_t N, int64_t K, cudaStream_t st) {
    const Problem p{codes, x, ldw, ldx, N, M, K, dtype};
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
    return with_activation(act, [&](auto a) { return launch_typed<false, false, decltype(a)::value>(p, e, st); });
}

int tensor_gated_product(int dtype, const void *x, int64_t ldx, const void *codes, int64_t ldw, const float *scale, int bits,
                         const void *bias, int bias_dtype, const void *bias2, int bias2_dtype, int act, void *y, int64_t ldy,
                         float *z, int64_t ldz, int64_t M, int64_t N, int64_t Np, int64_t K, cudaStream_t st) {
    const Problem p{codes, x, ldw, ldx, N, M, K, dtype};
    Epilogue e{};
    e.scale = scale;
    e.bias = bias;
    e.bias2 = bias2;
    e.half = Np;
    e.zf = z;
    e.y = y;
    e.unit = 1.0f / (float)(1 << (bits - 1));
    e.bias_dtype = bias_dtype;
    e.bias2_dtype = bias2_dtype;
    e.y_dtype = dtype;
    e.ldz = ldz;
    e.ldy = ldy;
    return with_activation(act, [&](auto a) { return launch_typed<false, false, decltype(a)::value, true>(p, e, st); });
}

int tensor_grad_x(int dtype, const void *dzs, int64_t ldd, const void *codes, int64_t ldw, const float *top, int bits,
                  void *dx, int64_t ldx, int64_t M, int64_t N, int64_t K, cudaStream_t st) {
    const Problem p{codes, dzs, ldw, ldd, K, M, N, dtype};
    Epilogue e{};
    e.alpha = top;
    e.y = dx;
    e.unit = top ? 1.0f / (float)(1 << (bits - 1)) : 1.0f;
    e.y_dtype = dtype;
    e.ldy = ldx;
    return launch_typed<true, false, SFB_ACT_NONE>(p, e, st);
}

int tensor_grad_w(int dtype, const void *dz, int64_t ldd, const void *x, int64_t ldx, void *dw, int dw_dtype,
                  int64_t ldw, int64_t M, int64_t N, int64_t K, const Sums &sums, cudaStream_t st) {
    const Problem p{x, dz, ldx, ldd, K, N, M, dtype};
    Epilogue e{};
    e.y = dw;
    e.unit = 1.0f;
    e.y_dtype = dw_dtype;
    e.ldy = ldw;
    e.sums = sums;
    return launch_typed<true, true, SFB_ACT_NONE>(p, e, st);
}

}  // namespace sfb

extern "C" int sfb_tensor_failures(int64_t *count) {
    using namespace sfb;
    unsigned long long n = 0;
    if (!count) return set_error(SFB_EINVAL, "sfb_tensor_failures: null pointer");
    if (cudaMemcpyFromSymbol(&n, g_failures, sizeof n) != cudaSuccess) return check_launch("sfb_tensor_failures");
    *count = (int64_t)n;
    return SFB_OK;
}
