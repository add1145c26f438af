// The forward product for few rows, straight from the packed codes.
//
//   y = act((x code^T) s[n] 2^-(bits-1) + b[n]) + r,  at most 48 rows
//
// Bound by the codes' bytes: each is read once, and turned into the activations'
// type in registers (exact: a code has at most 7 bits).  The products go to the
// warps' matrix instruction with the CODES as its 16-row operand and x as its
// 8-column one, so one row of x wastes 7 of 8 columns of a pipe that is idle
// anyway, where a tile of 128 rows on tcgen05 would need the codes in 16 bits in
// shared memory first.  The contraction index may be permuted freely as long as
// both operands agree: a lane takes 16 consecutive codes of a row with one load
// and the same 16 elements of x, and four steps of 16 use four of each.
// Codes arrive by cp.async, DEEP segments ahead, in places of shared memory that
// only the lane that asked for them reads: nothing to synchronise, and 32 KB a CTA
// in flight without a register.  (Two segments ahead in registers: 10.8 us for one
// row of 4096 x 4096; eight ahead: 14, a CTA of 155 registers a thread to an SM.)
// 48 rows is one number for where the products of 256 channels by 128 rows on tcgen05,
// with the codes expanded first, overtake it, which depends on the shape: for 48 rows
// 8192 x 4096 takes 27 us here and 38 there, 4096 x 4096 15 and 26, a head of 50257 x
// 768 46 and 41; for 64 rows 41 and 38, 22 and 26, 72 and 41.
// (32 channels a warp, to halve the loads of x, was slower: it spills.)
// A CTA of 8 warps covers 8 / ks groups of 16 channels; ks warps share a group,
// each every ks-th segment of 64, and their sums are added in a fixed order.
#include <algorithm>

#include "sfb_tensor_parts.cuh"

namespace sfb {
namespace {

constexpr int WARPS = 8, SEG = 64;

template <typename T>
__device__ __forceinline__ void mma16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                      uint32_t b1) {
    if constexpr (sizeof(T) == 2 && std::is_same<T, __half>::value)
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// 16 codes of a row from k on, those at or past K as 0: into `to` (where rows do not start on 16 bytes, shift_codes)
template <bool WHOLE>
__device__ __forceinline__ void fetch_codes(uint4 *to, const int8_t *row, int64_t k, int64_t K) {
    if constexpr (WHOLE) {
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(to)), "l"(row + k)
                     : "memory");
        return;
    }
    const int64_t left = K - k;
    const int bytes = left >= 16 ? 16 : left > 0 ? (int)left : 0;       // the rest is filled with zeros
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"((uint32_t)__cvta_generic_to_shared(to)),
                 "l"(bytes ? row + k : row), "r"(bytes)
                 : "memory");
}

// 16 elements of a row of x from k on, those at or past K as 0; rows start on 16 bytes
template <typename T>
__device__ __forceinline__ void load_x(const T *row, int64_t k, int64_t K, uint32_t (&x)[8]) {
#pragma unroll
    for (int h = 0; h < 2; h++) {
        uint4 q = make_uint4(0, 0, 0, 0);
        const int64_t at = k + 8 * h;
        if (at < K) {
            q = __ldg(reinterpret_cast<const uint4 *>(row + at));
            if (at + 8 > K) {
                uint32_t w[4] = {q.x, q.y, q.z, q.w};
                const int left = (int)(K - at);
#pragma unroll
                for (int i = 0; i < 4; i++) w[i] &= left >= 2 * i + 2 ? 0xFFFFFFFFu : left == 2 * i + 1 ? 0xFFFFu : 0u;
                q = make_uint4(w[0], w[1], w[2], w[3]);
            }
        }
        x[4 * h] = q.x, x[4 * h + 1] = q.y, x[4 * h + 2] = q.z, x[4 * h + 3] = q.w;
    }
}

struct Small {
    const void *x;
    const int8_t *codes;
    const float *scale;
    const void *bias, *residual;
    const int8_t *codes2;                      // of a gated product: the up half's
    const float *scale2;
    const void *bias2;
    int64_t ldc2;
    int bias2_dtype;
    void *y;
    int64_t ldx, ldc, ldr, ldy, N, K;
    float unit;
    int M, ks, bias_dtype;
};

constexpr int DEEP = 4;

// How K and the codes' rows lie: WHOLE, in whole segments on 16 bytes, asks nothing
// in the loop (the questions are half of its instructions); ON16, rows on 16 bytes; ANY.
enum { WHOLE, ON16, ANY };

// GATED: the 16 rows of a group are 8 channels of the gate and the same 8 of the other weight
template <typename T, int MT, int LIE, int ACT, bool GATED>
__global__ void __launch_bounds__(32 * WARPS, MT <= 2 ? 4 : MT == 4 ? 3 : 2) small_kernel(Small p) {
    __shared__ union {
        uint4 codes[DEEP][2][32 * WARPS];
        float sum[WARPS][16][8 * MT];
    } s;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int groups = WARPS / p.ks, group = warp / p.ks, part = warp % p.ks;
    constexpr int CHANS = GATED ? 8 : 16;      // channels of a group
    const int64_t n0 = ((int64_t)blockIdx.x * groups + group) * CHANS;
    // channels past the last read the last one's codes, rows past the last the last one: their sums are not stored
    const int8_t *row0 = p.codes + min(n0 + g, p.N - 1) * p.ldc, *row1 = GATED ? p.codes2 + min(n0 + g, p.N - 1) * p.ldc2 : p.codes + min(n0 + g + 8, p.N - 1) * p.ldc;
    const T *x[MT];
#pragma unroll
    for (int i = 0; i < MT; i++) x[i] = static_cast<const T *>(p.x) + (int64_t)min(i * 8 + g, p.M - 1) * p.ldx;
    float d[MT][4] = {};
    const int segs = n0 < p.N ? (int)((p.K + SEG - 1) / SEG) : 0;
    const int first = part * SEG + t * 16, step = p.ks * SEG;
    auto fetch = [&](int u, int seg, int64_t k) {
        if constexpr (LIE != ANY) {
            if (seg < segs) {
                fetch_codes<LIE == WHOLE>(&s.codes[u][0][threadIdx.x], row0, k, p.K);
                fetch_codes<LIE == WHOLE>(&s.codes[u][1][threadIdx.x], row1, k, p.K);
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
        }
    };
#pragma unroll
    for (int u = 0; u < DEEP; u++) fetch(u, part + u * p.ks, first + (int64_t)u * step);
    int u = 0;
    int64_t k = first;
#pragma unroll(LIE == ANY && MT == 1 ? 4 : 1)
    for (int seg = part; seg < segs; seg += p.ks, k += step) {
        uint32_t b[MT][8];
#pragma unroll
        for (int i = 0; i < MT; i++) {
            if constexpr (LIE == WHOLE) {
                const uint4 lo = __ldg(reinterpret_cast<const uint4 *>(x[i] + k));
                const uint4 hi = __ldg(reinterpret_cast<const uint4 *>(x[i] + k) + 1);
                b[i][0] = lo.x, b[i][1] = lo.y, b[i][2] = lo.z, b[i][3] = lo.w;
                b[i][4] = hi.x, b[i][5] = hi.y, b[i][6] = hi.z, b[i][7] = hi.w;
            } else {
                load_x(x[i], k, p.K, b[i]);
            }
        }
        uint4 c0, c1;
        if constexpr (LIE != ANY) {
            asm volatile("cp.async.wait_group %0;" ::"n"(DEEP - 1) : "memory");
            c0 = s.codes[u][0][threadIdx.x];
            c1 = s.codes[u][1][threadIdx.x];
            fetch(u, seg + DEEP * p.ks, k + (int64_t)DEEP * step);
            u = (u + 1) % DEEP;
        } else {
            c0 = shift_codes(row0, k, p.K);
            c1 = shift_codes(row1, k, p.K);
        }
        const uint32_t w0[4] = {c0.x, c0.y, c0.z, c0.w}, w1[4] = {c1.x, c1.y, c1.z, c1.w};
#pragma unroll
        for (int j = 0; j < 4; j++) {
            uint32_t a0, a1, a2, a3;
            widen<T>(w0[j], a0, a2);
            widen<T>(w1[j], a1, a3);
#pragma unroll
            for (int i = 0; i < MT; i++) mma16<T>(d[i], a0, a1, a2, a3, b[i][2 * j], b[i][2 * j + 1]);
        }
    }
    if constexpr (LIE != ANY) asm volatile("cp.async.wait_group 0;" ::: "memory");
    __syncthreads();                                   // the codes' places become the sums'
#pragma unroll
    for (int i = 0; i < MT; i++) {
        s.sum[warp][g][i * 8 + 2 * t] = d[i][0];
        s.sum[warp][g][i * 8 + 2 * t + 1] = d[i][1];
        s.sum[warp][g + 8][i * 8 + 2 * t] = d[i][2];
        s.sum[warp][g + 8][i * 8 + 2 * t + 1] = d[i][3];
    }
    __syncthreads();
    for (int o = threadIdx.x; o < groups * CHANS * p.M; o += 32 * WARPS) {
        const int c = o % (groups * CHANS), m = o / (groups * CHANS);
        const int64_t n = (int64_t)blockIdx.x * groups * CHANS + c;
        if (n >= p.N) continue;
        float v = 0.0f;
        for (int i = 0; i < p.ks; i++) v += s.sum[(c / CHANS) * p.ks + i][c % CHANS][m];
        v = fmaf(v, p.scale[n] * p.unit, p.bias ? load_as(p.bias, n, p.bias_dtype) : 0.0f);
        v = activate<ACT>(v);
        if constexpr (GATED) {
            float u = 0.0f;
            for (int i = 0; i < p.ks; i++) u += s.sum[(c / CHANS) * p.ks + i][c % CHANS + 8][m];
            v *= fmaf(u, p.scale2[n] * p.unit, p.bias2 ? load_as(p.bias2, n, p.bias2_dtype) : 0.0f);
        }
        if (p.residual) v += to_f(static_cast<const T *>(p.residual)[m * p.ldr + n]);
        static_cast<T *>(p.y)[m * p.ldy + n] = from_f<T>(v);
    }
}

template <typename T, int MT, int LIE, bool GATED>
int launch(const Small &p, int act, cudaStream_t st) {
    const int64_t groups = GATED ? (p.N + 7) / 8 : (p.N + 15) / 16;
    const int per = WARPS / p.ks;
    const unsigned grid = (unsigned)((groups + per - 1) / per);
    return with_activation(act, [&](auto a) {
        small_kernel<T, MT, LIE, decltype(a)::value, GATED><<<grid, 32 * WARPS, 0, st>>>(p);
        return check_launch("sf tensor linear (few rows)");
    });
}

bool on16(const int8_t *p, int64_t ld) { return p == nullptr || (ld % 16 == 0 && (reinterpret_cast<uintptr_t>(p) & 15) == 0); }

template <typename T, int MT, bool GATED>
int by_lie(const Small &p, int act, cudaStream_t st) {
    if (!on16(p.codes, p.ldc) || !on16(p.codes2, p.ldc2)) return launch<T, MT, ANY, GATED>(p, act, st);
    return p.K % SEG ? launch<T, MT, ON16, GATED>(p, act, st) : launch<T, MT, WHOLE, GATED>(p, act, st);
}

template <typename T, bool GATED>
int by_rows(const Small &p, int act, cudaStream_t st) {
    if (p.M <= 8) return by_lie<T, 1, GATED>(p, act, st);
    if (p.M <= 16) return by_lie<T, 2, GATED>(p, act, st);
    if (p.M <= 32) return by_lie<T, 4, GATED>(p, act, st);
    return by_lie<T, 6, GATED>(p, act, st);
}

// warps that share a group of channels: as many as fill the SMs, each with two segments at least
int share(int64_t groups, int64_t K) {
    const int64_t segs = (K + SEG - 1) / SEG;
    int ks = 8;
    while (ks > 1 && (segs < 2 * ks || groups * ks > 32ll * sm_count())) ks /= 2;
    return ks;
}

}  // namespace

int tensor_small(int dtype, const void *x, int64_t ldx, const int8_t *codes, int64_t ldc, const float *scale, int bits,
                 const void *bias, int bias_dtype, int act, const void *residual, int64_t ldr, void *y, int64_t ldy,
                 int64_t M, int64_t N, int64_t K, cudaStream_t st) {
    Small p{};
    p.x = x;
    p.codes = codes;
    p.scale = scale;
    p.bias = bias;
    p.residual = residual;
    p.y = y;
    p.ldx = ldx;
    p.ldc = ldc;
    p.ldr = ldr;
    p.ldy = ldy;
    p.N = N;
    p.K = K;
    p.unit = 1.0f / (float)(1 << (bits - 1));
    p.M = (int)M;
    p.bias_dtype = bias_dtype;
    p.ks = share((N + 15) / 16, K);
    return dtype == SFB_BF16 ? by_rows<__nv_bfloat16, false>(p, act, st) : by_rows<__half, false>(p, act, st);
}

int tensor_gated_small(int dtype, const void *x, int64_t ldx, const int8_t *gate, int64_t ldg, const float *gate_scale,
                       const int8_t *up, int64_t ldu, const float *up_scale, int bits, const void *bias, int bias_dtype,
                       const void *bias2, int bias2_dtype, int act, void *y, int64_t ldy, int64_t M, int64_t N, int64_t K,
                       cudaStream_t st) {
    Small p{};
    p.x = x;
    p.codes = gate;
    p.codes2 = up;
    p.scale = gate_scale;
    p.scale2 = up_scale;
    p.bias = bias;
    p.bias2 = bias2;
    p.y = y;
    p.ldx = ldx;
    p.ldc = ldg;
    p.ldc2 = ldu;
    p.ldy = ldy;
    p.N = N;
    p.K = K;
    p.unit = 1.0f / (float)(1 << (bits - 1));
    p.M = (int)M;
    p.bias_dtype = bias_dtype;
    p.bias2_dtype = bias2_dtype;
    p.ks = share((N + 7) / 8, K);
    return dtype == SFB_BF16 ? by_rows<__nv_bfloat16, true>(p, act, st) : by_rows<__half, true>(p, act, st);
}

}  // namespace sfb
