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

// four codes as two pairs of the activations' type
template <typename T> __device__ __forceinline__ void widen(uint32_t w, uint32_t &lo, uint32_t &hi);

// 0x43cc as bf16 is 128 + (c mod 128), or twice that form's 128 where bit 7 is set: the
// difference of the two is c in two's complement, exactly
template <>
__device__ __forceinline__ void widen<__nv_bfloat16>(uint32_t w, uint32_t &lo, uint32_t &hi) {
    const uint32_t a = __byte_perm(w, 0x43434343u, 0x4140), b = __byte_perm(w, 0x43434343u, 0x4342);
    const uint32_t a0 = a & 0xFF7FFF7Fu, a1 = a & 0xFF80FF80u, b0 = b & 0xFF7FFF7Fu, b1 = b & 0xFF80FF80u;
    __nv_bfloat162 x = __hsub2(reinterpret_cast<const __nv_bfloat162 &>(a0), reinterpret_cast<const __nv_bfloat162 &>(a1));
    __nv_bfloat162 y = __hsub2(reinterpret_cast<const __nv_bfloat162 &>(b0), reinterpret_cast<const __nv_bfloat162 &>(b1));
    lo = reinterpret_cast<uint32_t &>(x);
    hi = reinterpret_cast<uint32_t &>(y);
}

// 0x64uu as fp16 is 1024 + u; with u = c + 128 less 1152 it is c
template <>
__device__ __forceinline__ void widen<__half>(uint32_t w, uint32_t &lo, uint32_t &hi) {
    w ^= 0x80808080u;
    const uint32_t a = __byte_perm(w, 0x64646464u, 0x4140), b = __byte_perm(w, 0x64646464u, 0x4342);
    const __half2 c = __half2half2(__ushort_as_half((unsigned short)0x6480));
    __half2 x = __hsub2(reinterpret_cast<const __half2 &>(a), c), y = __hsub2(reinterpret_cast<const __half2 &>(b), c);
    lo = reinterpret_cast<uint32_t &>(x);
    hi = reinterpret_cast<uint32_t &>(y);
}

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

// 16 codes of a row from k on, those at or past K as 0: into `to` ...
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

// ... or, where rows do not start on 16 bytes, from the whole words around them, each holding at least one of the
// row's codes, shifted into place
__device__ __forceinline__ uint4 shift_codes(const int8_t *row, int64_t k, int64_t K) {
    uint32_t w[4] = {0, 0, 0, 0};
    if (k >= K) return make_uint4(0, 0, 0, 0);
    const uintptr_t at = reinterpret_cast<uintptr_t>(row + k), end = reinterpret_cast<uintptr_t>(row + K);
    const uint32_t *from = reinterpret_cast<const uint32_t *>(at & ~(uintptr_t)3);
    const uint32_t shift = 8 * (uint32_t)(at & 3);
    uint32_t a = __ldg(from);
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const uint32_t b = reinterpret_cast<uintptr_t>(from + i + 1) < end ? __ldg(from + i + 1) : 0u;
        w[i] = __funnelshift_r(a, b, shift);
        a = b;
    }
    const int left = (int)min((int64_t)16, K - k);
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const int keep = left - 4 * i;
        w[i] &= keep >= 4 ? 0xFFFFFFFFu : keep <= 0 ? 0u : (1u << (8 * keep)) - 1u;
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
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
    void *y;
    int64_t ldx, ldc, ldr, ldy, N, K;
    float unit;
    int M, ks, bias_dtype;
};

constexpr int DEEP = 4;

// How K and the codes' rows lie: WHOLE, in whole segments on 16 bytes, asks nothing
// in the loop (the questions are half of its instructions); ON16, rows on 16 bytes; ANY.
enum { WHOLE, ON16, ANY };

template <typename T, int MT, int LIE, int ACT>
__global__ void __launch_bounds__(32 * WARPS, MT <= 2 ? 4 : MT == 4 ? 3 : 2) small_kernel(Small p) {
    __shared__ union {
        uint4 codes[DEEP][2][32 * WARPS];
        float sum[WARPS][16][8 * MT];
    } s;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int groups = WARPS / p.ks, group = warp / p.ks, part = warp % p.ks;
    const int64_t n0 = ((int64_t)blockIdx.x * groups + group) * 16;
    // channels past the last read the last one's codes, rows past the last the last one: their sums are not stored
    const int8_t *row0 = p.codes + min(n0 + g, p.N - 1) * p.ldc, *row1 = p.codes + min(n0 + g + 8, p.N - 1) * p.ldc;
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
    for (int o = threadIdx.x; o < groups * 16 * p.M; o += 32 * WARPS) {
        const int c = o % (groups * 16), m = o / (groups * 16);
        const int64_t n = (int64_t)blockIdx.x * groups * 16 + c;
        if (n >= p.N) continue;
        float v = 0.0f;
        for (int i = 0; i < p.ks; i++) v += s.sum[(c / 16) * p.ks + i][c % 16][m];
        v = fmaf(v, p.scale[n] * p.unit, p.bias ? load_as(p.bias, n, p.bias_dtype) : 0.0f);
        v = activate<ACT>(v);
        if (p.residual) v += to_f(static_cast<const T *>(p.residual)[m * p.ldr + n]);
        static_cast<T *>(p.y)[m * p.ldy + n] = from_f<T>(v);
    }
}

template <typename T, int MT, int LIE>
int launch(const Small &p, int act, cudaStream_t st) {
    const int64_t groups = (p.N + 15) / 16;
    const int per = WARPS / p.ks;
    const unsigned grid = (unsigned)((groups + per - 1) / per);
    return with_activation(act, [&](auto a) {
        small_kernel<T, MT, LIE, decltype(a)::value><<<grid, 32 * WARPS, 0, st>>>(p);
        return check_launch("sf tensor linear (few rows)");
    });
}

template <typename T, int MT>
int by_lie(const Small &p, int act, cudaStream_t st) {
    if (p.ldc % 16 || (reinterpret_cast<uintptr_t>(p.codes) & 15)) return launch<T, MT, ANY>(p, act, st);
    return p.K % SEG ? launch<T, MT, ON16>(p, act, st) : launch<T, MT, WHOLE>(p, act, st);
}

template <typename T>
int by_rows(const Small &p, int act, cudaStream_t st) {
    if (p.M <= 8) return by_lie<T, 1>(p, act, st);
    if (p.M <= 16) return by_lie<T, 2>(p, act, st);
    if (p.M <= 32) return by_lie<T, 4>(p, act, st);
    return by_lie<T, 6>(p, act, st);
}

}  // namespace

int tensor_small(int dtype, const void *x, int64_t ldx, const int8_t *codes, int64_t ldc, const float *scale, int bits,
                 const void *bias, int bias_dtype, int act, const void *residual, int64_t ldr, void *y, int64_t ldy,
                 int64_t M, int64_t N, int64_t K, cudaStream_t st) {
    Small p{x, codes, scale, bias, residual, y, ldx, ldc, ldr, ldy, N, K, 1.0f / (float)(1 << (bits - 1)), (int)M, 8,
            bias_dtype};
    // warps that share a group of channels: as many as fill the SMs, each with two segments at least
    const int64_t groups = (N + 15) / 16, segs = (K + SEG - 1) / SEG;
    while (p.ks > 1 && (segs < 2 * p.ks || groups * p.ks > 32ll * sm_count())) p.ks /= 2;
    return dtype == SFB_BF16 ? by_rows<__nv_bfloat16>(p, act, st) : by_rows<__half>(p, act, st);
}

}  // namespace sfb
