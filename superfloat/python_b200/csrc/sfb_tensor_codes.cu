// The operands of the tensor-core linear other than the product itself: a float
// weight's codes and scales, packed codes in the activations' type, and the
// gradient of the pre-activation.
#include <math.h>

#include <algorithm>

#include "sfb_tensor_parts.cuh"

namespace sfb {
namespace {

constexpr int QT = 256;

// --- rows on 16-byte boundaries ----------------------------------------------------------------------

// 64 threads along a row, 8 elements each, 4 rows a block of 256; block (bx, by) of gx by gy
__device__ __forceinline__ void pad_rows(const Rows &r, int tx, int ty, int bx, int gx, int by, int gy) {
    const uint16_t *x = static_cast<const uint16_t *>(r.x);
    for (int64_t m = (int64_t)by * 4 + ty; m < r.M; m += 4ll * gy)
        for (int64_t k = ((int64_t)bx * 64 + tx) * 8; k < r.K; k += 512ll * gx) {
            Vec<uint16_t, 8> q;
#pragma unroll
            for (int j = 0; j < 8; j++) q.v[j] = k + j < r.K ? x[m * r.ldx + k + j] : (uint16_t)0;
            *reinterpret_cast<Vec<uint16_t, 8> *>(static_cast<uint16_t *>(r.out) + m * r.ldo + k) = q;
        }
}

__global__ void __launch_bounds__(QT) pad_kernel(Rows r) {
    pad_rows(r, threadIdx.x, threadIdx.y, blockIdx.x, gridDim.x, blockIdx.y, gridDim.y);
}

// --- codes of a float weight -------------------------------------------------------------------------
//
// s = amax / m (m = M / 2^(N-1), 1 where amax is 0) in float64, kept as float32;
// code = rint(w / s 2^(N-1)), held within +-M.  The quotient is first taken in
// float32, off by at most 2^-16 of a code; where that lies within 2^-10 of a border of two
// codes it is made again as a float64 division, so the codes are those of the
// division.  A row that holds a NaN or an infinity gets that as its scale and its
// outputs are NaN.
// A warp has a row and reads it twice, the second time from L1 or L2; 8 elements a lane
// at a time where rows start on 16 bytes.  4096 x 4096 of fp16 under one
// scale take 12 us for the largest magnitude and 23 for the codes, 2304 x 768 of bf16
// with a scale a row 9.5.  With one scale every CTA of 8 rows reads all N rows' maxima,
// N^2 / 2 bytes from L2: nothing beside 4096 rows, and for 50257 rows of 768 78 us where
// the codes with a scale a row take 59.  (A CTA to a row, an element a thread and every quotient in
// float64: 51 us for the former's codes.)

__device__ __forceinline__ float scale_from(uint32_t amax_bits, double m) {
    const float amax = __uint_as_float(amax_bits);
    return amax == 0.0f ? 1.0f : (float)((double)amax / m);
}

__device__ __forceinline__ float code_from(float w, float s, float inv, float M, double unit) {
    // the nearest integer, ties to even: adding 1.5 2^23 leaves it in the last bits
    // (rintf is a conversion, which an SM makes at an eighth of the rate of sums)
    const float t = w * inv, r = __fsub_rn(__fadd_rn(t, 12582912.0f), 12582912.0f);
    if (fabsf(t - r) <= 0.4990234375f) return r > M ? M : r < -M ? -M : r;
    const double d = rint((double)w / (double)s * unit);            // near a border, or not finite
    return d >= M ? M : d <= -M ? -M : d == d ? (float)d : 0.0f;
}

// 8 elements from k on, those past K as 0
template <typename W>
__device__ __forceinline__ void load8f(const W *row, int64_t k, int64_t K, bool vec, float (&v)[8]) {
    if (vec && k + 8 <= K) {
        constexpr int P = 16 / sizeof(W);
#pragma unroll
        for (int i = 0; i < 8 / P; i++) {
            const Vec<W, P> q = *reinterpret_cast<const Vec<W, P> *>(row + k + i * P);
#pragma unroll
            for (int j = 0; j < P; j++) v[i * P + j] = to_f(q.v[j]);
        }
    } else {
#pragma unroll
        for (int j = 0; j < 8; j++) v[j] = k + j < K ? to_f(row[k + j]) : 0.0f;
    }
}

// magnitudes order as their bits, NaN above infinity
template <typename W>
__device__ __forceinline__ uint32_t row_top(const W *row, int64_t K, bool vec, int lane) {
    uint32_t top = 0;
#pragma unroll 4
    for (int64_t k = lane * 8; k < K; k += 256) {
        float v[8];
        load8f(row, k, K, vec, v);
#pragma unroll
        for (int j = 0; j < 8; j++) top = max(top, __float_as_uint(v[j]) & 0x7FFFFFFFu);
    }
    return __reduce_max_sync(0xffffffffu, top);
}

template <typename W>
__global__ void __launch_bounds__(QT) amax_kernel(const W *__restrict__ w, int64_t N, int64_t K, int64_t ldw, bool vec,
                                                  uint32_t *amax) {
    const int64_t n = (int64_t)blockIdx.x * (QT / 32) + threadIdx.x / 32;
    if (n >= N) return;
    const uint32_t top = row_top(w + n * ldw, K, vec, threadIdx.x & 31);
    if ((threadIdx.x & 31) == 0) amax[n] = top;
}

// amax: of the rows, for one scale; null for a scale a row
template <typename W, typename O>
__global__ void __launch_bounds__(QT) code_kernel(const W *__restrict__ w, int64_t N, int64_t K, int64_t ldw, bool vec,
                                                  int bits, const uint32_t *__restrict__ amax, O *codes, int64_t ldc,
                                                  bool whole, float *scale, Rows rows) {
    if (blockIdx.y == 1) {                     // x's copy, in the launch that the call makes anyway
        pad_rows(rows, threadIdx.x & 63, threadIdx.x >> 6, 0, 1, blockIdx.x, gridDim.x);
        return;
    }
    if ((int64_t)blockIdx.x * (QT / 32) >= N) return;
    __shared__ uint32_t s_top[QT / 32];
    const int lane = threadIdx.x & 31;
    const int64_t n = (int64_t)blockIdx.x * (QT / 32) + threadIdx.x / 32;
    uint32_t top = 0;
    if (amax) {
        for (int64_t i = threadIdx.x; i < N; i += QT) top = max(top, amax[i]);
        top = __reduce_max_sync(0xffffffffu, top);
        if (lane == 0) s_top[threadIdx.x >> 5] = top;
        __syncthreads();
        for (int i = 0; i < QT / 32; i++) top = max(top, s_top[i]);
    }
    if (n >= N) return;
    const W *row = w + n * ldw;
    if (!amax) top = row_top(row, K, vec, lane);
    const double unit = (double)(1 << (bits - 1));
    const float M = (float)((1 << (bits - 1)) - 1), s = scale_from(top, (double)M / unit), inv = (float)(unit / (double)s);
    if (lane == 0) scale[n] = s;
    O *out = codes + n * ldc;
#pragma unroll 2
    for (int64_t k = lane * 8; k < K; k += 256) {
        float v[8];
        load8f(row, k, K, vec, v);
        Vec<O, 8> q;
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const float c = code_from(v[j], s, inv, M, unit);
            if constexpr (sizeof(O) == 1) q.v[j] = (O)(__float_as_uint(c + 12582912.0f) & 0xFFu);
            else q.v[j] = from_f<O>(c);
        }
        if (whole) {
            *reinterpret_cast<Vec<O, 8> *>(out + k) = q;         // a row's padding may be written
        } else {
#pragma unroll
            for (int j = 0; j < 8; j++)
                if (k + j < K) out[k + j] = q.v[j];
        }
    }
}

// --- packed codes in the activations' type -----------------------------------------------------------

// A thread turns 16 codes of a row at a time; where rows do not start on 16
// bytes it loads them one by one (the stores are aligned: the rows of `out` are).
// Rows without gaps are one long row.  64 threads along a row, 4 rows a CTA.
// Where x has to be copied too, the grid's second layer does it: a launch less for
// a call that waits for the host (777 x 1031 x 2049: 24.6 to 21.1 us).
template <typename O>
__global__ void __launch_bounds__(QT) expand_kernel(const int8_t *__restrict__ codes, int64_t N, int64_t K, int64_t ldc,
                                                    O *__restrict__ out, int64_t ldo, bool vec, Rows rows) {
    if (blockIdx.z == 1) {
        pad_rows(rows, threadIdx.x, threadIdx.y, blockIdx.x, gridDim.x, blockIdx.y, gridDim.y);
        return;
    }
    for (int64_t n = (int64_t)blockIdx.y * 4 + threadIdx.y; n < N; n += 4ll * gridDim.y) {
#pragma unroll 4
        for (int64_t k = ((int64_t)blockIdx.x * 64 + threadIdx.x) * 16; k < K; k += 1024ll * gridDim.x) {
            const int8_t *from = codes + n * ldc + k;
            O *to = out + n * ldo + k;
            Vec<int8_t, 16> q;
            if (vec && k + 16 <= K) {
                q = *reinterpret_cast<const Vec<int8_t, 16> *>(from);
            } else {
#pragma unroll
                for (int j = 0; j < 16; j++) q.v[j] = k + j < K ? from[j] : (int8_t)0;
            }
#pragma unroll
            for (int h = 0; h < 2; h++) {
                Vec<O, 8> r;
#pragma unroll
                for (int j = 0; j < 8; j++) r.v[j] = from_f<O>((float)q.v[8 * h + j]);
                if (k + 8 * h < K) *reinterpret_cast<Vec<O, 8> *>(to + 8 * h) = r;   // a row's padding may be written
            }
        }
    }
}

// --- the gradient of the pre-activation --------------------------------------------------------------
//
// dz = dy act'(z); written as dz (the operand of the weight's gradient) and
// as dz[n] s[n] / top (the operand of x's gradient: the channel's scale cannot
// wait for the product, which sums over channels; top keeps fp16 within its range),
// each rounded once from float32: both operands of a product have one type, and the
// other one is 16 bits.  A bf16 gradient is then off by 2.3e-3 in the 2-norm, 1.7e-3 of
// it the result's own rounding; an fp16 one by 3.0e-4 and 2.1e-4.
// db = sum over rows, in a fixed order: every
// CTA sums its 64 rows, and an idle warp of the weight's product (or, without
// it, a kernel) the CTAs' sums.
// Memory bound: dy and z read, dz and / or dz s written (8192 x 4096 of fp16, one scale:
// 201 MB in 31 us, 6.5 TB/s).

constexpr int BR = 64;                   // rows of a CTA
constexpr int BC = 256;                  // columns: 32 threads of 8

// A CTA's place: its columns first, in one grid dimension, as a convolution's rows
// (images x their pixels) pass the 65535 x 64 that the others reach.
__device__ __forceinline__ void place_of(int64_t N, int64_t &row, int64_t &column) {
    const unsigned across = (unsigned)((N + BC - 1) / BC);
    row = blockIdx.x / across;
    column = blockIdx.x % across;
}

template <bool VEC, typename T>
__device__ __forceinline__ Vec<T, 8> load8t(const T *from, int64_t left) {
    if constexpr (VEC) {
        return *reinterpret_cast<const Vec<T, 8> *>(from);
    } else {
        Vec<T, 8> q;
#pragma unroll
        for (int j = 0; j < 8; j++) q.v[j] = j < left ? from[j] : from_f<T>(0.0f);
        return q;
    }
}

// VEC: N is a multiple of 8 and the rows of dy and z start on 16 bytes
template <typename T, int ACT, bool VEC>
__global__ void __launch_bounds__(256, VEC ? 4 : 2)
slope_kernel(const T *__restrict__ dy, int64_t ldy, const __half *__restrict__ z, int64_t ldz, int64_t M, int64_t N,
             const float *__restrict__ scale, float unit, const float *__restrict__ top, T *__restrict__ dz,
             T *__restrict__ dzs, int64_t ldd, float *__restrict__ sums) {
    __shared__ float s_sum[8][BC];
    const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
    int64_t by, bx;
    place_of(N, by, bx);
    const int64_t n0 = bx * BC + tx * 8, left = N - n0;
    const int64_t r1 = min(M, (by + 1) * BR);
    float acc[8] = {}, f[8];
    if (dzs) {
        const float share = top ? __fdiv_rn(1.0f, *top) : unit;
#pragma unroll
        for (int j = 0; j < 8; j++) {
            f[j] = j < left ? scale[n0 + j] * share : 0.0f;
            if (fabsf(f[j]) > 1.001f && top) f[j] = 1.0f;        // a channel without a code, larger than `top`
        }
    }
    auto row = [&](int64_t r, const Vec<T, 8> &g, const Vec<__half, 8> &h) {
        float d[8];
#pragma unroll
        for (int j = 0; j < 8; j++) {
            d[j] = to_f(g.v[j]);
            // (one rounding, whatever else is wanted: contracted with the sum it would be none)
            if constexpr (ACT != SFB_ACT_NONE) d[j] = __fmul_rn(d[j], slope<ACT>(to_f(h.v[j])));
            acc[j] += d[j];
        }
        // ldd is a multiple of 8 and the buffers are aligned: the vector's tail lands in the row's padding
        if (dz) {
            Vec<T, 8> q;
#pragma unroll
            for (int j = 0; j < 8; j++) q.v[j] = from_f<T>(d[j]);
            *reinterpret_cast<Vec<T, 8> *>(dz + r * ldd + n0) = q;
        }
        if (dzs) {
            Vec<T, 8> q;
#pragma unroll
            for (int j = 0; j < 8; j++) q.v[j] = from_f<T>(d[j] * f[j]);
            *reinterpret_cast<Vec<T, 8> *>(dzs + r * ldd + n0) = q;
        }
    };
    if (left > 0) {
        int64_t r = by * BR + ty;
#pragma unroll 1
        for (; r + 8 < r1; r += 16) {                     // two rows' loads in flight
            const Vec<T, 8> g0 = load8t<VEC>(dy + r * ldy + n0, left), g1 = load8t<VEC>(dy + (r + 8) * ldy + n0, left);
            Vec<__half, 8> h0, h1;
            if constexpr (ACT != SFB_ACT_NONE) {
                h0 = load8t<VEC>(z + r * ldz + n0, left);
                h1 = load8t<VEC>(z + (r + 8) * ldz + n0, left);
            }
            row(r, g0, h0);
            row(r + 8, g1, h1);
        }
        if (r < r1) {
            const Vec<T, 8> g = load8t<VEC>(dy + r * ldy + n0, left);
            Vec<__half, 8> h;
            if constexpr (ACT != SFB_ACT_NONE) h = load8t<VEC>(z + r * ldz + n0, left);
            row(r, g, h);
        }
    }
    if (sums) {
#pragma unroll
        for (int j = 0; j < 8; j++) s_sum[ty][tx * 8 + j] = acc[j];
        __syncthreads();
        const int64_t n = bx * BC + threadIdx.x;
        if (n < N) {
            float v = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; i++) v += s_sum[i][threadIdx.x];
            sums[by * N + n] = v;
        }
    }
}

__global__ void __launch_bounds__(32) sum_kernel(Sums s) {
    const int64_t n = (int64_t)blockIdx.x * 32 + threadIdx.x;
    if (n < s.N) store_as(s.db, n, s.dtype, column_sum(s, n));
}

// The largest of the scales whose channel has a code other than 0: a row of zeros has
// the scale 1 by rule, and beside weights of 1e-3 would leave dz s / 1 below fp16's
// normal range.  Only rows of that scale are looked at, and only where no larger one
// makes it idle; others without a code (a caller's own scales) stay within the range by
// what they give.  At least 2^-126, so that its reciprocal is finite.
// One CTA: 2.4 us for 4096 scales, and the whole of it reads the rows in question, 16
// bytes a thread (a thread to a row took 82 us for one row of 4096).
__global__ void __launch_bounds__(1024) top_kernel(const float *__restrict__ scale, int64_t N,
                                                   const uint16_t *__restrict__ codes, int64_t ldc, int64_t K, float *top) {
    constexpr uint32_t ONE = 0x3F800000u;
    __shared__ uint32_t s_top[32];
    __shared__ int s_rows[1024], s_count;
    uint32_t t = 0x00800000u;                          // magnitudes order as their bits, NaN above all
    int ones = 0;
    for (int64_t n = threadIdx.x; n < N; n += 1024) {
        const uint32_t s = __float_as_uint(scale[n]) & 0x7FFFFFFFu;
        if (s == ONE) ones = 1;
        else t = max(t, s);
    }
    t = __reduce_max_sync(0xffffffffu, t);
    if ((threadIdx.x & 31) == 0) s_top[threadIdx.x >> 5] = t;
    ones = __syncthreads_or(ones);
    t = __reduce_max_sync(0xffffffffu, s_top[threadIdx.x & 31]);
    if (ones && t < ONE) {                             // the same for all threads
        const int64_t per = (K + 7) / 8;               // pieces of 16 bytes a row
        int live = 0;
        for (int64_t n0 = 0; n0 < N && !live; n0 += 1024) {
            __syncthreads();
            if (threadIdx.x == 0) s_count = 0;
            __syncthreads();
            const int64_t n = n0 + threadIdx.x;
            if (n < N && (__float_as_uint(scale[n]) & 0x7FFFFFFFu) == ONE) s_rows[atomicAdd(&s_count, 1)] = threadIdx.x;
            __syncthreads();
            const int64_t pieces = s_count * per;
            for (int64_t i = threadIdx.x; i - threadIdx.x < pieces && !live; i += 4 * 1024) {
                uint4 q[4];
#pragma unroll
                for (int u = 0; u < 4; u++) {
                    const int64_t at = i + 1024 * u;
                    q[u] = at < pieces ? __ldg(reinterpret_cast<const uint4 *>(codes + (n0 + s_rows[at / per]) * ldc) + at % per)
                                       : make_uint4(0, 0, 0, 0);
                }
                int any = 0;
#pragma unroll
                for (int u = 0; u < 4; u++) {
                    const uint32_t w[4] = {q[u].x, q[u].y, q[u].z, q[u].w};
                    const int64_t k = (i + 1024 * u) % per * 8;
#pragma unroll
                    for (int j = 0; j < 4; j++)        // (what is past K is a row's padding)
                        any |= ((w[j] & 0x7FFFu) && k + 2 * j < K) || ((w[j] & 0x7FFF0000u) && k + 2 * j + 1 < K);
                }
                live = __syncthreads_or(any);
            }
        }
        if (live) t = ONE;
    } else if (ones) {
        t = max(t, ONE);
    }
    if (threadIdx.x == 0) *top = __uint_as_float(t);
}

template <typename W>
int quantize_from(const W *w, int64_t N, int64_t K, int64_t ldw, int bits, bool per_channel, void *codes, int64_t ldc,
                  int out, float *scale, uint32_t *amax, const Rows &rows, cudaStream_t st) {
    const bool vec = (reinterpret_cast<uintptr_t>(w) & 15) == 0 && ldw * sizeof(W) % 16 == 0;
    const unsigned grid = (unsigned)((N + QT / 32 - 1) / (QT / 32));
    if (!per_channel) amax_kernel<W><<<grid, QT, 0, st>>>(w, N, K, ldw, vec, amax);
    const uint32_t *top = per_channel ? nullptr : amax;
    const dim3 both(std::max<unsigned>(grid, rows.x ? (unsigned)std::min<int64_t>((rows.M + 3) / 4, 16ll * sm_count()) : 0),
                    rows.x ? 2 : 1);
    // a row of 16-bit codes is padded to a multiple of 8; one of int8 only where the caller's stride says so
    if (out == SFB_I8)
        code_kernel<W, int8_t><<<both, QT, 0, st>>>(w, N, K, ldw, vec, bits, top, static_cast<int8_t *>(codes), ldc,
                                                    K % 8 == 0 && ldc % 8 == 0 && (reinterpret_cast<uintptr_t>(codes) & 7) == 0,
                                                    scale, rows);
    else if (out == SFB_BF16)
        code_kernel<W, __nv_bfloat16><<<both, QT, 0, st>>>(w, N, K, ldw, vec, bits, top,
                                                           static_cast<__nv_bfloat16 *>(codes), ldc, true, scale, rows);
    else
        code_kernel<W, __half><<<both, QT, 0, st>>>(w, N, K, ldw, vec, bits, top, static_cast<__half *>(codes), ldc,
                                                    true, scale, rows);
    return check_launch("sf weight codes");
}

}  // namespace

int tensor_quantize(const void *w, int dtype, int64_t N, int64_t K, int64_t ldw, int bits, bool per_channel, void *codes,
                    int64_t ldc, int codes_dtype, float *scale, void *work, const Rows &rows,
                    cudaStream_t st) {
    uint32_t *amax = static_cast<uint32_t *>(work);
    if (dtype == SFB_F32)
        return quantize_from(static_cast<const float *>(w), N, K, ldw, bits, per_channel, codes, ldc, codes_dtype,
                             scale, amax, rows, st);
    if (dtype == SFB_BF16)
        return quantize_from(static_cast<const __nv_bfloat16 *>(w), N, K, ldw, bits, per_channel, codes, ldc,
                             codes_dtype, scale, amax, rows, st);
    return quantize_from(static_cast<const __half *>(w), N, K, ldw, bits, per_channel, codes, ldc, codes_dtype, scale,
                         amax, rows, st);
}

namespace {
// blocks along a row of K elements, `step` a block, and over N rows, 4 a block
dim3 rows_grid(int64_t N, int64_t K, int step) {
    const int64_t room = 16ll * sm_count(), gy = std::min<int64_t>((N + 3) / 4, room);
    return dim3((unsigned)std::min<int64_t>((K + step - 1) / step, std::max<int64_t>(1, room / gy)), (unsigned)gy);
}
}  // namespace

int tensor_expand(const int8_t *codes, int64_t N, int64_t K, int64_t ldc, void *out, int64_t ldo, int dtype,
                  const Rows &rows, cudaStream_t st) {
    const bool vec = ldc % 16 == 0 && (reinterpret_cast<uintptr_t>(codes) & 15) == 0;
    dim3 grid, block(64, 4);
    if (rows.x) {
        const dim3 g = rows_grid(N, K, 1024), h = rows_grid(rows.M, rows.K, 512);
        grid = dim3(std::max(g.x, h.x), std::max(g.y, h.y), 2);
    } else if (ldc == K && ldo == K && K % 16 == 0) {
        K *= N, N = 1, ldc = ldo = K;
        grid = dim3((unsigned)std::min<int64_t>((K + 1023) / 1024, 64ll * sm_count()));
        block.y = 1;
    } else {
        grid = rows_grid(N, K, 1024);
    }
    if (dtype == SFB_BF16)
        expand_kernel<<<grid, block, 0, st>>>(codes, N, K, ldc, static_cast<__nv_bfloat16 *>(out), ldo, vec, rows);
    else
        expand_kernel<<<grid, block, 0, st>>>(codes, N, K, ldc, static_cast<__half *>(out), ldo, vec, rows);
    return check_launch("sf tensor linear (packed codes)");
}

int tensor_pad(const Rows &rows, cudaStream_t st) {
    pad_kernel<<<rows_grid(rows.M, rows.K, 512), dim3(64, 4), 0, st>>>(rows);
    return check_launch("sf tensor linear (rows of x)");
}

int tensor_top(const float *scale, int64_t N, const void *codes, int64_t ldc, int64_t K, float *top, cudaStream_t st) {
    top_kernel<<<1, 1024, 0, st>>>(scale, N, static_cast<const uint16_t *>(codes), ldc, K, top);
    return check_launch("sf tensor linear (largest scale)");
}

int64_t tensor_slope_parts(int64_t M) { return (M + BR - 1) / BR; }

int tensor_slope(int dtype, int act, const void *dy, int64_t ldy, const void *z, int64_t ldz, int64_t M, int64_t N,
                 const float *scale, int bits, const float *top, void *dz, void *dzs, int64_t ldd, float *sums,
                 cudaStream_t st) {
    const int64_t blocks = tensor_slope_parts(M) * ((N + BC - 1) / BC);
    if (blocks >= 1ll << 31)
        return set_error(SFB_ERANGE, "sf tensor linear: a gradient of %lld x %lld", (long long)M, (long long)N);
    const float unit = 1.0f / (float)(1 << (bits - 1));
    const unsigned grid = (unsigned)blocks;
    const bool vec = N % 8 == 0 && ldy % 8 == 0 && (reinterpret_cast<uintptr_t>(dy) & 15) == 0 &&
                     (act == SFB_ACT_NONE || (ldz % 8 == 0 && (reinterpret_cast<uintptr_t>(z) & 15) == 0));
    return with_activation(act, [&](auto a) {
        constexpr int A = decltype(a)::value;
        auto go = [&](auto *kernel, auto type) {
            using T = decltype(type);
            kernel<<<grid, 256, 0, st>>>(static_cast<const T *>(dy), ldy, static_cast<const __half *>(z), ldz, M, N, scale,
                                         unit, top, static_cast<T *>(dz), static_cast<T *>(dzs), ldd, sums);
        };
        if (dtype == SFB_BF16)
            vec ? go(slope_kernel<__nv_bfloat16, A, true>, __nv_bfloat16()) : go(slope_kernel<__nv_bfloat16, A, false>, __nv_bfloat16());
        else
            vec ? go(slope_kernel<__half, A, true>, __half()) : go(slope_kernel<__half, A, false>, __half());
        return check_launch("sf tensor linear (activation's gradient)");
    });
}

int tensor_sum(const Sums &sums, cudaStream_t st) {
    sum_kernel<<<(unsigned)((sums.N + 31) / 32), 32, 0, st>>>(sums);
    return check_launch("sf tensor linear (bias's gradient)");
}

}  // namespace sfb

extern "C" int sfb_code_quantize(const void *w, int dtype, int64_t N, int64_t K, int64_t ldw, int bits,
                                 int per_channel, void *codes, int64_t ldc, float *scale, void *work,
                                 sfb_stream stream) {
    using namespace sfb;
    if (bits < 4 || bits > 8) return set_error(SFB_EINVAL, "sfb_code_quantize: width %d is not in 4..8", bits);
    if (dtype != SFB_F32 && dtype != SFB_BF16 && dtype != SFB_F16)
        return set_error(SFB_EINVAL, "sfb_code_quantize: element type %d", dtype);
    if (N < 0 || K < 0 || ldw < K || ldc < K) return set_error(SFB_EINVAL, "sfb_code_quantize: bad shape");
    if (N >= (1ll << 31)) return set_error(SFB_ERANGE, "sfb_code_quantize: %lld rows", (long long)N);
    if (N == 0 || K == 0) return SFB_OK;
    if (!w || !codes || !scale || (!per_channel && !work)) return set_error(SFB_EINVAL, "sfb_code_quantize: null pointer");
    return tensor_quantize(w, dtype, N, K, ldw, bits, per_channel != 0, codes, ldc, SFB_I8, scale, work, Rows{},
                           static_cast<cudaStream_t>(stream));
}
