// The operands of the tensor-core linear other than the product itself: a float
// weight's codes and scales, packed codes in the activations' type, and the
// gradient of the pre-activation.
#include <math.h>

#include <algorithm>

#include "sfb_tensor.cuh"

namespace sfb {
namespace {

constexpr int QT = 256;

// --- codes of a float weight -------------------------------------------------------------------------
//
// s = amax / m (m = M / 2^(N-1), 1 where amax is 0) in float64, kept as float32;
// code = rint(w / s 2^(N-1)), held within +-M.  The quotient is taken as a
// product with 2^(N-1) / s in float64, 1e-16 off the true one; only where that
// lies within 1e-9 of a border of two codes is the division itself made, so the
// codes are those of the division.  A row that holds a NaN or an infinity gets
// that as its scale and its outputs are NaN.
// Memory bound: a row is read twice, the second time from L1 / L2.

__device__ __forceinline__ float scale_from(uint32_t amax_bits, double m) {
    const float amax = __uint_as_float(amax_bits);
    return amax == 0.0f ? 1.0f : (float)((double)amax / m);
}

__device__ __forceinline__ int code_from(float w, double s, double inv, int M, double unit) {
    double t = (double)w * inv;
    if (fabs(t - rint(t)) > 0.5 - 1e-9) t = (double)w / s * unit;
    const double r = rint(t);
    return r >= M ? M : r <= -M ? -M : r == r ? (int)r : 0;
}

// magnitudes order as their bits, NaN above infinity
template <typename W>
__global__ void __launch_bounds__(QT) amax_kernel(const W *__restrict__ w, int64_t K, int64_t ldw, uint32_t *amax) {
    __shared__ uint32_t s_top[QT / 32];
    const W *row = w + (int64_t)blockIdx.x * ldw;
    uint32_t top = 0;
    for (int64_t k = threadIdx.x; k < K; k += QT) top = max(top, __float_as_uint(to_f(row[k])) & 0x7FFFFFFFu);
    top = __reduce_max_sync(0xffffffffu, top);
    if ((threadIdx.x & 31) == 0) s_top[threadIdx.x >> 5] = top;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int i = 1; i < QT / 32; i++) top = max(top, s_top[i]);
        amax[blockIdx.x] = top;
    }
}

template <typename W, typename O>
__global__ void __launch_bounds__(QT) code_kernel(const W *__restrict__ w, int64_t N, int64_t K, int64_t ldw, int bits,
                                                  const uint32_t *__restrict__ amax, int per_channel, O *codes,
                                                  int64_t ldc, float *scale) {
    __shared__ uint32_t s_top[QT / 32];
    const int M = (1 << (bits - 1)) - 1;
    const double unit = (double)(1 << (bits - 1)), m = M / unit;
    uint32_t top = 0;
    if (per_channel) {
        top = amax[blockIdx.x];
    } else {
        for (int64_t n = threadIdx.x; n < N; n += QT) top = max(top, amax[n]);
        top = __reduce_max_sync(0xffffffffu, top);
        if ((threadIdx.x & 31) == 0) s_top[threadIdx.x >> 5] = top;
        __syncthreads();
        for (int i = 0; i < QT / 32; i++) top = max(top, s_top[i]);
    }
    const float s = scale_from(top, m);
    if (threadIdx.x == 0) scale[blockIdx.x] = s;
    const double inv = unit / (double)s;
    const W *row = w + (int64_t)blockIdx.x * ldw;
    O *out = codes + (int64_t)blockIdx.x * ldc;
    for (int64_t k = threadIdx.x; k < K; k += QT) {
        const int c = code_from(to_f(row[k]), (double)s, inv, M, unit);
        if constexpr (sizeof(O) == 1) out[k] = (O)c;
        else out[k] = from_f<O>((float)c);
    }
}

// --- packed codes in the activations' type -----------------------------------------------------------

// A thread turns 16 codes of a row at a time; where rows do not start on 16
// bytes it loads them one by one (the stores are aligned: the rows of `out` are).
template <typename O>
__global__ void __launch_bounds__(QT) expand_kernel(const int8_t *__restrict__ codes, int64_t N, int64_t K, int64_t ldc,
                                                    O *__restrict__ out, int64_t ldo, bool vec) {
    const int64_t per = (K + 15) / 16, total = N * per;
    for (int64_t i = (int64_t)blockIdx.x * QT + threadIdx.x; i < total; i += (int64_t)gridDim.x * QT) {
        const int64_t n = i / per, k = (i - n * per) * 16;
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

// --- the gradient of the pre-activation --------------------------------------------------------------
//
// dz = dy act'(z); written as dz (the operand of the weight's gradient) and
// as dz[n] s[n] / top (the operand of x's gradient: the channel's scale cannot
// wait for the product, which sums over channels; top keeps fp16 within its range),
// each rounded once from float32.  db = sum over rows, in a fixed order: every
// CTA sums its 128 rows, and a second kernel the CTAs' sums.
// Memory bound: dy and z read, dz and / or dz s written.

constexpr int BR = 128;                  // rows of a CTA
constexpr int BC = 256;                  // columns: 32 threads of 8

template <typename T, int ACT>
__global__ void __launch_bounds__(256) slope_kernel(const T *__restrict__ dy, int64_t ldy, const __half *__restrict__ z,
                                                    int64_t ldz, int64_t M, int64_t N, const float *__restrict__ scale,
                                                    float unit, const float *__restrict__ top, T *__restrict__ dz,
                                                    T *__restrict__ dzs, int64_t ldd, float *__restrict__ sums) {
    __shared__ float s_sum[8][BC];
    const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
    const int64_t n0 = (int64_t)blockIdx.x * BC + tx * 8;
    const int64_t r0 = (int64_t)blockIdx.y * BR, r1 = min(M, r0 + BR);
    const bool whole = n0 + 8 <= N;
    const bool vy = whole && ldy % 8 == 0 && (reinterpret_cast<uintptr_t>(dy) & 15) == 0;
    const bool vz = ACT != SFB_ACT_NONE && whole && ldz % 8 == 0 && (reinterpret_cast<uintptr_t>(z) & 15) == 0;
    float acc[8] = {}, f[8];
    if (dzs) {
        const float by = top ? __fdiv_rn(1.0f, *top) : unit;
#pragma unroll
        for (int j = 0; j < 8; j++) f[j] = n0 + j < N ? scale[n0 + j] * by : 0.0f;
    }
    if (n0 < N) {
        for (int64_t r = r0 + ty; r < r1; r += 8) {
            float g[8], d[8];
            if (vy) {
                const Vec<T, 8> q = *reinterpret_cast<const Vec<T, 8> *>(dy + r * ldy + n0);
#pragma unroll
                for (int j = 0; j < 8; j++) g[j] = to_f(q.v[j]);
            } else {
#pragma unroll
                for (int j = 0; j < 8; j++) g[j] = n0 + j < N ? to_f(dy[r * ldy + n0 + j]) : 0.0f;
            }
            if constexpr (ACT != SFB_ACT_NONE) {
                if (vz) {
                    const Vec<__half, 8> q = *reinterpret_cast<const Vec<__half, 8> *>(z + r * ldz + n0);
#pragma unroll
                    for (int j = 0; j < 8; j++) d[j] = g[j] * slope<ACT>(to_f(q.v[j]));
                } else {
#pragma unroll
                    for (int j = 0; j < 8; j++) d[j] = n0 + j < N ? g[j] * slope<ACT>(to_f(z[r * ldz + n0 + j])) : 0.0f;
                }
            } else {
#pragma unroll
                for (int j = 0; j < 8; j++) d[j] = g[j];
            }
#pragma unroll
            for (int j = 0; j < 8; j++) acc[j] += d[j];
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
        }
    }
    if (sums) {
#pragma unroll
        for (int j = 0; j < 8; j++) s_sum[ty][tx * 8 + j] = acc[j];
        __syncthreads();
        const int64_t n = (int64_t)blockIdx.x * BC + threadIdx.x;
        if (n < N) {
            float v = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; i++) v += s_sum[i][threadIdx.x];
            sums[(int64_t)blockIdx.y * N + n] = v;
        }
    }
}

__global__ void __launch_bounds__(QT) sum_kernel(const float *__restrict__ sums, int64_t parts, int64_t N, void *db,
                                                 int dtype) {
    const int64_t n = (int64_t)blockIdx.x * QT + threadIdx.x;
    if (n >= N) return;
    float v = 0.0f;
    for (int64_t i = 0; i < parts; i++) v += sums[i * N + n];
    store_as(db, n, dtype, v);
}

bool is_float(int dtype) { return dtype == SFB_F32 || dtype == SFB_BF16 || dtype == SFB_F16; }

template <typename W>
int quantize_from(const W *w, int64_t N, int64_t K, int64_t ldw, int bits, int per_channel, void *codes, int64_t ldc,
                  int out, float *scale, uint32_t *amax, cudaStream_t st) {
    amax_kernel<W><<<(unsigned)N, QT, 0, st>>>(w, K, ldw, amax);
    if (out == SFB_I8)
        code_kernel<W, int8_t><<<(unsigned)N, QT, 0, st>>>(w, N, K, ldw, bits, amax, per_channel,
                                                           static_cast<int8_t *>(codes), ldc, scale);
    else if (out == SFB_BF16)
        code_kernel<W, __nv_bfloat16><<<(unsigned)N, QT, 0, st>>>(w, N, K, ldw, bits, amax, per_channel,
                                                                  static_cast<__nv_bfloat16 *>(codes), ldc, scale);
    else
        code_kernel<W, __half><<<(unsigned)N, QT, 0, st>>>(w, N, K, ldw, bits, amax, per_channel,
                                                           static_cast<__half *>(codes), ldc, scale);
    return check_launch("sfb_code_quantize");
}

}  // namespace
}  // namespace sfb

extern "C" int sfb_code_quantize(const void *w, int dtype, int64_t N, int64_t K, int64_t ldw, int bits,
                                 int per_channel, void *codes, int64_t ldc, int codes_dtype, float *scale, void *work,
                                 sfb_stream stream) {
    using namespace sfb;
    if (bits < 4 || bits > 8) return set_error(SFB_EINVAL, "sfb_code_quantize: width %d is not in 4..8", bits);
    if (!is_float(dtype)) return set_error(SFB_EINVAL, "sfb_code_quantize: element type %d", dtype);
    if (codes_dtype != SFB_I8 && codes_dtype != SFB_BF16 && codes_dtype != SFB_F16)
        return set_error(SFB_EINVAL, "sfb_code_quantize: codes of type %d", codes_dtype);
    if (N < 0 || K < 0 || ldw < K || ldc < K) return set_error(SFB_EINVAL, "sfb_code_quantize: bad shape");
    if (N >= (1ll << 31)) return set_error(SFB_ERANGE, "sfb_code_quantize: %lld rows", (long long)N);
    if (N == 0 || K == 0) return SFB_OK;
    if (!w || !codes || !scale || !work) return set_error(SFB_EINVAL, "sfb_code_quantize: null pointer");
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    uint32_t *amax = static_cast<uint32_t *>(work);
    if (dtype == SFB_F32)
        return quantize_from(static_cast<const float *>(w), N, K, ldw, bits, per_channel, codes, ldc, codes_dtype,
                             scale, amax, st);
    if (dtype == SFB_BF16)
        return quantize_from(static_cast<const __nv_bfloat16 *>(w), N, K, ldw, bits, per_channel, codes, ldc,
                             codes_dtype, scale, amax, st);
    return quantize_from(static_cast<const __half *>(w), N, K, ldw, bits, per_channel, codes, ldc, codes_dtype, scale,
                         amax, st);
}

extern "C" int sfb_code_expand(const int8_t *codes, int64_t N, int64_t K, int64_t ldc, void *out, int64_t ldo,
                               int dtype, sfb_stream stream) {
    using namespace sfb;
    if (dtype != SFB_BF16 && dtype != SFB_F16) return set_error(SFB_EINVAL, "sfb_code_expand: element type %d", dtype);
    if (N < 0 || K < 0 || ldc < K || ldo < K) return set_error(SFB_EINVAL, "sfb_code_expand: bad shape");
    if (N == 0 || K == 0) return SFB_OK;
    if (!codes || !out) return set_error(SFB_EINVAL, "sfb_code_expand: null pointer");
    if ((reinterpret_cast<uintptr_t>(out) & 15) || ldo % 8)
        return set_error(SFB_EINVAL, "sfb_code_expand: the rows of the result must be aligned to 16 bytes");
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const int64_t total = N * ((K + 15) / 16);
    const unsigned grid = (unsigned)std::min<int64_t>((total + QT - 1) / QT, 16ll * sm_count());
    const bool vec = ldc % 16 == 0 && (reinterpret_cast<uintptr_t>(codes) & 15) == 0;
    if (dtype == SFB_BF16)
        expand_kernel<<<grid, QT, 0, st>>>(codes, N, K, ldc, static_cast<__nv_bfloat16 *>(out), ldo, vec);
    else
        expand_kernel<<<grid, QT, 0, st>>>(codes, N, K, ldc, static_cast<__half *>(out), ldo, vec);
    return check_launch("sfb_code_expand");
}

extern "C" int64_t sfb_slope_workspace(int64_t M, int64_t N) { return 4 * ((M + sfb::BR - 1) / sfb::BR) * N; }

extern "C" int sfb_slope(int dtype, int act, const void *dy, int64_t ldy, const void *z, int64_t ldz, int64_t M,
                         int64_t N, const float *scale, int bits, const float *top, void *dz, void *dzs, int64_t ldd,
                         void *db, int db_dtype, void *work, sfb_stream stream) {
    using namespace sfb;
    if (dtype != SFB_BF16 && dtype != SFB_F16) return set_error(SFB_EINVAL, "sfb_slope: element type %d", dtype);
    if (bits < 4 || bits > 8) return set_error(SFB_EINVAL, "sfb_slope: width %d is not in 4..8", bits);
    if (M < 0 || N < 0 || ldy < N || (act != SFB_ACT_NONE && ldz < N) || ((dz || dzs) && (ldd < N || ldd % 8)))
        return set_error(SFB_EINVAL, "sfb_slope: bad shape");
    if ((reinterpret_cast<uintptr_t>(dz) | reinterpret_cast<uintptr_t>(dzs)) & 15)
        return set_error(SFB_EINVAL, "sfb_slope: the outputs must be aligned to 16 bytes");
    if (db && !is_float(db_dtype)) return set_error(SFB_EINVAL, "sfb_slope: bias type %d", db_dtype);
    if (N == 0) return SFB_OK;
    if ((M > 0 && (!dy || (act != SFB_ACT_NONE && !z))) || (dzs && !scale) || (db && M > 0 && !work))
        return set_error(SFB_EINVAL, "sfb_slope: null pointer");
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const int64_t parts = (M + BR - 1) / BR;
    if (parts > 65535) return set_error(SFB_ERANGE, "sfb_slope: %lld rows", (long long)M);
    float *sums = db ? static_cast<float *>(work) : nullptr;
    const float unit = 1.0f / (float)(1 << (bits - 1));
    if (M > 0) {
        const dim3 grid((unsigned)((N + BC - 1) / BC), (unsigned)parts);
        const int rc = with_activation(act, [&](auto a) {
            constexpr int A = decltype(a)::value;
            if (dtype == SFB_BF16)
                slope_kernel<__nv_bfloat16, A><<<grid, 256, 0, st>>>(
                    static_cast<const __nv_bfloat16 *>(dy), ldy, static_cast<const __half *>(z), ldz, M, N, scale,
                    unit, top, static_cast<__nv_bfloat16 *>(dz), static_cast<__nv_bfloat16 *>(dzs), ldd, sums);
            else
                slope_kernel<__half, A><<<grid, 256, 0, st>>>(
                    static_cast<const __half *>(dy), ldy, static_cast<const __half *>(z), ldz, M, N, scale, unit, top,
                    static_cast<__half *>(dz), static_cast<__half *>(dzs), ldd, sums);
            return check_launch("sfb_slope");
        });
        if (rc) return rc;
    }
    if (db) {
        sum_kernel<<<(unsigned)((N + QT - 1) / QT), QT, 0, st>>>(sums, parts, N, db, db_dtype);
        return check_launch("sfb_slope (bias)");
    }
    return SFB_OK;
}
