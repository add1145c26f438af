// The gated feed-forward product over sf codes: entry points, and the launches that the linear layer does not have.
//
//   h = act(g) u,  g = x Wg^T + bg,  u = x Wu^T + bu
//   dg = dh u act'(g),  du = dh act(g)
//   dx = dg Wg + du Wu,  dWg = dg^T x,  dWu = du^T x
//
// Both products of the forward pass are one (sfb_tensor_gemm.cu), over the codes of both weights, of which operand A has
// 16 rows of the one and 16 of the other in turn: x is read once, and act(g) u is made where both are in registers.
// (g and u as two layers: another write and read of M x N each, and the product as a third launch.)
// 4096 x 4096 by 2 x 8192 of bf16: 328 us, 1676 TFLOP/s, the tensor pipe 93 % busy; one row from packed codes of these
// sizes 20 us (two calls of the linear layer 22), 16 rows 26 (30).
// The backward pass is two products over both weights' channels together, [dg s | du s] times the codes and [dg | du]^T x.
#include <algorithm>

#include "sfb_tensor_parts.cuh"

namespace sfb {
namespace {

// --- packed codes in the activations' type ---------------------------------------------------------------------
// Both weights, 16 codes a thread; the rows between them zeros, and the scales of both side by side.

struct Packed {
    const int8_t *codes[2];
    const float *scale[2];
    int64_t ldc[2];
};

// VEC: rows of both start on 16 bytes and have a multiple of 16 codes
template <typename O, bool VEC>
__global__ void __launch_bounds__(256) gated_expand_kernel(const __grid_constant__ Packed p, int64_t N, int64_t Np, int64_t K,
                                                           O *__restrict__ out, int64_t ldo, float *__restrict__ scale, Rows rows) {
    const int y = blockIdx.z;
    if (y == 2) {                              // x's copy, in the launch that the call makes anyway
        pad_rows(rows, threadIdx.x, threadIdx.y, blockIdx.x, gridDim.x, blockIdx.y, gridDim.y);
        return;
    }
    const int8_t *codes = p.codes[y];
    const int64_t ldc = p.ldc[y];
    out += y * Np * ldo;
    scale += y * Np;
    for (int64_t n = (int64_t)blockIdx.y * 4 + threadIdx.y; n < Np; n += 4ll * gridDim.y) {
        if (blockIdx.x == 0 && threadIdx.x == 0) scale[n] = n < N ? p.scale[y][n] : 1.0f;
#pragma unroll 4
        for (int64_t k = ((int64_t)blockIdx.x * 64 + threadIdx.x) * 16; k < K; k += 1024ll * gridDim.x) {
            uint4 q = make_uint4(0, 0, 0, 0);
            if (n < N) {
                if constexpr (VEC) q = *reinterpret_cast<const uint4 *>(codes + n * ldc + k);
                else q = shift_codes(codes + n * ldc, k, K);
            }
            // (without conversions, which an SM makes at an eighth of the rate of sums: 43.5 us for 2 x 8192 x 4096, now 41)
            const uint32_t four[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
            for (int h = 0; h < 2; h++) {
                uint4 r;
                widen<O>(four[2 * h], r.x, r.y);
                widen<O>(four[2 * h + 1], r.z, r.w);
                if (k + 8 * h < K) *reinterpret_cast<uint4 *>(out + n * ldo + k + 8 * h) = r;   // a row's padding may be written
            }
        }
    }
}

// --- the gradients of both products ------------------------------------------------------------------------------
//
// dg and du, side by side (du Np columns on), once as they are (the operand of the weights' gradients) and once times the
// channel's scale (that of x's), each rounded once; g and u come in float32, as dg = dh u act'(g) has u's whole rounding:
// in fp16 a u of 11 bits would add to dz's and the result's rounding a third of the same size.
// Sums over the rows, for the biases, as the linear layer's: 64 rows a CTA, in a fixed order.
// Memory bound: 2 + 8 bytes a channel and row read, 4 or 8 written.  8192 x 5632 of fp16, 830 MB: 146 us, 5.7 TB/s.

constexpr int BR = 64, BC = 256;

template <bool VEC, typename T>
__device__ __forceinline__ void load8(const T *from, int64_t left, float (&v)[8]) {
    if constexpr (VEC) {
        constexpr int P = 16 / sizeof(T);
#pragma unroll
        for (int i = 0; i < 8 / P; i++) {
            const Vec<T, P> q = *reinterpret_cast<const Vec<T, P> *>(from + i * P);
#pragma unroll
            for (int j = 0; j < P; j++) v[i * P + j] = to_f(q.v[j]);
        }
    } else {
#pragma unroll
        for (int j = 0; j < 8; j++) v[j] = j < left ? to_f(from[j]) : 0.0f;
    }
}

template <typename T>
__device__ __forceinline__ void store8(T *to, const float (&v)[8]) {
    Vec<T, 8> q;
#pragma unroll
    for (int j = 0; j < 8; j++) q.v[j] = from_f<T>(v[j]);
    *reinterpret_cast<Vec<T, 8> *>(to) = q;
}

// VEC: N is a multiple of 8 and the rows of dh start on 16 bytes
template <typename T, int ACT, bool VEC>
__global__ void __launch_bounds__(256, 2)
gated_slope_kernel(const T *__restrict__ dh, int64_t ldh, const float *__restrict__ z, int64_t ldz, int64_t M, int64_t N,
                   int64_t Np, const float *__restrict__ scale, float unit, const float *__restrict__ top,
                   T *__restrict__ dz, T *__restrict__ dzs, int64_t ldd, float *__restrict__ sums) {
    __shared__ float s_sum[8][BC];
    const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
    const unsigned across = (unsigned)((Np + BC - 1) / BC);
    const int64_t by = blockIdx.x / across, bx = blockIdx.x % across;
    const int64_t n0 = bx * BC + tx * 8, left = N - n0;
    const int64_t r1 = min(M, (by + 1) * BR);
    float acc[2][8] = {}, f[2][8];
    if (dzs) {
        const float share = top ? __fdiv_rn(1.0f, *top) : unit;
#pragma unroll
        for (int h = 0; h < 2; h++)
#pragma unroll
            for (int j = 0; j < 8; j++) {
                f[h][j] = j < left ? scale[h * Np + n0 + j] * share : 0.0f;
                if (fabsf(f[h][j]) > 1.001f && top) f[h][j] = 1.0f;      // a channel without a code, larger than `top`
            }
    }
    if (n0 < Np) {
#pragma unroll 2
        for (int64_t r = by * BR + ty; r < r1; r += 8) {
            float d[8] = {}, g[8] = {}, u[8] = {};     // (columns between the two halves are zeros)
            if (VEC ? left > 0 : left >= 8) {
                load8<VEC>(dh + r * ldh + n0, left, d);
                load8<true>(z + r * ldz + n0, left, g);
                load8<true>(z + r * ldz + Np + n0, left, u);
            } else if (!VEC && left > 0) {
                load8<false>(dh + r * ldh + n0, left, d);
                load8<false>(z + r * ldz + n0, left, g);
                load8<false>(z + r * ldz + Np + n0, left, u);
            }
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const float a = activate<ACT>(g[j]), s = slope<ACT>(g[j]);
                g[j] = __fmul_rn(__fmul_rn(d[j], u[j]), s);
                u[j] = __fmul_rn(d[j], a);
                acc[0][j] += g[j];
                acc[1][j] += u[j];
            }
            if (dz) {
                store8(dz + r * ldd + n0, g);
                store8(dz + r * ldd + Np + n0, u);
            }
            if (dzs) {
#pragma unroll
                for (int j = 0; j < 8; j++) g[j] *= f[0][j], u[j] *= f[1][j];
                store8(dzs + r * ldd + n0, g);
                store8(dzs + r * ldd + Np + n0, u);
            }
        }
    }
    if (!sums) return;
#pragma unroll
    for (int h = 0; h < 2; h++) {
        __syncthreads();
#pragma unroll
        for (int j = 0; j < 8; j++) s_sum[ty][tx * 8 + j] = acc[h][j];
        __syncthreads();
        const int64_t n = bx * BC + threadIdx.x;
        if (n < Np) {
            float v = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; i++) v += s_sum[i][threadIdx.x];
            sums[(by * 2 + h) * Np + n] = v;
        }
    }
}

bool is_16(int64_t t) { return t == SFB_BF16 || t == SFB_F16; }
bool is_float(int64_t t) { return t == SFB_F32 || is_16(t); }
bool on16(const void *p, int64_t ld) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && ld % 8 == 0; }
int64_t padded(int64_t N) { return (N + 15) & ~15ll; }

int check(const sfb_gated_call *c, const char *what, bool codes) {
    if (!is_16(c->dtype)) return set_error(SFB_EINVAL, "%s: element type %d", what, (int)c->dtype);
    if (c->bits < 4 || c->bits > 8) return set_error(SFB_EINVAL, "%s: width %d is not in 4..8", what, (int)c->bits);
    if (c->act < SFB_ACT_NONE || c->act > SFB_ACT_SILU)
        return set_error(SFB_EINVAL, "%s: activation %d", what, (int)c->act);
    if (c->M < 0 || c->N < 1 || c->K < 1) return set_error(SFB_EINVAL, "%s: bad shape", what);
    // tile coordinates are 32-bit
    const int64_t most = (1ll << 31) - 512;
    if (c->M >= most || c->N >= most / 2 || c->K >= most || ((c->N + 63) / 64) * ((c->M + 127) / 128) >= most ||
        ((c->K + 255) / 256) * ((c->M + 127) / 128) >= most || ((c->K + 255) / 256) * ((c->N + 63) / 64) >= most)
        return set_error(SFB_ERANGE, "%s: a size of %lld x %lld x %lld", what, (long long)c->M, (long long)c->N, (long long)c->K);
    const uintptr_t w = size_of(c->w_dtype), g = size_of(c->gate_bias_dtype), u = size_of(c->up_bias_dtype);
    if (!lies_on(c->x, 2) || !lies_on(c->y, 2) || !lies_on(c->dx, 2) || !lies_on(c->gate, w) || !lies_on(c->up, w) ||
        !lies_on(c->dgate, w) || !lies_on(c->dup, w) || !lies_on(c->gate_bias, g) || !lies_on(c->dgate_bias, g) ||
        !lies_on(c->up_bias, u) || !lies_on(c->dup_bias, u) || !lies_on(c->gate_scale, 4) || !lies_on(c->up_scale, 4) ||
        !lies_on(c->scale, 4) || !lies_on(c->z, 4) || !lies_on(c->work, 4) || !lies_on(c->top, 4))
        return set_error(SFB_EINVAL, "%s: an operand does not start on an element", what);
    if (codes && (!c->codes || !on16(c->codes, c->ldc) || c->ldc < c->K || !c->scale))
        return set_error(SFB_EINVAL, "%s: the codes' rows must start on 16 bytes", what);
    return SFB_OK;
}

}  // namespace
}  // namespace sfb

extern "C" int sfb_gated_forward(const sfb_gated_call *c, sfb_stream stream) {
    using namespace sfb;
    const char *what = "sfb_gated_forward";
    if (!c) return set_error(SFB_EINVAL, "%s: null pointer", what);
    const bool packed = c->w_dtype == SFB_I8, small = packed && c->codes == nullptr;
    int rc = check(c, what, !small);
    if (rc) return rc;
    if (small && (c->M > SFB_SMALL_ROWS || c->z))
        return set_error(SFB_EINVAL, "%s: more than %d rows, or products to keep, and no room for the codes", what, SFB_SMALL_ROWS);
    if (!packed && !is_float(c->w_dtype)) return set_error(SFB_EINVAL, "%s: weight type %d", what, (int)c->w_dtype);
    const int64_t Np = padded(c->N);
    if (c->ldx < c->K || c->ldg < c->K || c->ldu < c->K || c->ldy < c->N || (c->z && c->ldz < 2 * Np))
        return set_error(SFB_EINVAL, "%s: a row stride is shorter than its row", what);
    if ((c->gate_bias && !is_float(c->gate_bias_dtype)) || (c->up_bias && !is_float(c->up_bias_dtype)))
        return set_error(SFB_EINVAL, "%s: a bias's type", what);
    if (!c->gate || !c->up || (packed && (!c->gate_scale || !c->up_scale)) || (!packed && !c->per_channel && !c->work) ||
        (c->M > 0 && (!c->x || !c->y)))
        return set_error(SFB_EINVAL, "%s: null pointer", what);
    const bool pad = c->M > 0 && !on16(c->x, c->ldx);
    if (pad && (!c->xpad || !on16(c->xpad, c->ldp) || c->ldp < c->K))
        return set_error(SFB_EINVAL, "%s: x does not start on 16 bytes and there is no room for a copy", what);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const int t = (int)c->dtype, bits = (int)c->bits, act = (int)c->act;
    const Rows rows{pad ? c->x : nullptr, c->M, c->K, c->ldx, c->xpad, c->ldp};
    if (!packed) {
        rc = tensor_quantize2(c->gate, c->ldg, c->up, c->ldu, (int)c->w_dtype, c->N, Np, c->K, bits, c->per_channel != 0,
                              c->codes, c->ldc, t, c->scale, c->work, rows, st);
    } else {
        if (small) {
            if (pad) rc = tensor_pad(rows, st);
        } else {
            auto on = [](const void *p, int64_t ld) { return ld % 16 == 0 && (reinterpret_cast<uintptr_t>(p) & 15) == 0; };
            const bool vec = c->K % 16 == 0 && on(c->gate, c->ldg) && on(c->up, c->ldu);
            const Packed p{{static_cast<const int8_t *>(c->gate), static_cast<const int8_t *>(c->up)},
                           {c->gate_scale, c->up_scale},
                           {c->ldg, c->ldu}};
            const int64_t room = 8ll * sm_count(), gy = std::min<int64_t>((Np + 3) / 4, 65535);
            const dim3 grid((unsigned)std::min<int64_t>((c->K + 1023) / 1024, std::max<int64_t>(1, room / gy)), (unsigned)gy, pad ? 3 : 2);
            auto go = [&](auto *kernel, auto type) {
                kernel<<<grid, dim3(64, 4), 0, st>>>(p, c->N, Np, c->K, static_cast<decltype(type) *>(c->codes), c->ldc, c->scale, rows);
            };
            if (t == SFB_BF16)
                vec ? go(gated_expand_kernel<__nv_bfloat16, true>, __nv_bfloat16()) : go(gated_expand_kernel<__nv_bfloat16, false>, __nv_bfloat16());
            else
                vec ? go(gated_expand_kernel<__half, true>, __half()) : go(gated_expand_kernel<__half, false>, __half());
            rc = check_launch("sf gated product (packed codes)");
        }
    }
    if (rc || c->M == 0) return rc;
    const void *x = pad ? c->xpad : c->x;
    const int64_t ldx = pad ? c->ldp : c->ldx;
    if (small)
        return tensor_gated_small(t, x, ldx, static_cast<const int8_t *>(c->gate), c->ldg, c->gate_scale,
                                  static_cast<const int8_t *>(c->up), c->ldu, c->up_scale, bits, c->gate_bias,
                                  (int)c->gate_bias_dtype, c->up_bias, (int)c->up_bias_dtype, act, c->y, c->ldy, c->M, c->N,
                                  c->K, st);
    return tensor_gated_product(t, x, ldx, c->codes, c->ldc, c->scale, bits, c->gate_bias, (int)c->gate_bias_dtype,
                                c->up_bias, (int)c->up_bias_dtype, act, c->y, c->ldy, c->z, c->ldz, c->M, c->N, Np, c->K, st);
}

extern "C" int64_t sfb_gated_sums(int64_t M, int64_t N) { return 8 * sfb::tensor_slope_parts(M) * sfb::padded(N); }

extern "C" int sfb_gated_backward(const sfb_gated_call *c, sfb_stream stream) {
    using namespace sfb;
    const char *what = "sfb_gated_backward";
    if (!c) return set_error(SFB_EINVAL, "%s: null pointer", what);
    int rc = check(c, what, true);
    if (rc) return rc;
    if (c->M == 0) return set_error(SFB_EINVAL, "%s: no rows", what);
    const int64_t Np = padded(c->N);
    if (c->ldx < c->K || c->ldy < c->N || c->ldz < 2 * Np || c->ldz % 4 || c->ldd < 2 * Np || c->ldd % 8)
        return set_error(SFB_EINVAL, "%s: a row stride is shorter than its row", what);
    if (!c->x || !c->y || !c->z || (reinterpret_cast<uintptr_t>(c->z) & 15)) return set_error(SFB_EINVAL, "%s: null pointer", what);
    if (!on16(c->x, c->ldx)) return set_error(SFB_EINVAL, "%s: x does not start on 16 bytes", what);
    const bool bias = c->dgate_bias || c->dup_bias, weight = c->dgate || c->dup;
    if ((bias && !c->work) || (c->dgate_bias && !is_float(c->gate_bias_dtype)) || (c->dup_bias && !is_float(c->up_bias_dtype)) ||
        (weight && !is_float(c->w_dtype)))
        return set_error(SFB_EINVAL, "%s: a gradient's type", what);
    if ((weight && (!c->dz || !on16(c->dz, 0))) || (c->dx && (!c->dzs || !on16(c->dzs, 0))))
        return set_error(SFB_EINVAL, "%s: no room for the products' gradients", what);
    const int size = c->w_dtype == SFB_F32 ? 4 : 2;
    const bool together = c->dgate && c->dup == static_cast<char *>(c->dgate) + Np * c->K * size;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const int t = (int)c->dtype, bits = (int)c->bits;
    // fp16: dz s would leave its range where the scales are small; s over the largest one with a code is within it
    const float *top = nullptr;
    if (c->dx && t == SFB_F16) {
        if (!c->top) return set_error(SFB_EINVAL, "%s: null pointer", what);
        top = c->top;
        rc = tensor_top(c->scale, 2 * Np, c->codes, c->ldc, c->K, c->top, st);
        if (rc) return rc;
    }
    float *parts = bias ? static_cast<float *>(c->work) : nullptr;
    const int64_t blocks = tensor_slope_parts(c->M) * ((Np + BC - 1) / BC);
    if (blocks >= 1ll << 31) return set_error(SFB_ERANGE, "%s: a gradient of %lld x %lld", what, (long long)c->M, (long long)c->N);
    if (weight || c->dx || bias) {
        const bool vec = c->N % 8 == 0 && on16(c->y, c->ldy);
        const float unit = 1.0f / (float)(1 << (bits - 1));
        rc = with_activation((int)c->act, [&](auto a) {
            constexpr int A = decltype(a)::value;
            auto go = [&](auto *kernel, auto type) {
                using T = decltype(type);
                kernel<<<(unsigned)blocks, 256, 0, st>>>(static_cast<const T *>(c->y), c->ldy, c->z, c->ldz, c->M, c->N, Np,
                                                         c->scale, unit, top, weight ? static_cast<T *>(c->dz) : nullptr,
                                                         c->dx ? static_cast<T *>(c->dzs) : nullptr, c->ldd, parts);
            };
            if (t == SFB_BF16)
                vec ? go(gated_slope_kernel<__nv_bfloat16, A, true>, __nv_bfloat16()) : go(gated_slope_kernel<__nv_bfloat16, A, false>, __nv_bfloat16());
            else
                vec ? go(gated_slope_kernel<__half, A, true>, __half()) : go(gated_slope_kernel<__half, A, false>, __half());
            return check_launch("sf gated product (its gradient)");
        });
        if (rc) return rc;
    }
    Sums sums{parts, tensor_slope_parts(c->M), 2 * Np, c->dgate_bias, (int)c->gate_bias_dtype, c->dup_bias, (int)c->up_bias_dtype, Np, c->N};
    if (c->dx) rc = tensor_grad_x(t, c->dzs, c->ldd, c->codes, c->ldc, top, bits, c->dx, c->K, c->M, 2 * Np, c->K, st);
    if (rc) return rc;
    if (together) return tensor_grad_w(t, c->dz, c->ldd, c->x, c->ldx, c->dgate, (int)c->w_dtype, c->K, c->M, 2 * Np, c->K, sums, st);
    if (c->dgate) {
        rc = tensor_grad_w(t, c->dz, c->ldd, c->x, c->ldx, c->dgate, (int)c->w_dtype, c->K, c->M, c->N, c->K, sums, st);
        sums.parts = nullptr;
    }
    if (!rc && c->dup) {
        rc = tensor_grad_w(t, static_cast<uint16_t *>(c->dz) + Np, c->ldd, c->x, c->ldx, c->dup, (int)c->w_dtype, c->K, c->M, c->N, c->K, sums, st);
        sums.parts = nullptr;
    }
    if (!rc && sums.parts) rc = tensor_sum(sums, st);
    return rc;
}
