// The launches that the tensor-core linear is made of.  Arguments are checked by
// its entry points (sfb_tensor.cu).
#pragma once

#include "sfb_tensor.cuh"

namespace sfb {

// The bias's gradient from its partial sums, a row of N for every 64 rows of dz, in
// 32 running sums, the same whoever computes it: an idle warp of the weight's
// product where that is wanted, else a kernel.  A pair of SMs has 8 warps' columns to
// a tile at most, and the 32 loads in flight take about a microsecond for every 2048 rows of
// dz, where a tile takes 8 us and more: it never waits for them.
struct Sums {
    const float *parts;                       // null: none wanted
    int64_t count, N;
    void *db;
    int dtype;
    // of a gated product: columns from `half` on are the second bias's, each of the two having `width`; else half is 0
    void *db2;
    int dtype2;
    int64_t half, width;
};

__device__ __forceinline__ void store_sum(const Sums &s, int64_t n, float v) {
    if (s.half == 0) store_as(s.db, n, s.dtype, v);
    else if (n < s.width && s.db) store_as(s.db, n, s.dtype, v);
    else if (n >= s.half && n - s.half < s.width && s.db2) store_as(s.db2, n - s.half, s.dtype2, v);
}

__device__ __forceinline__ float column_sum(const Sums &s, int64_t n) {
    float v[32] = {};
    for (int64_t i = 0; i < s.count; i += 32) {
        float q[32];                          // all asked for before the first is waited for
#pragma unroll
        for (int u = 0; u < 32; u++) q[u] = __ldg(s.parts + (i + u < s.count ? i + u : i) * s.N + n);
#pragma unroll
        for (int u = 0; u < 32; u++) v[u] += i + u < s.count ? q[u] : 0.0f;
    }
#pragma unroll
    for (int u = 1; u < 32; u++) v[0] += v[u];
    return v[0];
}

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

// 16 codes of a row from k on, those at or past K as 0, where rows do not start on 16 bytes: from the whole words around
// them, each holding at least one of the row's codes, shifted into place
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

// a matrix of 16-bit elements, and where it is copied with its rows on 16-byte boundaries
struct Rows {
    const void *x;                            // null: no copy
    int64_t M, K, ldx;
    void *out;
    int64_t ldo;
};

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

// codes and scales of a float weight (work: 4 N bytes, for one scale only), and in the same launch a copy of
// `rows`, if any
int tensor_quantize(const void *w, int dtype, int64_t N, int64_t K, int64_t ldw, int bits, bool per_channel, void *codes,
                    int64_t ldc, int codes_dtype, float *scale, void *work, const Rows &rows,
                    cudaStream_t st);
// the same of two weights of N rows, the second one's codes and scales Np rows on; rows between are zeros of scale 1
// (work: 8 N bytes)
int tensor_quantize2(const void *w, int64_t ldw, const void *w2, int64_t ldw2, int dtype, int64_t N, int64_t Np, int64_t K,
                     int bits, bool per_channel, void *codes, int64_t ldc, int codes_dtype, float *scale, void *work,
                     const Rows &rows, cudaStream_t st);
// packed codes as the products' operand, and in the same launch a copy of `rows`, if any
int tensor_expand(const int8_t *codes, int64_t N, int64_t K, int64_t ldc, void *out, int64_t ldo, int dtype,
                  const Rows &rows, cudaStream_t st);
int tensor_pad(const Rows &rows, cudaStream_t st);
int tensor_top(const float *scale, int64_t N, const void *codes, int64_t ldc, int64_t K, float *top, cudaStream_t st);
int tensor_small(int dtype, const void *x, int64_t ldx, const int8_t *codes, int64_t ldc, const float *scale, int bits,
                 const void *bias, int bias_dtype, int act, const void *residual, int64_t ldr, void *y, int64_t ldy,
                 int64_t M, int64_t N, int64_t K, cudaStream_t st);
int tensor_product(int dtype, const void *x, int64_t ldx, const void *codes, int64_t ldw, const float *scale, int bits,
                   const void *bias, int bias_dtype, int act, const void *residual, int64_t ldr, void *y, int64_t ldy,
                   void *z, int64_t ldz, int64_t M, int64_t N, int64_t K, cudaStream_t st);
// act(gate) up of the two products, codes (2 Np rows) as tensor_quantize2 leaves them; z (nullable): both products, 2 Np float32 a row
int tensor_gated_product(int dtype, const void *x, int64_t ldx, const void *codes, int64_t ldw, const float *scale, int bits,
                         const void *bias, int bias_dtype, const void *bias2, int bias2_dtype, int act, void *y, int64_t ldy,
                         float *z, int64_t ldz, int64_t M, int64_t N, int64_t Np, int64_t K, cudaStream_t st);
int tensor_gated_small(int dtype, const void *x, int64_t ldx, const int8_t *gate, int64_t ldg, const float *gate_scale,
                       const int8_t *up, int64_t ldu, const float *up_scale, int bits, const void *bias, int bias_dtype,
                       const void *bias2, int bias2_dtype, int act, void *y, int64_t ldy, int64_t M, int64_t N, int64_t K,
                       cudaStream_t st);
int64_t tensor_slope_parts(int64_t M);          // rows of partial sums
int tensor_slope(int dtype, int act, const void *dy, int64_t ldy, const void *z, int64_t ldz, int64_t M, int64_t N,
                 const float *scale, int bits, const float *top, void *dz, void *dzs, int64_t ldd, float *sums,
                 cudaStream_t st);
int tensor_sum(const Sums &sums, cudaStream_t st);
// the products of the backward pass; the weight's adds `sums` up beside its own
int tensor_grad_x(int dtype, const void *dzs, int64_t ldd, const void *codes, int64_t ldw, const float *top, int bits,
                  void *dx, int64_t ldx, int64_t M, int64_t N, int64_t K, cudaStream_t st);
int tensor_grad_w(int dtype, const void *dz, int64_t ldd, const void *x, int64_t ldx, void *dw, int dw_dtype,
                  int64_t ldw, int64_t M, int64_t N, int64_t K, const Sums &sums, cudaStream_t st);

}  // namespace sfb
