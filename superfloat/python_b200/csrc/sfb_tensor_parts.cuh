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
};

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

// a matrix of 16-bit elements, and where it is copied with its rows on 16-byte boundaries
struct Rows {
    const void *x;                            // null: no copy
    int64_t M, K, ldx;
    void *out;
    int64_t ldo;
};

// codes and scales of a float weight (work: 4 N bytes, for one scale only), and in the same launch a copy of
// `rows`, if any
int tensor_quantize(const void *w, int dtype, int64_t N, int64_t K, int64_t ldw, int bits, bool per_channel, void *codes,
                    int64_t ldc, int codes_dtype, float *scale, void *work, const Rows &rows,
                    cudaStream_t st);
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
