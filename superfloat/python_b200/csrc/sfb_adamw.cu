// The AdamW step over many tensors at once, moments in float32 or in sf8.
//
//   p <- p (1 - lr wd) - lr / bc1 * m / (sqrt(v) / sqrt(bc2) + eps)
//   m <- b1 m + (1 - b1) g,   v <- b2 v + (1 - b2) g^2,   bc_i = 1 - b_i^step
//
// all in float32 whatever the type of p and g; p is rounded once (to nearest)
// when it is stored in 16 bits.
//
// sf8 moments.  Blocks of 256 elements share one float32 scale s, the block's
// largest magnitude.  A code c in [-127, 127] stands for s (c / 127)^2 with c's
// sign (first moment) or s (c / 127)^4 (second): equal steps in sqrt|m| and in
// v^(1/4), so that 127 levels span a range of 1.6e4 in m and in sqrt v, where
// equal steps in the moment itself would set everything below 1/254 of the
// block's largest to zero.  A new moment is rounded to one of its two levels by a dither, the upper
// with the probability that keeps the VALUE unbiased: with rounding to nearest a
// moment that changes by less than half a step per call (v does: 1 - b2 = 0.001)
// would never move.  A second moment above zero keeps a code of at least one, or
// the quotient would divide by eps alone.  A block whose largest moment is below
// 1e-30 is held as zero.  A moment that is not finite makes the block's scale
// infinite or NaN; every moment of the block then reads as that or as NaN, and as NaN
// after the next step.
// The codes depend on the last bits of m and v, so each float32 operation on the
// way to a code is one IEEE rounding (the __f*_rn forms are not contracted to fma).
//
// One launch takes a table of tensors as its parameter (no table in device
// memory: nothing to copy, and nothing that two captured graphs could share).
// A CTA takes one chunk of one tensor, found by bisection over the chunk counts.
// Float32 moments: bound by memory, 28 bytes an element with float32 p and g, 6430
// GB/s for 46.5 M elements (202 us).  sf8 moments: 16.06 bytes an element with float32
// p and g, 10.06 with 16-bit ones, against about 85 instructions of arithmetic: 133
// us for 46.5 M float32 elements (5600 GB/s), 318 us for 117 M of bf16 (3700 GB/s,
// bound by instruction issue).
#include <math.h>

#include <algorithm>
#include <exception>
#include <vector>

#include "sfb_tensor.cuh"

namespace sfb {
namespace {

constexpr int AT = 128;                       // threads of a CTA: 8 of them an SM were faster than 4 of 256 (136 against 155 us)
constexpr int AB = 256;                       // elements of one sf8 block
// elements of one CTA: sf8 blocks in turn to its warps
template <bool SF8> constexpr int CHUNK = SF8 ? 8192 : 4096;
constexpr float UNIT2 = (float)(1.0 / 16129.0), UNIT4 = (float)(1.0 / 260144641.0);
constexpr float TOP2 = 16129.0f, TOP4 = 260144641.0f;

struct Coefs {
    float shrink, size, root, eps, b1, a1, b2, a2;     // a_i = 1 - b_i
    uint32_t dither;
};

struct Entry {
    void *p;
    const void *g;
    void *m, *v;
    float *ms, *vs;
    int64_t n;
    uint32_t seed;                            // of the dither, less the call's
    uint32_t vec;                             // all are aligned for vectors of four (sf8: eight) elements
};

template <int CAP>
struct Table {
    int count;
    uint32_t start[CAP + 1];                  // first chunk of each tensor
    Entry e[CAP];
};

// elements i .. i + 3 (those below n) as float
template <typename T>
__device__ __forceinline__ void load4(const T *x, int64_t i, int64_t n, bool vec, float (&r)[4]) {
    if (vec && i + 4 <= n) {
        const Vec<T, 4> q = *reinterpret_cast<const Vec<T, 4> *>(x + i);
#pragma unroll
        for (int j = 0; j < 4; j++) r[j] = to_f(q.v[j]);
    } else {
#pragma unroll
        for (int j = 0; j < 4; j++) r[j] = i + j < n ? to_f(x[i + j]) : 0.0f;
    }
}

template <typename T>
__device__ __forceinline__ void store4(T *x, int64_t i, int64_t n, bool vec, const float (&r)[4]) {
    if (vec && i + 4 <= n) {
        Vec<T, 4> q;
#pragma unroll
        for (int j = 0; j < 4; j++) q.v[j] = from_f<T>(r[j]);
        *reinterpret_cast<Vec<T, 4> *>(x + i) = q;
    } else {
#pragma unroll
        for (int j = 0; j < 4; j++)
            if (i + j < n) x[i + j] = from_f<T>(r[j]);
    }
}

__device__ __forceinline__ float sqrt_fast(float x) {
    float r;
    asm("sqrt.approx.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

__device__ __forceinline__ float stepped(float p, float m, float v, const Coefs &c) {
    return p * c.shrink - c.size * __fdividef(m, fmaf(sqrt_fast(v), c.root, c.eps));
}

__device__ __forceinline__ void moments(float &m, float &v, float g, const Coefs &c) {
    m = __fadd_rn(__fmul_rn(m, c.b1), __fmul_rn(g, c.a1));
    v = __fadd_rn(__fmul_rn(v, c.b2), __fmul_rn(__fmul_rn(g, c.a2), g));
}

// 32 mixed bits of a counter: two rounds of multiply and xor-shift, with the shifts and
// multipliers of Chris Wellons' published search for integer hashes of least bias.  A
// seed is a place in the counter's sequence: two seeds give the same draws, shifted.
__device__ __forceinline__ uint32_t mixed(uint32_t i, uint32_t seed) {
    uint32_t h = i * 0x9E3779B1u + seed;
    h ^= h >> 16;
    h *= 0x7FEB352Du;
    h ^= h >> 15;
    h *= 0x846CA68Bu;
    h ^= h >> 16;
    return h;
}

// Two elements at a time: one instruction for both, each result rounded as the
// scalar operation's.  Unlike the scalar forms, a mul2 whose result is added may be
// contracted with the addition: products that are summed are scalar (`once`).
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
    float2 r;
    asm("{\n\t.reg .b64 x, y;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmul.rn.f32x2 x, x, y;\n\t"
        "mov.b64 {%0, %1}, x;\n\t}"
        : "=f"(r.x), "=f"(r.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return r;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    float2 r;
    asm("{\n\t.reg .b64 x, y;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tadd.rn.f32x2 x, x, y;\n\t"
        "mov.b64 {%0, %1}, x;\n\t}"
        : "=f"(r.x), "=f"(r.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return r;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    float2 r;
    asm("{\n\t.reg .b64 x, y, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmov.b64 z, {%6, %7};\n\t"
        "fma.rn.f32x2 x, x, y, z;\n\tmov.b64 {%0, %1}, x;\n\t}"
        : "=f"(r.x), "=f"(r.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return r;
}
__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }
// a - b: b (-1) + a, the product exact
__device__ __forceinline__ float2 sub2(float2 a, float2 b) { return fma2(b, both(-1.0f), a); }

__device__ __forceinline__ float2 once(float2 a, float2 b) { return make_float2(__fmul_rn(a.x, b.x), __fmul_rn(a.y, b.y)); }

// 1 where a < b, else 0
__device__ __forceinline__ float less(float a, float b) {
    float r;
    asm("set.lt.f32.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float2 less2(float2 a, float2 b) { return make_float2(less(a.x, b.x), less(a.y, b.y)); }

__device__ __forceinline__ float root_ftz(float x) {
    float r;
    asm("sqrt.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

__device__ __forceinline__ float top_nan(float a, float b) {           // NaN above all
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

template <int POWER>
__device__ __forceinline__ float2 level(float2 c) {
    const float2 c2 = mul2(c, c);
    return POWER == 2 ? c2 : mul2(c2, c2);
}

// the level of c + 1, its last product not to be contracted
template <int POWER>
__device__ __forceinline__ float2 above(float2 c) {
    const float2 d = add2(c, both(1.0f)), d2 = mul2(d, d);
    return POWER == 2 ? once(d, d) : once(d2, d2);
}

// Conversions between integers and floats share a unit of 16 lanes with the square
// roots, and ten of them an element made the kernel wait for it (281 us for 46.5 M
// float32 elements; 199 without them, 136 with two elements to an instruction).  Adding 2^23 to a float in [0, 2^23) leaves the nearest
// integer in its low bits, and putting an integer there and subtracting is the way back.
constexpr float MAGIC = 8388608.0f;

// bytes J and J + 1 of a word of codes, exactly
template <int J>
__device__ __forceinline__ float2 code_values(uint32_t biased) {        // each byte c + 128
    return add2(make_float2(__uint_as_float(__byte_perm(biased, 0x4B000000u, 0x7650 | J)),
                            __uint_as_float(__byte_perm(biased, 0x4B000000u, 0x7650 | (J + 1)))),
                both(-MAGIC - 128.0f));
}

// The codes of t = |value| * top / s as floats in [0, 127]: the largest c with
// level(c) <= t, or the next one by the dither u.  `root` is t^(1/POWER) to within a few
// units, so its nearest integer is that c or one more.  Where t is not finite the
// code is any: the scale tells.
template <int POWER>
__device__ __forceinline__ float2 codes_of(float2 t, float2 root, float2 u) {
    float2 c = add2(add2(root, both(MAGIC)), both(-MAGIC));
    c = sub2(c, less2(t, level<POWER>(c)));
    const float2 low = POWER == 2 ? once(c, c) : once(mul2(c, c), mul2(c, c));
    // the step to the next level: 2 c + 1 of the squares, exactly
    const float2 wide = POWER == 2 ? fma2(c, both(2.0f), both(1.0f)) : sub2(above<POWER>(c), low);
    c = add2(c, less2(mul2(u, wide), sub2(t, low)));
    c.x = fminf(c.x, 127.0f);
    c.y = fminf(c.y, 127.0f);
    if (POWER == 4) {
        if (t.x > 0.0f) c.x = fmaxf(c.x, 1.0f);
        if (t.y > 0.0f) c.y = fmaxf(c.y, 1.0f);
    }
    return c;
}

__device__ __forceinline__ float scale_of(uint32_t bits) {
    const float s = __uint_as_float(bits);
    return s < 1e-30f ? 0.0f : s;
}

// the low bytes of four floats c + 1.5 2^23
__device__ __forceinline__ uint32_t bytes_of(const float (&c)[4]) {
    const float m = 1.5f * MAGIC;
    const uint32_t a = __byte_perm(__float_as_uint(__fadd_rn(c[0], m)), __float_as_uint(__fadd_rn(c[1], m)), 0x0040);
    const uint32_t b = __byte_perm(__float_as_uint(__fadd_rn(c[2], m)), __float_as_uint(__fadd_rn(c[3], m)), 0x0040);
    return __byte_perm(a, b, 0x5410);
}

// A block of 256 elements by one warp: lane l has elements 8 l .. 8 l + 7, one access
// an array.  (With four elements an access, 16 accesses a lane and block for 9, 117 M
// elements of bf16 took 328 us, now 318.  Loading the next block under this one's arithmetic
// was slower, too: its registers cost warps.)
template <typename T>
struct Loaded {
    Vec<T, 8> p, g;
    uint2 cm, cv;
    float sm, sv;
};

template <typename T>
__device__ __forceinline__ void load_block(const Entry &e, int64_t blk, int lane, Loaded<T> &q) {
    const int64_t i = blk * AB + lane * 8;
    const T *p = static_cast<const T *>(e.p) + i, *g = static_cast<const T *>(e.g) + i;
    const uint8_t *mc = static_cast<const uint8_t *>(e.m) + i, *vc = static_cast<const uint8_t *>(e.v) + i;
    q.sm = e.ms[blk];
    q.sv = e.vs[blk];
    if (blk * AB + AB <= e.n && e.vec) {
        q.g = *reinterpret_cast<const Vec<T, 8> *>(g);
        q.cm = *reinterpret_cast<const uint2 *>(mc);
        q.cv = *reinterpret_cast<const uint2 *>(vc);
        q.p = *reinterpret_cast<const Vec<T, 8> *>(p);
        return;
    }
    uint32_t a[2] = {0, 0}, b[2] = {0, 0};
#pragma unroll
    for (int j = 0; j < 8; j++) {
        const bool in = i + j < e.n;
        q.g.v[j] = in ? g[j] : from_f<T>(0.0f);
        q.p.v[j] = in ? p[j] : from_f<T>(0.0f);
        if (in) {
            a[j / 4] |= (uint32_t)mc[j] << (8 * (j % 4));
            b[j / 4] |= (uint32_t)vc[j] << (8 * (j % 4));
        }
    }
    q.cm = make_uint2(a[0], a[1]);
    q.cv = make_uint2(b[0], b[1]);
}

template <typename T>
__device__ __forceinline__ void block_sf8(const Entry &e, int64_t blk, const Coefs &c, int lane, const Loaded<T> &q) {
    const int64_t i = blk * AB + lane * 8;
    T *p = static_cast<T *>(e.p) + i;
    uint8_t *mc = static_cast<uint8_t *>(e.m) + i, *vc = static_cast<uint8_t *>(e.v) + i;
    const bool vec = blk * AB + AB <= e.n && e.vec;
    const uint32_t cm[2] = {q.cm.x, q.cm.y}, cv[2] = {q.cv.x, q.cv.y};
    const float sm = q.sm, sv = q.sv;
    float P[8], G[8];
    float2 M[4], V[4], S[4];                        // pairs of elements
#pragma unroll
    for (int j = 0; j < 8; j++) {
        P[j] = to_f(q.p.v[j]);
        G[j] = to_f(q.g.v[j]);
    }
    const float um = __fmul_rn(sm, UNIT2), uv = __fmul_rn(sv, UNIT4);
    float tm = 0.0f, tv = 0.0f;
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const uint32_t a = cm[j / 2] ^ 0x80808080u, b = cv[j / 2] ^ 0x80808080u;
        const float2 x = j % 2 ? code_values<2>(a) : code_values<0>(a), y = j % 2 ? code_values<2>(b) : code_values<0>(b);
        const float2 gg = make_float2(G[2 * j], G[2 * j + 1]);
        const float2 m0 = mul2(mul2(x, make_float2(fabsf(x.x), fabsf(x.y))), both(um)), v0 = mul2(level<4>(y), both(uv));
        M[j] = add2(once(m0, both(c.b1)), once(gg, both(c.a1)));
        V[j] = add2(once(v0, both(c.b2)), once(mul2(gg, both(c.a2)), gg));
        tm = top_nan(tm, top_nan(fabsf(M[j].x), fabsf(M[j].y)));
        tv = top_nan(tv, top_nan(V[j].x, V[j].y));
        // (2^-126 more, so that a v below float32's normal range is not taken for 0; its root is far below any eps)
        const float2 vv = add2(V[j], both(0x1p-126f));
        S[j] = make_float2(root_ftz(vv.x), root_ftz(vv.y));
        const float2 d = fma2(S[j], both(c.root), both(c.eps));
        const float2 by = mul2(M[j], make_float2(rcp_fast(d.x), rcp_fast(d.y)));
        const float2 r = fma2(by, both(-c.size), mul2(make_float2(P[2 * j], P[2 * j + 1]), both(c.shrink)));
        P[2 * j] = r.x;
        P[2 * j + 1] = r.y;
    }
    if (vec) {
        Vec<T, 8> r;
#pragma unroll
        for (int j = 0; j < 8; j++) r.v[j] = from_f<T>(P[j]);
        *reinterpret_cast<Vec<T, 8> *>(p) = r;
    } else {
#pragma unroll
        for (int j = 0; j < 8; j++)
            if (i + j < e.n) p[j] = from_f<T>(P[j]);
    }
    // magnitudes order as their bits, NaN above all
    const float sm1 = scale_of(__reduce_max_sync(0xffffffffu, __float_as_uint(tm) & 0x7FFFFFFFu));
    const float sv1 = scale_of(__reduce_max_sync(0xffffffffu, __float_as_uint(tv) & 0x7FFFFFFFu));
    const float im = sm1 != 0.0f ? __fdiv_rn(TOP2, sm1) : 0.0f, iv = sv1 != 0.0f ? __fdiv_rn(TOP4, sv1) : 0.0f;
    const float siv = sqrt_fast(iv);
    if (lane == 0) {
        e.ms[blk] = sm1;
        e.vs[blk] = sv1;
    }
    const uint32_t seed = e.seed + c.dither, i0 = (uint32_t)i;
    uint32_t xs[2], ys[2];
#pragma unroll
    for (int h = 0; h < 2; h++) {
        float a[4], b[4];
#pragma unroll
        for (int k = 0; k < 2; k++) {
            const int j = 2 * h + k;
            const uint32_t r0 = mixed(i0 + 2 * j, seed), r1 = mixed(i0 + 2 * j + 1, seed);
            // a 16-bit number u under 2^23 as a float, then (2^23 + u) 2^-16 - 2^7 = u 2^-16 exactly
            const float2 lo = fma2(make_float2(__uint_as_float(__byte_perm(r0, 0x4B000000u, 0x7610)),
                                               __uint_as_float(__byte_perm(r1, 0x4B000000u, 0x7610))),
                                   both(0x1p-16f), both(-128.0f));
            const float2 hi = fma2(make_float2(__uint_as_float(__byte_perm(r0, 0x4B000000u, 0x7632)),
                                               __uint_as_float(__byte_perm(r1, 0x4B000000u, 0x7632))),
                                   both(0x1p-16f), both(-128.0f));
            const float2 t = mul2(make_float2(fabsf(M[j].x), fabsf(M[j].y)), both(im)), tq = mul2(V[j], both(iv));
            const float2 rq = mul2(S[j], both(siv));
            const float2 x = codes_of<2>(t, make_float2(root_ftz(t.x), root_ftz(t.y)), lo);
            const float2 y = codes_of<4>(tq, make_float2(root_ftz(rq.x), root_ftz(rq.y)), hi);
            a[2 * k] = copysignf(x.x, M[j].x);
            a[2 * k + 1] = copysignf(x.y, M[j].y);
            b[2 * k] = y.x;
            b[2 * k + 1] = y.y;
        }
        xs[h] = bytes_of(a);
        ys[h] = bytes_of(b);
    }
    if (vec) {
        *reinterpret_cast<uint2 *>(mc) = make_uint2(xs[0], xs[1]);
        *reinterpret_cast<uint2 *>(vc) = make_uint2(ys[0], ys[1]);
    } else {
#pragma unroll
        for (int j = 0; j < 8; j++)
            if (i + j < e.n) {
                mc[j] = (uint8_t)(xs[j / 4] >> (8 * (j % 4)));
                vc[j] = (uint8_t)(ys[j / 4] >> (8 * (j % 4)));
            }
    }
}

template <typename T>
__device__ __forceinline__ void four_f32(const Entry &e, int64_t i, const Coefs &c) {
    T *p = static_cast<T *>(e.p);
    const T *g = static_cast<const T *>(e.g);
    float *m = static_cast<float *>(e.m), *v = static_cast<float *>(e.v);
    float P[4], G[4], M[4], V[4];
    load4(g, i, e.n, e.vec, G);
    load4(m, i, e.n, e.vec, M);
    load4(v, i, e.n, e.vec, V);
    load4(p, i, e.n, e.vec, P);
#pragma unroll
    for (int j = 0; j < 4; j++) {
        moments(M[j], V[j], G[j], c);
        P[j] = stepped(P[j], M[j], V[j], c);
    }
    store4(m, i, e.n, e.vec, M);
    store4(v, i, e.n, e.vec, V);
    store4(p, i, e.n, e.vec, P);
}

template <int CAP>
__device__ __forceinline__ int tensor_of(const Table<CAP> &t, uint32_t chunk) {
    int lo = 0, hi = t.count;
    while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (t.start[mid] <= chunk) lo = mid;
        else hi = mid;
    }
    return lo;
}

template <typename T, bool SF8, int CAP>
__global__ void __launch_bounds__(AT, SF8 ? 8 : 12) adamw_kernel(const __grid_constant__ Table<CAP> t, Coefs given,
                                                   const Coefs *__restrict__ on_device) {
    const int k = tensor_of(t, blockIdx.x);
    const Entry &e = t.e[k];
    const Coefs c = on_device ? *on_device : given;
    const int64_t first = (int64_t)(blockIdx.x - t.start[k]) * CHUNK<SF8>, last = min(e.n, first + CHUNK<SF8>);
    if constexpr (SF8) {
        const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
#pragma unroll 1
        for (int64_t b = first / AB + warp; b * AB < last; b += AT / 32) {
            Loaded<T> q;
            load_block(e, b, lane, q);
            block_sf8<T>(e, b, c, lane, q);
        }
    } else {
#pragma unroll 2
        for (int64_t i = first + 4 * threadIdx.x; i < last; i += 4 * AT) four_f32<T>(e, i, c);
    }
}

Coefs coefs_of(double lr, double b1, double b2, double eps, double wd, int64_t step, uint32_t dither) {
    Coefs c;
    c.shrink = (float)(1.0 - lr * wd);
    c.size = (float)(lr / (1.0 - pow(b1, (double)step)));
    c.root = (float)(1.0 / sqrt(1.0 - pow(b2, (double)step)));
    c.eps = (float)eps;
    c.b1 = (float)b1;
    c.a1 = (float)(1.0 - b1);
    c.b2 = (float)b2;
    c.a2 = (float)(1.0 - b2);
    c.dither = dither;
    return c;
}

// the step counter and the constants of a captured step, in device memory
__global__ void advance_kernel(long long *step, Coefs *out, double lr, double b1, double b2, double eps, double wd,
                               uint32_t seed) {
    const long long t = ++*step;
    Coefs c;
    c.shrink = (float)(1.0 - lr * wd);
    c.size = (float)(lr / (1.0 - pow(b1, (double)t)));
    c.root = (float)(1.0 / sqrt(1.0 - pow(b2, (double)t)));
    c.eps = (float)eps;
    c.b1 = (float)b1;
    c.a1 = (float)(1.0 - b1);
    c.b2 = (float)b2;
    c.a2 = (float)(1.0 - b2);
    c.dither = seed + (uint32_t)t;
    *out = c;
}

// the values of four sf8 codes
__device__ __forceinline__ void four_values(const char4 &x, float s, int power, float (&r)[4]) {
    const float u = __fmul_rn(s, power == 2 ? UNIT2 : UNIT4);
    const int q[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const float y = (float)(q[j] * q[j]), l = power == 2 ? y : __fmul_rn(y, y);
        r[j] = __fmul_rn(q[j] < 0 ? -l : l, u);
    }
}

// the values that sf8 codes stand for: a whole chunk's loads are asked for before the
// first store, which the compiler cannot do by itself as the two could overlap
// (117 M codes in 91.5 us, 6410 GB/s; 106.6 us in its order)
template <int CAP>
__global__ void __launch_bounds__(AT) values_kernel(const __grid_constant__ Table<CAP> t, int power) {
    constexpr int SIZE = CHUNK<false>, STEPS = SIZE / (4 * AT);
    const int k = tensor_of(t, blockIdx.x);
    const Entry &e = t.e[k];
    const int64_t first = (int64_t)(blockIdx.x - t.start[k]) * SIZE, last = min(e.n, first + SIZE);
    const int8_t *code = static_cast<const int8_t *>(e.g);
    float *out = static_cast<float *>(e.p);
    if (first + SIZE <= e.n) {
        char4 x[STEPS];
        float s[STEPS];
#pragma unroll
        for (int i = 0; i < STEPS; i++) {
            const int64_t at = first + 4 * (threadIdx.x + AT * i);
            x[i] = __ldcs(reinterpret_cast<const char4 *>(code + at));
            s[i] = __ldg(e.ms + at / AB);
        }
#pragma unroll
        for (int i = 0; i < STEPS; i++) {
            float r[4];
            four_values(x[i], s[i], power, r);
            store4(out, first + 4 * (threadIdx.x + AT * i), last, true, r);
        }
        return;
    }
    for (int64_t i = first + 4 * threadIdx.x; i < last; i += 4 * AT) {
        char4 x = make_char4(0, 0, 0, 0);
        if (i + 4 <= last) {
            x = *reinterpret_cast<const char4 *>(code + i);
        } else {
            x.x = code[i];
            if (i + 1 < last) x.y = code[i + 1];
            if (i + 2 < last) x.z = code[i + 2];
        }
        float r[4];
        four_values(x, e.ms[i / AB], power, r);
        store4(out, i, last, true, r);
    }
}

constexpr int WORDS = 8;                      // of one table entry as the caller gives it
constexpr int MAX_CAP = 448;

template <int CAP, bool SF8, typename F>
int each_table(const int64_t *rows, int count, F launch) {
    // one launch for every CAP tensors, or sooner where the grid would pass 2^30 chunks
    Table<CAP> t;
    int at = 0;
    while (at < count) {
        t.count = 0;
        uint64_t chunks = 0;
        for (; at < count && t.count < CAP; at++) {
            const int64_t *r = rows + (int64_t)at * WORDS;
            const int64_t n = r[6];
            if (n == 0) continue;
            const uint64_t need = (uint64_t)((n + CHUNK<SF8> - 1) / CHUNK<SF8>);
            if (need > (1u << 30)) return set_error(SFB_ERANGE, "sfb_adamw: a tensor of %lld elements", (long long)n);
            if (chunks + need > (1u << 30)) break;
            Entry &e = t.e[t.count];
            e.p = reinterpret_cast<void *>(r[0]);
            e.g = reinterpret_cast<const void *>(r[1]);
            e.m = reinterpret_cast<void *>(r[2]);
            e.v = reinterpret_cast<void *>(r[3]);
            e.ms = reinterpret_cast<float *>(r[4]);
            e.vs = reinterpret_cast<float *>(r[5]);
            e.n = n;
            e.seed = (uint32_t)r[7];
            e.vec = 0;
            t.start[t.count++] = (uint32_t)chunks;
            chunks += need;
        }
        t.start[t.count] = (uint32_t)chunks;
        if (t.count == 0) break;
        const int rc = launch(t, (unsigned)chunks);
        if (rc) return rc;
    }
    return SFB_OK;
}

// writes to memory that another entry of the call writes or reads would race
int check_overlap(const int64_t *rows, int count, int size, bool sf8) {
    struct Span {
        int64_t lo, hi;
        bool written;
    };
    std::vector<Span> s;
    s.reserve((size_t)count * 6);
    for (int i = 0; i < count; i++) {
        const int64_t *r = rows + (int64_t)i * WORDS, n = r[6];
        if (n <= 0) continue;
        const int64_t state = n * (sf8 ? 1 : 4), scales = 4 * ((n + AB - 1) / AB);
        s.push_back({r[0], r[0] + n * size, true});
        s.push_back({r[1], r[1] + n * size, false});
        s.push_back({r[2], r[2] + state, true});
        s.push_back({r[3], r[3] + state, true});
        if (sf8) {
            s.push_back({r[4], r[4] + scales, true});
            s.push_back({r[5], r[5] + scales, true});
        }
    }
    std::sort(s.begin(), s.end(), [](const Span &a, const Span &b) { return a.lo < b.lo; });
    int64_t end = INT64_MIN, written_end = INT64_MIN;   // of all spans so far, of the written ones
    for (const Span &x : s) {
        if (x.lo < (x.written ? end : written_end))
            return set_error(SFB_EINVAL, "sfb_adamw: a tensor is given twice, or overlaps one that the step writes");
        end = std::max(end, x.hi);
        if (x.written) written_end = std::max(written_end, x.hi);
    }
    return SFB_OK;
}

template <typename T, bool SF8, int CAP>
int run_adamw(const int64_t *rows, int count, const Coefs &c, const Coefs *dev, cudaStream_t st) {
    return each_table<CAP, SF8>(rows, count, [&](Table<CAP> &t, unsigned grid) {
        for (int i = 0; i < t.count; i++) {
            Entry &e = t.e[i];
            const uintptr_t a = reinterpret_cast<uintptr_t>(e.p) | reinterpret_cast<uintptr_t>(e.g);
            const uintptr_t b = reinterpret_cast<uintptr_t>(e.m) | reinterpret_cast<uintptr_t>(e.v);
            // float32 moments: four elements an access; sf8: eight
            e.vec = (a & ((SF8 ? 8 : 4) * sizeof(T) - 1)) == 0 && (b & (SF8 ? 7 : 15)) == 0;
        }
        adamw_kernel<T, SF8, CAP><<<grid, AT, 0, st>>>(t, c, dev);
        return check_launch("sfb_adamw");
    });
}

template <typename T>
int run_typed(const int64_t *rows, int count, bool sf8, const Coefs &c, const Coefs *dev, cudaStream_t st) {
    // the table is the launch's parameter: a short one costs less to send
    if (sf8)
        return count <= 16 ? run_adamw<T, true, 16>(rows, count, c, dev, st)
               : count <= 96 ? run_adamw<T, true, 96>(rows, count, c, dev, st)
                             : run_adamw<T, true, MAX_CAP>(rows, count, c, dev, st);
    return count <= 16 ? run_adamw<T, false, 16>(rows, count, c, dev, st)
           : count <= 96 ? run_adamw<T, false, 96>(rows, count, c, dev, st)
                         : run_adamw<T, false, MAX_CAP>(rows, count, c, dev, st);
}

int check_table(const int64_t *table, int count, int dtype, bool sf8) {
    if (count < 0 || (count > 0 && !table)) return set_error(SFB_EINVAL, "sfb_adamw: no table");
    if (dtype != SFB_F32 && dtype != SFB_BF16 && dtype != SFB_F16)
        return set_error(SFB_EINVAL, "sfb_adamw: element type %d", dtype);
    const int size = dtype == SFB_F32 ? 4 : 2;
    for (int i = 0; i < count; i++) {
        const int64_t *r = table + (int64_t)i * WORDS;
        if (r[6] < 0) return set_error(SFB_EINVAL, "sfb_adamw: tensor %d has %lld elements", i, (long long)r[6]);
        if (r[6] == 0) continue;
        for (int j = 0; j < (sf8 ? 6 : 4); j++)
            if (!r[j]) return set_error(SFB_EINVAL, "sfb_adamw: tensor %d has a null pointer", i);
        if ((r[0] | r[1]) % size || (!sf8 && (r[2] | r[3]) % 4) || (sf8 && ((r[2] | r[3] | r[4] | r[5]) % 4)))
            return set_error(SFB_EINVAL, "sfb_adamw: tensor %d is not aligned to its type", i);
    }
    try {
        return check_overlap(table, count, size, sf8);
    } catch (const std::exception &) {
        return set_error(SFB_ERANGE, "sfb_adamw: no host memory for a table of %d tensors", count);
    }
}

}  // namespace
}  // namespace sfb

extern "C" int sfb_adamw_check(const int64_t *table, int count, int dtype, int sf8) {
    return sfb::check_table(table, count, dtype, sf8 != 0);
}

extern "C" int sfb_adamw(const int64_t *table, int count, int dtype, int sf8, double lr, double beta1, double beta2,
                         double eps, double weight_decay, int64_t step, unsigned dither, const void *constants,
                         sfb_stream stream) {
    using namespace sfb;
    if (!constants && step < 1) return set_error(SFB_EINVAL, "sfb_adamw: step %lld", (long long)step);
    const int rc = check_table(table, count, dtype, sf8 != 0);
    if (rc) return rc;
    const Coefs c = constants ? Coefs{} : coefs_of(lr, beta1, beta2, eps, weight_decay, step, dither);
    const Coefs *dev = static_cast<const Coefs *>(constants);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (dtype == SFB_F32) return run_typed<float>(table, count, sf8 != 0, c, dev, st);
    if (dtype == SFB_BF16) return run_typed<__nv_bfloat16>(table, count, sf8 != 0, c, dev, st);
    return run_typed<__half>(table, count, sf8 != 0, c, dev, st);
}

extern "C" int sfb_adamw_advance(int64_t *step, void *constants, double lr, double beta1, double beta2, double eps,
                                 double weight_decay, unsigned seed, sfb_stream stream) {
    using namespace sfb;
    static_assert(sizeof(Coefs) <= SFB_ADAMW_CONSTANTS, "the caller's buffer holds the constants");
    if (!step || !constants) return set_error(SFB_EINVAL, "sfb_adamw_advance: null pointer");
    advance_kernel<<<1, 1, 0, static_cast<cudaStream_t>(stream)>>>(reinterpret_cast<long long *>(step),
                                                                   static_cast<Coefs *>(constants), lr, beta1, beta2,
                                                                   eps, weight_decay, seed);
    return check_launch("sfb_adamw_advance");
}

extern "C" int sfb_sf8_values(const int64_t *table, int count, int power, sfb_stream stream) {
    using namespace sfb;
    if (count < 0 || (count > 0 && !table)) return set_error(SFB_EINVAL, "sfb_sf8_values: no table");
    if (power != 2 && power != 4) return set_error(SFB_EINVAL, "sfb_sf8_values: power %d", power);
    for (int i = 0; i < count; i++) {
        const int64_t *r = table + (int64_t)i * WORDS;
        if (r[6] < 0 || (r[6] > 0 && (!r[0] || !r[1] || !r[4] || r[0] % 16 || r[1] % 4)))
            return set_error(SFB_EINVAL, "sfb_sf8_values: tensor %d has a bad pointer or size", i);
    }
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (count <= 16)
        return each_table<16, false>(table, count, [&](Table<16> &t, unsigned grid) {
            values_kernel<16><<<grid, AT, 0, st>>>(t, power);
            return check_launch("sfb_sf8_values");
        });
    return each_table<MAX_CAP, false>(table, count, [&](Table<MAX_CAP> &t, unsigned grid) {
        values_kernel<MAX_CAP><<<grid, AT, 0, st>>>(t, power);
        return check_launch("sfb_sf8_values");
    });
}
