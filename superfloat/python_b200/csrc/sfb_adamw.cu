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
// infinite or NaN, and every moment of the block then reads as NaN.
// The codes depend on the last bits of m and v, so each float32 operation on the
// way to a code is one IEEE rounding (the __f*_rn forms are not contracted to fma).
//
// One launch takes a table of tensors as its parameter (no table in device
// memory: nothing to copy, and nothing that two captured graphs could share).
// A CTA takes one chunk of one tensor, found by bisection over the chunk counts.
// Memory bound: 28 bytes an element with float32 p, g and moments, 16.06 with sf8
// moments, 10.06 with 16-bit p and g besides.
#include <math.h>

#include <algorithm>
#include <exception>
#include <vector>

#include "sfb_tensor.cuh"

namespace sfb {
namespace {

constexpr int AT = 256;                       // threads of a CTA
constexpr int AB = 256;                       // elements of one sf8 block
constexpr int CHUNK = 4096;                   // elements of one CTA
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
    uint32_t vec;                             // p and g are aligned for vectors of four
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

// 32 mixed bits of a counter (two rounds of multiply and xor-shift)
__device__ __forceinline__ uint32_t mixed(uint32_t i, uint32_t seed) {
    uint32_t h = i * 0x9E3779B1u + seed;
    h ^= h >> 16;
    h *= 0x7FEB352Du;
    h ^= h >> 15;
    h *= 0x846CA68Bu;
    h ^= h >> 16;
    return h;
}

template <int POWER>
__device__ __forceinline__ float level(float c) {
    const float c2 = __fmul_rn(c, c);
    return POWER == 2 ? c2 : __fmul_rn(c2, c2);
}

// the code of t = |value| * top / s: the largest c with level(c) <= t, or the next one by the dither
template <int POWER>
__device__ __forceinline__ int code_of(float t, float u) {
    float r = sqrt_fast(t);
    if (POWER == 4) r = sqrt_fast(r);
    int k = t < 3.0e38f ? (int)r : 127;               // NaN and infinity: any code, the scale tells
    float c = (float)k;
    if (level<POWER>(c) > t) c -= 1.0f;
    else if (level<POWER>(c + 1.0f) <= t) c += 1.0f;
    if (c >= 127.0f) return 127;
    const float low = level<POWER>(c), wide = __fsub_rn(level<POWER>(c + 1.0f), low);
    if (__fmul_rn(u, wide) < __fsub_rn(t, low)) c += 1.0f;
    if (POWER == 4 && t > 0.0f) c = fmaxf(c, 1.0f);
    return (int)c;
}

__device__ __forceinline__ uint32_t warp_top(const float (&x)[8]) {
    uint32_t top = 0;
#pragma unroll
    for (int j = 0; j < 8; j++) top = max(top, __float_as_uint(x[j]) & 0x7FFFFFFFu);
    return __reduce_max_sync(0xffffffffu, top);       // magnitudes order as their bits, NaN above all
}

__device__ __forceinline__ float scale_of(uint32_t bits) {
    const float s = __uint_as_float(bits);
    return s < 1e-30f ? 0.0f : s;
}

// a block of 256 elements by one warp: lane l has elements 4 l .. 4 l + 3 of each half
template <typename T>
__device__ __forceinline__ void block_sf8(const Entry &e, int64_t blk, const Coefs &c, int lane) {
    const int64_t base = blk * AB;
    T *p = static_cast<T *>(e.p);
    const T *g = static_cast<const T *>(e.g);
    int8_t *mc = static_cast<int8_t *>(e.m), *vc = static_cast<int8_t *>(e.v);
    const bool whole = base + AB <= e.n;
    float P[8], G[8], M[8], V[8];
    char4 cm[2], cv[2];
    const float sm = e.ms[blk], sv = e.vs[blk];
#pragma unroll
    for (int h = 0; h < 2; h++) {
        const int64_t i = base + h * 128 + lane * 4;
        load4(g, i, e.n, e.vec, *reinterpret_cast<float(*)[4]>(G + 4 * h));
        if (whole) {
            cm[h] = *reinterpret_cast<const char4 *>(mc + i);
            cv[h] = *reinterpret_cast<const char4 *>(vc + i);
        } else {
            signed char a[4], b[4];
#pragma unroll
            for (int j = 0; j < 4; j++) {
                a[j] = i + j < e.n ? mc[i + j] : (signed char)0;
                b[j] = i + j < e.n ? vc[i + j] : (signed char)0;
            }
            cm[h] = make_char4(a[0], a[1], a[2], a[3]);
            cv[h] = make_char4(b[0], b[1], b[2], b[3]);
        }
        load4(p, i, e.n, e.vec, *reinterpret_cast<float(*)[4]>(P + 4 * h));
    }
    const float um = __fmul_rn(sm, UNIT2), uv = __fmul_rn(sv, UNIT4);
#pragma unroll
    for (int j = 0; j < 8; j++) {
        const char4 a = cm[j / 4], b = cv[j / 4];
        const int x = j % 4 == 0 ? a.x : j % 4 == 1 ? a.y : j % 4 == 2 ? a.z : a.w;
        const int y = j % 4 == 0 ? b.x : j % 4 == 1 ? b.y : j % 4 == 2 ? b.z : b.w;
        M[j] = __fmul_rn((float)(x * abs(x)), um);
        const float y2 = (float)(y * y);
        V[j] = __fmul_rn(__fmul_rn(y2, y2), uv);
        moments(M[j], V[j], G[j], c);
        P[j] = stepped(P[j], M[j], V[j], c);
    }
    const float sm1 = scale_of(warp_top(M)), sv1 = scale_of(warp_top(V));
    const float im = sm1 != 0.0f ? __fdiv_rn(TOP2, sm1) : 0.0f, iv = sv1 != 0.0f ? __fdiv_rn(TOP4, sv1) : 0.0f;
    if (lane == 0) {
        e.ms[blk] = sm1;
        e.vs[blk] = sv1;
    }
#pragma unroll
    for (int h = 0; h < 2; h++) {
        const int64_t i = base + h * 128 + lane * 4;
        store4(p, i, e.n, e.vec, *reinterpret_cast<float(*)[4]>(P + 4 * h));
        int a[4], b[4];
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const uint32_t r = mixed((uint32_t)(i + j), e.seed + c.dither);
            const float m = M[4 * h + j];
            const int k = code_of<2>(__fmul_rn(fabsf(m), im), (float)(r & 0xFFFFu) * 0x1p-16f);
            a[j] = m < 0.0f ? -k : k;
            b[j] = code_of<4>(__fmul_rn(V[4 * h + j], iv), (float)(r >> 16) * 0x1p-16f);
        }
        if (whole) {
            *reinterpret_cast<char4 *>(mc + i) = make_char4(a[0], a[1], a[2], a[3]);
            *reinterpret_cast<char4 *>(vc + i) = make_char4(b[0], b[1], b[2], b[3]);
        } else {
#pragma unroll
            for (int j = 0; j < 4; j++)
                if (i + j < e.n) {
                    mc[i + j] = (int8_t)a[j];
                    vc[i + j] = (int8_t)b[j];
                }
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
__global__ void __launch_bounds__(AT) adamw_kernel(const __grid_constant__ Table<CAP> t, Coefs given,
                                                   const Coefs *__restrict__ on_device) {
    const int k = tensor_of(t, blockIdx.x);
    const Entry &e = t.e[k];
    const Coefs c = on_device ? *on_device : given;
    const int64_t first = (int64_t)(blockIdx.x - t.start[k]) * CHUNK, last = min(e.n, first + CHUNK);
    if constexpr (SF8) {
        const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
        for (int64_t b = first / AB + warp; b * AB < last; b += AT / 32) block_sf8<T>(e, b, c, lane);
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

// the values that sf8 codes stand for
template <int CAP>
__global__ void __launch_bounds__(AT) values_kernel(const __grid_constant__ Table<CAP> t, int power) {
    const int k = tensor_of(t, blockIdx.x);
    const Entry &e = t.e[k];
    const int64_t first = (int64_t)(blockIdx.x - t.start[k]) * CHUNK, last = min(e.n, first + CHUNK);
    const int8_t *code = static_cast<const int8_t *>(e.g);
    float *out = static_cast<float *>(e.p);
    for (int64_t i = first + 4 * threadIdx.x; i < last; i += 4 * AT) {
        const float s = e.ms[i / AB], u = __fmul_rn(s, power == 2 ? UNIT2 : UNIT4);
        float r[4];
        signed char q[4] = {0, 0, 0, 0};
        if (i + 4 <= last) {
            const char4 x = *reinterpret_cast<const char4 *>(code + i);
            q[0] = x.x, q[1] = x.y, q[2] = x.z, q[3] = x.w;
        } else {
            for (int j = 0; j < 4; j++)
                if (i + j < last) q[j] = code[i + j];
        }
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const int x = q[j];
            const float y = (float)(x * x), l = power == 2 ? y : __fmul_rn(y, y);
            r[j] = __fmul_rn(x < 0 ? -l : l, u);
        }
        store4(out, i, last, true, r);
    }
}

constexpr int WORDS = 8;                      // of one table entry as the caller gives it
constexpr int MAX_CAP = 448;

template <int CAP, typename F>
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
            const uint64_t need = (uint64_t)((n + CHUNK - 1) / CHUNK);
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
    return each_table<CAP>(rows, count, [&](Table<CAP> &t, unsigned grid) {
        for (int i = 0; i < t.count; i++) {
            Entry &e = t.e[i];
            const uintptr_t a = reinterpret_cast<uintptr_t>(e.p) | reinterpret_cast<uintptr_t>(e.g);
            const uintptr_t b = SF8 ? 0 : reinterpret_cast<uintptr_t>(e.m) | reinterpret_cast<uintptr_t>(e.v);
            e.vec = (a & (4 * sizeof(T) - 1)) == 0 && (b & 15) == 0;
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

}  // namespace
}  // namespace sfb

extern "C" int sfb_adamw(const int64_t *table, int count, int dtype, int sf8, double lr, double beta1, double beta2,
                         double eps, double weight_decay, int64_t step, unsigned dither, const void *constants,
                         sfb_stream stream) {
    using namespace sfb;
    if (count < 0 || (count > 0 && !table)) return set_error(SFB_EINVAL, "sfb_adamw: no table");
    if (dtype != SFB_F32 && dtype != SFB_BF16 && dtype != SFB_F16)
        return set_error(SFB_EINVAL, "sfb_adamw: element type %d", dtype);
    if (!constants && step < 1) return set_error(SFB_EINVAL, "sfb_adamw: step %lld", (long long)step);
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
        const int rc = check_overlap(table, count, size, sf8 != 0);
        if (rc) return rc;
    } catch (const std::exception &) {
        return set_error(SFB_ERANGE, "sfb_adamw: no host memory for a table of %d tensors", count);
    }
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
        return each_table<16>(table, count, [&](Table<16> &t, unsigned grid) {
            values_kernel<16><<<grid, AT, 0, st>>>(t, power);
            return check_launch("sfb_sf8_values");
        });
    return each_table<MAX_CAP>(table, count, [&](Table<MAX_CAP> &t, unsigned grid) {
        values_kernel<MAX_CAP><<<grid, AT, 0, st>>>(t, power);
        return check_launch("sfb_sf8_values");
    });
}
