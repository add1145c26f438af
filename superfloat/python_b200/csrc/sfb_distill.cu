// Distillation from a teacher's top logits: the loss of a row and its gradient.
//
//   p_i = softmax of the teacher's entries / T,  q_j = softmax of the row / T
//   l = T^2 sum_i p_i (log p_i - log q_i),  dl / d logit_j = T (q_j - sum of the p_i whose index is j)
//
// times the row's weight and, for the mean, 1 / (the sum of the weights of the rows that
// count).  An entry is absent where its index is outside the vocabulary or its logit
// -inf; a row without entries, or of weight 0, gives 0 whatever stands in it and is not read.
//
// Bound by memory: the row is read once, into shared memory, and its gradient written
// once, from there.  Maximum and sum are taken in one pass; the gradient is a second one
// over shared memory.  A row is split over a cluster of up to 8 CTAs, so that two
// or more CTAs fit an SM (one computes while the other's copy is in flight), and so that
// few rows still occupy the GPU; they exchange (maximum, sum) through one another's memory.
// Rows start anywhere: a position in shared memory has the alignment of its address; whole
// 16-byte vectors come by cp.async, the elements around them one by one.  A thread reads
// what it has copied itself, so nothing waits for the whole row.  What shared memory does
// not hold is read from memory twice.
// Statistics and sums are float32.  2^x is taken of (x - max) log2(e) / T, so that neither
// the maximum nor the sum's logarithm, which are larger, is rounded with it.
#include <math.h>

#include <algorithm>
#include <mutex>

#include "sfb_tensor.cuh"

namespace sfb {
namespace {

constexpr int THREADS = 512;
constexpr int MAX_K = 1024;

struct Distill {
    const void *logits;
    const void *teacher, *index, *weight;
    float *rows;                         // the rows' losses
    float *stats;                        // maximum, sum, share of every row
    void *grad;
    const float *upstream;               // one, or one a row
    const float *parts;                  // the mean: partial sums of weights
    int64_t inner, so, si;               // row r starts at (r / inner) so + (r % inner) si
    int64_t go, gi;                      // the gradient's
    int64_t V, K, ldt, ldi, n_parts, M;
    int t_dtype, i_long, w_dtype, each;  // w_dtype: of the weights, -1 for bytes (truth values), -2 for none
    int chunk, held;                     // positions of a CTA; how many of them shared memory holds
    int same;                            // the gradient's rows lie on 16 bytes as the logits' do
    int skip;                            // nothing to do where the upstream gradient is one
    float temperature, unit;             // unit = log2(e) / T
};

enum Mode { LOSS, BOTH, GRADIENT };

__device__ __forceinline__ uint32_t cluster_size() {
    uint32_t n;
    asm("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(n));
    return n;
}

__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}

__device__ __forceinline__ void cluster_barrier() {
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

__device__ __forceinline__ float exp2_fast(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

__device__ __forceinline__ float ninf() { return __int_as_float(0xFF800000); }

template <typename T> struct Wide { static constexpr int E = 16 / sizeof(T); };

template <typename T> __device__ __forceinline__ void open16(uint4 q, float (&v)[Wide<T>::E]) {
    const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int i = 0; i < 4; i++) {
        if constexpr (sizeof(T) == 4) {
            v[i] = __uint_as_float(w[i]);
        } else if constexpr (std::is_same<T, __half>::value) {
            const float2 f = __half22float2(reinterpret_cast<const __half2 &>(w[i]));
            v[2 * i] = f.x;
            v[2 * i + 1] = f.y;
        } else {
            v[2 * i] = __uint_as_float(w[i] << 16);
            v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
        }
    }
}

template <typename T> __device__ __forceinline__ uint4 close16(const float (&v)[Wide<T>::E]) {
    Vec<T, Wide<T>::E> q;
#pragma unroll
    for (int j = 0; j < Wide<T>::E; j++) q.v[j] = from_f<T>(v[j]);
    return *reinterpret_cast<uint4 *>(&q);
}

__device__ __forceinline__ float weight_of(const Distill &p, int64_t r) {
    if (p.w_dtype == -2) return 1.0f;
    if (p.w_dtype == -1) return static_cast<const uint8_t *>(p.weight)[r] ? 1.0f : 0.0f;
    return load_as(p.weight, r, p.w_dtype);
}

__device__ __forceinline__ int64_t index_of(const Distill &p, int64_t r, int64_t i) {
    const int64_t at = r * p.ldi + i;
    const int64_t j = p.i_long ? static_cast<const int64_t *>(p.index)[at] : static_cast<const int32_t *>(p.index)[at];
    return j >= 0 && j < p.V ? j : -1;
}

// an entry's logit, -inf where it is absent
__device__ __forceinline__ float entry_of(const Distill &p, int64_t r, int64_t i, int64_t j) {
    return j >= 0 ? load_as(p.teacher, r * p.ldt + i, p.t_dtype) : ninf();
}

// --- the mean's denominator ----------------------------------------------------------------------------------
// A row counts with its weight if it has an entry, mostly its first: 256 rows a CTA, their sum in a fixed order.

constexpr int PART = 256;

__global__ void __launch_bounds__(PART) count_kernel(const __grid_constant__ Distill p, float *parts) {
    __shared__ float s[PART / 32];
    const int64_t r = (int64_t)blockIdx.x * PART + threadIdx.x;
    float w = 0.0f;
    if (r < p.M) {
        w = weight_of(p, r);
        bool some = false;
        if (w != 0.0f)
            for (int64_t i = 0; i < p.K && !some; i++) some = !(entry_of(p, r, i, index_of(p, r, i)) == ninf());
        if (!some) w = 0.0f;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) w += __shfl_xor_sync(0xffffffffu, w, o);
    if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = w;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int i = 1; i < PART / 32; i++) w += s[i];
        parts[blockIdx.x] = w;
    }
}

// the rows' losses added up, in a fixed order
__global__ void __launch_bounds__(1024) total_kernel(const float *__restrict__ rows, int64_t M, float *loss) {
    __shared__ float s[32];
    float v = 0.0f;
#pragma unroll 4
    for (int64_t i = threadIdx.x; i < M; i += 1024) v += rows[i];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = v;
    __syncthreads();
    if (threadIdx.x < 32) {
        v = s[threadIdx.x];
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
        if (threadIdx.x == 0) *loss = v;
    }
}

// --- a row ---------------------------------------------------------------------------------------------------

struct Shared {
    float red[THREADS / 32];
    float2 soft[THREADS / 32];
    float2 ctas[2][8];
};

__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// over the CTA; the barriers before and after let the places be used again
__device__ __forceinline__ float cta_max(float v, Shared &s) {
    v = warp_max(v);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) s.red[threadIdx.x >> 5] = v;
    __syncthreads();
    v = s.red[0];
#pragma unroll
    for (int i = 1; i < THREADS / 32; i++) v = fmaxf(v, s.red[i]);
    return v;
}

__device__ __forceinline__ float cta_sum(float v, Shared &s) {
    v = warp_sum(v);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) s.red[threadIdx.x >> 5] = v;
    __syncthreads();
    v = s.red[0];
#pragma unroll
    for (int i = 1; i < THREADS / 32; i++) v += s.red[i];
    return v;
}

// (maximum, sum of 2^((x - maximum) unit)) of two parts of a row; a part of nothing is (-inf, 0)
__device__ __forceinline__ float2 soft_join(float2 a, float2 b, float unit) {
    const float m = fmaxf(a.x, b.x), base = m == ninf() ? 0.0f : m;
    return make_float2(m, a.y * exp2_fast((a.x - base) * unit) + b.y * exp2_fast((b.x - base) * unit));
}

template <typename T, int MODE>
__global__ void __launch_bounds__(THREADS, 2) row_kernel(const __grid_constant__ Distill p) {
    constexpr int E = Wide<T>::E;
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ Shared s;
    // the teacher's entries: logits, then p; indexes; the student's logits there
    float *entry = reinterpret_cast<float *>(smem);
    const int k4 = (int)((p.K + 3) & ~3);
    int *where = reinterpret_cast<int *>(entry + k4);
    float *near = reinterpret_cast<float *>(where + k4);
    T *row = reinterpret_cast<T *>(near + k4);
    const int tid = threadIdx.x;
    const uint32_t n = cluster_size(), rank = cluster_rank();
    if (MODE == GRADIENT && p.skip && *p.upstream == 1.0f) return;
    if (MODE != GRADIENT && n > 1) cluster_barrier();  // the others' memory is there
    float share = 1.0f;                               // of a row's loss, before its weight
    if (MODE != GRADIENT && p.parts) {
        float w = 0.0f;
        for (int64_t i = tid; i < p.n_parts; i += THREADS) w += p.parts[i];
        w = cta_sum(w, s);
        share = w == 0.0f ? 0.0f : __fdiv_rn(1.0f, w);
    }
    int turn = 0;
    for (int64_t r = blockIdx.x / n; r < p.M; r += gridDim.x / n) {
        const T *from = static_cast<const T *>(p.logits) + (r / p.inner) * p.so + (r % p.inner) * p.si;
        T *to = static_cast<T *>(p.grad) + (r / p.inner) * p.go + (r % p.inner) * p.gi;
        const float weight = weight_of(p, r);
        // Positions count from the 16-byte border before the row: element j is at j + lead.
        const int lead = (int)((reinterpret_cast<uintptr_t>(from) & 15) / sizeof(T));
        const int64_t lo = (int64_t)rank * p.chunk, hi = min(lo + p.chunk, p.V + lead);     // of this CTA
        const int64_t first = max(lo, (int64_t)lead);                                      // with an element
        const T *at0 = from - lead;                   // (the address of position 0: not read before `lead`)
        const int held = (int)max((int64_t)0, min((int64_t)p.held, hi - lo));
        // the whole vectors that shared memory holds, and the elements around them
        const int64_t whole = (first + E - 1) / E * E, end = (lo + held) / E * E;
        const bool live = weight != 0.0f;
        const int vectors = hi > lo ? (int)((hi - lo + E - 1) / E) : 0, inside = held / E;
        __syncthreads();                              // the row before has been read
        if (MODE != GRADIENT && live) {
            for (int i = tid; i < inside; i += THREADS) {
                const int64_t u = lo + (int64_t)i * E;
                if (u >= whole && u < end)
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(
                                     (uint32_t)__cvta_generic_to_shared(row + (u - lo))),
                                 "l"(at0 + u)
                                 : "memory");
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
        }
        // the entries
        float top = ninf();
        bool some = false;
        for (int i = tid; i < p.K && live; i += THREADS) {
            const int64_t j = index_of(p, r, i);
            const float t = entry_of(p, r, i, j);
            const bool here = !(t == ninf());
            entry[i] = t;
            where[i] = here ? (int)j : -1;
            near[i] = here ? to_f(from[j]) : 0.0f;
            top = fmaxf(top, t);
            some |= here;
        }
        some = __syncthreads_or(some) != 0;
        const bool counts = live && some;             // the same for all threads, and for the cluster
        float total = 0.0f;
        if (counts) {
            top = cta_max(top, s);
            for (int i = tid; i < p.K; i += THREADS)
                if (where[i] >= 0) total += exp2_fast((entry[i] - top) * p.unit);
            total = cta_sum(total, s);
        }
        const float inv_total = __fdiv_rn(1.0f, total);

        // elements that shared memory does not get by the copy: before the first whole vector, after the last
        auto vector_at = [&](int64_t u) {             // the vector of positions u .. u + E - 1 from memory
            if (u >= first && u + E <= hi) return __ldg(reinterpret_cast<const uint4 *>(at0 + u));
            float v[E];
#pragma unroll
            for (int j = 0; j < E; j++) v[j] = u + j >= first && u + j < hi ? to_f(at0[u + j]) : ninf();
            return close16<T>(v);
        };
        float2 soft = make_float2(ninf(), 0.0f);
        if constexpr (MODE != GRADIENT) {
            asm volatile("cp.async.wait_group 0;" ::: "memory");
            if (counts) {
                for (int i = tid; i < vectors; i += THREADS) {
                    const int64_t u = lo + (int64_t)i * E;
                    uint4 q;
                    if (u >= whole && u < end) {
                        q = *reinterpret_cast<const uint4 *>(row + (u - lo));
                    } else {
                        q = vector_at(u);
                        if (i < inside) *reinterpret_cast<uint4 *>(row + (u - lo)) = q;
                    }
                    float v[E];
                    open16<T>(q, v);
                    float m = v[0];
#pragma unroll
                    for (int j = 1; j < E; j++) m = fmaxf(m, v[j]);
                    if (m > soft.x) {
                        soft.y *= exp2_fast((soft.x - m) * p.unit);
                        soft.x = m;
                    }
                    const float base = soft.x == ninf() ? 0.0f : soft.x;
                    float e = 0.0f;
#pragma unroll
                    for (int j = 0; j < E; j++) e += exp2_fast((v[j] - base) * p.unit);
                    soft.y += e;
                }
#pragma unroll
                for (int o = 16; o > 0; o >>= 1)
                    soft = soft_join(soft, make_float2(__shfl_xor_sync(0xffffffffu, soft.x, o),
                                                       __shfl_xor_sync(0xffffffffu, soft.y, o)), p.unit);
                if ((tid & 31) == 0) s.soft[tid >> 5] = soft;
            }
            __syncthreads();
            if (counts) {
                soft = s.soft[0];
                for (int i = 1; i < THREADS / 32; i++) soft = soft_join(soft, s.soft[i], p.unit);
            }
            if (n > 1) {
                // (the places alternate: what is overwritten was read before the barrier of the row between)
                if (tid < (int)n) {
                    const uint32_t mine = (uint32_t)__cvta_generic_to_shared(&s.ctas[turn][rank]);
                    uint32_t there;
                    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"(mine), "r"((uint32_t)tid));
                    asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};" ::"r"(there), "f"(soft.x), "f"(soft.y) : "memory");
                }
                cluster_barrier();
                soft = s.ctas[turn][0];
                for (uint32_t i = 1; i < n; i++) soft = soft_join(soft, s.ctas[turn][i], p.unit);
                turn ^= 1;
            }
            if (rank == 0) {
                float loss = 0.0f;
                if (counts) {
                    // log p - log q = (entry - top) / T - log total - (logit - maximum) / T + log sum, in base 2
                    const float base = soft.x == ninf() ? 0.0f : soft.x;
                    const float off = log2f(soft.y) - log2f(total);
                    for (int i = tid; i < p.K; i += THREADS) {
                        if (where[i] < 0) continue;
                        const float a = (entry[i] - top) * p.unit;
                        const float q = exp2_fast(a) * inv_total;
                        if (!(q == 0.0f)) loss = fmaf(q, a - (near[i] - base) * p.unit + off, loss);
                    }
                    loss = cta_sum(loss, s) * (0.69314718056f * p.temperature * p.temperature) * (weight * share);
                }
                if (tid == 0) {
                    p.rows[r] = loss;
                    if (p.stats) {
                        p.stats[3 * r] = soft.x == ninf() ? 0.0f : soft.x;
                        p.stats[3 * r + 1] = soft.y;
                        p.stats[3 * r + 2] = counts ? weight * share : 0.0f;
                    }
                }
            }
        }
        if constexpr (MODE != LOSS) {
            float base, factor, inv;
            if constexpr (MODE == BOTH) {
                base = soft.x == ninf() ? 0.0f : soft.x;
                inv = __fdiv_rn(1.0f, soft.y);
                factor = counts ? weight * share * p.temperature : 0.0f;
            } else {
                base = p.stats[3 * r];
                inv = __fdiv_rn(1.0f, p.stats[3 * r + 1]);
                factor = counts ? p.stats[3 * r + 2] * p.temperature * p.upstream[p.each ? r : 0] : 0.0f;
            }
            const float scale = inv * factor;
            if (p.same) {
                T *to0 = to - lead;
                for (int i = tid; i < vectors; i += THREADS) {
                    const int64_t u = lo + (int64_t)i * E;
                    float v[E];
                    if (counts) {
                        open16<T>(MODE == BOTH && i < inside ? *reinterpret_cast<const uint4 *>(row + (u - lo)) : vector_at(u), v);
#pragma unroll
                        for (int j = 0; j < E; j++) v[j] = exp2_fast((v[j] - base) * p.unit) * scale;
                    } else {
#pragma unroll
                        for (int j = 0; j < E; j++) v[j] = 0.0f;
                    }
                    if (u >= first && u + E <= hi) {
                        *reinterpret_cast<uint4 *>(to0 + u) = close16<T>(v);
                    } else {
#pragma unroll
                        for (int j = 0; j < E; j++)
                            if (u + j >= first && u + j < hi) to0[u + j] = from_f<T>(v[j]);
                    }
                }
            } else {
                for (int64_t u = first + tid; u < hi; u += THREADS) {
                    float v = 0.0f;
                    if (counts)
                        v = exp2_fast((to_f(MODE == BOTH && u < lo + inside * E ? row[u - lo] : at0[u]) - base) * p.unit) * scale;
                    to[u - lead] = from_f<T>(v);
                }
            }
            __syncthreads();                          // the entries' elements are written again, after that
            for (int i = tid; i < p.K && counts; i += THREADS) {
                const int64_t u = (int64_t)where[i] + lead;
                if (where[i] < 0 || u < lo || u >= hi) continue;
                // an index that comes more than once has all its entries' shares, whichever thread writes it
                float mine = 0.0f;
                for (int j = 0; j < p.K; j++)
                    if (where[j] == where[i]) mine += exp2_fast((entry[j] - top) * p.unit) * inv_total;
                to[where[i]] = from_f<T>(factor * (exp2_fast((near[i] - base) * p.unit) * inv - mine));
            }
        }
    }
    // (a CTA ends only once the others have written into its memory: their writes precede a barrier that it has passed)
}

// --- launches ------------------------------------------------------------------------------------------------

constexpr int64_t HALF = 106 * 1024;     // shared memory of a CTA of which two fit an SM
constexpr int64_t MOST = 200 * 1024;

template <typename T, int MODE>
int launch(Distill p, cudaStream_t st) {
    const char *what = MODE == GRADIENT ? "sf distillation (backward)" : "sf distillation";
    auto *kernel = row_kernel<T, MODE>;
    static std::mutex lock;
    static unsigned long long ready[64] = {};          // the CUDA context whose attribute is set, per device
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return set_error(SFB_ECUDA, "%s: no current CUDA device", what);
    if (MODE != GRADIENT) {
        std::lock_guard<std::mutex> g(lock);
        const unsigned long long ctx = context_id();
        if (ctx == 0 || ready[dev] != ctx) {
            if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)MOST) != cudaSuccess)
                return check_launch(what);
            ready[dev] = context_id();
        }
    }
    constexpr int64_t E = 16 / sizeof(T);
    const int64_t entries = 12 * ((p.K + 3) & ~3ll), span = p.V + E - 1;
    auto chunk_of = [&](int64_t c) { return ((span + c - 1) / c + E - 1) / E * E; };
    int64_t c = 1;
    // A cluster as large as lets two CTAs share an SM; larger ones where rows are few, a chunk being 4096 elements at least.
    while (c < 8 && ((MODE != GRADIENT && entries + chunk_of(c) * (int64_t)sizeof(T) > HALF) ||
                     (p.M * c < 2 * sm_count() && chunk_of(2 * c) >= 4096)))
        c *= 2;
    const int64_t chunk = chunk_of(c);
    p.chunk = (int)chunk;
    p.held = MODE == GRADIENT ? 0 : (int)std::min(chunk, (MOST - entries) / 16 * E);
    const int64_t bytes = entries + p.held * (int64_t)sizeof(T);
    const int64_t resident = std::max<int64_t>(1, (bytes > HALF ? 1 : 2) * sm_count() / c);
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)(std::min(p.M, resident) * c));
    cfg.blockDim = dim3(THREADS);
    cfg.dynamicSmemBytes = (size_t)bytes;
    cfg.stream = st;
    cudaLaunchAttribute a{};
    a.id = cudaLaunchAttributeClusterDimension;
    a.val.clusterDim.x = (unsigned)c;
    a.val.clusterDim.y = a.val.clusterDim.z = 1;
    cfg.attrs = &a;
    cfg.numAttrs = c > 1 ? 1 : 0;
    cudaLaunchKernelEx(&cfg, kernel, p);
    return check_launch(what);
}

template <int MODE>
int by_type(int64_t dtype, const Distill &p, cudaStream_t st) {
    if (dtype == SFB_F32) return launch<float, MODE>(p, st);
    if (dtype == SFB_BF16) return launch<__nv_bfloat16, MODE>(p, st);
    return launch<__half, MODE>(p, st);
}

bool is_float(int64_t t) { return t == SFB_F32 || t == SFB_BF16 || t == SFB_F16; }

int check(const sfb_distill_call *c, const char *what) {
    if (!c) return set_error(SFB_EINVAL, "%s: null pointer", what);
    if (!is_float(c->dtype) || !is_float(c->t_dtype))
        return set_error(SFB_EINVAL, "%s: element types %d and %d", what, (int)c->dtype, (int)c->t_dtype);
    if (c->w_dtype != SFB_WEIGHT_NONE && c->w_dtype != SFB_WEIGHT_BYTES && !is_float(c->w_dtype))
        return set_error(SFB_EINVAL, "%s: the weights' type %d", what, (int)c->w_dtype);
    if (c->M < 0 || c->V < 1 || c->K < 0 || c->inner < 1 || c->ldt < c->K || c->ldi < c->K)
        return set_error(SFB_EINVAL, "%s: bad shape", what);
    if (c->V >= (1ll << 31) - 4096) return set_error(SFB_ERANGE, "%s: a vocabulary of %lld", what, (long long)c->V);
    if (c->K > MAX_K) return set_error(SFB_ERANGE, "%s: %lld entries a row, %d at most", what, (long long)c->K, MAX_K);
    if (!(c->temperature > 0.0) || !(c->temperature <= 1e6) || !(c->temperature >= 1e-6))
        return set_error(SFB_EINVAL, "%s: a temperature is between 1e-6 and 1e6", what);
    if (c->reduction < SFB_REDUCE_NONE || c->reduction > SFB_REDUCE_MEAN)
        return set_error(SFB_EINVAL, "%s: reduction %d", what, (int)c->reduction);
    if (c->M > 0 && (!c->logits || (c->K > 0 && (!c->teacher || !c->index)) || (c->w_dtype != SFB_WEIGHT_NONE && !c->weight)))
        return set_error(SFB_EINVAL, "%s: null pointer", what);
    const uintptr_t size = c->dtype == SFB_F32 ? 4 : 2;
    if (reinterpret_cast<uintptr_t>(c->logits) % size || reinterpret_cast<uintptr_t>(c->grad) % size)
        return set_error(SFB_EINVAL, "%s: the logits or their gradient do not start on an element", what);
    return SFB_OK;
}

Distill distill_of(const sfb_distill_call *c) {
    Distill p{};
    p.logits = c->logits;
    p.teacher = c->teacher;
    p.index = c->index;
    p.weight = c->weight;
    p.stats = c->stats;
    p.grad = c->grad;
    p.inner = c->inner;
    p.so = c->so;
    p.si = c->si;
    p.go = c->go;
    p.gi = c->gi;
    p.V = c->V;
    p.K = c->K;
    p.M = c->M;
    p.ldt = c->ldt;
    p.ldi = c->ldi;
    p.t_dtype = (int)c->t_dtype;
    p.i_long = c->i_long != 0;
    p.w_dtype = (int)c->w_dtype;
    p.temperature = (float)c->temperature;
    p.unit = (float)(1.4426950408889634 / c->temperature);
    // the rows of both lie alike on 16 bytes
    const int64_t size = c->dtype == SFB_F32 ? 4 : 2;
    p.same = c->grad && ((reinterpret_cast<uintptr_t>(c->logits) ^ reinterpret_cast<uintptr_t>(c->grad)) & 15) == 0 &&
             (c->so - c->go) * size % 16 == 0 && (c->si - c->gi) * size % 16 == 0;
    return p;
}

}  // namespace
}  // namespace sfb

extern "C" int64_t sfb_distill_parts(int64_t M) { return M > 0 ? (M + sfb::PART - 1) / sfb::PART : 0; }

extern "C" int sfb_distill_forward(const sfb_distill_call *c, sfb_stream stream) {
    using namespace sfb;
    const char *what = "sfb_distill_forward";
    int rc = check(c, what);
    if (rc) return rc;
    const bool mean = c->reduction == SFB_REDUCE_MEAN, one = c->reduction != SFB_REDUCE_NONE;
    if ((one && !c->loss) || (c->M > 0 && (!c->rows || (mean && !c->parts))))
        return set_error(SFB_EINVAL, "%s: null pointer", what);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (c->M > 0) {
        Distill p = distill_of(c);
        p.rows = c->rows;
        if (mean) {
            p.n_parts = sfb_distill_parts(c->M);
            if (p.n_parts >= 1ll << 31) return set_error(SFB_ERANGE, "%s: %lld rows", what, (long long)c->M);
            count_kernel<<<(unsigned)p.n_parts, PART, 0, st>>>(p, c->parts);
            if ((rc = check_launch("sf distillation (rows that count)"))) return rc;
            p.parts = c->parts;
        }
        rc = c->grad ? by_type<BOTH>(c->dtype, p, st) : by_type<LOSS>(c->dtype, p, st);
        if (rc) return rc;
    }
    if (!one) return SFB_OK;
    total_kernel<<<1, 1024, 0, st>>>(c->rows, c->M, c->loss);
    return check_launch("sf distillation (sum of the rows)");
}

extern "C" int sfb_distill_backward(const sfb_distill_call *c, sfb_stream stream) {
    using namespace sfb;
    const char *what = "sfb_distill_backward";
    const int rc = check(c, what);
    if (rc) return rc;
    if (c->M == 0) return SFB_OK;
    if (!c->grad || !c->stats || !c->upstream) return set_error(SFB_EINVAL, "%s: null pointer", what);
    Distill p = distill_of(c);
    p.upstream = c->upstream;
    p.each = c->reduction == SFB_REDUCE_NONE;
    p.skip = c->skip != 0 && !p.each;
    return by_type<GRADIENT>(c->dtype, p, static_cast<cudaStream_t>(stream));
}
