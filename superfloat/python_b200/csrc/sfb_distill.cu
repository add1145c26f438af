// Distillation from a teacher's top logits: the loss of a row and its gradient.
//
//   p_i = softmax of the teacher's entries / T,  q_j = softmax of the row / T
//   l = T^2 sum_i p_i (log p_i - log q_i),  dl / d logit_j = T (q_j - sum of the p_i whose index is j)
//
// times the row's weight and, for the mean, 1 / (the sum of the weights of the rows that
// count).  An entry is absent where its index is outside the vocabulary or its logit
// -inf; a row without entries, or of weight 0, gives 0 whatever stands in it and is not read.
//
// Neither memory nor the rate of exponentials (two an element, 16 a cycle and SM) is full, both stand at half:
// the row is read once, into shared memory, and its gradient written once, from there.  Maximum,
// sum and gradient are three passes over shared memory, of which a thread reads what it has
// copied itself (cp.async), so that nothing waits for the whole row, and asks for the next row's
// vectors once it has used its own of this one.  A row is split over a cluster of up to 8 CTAs, so that
// four fit an SM, one's sums running under another's copies and a third one's stores, and so that
// few rows still occupy the GPU.  What depends on the teacher's entries alone is made by a launch
// before; a warp of its own makes the row's loss and the elements of the gradient that have an
// entry.
// 4096 x 50257 of bf16, a fifth of the rows masked, which are written and not read: 164 us for 735 MB, 4.5 TB/s; 2047 x
// 32001 of float32 likewise: 103 us for 467 MB, 4.5 TB/s.
// Measured on the way, each beside 162: two CTAs an SM with 100 KB of a row each 176, five with 34 KB 197; two buffers
// a CTA, the next row's copy under this one's sums, 188 (two CTAs) and 196 (one, of a whole row);
// the gradient one row behind the sums 243.
// Rows start anywhere: a position in shared memory has the alignment of its address.  What
// shared memory does not hold is read from memory three times.
// Statistics and sums are float32.  2^x is taken of x log2(e) / T - b, with one b, the
// rounded maximum's, for all of a row: its rounding cancels between q and the sum.  Rows so
// far from 0 that this rounding counts take the difference first.
#include <math.h>

#include <algorithm>
#include <mutex>

#include "sfb_tensor.cuh"

namespace sfb {

unsigned wait_polls();                        // the calling thread's sfb_wide_wait_limit
int wait_stall();

namespace {

constexpr int THREADS = 224, WARPS = THREADS / 32;   // that have the row
constexpr int ALL = THREADS + 32;                    // and the warp that has the entries
constexpr int MAX_K = 1024;
constexpr int PART = 8;                              // rows of a CTA that takes entries, a warp each
constexpr int BITS = 8192;                           // of the table in which entries look for their like

struct Distill {
    const void *logits;
    const void *teacher, *index, *weight;
    float *rows;                         // the rows' losses
    float *stats;                        // maximum, 1 / sum, weight x share of every row
    float *block;                        // of every row 4 k4 words: its entries' p, mass, near, where
    float *weights;                      // of every row, 0 where it does not count
    void *grad;
    const float *upstream;               // one, or one a row
    const float *parts;                  // the mean: partial sums of weights
    float *loss;                         // the rows' sum, null where none is wanted
    unsigned *ended;                     // counts the clusters that have ended
    int64_t inner, so, si;               // row r starts at (r / inner) so + (r % inner) si
    int64_t go, gi;                      // the gradient's
    int64_t V, K, ldt, ldi, n_parts, M;
    int64_t last;                        // the element after the last row's last
    int t_dtype, i_long, w_dtype, each;  // w_dtype: of the weights, -1 for bytes (truth values), -2 for none
    int chunk, held;                     // positions of a CTA; how many of them shared memory holds
    int same;                            // the gradient's rows lie on 16 bytes as the logits' do
    int skip;                            // nothing to do where the upstream gradient is one
    float temperature, unit;             // unit = log2(e) / T
    unsigned spin;                       // polls of a wait
    int stall;                           // the tests': the first row's parts never come
};

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

__device__ __forceinline__ int64_t place(const Distill &p, int64_t r, int64_t outer, int64_t inner) {
    if (r < p.inner) return r * inner;
    if ((r | p.inner) >> 32) return r / p.inner * outer + r % p.inner * inner;
    const uint32_t o = (uint32_t)r / (uint32_t)p.inner;
    return o * outer + (r - o * p.inner) * inner;
}

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

// what is taken from x unit before 2^x; a row (or part) of nothing but -inf has none
__device__ __forceinline__ float base_of(float m, float unit) { return m == ninf() ? 0.0f : __fmul_rn(m, unit); }

// Where the rounding of m log2(e) / T is not small (half a step is 1 from 2^24 on and 64 from 2^30 on, so that powers would
// leave float32's range) the difference of x and m is taken first: a row at -1e30, as masks leave it, or a temperature of 1e-6.
constexpr float BORDER = 16777216.0f;

__device__ __forceinline__ bool far(float m, float unit) { return fabsf(m) * unit > BORDER && m != ninf(); }

template <bool FAR>
__device__ __forceinline__ float power(float x, float m, float base, float unit) {
    return exp2_fast(FAR ? (x - m) * unit : fmaf(x, unit, -base));
}

__device__ __forceinline__ float power_of(float x, float m, float base, float unit) {
    return far(m, unit) ? power<true>(x, m, base, unit) : power<false>(x, m, base, unit);
}

// --- entries -------------------------------------------------------------------------------------------------
// A warp a row.  Of each entry: p, the teacher's share; mass, that of all entries with its index; near, the student's
// logit there; where, its index, -1 where it has none.  Also the row's weight, 0 where it has no entry, and for the mean
// the sum of 8 rows' weights.  (Made by a warp of the row's CTA, their chain of loads was waited for at every row:
// 4096 x 50257 of bf16 took 240 us.)

template <typename T>
__global__ void __launch_bounds__(32 * PART) entry_kernel(const __grid_constant__ Distill p, float *parts) {
    static_assert(BITS == 1 << 13, "the hash keeps 13 bits");
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ float sum[PART];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int k = (int)p.K, k4 = (k + 3) & ~3;
    float *a = reinterpret_cast<float *>(smem) + warp * (2 * k4 + BITS / 32);
    int *where = reinterpret_cast<int *>(a + k4);
    uint32_t *seen = reinterpret_cast<uint32_t *>(where + k4);
    const int64_t r = (int64_t)blockIdx.x * PART + warp;
    float weight = r < p.M ? weight_of(p, r) : 0.0f;
    if (weight != 0.0f) {
        float *out = p.block + r * 4 * k4;
        const T *from = static_cast<const T *>(p.logits) + place(p, r, p.so, p.si);
        float top = ninf();
        bool some = false;
#pragma unroll 4
        for (int i = lane; i < k; i += 32) {
            const int64_t j = index_of(p, r, i);
            const float t = j >= 0 ? load_as(p.teacher, r * p.ldt + i, p.t_dtype) : ninf();
            out[2 * k4 + i] = j >= 0 ? to_f(from[j]) : 0.0f;
            reinterpret_cast<int *>(out)[3 * k4 + i] = where[i] = (int)j;
            a[i] = t;
            some |= !(t == ninf());
            top = fmaxf(top, t);
        }
        if (__any_sync(0xffffffffu, some)) {
            for (int i = lane; i < BITS / 32; i += 32) seen[i] = 0;
            top = warp_max(top);
            float total = 0.0f;
            for (int i = lane; i < k; i += 32) total += a[i] = a[i] == ninf() ? 0.0f : exp2_fast((a[i] - top) * p.unit);
            const float inv = __fdiv_rn(1.0f, warp_sum(total));
            for (int i = lane; i < k; i += 32) out[i] = out[k4 + i] = a[i] *= inv;
            __syncwarp();
            // An entry that finds its index's bit set may have come before: those are compared with all.
            for (int i0 = 0; i0 < k; i0 += 32) {
                const int j = i0 + lane < k ? where[i0 + lane] : -1;
                const uint32_t h = ((uint32_t)j * 0x9E3779B1u) >> 19;
                const bool again = j >= 0 && (atomicOr(&seen[h / 32], 1u << (h % 32)) >> (h % 32) & 1u);
                for (uint32_t left = __ballot_sync(0xffffffffu, again); left; left &= left - 1) {
                    const int mine = __shfl_sync(0xffffffffu, j, __ffs(left) - 1);
                    float all = 0.0f;
                    for (int n = lane; n < k; n += 32)
                        if (where[n] == mine) all += a[n];
                    all = warp_sum(all);
                    for (int n = lane; n < k; n += 32)
                        if (where[n] == mine) out[k4 + n] = all;
                }
            }
        } else {
            weight = 0.0f;
        }
    }
    if (lane == 0) {
        if (r < p.M) p.weights[r] = weight;
        sum[warp] = weight;
    }
    __syncthreads();
    if (threadIdx.x == 0 && blockIdx.x == 0 && p.ended) *p.ended = 0;
    if (threadIdx.x == 0 && parts) {
        for (int i = 1; i < PART; i++) weight += sum[i];
        parts[blockIdx.x] = weight;
    }
}

// --- a row ---------------------------------------------------------------------------------------------------

struct Shared {
    float2 soft[2][8 * (WARPS + 1)];     // (maximum, sum) of every warp of the cluster
    unsigned long long bar[2];
    unsigned long long done;             // counts the warps that have written their part of a row's gradient
    unsigned long long left;             // the first row at which a warp has left the exchange
    float share[ALL / 32];
    int last;
};

constexpr unsigned long long NONE = ~0ull;

constexpr unsigned kSpinLimit = 1u << 26;             // polls of one wait, some seconds

__device__ unsigned long long g_failures;             // CTAs that gave up a wait

// A row's exchange.  Every warp sends its part to every CTA of the cluster, each part counted by the receiver's barrier:
// a cluster's own barrier also waits until the row before has reached memory.  Places and barriers alternate between two:
// a part of the row after next is sent once the next row's are complete, that is, after all have read this row's.
__device__ __forceinline__ void send_part(Shared &s, int turn, uint32_t n, uint32_t rank, float2 v) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    __syncwarp();
    if (lane >= (int)n) return;
    uint32_t place, bar;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(place) : "r"((uint32_t)__cvta_generic_to_shared(&s.soft[turn][rank * (WARPS + 1) + warp])), "r"(lane));
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(bar) : "r"((uint32_t)__cvta_generic_to_shared(&s.bar[turn])), "r"(lane));
    asm volatile("st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.v2.f32 [%0], {%1, %2}, [%3];" ::"r"(place), "f"(v.x),
                 "f"(v.y), "r"(bar)
                 : "memory");
}

// False where the wait has run out, for the whole warp.  It sends and waits no more then: parts of a later row would be
// counted as this one's by a CTA that is still at it, and the others' waits run out in turn.
__device__ __forceinline__ bool wait_for(const unsigned long long &on, int parity, unsigned spin) {
    const uint32_t bar = (uint32_t)__cvta_generic_to_shared(&on);
    uint32_t ok = 0;
    for (unsigned i = 0; !ok && i < spin; i++)
        asm volatile(
            "{\n\t.reg .pred q;\n\t"
            "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 q, [%1], %2;\n\t"
            "selp.u32 %0, 1, 0, q;\n\t}"
            : "=r"(ok)
            : "r"(bar), "r"(parity)
            : "memory");
    return __all_sync(0xffffffffu, ok);
}

// What a part's sum is multiplied with where the whole has the maximum m, of base `base`; a part of nothing is (-inf, 0).
// Where one side is far and the other is not, what a base is rounded by counts.
__device__ __noinline__ float factor_far(float x, float m, float unit) {
    if (x == m || x == ninf()) return x == m ? 1.0f : 0.0f;
    return exp2_fast(fmaf(x - m, unit, far(x, unit) ? 0.0f : -fmaf(x, unit, -base_of(x, unit))));
}

// (the rows that hardly occur in a function of their own: within this one they cost all others 1.5 us of 179)
__device__ __forceinline__ float factor_of(float x, float m, float base, float unit) {
    if (m == ninf() || far(m, unit)) return factor_far(x, m, unit);
    const float at = __fmul_rn(x, unit);              // (the base of the part's sum, rounded as it is)
    float e = at - base;
    if (e > -200.0f && at < -BORDER) e += fmaf(x, unit, -at);    // a far x; below -200 there is nothing
    return exp2_fast(e);
}

// (maximum, sum of the powers) of a warp's parts: the same in all lanes
__device__ __forceinline__ float2 soft_warp(float2 v, float unit) {
    const float m = warp_max(v.x);
    return make_float2(m, warp_sum(v.y * factor_of(v.x, m, base_of(m, unit), unit)));
}

// of all warps of the cluster
__device__ __forceinline__ float2 soft_all(const float2 *parts, int count, float unit) {
    const int lane = threadIdx.x & 31;
    float m = ninf(), sum = 0.0f;
    for (int i = lane; i < count; i += 32) m = fmaxf(m, parts[i].x);
    m = warp_max(m);
    const float base = base_of(m, unit);
    for (int i = lane; i < count; i += 32) sum = fmaf(parts[i].y, factor_of(parts[i].x, m, base, unit), sum);
    return make_float2(m, warp_sum(sum));
}

// the largest of a vector's elements, a NaN left out
template <typename T> __device__ __forceinline__ float max16(uint4 q) {
    if constexpr (sizeof(T) == 4) {
        return fmaxf(fmaxf(__uint_as_float(q.x), __uint_as_float(q.y)), fmaxf(__uint_as_float(q.z), __uint_as_float(q.w)));
    } else if constexpr (std::is_same<T, __half>::value) {
        const __half2 m = __hmax2(__hmax2(reinterpret_cast<__half2 &>(q.x), reinterpret_cast<__half2 &>(q.y)),
                                  __hmax2(reinterpret_cast<__half2 &>(q.z), reinterpret_cast<__half2 &>(q.w)));
        const float2 f = __half22float2(m);
        return fmaxf(f.x, f.y);
    } else {
        const __nv_bfloat162 m = __hmax2(__hmax2(reinterpret_cast<__nv_bfloat162 &>(q.x), reinterpret_cast<__nv_bfloat162 &>(q.y)),
                                         __hmax2(reinterpret_cast<__nv_bfloat162 &>(q.z), reinterpret_cast<__nv_bfloat162 &>(q.w)));
        const uint32_t w = reinterpret_cast<const uint32_t &>(m);
        return fmaxf(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
    }
}

// A CTA's part of a row.  Positions count from the 16-byte border before the row: element j is at j + lead.
template <typename T> struct Part {
    const T *from, *at;                  // the row; the address of the part's first position (not read before the row)
    int64_t first;                       // the part's first position
    int lead;
    int vectors, inside;                 // of 16 bytes, those that shared memory holds
    int begin, end;                      // elements of the row lie from `begin` to `end`, from the part's first position on
    int lo, hi;                          // vectors within the logits' memory: those around a row's ends are its neighbours'
};

template <typename T>
__device__ __forceinline__ Part<T> part_of(const Distill &p, int64_t r, uint32_t rank) {
    constexpr int E = Wide<T>::E;
    Part<T> q;
    q.from = static_cast<const T *>(p.logits) + place(p, r, p.so, p.si);
    q.lead = (int)((reinterpret_cast<uintptr_t>(q.from) & 15) / sizeof(T));
    q.first = (int64_t)rank * p.chunk;
    q.at = q.from - q.lead + q.first;
    q.begin = rank ? 0 : q.lead;
    q.end = (int)max(min((int64_t)p.chunk, p.V + q.lead - q.first), (int64_t)0);
    q.vectors = (q.end + E - 1) / E;
    q.inside = min(q.vectors, p.held / E);
    const T *base = static_cast<const T *>(p.logits);
    q.lo = q.at < base;
    q.hi = q.vectors - (q.at + (int64_t)q.vectors * E > base + p.last);
    return q;
}

// whether all elements of vector i are the row's
template <typename T> __device__ __forceinline__ bool whole(const Part<T> &q, int i) {
    return i * Wide<T>::E >= q.begin && (i + 1) * Wide<T>::E <= q.end;
}

// the vector i from memory, what is not the row's as -inf
template <typename T>
__device__ __forceinline__ uint4 vector_at(const Part<T> &q, int i) {
    constexpr int E = Wide<T>::E;
    if (whole(q, i)) return __ldg(reinterpret_cast<const uint4 *>(q.at + (int64_t)i * E));
    float v[E];
#pragma unroll
    for (int j = 0; j < E; j++) v[j] = i * E + j >= q.begin && i * E + j < q.end ? to_f(q.at[(int64_t)i * E + j]) : ninf();
    return close16<T>(v);
}

// this thread's copies of the row, as one group
template <typename T>
__device__ __forceinline__ void copy_row(const Part<T> &q, T *row, bool live) {
    constexpr int E = Wide<T>::E;
    if (live) {
        const uint32_t to = (uint32_t)__cvta_generic_to_shared(row);
        const int stop = min(q.inside, q.hi);
        for (int i = threadIdx.x; i < stop; i += THREADS)
            if (i >= q.lo)
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to + i * 16), "l"(q.at + (int64_t)i * E) : "memory");
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
}

// What a CTA that gave up a wait leaves of the row `r` and of those after it: NaN, and 0 as ever where a row does not count.
template <typename T, bool GRAD>
__device__ __noinline__ void lost_rows(const Distill &p, int64_t r, int64_t step, uint32_t rank) {
    for (; r < p.M; r += step) {
        const float lost = p.weights[r] != 0.0f ? __int_as_float(0x7FC00000) : 0.0f;
        if (rank == 0 && threadIdx.x == 0) {
            p.rows[r] = lost;
            if (p.stats) p.stats[3 * r] = p.stats[3 * r + 1] = p.stats[3 * r + 2] = lost;
        }
        if constexpr (GRAD) {
            const Part<T> q = part_of<T>(p, r, rank);
            T *to0 = static_cast<T *>(p.grad) + place(p, r, p.go, p.gi) - q.lead + q.first;
            for (int u = q.begin + threadIdx.x; u < q.end; u += ALL) to0[u] = from_f<T>(lost);
        }
    }
}

// --- a row's kernel ------------------------------------------------------------------------------------------

template <typename T, bool GRAD>
__global__ void __launch_bounds__(ALL, 4) row_kernel(const __grid_constant__ Distill p) {
    constexpr int E = Wide<T>::E;
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ Shared s;
    const int k4 = (int)((p.K + 3) & ~3);
    float *entries = reinterpret_cast<float *>(smem);                 // two rows' p, mass, near, where
    T *row = reinterpret_cast<T *>(entries + 8 * k4);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t n = cluster_size(), rank = cluster_rank();
    const int64_t step = gridDim.x / n;
    const uint32_t expected = n * (WARPS + 1) * 8;    // bytes of a row's parts
    if (tid == 0) {
        for (int i = 0; i < 2; i++) {
            const uint32_t bar = (uint32_t)__cvta_generic_to_shared(&s.bar[i]);
            asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(bar) : "memory");
        }
        asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"((uint32_t)__cvta_generic_to_shared(&s.done)), "n"(WARPS) : "memory");
        s.left = NONE;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (n > 1) cluster_barrier();                     // the others' barriers are set
    else __syncthreads();
    float share = 1.0f;                               // of a row's loss, before its weight
    if (p.parts) {
        float w = 0.0f;
        for (int64_t i = tid; i < p.n_parts; i += ALL) w += p.parts[i];
        w = warp_sum(w);
        if (lane == 0) s.share[warp] = w;
        __syncthreads();
        w = s.share[0];
        for (int i = 1; i < ALL / 32; i++) w += s.share[i];
        share = w == 0.0f ? 0.0f : __fdiv_rn(1.0f, w);
    }
    int turn = 0, parity = 0;
    int64_t left = -1;                                // the row at which a wait of this warp has run out
    const int64_t r0 = blockIdx.x / n;
    if (warp < WARPS) {
        float weight = p.weights[r0], next = r0 + step < p.M ? p.weights[r0 + step] : 0.0f;
        Part<T> ahead = part_of<T>(p, r0, rank);
        copy_row(ahead, row, weight != 0.0f);
        for (int64_t r = r0; r < p.M; r += step) {
            const bool live = weight != 0.0f;
            const Part<T> q = ahead;
            if (tid == 0)
                asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(
                                 (uint32_t)__cvta_generic_to_shared(&s.bar[turn])),
                             "r"(expected + (p.stall ? 8 : 0))
                             : "memory");
            const float after = r + 2 * step < p.M ? p.weights[r + 2 * step] : 0.0f;
            asm volatile("cp.async.wait_group 0;" ::: "memory");
            float2 soft = make_float2(ninf(), 0.0f);
            if (live) {
                // the vectors around the row's ends: what is not the row's becomes -inf
                auto mend = [&](int i) {
                    if (i >= q.inside || i % THREADS != tid || whole(q, i)) return;
                    if (i >= q.lo && i < q.hi) {
#pragma unroll
                        for (int j = 0; j < E; j++)
                            if (i * E + j < q.begin || i * E + j >= q.end) row[i * E + j] = from_f<T>(ninf());
                    } else {
                        *reinterpret_cast<uint4 *>(row + i * E) = vector_at(q, i);
                    }
                };
                mend(0);
                mend(q.vectors - 1);
                asm volatile("" ::: "memory");        // (the elements written are read as vectors)
                float m = ninf();
#pragma unroll 4
                for (int i = tid; i < q.inside; i += THREADS) m = fmaxf(m, max16<T>(*reinterpret_cast<const uint4 *>(row + i * E)));
                for (int i = q.inside + tid; i < q.vectors; i += THREADS) m = fmaxf(m, max16<T>(vector_at(q, i)));
                const float base = base_of(m, p.unit);
                float sum[2] = {0.0f, 0.0f};
                auto add = [&](uint4 w, auto is_far) {
                    float v[E];
                    open16<T>(w, v);
#pragma unroll
                    for (int j = 0; j < E; j++) sum[j & 1] += power<decltype(is_far)::value>(v[j], m, base, p.unit);
                };
                if (far(m, p.unit)) {
                    for (int i = tid; i < q.inside; i += THREADS) add(*reinterpret_cast<const uint4 *>(row + i * E), std::true_type());
                    for (int i = q.inside + tid; i < q.vectors; i += THREADS) add(vector_at(q, i), std::true_type());
                } else {
#pragma unroll 2
                    for (int i = tid; i < q.inside; i += THREADS) add(*reinterpret_cast<const uint4 *>(row + i * E), std::false_type());
                    for (int i = q.inside + tid; i < q.vectors; i += THREADS) add(vector_at(q, i), std::false_type());
                }
                soft = soft_warp(make_float2(m, sum[0] + sum[1]), p.unit);
            }
            send_part(s, turn, n, rank, soft);
            if (!wait_for(s.bar[turn], parity, p.spin)) {
                left = r;
                break;
            }
            if constexpr (GRAD) {
                soft = soft_all(s.soft[turn], (int)n * (WARPS + 1), p.unit);
                const float base = base_of(soft.x, p.unit);
                const float scale = __fdiv_rn(1.0f, soft.y) * (weight * share * p.temperature);
                T *to = static_cast<T *>(p.grad) + place(p, r, p.go, p.gi);
                if (p.same) {
                    T *to0 = to - q.lead + q.first;
                    uint4 *out = reinterpret_cast<uint4 *>(to0);
                    // the vectors of the row alone, from `from` on `count` of them
                    const int from = q.begin > 0, count = max(q.end / E - from, 0);
                    if (!live) {
                        for (int i = tid; i < count; i += THREADS) out[from + i] = make_uint4(0, 0, 0, 0);
                    } else {
                        auto slope = [&](uint4 w, auto is_far) {
                            float v[E];
                            open16<T>(w, v);
#pragma unroll
                            for (int j = 0; j < E; j++) v[j] = power<decltype(is_far)::value>(v[j], soft.x, base, p.unit) * scale;
                            return close16<T>(v);
                        };
                        auto all = [&](auto is_far) {
                            // (a thread's vectors are those that it has copied)
#pragma unroll 2
                            for (int i = tid; i < q.inside; i += THREADS)
                                if ((unsigned)(i - from) < (unsigned)count) out[i] = slope(*reinterpret_cast<const uint4 *>(row + i * E), is_far);
                            for (int i = q.inside + tid; i < q.vectors; i += THREADS)
                                if ((unsigned)(i - from) < (unsigned)count) out[i] = slope(vector_at(q, i), is_far);
                        };
                        if (far(soft.x, p.unit)) all(std::true_type());
                        else all(std::false_type());
                    }
                    // the elements around them, fewer than a vector's at either end
                    if (warp == 0) {
                        const int head = from ? min(E, q.end) : 0, tail = max(q.end / E * E, head);
                        for (int u = lane; u < q.end - tail + head; u += 32) {
                            const int at = u < head ? u : tail + u - head;
                            if (at >= q.begin)
                                to0[at] = from_f<T>(live ? power_of(to_f(q.at[at]), soft.x, base, p.unit) * scale : 0.0f);
                        }
                    }
                } else {
                    // Rows of the gradient that lie differently: elements, a warp those of the vectors that its own lanes
                    // have copied (32 in a row), so that it waits for nobody else's copies and nobody for its reading.
                    T *to0 = to - q.lead + q.first;
                    __syncwarp();
                    for (int i0 = warp * 32; i0 < q.vectors; i0 += THREADS)
#pragma unroll
                        for (int j = 0; j < E; j++) {
                            const int u = i0 * E + j * 32 + lane;
                            if (u < q.begin || u >= q.end) continue;
                            float v = 0.0f;
                            if (live) v = power_of(to_f(u < q.inside * E ? row[u] : q.at[u]), soft.x, base, p.unit) * scale;
                            to0[u] = from_f<T>(v);
                        }
                    __syncwarp();                     // the next copies go over what was read here
                }
            }
            // the next row's copies, to where this thread has read what it needs
            if (r + step < p.M) {
                ahead = part_of<T>(p, r + step, rank);
                copy_row(ahead, row, next != 0.0f);
            }
            if constexpr (GRAD) {
                __syncwarp();
                if (lane == 0)
                    asm volatile("mbarrier.arrive.release.cta.shared::cta.b64 _, [%0];" ::"r"((uint32_t)__cvta_generic_to_shared(&s.done))
                                 : "memory");
            }
            weight = next;
            next = after;
            parity ^= turn;
            turn ^= 1;
        }
    } else {
        // the next row's entries are copied while this one's are used
        auto copy = [&](int64_t r, int i) {
            if (r < p.M)
                for (int j = lane; j < k4; j += 32)
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(
                                     (uint32_t)__cvta_generic_to_shared(entries + (i * k4 + j) * 4)),
                                 "l"(p.block + (r * k4 + j) * 4)
                                 : "memory");
            asm volatile("cp.async.commit_group;" ::: "memory");
        };
        float weight = p.weights[r0];
        copy(r0, 0);
        for (int64_t r = r0; r < p.M; r += step) {
            const float *e = entries + turn * 4 * k4, *mass = e + k4, *near = mass + k4;
            const int *where = reinterpret_cast<const int *>(near + k4);
            copy(r + step, turn ^ 1);
            const float next = r + step < p.M ? p.weights[r + step] : 0.0f;
            asm volatile("cp.async.wait_group 1;" ::: "memory");
            __syncwarp();
            const bool live = weight != 0.0f;         // (if not, its entries were not made)
            send_part(s, turn, n, rank, make_float2(ninf(), 0.0f));      // what it read of the row before is free
            if (!wait_for(s.bar[turn], parity, p.spin)) {
                left = r;
                break;
            }
            const float2 soft = soft_all(s.soft[turn], (int)n * (WARPS + 1), p.unit);
            const float base = base_of(soft.x, p.unit), inv = __fdiv_rn(1.0f, soft.y);
            if (rank == 0) {
                float loss = 0.0f;
                if (live) {
                    // p (log p - log q) in base 2; where that leaves float32's range (a logit of the type's lowest value) the
                    // difference of the logits itself, beside which the logarithms are nothing (but for a NaN, of a row
                    // with an infinity)
                    const float off = log2f(soft.y);
                    float low = 0.0f;
                    for (int i = lane; i < (int)p.K; i += 32) {
                        const float z = far(soft.x, p.unit) ? (near[i] - soft.x) * p.unit : fmaf(near[i], p.unit, -base);
                        if (e[i] == 0.0f) continue;
                        const bool in = z > -1e30f;
                        loss = fmaf(e[i], (in ? log2f(e[i]) - z : 0.0f) + off, loss);
                        if (!in) low = fmaf(e[i], soft.x - near[i], low);
                    }
                    loss = warp_sum(loss) * (0.69314718056f * p.temperature * p.temperature) * (weight * share);
                    if (__any_sync(0xffffffffu, low != 0.0f)) loss += warp_sum(low) * p.temperature * (weight * share);
                }
                if (lane == 0) {
                    p.rows[r] = loss;
                    if (p.stats) {
                        p.stats[3 * r] = soft.x;
                        p.stats[3 * r + 1] = inv;
                        p.stats[3 * r + 2] = live ? weight * share : 0.0f;
                    }
                }
            }
            if constexpr (GRAD) {
                // the elements with an entry, after the others have written the whole row (a warp that has left the
                // exchange does not say so: hence a wait with a limit here too)
                if (!wait_for(s.done, turn, p.spin)) {
                    left = r;
                    break;
                }
                T *to = static_cast<T *>(p.grad) + place(p, r, p.go, p.gi);
                const int64_t lo = (int64_t)rank * p.chunk - part_of<T>(p, r, rank).lead, hi = lo + p.chunk;     // of this CTA
                const float factor = weight * share * p.temperature;
                for (int i = lane; i < (int)p.K && live; i += 32)
                    if (where[i] >= 0 && where[i] >= lo && where[i] < hi)
                        to[where[i]] = from_f<T>(factor * fmaf(power_of(near[i], soft.x, base, p.unit), inv, -mass[i]));
            }
            weight = next;
            parity ^= turn;
            turn ^= 1;
            __syncwarp();                             // the row's entries have been read
        }
        asm volatile("cp.async.wait_group 0;" ::: "memory");
    }
    // (a CTA ends only once all parts sent to it have come, unless a wait ran out)
    if (left >= 0 && lane == 0) atomicMin(&s.left, (unsigned long long)left);
    __syncthreads();
    if (s.left != NONE) {
        lost_rows<T, GRAD>(p, (int64_t)s.left, step, rank);
        if (tid == 0) atomicAdd(&g_failures, 1ull);
        __syncthreads();
        if (n > 1) cluster_barrier();
    }
    // the last cluster to end adds the rows' losses up, in a fixed order (a launch of its own was 3 us, and 4 of the host's)
    if (!p.loss || rank != 0) return;
    if (tid == 0) {
        __threadfence();
        s.last = atomicAdd(p.ended, 1) == gridDim.x / n - 1;
    }
    __syncthreads();
    if (!s.last) return;
    __threadfence();
    float sum = 0.0f;
#pragma unroll 8
    for (int64_t i = tid; i < p.M; i += ALL) sum += __ldcg(p.rows + i);
    sum = warp_sum(sum);
    if (lane == 0) s.share[warp] = sum;
    __syncthreads();
    if (tid) return;
    for (int i = 1; i < ALL / 32; i++) sum += s.share[i];
    *p.loss = sum;
}

// --- the gradient alone --------------------------------------------------------------------------------------
// From what the forward pass kept: the row's statistics, and of each entry its index's share.  A CTA takes pieces of 8
// vectors a thread, all of their loads in flight.

constexpr int PIECE = 8, GT = 256;

template <typename T>
__global__ void __launch_bounds__(GT, 3) gradient_kernel(const __grid_constant__ Distill p) {
    constexpr int E = Wide<T>::E;
    if (p.skip && *p.upstream == 1.0f) return;
    const int tid = threadIdx.x, k4 = (int)((p.K + 3) & ~3);
    const int64_t pieces = (p.V + E - 1 + p.chunk - 1) / p.chunk;
    for (int64_t item = blockIdx.x; item < p.M * pieces; item += gridDim.x) {
        const int64_t r = item / pieces;
        const Part<T> q = part_of<T>(p, r, (uint32_t)(item % pieces));
        const float top = p.stats[3 * r], inv = p.stats[3 * r + 1], share = p.stats[3 * r + 2];
        const float base = base_of(top, p.unit);
        const float factor = share * p.temperature * p.upstream[p.each ? r : 0];
        const bool counts = share != 0.0f;
        const float scale = inv * factor;
        T *to = static_cast<T *>(p.grad) + place(p, r, p.go, p.gi), *to0 = to - q.lead + q.first;
        if (p.same) {
            uint4 w[PIECE];
#pragma unroll
            for (int n = 0; n < PIECE; n++) {
                const int i = tid + n * GT;
                w[n] = make_uint4(0, 0, 0, 0);
                if (i < q.vectors && counts) w[n] = vector_at(q, i);
            }
#pragma unroll
            for (int n = 0; n < PIECE; n++) {
                const int i = tid + n * GT;
                if (i >= q.vectors) continue;
                float v[E];
                open16<T>(w[n], v);
#pragma unroll
                for (int j = 0; j < E; j++) v[j] = counts ? power_of(v[j], top, base, p.unit) * scale : 0.0f;
                if (whole(q, i)) {
                    *reinterpret_cast<uint4 *>(to0 + (int64_t)i * E) = close16<T>(v);
                } else {
#pragma unroll
                    for (int j = 0; j < E; j++)
                        if (i * E + j >= q.begin && i * E + j < q.end) to0[(int64_t)i * E + j] = from_f<T>(v[j]);
                }
            }
        } else {
#pragma unroll 4
            for (int u = q.begin + tid; u < q.end; u += GT)
                to0[u] = from_f<T>(counts ? power_of(to_f(q.at[u]), top, base, p.unit) * scale : 0.0f);
        }
        __syncthreads();                              // the elements with an entry are written again, after that
        const float *mass = p.block + (r * 4 + 1) * k4, *near = mass + k4;
        for (int i = tid; i < p.K && counts; i += GT) {
            const int j = reinterpret_cast<const int *>(near + k4)[i];
            if (j >= 0 && j + q.lead - q.first >= q.begin && j + q.lead - q.first < q.end)
                to[j] = from_f<T>(factor * fmaf(power_of(near[i], top, base, p.unit), inv, -mass[i]));
        }
    }
}

// --- launches ------------------------------------------------------------------------------------------------

constexpr int64_t ROOM = 53 * 1024;      // dynamic shared memory of a CTA of which four fit an SM

// the kernel's shared memory, once a device and context
template <typename K>
int allow(K *kernel, unsigned long long (&ready)[64], int64_t bytes) {
    static std::mutex lock;
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64)
        return set_error(SFB_ECUDA, "sf distillation: no current CUDA device");
    std::lock_guard<std::mutex> g(lock);
    const unsigned long long ctx = context_id();
    if (ctx == 0 || ready[dev] != ctx) {
        if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes) != cudaSuccess)
            return check_launch("sf distillation (attributes)");
        ready[dev] = context_id();
    }
    return SFB_OK;
}

template <typename T>
int launch_entries(const Distill &p, float *parts, cudaStream_t st) {
    static unsigned long long ready[64] = {};
    const int64_t blocks = (p.M + PART - 1) / PART;
    if (blocks >= 1ll << 31) return set_error(SFB_ERANGE, "sf distillation: %lld rows", (long long)p.M);
    auto bytes = [](int64_t k) { return PART * 4 * (2 * ((k + 3) & ~3ll) + BITS / 32); };
    const int rc = allow(entry_kernel<T>, ready, bytes(MAX_K));
    if (rc) return rc;
    entry_kernel<T><<<(unsigned)blocks, 32 * PART, (size_t)bytes(p.K), st>>>(p, parts);
    return check_launch("sf distillation (entries)");
}

template <typename T, bool GRAD>
int launch_rows(Distill p, cudaStream_t st) {
    static unsigned long long ready[64] = {};
    const int rc = allow(row_kernel<T, GRAD>, ready, ROOM);
    if (rc) return rc;
    constexpr int64_t E = 16 / sizeof(T);
    const int64_t entries = 32 * ((p.K + 3) & ~3ll), room = (ROOM - entries) / 16 * E, span = p.V + E - 1;
    auto chunk_of = [&](int64_t c) { return ((span + c - 1) / c + E - 1) / E * E; };
    int64_t c = 1;
    // A cluster as large as lets shared memory hold its part; larger ones where rows are few, a chunk being 4096
    // elements at least.
    while (c < 8 && (chunk_of(c) > room || (p.M * c < 2 * sm_count() && chunk_of(2 * c) >= 4096))) c *= 2;
    p.chunk = (int)chunk_of(c);
    p.held = (int)std::min<int64_t>(p.chunk, room);
    cudaLaunchConfig_t cfg{};
    cfg.blockDim = dim3(ALL);
    cfg.dynamicSmemBytes = (size_t)(entries + p.held * (int64_t)sizeof(T));
    cfg.gridDim = dim3((unsigned)c);
    cfg.stream = st;
    cudaLaunchAttribute a{};
    a.id = cudaLaunchAttributeClusterDimension;
    a.val.clusterDim.x = (unsigned)c;
    a.val.clusterDim.y = a.val.clusterDim.z = 1;
    cfg.attrs = &a;
    cfg.numAttrs = 1;
    // No more clusters than the GPU has room for: what waits for a place would begin its rows when all others end theirs.
    static std::mutex lock;
    static struct { unsigned long long ctx; size_t bytes; int64_t c; int clusters; } known;
    int clusters = 0;
    const unsigned long long ctx = context_id();
    {
        std::lock_guard<std::mutex> g(lock);
        if (ctx != 0 && known.ctx == ctx && known.bytes == cfg.dynamicSmemBytes && known.c == c) clusters = known.clusters;
    }
    if (clusters == 0) {
        if (cudaOccupancyMaxActiveClusters(&clusters, row_kernel<T, GRAD>, &cfg) != cudaSuccess)
            return check_launch("sf distillation (clusters)");
        if (clusters < 1) return set_error(SFB_ECUDA, "sf distillation: no room for a cluster of %d", (int)c);
        std::lock_guard<std::mutex> g(lock);
        known = {ctx, cfg.dynamicSmemBytes, c, clusters};
    }
    cfg.gridDim = dim3((unsigned)(std::min<int64_t>(p.M, clusters) * c));
    cudaLaunchKernelEx(&cfg, row_kernel<T, GRAD>, p);
    return check_launch("sf distillation");
}

template <typename T>
int launch_forward(const Distill &p, float *parts, cudaStream_t st) {
    const int rc = launch_entries<T>(p, parts, st);
    if (rc) return rc;
    return p.grad ? launch_rows<T, true>(p, st) : launch_rows<T, false>(p, st);
}

template <typename T>
int launch_gradient(Distill p, cudaStream_t st) {
    constexpr int64_t E = 16 / sizeof(T);
    p.chunk = (int)(PIECE * GT * E);
    p.held = 0;
    const int64_t pieces = (p.V + E - 1 + p.chunk - 1) / p.chunk;
    gradient_kernel<T><<<(unsigned)std::min<int64_t>(p.M * pieces, 3 * sm_count()), GT, 0, st>>>(p);
    return check_launch("sf distillation (backward)");
}

bool is_float(int64_t t) { return t == SFB_F32 || t == SFB_BF16 || t == SFB_F16; }

int check(const sfb_distill_call *c, const char *what, bool forward) {
    if (!c) return set_error(SFB_EINVAL, "%s: null pointer", what);
    if (!is_float(c->dtype) || !is_float(c->t_dtype))
        return set_error(SFB_EINVAL, "%s: element types %d and %d", what, (int)c->dtype, (int)c->t_dtype);
    if (c->w_dtype != SFB_WEIGHT_NONE && c->w_dtype != SFB_WEIGHT_BYTES && !is_float(c->w_dtype))
        return set_error(SFB_EINVAL, "%s: the weights' type %d", what, (int)c->w_dtype);
    if (c->M < 0 || c->V < 1 || c->K < 0 || c->inner < 1 || c->so < 0 || c->si < 0 || c->go < 0 || c->gi < 0 || c->ldt < c->K || c->ldi < c->K)
        return set_error(SFB_EINVAL, "%s: bad shape", what);
    if (c->V >= (1ll << 31) - 4096) return set_error(SFB_ERANGE, "%s: a vocabulary of %lld", what, (long long)c->V);
    if (c->K > MAX_K) return set_error(SFB_ERANGE, "%s: %lld entries a row, %d at most", what, (long long)c->K, MAX_K);
    if (!(c->temperature > 0.0) || !(c->temperature <= 1e6) || !(c->temperature >= 1e-6))
        return set_error(SFB_EINVAL, "%s: a temperature is between 1e-6 and 1e6", what);
    if (c->reduction < SFB_REDUCE_NONE || c->reduction > SFB_REDUCE_MEAN)
        return set_error(SFB_EINVAL, "%s: reduction %d", what, (int)c->reduction);
    if (c->M > 0 && (!c->logits || (c->K > 0 && !c->block) ||
                     (forward && ((c->K > 0 && (!c->teacher || !c->index)) || (c->w_dtype != SFB_WEIGHT_NONE && !c->weight)))))
        return set_error(SFB_EINVAL, "%s: null pointer", what);
    const uintptr_t size = size_of(c->dtype);
    if (!lies_on(c->block, 16)) return set_error(SFB_EINVAL, "%s: the entries' scratch starts on 16 bytes", what);
    if (!lies_on(c->logits, size) || !lies_on(c->grad, size) || !lies_on(c->teacher, size_of(c->t_dtype)) ||
        !lies_on(c->index, c->i_long ? 8 : 4) || (is_float(c->w_dtype) && !lies_on(c->weight, size_of(c->w_dtype))))
        return set_error(SFB_EINVAL, "%s: an operand does not start on an element", what);
    for (const void *p : {static_cast<const float *>(c->loss), static_cast<const float *>(c->rows), static_cast<const float *>(c->parts),
                          static_cast<const float *>(c->weights), static_cast<const float *>(c->stats), c->upstream})
        if (!lies_on(p, 4)) return set_error(SFB_EINVAL, "%s: a float32 buffer does not start on an element", what);
    return SFB_OK;
}

Distill distill_of(const sfb_distill_call *c) {
    Distill p{};
    p.logits = c->logits;
    p.teacher = c->teacher;
    p.index = c->index;
    p.weight = c->weight;
    p.stats = c->stats;
    p.block = c->block;
    p.weights = c->weights;
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
    p.spin = wait_polls() ? wait_polls() : kSpinLimit;
    p.stall = wait_stall();
    if (c->M > 0) {
        const int64_t outer = (c->M - 1) / c->inner, in = std::min(c->M, c->inner) - 1;
        p.last = outer * c->so + in * c->si + c->V;
        if (outer > 0) p.last = std::max(p.last - in * c->si + ((c->M - 1) % c->inner) * c->si, (outer - 1) * c->so + in * c->si + c->V);
    }
    // the rows of both lie alike on 16 bytes
    const int64_t size = c->dtype == SFB_F32 ? 4 : 2;
    p.same = c->grad && ((reinterpret_cast<uintptr_t>(c->logits) ^ reinterpret_cast<uintptr_t>(c->grad)) & 15) == 0 &&
             (c->so - c->go) * size % 16 == 0 && (c->si - c->gi) * size % 16 == 0;
    return p;
}

}  // namespace
}  // namespace sfb

extern "C" int sfb_distill_failures(int64_t *count) {
    using namespace sfb;
    unsigned long long n = 0;
    if (!count) return set_error(SFB_EINVAL, "sfb_distill_failures: null pointer");
    if (cudaMemcpyFromSymbol(&n, g_failures, sizeof n) != cudaSuccess) return check_launch("sfb_distill_failures");
    *count = (int64_t)n;
    return SFB_OK;
}

extern "C" int64_t sfb_distill_parts(int64_t M) { return M > 0 ? (M + sfb::PART - 1) / sfb::PART : 0; }

extern "C" int sfb_distill_forward(const sfb_distill_call *c, sfb_stream stream) {
    using namespace sfb;
    const char *what = "sfb_distill_forward";
    int rc = check(c, what, true);
    if (rc) return rc;
    const bool mean = c->reduction == SFB_REDUCE_MEAN, one = c->reduction != SFB_REDUCE_NONE;
    if ((one && !c->loss) || (c->M > 0 && (!c->rows || !c->weights || (mean && !c->parts))))
        return set_error(SFB_EINVAL, "%s: null pointer", what);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (c->M > 0) {
        Distill p = distill_of(c);
        p.rows = c->rows;
        p.loss = one ? c->loss : nullptr;
        p.ended = reinterpret_cast<unsigned *>(c->weights + c->M);
        float *parts = nullptr;
        if (mean) {
            p.n_parts = sfb_distill_parts(c->M);
            p.parts = parts = c->parts;
        }
        if (c->dtype == SFB_F32) rc = launch_forward<float>(p, parts, st);
        else if (c->dtype == SFB_BF16) rc = launch_forward<__nv_bfloat16>(p, parts, st);
        else rc = launch_forward<__half>(p, parts, st);
        if (rc) return rc;
    }
    if (!one || c->M > 0) return SFB_OK;
    return cudaMemsetAsync(c->loss, 0, sizeof(float), st) == cudaSuccess ? SFB_OK : check_launch("sf distillation (no rows)");
}

extern "C" int sfb_distill_backward(const sfb_distill_call *c, sfb_stream stream) {
    using namespace sfb;
    const char *what = "sfb_distill_backward";
    const int rc = check(c, what, false);
    if (rc) return rc;
    if (c->M == 0) return SFB_OK;
    if (!c->grad || !c->stats || !c->upstream) return set_error(SFB_EINVAL, "%s: null pointer", what);
    Distill p = distill_of(c);
    p.upstream = c->upstream;
    p.each = c->reduction == SFB_REDUCE_NONE;
    p.skip = c->skip != 0 && !p.each;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (c->dtype == SFB_F32) return launch_gradient<float>(p, st);
    if (c->dtype == SFB_BF16) return launch_gradient<__nv_bfloat16>(p, st);
    return launch_gradient<__half>(p, st);
}
