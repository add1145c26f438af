// Layer norm over the last dimension, forward and backward.
//
//   y  = xh w + b,  xh = (x - mean) r,  r = 1 / sqrt(var + eps)
//   dx = r (gy - mean(gy) - xh mean(gy xh)),  gy = dy w
//   dw = sum over rows of dy xh,  db = sum over rows of dy
//
// A row is read once and written once.  Bound by the wait for a row's sums: at 16384 x 4096 of bf16 neither
// DRAM (47 % of its rate forward, 63 % backward) nor issue (57 %, 70 %) is full.  The
// variance is taken from the deviations, not from a sum of squares, which would cancel where
// a row's mean is far from 0.  All sums are float32; results are rounded once.
// A row belongs to a team: a warp (up to 1024 elements), a CTA (up to 8192) or a cluster
// of up to 8 CTAs, which add their sums up through one another's shared memory.
// Teams take row after row, the next ones' copies in flight.  The backward pass keeps dw and db of a
// team's own columns in registers; what the teams leave, one row of partial sums for every
// CTA (or cluster), is added up by a second launch in a fixed order.
// 16384 x 4096 of bf16: forward 55 us (4.8 TB/s), backward 71 us (5.7 TB/s) and 7 for the sums.
#include <algorithm>
#include <mutex>

#include "sfb_tensor.cuh"

namespace sfb {

unsigned wait_polls();                        // the calling thread's sfb_wide_wait_limit
int wait_stall();

namespace {

constexpr int E = 8;                     // neighbouring elements of a thread
constexpr int TEAM = 512;                // threads of a CTA at most
constexpr int WIDE = TEAM * E * 2;       // elements of a row that a CTA has at most

struct Norm {
    const void *x, *dy;
    void *y, *dx;
    const void *w, *b;
    float *stats;                        // mean and r of every row
    float *parts;                        // rows of 2 D partial sums: dw, then db
    int64_t M, D, ldx, ldy, lddy, lddx;
    int w_dtype, b_dtype;
    float eps, share;                    // share = 1 / D
    unsigned spin;                       // polls of a wait
    int stall;                           // the tests': the first exchange never ends
};

constexpr unsigned kSpinLimit = 1u << 26;             // polls of one wait, some seconds

__device__ unsigned long long g_failures;             // CTAs that gave up a wait

// Where a thread's elements lie: E neighbouring ones (VEC: rows, weight and bias start on 16 bytes), or one in every
// `step`, so that unaligned accesses of a warp are to neighbouring elements.
template <bool VEC>
__device__ __forceinline__ int64_t place(int64_t base, int i, int j, int t, int step) {
    return VEC ? base + ((int64_t)i * step + t) * E + j : base + ((int64_t)i * E + j) * step + t;
}

template <typename T, bool VEC>
__device__ __forceinline__ void fetch(Vec<T, E> &q, const T *row, int64_t base, int i, int t, int step, int64_t end) {
    if constexpr (VEC) {
        const int64_t at = place<VEC>(base, i, 0, t, step);
        if (at + E <= end) {
            constexpr int P = 16 / sizeof(T);
#pragma unroll
            for (int h = 0; h < E / P; h++)
                *reinterpret_cast<uint4 *>(&q.v[h * P]) = *reinterpret_cast<const uint4 *>(row + at + h * P);
            return;
        }
    }
#pragma unroll
    for (int j = 0; j < E; j++) {
        const int64_t at = place<VEC>(base, i, j, t, step);
        q.v[j] = at < end ? row[at] : from_f<T>(0.0f);
    }
}

template <typename T, bool VEC>
__device__ __forceinline__ void put(T *row, const float (&v)[E], int64_t base, int i, int t, int step, int64_t end) {
    if constexpr (VEC) {
        const int64_t at = place<VEC>(base, i, 0, t, step);
        if (at + E <= end) {
            Vec<T, E> q;
#pragma unroll
            for (int j = 0; j < E; j++) q.v[j] = from_f<T>(v[j]);
            constexpr int P = 16 / sizeof(T);
#pragma unroll
            for (int h = 0; h < E / P; h++)
                *reinterpret_cast<uint4 *>(row + at + h * P) = *reinterpret_cast<const uint4 *>(&q.v[h * P]);
            return;
        }
    }
#pragma unroll
    for (int j = 0; j < E; j++) {
        const int64_t at = place<VEC>(base, i, j, t, step);
        if (at < end) row[at] = from_f<T>(v[j]);
    }
}

// a parameter's elements, `none` where there is no parameter
template <bool VEC>
__device__ __forceinline__ void param(float (&v)[E], const void *p, int dtype, float none, int64_t base, int i, int t,
                                      int step, int64_t end) {
    if (VEC && p && place<VEC>(base, i, 0, t, step) + E <= end) {
        const int64_t at = place<VEC>(base, i, 0, t, step);
        if (dtype == SFB_F32) {
            const float4 lo = __ldg(reinterpret_cast<const float4 *>(static_cast<const float *>(p) + at));
            const float4 hi = __ldg(reinterpret_cast<const float4 *>(static_cast<const float *>(p) + at) + 1);
            v[0] = lo.x, v[1] = lo.y, v[2] = lo.z, v[3] = lo.w, v[4] = hi.x, v[5] = hi.y, v[6] = hi.z, v[7] = hi.w;
        } else {
            const uint4 q = __ldg(reinterpret_cast<const uint4 *>(static_cast<const uint16_t *>(p) + at));
            const uint32_t h[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
            for (int j = 0; j < 4; j++) {
                if (dtype == SFB_BF16) {
                    v[2 * j] = __uint_as_float(h[j] << 16);
                    v[2 * j + 1] = __uint_as_float(h[j] & 0xFFFF0000u);
                } else {
                    const float2 f = __half22float2(reinterpret_cast<const __half2 &>(h[j]));
                    v[2 * j] = f.x;
                    v[2 * j + 1] = f.y;
                }
            }
        }
        return;
    }
#pragma unroll
    for (int j = 0; j < E; j++) {
        const int64_t at = place<VEC>(base, i, j, t, step);
        v[j] = p && at < end ? load_as(p, at, dtype) : none;
    }
}

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

// Sums over a team, known to all of it.  The places in shared memory alternate, so that one barrier a use is
// enough: what a use overwrites was read before the barrier of the use between.  Those of warps that a CTA does not have
// are zeros: the others are read four at a time (one at a time, in a loop, they were a third of the forward pass's
// instructions, which bound it).
// (a kernel for clusters of its own: with both in one, rows that a CTA holds took 34.8 us of 8192 x 4096 forward, not 32.8)
enum Of { WARPS, CTAS, CLUSTERS };

struct __align__(16) Team {
    float one[2][TEAM / 32];
    float2 two[2][TEAM / 32];
    float2 ctas[2][8];
    unsigned long long bar[2];
    int gave_up;
};

template <Of TO>
__device__ __forceinline__ void clear(Team &s) {
    if (threadIdx.x < TEAM / 32) {
        s.one[0][threadIdx.x] = s.one[1][threadIdx.x] = 0.0f;
        s.two[0][threadIdx.x] = s.two[1][threadIdx.x] = make_float2(0.0f, 0.0f);
    }
    if (TO == CLUSTERS && threadIdx.x == 0) {
        s.gave_up = 0;
        for (int i = 0; i < 2; i++)
            asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"((uint32_t)__cvta_generic_to_shared(&s.bar[i])) : "memory");
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if constexpr (TO == CLUSTERS) cluster_barrier();  // the others' barriers are set
    else __syncthreads();
}

// once all rows are done: a CTA ends only when all parts sent to it have come, unless a wait ran out
__device__ __forceinline__ void leave(Team &s) {
    __syncthreads();
    if (!s.gave_up) return;
    if (threadIdx.x == 0) atomicAdd(&g_failures, 1ull);
    cluster_barrier();
}

// Of the cluster's CTAs, each of which sends its part to all, counted by the receiver's barrier: a cluster's own barrier
// also waits until the row before has reached memory (bf16 forward and backward, 8192 x 8200: 425 us and 330, 4096 x
// 16384: 270 and 212).  Places and barriers alternate between two: a part of the use after next is sent once the next
// one's are complete, that is, after all have read this one's.  A wait that runs out makes the row NaN and ends the CTA's part in the exchange: the others'
// waits run out in turn, and nothing is on its way to a CTA that ends.
__device__ __forceinline__ float2 cluster_sum(float2 v, Team &s, int turn, uint32_t n, const Norm &p) {
    const int at = turn & 1, parity = turn >> 1 & 1;
    const uint32_t bar = (uint32_t)__cvta_generic_to_shared(&s.bar[at]);
    const bool fine = *reinterpret_cast<volatile int *>(&s.gave_up) == 0;
    if (threadIdx.x == 0 && fine)
        asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(n * 8 + (p.stall ? 8 : 0))
                     : "memory");
    if (threadIdx.x < n && fine) {
        uint32_t place, there;
        const uint32_t mine = (uint32_t)__cvta_generic_to_shared(&s.ctas[at][cluster_rank()]);
        asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(place) : "r"(mine), "r"((uint32_t)threadIdx.x));
        asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"(bar), "r"((uint32_t)threadIdx.x));
        asm volatile("st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.v2.f32 [%0], {%1, %2}, [%3];" ::"r"(place),
                     "f"(v.x), "f"(v.y), "r"(there)
                     : "memory");
    }
    uint32_t ok = 0;
    for (unsigned i = 0; fine && !ok && i < p.spin; i++)
        asm volatile(
            "{\n\t.reg .pred q;\n\t"
            "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 q, [%1], %2;\n\t"
            "selp.u32 %0, 1, 0, q;\n\t}"
            : "=r"(ok)
            : "r"(bar), "r"(parity)
            : "memory");
    if (!ok) {
        *reinterpret_cast<volatile int *>(&s.gave_up) = 1;
        return make_float2(__int_as_float(0x7FC00000), __int_as_float(0x7FC00000));
    }
    v = s.ctas[at][0];
    for (uint32_t i = 1; i < n; i++) v.x += s.ctas[at][i].x, v.y += s.ctas[at][i].y;
    return v;
}

template <Of TO>
__device__ __forceinline__ float team_sum(float v, Team &s, int &turn, const Norm &n) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if constexpr (TO != WARPS) {
        const int p = turn & 1;
        if ((threadIdx.x & 31) == 0) s.one[p][threadIdx.x >> 5] = v;
        __syncthreads();
        v = 0.0f;
#pragma unroll
        for (int i = 0; i < TEAM / 128; i++) {
            if (i * 128 >= (int)blockDim.x) break;
            const float4 q = reinterpret_cast<const float4 *>(s.one[p])[i];
            v += (q.x + q.y) + (q.z + q.w);
        }
        if constexpr (TO == CLUSTERS) v = cluster_sum(make_float2(v, 0.0f), s, turn, cluster_size(), n).x;
        turn++;
    }
    return v;
}

template <Of TO>
__device__ __forceinline__ float2 team_sum(float2 v, Team &s, int &turn, const Norm &n) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        v.x += __shfl_xor_sync(0xffffffffu, v.x, o);
        v.y += __shfl_xor_sync(0xffffffffu, v.y, o);
    }
    if constexpr (TO != WARPS) {
        const int p = turn & 1;
        if ((threadIdx.x & 31) == 0) s.two[p][threadIdx.x >> 5] = v;
        __syncthreads();
        v = make_float2(0.0f, 0.0f);
#pragma unroll
        for (int i = 0; i < TEAM / 128; i++) {
            if (i * 128 >= (int)blockDim.x) break;
            const float4 a = reinterpret_cast<const float4 *>(s.two[p])[2 * i], b = reinterpret_cast<const float4 *>(s.two[p])[2 * i + 1];
            v.x += (a.x + a.z) + (b.x + b.z);
            v.y += (a.y + a.w) + (b.y + b.w);
        }
        if constexpr (TO == CLUSTERS) v = cluster_sum(v, s, turn, cluster_size(), n);
        turn++;
    }
    return v;
}

// The team's place: its first row, the rows from one of its own to the next, its columns.
struct Place {
    int64_t row, rows, base, end;
    int t, step;
};

template <Of TO, int C>
__device__ __forceinline__ Place team_place(const Norm &p) {
    Place q;
    if constexpr (TO == WARPS) {
        q.row = (int64_t)blockIdx.x * (blockDim.x / 32) + threadIdx.x / 32;
        q.rows = (int64_t)gridDim.x * (blockDim.x / 32);
        q.base = 0;
        q.end = p.D;
        q.t = threadIdx.x & 31;
        q.step = 32;
    } else {
        const uint32_t n = TO == CLUSTERS ? cluster_size() : 1;
        q.row = blockIdx.x / n;
        q.rows = gridDim.x / n;
        q.t = threadIdx.x;
        q.step = blockDim.x;
        q.base = (int64_t)(TO == CLUSTERS ? cluster_rank() : 0) * q.step * C * E;
        q.end = min(p.D, q.base + (int64_t)q.step * C * E);
    }
    return q;
}

// A team's next rows: copies to shared memory, S - 1 rows ahead, of which a thread reads its own (nothing to
// synchronise).  With one row ahead in registers 16384 x 4096 of bf16 took 118 us backward, 32 KB an SM in flight.
// Unaligned rows have one row ahead in registers.
template <typename T, int C> struct Slot { static constexpr int H = E * sizeof(T) / 16, LINES = C * H; };   // lines of 16 bytes a thread

template <typename T, int C>
__device__ __forceinline__ void copy_in(uint32_t slot, const T *row, const Place &q) {
    constexpr int H = Slot<T, C>::H, P = 16 / sizeof(T);
#pragma unroll
    for (int i = 0; i < C; i++) {
        const int64_t at = place<true>(q.base, i, 0, q.t, q.step);
        const int bytes = at + E <= q.end ? 16 : 0;              // (else filled with zeros)
        const T *from = row + (bytes ? at : 0);
#pragma unroll
        for (int h = 0; h < H; h++)
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(slot + ((i * H + h) * blockDim.x + threadIdx.x) * 16),
                         "l"(from + h * P), "r"(bytes)
                         : "memory");
    }
}

template <typename T, int C>
__device__ __forceinline__ void copied(Vec<T, E> (&q)[C], const uint4 *slot) {
    constexpr int H = Slot<T, C>::H, P = 16 / sizeof(T);
#pragma unroll
    for (int i = 0; i < C; i++)
#pragma unroll
        for (int h = 0; h < H; h++) *reinterpret_cast<uint4 *>(&q[i].v[h * P]) = slot[(i * H + h) * blockDim.x + threadIdx.x];
}

template <typename T> struct Ahead { static constexpr int FORWARD = sizeof(T) == 2 ? 4 : 3, BACKWARD = sizeof(T) == 2 ? 3 : 2; };

template <typename T, bool VEC, Of TO, int C>
__global__ void __launch_bounds__(TO == WARPS ? 128 : TEAM) forward_kernel(const __grid_constant__ Norm p) {
    constexpr int S = Ahead<T>::FORWARD;
    extern __shared__ __align__(16) uint4 ring[];
    __shared__ Team s;
    int turn = 0;
    const Place q = team_place<TO, C>(p);
    if constexpr (TO != WARPS) clear<TO>(s);
    const int lines = Slot<T, C>::LINES * blockDim.x;
    const uint32_t at = (uint32_t)__cvta_generic_to_shared(ring);
    const T *x = static_cast<const T *>(p.x);
    float w[C][E], b[C][E];
#pragma unroll
    for (int i = 0; i < C; i++) {
        param<VEC>(w[i], p.w, p.w_dtype, 1.0f, q.base, i, q.t, q.step, q.end);
        param<VEC>(b[i], p.b, p.b_dtype, 0.0f, q.base, i, q.t, q.step, q.end);
    }
    Vec<T, E> raw[C];
    if constexpr (VEC) {
#pragma unroll
        for (int n = 0; n < S - 1; n++) {
            if (q.row + n * q.rows < p.M) copy_in<T, C>(at + n * lines * 16, x + (q.row + n * q.rows) * p.ldx, q);
            asm volatile("cp.async.commit_group;" ::: "memory");
        }
    } else if (q.row < p.M) {
#pragma unroll
        for (int i = 0; i < C; i++) fetch<T, VEC>(raw[i], x + q.row * p.ldx, q.base, i, q.t, q.step, q.end);
    }
    int slot = 0;
    for (int64_t r = q.row; r < p.M; r += q.rows) {
        if constexpr (VEC) {
            const int64_t next = r + (S - 1) * q.rows;
            if (next < p.M) copy_in<T, C>(at + (slot == 0 ? S - 1 : slot - 1) * lines * 16, x + next * p.ldx, q);
            asm volatile("cp.async.commit_group;" ::: "memory");
            asm volatile("cp.async.wait_group %0;" ::"n"(S - 1) : "memory");
            copied<T, C>(raw, ring + slot * lines);
            slot = slot == S - 1 ? 0 : slot + 1;
        }
        float v[C][E], sum = 0.0f;
#pragma unroll
        for (int i = 0; i < C; i++)
#pragma unroll
            for (int j = 0; j < E; j++) {
                v[i][j] = to_f(raw[i].v[j]);
                sum += v[i][j];
            }
        if constexpr (!VEC) {
            if (r + q.rows < p.M)
#pragma unroll
                for (int i = 0; i < C; i++) fetch<T, VEC>(raw[i], x + (r + q.rows) * p.ldx, q.base, i, q.t, q.step, q.end);
        }
        const float mean = team_sum<TO>(sum, s, turn, p) * p.share;
        sum = 0.0f;
#pragma unroll
        for (int i = 0; i < C; i++) {
            if (VEC && place<VEC>(q.base, i, 0, q.t, q.step) >= q.end) continue;       // (not stored either)
#pragma unroll
            for (int j = 0; j < E; j++) {
                v[i][j] = VEC || place<VEC>(q.base, i, j, q.t, q.step) < q.end ? v[i][j] - mean : 0.0f;
                sum = fmaf(v[i][j], v[i][j], sum);
            }
        }
        const float rs = rsqrtf(fmaf(team_sum<TO>(sum, s, turn, p), p.share, p.eps));
        if (p.stats && q.t == 0 && q.base == 0) *reinterpret_cast<float2 *>(p.stats + 2 * r) = make_float2(mean, rs);
        T *out = static_cast<T *>(p.y) + r * p.ldy;
#pragma unroll
        for (int i = 0; i < C; i++) {
            float y[E];
#pragma unroll
            for (int j = 0; j < E; j++) y[j] = fmaf(v[i][j] * rs, w[i][j], b[i][j]);
            put<T, VEC>(out, y, q.base, i, q.t, q.step, q.end);
        }
    }
    if constexpr (TO == CLUSTERS) leave(s);
}

template <typename T, bool VEC, Of TO, int C>
__global__ void __launch_bounds__(TO == WARPS ? 128 : TEAM, 1) backward_kernel(const __grid_constant__ Norm p) {
    constexpr int S = Ahead<T>::BACKWARD;
    extern __shared__ __align__(16) uint4 ring[];
    __shared__ Team s;
    __shared__ float joined[TO == WARPS ? 2 * 32 * C * E : 1];
    int turn = 0;
    const Place q = team_place<TO, C>(p);
    if constexpr (TO != WARPS) clear<TO>(s);
    const int lines = Slot<T, C>::LINES * blockDim.x;
    const uint32_t at = (uint32_t)__cvta_generic_to_shared(ring);
    const T *x = static_cast<const T *>(p.x), *dy = static_cast<const T *>(p.dy);
    float w[C][E], dw[C][E] = {}, db[C][E] = {};
#pragma unroll
    for (int i = 0; i < C; i++) param<VEC>(w[i], p.w, p.w_dtype, 1.0f, q.base, i, q.t, q.step, q.end);
    Vec<T, E> xr[C], gr[C];
    float2 stats = make_float2(0.0f, 0.0f);
    auto load = [&](int64_t r) {
#pragma unroll
        for (int i = 0; i < C; i++) {
            fetch<T, VEC>(xr[i], x + r * p.ldx, q.base, i, q.t, q.step, q.end);
            fetch<T, VEC>(gr[i], dy + r * p.lddy, q.base, i, q.t, q.step, q.end);
        }
    };
    auto copy = [&](int64_t r, int n) {
        if (r < p.M) {
            copy_in<T, C>(at + 2 * n * lines * 16, x + r * p.ldx, q);
            copy_in<T, C>(at + (2 * n + 1) * lines * 16, dy + r * p.lddy, q);
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    if constexpr (VEC) {
#pragma unroll
        for (int n = 0; n < S - 1; n++) copy(q.row + n * q.rows, n);
    } else if (q.row < p.M) {
        load(q.row);
    }
    if (q.row < p.M) stats = __ldg(reinterpret_cast<const float2 *>(p.stats) + q.row);
    int slot = 0;
    for (int64_t r = q.row; r < p.M; r += q.rows) {
        if constexpr (VEC) {
            copy(r + (S - 1) * q.rows, slot == 0 ? S - 1 : slot - 1);
            asm volatile("cp.async.wait_group %0;" ::"n"(S - 1) : "memory");
            copied<T, C>(xr, ring + 2 * slot * lines);
            copied<T, C>(gr, ring + (2 * slot + 1) * lines);
            slot = slot == S - 1 ? 0 : slot + 1;
        }
        // (elements past the row have a gradient of 0, and add nothing)
        float xh[C][E], gy[C][E];
        float2 sum = make_float2(0.0f, 0.0f);
        const float mean = stats.x, rs = stats.y;
#pragma unroll
        for (int i = 0; i < C; i++)
#pragma unroll
            for (int j = 0; j < E; j++) {
                const float g = to_f(gr[i].v[j]);
                xh[i][j] = (to_f(xr[i].v[j]) - mean) * rs;
                gy[i][j] = g * w[i][j];
                dw[i][j] = fmaf(g, xh[i][j], dw[i][j]);
                db[i][j] += g;
                sum.x += gy[i][j];
                sum.y = fmaf(gy[i][j], xh[i][j], sum.y);
            }
        if (r + q.rows < p.M) {
            if constexpr (!VEC) load(r + q.rows);
            stats = __ldg(reinterpret_cast<const float2 *>(p.stats) + r + q.rows);
        }
        sum = team_sum<TO>(sum, s, turn, p);
        const float a = sum.x * p.share, c = sum.y * p.share;
        if (p.dx) {
            T *out = static_cast<T *>(p.dx) + r * p.lddx;
#pragma unroll
            for (int i = 0; i < C; i++) {
                float d[E];
#pragma unroll
                for (int j = 0; j < E; j++) d[j] = rs * (gy[i][j] - a - xh[i][j] * c);
                put<T, VEC>(out, d, q.base, i, q.t, q.step, q.end);
            }
        }
    }
    if constexpr (TO == CLUSTERS) leave(s);
    if (!p.parts) return;
    if constexpr (TO == WARPS) {
        // the CTA's warps, one after another
        for (int n = 0; n < (int)blockDim.x / 32; n++) {
            if ((int)threadIdx.x / 32 == n)
#pragma unroll
                for (int i = 0; i < C; i++)
#pragma unroll
                    for (int j = 0; j < E; j++) {
                        const int o = (i * E + j) * 32 + q.t;
                        dw[i][j] += n ? joined[o] : 0.0f;
                        db[i][j] += n ? joined[32 * C * E + o] : 0.0f;
                        joined[o] = dw[i][j];
                        joined[32 * C * E + o] = db[i][j];
                    }
            __syncthreads();
        }
        if (threadIdx.x / 32 != blockDim.x / 32 - 1) return;
    }
    float *out = p.parts + (int64_t)(TO == WARPS ? blockIdx.x : q.row) * 2 * p.D;
    // (partial sums start on 16 bytes where D is a multiple of 4: VEC has multiples of 8)
#pragma unroll
    for (int i = 0; i < C; i++) {
        put<float, VEC>(out, dw[i], q.base, i, q.t, q.step, q.end);
        put<float, VEC>(out + p.D, db[i], q.base, i, q.t, q.step, q.end);
    }
}

// dw and db from `count` rows of partial sums: W columns a CTA, 512 / W sums to a column, joined in order.  8 columns (a
// sector of 32 bytes) where 32 would leave SMs idle: 768 features 5.7 us and 6.3, 4096 features 10.5 and 6.0.
template <int W>
__global__ void __launch_bounds__(512) join_kernel(const float *__restrict__ parts, int64_t count, int64_t D, void *dw,
                                                   int w_dtype, void *db, int b_dtype) {
    constexpr int H = 512 / W;
    __shared__ float s[H][W + 1];
    const int x = threadIdx.x % W, y = threadIdx.x / W;
    const int64_t c = (int64_t)blockIdx.x * W + x;
    float v = 0.0f;
    if (c < 2 * D) {
#pragma unroll 8
        for (int64_t i = y; i < count; i += H) v += parts[i * 2 * D + c];
    }
    s[y][x] = v;
    __syncthreads();
    if (y || c >= 2 * D) return;
#pragma unroll 8
    for (int i = 1; i < H; i++) v += s[i][x];
    if (c < D) {
        if (dw) store_as(dw, c, w_dtype, v);
    } else if (db) {
        store_as(db, c - D, b_dtype, v);
    }
}

// --- launches ------------------------------------------------------------------------------------------------

// How rows of D elements are dealt out: elements a thread and the team's threads.
struct Teams {
    bool warp;
    int chunks, threads, ctas;           // threads of a CTA, CTAs of a cluster
};

Teams teams_of(int64_t D) {
    Teams t{D <= 1024, 0, 128, 1};
    if (t.warp) {
        t.chunks = (int)((D + 32 * E - 1) / (32 * E));
    } else {
        while ((int64_t)t.ctas * WIDE < D) t.ctas *= 2;
        t.chunks = 2;
        const int64_t each = (D + t.ctas - 1) / t.ctas;
        t.threads = (int)((each + 64 * E - 1) / (64 * E)) * 32;
    }
    return t;
}

constexpr int64_t MOST = 8 * (int64_t)WIDE;

// CTAs (or clusters) that take rows of the backward pass in turn: as many as registers leave room for (128 a thread, 96 to
// 250 of a warp's kernels), so that none waits for another's end.
int64_t backward_teams(int64_t M, const Teams &t) {
    static const int of_warps[5] = {0, 5, 3, 2, 2};
    const int64_t per = t.warp ? of_warps[t.chunks] : std::max<int64_t>(1, 512 / t.threads);
    const int64_t rows = t.warp ? (M + 3) / 4 : M;
    return std::max<int64_t>(1, std::min<int64_t>(rows, per * sm_count() / t.ctas));
}

constexpr int RING = 160 * 1024;         // dynamic shared memory of a CTA at most

// A kernel's CUDA context whose attributes are set, per device, and how many CTAs of a size (clusters of 2, 4 or 8 of them)
// the device holds at once: more clusters than that are a second wave, as long as the first (2048 x 65536 of bf16 forward
// 405 us and 248, backward included 828 and 504)
struct Known {
    std::mutex lock;
    unsigned long long ctx[64];
    int at_once[64][4][TEAM / 32 + 1];
};

cudaLaunchConfig_t config(const Teams &t, int64_t grid, int64_t ring, cudaStream_t st, cudaLaunchAttribute &a) {
    cudaLaunchConfig_t c{};
    c.gridDim = dim3((unsigned)(grid * t.ctas));
    c.blockDim = dim3(t.threads);
    c.dynamicSmemBytes = (size_t)ring;
    c.stream = st;
    a = cudaLaunchAttribute{};
    a.id = cudaLaunchAttributeClusterDimension;
    a.val.clusterDim.x = t.ctas;
    a.val.clusterDim.y = a.val.clusterDim.z = 1;
    c.attrs = &a;
    c.numAttrs = t.ctas > 1 ? 1 : 0;
    return c;
}

// CTAs or clusters at once, 0 on an error
template <typename K>
int ready(K *kernel, Known &known, const Teams &t, int64_t ring, const char *what) {
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return set_error(0, "%s: no current CUDA device", what);
    std::lock_guard<std::mutex> g(known.lock);
    const unsigned long long ctx = context_id();
    if (ctx == 0 || known.ctx[dev] != ctx) {
        if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, RING) != cudaSuccess)
            return check_launch(what), 0;
        for (auto &sizes : known.at_once[dev])
            for (int &n : sizes) n = 0;
        known.ctx[dev] = context_id();
    }
    int &n = known.at_once[dev][t.ctas == 8 ? 3 : t.ctas / 2][t.threads / 32];
    if (n == 0) {
        int found = 0;
        cudaLaunchAttribute a;
        const cudaLaunchConfig_t c = config(t, sm_count(), ring, nullptr, a);
        if (t.ctas > 1 ? cudaOccupancyMaxActiveClusters(&found, kernel, &c) != cudaSuccess
                       : cudaOccupancyMaxActiveBlocksPerMultiprocessor(&found, kernel, t.threads, (size_t)ring) != cudaSuccess)
            return check_launch(what), 0;
        n = std::max(found, 1) * (t.ctas > 1 ? 1 : sm_count());
    }
    return n;
}

template <typename K>
int launch(K *kernel, const Norm &p, const Teams &t, int64_t grid, int64_t ring, cudaStream_t st, const char *what) {
    cudaLaunchAttribute a;
    const cudaLaunchConfig_t c = config(t, grid, ring, st, a);
    cudaLaunchKernelEx(&c, kernel, p);
    return check_launch(what);
}

template <typename T, bool VEC, Of TO, int C>
int forward(const Norm &p, const Teams &t, cudaStream_t st) {
    const int64_t ring = VEC ? Ahead<T>::FORWARD * Slot<T, C>::LINES * 16ll * t.threads : 0;
    static Known known;
    const char *what = "sf layer norm";
    const int at_once = ready(forward_kernel<T, VEC, TO, C>, known, t, ring, what);
    if (at_once == 0) return SFB_ECUDA;
    const int64_t rows = TO == WARPS ? (p.M + 3) / 4 : p.M;
    return launch(forward_kernel<T, VEC, TO, C>, p, t, std::min<int64_t>(rows, at_once), ring, st, what);
}

template <typename T, bool VEC, Of TO, int C>
int backward(const Norm &p, const Teams &t, cudaStream_t st, int64_t &teams) {
    const int64_t ring = VEC ? 2 * Ahead<T>::BACKWARD * Slot<T, C>::LINES * 16ll * t.threads : 0;
    static Known known;
    const char *what = "sf layer norm (backward)";
    const int at_once = ready(backward_kernel<T, VEC, TO, C>, known, t, ring, what);
    if (at_once == 0) return SFB_ECUDA;
    teams = backward_teams(p.M, t);
    if (TO == CLUSTERS) teams = std::min<int64_t>(teams, at_once);
    return launch(backward_kernel<T, VEC, TO, C>, p, t, teams, ring, st, what);
}

// the kernel for a type, alignment and length; backwards also how many rows of partial sums there are
template <typename T, bool VEC>
int run(const Norm &p, const Teams &t, int64_t *teams, cudaStream_t st) {
    using std::integral_constant;
    auto go = [&](auto to, auto chunks) {
        constexpr Of TO = decltype(to)::value;
        constexpr int C = decltype(chunks)::value;
        return teams ? backward<T, VEC, TO, C>(p, t, st, *teams) : forward<T, VEC, TO, C>(p, t, st);
    };
    const integral_constant<Of, WARPS> warps;
    if (t.ctas > 1) return go(integral_constant<Of, CLUSTERS>(), integral_constant<int, 2>());
    if (!t.warp) return go(integral_constant<Of, CTAS>(), integral_constant<int, 2>());
    switch (t.chunks) {
        case 1: return go(warps, integral_constant<int, 1>());
        case 2: return go(warps, integral_constant<int, 2>());
        case 3: return go(warps, integral_constant<int, 3>());
    }
    return go(warps, integral_constant<int, 4>());
}

int run(const Norm &p, int64_t dtype, bool vec, int64_t *teams, cudaStream_t st) {
    const Teams t = teams_of(p.D);
    if (dtype == SFB_F32) return vec ? run<float, true>(p, t, teams, st) : run<float, false>(p, t, teams, st);
    if (dtype == SFB_BF16) return vec ? run<__nv_bfloat16, true>(p, t, teams, st) : run<__nv_bfloat16, false>(p, t, teams, st);
    return vec ? run<__half, true>(p, t, teams, st) : run<__half, false>(p, t, teams, st);
}

bool is_float(int64_t t) { return t == SFB_F32 || t == SFB_BF16 || t == SFB_F16; }

bool rows16(const void *p, int64_t ld, int64_t size) {
    return p == nullptr || ((reinterpret_cast<uintptr_t>(p) & 15) == 0 && ld * size % 16 == 0);
}

int check(const sfb_norm_call *c, const char *what) {
    if (!c) return set_error(SFB_EINVAL, "%s: null pointer", what);
    if (!is_float(c->dtype)) return set_error(SFB_EINVAL, "%s: element type %d", what, (int)c->dtype);
    if (c->M < 0 || c->D < 1) return set_error(SFB_EINVAL, "%s: bad shape", what);
    if (c->D > MOST) return set_error(SFB_ERANGE, "%s: rows of %lld elements, %lld at most", what, (long long)c->D, (long long)MOST);
    if ((c->w && !is_float(c->w_dtype)) || (c->b && !is_float(c->b_dtype)))
        return set_error(SFB_EINVAL, "%s: a parameter's type", what);
    if (c->ldx < c->D || c->ldy < c->D) return set_error(SFB_EINVAL, "%s: a row stride is shorter than its row", what);
    if (c->M > 0 && (!c->x || !c->y)) return set_error(SFB_EINVAL, "%s: null pointer", what);
    if (!lies_on(c->stats, 8)) return set_error(SFB_EINVAL, "%s: the statistics start on 8 bytes", what);
    const uintptr_t size = size_of(c->dtype), w = size_of(c->w_dtype), b = size_of(c->b_dtype);
    if (!lies_on(c->x, size) || !lies_on(c->y, size) || !lies_on(c->dx, size) || !lies_on(c->w, w) || !lies_on(c->dw, w) ||
        !lies_on(c->b, b) || !lies_on(c->db, b))
        return set_error(SFB_EINVAL, "%s: an operand does not start on an element", what);
    return SFB_OK;
}

Norm norm_of(const sfb_norm_call *c) {
    Norm p{};
    p.x = c->x;
    p.w = c->w;
    p.b = c->b;
    p.stats = c->stats;
    p.M = c->M;
    p.D = c->D;
    p.ldx = c->ldx;
    p.w_dtype = (int)c->w_dtype;
    p.b_dtype = (int)c->b_dtype;
    p.eps = (float)c->eps;
    p.share = (float)(1.0 / (double)c->D);
    p.spin = wait_polls() ? wait_polls() : kSpinLimit;
    p.stall = wait_stall();
    return p;
}

}  // namespace
}  // namespace sfb

extern "C" int sfb_norm_forward(const sfb_norm_call *c, sfb_stream stream) {
    using namespace sfb;
    const char *what = "sfb_norm_forward";
    const int rc = check(c, what);
    if (rc) return rc;
    if (!(c->eps >= 0.0)) return set_error(SFB_EINVAL, "%s: eps is negative or not a number", what);
    if (c->M == 0) return SFB_OK;
    Norm p = norm_of(c);
    p.y = c->y;
    p.ldy = c->ldy;
    const int size = c->dtype == SFB_F32 ? 4 : 2;
    const bool vec = c->D % 8 == 0 && rows16(c->x, c->ldx, size) && rows16(c->y, c->ldy, size) && rows16(c->w, 0, 0) && rows16(c->b, 0, 0);
    return run(p, c->dtype, vec, nullptr, static_cast<cudaStream_t>(stream));
}

extern "C" int sfb_norm_failures(int64_t *count) {
    using namespace sfb;
    unsigned long long n = 0;
    if (!count) return set_error(SFB_EINVAL, "sfb_norm_failures: null pointer");
    if (cudaMemcpyFromSymbol(&n, g_failures, sizeof n) != cudaSuccess) return check_launch("sfb_norm_failures");
    *count = (int64_t)n;
    return SFB_OK;
}

extern "C" int64_t sfb_norm_work(int64_t M, int64_t D) {
    using namespace sfb;
    if (M < 0 || D < 1 || D > MOST) return 0;
    return 8 * D * backward_teams(M, teams_of(D));
}

extern "C" int sfb_norm_backward(const sfb_norm_call *c, sfb_stream stream) {
    using namespace sfb;
    const char *what = "sfb_norm_backward";
    int rc = check(c, what);
    if (rc) return rc;
    if (c->M == 0) return set_error(SFB_EINVAL, "%s: no rows", what);
    if (!c->stats || (c->dx && c->lddx < c->D) || ((c->dw || c->db) && !c->work))
        return set_error(SFB_EINVAL, "%s: null pointer, or a row stride that is shorter than its row", what);
    if ((c->dw && !is_float(c->w_dtype)) || (c->db && !is_float(c->b_dtype)))
        return set_error(SFB_EINVAL, "%s: a gradient's type", what);
    if (!lies_on(c->work, 16)) return set_error(SFB_EINVAL, "%s: the scratch starts on 16 bytes", what);
    if (!c->dx && !c->dw && !c->db) return SFB_OK;
    Norm p = norm_of(c);
    p.dy = c->y;
    p.lddy = c->ldy;
    p.dx = c->dx;
    p.lddx = c->lddx;
    p.parts = c->dw || c->db ? static_cast<float *>(c->work) : nullptr;
    const int size = c->dtype == SFB_F32 ? 4 : 2;
    const bool vec = c->D % 8 == 0 && rows16(c->x, c->ldx, size) && rows16(c->y, c->ldy, size) &&
                     rows16(c->dx, c->lddx, size) && rows16(c->w, 0, 0);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    int64_t teams = 0;
    rc = run(p, c->dtype, vec, &teams, st);
    if (rc || !p.parts) return rc;
    auto join = [&](auto *kernel, int64_t columns) {
        kernel<<<(unsigned)((2 * c->D + columns - 1) / columns), 512, 0, st>>>(
            p.parts, teams, c->D, c->dw, (int)c->w_dtype, c->db, (int)c->b_dtype);
    };
    if (2 * c->D < 32ll * sm_count()) join(join_kernel<8>, 8);
    else join(join_kernel<32>, 32);
    return check_launch("sf layer norm (sums over the rows)");
}
