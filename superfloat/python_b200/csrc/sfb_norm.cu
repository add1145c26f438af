// Layer norm over the last dimension, forward and backward.
//
//   y  = xh w + b,  xh = (x - mean) r,  r = 1 / sqrt(var + eps)
//   dx = r (gy - mean(gy) - xh mean(gy xh)),  gy = dy w
//   dw = sum over rows of dy xh,  db = sum over rows of dy
//
// Bound by memory: a row is read once, into registers, and written once.  The
// variance is taken from the deviations that are there anyway, not from a sum of
// squares, which would cancel where a row's mean is far from 0.  All sums are
// float32; results are rounded once.
// A row belongs to a team: a warp (up to 1024 elements), a CTA (up to 8192) or a cluster
// of up to 8 CTAs, which add their sums up through one another's shared memory.
// The backward pass's teams take row after row, the next one's loads in flight,
// and keep dw and db of their own columns in registers; what they leave, one
// row of partial sums for every CTA (or cluster), is added up by a second launch in a fixed order.
#include <algorithm>

#include "sfb_tensor.cuh"

namespace sfb {
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
};

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

// Two sums over a team, known to all of it.  The places in shared memory alternate, so that one barrier a use is
// enough: what a use overwrites was read before the barrier of the use between.
struct Team {
    float2 warps[2][TEAM / 32];
    float2 ctas[2][8];
};

template <bool WARP>
__device__ __forceinline__ float2 team_sum(float2 v, Team &s, int &turn) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        v.x += __shfl_xor_sync(0xffffffffu, v.x, o);
        v.y += __shfl_xor_sync(0xffffffffu, v.y, o);
    }
    if constexpr (!WARP) {
        const int p = turn;
        turn ^= 1;
        if ((threadIdx.x & 31) == 0) s.warps[p][threadIdx.x >> 5] = v;
        __syncthreads();
        v = s.warps[p][0];
        for (int i = 1; i < (int)blockDim.x / 32; i++) v.x += s.warps[p][i].x, v.y += s.warps[p][i].y;
        const uint32_t n = cluster_size();
        if (n > 1) {
            if (threadIdx.x < n) {
                const uint32_t mine = (uint32_t)__cvta_generic_to_shared(&s.ctas[p][cluster_rank()]);
                uint32_t there;
                asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"(mine), "r"((uint32_t)threadIdx.x));
                asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};" ::"r"(there), "f"(v.x), "f"(v.y) : "memory");
            }
            cluster_barrier();
            v = s.ctas[p][0];
            for (uint32_t i = 1; i < n; i++) v.x += s.ctas[p][i].x, v.y += s.ctas[p][i].y;
        }
    }
    return v;
}

// The team's place: its first row, the rows from one of its own to the next, its columns.
struct Place {
    int64_t row, rows, base, end;
    int t, step;
};

template <bool WARP, int C>
__device__ __forceinline__ Place team_place(const Norm &p) {
    Place q;
    if constexpr (WARP) {
        q.row = (int64_t)blockIdx.x * (blockDim.x / 32) + threadIdx.x / 32;
        q.rows = (int64_t)gridDim.x * (blockDim.x / 32);
        q.base = 0;
        q.end = p.D;
        q.t = threadIdx.x & 31;
        q.step = 32;
    } else {
        const uint32_t n = cluster_size();
        q.row = blockIdx.x / n;
        q.rows = gridDim.x / n;
        q.t = threadIdx.x;
        q.step = blockDim.x;
        q.base = (int64_t)cluster_rank() * q.step * C * E;
        q.end = min(p.D, q.base + (int64_t)q.step * C * E);
    }
    return q;
}

template <typename T, bool VEC, bool WARP, int C>
__global__ void __launch_bounds__(WARP ? 128 : TEAM) forward_kernel(const __grid_constant__ Norm p) {
    __shared__ Team s;
    int turn = 0;
    const Place q = team_place<WARP, C>(p);
    if (!WARP && cluster_size() > 1) cluster_barrier();  // the others' memory is there
    for (int64_t r = q.row; r < p.M; r += q.rows) {
        const T *row = static_cast<const T *>(p.x) + r * p.ldx;
        float v[C][E];
        float2 sum = make_float2(0.0f, 0.0f);
        {
            Vec<T, E> raw[C];
#pragma unroll
            for (int i = 0; i < C; i++) fetch<T, VEC>(raw[i], row, q.base, i, q.t, q.step, q.end);
#pragma unroll
            for (int i = 0; i < C; i++)
#pragma unroll
                for (int j = 0; j < E; j++) {
                    v[i][j] = to_f(raw[i].v[j]);
                    sum.x += v[i][j];
                }
        }
        const float mean = team_sum<WARP>(sum, s, turn).x * p.share;
        sum.x = 0.0f;
#pragma unroll
        for (int i = 0; i < C; i++)
#pragma unroll
            for (int j = 0; j < E; j++) {
                v[i][j] = place<VEC>(q.base, i, j, q.t, q.step) < q.end ? v[i][j] - mean : 0.0f;
                sum.x = fmaf(v[i][j], v[i][j], sum.x);
            }
        const float rs = rsqrtf(fmaf(team_sum<WARP>(sum, s, turn).x, p.share, p.eps));
        if (p.stats && q.t == 0 && q.base == 0) {
            p.stats[2 * r] = mean;
            p.stats[2 * r + 1] = rs;
        }
        T *out = static_cast<T *>(p.y) + r * p.ldy;
#pragma unroll
        for (int i = 0; i < C; i++) {
            float w[E], b[E];
            param<VEC>(w, p.w, p.w_dtype, 1.0f, q.base, i, q.t, q.step, q.end);
            param<VEC>(b, p.b, p.b_dtype, 0.0f, q.base, i, q.t, q.step, q.end);
#pragma unroll
            for (int j = 0; j < E; j++) w[j] = fmaf(v[i][j] * rs, w[j], b[j]);
            put<T, VEC>(out, w, q.base, i, q.t, q.step, q.end);
        }
    }
    // (a CTA of a cluster ends only once the others have written into its memory: their writes precede a barrier that
    // it has passed)
}

template <typename T, bool VEC, bool WARP, int C>
__global__ void __launch_bounds__(WARP ? 128 : TEAM, 1) backward_kernel(const __grid_constant__ Norm p) {
    __shared__ Team s;
    __shared__ float joined[WARP ? 2 * 32 * C * E : 1];
    int turn = 0;
    const Place q = team_place<WARP, C>(p);
    if (!WARP && cluster_size() > 1) cluster_barrier();
    float w[C][E], dw[C][E] = {}, db[C][E] = {};
#pragma unroll
    for (int i = 0; i < C; i++) param<VEC>(w[i], p.w, p.w_dtype, 1.0f, q.base, i, q.t, q.step, q.end);
    Vec<T, E> xr[C], gr[C];
    float mean = 0.0f, rs = 0.0f;
    auto load = [&](int64_t r) {
        const T *x = static_cast<const T *>(p.x) + r * p.ldx, *g = static_cast<const T *>(p.dy) + r * p.lddy;
#pragma unroll
        for (int i = 0; i < C; i++) {
            fetch<T, VEC>(xr[i], x, q.base, i, q.t, q.step, q.end);
            fetch<T, VEC>(gr[i], g, q.base, i, q.t, q.step, q.end);
        }
        const float2 st = __ldg(reinterpret_cast<const float2 *>(p.stats) + r);
        mean = st.x;
        rs = st.y;
    };
    if (q.row < p.M) load(q.row);
    for (int64_t r = q.row; r < p.M; r += q.rows) {
        float xh[C][E], gy[C][E];
        float2 sum = make_float2(0.0f, 0.0f);
        const float scale = rs;
#pragma unroll
        for (int i = 0; i < C; i++)
#pragma unroll
            for (int j = 0; j < E; j++) {
                const bool in = place<VEC>(q.base, i, j, q.t, q.step) < q.end;
                const float g = to_f(gr[i].v[j]);
                xh[i][j] = in ? (to_f(xr[i].v[j]) - mean) * rs : 0.0f;
                gy[i][j] = in ? g * w[i][j] : 0.0f;
                dw[i][j] = fmaf(g, xh[i][j], dw[i][j]);
                db[i][j] += g;
                sum.x += gy[i][j];
                sum.y = fmaf(gy[i][j], xh[i][j], sum.y);
            }
        if (r + q.rows < p.M) load(r + q.rows);
        sum = team_sum<WARP>(sum, s, turn);
        const float a = sum.x * p.share, c = sum.y * p.share;
        if (p.dx) {
            T *out = static_cast<T *>(p.dx) + r * p.lddx;
#pragma unroll
            for (int i = 0; i < C; i++) {
                float d[E];
#pragma unroll
                for (int j = 0; j < E; j++) d[j] = scale * (gy[i][j] - a - xh[i][j] * c);
                put<T, VEC>(out, d, q.base, i, q.t, q.step, q.end);
            }
        }
    }
    if (!p.parts) return;
    if constexpr (WARP) {
        // the CTA's warps, one after another
        for (int n = 0; n < (int)blockDim.x / 32; n++) {
            if ((int)threadIdx.x / 32 == n)
#pragma unroll
                for (int i = 0; i < C; i++)
#pragma unroll
                    for (int j = 0; j < E; j++) {
                        const int at = (i * E + j) * 32 + q.t;
                        dw[i][j] += n ? joined[at] : 0.0f;
                        db[i][j] += n ? joined[32 * C * E + at] : 0.0f;
                        joined[at] = dw[i][j];
                        joined[32 * C * E + at] = db[i][j];
                    }
            __syncthreads();
        }
        if (threadIdx.x / 32 != blockDim.x / 32 - 1) return;
    }
    float *out = p.parts + (int64_t)(WARP ? blockIdx.x : q.row) * 2 * p.D;
    // (partial sums start on 16 bytes where D is a multiple of 4: VEC has multiples of 8)
#pragma unroll
    for (int i = 0; i < C; i++) {
        put<float, VEC>(out, dw[i], q.base, i, q.t, q.step, q.end);
        put<float, VEC>(out + p.D, db[i], q.base, i, q.t, q.step, q.end);
    }
}

// dw and db from `count` rows of partial sums: 32 columns a CTA, 16 sums to a column, joined in order
__global__ void __launch_bounds__(512) join_kernel(const float *__restrict__ parts, int64_t count, int64_t D, void *dw,
                                                   int w_dtype, void *db, int b_dtype) {
    __shared__ float s[16][33];
    const int64_t c = (int64_t)blockIdx.x * 32 + threadIdx.x;
    float v = 0.0f;
    if (c < 2 * D) {
#pragma unroll 8
        for (int64_t i = threadIdx.y; i < count; i += 16) v += parts[i * 2 * D + c];
    }
    s[threadIdx.y][threadIdx.x] = v;
    __syncthreads();
    if (threadIdx.y || c >= 2 * D) return;
#pragma unroll
    for (int i = 1; i < 16; i++) v += s[i][threadIdx.x];
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

int64_t backward_teams(int64_t M, const Teams &t) {
    // CTAs (or clusters) that take rows in turn: two CTAs of 256 threads an SM, as registers allow, and four of small ones
    const int64_t per = t.warp ? 3 : std::max<int64_t>(1, 512 / t.threads);
    const int64_t rows = t.warp ? (M + 3) / 4 : M;
    return std::max<int64_t>(1, std::min<int64_t>(rows, per * sm_count() / t.ctas));
}

template <typename K>
int launch(K *kernel, const Norm &p, const Teams &t, int64_t grid, cudaStream_t st, const char *what) {
    cudaLaunchConfig_t c{};
    c.gridDim = dim3((unsigned)(grid * t.ctas));
    c.blockDim = dim3(t.threads);
    c.stream = st;
    cudaLaunchAttribute a{};
    a.id = cudaLaunchAttributeClusterDimension;
    a.val.clusterDim.x = t.ctas;
    a.val.clusterDim.y = a.val.clusterDim.z = 1;
    c.attrs = &a;
    c.numAttrs = t.ctas > 1 ? 1 : 0;
    cudaLaunchKernelEx(&c, kernel, p);
    return check_launch(what);
}

template <typename T, bool VEC>
int forward(const Norm &p, const Teams &t, cudaStream_t st) {
    const char *what = "sf layer norm";
    const int64_t grid = std::min<int64_t>(t.warp ? (p.M + 3) / 4 : p.M, 1 << 24);
    if (!t.warp) return launch(forward_kernel<T, VEC, false, 2>, p, t, grid, st, what);
    switch (t.chunks) {
        case 1: return launch(forward_kernel<T, VEC, true, 1>, p, t, grid, st, what);
        case 2: return launch(forward_kernel<T, VEC, true, 2>, p, t, grid, st, what);
        case 3: return launch(forward_kernel<T, VEC, true, 3>, p, t, grid, st, what);
    }
    return launch(forward_kernel<T, VEC, true, 4>, p, t, grid, st, what);
}

template <typename T, bool VEC>
int backward(const Norm &p, const Teams &t, cudaStream_t st) {
    const char *what = "sf layer norm (backward)";
    const int64_t grid = backward_teams(p.M, t);
    if (!t.warp) return launch(backward_kernel<T, VEC, false, 2>, p, t, grid, st, what);
    switch (t.chunks) {
        case 1: return launch(backward_kernel<T, VEC, true, 1>, p, t, grid, st, what);
        case 2: return launch(backward_kernel<T, VEC, true, 2>, p, t, grid, st, what);
        case 3: return launch(backward_kernel<T, VEC, true, 3>, p, t, grid, st, what);
    }
    return launch(backward_kernel<T, VEC, true, 4>, p, t, grid, st, what);
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
    const Teams t = teams_of(c->D);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (c->dtype == SFB_F32) return vec ? forward<float, true>(p, t, st) : forward<float, false>(p, t, st);
    if (c->dtype == SFB_BF16) return vec ? forward<__nv_bfloat16, true>(p, t, st) : forward<__nv_bfloat16, false>(p, t, st);
    return vec ? forward<__half, true>(p, t, st) : forward<__half, false>(p, t, st);
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
    if ((reinterpret_cast<uintptr_t>(c->stats) & 7) || (reinterpret_cast<uintptr_t>(c->work) & 15))
        return set_error(SFB_EINVAL, "%s: the statistics start on 8 bytes, the scratch on 16", what);
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
    const Teams t = teams_of(c->D);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (c->dtype == SFB_F32) rc = vec ? backward<float, true>(p, t, st) : backward<float, false>(p, t, st);
    else if (c->dtype == SFB_BF16) rc = vec ? backward<__nv_bfloat16, true>(p, t, st) : backward<__nv_bfloat16, false>(p, t, st);
    else rc = vec ? backward<__half, true>(p, t, st) : backward<__half, false>(p, t, st);
    if (rc || !p.parts) return rc;
    join_kernel<<<(unsigned)((2 * c->D + 31) / 32), dim3(32, 16), 0, st>>>(p.parts, backward_teams(c->M, t), c->D, c->dw,
                                                                          (int)c->w_dtype, c->db, (int)c->b_dtype);
    return check_launch("sf layer norm (sums over the rows)");
}
