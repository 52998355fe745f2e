// Group norm + activation on channels-last tensors, forward (the batchnorm layer's place,
// batchnorm.zig:129-153, with statistics per image and group instead of per batch).
//
//   mean = sum(x)/n,  rstd = 1/sqrt(sum((x - mean)^2)/n + eps),  y = act(((x - mean)*rstd)*scale + bias)
//
// Bound by memory: x in, y out, nothing else of that size. k_gn_fwd reads a unit (see dnb_gn.cuh) once
// into shared memory, adds it up on the way, takes the squared deviations from the true mean in a second
// walk over shared memory (no cancellation, whatever the mean), and writes y in a third. Per-thread sums
// run over a column's rows / RL elements in fp32; they are added across threads and CTAs in fp64, in a
// fixed order.
#include "dnb_gn.cuh"

namespace dnb {
namespace {

struct GnFwd {
    const void *x;
    void *y;
    const float *scales, *biases;
    float *mean, *rstd;
    double *pieces;  // streaming path: [batch][groups][chunks][2] = (mean, M2) of a row chunk
    int64_t spatial, filters, groups, cg, cb, nu, rows, chunks;
    float eps;
    int act, cluster;
    unsigned slab, part;  // bytes, floats
};

// Adds part[rl][c] over rl and the channels of each group: a warp per group, fp64.
__device__ __forceinline__ void group_sums(const float *part, int rl_n, int cb, int ng, int cg, double *out) {
    const int lane = threadIdx.x & 31;
    for (int g = threadIdx.x >> 5; g < ng; g += blockDim.x >> 5) {
        double s = 0.0;
        if (cg >= 32) {
            for (int r = 0; r < rl_n; ++r)
                for (int c = lane; c < cg; c += 32) s += (double)part[r * cb + g * cg + c];
        } else {  // several rows at a time
            const int per = 32 / cg, r0 = lane / cg, c = lane % cg;
            if (r0 < per)
                for (int r = r0; r < rl_n; r += per) s += (double)part[r * cb + g * cg + c];
        }
        s = warp_sum(s);
        if (lane == 0) out[g] = s;
    }
}

template <class T, int VB, int A, bool STREAM>
__global__ void __launch_bounds__(512) k_gn_fwd(const __grid_constant__ GnFwd a) {
    using V = Vec<T, VB>;
    using Raw = typename V::Raw;
    constexpr int N = V::N;
    extern __shared__ __align__(16) unsigned char smem[];
    const Place p = place_of(a, STREAM ? a.chunks : a.cluster);
    T *slab = reinterpret_cast<T *>(smem);
    float *part = reinterpret_cast<float *>(smem + a.slab);
    double *gs = reinterpret_cast<double *>(smem + ((a.slab + a.part * 4 + 15) & ~15u));  // [2][ng] sums
    float *gm = reinterpret_cast<float *>(gs + 2 * p.ng), *gr = gm + p.ng;               // mean, rstd
    const int nt = blockDim.x, v = p.cb / N, vp = v < nt ? v : nt, rl_n = v < nt ? nt / v : 1;
    const int col0 = threadIdx.x % vp, rl = threadIdx.x / vp;
    const bool on = rl < rl_n;
    const T *x = static_cast<const T *>(a.x) + (p.b * a.spatial + p.r0) * a.filters + p.c0;
    const int cg = (int)a.cg;
    const double count = STREAM ? (double)p.nr * (double)a.cg : (double)a.spatial * (double)a.cg;

    // load, keep, and add up
    for (int col = col0; col < v; col += vp) {
        if (!on) break;
        float acc[N] = {};
        const T *src = x + (int64_t)col * N;
        T *dst = slab + col * N;
        int r = rl;
        constexpr int U = 4;
        for (; r + (U - 1) * rl_n < p.nr; r += U * rl_n) {
            Raw raw[U];
#pragma unroll
            for (int u = 0; u < U; ++u)
                raw[u] = *reinterpret_cast<const Raw *>(src + (int64_t)(r + u * rl_n) * a.filters);
#pragma unroll
            for (int u = 0; u < U; ++u) {
                float f[N];
                V::unpack(raw[u], f);
                *reinterpret_cast<Raw *>(dst + (r + u * rl_n) * p.cb) = raw[u];
#pragma unroll
                for (int j = 0; j < N; ++j) acc[j] += f[j];
            }
        }
        for (; r < p.nr; r += rl_n) {
            const Raw raw = *reinterpret_cast<const Raw *>(src + (int64_t)r * a.filters);
            float f[N];
            V::unpack(raw, f);
            *reinterpret_cast<Raw *>(dst + r * p.cb) = raw;
#pragma unroll
            for (int j = 0; j < N; ++j) acc[j] += f[j];
        }
#pragma unroll
        for (int j = 0; j < N; ++j) part[rl * p.cb + col * N + j] = acc[j];
    }
    __syncthreads();
    group_sums(part, rl_n, p.cb, p.ng, cg, gs);
    const int q_n = STREAM ? 1 : a.cluster;
    if (q_n > 1) gn_cluster_sync();
    else __syncthreads();
    for (int g = threadIdx.x; g < p.ng; g += nt) {
        double s = 0.0;
        if (q_n > 1)
            for (int q = 0; q < q_n; ++q) s += gn_peer_f64(gs + g, (unsigned)q);
        else
            s = gs[g];
        gm[g] = (float)(s / count);
    }
    __syncthreads();

    // squared deviations, from shared memory
    for (int col = col0; col < v; col += vp) {
        if (!on) break;
        float acc[N] = {}, m[N];
#pragma unroll
        for (int j = 0; j < N; ++j) m[j] = gm[(col * N + j) / cg];
        for (int r = rl; r < p.nr; r += rl_n) {
            float f[N];
            V::unpack(*reinterpret_cast<const Raw *>(slab + r * p.cb + col * N), f);
#pragma unroll
            for (int j = 0; j < N; ++j) {
                const float d = f[j] - m[j];
                acc[j] = __fmaf_rn(d, d, acc[j]);
            }
        }
#pragma unroll
        for (int j = 0; j < N; ++j) part[rl * p.cb + col * N + j] = acc[j];
    }
    __syncthreads();
    double *gv = gs + p.ng;
    group_sums(part, rl_n, p.cb, p.ng, cg, gv);
    if (q_n > 1) gn_cluster_sync();
    else __syncthreads();
    for (int g = threadIdx.x; g < p.ng; g += nt) {
        double s = 0.0;
        if (q_n > 1)
            for (int q = 0; q < q_n; ++q) s += gn_peer_f64(gv + g, (unsigned)q);
        else
            s = gv[g];
        if constexpr (STREAM) {
            // the deviations are from the rounded mean: their sum is M2 + n (mean - gm)^2, taken back here
            const double mean = gs[g] / count, e = mean - (double)gm[g];
            double *piece = a.pieces + ((p.b * a.groups + p.g0 + g) * a.chunks + blockIdx.x % a.chunks) * 2;
            const double m2 = s - count * e * e;
            piece[0] = mean;
            piece[1] = m2 < 0.0 ? 0.0 : m2;
        } else {
            const float rstd = (float)(1.0 / sqrt(s / count + (double)a.eps));
            gr[g] = rstd;
            if (p.r0 == 0) {  // the unit's first CTA
                a.mean[p.b * a.groups + p.g0 + g] = gm[g];
                a.rstd[p.b * a.groups + p.g0 + g] = rstd;
            }
        }
    }
    if constexpr (STREAM) return;
    // the peers may still read gv: no CTA leaves before all have
    if (q_n > 1) gn_cluster_sync();
    else __syncthreads();

    T *y = static_cast<T *>(a.y) + (p.b * a.spatial + p.r0) * a.filters + p.c0;
    for (int col = col0; col < v; col += vp) {
        if (!on) break;
        float m[N], rs[N], sc[N], bi[N];
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const int g = (col * N + j) / cg;
            m[j] = gm[g];
            rs[j] = gr[g];
            sc[j] = a.scales[p.c0 + col * N + j];
            bi[j] = a.biases[p.c0 + col * N + j];
        }
#pragma unroll 2
        for (int r = rl; r < p.nr; r += rl_n) {
            float f[N];
            V::unpack(*reinterpret_cast<const Raw *>(slab + r * p.cb + col * N), f);
#pragma unroll
            for (int j = 0; j < N; ++j) f[j] = act_fwd<A>(__fmaf_rn((f[j] - m[j]) * rs[j], sc[j], bi[j]), a.act);
            *reinterpret_cast<Raw *>(y + (int64_t)r * a.filters + (int64_t)col * N) = V::pack(f);
        }
    }
}

// Streaming path: merges the row chunks' (mean, M2) of a group (Chan, Golub and LeVeque's pairwise
// update), a warp per (image, group): each lane its chunks in order, then the lanes in a fixed tree.
struct Moments {
    double n, mean, m2;
    __device__ void add(double k, double pm, double p2) {
        const double t = n + k;
        if (t == 0.0) return;
        const double d = pm - mean;
        mean += d * (k / t);
        m2 += p2 + d * d * (n * k / t);
        n = t;
    }
};
__global__ void __launch_bounds__(256) k_gn_merge(const __grid_constant__ GnFwd a, int64_t total) {
    const int lane = threadIdx.x & 31;
    const int64_t i = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
    if (i >= total) return;
    Moments t{0.0, 0.0, 0.0};
    for (int64_t q = lane; q < a.chunks; q += 32) {
        const int64_t left = a.spatial - q * a.rows;
        const double k = (double)(left < a.rows ? left : a.rows) * (double)a.cg;
        t.add(k, a.pieces[(i * a.chunks + q) * 2], a.pieces[(i * a.chunks + q) * 2 + 1]);
    }
    for (int o = 16; o > 0; o >>= 1) {
        const double n = __shfl_down_sync(0xffffffffu, t.n, o), m = __shfl_down_sync(0xffffffffu, t.mean, o),
                     s = __shfl_down_sync(0xffffffffu, t.m2, o);
        t.add(n, m, s);
    }
    if (lane == 0) {
        a.mean[i] = (float)t.mean;
        a.rstd[i] = (float)(1.0 / sqrt(t.m2 / t.n + (double)a.eps));
    }
}

// Streaming path: the outputs, with the statistics from global memory.
template <class T, int VB, int A>
__global__ void __launch_bounds__(256) k_gn_apply(const __grid_constant__ GnFwd a) {
    using V = Vec<T, VB>;
    using Raw = typename V::Raw;
    constexpr int N = V::N;
    const Place p = place_of(a, a.chunks);
    const int nt = blockDim.x, v = p.cb / N, vp = v < nt ? v : nt, rl_n = v < nt ? nt / v : 1;
    const int col0 = threadIdx.x % vp, rl = threadIdx.x / vp;
    if (rl >= rl_n) return;
    const int cg = (int)a.cg;
    const int64_t base = (p.b * a.spatial + p.r0) * a.filters + p.c0;
    const T *x = static_cast<const T *>(a.x) + base;
    T *y = static_cast<T *>(a.y) + base;
    for (int col = col0; col < v; col += vp) {
        float m[N], rs[N], sc[N], bi[N];
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const int64_t g = p.b * a.groups + p.g0 + (col * N + j) / cg;
            m[j] = a.mean[g];
            rs[j] = a.rstd[g];
            sc[j] = a.scales[p.c0 + col * N + j];
            bi[j] = a.biases[p.c0 + col * N + j];
        }
#pragma unroll 4
        for (int r = rl; r < p.nr; r += rl_n) {
            const int64_t at = (int64_t)r * a.filters + (int64_t)col * N;
            float f[N];
            V::unpack(*reinterpret_cast<const Raw *>(x + at), f);
#pragma unroll
            for (int j = 0; j < N; ++j) f[j] = act_fwd<A>(__fmaf_rn((f[j] - m[j]) * rs[j], sc[j], bi[j]), a.act);
            *reinterpret_cast<Raw *>(y + at) = V::pack(f);
        }
    }
}

template <class T, int VB, int A>
dnb_status run_fwd(GnFwd a, const GnPlan &p, int64_t batch, const DeviceState *ds, cudaStream_t s) {
    const char *what = "gn_act_forward";
    const int64_t units = batch * p.nu;
    if (!p.stream) {
        static std::atomic<int> opted[kMaxDevices];
        return gn_launch(k_gn_fwd<T, VB, A, false>, a, units * p.cluster, p, ds, s, opted, what);
    }
    static std::atomic<int> opted[kMaxDevices];
    DNB_TRY(gn_launch(k_gn_fwd<T, VB, A, true>, a, units * p.chunks, p, ds, s, opted, what));
    const int64_t total = batch * a.groups;
    k_gn_merge<<<(unsigned)((total + 7) / 8), 256, 0, s>>>(a, total);
    DNB_TRY(after_launch(s, what));
    k_gn_apply<T, VB, A><<<(unsigned)(units * p.chunks), p.threads, 0, s>>>(a);
    return after_launch(s, what);
}

dnb_status gn_fwd_check(int dtype, int64_t batch, int64_t spatial, int64_t filters, int64_t groups, const char *what) {
    if (!valid_dtype(dtype)) return fail(DNB_ERR_INVALID, "%s: unknown dtype %d", what, dtype);
    return gn_shape_check(batch, spatial, filters, groups, what);
}

}  // namespace
}  // namespace dnb

using namespace dnb;

extern "C" {

dnb_status dnb_gn_act_forward_workspace(const void *x, const void *y, int dtype, int64_t batch, int64_t spatial,
                                        int64_t filters, int64_t groups, size_t *bytes) {
    if (!bytes) return fail(DNB_ERR_INVALID, "gn_act_forward_workspace: bytes is null");
    DNB_TRY(gn_fwd_check(dtype, batch, spatial, filters, groups, "gn_act_forward_workspace"));
    *bytes = 0;
    if (batch == 0 || spatial == 0) return DNB_OK;
    const uintptr_t align = reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(y);
    const GnPlan p = gn_plan(batch, spatial, filters, groups, dtype_size(dtype), align, 1, 1);
    if (p.stream) *bytes = (size_t)(batch * groups * p.chunks) * 16;
    return DNB_OK;
}

dnb_status dnb_gn_act_forward(const void *x, void *y, int dtype, int64_t batch, int64_t spatial, int64_t filters,
                              int64_t groups, const float *scales, const float *biases, float eps, float *mean,
                              float *rstd, int act, void *workspace, size_t workspace_bytes, dnb_stream stream) {
    const char *what = "gn_act_forward";
    DNB_TRY(gn_fwd_check(dtype, batch, spatial, filters, groups, what));
    if (!valid_act(act)) return fail(DNB_ERR_INVALID, "%s: unknown activation %d", what, act);
    if (!(eps >= 0.0f)) return fail(DNB_ERR_INVALID, "%s: eps must not be negative", what);
    if (batch == 0 || spatial == 0) return DNB_OK;
    if (!x || !y || !scales || !biases || !mean || !rstd) return fail(DNB_ERR_INVALID, "%s: null pointer", what);
    const int64_t e = dtype_size(dtype), bytes = batch * spatial * filters * e, st = batch * groups * 4;
    const uintptr_t align = reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(y);
    if (align % (uintptr_t)e) return fail(DNB_ERR_INVALID, "%s: misaligned pointer", what);
    if ((x != y && overlaps(x, bytes, y, bytes)) || overlaps(mean, st, rstd, st) || overlaps(mean, st, y, bytes) ||
        overlaps(rstd, st, y, bytes) || overlaps(mean, st, x, bytes) || overlaps(rstd, st, x, bytes))
        return fail(DNB_ERR_INVALID, "%s: overlapping tensors", what);
    const GnPlan p = gn_plan(batch, spatial, filters, groups, e, align, 1, 1);
    const size_t need = p.stream ? (size_t)(batch * groups * p.chunks) * 16 : 0;
    if (need && (!workspace || workspace_bytes < need || !aligned16(workspace)))
        return fail(DNB_ERR_INVALID, "%s: needs a 16-byte aligned workspace of %zu bytes, got %zu", what, need,
                    workspace ? workspace_bytes : (size_t)0);
    DeviceState *ds = nullptr;
    DNB_TRY(current_device(&ds));
    const cudaStream_t s = as_stream(stream);
    GnFwd a;
    a.x = x;
    a.y = y;
    a.scales = scales;
    a.biases = biases;
    a.mean = mean;
    a.rstd = rstd;
    a.pieces = static_cast<double *>(workspace);
    a.spatial = spatial;
    a.filters = filters;
    a.groups = groups;
    a.cg = filters / groups;
    a.cb = p.cb;
    a.nu = p.nu;
    a.rows = p.rows;
    a.chunks = p.chunks;
    a.eps = eps;
    a.act = act;
    a.cluster = p.cluster;
    a.slab = (unsigned)p.slab;
    a.part = (unsigned)p.part_floats;
    return dispatch_dtype(dtype, [&]<class T>() -> dnb_status {
        if (p.vb == 16)
            return dispatch_act(act, [&]<int A>() { return run_fwd<T, 16, A>(a, p, batch, ds, s); });
        if (p.vb == 4) return run_fwd<T, 4, -1>(a, p, batch, ds, s);
        return run_fwd<T, (int)sizeof(T), -1>(a, p, batch, ds, s);
    });
}

}  // extern "C"
