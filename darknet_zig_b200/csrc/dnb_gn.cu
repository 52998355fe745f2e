// Group norm + activation on channels-last tensors, forward (the batchnorm layer's place,
// batchnorm.zig:129-153, with statistics per image and group instead of per batch).
//
//   mean = sum(x)/n,  rstd = 1/sqrt(sum((x - mean)^2)/n + eps),  y = act((x - mean)*(rstd*scale) + bias)
//
// Bound by memory: x in, y out, nothing else of that size. k_gn_fwd reads a unit (see dnb_gn.cuh) once
// into shared memory and adds it up on the way; y comes from shared memory. The sums are of d = x - s and
// d^2 about a shift s of each thread's own, the first element it sees of the group: s is one of the group's
// elements, so s's own distance from the mean is among the deviations that make up the variance, and no mean,
// however far from 0, cancels. Each thread's (count, mean, squared deviations) are merged as Chan, Golub and LeVeque
// do, about one of the means, in a fixed order. With a second walk over shared memory for the deviations instead,
// [128,784,256] bf16 took 45 us, bound by instructions (30 an element); so it takes 23 us (16 an element; 103 MB at
// 4.5 TB/s).
#include "dnb_gn.cuh"

namespace dnb {
namespace {

struct GnFwd {
    const void *x;
    void *y;
    const float *scales, *biases;
    float *mean, *rstd;
    float2 *pieces;   // streaming path: [batch][groups][chunks] = (mean, M2) of a row chunk
    int64_t spatial, filters, groups, cg, cb, nu, rows, chunks;
    float eps, inv_count;  // 1 / n
    int act, cluster;
    int unit_groups;
    unsigned slab, part;  // bytes, entries
};

// Moments (weight, mean, M2) added up about a reference mean `ref` that is one of theirs, in fp32: the
// differences of the means are of the group's own spread, and small beside it.
struct About {
    float ref, n = 0.0f, s = 0.0f, q = 0.0f;
    __device__ __forceinline__ void add(float w, float mean, float m2) {
        const float d = mean - ref, wd = w * d;
        n += w;
        s += wd;
        q += __fmaf_rn(wd, d, m2);
    }
    __device__ __forceinline__ float2 close() const {  // (mean, M2)
        if (n == 0.0f) return make_float2(0.0f, 0.0f);
        const float shift = s / n, m2 = __fmaf_rn(-shift, s, q);
        return make_float2(ref + shift, m2 < 0.0f ? 0.0f : m2);
    }
};

// Merges the moments of a group's threads: entries (rl, e) with e < eg of the group, each `per` elements of a
// row times the thread's rows. A warp's lanes all get (mean, M2).
__device__ __forceinline__ float2 merge_group(const float *mean, const float *m2, int rl_n, int pitch, int e0, int eg,
                                              int per, int nr) {
    const int lane = threadIdx.x & 31, total = rl_n * eg, full = nr / rl_n, rem = nr - full * rl_n;
    const int step_r = 32 / eg, step_e = 32 - step_r * eg;
    About t;
    t.ref = mean[e0];
    int r = lane / eg, e = lane - r * eg;
    for (int i = lane; i < total; i += 32) {
        const int rows = full + (r < rem);
        if (rows) t.add((float)(rows * per), mean[r * pitch + e0 + e], m2[r * pitch + e0 + e]);
        r += step_r;
        e += step_e;
        if (e >= eg) {
            e -= eg;
            ++r;
        }
    }
    t.n = warp_sum(t.n);
    t.s = warp_sum(t.s);
    t.q = warp_sum(t.q);
    return t.close();
}

template <class T, int VB, int A, bool UNI, bool STREAM>
__global__ void __launch_bounds__(512) k_gn_fwd(const __grid_constant__ GnFwd a) {
    using V = Pairs<T, VB>;
    using Raw = typename V::Raw;
    constexpr int N = V::N, P = V::P;
    extern __shared__ __align__(16) unsigned char smem[];
    const Place p = place_of(a, STREAM ? (unsigned)a.chunks : (unsigned)a.cluster);
    T *slab = reinterpret_cast<T *>(smem);
    float *pm = reinterpret_cast<float *>(smem + a.slab), *pq = pm + a.part;  // the threads' means and M2
    float2 *gs = reinterpret_cast<float2 *>(smem + a.slab + a.part * 8);  // the CTA's, a group
    float *gm = reinterpret_cast<float *>(gs + p.ng), *gr = gm + p.ng;                       // mean, rstd
    float *sc = gr + p.ng, *bi = sc + p.cb;
    const int nt = blockDim.x, v = p.cb / N, vp = v < nt ? v : nt, rl_n = v < nt ? nt / v : 1;
    const int col0 = threadIdx.x % vp, rl = threadIdx.x / vp;
    const bool on = rl < rl_n;
    const T *x = static_cast<const T *>(a.x) + (p.b * a.spatial + p.r0) * a.filters + p.c0;
    const int cg = (int)a.cg;
    const int64_t pitch = a.filters * rl_n;

    if constexpr (!STREAM) {
        for (int col = col0; col < v; col += vp) {
            if (!on) break;
            const T *src = x + (int64_t)rl * a.filters + (int64_t)col * N;
            T *dst = slab + rl * p.cb + col * N;
#pragma unroll 4
            for (int r = rl; r < p.nr; r += rl_n) {
                gn_copy<VB>(dst, src);
                src += pitch;
                dst += rl_n * p.cb;
            }
        }
        gn_stage_params(sc, a.scales, a.biases, p);
        gn_arrived();
    }

    const int rows = p.nr > rl ? (p.nr - rl + rl_n - 1) / rl_n : 0;
    for (int col = col0; col < v; col += vp) {
        if (!on) break;
        float2 s1[P] = {}, s2[P] = {}, sh[P] = {};
        const T *src = STREAM ? x + (int64_t)rl * a.filters + (int64_t)col * N : slab + rl * p.cb + col * N;
        const int64_t step = STREAM ? pitch : rl_n * p.cb;
        if (rows) {
            V::unpack(*reinterpret_cast<const Raw *>(src), sh);
            if constexpr (UNI) {
#pragma unroll
                for (int i = P - 1; i >= 0; --i) sh[i] = both(sh[0].x);
            }
        }
#pragma unroll 4
        for (int r = 0; r < rows; ++r) {
            float2 f[P];
            V::unpack(*reinterpret_cast<const Raw *>(src), f);
            src += step;
#pragma unroll
            for (int i = 0; i < P; ++i) {
                const float2 d = __fadd2_rn(f[i], neg(sh[i]));
                s1[i] = __fadd2_rn(s1[i], d);
                s2[i] = __ffma2_rn(d, d, s2[i]);
            }
        }
        // (mean, M2) about the thread's own mean: M2 = sum d^2 - (sum d)^2 / count
        if constexpr (UNI) {
#pragma unroll
            for (int i = 1; i < P; ++i) {
                s1[0] = __fadd2_rn(s1[0], s1[i]);
                s2[0] = __fadd2_rn(s2[0], s2[i]);
            }
            const float t1 = N > 1 ? s1[0].x + s1[0].y : s1[0].x, t2 = N > 1 ? s2[0].x + s2[0].y : s2[0].x;
            const float inv = rows ? 1.0f / (float)(rows * N) : 0.0f;
            pm[rl * v + col] = __fmaf_rn(t1, inv, sh[0].x);
            const float q = __fmaf_rn(-t1 * inv, t1, t2);
            pq[rl * v + col] = q < 0.0f ? 0.0f : q;
        } else {
            const float inv = rows ? 1.0f / (float)rows : 0.0f;
#pragma unroll
            for (int j = 0; j < N; ++j) {
                const float t1 = j & 1 ? s1[j / 2].y : s1[j / 2].x, t2 = j & 1 ? s2[j / 2].y : s2[j / 2].x;
                const float q = __fmaf_rn(-t1 * inv, t1, t2);
                pm[rl * p.cb + col * N + j] = __fmaf_rn(t1, inv, j & 1 ? sh[j / 2].y : sh[j / 2].x);
                pq[rl * p.cb + col * N + j] = q < 0.0f ? 0.0f : q;
            }
        }
    }
    __syncthreads();
    const int eg = UNI ? cg / N : cg, lane = threadIdx.x & 31;
    const int q_n = STREAM ? 1 : a.cluster;
    for (int g = threadIdx.x >> 5; g < p.ng; g += nt >> 5) {
        const float2 s = merge_group(pm, pq, rl_n, UNI ? v : p.cb, g * eg, eg, UNI ? N : 1, p.nr);
        if (lane != 0) continue;
        if constexpr (STREAM) {
            a.pieces[(p.b * a.groups + p.g0 + g) * a.chunks + blockIdx.x % (unsigned)a.chunks] = s;
        } else if (q_n == 1) {
            gm[g] = s.x;
            gr[g] = rsqrtf(__fmaf_rn(s.y, a.inv_count, a.eps));
        } else {
            gs[g] = s;
        }
    }
    if constexpr (STREAM) return;
    if (q_n > 1) {
        gn_cluster_arrive();
        gn_cluster_wait();
        for (int g = threadIdx.x; g < p.ng; g += nt) {
            // the CTAs' moments in rank order
            About t;
            for (int q = 0; q < q_n; ++q) {
                const int64_t left = a.spatial - q * a.rows;
                if (left <= 0) break;
                const float2 s = gn_peer_f32x2(gs + g, (unsigned)q);
                if (q == 0) t.ref = s.x;
                t.add((float)(left < a.rows ? left : a.rows) * (float)cg, s.x, s.y);
            }
            const float2 s = t.close();
            gm[g] = s.x;
            gr[g] = rsqrtf(__fmaf_rn(s.y, a.inv_count, a.eps));
        }
        gn_cluster_arrive();  // met again at the end: no CTA leaves while its moments may be read
    }
    __syncthreads();
    if (p.r0 == 0)  // the unit's first CTA
        for (int g = threadIdx.x; g < p.ng; g += nt) {
            a.mean[p.b * a.groups + p.g0 + g] = gm[g];
            a.rstd[p.b * a.groups + p.g0 + g] = gr[g];
        }

    T *y = static_cast<T *>(a.y) + (p.b * a.spatial + p.r0) * a.filters + p.c0;
    for (int col = col0; col < v; col += vp) {
        if (!on) break;
        Affine<N, UNI> k;
        k.load(col, cg, gm, gr, sc, bi);
        const T *src = slab + rl * p.cb + col * N;
        T *dst = y + (int64_t)rl * a.filters + (int64_t)col * N;
#pragma unroll 2
        for (int r = rl; r < p.nr; r += rl_n) {
            float2 f[P];
            V::unpack(*reinterpret_cast<const Raw *>(src), f);
#pragma unroll
            for (int i = 0; i < P; ++i) {
                f[i] = act_pair<A>(k.z(f[i], i), a.act);
            }
            *reinterpret_cast<Raw *>(dst) = V::pack(f);
            src += rl_n * p.cb;
            dst += pitch;
        }
    }
    if (q_n > 1) gn_cluster_wait();
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
        const float2 piece = a.pieces[i * a.chunks + q];
        t.add(k, (double)piece.x, (double)piece.y);
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
template <class T, int VB, int A, bool UNI>
__global__ void __launch_bounds__(256) k_gn_apply(const __grid_constant__ GnFwd a) {
    using V = Pairs<T, VB>;
    using Raw = typename V::Raw;
    constexpr int N = V::N, P = V::P;
    const Place p = place_of(a, (unsigned)a.chunks);
    const int nt = blockDim.x, v = p.cb / N, vp = v < nt ? v : nt, rl_n = v < nt ? nt / v : 1;
    const int col0 = threadIdx.x % vp, rl = threadIdx.x / vp;
    extern __shared__ __align__(16) float params[];
    gn_stage_params(params, a.scales, a.biases, p);
    __syncthreads();
    if (rl >= rl_n) return;
    const int64_t base = (p.b * a.spatial + p.r0) * a.filters + p.c0, g0 = p.b * a.groups + p.g0;
    for (int col = col0; col < v; col += vp) {
        Affine<N, UNI> k;
        k.load(col, (int)a.cg, a.mean + g0, a.rstd + g0, params, params + p.cb);
#pragma unroll 4
        for (int r = rl; r < p.nr; r += rl_n) {
            const int64_t at = base + (int64_t)r * a.filters + (int64_t)col * N;
            float2 f[P];
            V::unpack(*reinterpret_cast<const Raw *>(static_cast<const T *>(a.x) + at), f);
#pragma unroll
            for (int i = 0; i < P; ++i) {
                f[i] = act_pair<A>(k.z(f[i], i), a.act);
            }
            *reinterpret_cast<Raw *>(static_cast<T *>(a.y) + at) = V::pack(f);
        }
    }
}

template <class T, int VB, int A, bool UNI>
dnb_status run_fwd(GnFwd a, const GnPlan &p, int64_t batch, const DeviceState *ds, cudaStream_t s) {
    const char *what = "gn_act_forward";
    const int64_t units = batch * p.nu;
    static std::atomic<int> opted[2][kMaxDevices];
    if (!p.stream) return gn_launch(k_gn_fwd<T, VB, A, UNI, false>, a, units * p.cluster, p, ds, s, opted[0], what);
    DNB_TRY(gn_launch(k_gn_fwd<T, VB, -1, UNI, true>, a, units * p.chunks, p, ds, s, opted[1], what));
    const int64_t total = batch * a.groups;
    k_gn_merge<<<(unsigned)((total + 7) / 8), 256, 0, s>>>(a, total);
    DNB_TRY(after_launch(s, what));
    k_gn_apply<T, VB, A, UNI><<<(unsigned)(units * p.chunks), p.threads, (size_t)p.cb * 8, s>>>(a);
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
    const GnPlan p = gn_plan(batch, spatial, filters, groups, dtype_size(dtype), align, false);
    if (p.stream) *bytes = (size_t)(batch * groups * p.chunks) * 8;
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
    const GnPlan p = gn_plan(batch, spatial, filters, groups, e, align, false);
    const size_t need = p.stream ? (size_t)(batch * groups * p.chunks) * 8 : 0;
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
    a.pieces = static_cast<float2 *>(workspace);
    a.spatial = spatial;
    a.filters = filters;
    a.groups = groups;
    a.cg = filters / groups;
    a.cb = p.cb;
    a.nu = p.nu;
    a.rows = p.rows;
    a.chunks = p.chunks;
    a.eps = eps;
    a.inv_count = (float)(1.0 / ((double)spatial * (double)a.cg));
    a.act = act;
    a.cluster = p.cluster;
    a.unit_groups = (int)(p.cb / a.cg);
    a.slab = (unsigned)p.slab;
    a.part = (unsigned)p.part;
    return dispatch_dtype(dtype, [&]<class T>() -> dnb_status {
        if (p.vb == 16 && p.uni)
            return dispatch_act(act, [&]<int A>() { return run_fwd<T, 16, A, true>(a, p, batch, ds, s); });
        if (p.vb == 16)
            return dispatch_act(act, [&]<int A>() { return run_fwd<T, 16, A, false>(a, p, batch, ds, s); });
        if (p.vb == 4)
            return dispatch_act(act, [&]<int A>() { return run_fwd<T, 4, A, sizeof(T) == 4>(a, p, batch, ds, s); });
        return run_fwd<T, (int)sizeof(T), -1, true>(a, p, batch, ds, s);
    });
}

}  // extern "C"
