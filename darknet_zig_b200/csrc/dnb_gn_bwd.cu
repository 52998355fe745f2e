// Group norm + activation on channels-last tensors, backward (the place of batchnorm.zig:155-169).
//
//   d = delta*act'(y), t = d*scale, xh = (x - mean)*rstd, n = spatial * channels of a group:
//   dx = rstd*(t - sum(t)/n - xh*sum(t*xh)/n);  bias_updates = sum(d);  scale_updates = sum(d*xh)
//
// Both group sums are sums over the group's channels of scale * (the channel's sums over the rows), and
// those channel sums, added over the images, are the updates: one reduction serves all four. Bound by
// memory: x, delta (and y) in, dx out. k_gn_bwd keeps a unit (see dnb_gn.cuh) of each input in shared
// memory: the channel sums are formed while it is loaded, dx from shared memory. A channel's rows are
// added in fp32 per thread (rows / RL terms), across threads, CTAs and images in fp64, in a fixed order;
// k_gn_updates adds the images up.
#include "dnb_gn.cuh"

namespace dnb {
namespace {

struct GnBwd {
    const void *x, *y, *delta;
    void *dx;
    const float *scales, *biases, *mean, *rstd;
    float2 *image;   // [batch][filters]: a channel's (sum d, sum d*xh) in an image
    float2 *pieces;  // streaming path: [batch][chunks][filters], the same of a row chunk
    float2 *moments; // streaming path: [batch][groups]: (sum t, sum t*xh) / n
    int64_t spatial, filters, groups, cg, cb, nu, rows, chunks;
    int act, cluster;
    unsigned slab, part;
};

// The activation's gradient times delta, from the given output or the recomputed one.
template <int A, bool Y>
__device__ __forceinline__ float through(float delta, float y, float xh, float sc, float bi, int act) {
    const float out = Y ? y : act_fwd<A>(__fmaf_rn(xh, sc, bi), act);
    return delta * act_grad<A>(out, act);
}

template <class T, int VB, int A, bool Y, bool STREAM>
__global__ void __launch_bounds__(512) k_gn_bwd(const __grid_constant__ GnBwd a) {
    using V = Vec<T, VB>;
    using Raw = typename V::Raw;
    constexpr int N = V::N;
    extern __shared__ __align__(16) unsigned char smem[];
    const Place p = place_of(a, STREAM ? a.chunks : a.cluster);
    T *sx = reinterpret_cast<T *>(smem), *sd = reinterpret_cast<T *>(smem + a.slab),
      *sy = reinterpret_cast<T *>(smem + 2 * a.slab);
    float *part = reinterpret_cast<float *>(smem + (STREAM ? 0u : (Y ? 3u : 2u) * a.slab));
    float2 *ch = reinterpret_cast<float2 *>(part + ((2 * a.part + 3) & ~3u));  // the CTA's channel sums
    float *m0 = reinterpret_cast<float *>(ch + p.cb), *m1 = m0 + p.ng;
    const int nt = blockDim.x, v = p.cb / N, vp = v < nt ? v : nt, rl_n = v < nt ? nt / v : 1;
    const int col0 = threadIdx.x % vp, rl = threadIdx.x / vp;
    const bool on = rl < rl_n;
    const int64_t base = (p.b * a.spatial + p.r0) * a.filters + p.c0;
    const T *x = static_cast<const T *>(a.x) + base, *delta = static_cast<const T *>(a.delta) + base;
    const T *y = Y ? static_cast<const T *>(a.y) + base : nullptr;
    const int cg = (int)a.cg;

    for (int col = col0; col < v; col += vp) {
        if (!on) break;
        float s0[N] = {}, s1[N] = {}, m[N], rs[N], sc[N], bi[N];
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const int64_t g = p.b * a.groups + p.g0 + (col * N + j) / cg;
            m[j] = a.mean[g];
            rs[j] = a.rstd[g];
            sc[j] = Y ? 0.0f : a.scales[p.c0 + col * N + j];
            bi[j] = Y ? 0.0f : a.biases[p.c0 + col * N + j];
        }
#pragma unroll 4
        for (int r = rl; r < p.nr; r += rl_n) {
            const int64_t at = (int64_t)r * a.filters + (int64_t)col * N;
            const int in = r * p.cb + col * N;
            const Raw rx = *reinterpret_cast<const Raw *>(x + at), rd = *reinterpret_cast<const Raw *>(delta + at);
            Raw ry{};
            if constexpr (Y) ry = *reinterpret_cast<const Raw *>(y + at);
            float fx[N], fd[N], fy[N] = {};
            V::unpack(rx, fx);
            V::unpack(rd, fd);
            if constexpr (Y) V::unpack(ry, fy);
            if constexpr (!STREAM) {
                *reinterpret_cast<Raw *>(sx + in) = rx;
                *reinterpret_cast<Raw *>(sd + in) = rd;
                if constexpr (Y) *reinterpret_cast<Raw *>(sy + in) = ry;
            }
#pragma unroll
            for (int j = 0; j < N; ++j) {
                const float xh = (fx[j] - m[j]) * rs[j];
                const float d = through<A, Y>(fd[j], fy[j], xh, sc[j], bi[j], a.act);
                s0[j] += d;
                s1[j] = __fmaf_rn(d, xh, s1[j]);
            }
        }
#pragma unroll
        for (int j = 0; j < N; ++j) {
            part[rl * p.cb + col * N + j] = s0[j];
            part[a.part + rl * p.cb + col * N + j] = s1[j];
        }
    }
    __syncthreads();
    for (int c = threadIdx.x; c < p.cb; c += nt) {
        double s0 = 0.0, s1 = 0.0;
        for (int r = 0; r < rl_n; ++r) {
            s0 += (double)part[r * p.cb + c];
            s1 += (double)part[a.part + r * p.cb + c];
        }
        const float2 s = make_float2((float)s0, (float)s1);
        if constexpr (STREAM)
            a.pieces[(p.b * a.chunks + blockIdx.x % a.chunks) * a.filters + p.c0 + c] = s;
        else
            ch[c] = s;
    }
    if constexpr (STREAM) return;
    const int q_n = a.cluster;
    if (q_n > 1) {  // the unit's sums: every CTA adds the CTAs' in rank order, into its (now free) partials
        gn_cluster_sync();
        for (int c = threadIdx.x; c < p.cb; c += nt) {
            double s0 = 0.0, s1 = 0.0;
            for (int q = 0; q < q_n; ++q) {
                s0 += (double)gn_peer_f32(&ch[c].x, (unsigned)q);
                s1 += (double)gn_peer_f32(&ch[c].y, (unsigned)q);
            }
            part[c] = (float)s0;
            part[a.part + c] = (float)s1;
        }
        gn_cluster_sync();  // no CTA overwrites or leaves before its peers have read it
        for (int c = threadIdx.x; c < p.cb; c += nt) ch[c] = make_float2(part[c], part[a.part + c]);
    }
    __syncthreads();
    if (p.r0 == 0)
        for (int c = threadIdx.x; c < p.cb; c += nt) a.image[p.b * a.filters + p.c0 + c] = ch[c];
    const double count = (double)a.spatial * (double)a.cg;
    const int lane = threadIdx.x & 31;
    for (int g = threadIdx.x >> 5; g < p.ng; g += nt >> 5) {
        double s0 = 0.0, s1 = 0.0;
        for (int c = lane; c < cg; c += 32) {
            const double sc = (double)a.scales[p.c0 + g * cg + c];
            s0 += sc * (double)ch[g * cg + c].x;
            s1 += sc * (double)ch[g * cg + c].y;
        }
        s0 = warp_sum(s0);
        s1 = warp_sum(s1);
        if (lane == 0) {
            m0[g] = (float)(s0 / count);
            m1[g] = (float)(s1 / count);
        }
    }
    __syncthreads();

    T *dx = static_cast<T *>(a.dx) + base;
    for (int col = col0; col < v; col += vp) {
        if (!on) break;
        float m[N], rs[N], sc[N], bi[N], k0[N], k1[N];
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const int lg = (col * N + j) / cg;
            const int64_t g = p.b * a.groups + p.g0 + lg;
            m[j] = a.mean[g];
            rs[j] = a.rstd[g];
            sc[j] = a.scales[p.c0 + col * N + j];
            bi[j] = Y ? 0.0f : a.biases[p.c0 + col * N + j];
            k0[j] = m0[lg];
            k1[j] = m1[lg];
        }
        for (int r = rl; r < p.nr; r += rl_n) {
            const int in = r * p.cb + col * N;
            float fx[N], fd[N], fy[N] = {};
            V::unpack(*reinterpret_cast<const Raw *>(sx + in), fx);
            V::unpack(*reinterpret_cast<const Raw *>(sd + in), fd);
            if constexpr (Y) V::unpack(*reinterpret_cast<const Raw *>(sy + in), fy);
#pragma unroll
            for (int j = 0; j < N; ++j) {
                const float xh = (fx[j] - m[j]) * rs[j];
                const float d = through<A, Y>(fd[j], fy[j], xh, sc[j], bi[j], a.act);
                fx[j] = rs[j] * (__fmaf_rn(d, sc[j], -k0[j]) - xh * k1[j]);
            }
            *reinterpret_cast<Raw *>(dx + (int64_t)r * a.filters + (int64_t)col * N) = V::pack(fx);
        }
    }
}

// Streaming path: a block per (image, group): the chunks' channel sums added in order, then the group's
// two means.
__global__ void __launch_bounds__(128) k_gn_bwd_merge(const __grid_constant__ GnBwd a) {
    __shared__ double red[2][4];
    const int64_t b = blockIdx.x / a.groups, g = blockIdx.x % a.groups;
    double t0 = 0.0, t1 = 0.0;
    for (int64_t c = threadIdx.x; c < a.cg; c += 128) {
        double s0 = 0.0, s1 = 0.0;
        for (int64_t q = 0; q < a.chunks; ++q) {
            const float2 s = a.pieces[(b * a.chunks + q) * a.filters + g * a.cg + c];
            s0 += (double)s.x;
            s1 += (double)s.y;
        }
        a.image[b * a.filters + g * a.cg + c] = make_float2((float)s0, (float)s1);
        const double sc = (double)a.scales[g * a.cg + c];
        t0 += sc * s0;
        t1 += sc * s1;
    }
    t0 = warp_sum(t0);
    t1 = warp_sum(t1);
    if ((threadIdx.x & 31) == 0) {
        red[0][threadIdx.x >> 5] = t0;
        red[1][threadIdx.x >> 5] = t1;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        const double n = (double)a.spatial * (double)a.cg;
        t0 = red[0][0] + red[0][1] + red[0][2] + red[0][3];
        t1 = red[1][0] + red[1][1] + red[1][2] + red[1][3];
        a.moments[blockIdx.x] = make_float2((float)(t0 / n), (float)(t1 / n));
    }
}

template <class T, int VB, int A, bool Y>
__global__ void __launch_bounds__(256) k_gn_bwd_apply(const __grid_constant__ GnBwd a) {
    using V = Vec<T, VB>;
    using Raw = typename V::Raw;
    constexpr int N = V::N;
    const Place p = place_of(a, a.chunks);
    const int nt = blockDim.x, v = p.cb / N, vp = v < nt ? v : nt, rl_n = v < nt ? nt / v : 1;
    const int col0 = threadIdx.x % vp, rl = threadIdx.x / vp;
    if (rl >= rl_n) return;
    const int cg = (int)a.cg;
    const int64_t base = (p.b * a.spatial + p.r0) * a.filters + p.c0;
    const T *x = static_cast<const T *>(a.x) + base, *delta = static_cast<const T *>(a.delta) + base;
    const T *y = Y ? static_cast<const T *>(a.y) + base : nullptr;
    T *dx = static_cast<T *>(a.dx) + base;
    for (int col = col0; col < v; col += vp) {
        float m[N], rs[N], sc[N], bi[N], k0[N], k1[N];
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const int64_t g = p.b * a.groups + p.g0 + (col * N + j) / cg;
            m[j] = a.mean[g];
            rs[j] = a.rstd[g];
            sc[j] = a.scales[p.c0 + col * N + j];
            bi[j] = Y ? 0.0f : a.biases[p.c0 + col * N + j];
            k0[j] = a.moments[g].x;
            k1[j] = a.moments[g].y;
        }
#pragma unroll 2
        for (int r = rl; r < p.nr; r += rl_n) {
            const int64_t at = (int64_t)r * a.filters + (int64_t)col * N;
            float fx[N], fd[N], fy[N] = {};
            V::unpack(*reinterpret_cast<const Raw *>(x + at), fx);
            V::unpack(*reinterpret_cast<const Raw *>(delta + at), fd);
            if constexpr (Y) V::unpack(*reinterpret_cast<const Raw *>(y + at), fy);
#pragma unroll
            for (int j = 0; j < N; ++j) {
                const float xh = (fx[j] - m[j]) * rs[j];
                const float d = through<A, Y>(fd[j], fy[j], xh, sc[j], bi[j], a.act);
                fx[j] = rs[j] * (__fmaf_rn(d, sc[j], -k0[j]) - xh * k1[j]);
            }
            *reinterpret_cast<Raw *>(dx + at) = V::pack(fx);
        }
    }
}

// The updates: a block per 32 channels, 8 slices of the images added in order, then the slices.
__global__ void __launch_bounds__(256) k_gn_updates(const float2 *image, int64_t batch, int64_t filters,
                                                    float *bias_updates, float *scale_updates, int add) {
    __shared__ double red[2][8][32];
    const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
    const int64_t c = (int64_t)blockIdx.x * 32 + tx;
    double s0 = 0.0, s1 = 0.0;
    if (c < filters) {
#pragma unroll 4
        for (int64_t b = ty; b < batch; b += 8) {
            const float2 v = image[b * filters + c];
            s0 += (double)v.x;
            s1 += (double)v.y;
        }
    }
    red[0][ty][tx] = s0;
    red[1][ty][tx] = s1;
    __syncthreads();
    if (ty == 0 && c < filters) {
        for (int k = 1; k < 8; ++k) {
            s0 += red[0][k][tx];
            s1 += red[1][k][tx];
        }
        bias_updates[c] = (float)(add ? (double)bias_updates[c] + s0 : s0);
        scale_updates[c] = (float)(add ? (double)scale_updates[c] + s1 : s1);
    }
}

struct BwdSpace {
    size_t image, pieces, moments, total;
};
BwdSpace space_of(const GnPlan &p, int64_t batch, int64_t filters, int64_t groups) {
    BwdSpace w;
    auto round = [](size_t b) { return (b + 15) / 16 * 16; };
    w.image = 0;
    w.pieces = round((size_t)(batch * filters) * 8);
    w.moments = w.pieces + (p.stream ? round((size_t)(batch * p.chunks * filters) * 8) : 0);
    w.total = w.moments + (p.stream ? round((size_t)(batch * groups) * 8) : 0);
    return w;
}

GnPlan plan_bwd(const void *x, const void *y, const void *delta, const void *dx, int dtype, int64_t batch,
                int64_t spatial, int64_t filters, int64_t groups) {
    const uintptr_t align = reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(y) |
                            reinterpret_cast<uintptr_t>(delta) | reinterpret_cast<uintptr_t>(dx);
    return gn_plan(batch, spatial, filters, groups, dtype_size(dtype), align, y ? 3 : 2, 2);
}

template <class T, int VB, int A, bool Y>
dnb_status run_bwd(const GnBwd &a, const GnPlan &p, int64_t batch, const DeviceState *ds, cudaStream_t s) {
    const char *what = "gn_act_backward";
    const int64_t units = batch * p.nu;
    if (!p.stream) {
        static std::atomic<int> opted[kMaxDevices];
        return gn_launch(k_gn_bwd<T, VB, A, Y, false>, a, units * p.cluster, p, ds, s, opted, what);
    }
    static std::atomic<int> opted[kMaxDevices];
    DNB_TRY(gn_launch(k_gn_bwd<T, VB, A, Y, true>, a, units * p.chunks, p, ds, s, opted, what));
    if (batch * a.groups > 0x7fffffffll) return fail(DNB_ERR_UNSUPPORTED, "%s: too many groups", what);
    k_gn_bwd_merge<<<(unsigned)(batch * a.groups), 128, 0, s>>>(a);
    DNB_TRY(after_launch(s, what));
    k_gn_bwd_apply<T, VB, A, Y><<<(unsigned)(units * p.chunks), p.threads, 0, s>>>(a);
    return after_launch(s, what);
}

}  // namespace
}  // namespace dnb

using namespace dnb;

extern "C" {

dnb_status dnb_gn_act_backward_workspace(const void *x, const void *y, const void *delta, const void *dx, int dtype,
                                         int64_t batch, int64_t spatial, int64_t filters, int64_t groups,
                                         size_t *bytes) {
    const char *what = "gn_act_backward_workspace";
    if (!bytes) return fail(DNB_ERR_INVALID, "%s: bytes is null", what);
    if (!valid_dtype(dtype)) return fail(DNB_ERR_INVALID, "%s: unknown dtype %d", what, dtype);
    DNB_TRY(gn_shape_check(batch, spatial, filters, groups, what));
    *bytes = 0;
    if (batch == 0 || spatial == 0) return DNB_OK;
    const GnPlan p = plan_bwd(x, y, delta, dx, dtype, batch, spatial, filters, groups);
    *bytes = space_of(p, batch, filters, groups).total;
    return DNB_OK;
}

dnb_status dnb_gn_act_backward(const void *x, const void *y, const void *delta, void *dx, int dtype, int64_t batch,
                               int64_t spatial, int64_t filters, int64_t groups, const float *scales,
                               const float *biases, const float *mean, const float *rstd, float *bias_updates,
                               float *scale_updates, int act, int accumulate, void *workspace,
                               size_t workspace_bytes, dnb_stream stream) {
    const char *what = "gn_act_backward";
    if (!valid_dtype(dtype)) return fail(DNB_ERR_INVALID, "%s: unknown dtype %d", what, dtype);
    DNB_TRY(gn_shape_check(batch, spatial, filters, groups, what));
    if (!valid_act(act)) return fail(DNB_ERR_INVALID, "%s: unknown activation %d", what, act);
    if (accumulate & ~DNB_ACC_UPDATES) return fail(DNB_ERR_INVALID, "%s: only the updates accumulate", what);
    if (!bias_updates || !scale_updates) return fail(DNB_ERR_INVALID, "%s: null pointer", what);
    DeviceState *ds = nullptr;
    const cudaStream_t s = as_stream(stream);
    const unsigned ublocks = (unsigned)((filters + 31) / 32);
    const int add = accumulate & DNB_ACC_UPDATES;
    if (filters > int64_t(1) << 35) return fail(DNB_ERR_UNSUPPORTED, "%s: too many filters", what);
    if (batch == 0 || spatial == 0) {  // sums over nothing
        if (add) return DNB_OK;
        DNB_TRY(current_device(&ds));
        k_gn_updates<<<ublocks, 256, 0, s>>>(nullptr, 0, filters, bias_updates, scale_updates, 0);
        return after_launch(s, what);
    }
    if (!x || !delta || !dx || !scales || !biases || !mean || !rstd)
        return fail(DNB_ERR_INVALID, "%s: null pointer", what);
    const int64_t e = dtype_size(dtype), bytes = batch * spatial * filters * e, fb = filters * 4;
    if ((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(y) | reinterpret_cast<uintptr_t>(delta) |
         reinterpret_cast<uintptr_t>(dx)) % (uintptr_t)e)
        return fail(DNB_ERR_INVALID, "%s: misaligned pointer", what);
    if (overlaps(dx, bytes, x, bytes) || overlaps(dx, bytes, y, bytes) ||
        (dx != delta && overlaps(dx, bytes, delta, bytes)) || overlaps(bias_updates, fb, scale_updates, fb) ||
        overlaps(dx, bytes, bias_updates, fb) || overlaps(dx, bytes, scale_updates, fb))
        return fail(DNB_ERR_INVALID, "%s: overlapping tensors", what);
    const GnPlan p = plan_bwd(x, y, delta, dx, dtype, batch, spatial, filters, groups);
    const BwdSpace w = space_of(p, batch, filters, groups);
    if (!workspace || workspace_bytes < w.total || !aligned16(workspace))
        return fail(DNB_ERR_INVALID, "%s: needs a 16-byte aligned workspace of %zu bytes, got %zu", what, w.total,
                    workspace ? workspace_bytes : (size_t)0);
    DNB_TRY(current_device(&ds));
    char *ws = static_cast<char *>(workspace);
    GnBwd a;
    a.x = x;
    a.y = y;
    a.delta = delta;
    a.dx = dx;
    a.scales = scales;
    a.biases = biases;
    a.mean = mean;
    a.rstd = rstd;
    a.image = reinterpret_cast<float2 *>(ws + w.image);
    a.pieces = reinterpret_cast<float2 *>(ws + w.pieces);
    a.moments = reinterpret_cast<float2 *>(ws + w.moments);
    a.spatial = spatial;
    a.filters = filters;
    a.groups = groups;
    a.cg = filters / groups;
    a.cb = p.cb;
    a.nu = p.nu;
    a.rows = p.rows;
    a.chunks = p.chunks;
    a.act = act;
    a.cluster = p.cluster;
    a.slab = (unsigned)p.slab;
    a.part = (unsigned)p.part_floats;
    auto with_y = [&]<class T, int VB, int A>() {
        return y ? run_bwd<T, VB, A, true>(a, p, batch, ds, s) : run_bwd<T, VB, A, false>(a, p, batch, ds, s);
    };
    const dnb_status st = dispatch_dtype(dtype, [&]<class T>() -> dnb_status {
        if (p.vb == 16)
            return dispatch_act(act, [&]<int A>() { return with_y.template operator()<T, 16, A>(); });
        if (p.vb == 4) return with_y.template operator()<T, 4, -1>();
        return with_y.template operator()<T, (int)sizeof(T), -1>();
    });
    DNB_TRY(st);
    k_gn_updates<<<ublocks, 256, 0, s>>>(a.image, batch, filters, bias_updates, scale_updates, add);
    return after_launch(s, what);
}

}  // extern "C"
