// Group norm + activation on channels-last tensors, backward (the place of batchnorm.zig:155-169).
//
//   d = delta*act'(y), t = d*scale, xh = (x - mean)*rstd, n = spatial * channels of a group:
//   dx = rstd*(t - sum(t)/n - xh*sum(t*xh)/n);  bias_updates = sum(d);  scale_updates = sum(d*xh)
//
// Both group sums are sums over the group's channels of scale * (the channel's sums over the rows), and
// those channel sums, added over the images, are the updates: one reduction serves all four. Bound by
// memory: x, delta (and y) in, dx out. k_gn_bwd walks a unit (see dnb_gn.cuh) twice: for the channel sums, then
// for dx = d*k - (x - mean)*c2 - c1 (k = rstd*scale, c1 = rstd*sum(t)/n, c2 = rstd^2*sum(t*xh)/n: two fused
// multiply-adds an element). The second walk finds the rows in the L2 cache (HBM reads each once: 103 MB at
// [128,784,256] bf16), which leaves shared memory free: three CTAs an SM and 62 us (logistic, recomputed) against
// two and 75 us with the rows, or the fp32 d, held there. Registers double-buffered over the loads: 69 us.
// A channel's rows are added in fp32 (per thread rows / RL terms, then the threads in two steps), across CTAs,
// images and a group's channels in fp64, in a fixed order; k_gn_updates adds the images up.
#include "dnb_gn.cuh"

namespace dnb {
namespace {

struct GnBwd {
    const void *x, *y, *delta;
    void *dx;
    const float *scales, *biases, *mean, *rstd;
    float2 *image;   // [batch][filters]: a channel's (sum d, sum d*xh) in an image
    float2 *pieces;  // streaming path: [batch][chunks][filters], the same of a row chunk
    float2 *moments; // streaming path: [batch][groups]: -(c1, c2)
    int64_t spatial, filters, groups, cg, cb, nu, rows, chunks;
    double inv_count;  // 1 / n
    int act, cluster, unit_groups;
    unsigned part;
};

// The activation's gradient times delta for a pair, from the given output or the recomputed one (z: its
// argument). The recomputed logistic's y(1 - y) shares one reciprocal between the two: 1/u and 1/v are v/(uv)
// and u/(uv). Exponents are cut off at 43 (y = 2e-19) so that uv stays finite; three special-function results
// a pair instead of four, which bound the kernel.
template <int A, bool Y>
__device__ __forceinline__ float2 through(float2 delta, float2 y, float2 z, int act) {
    if constexpr (A == DNB_ACT_LINEAR) return delta;
    if constexpr (A == DNB_ACT_LOGISTIC && !Y) {
        float tx, ty;
        asm("min.NaN.f32 %0, %1, %2;" : "=f"(tx) : "f"(-z.x), "f"(43.0f));
        asm("min.NaN.f32 %0, %1, %2;" : "=f"(ty) : "f"(-z.y), "f"(43.0f));
        const float2 e = make_float2(quick_exp(tx), quick_exp(ty)), u = __fadd2_rn(e, both(1.0f));
        const float rcp = quick_rcp(u.x * u.y);
        const float2 out = __fmul2_rn(both(rcp), make_float2(u.y, u.x));
        return __fmul2_rn(delta, __fmul2_rn(__fmul2_rn(e, out), out));  // 1 - y = e y
    }
    const float2 o = Y ? y : act_pair<A>(z, act);
    return make_float2(delta.x * act_grad<A>(o.x, act), delta.y * act_grad<A>(o.y, act));
}

template <int N>
__device__ __forceinline__ void store_pairs(float *p, const float2 (&s)[(N + 1) / 2]) {
    if constexpr (N == 1) *p = s[0].x;
    else if constexpr (N == 2) *reinterpret_cast<float2 *>(p) = s[0];
    else
#pragma unroll
        for (int i = 0; i < N / 2; i += 2)
            *reinterpret_cast<float4 *>(p + 2 * i) = make_float4(s[i].x, s[i].y, s[i + 1].x, s[i + 1].y);
}

// The group's (c1, c2) for a vector's channels.
template <int N, bool UNI>
__device__ __forceinline__ void load_moments(int col, int cg, const float2 *mo, float2 *c1, float2 *c2) {
    if constexpr (UNI) {
        const float2 m = mo[col * N / cg];
        c1[0] = both(m.x);
        c2[0] = both(m.y);
    } else {
        int g[N];
        groups_of<N>(col, cg, g);
#pragma unroll
        for (int i = 0; i < (N + 1) / 2; ++i) {
            const float2 m = mo[g[2 * i]], n = 2 * i + 1 < N ? mo[g[2 * i + 1 < N ? 2 * i + 1 : 0]] : both(0.0f);
            c1[i] = make_float2(m.x, n.x);
            c2[i] = make_float2(m.y, n.y);
        }
    }
}
// dx of a vector, in place of x.
template <int P, int A, bool Y, bool UNI, class K>
__device__ __forceinline__ void dx_of(float2 (&fx)[P], const float2 (&fd)[P], const float2 (&fy)[P], const K &k,
                                      const float2 *c1, const float2 *c2, int act) {
#pragma unroll
    for (int i = 0; i < P; ++i) {
        const float2 z = Y ? fy[i] : k.z(fx[i], i);
        const float2 d = through<A, Y>(fd[i], fy[i], z, act);
        const float2 xm = __fadd2_rn(fx[i], k.m[UNI ? 0 : i]);
        fx[i] = __ffma2_rn(d, k.k[i], __ffma2_rn(xm, c2[UNI ? 0 : i], c1[UNI ? 0 : i]));
    }
}

template <class T, int VB, int A, bool Y, bool UNI, bool STREAM>
__global__ void __launch_bounds__(256, 3) k_gn_bwd(const __grid_constant__ GnBwd a) {
    using V = Pairs<T, VB>;
    using Raw = typename V::Raw;
    constexpr int N = V::N, P = V::P;
    extern __shared__ __align__(16) unsigned char smem[];
    const Place p = place_of(a, STREAM ? (unsigned)a.chunks : (unsigned)a.cluster);
    float *part = reinterpret_cast<float *>(smem);
    float2 *slices = reinterpret_cast<float2 *>(part + 2 * a.part);
    const int nt = blockDim.x;
    float2 *ch = slices + nt;                                    // the channels' sums
    float *sc = reinterpret_cast<float *>(ch + p.cb), *bi = sc + p.cb;
    float2 *mo = reinterpret_cast<float2 *>(bi + p.cb);          // the groups' (c1, c2)
    const int v = p.cb / N, vp = v < nt ? v : nt, rl_n = v < nt ? nt / v : 1;
    const int col0 = threadIdx.x % vp, rl = threadIdx.x / vp;
    const bool on = rl < rl_n;
    const int64_t base = (p.b * a.spatial + p.r0) * a.filters + p.c0, g0 = p.b * a.groups + p.g0;
    const int64_t pitch = a.filters * rl_n;
    const int cg = (int)a.cg;

    gn_stage_params(sc, a.scales, a.biases, p);
    __syncthreads();

    for (int col = col0; col < v; col += vp) {
        if (!on) break;
        Affine<N, UNI> k;
        k.load(col, cg, a.mean + g0, a.rstd + g0, sc, bi);
        float2 s0[P] = {}, s1[P] = {};
        const int64_t at = base + (int64_t)rl * a.filters + (int64_t)col * N;
        const T *x = static_cast<const T *>(a.x) + at, *delta = static_cast<const T *>(a.delta) + at;
        const T *y = Y ? static_cast<const T *>(a.y) + at : nullptr;
        auto add = [&](Raw rx, Raw rd, Raw ry) {
            float2 fx[P], fd[P], fy[P] = {};
            V::unpack(rx, fx);
            V::unpack(rd, fd);
            if constexpr (Y) V::unpack(ry, fy);
#pragma unroll
            for (int i = 0; i < P; ++i) {
                const float2 z = Y ? fy[i] : k.z(fx[i], i);
                const float2 d = through<A, Y>(fd[i], fy[i], z, a.act);
                s0[i] = __fadd2_rn(s0[i], d);
                s1[i] = __ffma2_rn(d, __fadd2_rn(fx[i], k.m[UNI ? 0 : i]), s1[i]);
            }
        };
        constexpr int U = Y ? 2 : 4;
        int r = rl;
        for (; r + (U - 1) * rl_n < p.nr; r += U * rl_n) {
            Raw rx[U], rd[U], ry[U] = {};
#pragma unroll
            for (int u = 0; u < U; ++u) {
                rx[u] = *reinterpret_cast<const Raw *>(x + u * pitch);
                rd[u] = *reinterpret_cast<const Raw *>(delta + u * pitch);
                if constexpr (Y) ry[u] = *reinterpret_cast<const Raw *>(y + u * pitch);
            }
            x += U * pitch;
            delta += U * pitch;
            if constexpr (Y) y += U * pitch;
#pragma unroll
            for (int u = 0; u < U; ++u) add(rx[u], rd[u], ry[u]);
        }
        for (; r < p.nr; r += rl_n) {
            Raw ry{};
            if constexpr (Y) {
                ry = *reinterpret_cast<const Raw *>(y);
                y += pitch;
            }
            add(*reinterpret_cast<const Raw *>(x), *reinterpret_cast<const Raw *>(delta), ry);
            x += pitch;
            delta += pitch;
        }
        if constexpr (UNI) {
#pragma unroll
            for (int i = 0; i < P; ++i) s1[i] = __fmul2_rn(s1[i], both(k.rs));
        } else {
            int g[N];
            groups_of<N>(col, cg, g);
#pragma unroll
            for (int i = 0; i < P; ++i)
                s1[i] = __fmul2_rn(s1[i], make_float2(a.rstd[g0 + g[2 * i]], a.rstd[g0 + g[2 * i + 1 < N ? 2 * i + 1 : 0]]));
        }
        store_pairs<N>(part + rl * p.cb + col * N, s0);
        store_pairs<N>(part + a.part + rl * p.cb + col * N, s1);
    }
    __syncthreads();
    // a channel's sums: its row lanes in slices, one thread each, then the slices
    const int sl_n = p.cb < nt ? min(nt / p.cb, rl_n) : 1;
    if (sl_n > 1) {
        const int sl = threadIdx.x / p.cb, c = threadIdx.x - sl * p.cb;
        if (sl < sl_n) {
            float s0 = 0.0f, s1 = 0.0f;
            for (int r = sl; r < rl_n; r += sl_n) {
                s0 += part[r * p.cb + c];
                s1 += part[a.part + r * p.cb + c];
            }
            slices[sl * p.cb + c] = make_float2(s0, s1);
        }
        __syncthreads();
        if (threadIdx.x < p.cb) {
            float s0 = 0.0f, s1 = 0.0f;
            for (int q = 0; q < sl_n; ++q) {
                const float2 s = slices[q * p.cb + threadIdx.x];
                s0 += s.x;
                s1 += s.y;
            }
            ch[threadIdx.x] = make_float2(s0, s1);
        }
    } else {
        for (int c = threadIdx.x; c < p.cb; c += nt) {
            float s0 = 0.0f, s1 = 0.0f;
            for (int r = 0; r < rl_n; ++r) {
                s0 += part[r * p.cb + c];
                s1 += part[a.part + r * p.cb + c];
            }
            ch[c] = make_float2(s0, s1);
        }
    }
    if (STREAM || a.cluster == 1) __syncthreads();
    if constexpr (STREAM) {
        for (int c = threadIdx.x; c < p.cb; c += nt)
            a.pieces[(p.b * a.chunks + blockIdx.x % a.chunks) * a.filters + p.c0 + c] = ch[c];
        return;
    }
    const int q_n = a.cluster;
    float2 *all = ch;
    if (q_n > 1) {  // the unit's sums: every CTA adds the CTAs' in rank order, into its (now free) partials
        gn_cluster_arrive();
        gn_cluster_wait();
        all = reinterpret_cast<float2 *>(part);
        for (int c = threadIdx.x; c < p.cb; c += nt) {
            double s0 = 0.0, s1 = 0.0;
            for (int q = 0; q < q_n; ++q) {
                const float2 s = gn_peer_f32x2(ch + c, (unsigned)q);
                s0 += (double)s.x;
                s1 += (double)s.y;
            }
            all[c] = make_float2((float)s0, (float)s1);
        }
        gn_cluster_arrive();  // met again at the end: no CTA leaves while its sums may be read
        __syncthreads();
    }
    if (p.r0 == 0)
        for (int c = threadIdx.x; c < p.cb; c += nt) a.image[p.b * a.filters + p.c0 + c] = all[c];
    const int lane = threadIdx.x & 31;
    for (int g = threadIdx.x >> 5; g < p.ng; g += nt >> 5) {
        double s0 = 0.0, s1 = 0.0;
        for (int c = lane; c < cg; c += 32) {
            const double by = (double)sc[g * cg + c];
            s0 += by * (double)all[g * cg + c].x;
            s1 += by * (double)all[g * cg + c].y;
        }
        s0 = warp_sum(s0);
        s1 = warp_sum(s1);
        if (lane == 0) {
            const double rs = (double)a.rstd[g0 + g];
            mo[g] = make_float2((float)(-rs * s0 * a.inv_count), (float)(-rs * rs * s1 * a.inv_count));
        }
    }
    __syncthreads();

    for (int col = col0; col < v; col += vp) {
        if (!on) break;
        Affine<N, UNI> k;
        k.load(col, cg, a.mean + g0, a.rstd + g0, sc, bi);
        float2 c1[UNI ? 1 : P], c2[UNI ? 1 : P];
        load_moments<N, UNI>(col, cg, mo, c1, c2);
        // dx may be delta: a batch of rows is read before the first of it is written
        int64_t at = base + (int64_t)rl * a.filters + (int64_t)col * N;
        const T *x = static_cast<const T *>(a.x), *delta = static_cast<const T *>(a.delta),
                *y = static_cast<const T *>(a.y);
        T *dx = static_cast<T *>(a.dx);
        auto give = [&](Raw rx, Raw rd, Raw ry, int64_t to) {
            float2 fx[P], fd[P], fy[P] = {};
            V::unpack(rx, fx);
            V::unpack(rd, fd);
            if constexpr (Y) V::unpack(ry, fy);
            dx_of<P, A, Y, UNI>(fx, fd, fy, k, c1, c2, a.act);
            *reinterpret_cast<Raw *>(dx + to) = V::pack(fx);
        };
        constexpr int U = Y ? 2 : 4;
        int r = rl;
        for (; r + (U - 1) * rl_n < p.nr; r += U * rl_n) {
            Raw rx[U], rd[U], ry[U] = {};
#pragma unroll
            for (int u = 0; u < U; ++u) {
                rx[u] = *reinterpret_cast<const Raw *>(x + at + u * pitch);
                rd[u] = *reinterpret_cast<const Raw *>(delta + at + u * pitch);
                if constexpr (Y) ry[u] = *reinterpret_cast<const Raw *>(y + at + u * pitch);
            }
#pragma unroll
            for (int u = 0; u < U; ++u) give(rx[u], rd[u], ry[u], at + u * pitch);
            at += U * pitch;
        }
        for (; r < p.nr; r += rl_n) {
            Raw ry{};
            if constexpr (Y) ry = *reinterpret_cast<const Raw *>(y + at);
            give(*reinterpret_cast<const Raw *>(x + at), *reinterpret_cast<const Raw *>(delta + at), ry, at);
            at += pitch;
        }
    }
    if (q_n > 1) gn_cluster_wait();
}

// Streaming path: a block per (image, group): the chunks' channel sums added in order, then the group's
// (c1, c2).
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
        t0 = red[0][0] + red[0][1] + red[0][2] + red[0][3];
        t1 = red[1][0] + red[1][1] + red[1][2] + red[1][3];
        const double rs = (double)a.rstd[blockIdx.x];
        a.moments[blockIdx.x] = make_float2((float)(-rs * t0 * a.inv_count), (float)(-rs * rs * t1 * a.inv_count));
    }
}

template <class T, int VB, int A, bool Y, bool UNI>
__global__ void __launch_bounds__(256) k_gn_bwd_apply(const __grid_constant__ GnBwd a) {
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
        float2 c1[UNI ? 1 : P], c2[UNI ? 1 : P];
        load_moments<N, UNI>(col, (int)a.cg, a.moments + g0, c1, c2);
#pragma unroll 2
        for (int r = rl; r < p.nr; r += rl_n) {
            const int64_t at = base + (int64_t)r * a.filters + (int64_t)col * N;
            float2 fx[P], fd[P], fy[P] = {};
            V::unpack(*reinterpret_cast<const Raw *>(static_cast<const T *>(a.x) + at), fx);
            V::unpack(*reinterpret_cast<const Raw *>(static_cast<const T *>(a.delta) + at), fd);
            if constexpr (Y) V::unpack(*reinterpret_cast<const Raw *>(static_cast<const T *>(a.y) + at), fy);
            dx_of<P, A, Y, UNI>(fx, fd, fy, k, c1, c2, a.act);
            *reinterpret_cast<Raw *>(static_cast<T *>(a.dx) + at) = V::pack(fx);
        }
    }
}

// The updates: a block per 32 channels, 32 slices of the images (each added in order), then the slices.
__global__ void __launch_bounds__(1024) k_gn_updates(const float2 *image, int64_t batch, int64_t filters,
                                                     float *bias_updates, float *scale_updates, int add) {
    __shared__ double red[2][32][33];
    const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
    const int64_t c = (int64_t)blockIdx.x * 32 + tx;
    double s0 = 0.0, s1 = 0.0;
    if (c < filters) {
#pragma unroll 4
        for (int64_t b = ty; b < batch; b += 32) {
            const float2 v = image[b * filters + c];
            s0 += (double)v.x;
            s1 += (double)v.y;
        }
    }
    red[0][ty][tx] = s0;
    red[1][ty][tx] = s1;
    __syncthreads();
    // warp w: channel w's slices, a lane each
    s0 = warp_sum(red[0][tx][ty]);
    s1 = warp_sum(red[1][tx][ty]);
    const int64_t o = (int64_t)blockIdx.x * 32 + ty;
    if (tx == 0 && o < filters) {
        bias_updates[o] = (float)(add ? (double)bias_updates[o] + s0 : s0);
        scale_updates[o] = (float)(add ? (double)scale_updates[o] + s1 : s1);
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
    return gn_plan(batch, spatial, filters, groups, dtype_size(dtype), align, true);
}

template <class T, int VB, int A, bool Y, bool UNI>
dnb_status run_bwd(const GnBwd &a, const GnPlan &p, int64_t batch, const DeviceState *ds, cudaStream_t s) {
    const char *what = "gn_act_backward";
    const int64_t units = batch * p.nu;
    static std::atomic<int> opted[2][kMaxDevices];
    if (!p.stream) return gn_launch(k_gn_bwd<T, VB, A, Y, UNI, false>, a, units * p.cluster, p, ds, s, opted[0], what);
    DNB_TRY(gn_launch(k_gn_bwd<T, VB, A, Y, UNI, true>, a, units * p.chunks, p, ds, s, opted[1], what));
    if (batch * a.groups > 0x7fffffffll) return fail(DNB_ERR_UNSUPPORTED, "%s: too many groups", what);
    k_gn_bwd_merge<<<(unsigned)(batch * a.groups), 128, 0, s>>>(a);
    DNB_TRY(after_launch(s, what));
    k_gn_bwd_apply<T, VB, A, Y, UNI><<<(unsigned)(units * p.chunks), p.threads, (size_t)p.cb * 8, s>>>(a);
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
        k_gn_updates<<<ublocks, 1024, 0, s>>>(nullptr, 0, filters, bias_updates, scale_updates, 0);
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
    a.inv_count = 1.0 / ((double)spatial * (double)a.cg);
    a.act = act;
    a.cluster = p.cluster;
    a.unit_groups = (int)(p.cb / a.cg);
    a.part = (unsigned)p.part;
    auto with_y = [&]<class T, int VB, int A, bool UNI>() {
        return y ? run_bwd<T, VB, A, true, UNI>(a, p, batch, ds, s) : run_bwd<T, VB, A, false, UNI>(a, p, batch, ds, s);
    };
    const dnb_status st = dispatch_dtype(dtype, [&]<class T>() -> dnb_status {
        if (p.vb == 16 && p.uni)
            return dispatch_act(act, [&]<int A>() { return with_y.template operator()<T, 16, A, true>(); });
        if (p.vb == 16)
            return dispatch_act(act, [&]<int A>() { return with_y.template operator()<T, 16, A, false>(); });
        if (p.vb == 4)
            return dispatch_act(act, [&]<int A>() { return with_y.template operator()<T, 4, A, sizeof(T) == 4>(); });
        return with_y.template operator()<T, (int)sizeof(T), -1, true>();
    });
    DNB_TRY(st);
    k_gn_updates<<<ublocks, 1024, 0, s>>>(a.image, batch, filters, bias_updates, scale_updates, add);
    return after_launch(s, what);
}

}  // extern "C"
