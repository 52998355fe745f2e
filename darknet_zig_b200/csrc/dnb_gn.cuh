// Group norm on channels-last tensors: how the work is cut, shared by the forward (dnb_gn.cu) and the
// backward (dnb_gn_bwd.cu).
//
// A unit is one image's run of whole groups, `cb` channels wide (64 bytes of a row or more, so that the
// accesses of a row fill their sectors) and all `spatial` rows tall. A CTA, or a cluster of up to 8 CTAs
// that split the rows, takes a unit: the forward loads it into shared memory once, forms the statistics there
// and writes the outputs from there; the backward walks it twice, the second time in the L2 cache. So every
// tensor crosses HBM once. Units beyond what 8 CTAs can hold (or the cache keep) take the streaming path:
// partial statistics of row chunks, a merge, and a second read of the inputs.
//
// A thread owns one vector of channels (VB bytes) and every RL-th row, so per-channel values sit in its
// registers: V = cb / N vectors make a row; RL = T / V threads share a column, or, where a row is longer
// than the block, the block walks the columns in passes of T vectors. Where a group is a whole number of
// vectors (`uni`), what belongs to the group is one value per thread instead of one per channel.
#pragma once

#include <atomic>

#include "dnb_types.cuh"

namespace dnb {

struct GnPlan {
    int vb = 16;            // bytes of a vector
    int64_t cb = 0;         // channels of a unit (the last unit of an image may have fewer)
    int64_t nu = 0;         // units of an image
    int cluster = 1;        // CTAs of a unit
    int64_t rows = 0;       // rows of a CTA
    int threads = 256;
    bool stream = false;
    bool uni = false;       // a vector's channels are of one group
    int64_t chunks = 1;     // row chunks of a unit on the streaming path
    size_t slab = 0;        // bytes of one tensor's rows in shared memory, rounded to 16
    size_t part = 0;        // entries of a per-thread partial array
    size_t smem = 0;
};

constexpr size_t kGnSmemTarget = 112 * 1024;  // two CTAs an SM
constexpr size_t kGnSmemMax = 200 * 1024;
// Backward: bytes of one tensor's rows of a CTA that the L2 cache keeps from the sums to the outputs (two or
// three tensors, some 400 CTAs at a time: 60 MB of its 126).
constexpr size_t kGnReread = 64 * 1024;
constexpr size_t kGnStreamBytes = 64 * 1024;  // a streaming chunk's inputs
constexpr int kGnMaxCluster = 8;
constexpr int64_t kGnMaxGroup = 4096;         // channels of a group: a row of them, with the partials, fits an SM

inline dnb_status gn_shape_check(int64_t batch, int64_t spatial, int64_t filters, int64_t groups, const char *what) {
    if (batch < 0 || spatial < 0 || filters <= 0 || groups <= 0)
        return fail(DNB_ERR_INVALID, "%s: bad shape", what);
    if (filters % groups) return fail(DNB_ERR_INVALID, "%s: groups must divide filters", what);
    if (filters / groups > kGnMaxGroup)
        return fail(DNB_ERR_UNSUPPORTED, "%s: more than %lld channels in a group", what, (long long)kGnMaxGroup);
    if (filters > int64_t(1) << 30) return fail(DNB_ERR_UNSUPPORTED, "%s: too many filters", what);
    const int64_t most = int64_t(1) << 44;  // elements: offsets stay far inside 63 bits
    if (filters > most || (batch && spatial && (spatial > most / filters || batch > most / filters / spatial)))
        return fail(DNB_ERR_INVALID, "%s: too large", what);
    return DNB_OK;
}

inline int64_t gcd64(int64_t a, int64_t b) {
    while (b) {
        const int64_t t = a % b;
        a = b;
        b = t;
    }
    return a;
}

// align: the OR of the tensors' addresses.
inline GnPlan gn_plan(int64_t batch, int64_t spatial, int64_t filters, int64_t groups, int64_t esize, uintptr_t align,
                      bool backward) {
    constexpr int sms = 148;  // a B200's; the plan must not depend on the current device, for the workspace's size
    GnPlan p;
    const int64_t cg = filters / groups;
    const uintptr_t a = align | (uintptr_t)(filters * esize);
    p.vb = a % 16 == 0 ? 16 : a % 4 == 0 ? 4 : (int)esize;
    // groups that end on a vector's boundary; single elements where that makes units too wide to hold
    if (p.vb / esize / gcd64(p.vb / esize, cg) * cg > kGnMaxGroup) p.vb = (int)esize;
    const int64_t n = p.vb / esize;
    const int64_t step = n / gcd64(n, cg);
    p.uni = cg % n == 0 && (p.vb == 16 || n == 1);  // the narrower vectors' kernels take channels one by one
    auto cap = [&](int64_t g) { return g < groups ? g : groups; };
    int64_t per = cap(step * ((64 + step * cg * esize - 1) / (step * cg * esize)));
    auto slab_of = [&](int64_t g, int64_t rows) { return (size_t)((rows * g * cg * esize + 15) / 16 * 16); };
    auto units_of = [&](int64_t g) { return batch * ((groups + g - 1) / g); };
    // short planes: wider units, while they still fill the SMs twice
    while (per < groups && cap(2 * per) * cg <= 2048 && slab_of(cap(2 * per), spatial) <= (backward ? 8 : 16) * 1024 &&
           units_of(cap(2 * per)) >= 2 * sms)
        per = cap(2 * per);
    // rows narrower than 64 bytes rather than a second read of the inputs
    // (backward: rows that the L2 cache would not keep until they are read again)
    if (slab_of(per, (spatial + kGnMaxCluster - 1) / kGnMaxCluster) > (backward ? kGnReread : kGnSmemMax) && step < per)
        per = cap(step);
    p.cb = per * cg;
    p.nu = (groups + per - 1) / per;
    auto sizes = [&](bool held) {
        const int64_t v = p.cb / n, wide = p.threads > v ? p.threads : v;
        // forward: two floats a thread and vector (or channel), four floats a group;
        // backward: two floats a channel of a thread, two a thread (slices), two a channel, two a group
        p.part = (size_t)(((backward || !p.uni ? wide * n : wide) + 3) / 4 * 4);
        p.smem = (held ? p.slab : 0) + p.part * 8 + 64;
        p.smem += backward ? (size_t)p.threads * 8 + (size_t)p.cb * 8 + (size_t)per * 8 : (size_t)per * 16;
        p.smem += (size_t)p.cb * 8;  // scales and biases
    };
    auto shape = [&](int q) {
        p.cluster = q;
        p.rows = (spatial + q - 1) / q;
        p.slab = slab_of(per, p.rows);
        // a warp's fixed work (places, reductions) is that of a dozen vectors: no more threads than get those
        p.threads = !backward && p.rows * (p.cb / n) >= 12 * 512 ? 512 : 256;
        sizes(!backward);
    };
    auto too_big = [&] { return backward ? p.slab > kGnReread : p.smem > kGnSmemTarget; };
    int q = 1;
    shape(q);
    while (q < kGnMaxCluster && too_big()) shape(q *= 2);
    if (backward ? p.slab > kGnReread : p.smem > kGnSmemMax) {
        p.stream = true;
        p.cluster = 1;
        p.rows = (int64_t)(kGnStreamBytes / (size_t)(p.cb * esize * (backward ? 2 : 1)));
        if (p.rows < 1) p.rows = 1;
        p.chunks = (spatial + p.rows - 1) / p.rows;
        p.slab = 0;
        p.threads = 256;
        sizes(false);
        return p;
    }
    // few units: more CTAs for each, while a CTA keeps 8 KB (backward: of each tensor)
    while (q < kGnMaxCluster && units_of(per) * q < sms && p.slab > 16 * 1024) shape(q *= 2);
    return p;
}

// ---- device helpers ----

// Where a CTA works: unit, rows, columns. (32-bit arithmetic: a 64-bit division costs a hundred instructions,
// and a warp has a few hundred to run; gn_shape_check and gn_launch keep every count below 2^31.)
struct Place {
    int64_t b, c0, r0;
    int nr, cb, ng, g0;
};
template <class Args>
__device__ __forceinline__ Place place_of(const Args &a, unsigned per_unit) {
    Place p;
    const unsigned unit = blockIdx.x / per_unit, q = blockIdx.x - unit * per_unit;
    const unsigned b = unit / (unsigned)a.nu, u = unit - b * (unsigned)a.nu;
    p.b = b;
    const int c0 = (int)u * (int)a.cb, left_c = (int)a.filters - c0;
    p.c0 = c0;
    p.cb = (int)a.cb < left_c ? (int)a.cb : left_c;
    p.g0 = (int)u * a.unit_groups;
    p.ng = (int)a.groups - p.g0 < a.unit_groups ? (int)a.groups - p.g0 : a.unit_groups;
    p.r0 = (int64_t)q * a.rows;
    const int64_t left = a.spatial - p.r0;
    p.nr = (int)(left < 0 ? 0 : left < a.rows ? left : a.rows);
    return p;
}

// A vector from global to shared memory without passing through registers, where the hardware has such a copy
// (16 or 4 bytes): a thread has all its rows in flight at once. gn_arrived(): the thread's own copies are there.
template <int VB>
__device__ __forceinline__ void gn_copy(void *dst, const void *src) {
    if constexpr (VB == 16)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(dst)), "l"(src)
                     : "memory");
    else if constexpr (VB == 4)
        asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"((uint32_t)__cvta_generic_to_shared(dst)), "l"(src)
                     : "memory");
    else
        *static_cast<typename RawVec<VB>::type *>(dst) = *static_cast<const typename RawVec<VB>::type *>(src);
}
__device__ __forceinline__ void gn_arrived() { asm volatile("cp.async.wait_all;" ::: "memory"); }

__device__ __forceinline__ void gn_cluster_arrive() {
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
}
__device__ __forceinline__ void gn_cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
// The address of `p` (shared memory) in the cluster's CTA `rank`.
__device__ __forceinline__ uint32_t gn_peer(const void *p, unsigned rank) {
    uint32_t a = (uint32_t)__cvta_generic_to_shared(p), r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(rank));
    return r;
}
__device__ __forceinline__ float2 gn_peer_f32x2(const void *p, unsigned rank) {
    float2 v;
    asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(gn_peer(p, rank)) : "memory");
    return v;
}
// The local group of each channel of the vector at column `col`, in order (one division a vector).
template <int N>
__device__ __forceinline__ void groups_of(int col, int cg, int (&g)[N]) {
    g[0] = col * N / cg;
    int left = cg - (col * N - g[0] * cg);
#pragma unroll
    for (int j = 1; j < N; ++j) {
        const bool next = --left == 0;
        g[j] = g[j - 1] + next;
        if (next) left = cg;
    }
}

// The unit's scales and biases into shared memory, early: by the time they are needed their latency is over.
__device__ __forceinline__ void gn_stage_params(float *sc, const float *scales, const float *biases, const Place &p) {
    for (int c = threadIdx.x; c < p.cb; c += blockDim.x) {
        sc[c] = scales[p.c0 + c];
        sc[p.cb + c] = biases[p.c0 + c];
    }
}

// N consecutive floats as pairs, in the widest accesses the alignment of p allows for every N (16 bytes from
// N = 4 on: the units start on whole vectors). From global memory one by one (the caller's vectors are
// aligned to their element alone).
template <int N>
__device__ __forceinline__ void load_pairs(const float *p, float2 (&f)[(N + 1) / 2]) {
    if constexpr (N == 1) {
        f[0] = make_float2(*p, 0.0f);
    } else if constexpr (N == 2) {
        f[0] = *reinterpret_cast<const float2 *>(p);
    } else {
#pragma unroll
        for (int i = 0; i < N / 2; i += 2) {
            const float4 v = *reinterpret_cast<const float4 *>(p + 2 * i);
            f[i] = make_float2(v.x, v.y);
            f[i + 1] = make_float2(v.z, v.w);
        }
    }
}

// z = (x - mean)*(rstd*scale) + bias for a vector's channels; the forward and the backward's recomputed output
// share it, so that both see the same z.
template <int N, bool UNI>
struct Affine {
    static constexpr int P = (N + 1) / 2;
    float2 m[UNI ? 1 : P], k[P], b[P];
    float rs;  // UNI: the group's rstd
    __device__ __forceinline__ void load(int col, int cg, const float *mean, const float *rstd, const float *scales,
                                         const float *biases) {
        int g[N];
        if constexpr (!UNI) groups_of<N>(col, cg, g);
        const int lg = UNI ? col * N / cg : 0;
        const float um = UNI ? mean[lg] : 0.0f, ur = UNI ? rstd[lg] : 0.0f;
        if constexpr (UNI) m[0] = both(-um);
        rs = ur;
        load_pairs<N>(scales + col * N, k);
        load_pairs<N>(biases + col * N, b);
#pragma unroll
        for (int i = 0; i < P; ++i) {
            const bool two = 2 * i + 1 < N;
            if constexpr (!UNI) m[i] = make_float2(-mean[g[2 * i]], two ? -mean[g[two ? 2 * i + 1 : 0]] : 0.0f);
            k[i] = __fmul2_rn(k[i], UNI ? both(ur) : make_float2(rstd[g[2 * i]], two ? rstd[g[two ? 2 * i + 1 : 0]] : 0.0f));
        }
    }
    __device__ __forceinline__ float2 z(float2 x, int i) const {
        return __ffma2_rn(__fadd2_rn(x, m[UNI ? 0 : i]), k[i], b[i]);
    }
};

// Launches a GN kernel with its shared memory and cluster size.
template <class K, class Args>
dnb_status gn_launch(K kernel, const Args &args, int64_t blocks, const GnPlan &p, const DeviceState *ds,
                     cudaStream_t s, std::atomic<int> *opted, const char *what) {
    if (!opted[ds->device].load(std::memory_order_acquire)) {
        DNB_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, ds->max_smem_optin));
        opted[ds->device].store(1, std::memory_order_release);
    }
    if (blocks > 0x7fffffffll || p.smem > (size_t)ds->max_smem_optin)
        return fail(DNB_ERR_UNSUPPORTED, "%s: too many units, or too many channels in a group", what);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)blocks);
    cfg.blockDim = dim3((unsigned)p.threads);
    cfg.dynamicSmemBytes = p.smem;
    cfg.stream = s;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = (unsigned)p.cluster;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = p.cluster > 1 ? 1 : 0;
    DNB_CUDA(cudaLaunchKernelEx(&cfg, kernel, args));
    return after_launch(s, what);
}

}  // namespace dnb
