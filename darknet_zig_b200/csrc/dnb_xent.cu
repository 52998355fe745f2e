// Softmax + cross entropy of a connected layer's outputs, never stored (the place of misc.zig:41-77 after
// connected.zig:92-119, at numbers of classes whose outputs would not fit or not pay).
//
//   z = x w^T + b;  lse = log sum exp z;  loss = lse - z[label];  d = f ((n == label) - exp(z - lse))
//
// Forward: k_gemm's epilogue takes each tile's rows to (max, sum of exponentials) and picks out the label's z;
// k_xent_close merges the tiles. 2 * rows * classes * inputs operations, x and w read: bound by the tensor
// cores from a few hundred rows on, by reading w below.
//
// Backward: for a piece of the classes at a time, the product again with an epilogue that leaves
// d / f * 2^14 in 16 bits (d / f lies in [-1, 1]; the factor keeps probabilities down to 2^-28 among f16's
// normal numbers), then dx += d w and dW = d^T x. Three products of the same size, the recomputed one in
// place of rows * classes stored outputs. A piece is as wide as 256 MB of d allow: dx is added up in fp32
// over the pieces (one read and write of it a piece), so fewer pieces cost less.
//
// Padding rows are left out of all products: their indices are squeezed out of the row list first, and the
// kernels take the number of rows that are left from the device.
#include "dnb_epilogue.cuh"
#include "dnb_pack.cuh"

namespace dnb {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kDeltaScale = 16384.0f;

// ---- the rows that count ----

// rows[0 .. *count) = the rows whose label is in [0, classes), in order. With factors, meta = {norm, back}:
// norm * the largest |factor| of those rows lies in [1, 2), back = scale / norm (so that a product with
// norm * factor needs back).
__global__ void __launch_bounds__(1024) k_kept_rows(const int32_t *labels, int64_t batch, int64_t classes, int *rows,
                                                    int *count, const float *factor, float scale, float *meta) {
    __shared__ int sums[32];
    __shared__ float tops[32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    // a warp takes a run of 32-row blocks; a lane a row of each
    const int64_t blocks = (batch + 31) / 32, run = (blocks + 31) / 32, b0 = warp * run,
                  b1 = b0 + run < blocks ? b0 + run : blocks;
    auto keeps = [&](int64_t b) {
        const int64_t r = b * 32 + lane;
        if (r >= batch) return false;
        const int l = labels[r];
        return l >= 0 && l < classes;
    };
    int mine = 0;
#pragma unroll 8
    for (int64_t b = b0; b < b1; ++b) mine += keeps(b);
    mine = __reduce_add_sync(0xffffffffu, mine);
    if (lane == 0) sums[warp] = mine;
    __syncthreads();
    int base = 0, all = 0;
    for (int w = 0; w < 32; ++w) {
        if (w < warp) base += sums[w];
        all += sums[w];
    }
    if (threadIdx.x == 0) *count = all;
    float top = 0.0f;
#pragma unroll 8
    for (int64_t b = b0; b < b1; ++b) {
        const bool keep = keeps(b);
        const unsigned mask = __ballot_sync(0xffffffffu, keep);
        if (keep) {
            const int64_t r = b * 32 + lane;
            rows[base + __popc(mask & ((1u << lane) - 1u))] = (int)r;
            if (factor) top = fmaxf(top, fabsf(factor[r]));
        }
        base += __popc(mask);
    }
    if (!factor) return;
    top = warp_max(top);
    if (lane == 0) tops[warp] = top;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < 32; ++w) top = fmaxf(top, tops[w]);
        int e = 1;
        if (top > 0.0f && top <= 3.4e38f) frexpf(top, &e);
        if (e > 120) e = 120;
        if (e < -120) e = -120;
        meta[0] = ldexpf(1.0f, 1 - e);
        meta[1] = scale * ldexpf(1.0f, e - 1) / kDeltaScale;
    }
}

// ---- forward ----

// Each row's (max, sum of exp(z - max)) over a tile's columns, and the label's z.
struct EpiStats {
    const float *bias;
    const int32_t *labels;
    const int *rows, *m_dev;  // NULL: every row
    float2 *part;             // [tile][m]
    float *at_label;          // [m]
    int64_t m, n;
    int bn;  // columns of a thread's part of a tile

    struct State {
        float top, sum;
        int label;
    };
    __device__ __forceinline__ void begin(State &s, int64_t row, int64_t) const {
        s.top = __int_as_float(0xff800000);  // -inf
        s.sum = 0.0f;
        s.label = -1;
        if (row < (m_dev ? *m_dev : m)) s.label = labels[rows ? rows[row] : row];
    }
    // what the exponents are taken from: the maximum, or 0 while it is infinite (then no z but infinities or
    // nothing has been seen, and the sums come out as log sum exp's limits)
    static __device__ __forceinline__ float shift(float top) { return fabsf(top) < __int_as_float(0x7f800000) ? top : 0.0f; }

    struct Ahead {};
    __device__ __forceinline__ void fetch(const State &, Ahead &, int64_t) const {}

    __device__ __forceinline__ void columns(State &s, float2 (&v)[16], const float *tile_bias, const Ahead &,
                                            int64_t row, int64_t col) const {
        const int cols = (int)(n - col < 32 ? n - col : 32);
        const float none = __int_as_float(0xff800000);
        if (bias) add_bias32(v, tile_bias);
        if (cols < 32) {
#pragma unroll
            for (int j = 0; j < 16; ++j) {
                if (2 * j >= cols) v[j].x = none;
                if (2 * j + 1 >= cols) v[j].y = none;
            }
        }
        const int64_t at = (int64_t)s.label - col;
        if (at >= 0 && at < cols) {
#pragma unroll
            for (int j = 0; j < 16; ++j) {
                if (2 * j == at) at_label[row] = v[j].x;
                if (2 * j + 1 == at) at_label[row] = v[j].y;
            }
        }
        float top = s.top;
#pragma unroll
        for (int j = 0; j < 16; ++j) top = fmaxf(top, fmaxf(v[j].x, v[j].y));
        const float to = shift(top);
        float2 sum = make_float2(s.sum == 0.0f ? 0.0f : s.sum * quick_exp(shift(s.top) - to), 0.0f);
#pragma unroll
        for (int j = 0; j < 16; ++j) {
            const float2 d = __fadd2_rn(v[j], both(-to));
            sum = __fadd2_rn(sum, make_float2(quick_exp(d.x), quick_exp(d.y)));
        }
        s.top = top;
        s.sum = sum.x + sum.y;
    }
    __device__ __forceinline__ void end(State &s, int64_t row, int64_t col0) const {
        if (row < (m_dev ? *m_dev : m)) part[(col0 / bn) * m + row] = make_float2(shift(s.top), s.sum);
    }
};

// Merges the tiles of a row: 32 rows a block, 32 slices of the tiles each; the maximum first, so that the sums
// need no order, then the slices in a fixed one.
__global__ void __launch_bounds__(1024) k_xent_close(const float2 *part, const float *at_label, const int32_t *labels,
                                                     const int *rows, const int *m_dev, int64_t m, int64_t tiles,
                                                     int64_t classes, float *loss, float *lse) {
    __shared__ float red[32][33];
    const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
    const int64_t row = (int64_t)blockIdx.x * 32 + tx, count = m_dev ? *m_dev : m;
    // a tile whose sum is 0 has only classes of -inf: its maximum stands for nothing
    const float none = __int_as_float(0xff800000);
    auto load = [&](int64_t t) {
        float2 p = part[t * m + row];
        if (p.y == 0.0f) p.x = none;
        return p;
    };
    constexpr int kHeld = 8;
    float2 held[kHeld];  // a slice's first tiles, read once
    float top = none;
    if (row < count) {
#pragma unroll
        for (int i = 0; i < kHeld; ++i) {
            const int64_t t = ty + 32 * i;
            held[i] = t < tiles ? load(t) : make_float2(none, 0.0f);
            top = fmaxf(top, held[i].x);
        }
        for (int64_t t = ty + 32 * kHeld; t < tiles; t += 32) top = fmaxf(top, load(t).x);
    }
    red[ty][tx] = top;
    __syncthreads();
    top = warp_max(red[tx][ty]);  // warp w: row w's slices
    __syncthreads();
    if (tx == 0) red[0][ty] = top;
    __syncthreads();
    top = red[0][tx];
    __syncthreads();
    float sum = 0.0f;
    if (row < count) {
#pragma unroll
        for (int i = 0; i < kHeld; ++i)
            if (held[i].y != 0.0f) sum += held[i].y * exp2f((held[i].x - top) * kLog2e);
        for (int64_t t = ty + 32 * kHeld; t < tiles; t += 32) {
            const float2 p = load(t);
            if (p.y != 0.0f) sum += p.y * exp2f((p.x - top) * kLog2e);
        }
    }
    red[ty][tx] = sum;
    __syncthreads();
    sum = warp_sum(red[tx][ty]);
    __syncthreads();
    if (tx == 0) red[0][ty] = sum;
    __syncthreads();
    if (ty != 0) return;
    if (row < count) {
        const int64_t at = rows ? rows[row] : row;
        if (rows || (labels[at] >= 0 && labels[at] < classes)) {
            const float l = top + logf(red[0][tx]);
            lse[at] = l;
            loss[at] = l - at_label[row];
        }
    }
    // padding rows, each by the thread of its own index
    if (row < m && (labels[row] < 0 || labels[row] >= classes)) lse[row] = loss[row] = 0.0f;
}

// ---- backward ----

// d / f * 2^14 of a piece of the classes, in 16 bits, and each 32 rows' column sums of d.
struct EpiDelta {
    const float *bias;
    const int32_t *labels;
    const float *lse, *row_factor;
    const int *rows, *count;
    void *d;
    int64_t ld, n, c0;  // row stride, classes of the piece, the piece's first class
    float *sums;        // [32 rows][ld]; NULL: no bias updates
    float scale;
    int dtype;

    struct State {
        int at;       // label - c0
        float lse, f;
        int kept;
        int zero;     // rows that follow the kept ones up to a multiple of 64: zeros
    };
    __device__ __forceinline__ void begin(State &s, int64_t row, int64_t) const {
        const int m = *count;
        s.kept = row < m;
        s.zero = !s.kept && row < (m + 63) / 64 * 64;
        s.at = -1;
        s.lse = s.f = 0.0f;
        if (!s.kept) return;
        const int r = rows[row];
        s.at = labels[r] - (int)c0;
        s.lse = lse[r];
        s.f = scale * (row_factor ? row_factor[r] : 1.0f);
    }
    __device__ __forceinline__ void end(State &, int64_t, int64_t) const {}

    template <class T>
    __device__ __forceinline__ void store(const float2 (&v)[16], int64_t row, int64_t col, int cols) const {
        T *p = static_cast<T *>(d) + row * ld + col;
        if (cols == 32) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                float2 f[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) f[i] = __fmul2_rn(v[4 * j + i], both(kDeltaScale));
                reinterpret_cast<uint4 *>(p)[j] = Pairs<T, 16>::pack(f);
            }
        } else {
#pragma unroll
            for (int j = 0; j < 16; ++j) {
                if (2 * j < cols) p[2 * j] = Elem<T>::from(v[j].x * kDeltaScale);
                if (2 * j + 1 < cols) p[2 * j + 1] = Elem<T>::from(v[j].y * kDeltaScale);
            }
        }
    }
    struct Ahead {};
    __device__ __forceinline__ void fetch(const State &, Ahead &, int64_t) const {}
    __device__ __forceinline__ void columns(State &s, float2 (&v)[16], const float *tile_bias, const Ahead &,
                                            int64_t row, int64_t col) const {
        const int cols = (int)(n - col < 32 ? n - col : 32);
        if (s.kept) {
            if (bias) add_bias32(v, tile_bias);
#pragma unroll
            for (int j = 0; j < 16; ++j) {
                const float2 z = __fadd2_rn(v[j], both(-s.lse));
                v[j] = make_float2(-quick_exp(z.x), -quick_exp(z.y));
            }
            const int64_t at = (int64_t)s.at - col;
            if (at >= 0 && at < 32) {
#pragma unroll
                for (int j = 0; j < 16; ++j) {
                    if (2 * j == at) v[j].x += 1.0f;
                    if (2 * j + 1 == at) v[j].y += 1.0f;
                }
            }
        } else {
#pragma unroll
            for (int j = 0; j < 16; ++j) v[j] = both(0.0f);
        }
        if (s.kept || s.zero) {
            if (dtype == DNB_BF16) store<__nv_bfloat16>(v, row, col, cols);
            else store<__half>(v, row, col, cols);
        }
        if (sums) {  // lane j ends up with column j's sum over the warp's 32 rows
            const int lane = threadIdx.x & 31;
            float u[32];
#pragma unroll
            for (int j = 0; j < 16; ++j) {
                u[2 * j] = v[j].x * s.f;
                u[2 * j + 1] = v[j].y * s.f;
            }
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) {
                const bool up = lane & o;
#pragma unroll
                for (int j = 0; j < o; ++j) {
                    const float send = up ? u[j] : u[j + o], keep = up ? u[j + o] : u[j];
                    u[j] = keep + __shfl_xor_sync(0xffffffffu, send, o);
                }
            }
            const int64_t block = row / 32;
            if (block * 32 < *count && lane < cols) sums[block * ld + col + lane] = u[0];
        }
    }
};

// Column sums over the row blocks that hold kept rows.
__global__ void __launch_bounds__(256) k_delta_sums(const float *sums, const int *count, int64_t n, int64_t ld,
                                                    float *out, int add) {
    __shared__ double red[8][32];
    const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
    const int64_t c = (int64_t)blockIdx.x * 32 + tx, blocks = (*count + 31) / 32;
    double s = 0.0;
    if (c < n)
#pragma unroll 4
        for (int64_t q = ty; q < blocks; q += 8) s += (double)sums[q * ld + c];
    red[ty][tx] = s;
    __syncthreads();
    if (ty == 0 && c < n) {
        for (int i = 1; i < 8; ++i) s += red[i][tx];
        out[c] = (float)(add ? (double)out[c] + s : s);
    }
}

// The products whose results stay in the epilogue.
template <class Epi>
dnb_status xent_product(const Tiles &t, const Operand &a, const Operand &b, int dtype, int64_t m, int64_t n, int64_t k,
                        const Epi &e, const DeviceState *ds, cudaStream_t s, const char *what, const int *m_dev) {
    if (t.ctas == 2) return launch_gemm<GemmCfg<2, 256, false, false>>(a, b, dtype, m, n, k, e, ds, s, what, 1, m_dev);
    if (t.split > 1)
        return launch_gemm<GemmCfg<1, 128, false, false, true>>(a, b, dtype, m, n, k, e, ds, s, what, t.split, m_dev);
    return launch_gemm<GemmCfg<1, 128, false, false>>(a, b, dtype, m, n, k, e, ds, s, what, 1, m_dev);
}

// ---- the caller's workspace ----

// Squeezing out padding rows pays from a few tiles of rows on: below, a forward takes every row.
bool squeezes(int64_t m) { return m > 512; }

struct FwdSpace {
    void *x, *w;
    float2 *part;
    float *at_label;
    int *rows, *count;
    int64_t tiles;
    Tiles shape;
    size_t total;
};
FwdSpace fwd_space(void *ws, const void *x, int64_t ldx, const void *w, int64_t ldw, int64_t m, int64_t k, int64_t n) {
    Carver c(ws);
    FwdSpace f{};
    f.shape = pick_tiles(m, n, k);
    f.tiles = (n + f.shape.ew - 1) / f.shape.ew;
    f.part = static_cast<float2 *>(c.take(f.tiles * m * 8));
    f.at_label = static_cast<float *>(c.take(m * 4));
    if (squeezes(m)) {
        f.rows = static_cast<int *>(c.take(m * 4));
        f.count = static_cast<int *>(c.take(4));
        f.x = c.take(packed_bytes((m + 63) / 64 * 64, k));
    } else if (!tma_ready(x, m > 1 ? ldx : 8)) {
        f.x = c.take(packed_bytes(m, k));
    }
    if (!tma_ready(w, n > 1 ? ldw : 8)) f.w = c.take(packed_bytes(n, k));
    f.total = c.used;
    return f;
}

struct BwdSpace {
    void *x, *xs, *w, *d;
    float *dx, *sums, *meta;
    int *rows, *count;
    int64_t piece, pieces;
    size_t total;
};
constexpr int64_t kPieceBytes = 256ll << 20;
BwdSpace bwd_space(void *ws, const void *w, int64_t ldw, int64_t m, int64_t k, int64_t n) {
    Carver c(ws);
    BwdSpace b{};
    const int64_t rows = (m + 63) / 64 * 64;
    int64_t p = kPieceBytes / (rows * 2) / 256 * 256;
    if (p < 2048) p = 2048;
    if (p > (n + 7) / 8 * 8) p = (n + 7) / 8 * 8;
    b.pieces = (n + p - 1) / p;
    // pieces of the same width, but for the last
    b.piece = b.pieces == 1 ? p : ((n + b.pieces - 1) / b.pieces + 255) / 256 * 256;
    b.pieces = (n + b.piece - 1) / b.piece;
    b.rows = static_cast<int *>(c.take(m * 4));
    b.count = static_cast<int *>(c.take(4));
    b.meta = static_cast<float *>(c.take(8));
    b.x = c.take(packed_bytes(rows, k));
    b.xs = c.take(packed_bytes(rows, k));
    if (!tma_ready(w, n > 1 ? ldw : 8)) b.w = c.take(packed_bytes(n, k));
    b.d = c.take(rows * b.piece * 2);
    b.dx = static_cast<float *>(c.take(b.pieces > 1 ? m * k * 4 : 0));
    b.sums = static_cast<float *>(c.take((m + 31) / 32 * b.piece * 4));
    b.total = c.used;
    return b;
}

}  // namespace
}  // namespace dnb

using namespace dnb;

extern "C" {

dnb_status dnb_connected_xent_forward_workspace(const void *x, int64_t ldx, const void *w, int64_t ldw, int dtype,
                                                int64_t batch, int64_t inputs, int64_t classes, size_t *bytes) {
    const char *what = "connected_xent_forward_workspace";
    if (!bytes) return fail(DNB_ERR_INVALID, "%s: bytes is null", what);
    DNB_TRY(product_shape_check(dtype, batch, inputs, classes, what));
    *bytes = 0;
    if (batch == 0 || classes == 0 || inputs == 0) return DNB_OK;
    *bytes = fwd_space(nullptr, x, ldx, w, ldw, batch, inputs, classes).total;
    return DNB_OK;
}

dnb_status dnb_connected_xent_forward(const void *x, int64_t ldx, const void *w, int64_t ldw, const float *biases,
                                      const int32_t *labels, float *loss, float *lse, int dtype, int64_t batch,
                                      int64_t inputs, int64_t classes, void *workspace, size_t workspace_bytes,
                                      dnb_stream stream) {
    const char *what = "connected_xent_forward";
    DNB_TRY(product_shape_check(dtype, batch, inputs, classes, what));
    if (batch == 0) return DNB_OK;
    if (classes == 0 || inputs == 0) return fail(DNB_ERR_INVALID, "%s: no classes or no inputs", what);
    if (!x || !w || !labels || !loss || !lse) return fail(DNB_ERR_INVALID, "%s: null pointer", what);
    if (!matrix_ok(x, batch, inputs, ldx, dtype) || !matrix_ok(w, classes, inputs, ldw, dtype) ||
        (reinterpret_cast<uintptr_t>(biases) | reinterpret_cast<uintptr_t>(labels) |
         reinterpret_cast<uintptr_t>(loss) | reinterpret_cast<uintptr_t>(lse)) % 4)
        return fail(DNB_ERR_INVALID, "%s: a row stride is shorter than its row, too large, or a pointer is misaligned",
                    what);
    const int64_t sx = matrix_span(batch, inputs, ldx, 2), sw = matrix_span(classes, inputs, ldw, 2), v = batch * 4;
    for (const void *o : {(const void *)loss, (const void *)lse})
        if (overlaps(o, v, x, sx) || overlaps(o, v, w, sw) || overlaps(o, v, biases, classes * 4) ||
            overlaps(o, v, labels, v))
            return fail(DNB_ERR_INVALID, "%s: overlapping tensors", what);
    if (overlaps(loss, v, lse, v)) return fail(DNB_ERR_INVALID, "%s: overlapping tensors", what);
    const FwdSpace f = fwd_space(workspace, x, ldx, w, ldw, batch, inputs, classes);
    DNB_TRY(workspace_check(workspace, workspace_bytes, f.total, what));
    DeviceState *ds = nullptr;
    DNB_TRY(current_device(&ds));
    const cudaStream_t s = as_stream(stream);
    Operand a{x, ldx}, b{w, ldw};
    if (f.rows) {
        k_kept_rows<<<1, 1024, 0, s>>>(labels, batch, classes, f.rows, f.count, nullptr, 1.0f, nullptr);
        DNB_TRY(after_launch(s, what));
    }
    Gather g;
    g.rows = f.rows;
    g.count = f.count;
    DNB_TRY(pack_rows({x, ldx, f.x, batch, inputs}, {w, ldw, f.w, classes, inputs}, dtype, g, ds, s, what));
    if (f.x) a = {f.x, packed_ld(inputs)};
    if (f.w) b = {f.w, packed_ld(inputs)};
    EpiStats e{biases, labels, f.rows, f.count, f.part, f.at_label, batch, classes, f.shape.ew};
    DNB_TRY(xent_product(f.shape, a, b, dtype, batch, classes, inputs, e, ds, s, what, f.count));
    k_xent_close<<<(unsigned)((batch + 31) / 32), 1024, 0, s>>>(f.part, f.at_label, labels, f.rows, f.count, batch,
                                                               f.tiles, classes, loss, lse);
    return after_launch(s, what);
}

dnb_status dnb_connected_xent_backward_workspace(const void *x, int64_t ldx, const void *w, int64_t ldw, int dtype,
                                                 int64_t batch, int64_t inputs, int64_t classes, size_t *bytes) {
    const char *what = "connected_xent_backward_workspace";
    (void)x;
    (void)ldx;
    if (!bytes) return fail(DNB_ERR_INVALID, "%s: bytes is null", what);
    DNB_TRY(product_shape_check(dtype, batch, inputs, classes, what));
    *bytes = 0;
    if (batch == 0 || classes == 0 || inputs == 0) return DNB_OK;
    *bytes = bwd_space(nullptr, w, ldw, batch, inputs, classes).total;
    return DNB_OK;
}

dnb_status dnb_connected_xent_backward(const void *x, int64_t ldx, const void *w, int64_t ldw, const float *biases,
                                       const int32_t *labels, const float *lse, const float *row_scales, float scale,
                                       void *dx, int64_t lddx, float *bias_updates, void *weight_updates,
                                       int64_t lddw, int updates_dtype, int dtype, int64_t batch, int64_t inputs,
                                       int64_t classes, int accumulate, void *workspace, size_t workspace_bytes,
                                       dnb_stream stream) {
    const char *what = "connected_xent_backward";
    DNB_TRY(product_shape_check(dtype, batch, inputs, classes, what));
    if (accumulate & ~(DNB_ACC_UPDATES | DNB_ACC_DELTA)) return fail(DNB_ERR_INVALID, "%s: unknown accumulate bits", what);
    if (weight_updates && updates_dtype != dtype && updates_dtype != DNB_F32)
        return fail(DNB_ERR_INVALID, "%s: updates_dtype must be dtype or f32", what);
    if (classes == 0 || inputs == 0) return fail(DNB_ERR_INVALID, "%s: no classes or no inputs", what);
    if (batch > 0 && (!x || !w || !labels || !lse)) return fail(DNB_ERR_INVALID, "%s: null pointer", what);
    if (!matrix_ok(x, batch, inputs, ldx, dtype) || !matrix_ok(w, classes, inputs, ldw, dtype) ||
        (dx && !matrix_ok(dx, batch, inputs, lddx, dtype)) ||
        (weight_updates && !matrix_ok(weight_updates, classes, inputs, lddw, updates_dtype)) ||
        (reinterpret_cast<uintptr_t>(biases) | reinterpret_cast<uintptr_t>(labels) | reinterpret_cast<uintptr_t>(lse) |
         reinterpret_cast<uintptr_t>(row_scales) | reinterpret_cast<uintptr_t>(bias_updates)) % 4)
        return fail(DNB_ERR_INVALID, "%s: a row stride is shorter than its row, too large, or a pointer is misaligned",
                    what);
    struct Span {
        const void *p;
        int64_t n;
    };
    const Span in[6] = {{x, matrix_span(batch, inputs, ldx, 2)}, {w, matrix_span(classes, inputs, ldw, 2)},
                        {biases, classes * 4}, {labels, batch * 4}, {lse, batch * 4}, {row_scales, batch * 4}};
    const Span out[3] = {{dx, matrix_span(batch, inputs, lddx, 2)},
                         {weight_updates, matrix_span(classes, inputs, lddw, dtype_size(updates_dtype))},
                         {bias_updates, classes * 4}};
    for (int o = 0; o < 3; ++o) {
        for (const Span &i : in)
            if (overlaps(out[o].p, out[o].n, i.p, i.n)) return fail(DNB_ERR_INVALID, "%s: overlapping tensors", what);
        for (int q = 0; q < o; ++q)
            if (overlaps(out[o].p, out[o].n, out[q].p, out[q].n))
                return fail(DNB_ERR_INVALID, "%s: overlapping tensors", what);
    }
    DeviceState *ds = nullptr;
    const cudaStream_t s = as_stream(stream);
    const bool add_w = accumulate & DNB_ACC_UPDATES, add_x = accumulate & DNB_ACC_DELTA;
    if (batch == 0) {
        if (add_w || (!weight_updates && !bias_updates)) return DNB_OK;
        DNB_TRY(current_device(&ds));
        if (weight_updates)
            DNB_TRY(zero_rows(weight_updates, classes, inputs, lddw, dtype_size(updates_dtype), ds, s, what));
        if (bias_updates) DNB_TRY(zero_rows(bias_updates, 1, classes, classes, 4, ds, s, what));
        return DNB_OK;
    }
    const BwdSpace f = bwd_space(workspace, w, ldw, batch, inputs, classes);
    DNB_TRY(workspace_check(workspace, workspace_bytes, f.total, what));
    DNB_TRY(current_device(&ds));
    k_kept_rows<<<1, 1024, 0, s>>>(labels, batch, classes, f.rows, f.count, row_scales, scale, f.meta);
    DNB_TRY(after_launch(s, what));
    Gather g;
    g.rows = f.rows;
    g.count = f.count;
    DNB_TRY(pack_rows({x, ldx, f.x, batch, inputs}, {w, ldw, f.w, classes, inputs}, dtype, g, ds, s, what));
    const Operand xp{f.x, packed_ld(inputs)};
    Operand xs = xp, wp{w, ldw};
    if (weight_updates && row_scales) {
        g.factor = row_scales;
        g.norm = f.meta;
        DNB_TRY(pack_rows({x, ldx, f.xs, batch, inputs}, {}, dtype, g, ds, s, what));
        xs.p = f.xs;
    }
    if (f.w) wp = {f.w, packed_ld(inputs)};
    if (dx && !add_x) DNB_TRY(zero_rows(dx, batch, inputs, lddx, 2, ds, s, what, labels, classes));
    const int64_t rows = (batch + 63) / 64 * 64;
    for (int64_t p = 0; p < f.pieces; ++p) {
        const int64_t c0 = p * f.piece, n = classes - c0 < f.piece ? classes - c0 : f.piece;
        const Operand wq{static_cast<const char *>(wp.p) + c0 * wp.ld * 2, wp.ld};
        EpiDelta e;
        e.bias = biases ? biases + c0 : nullptr;
        e.labels = labels;
        e.lse = lse;
        e.row_factor = row_scales;
        e.rows = f.rows;
        e.count = f.count;
        e.d = f.d;
        e.ld = f.piece;
        e.n = n;
        e.c0 = c0;
        e.sums = bias_updates ? f.sums : nullptr;
        e.scale = scale;
        e.dtype = dtype;
        DNB_TRY(xent_product(pick_tiles(batch, n, inputs), xp, wq, dtype, rows, n, inputs, e, ds, s, what, f.count));
        if (bias_updates) {
            k_delta_sums<<<(unsigned)((n + 31) / 32), 256, 0, s>>>(f.sums, f.count, n, f.piece, bias_updates + c0, add_w);
            DNB_TRY(after_launch(s, what));
        }
        const Operand d{f.d, f.piece};
        if (dx) {
            const bool last = p + 1 == f.pieces;
            EpiOut o = last ? epilogue(dx, lddx, dtype, batch, inputs) : epilogue(f.dx, inputs, DNB_F32, batch, inputs);
            if (p > 0) add_to(o, f.dx, inputs, DNB_F32);
            else if (add_x) add_to(o, dx, lddx, dtype);
            o.alpha = scale / kDeltaScale;
            o.row_factor = row_scales;
            o.rows = f.rows;
            o.m_dev = f.count;
            const dnb_status sx = product(false, true, d, wq, dtype, rows, inputs, n, o, ds, s, what, f.count);
            DNB_TRY(sx);
        }
        if (weight_updates) {
            char *out = static_cast<char *>(weight_updates) + c0 * lddw * dtype_size(updates_dtype);
            EpiOut o = epilogue(out, lddw, updates_dtype, n, inputs);
            if (add_w) add_to(o, out, lddw, updates_dtype);
            o.alpha = scale / kDeltaScale;
            if (row_scales) {
                o.alpha = 1.0f;
                o.alpha_dev = f.meta + 1;
            }
            const dnb_status sw = product(true, true, d, xs, dtype, n, inputs, rows, o, ds, s, what, nullptr, f.count);
            DNB_TRY(sw);
        }
    }
    return DNB_OK;
}

}  // extern "C"
