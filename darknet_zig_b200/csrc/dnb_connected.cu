// The connected layer on 16-bit tensors: product, bias, residual and activation in one kernel
// (connected.zig:92-119 with misc.zig:244-270 and the activation after them), and its backward
// (connected.zig:121-138).
//
//   forward   y = act(x w^T + b + r)                       x, w K-major
//   backward  dz = delta act'(y); dx = dz w; dW = dz^T x   dz K-major with w MN-major, then both MN-major
//
// A few rows (a token's decode step) are bound by reading w: k_rows gives a warp an output and the lanes
// slices of its row of w, with no tensor core. Everything else runs on k_gemm (dnb_gemm.cuh).
#include "dnb_epilogue.cuh"
#include "dnb_pack.cuh"

namespace dnb {
namespace {

// ---- few rows ----

struct RowsArgs {
    const void *x, *w, *add;
    void *y;
    const float *bias;
    int64_t ldx, ldw, ld_add, ldy, m, n, k;
    int act, out_type;
};

// MB rows of x at a time; a block of 8 warps, WPR of them share an output and split its k. A lane has U vectors of
// w (and as many of x, which the L1 cache holds) on their way before it needs the first.
template <class T, int VB, int MB>
__global__ void __launch_bounds__(256) k_rows(const __grid_constant__ RowsArgs a, int wpr) {
    using V = Pairs<T, VB>;
    using Raw = typename V::Raw;
    constexpr int N = V::N, P = V::P, U = 4;
    __shared__ float red[8][MB];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, outs = 8 / wpr;
    const int64_t row = (int64_t)blockIdx.x * outs + warp / wpr;
    const int part = warp % wpr;
    const int64_t m0 = (int64_t)blockIdx.y * MB;
    const T *x = static_cast<const T *>(a.x) + m0 * a.ldx, *w = static_cast<const T *>(a.w) + row * a.ldw;
    const int rows = (int)(a.m - m0 < MB ? a.m - m0 : MB);
    float2 acc[MB] = {};
    if (row < a.n) {
        const int64_t vecs = a.k / N;
        const int step = wpr * 32;
        int64_t i = part * 32 + lane;
        auto take = [&](Raw rw, int64_t at) {
            float2 fw[P];
            V::unpack(rw, fw);
#pragma unroll
            for (int b = 0; b < MB; ++b) {
                if (b >= rows) break;
                float2 fx[P];
                V::unpack(__ldg(reinterpret_cast<const Raw *>(x + b * a.ldx + at * N)), fx);
#pragma unroll
                for (int j = 0; j < P; ++j) acc[b] = __ffma2_rn(fx[j], fw[j], acc[b]);
            }
        };
        for (; i + (U - 1) * step < vecs; i += U * step) {
            Raw rw[U];
#pragma unroll
            for (int u = 0; u < U; ++u) rw[u] = __ldcs(reinterpret_cast<const Raw *>(w + (i + u * step) * N));
#pragma unroll
            for (int u = 0; u < U; ++u) take(rw[u], i + u * step);
        }
        for (; i < vecs; i += step) take(__ldcs(reinterpret_cast<const Raw *>(w + i * N)), i);
        // the last k % N elements
        const int64_t last = vecs * N + lane;
        if (part == 0 && last < a.k)
#pragma unroll
            for (int b = 0; b < MB; ++b)
                if (b < rows) acc[b].x = __fmaf_rn(Elem<T>::to(x[b * a.ldx + last]), Elem<T>::to(w[last]), acc[b].x);
    }
#pragma unroll
    for (int b = 0; b < MB; ++b) {
        const float s = warp_sum(acc[b].x + acc[b].y);
        if (lane == 0) red[warp][b] = s;
    }
    __syncthreads();
    // a thread per (output, row): the parts added in order
    for (int t = threadIdx.x; t < outs * MB; t += 256) {
        const int o = t / MB, b = t % MB;
        const int64_t n = (int64_t)blockIdx.x * outs + o, m = m0 + b;
        if (n >= a.n || m >= a.m) continue;
        float v = 0.0f;
        for (int p = 0; p < wpr; ++p) v += red[o * wpr + p][b];
        if (a.bias) v += a.bias[n];
        if (a.add) v += Elem<T>::to(static_cast<const T *>(a.add)[m * a.ld_add + n]);
        static_cast<T *>(a.y)[m * a.ldy + n] = Elem<T>::from(act_fwd_any(v, a.act));
    }
}

template <class T, int VB>
dnb_status run_rows(const RowsArgs &a, cudaStream_t s, const char *what) {
    // a warp an output from 4096 of them on; fewer are shared by more warps, while a lane keeps two vectors.
    // [1,4096]x[4096,4096]^T: 1, 2 and 4 warps an output 5.9, 7.2 and 9.1 us; [1,4096]x[1000,4096]^T: 5.0, 3.8, 3.4
    int wpr = 1;
    while (wpr < 8 && a.n * wpr * 2 <= 4096 && a.k >= 512 * wpr) wpr *= 2;
    const int64_t outs = 8 / wpr, blocks = (a.n + outs - 1) / outs;
    if (blocks > 0x7fffffffll) return fail(DNB_ERR_UNSUPPORTED, "%s: too many outputs", what);
    if (a.m == 1) k_rows<T, VB, 1><<<dim3((unsigned)blocks, 1), 256, 0, s>>>(a, wpr);
    else k_rows<T, VB, 2><<<dim3((unsigned)blocks, (unsigned)((a.m + 1) / 2)), 256, 0, s>>>(a, wpr);
    return after_launch(s, what);
}

// ---- backward: delta through the activation ----

struct DzArgs {
    const void *y, *delta;
    void *dz, *copy;  // the caller's dz (NULL: linear) and an aligned copy for the products (NULL: none)
    float *part;      // [row chunks][n] column sums (NULL: no bias updates)
    int64_t ldy, ldd, lddz, ld_copy, m, n;
    int act, rows;    // rows of a chunk
};

// A block takes kDzRows rows of 64 vectors of columns: 4 row lanes, each with four rows on their way at a time
// (dz may be delta, so that nothing is hoisted past a store by itself). Bound by memory: [8192,4096] bf16 with
// an output, 201 MB, 50 us with one row lane of 256 vectors and 33 us so.
template <class T, int VB, int A>
__global__ void __launch_bounds__(256) k_dz(const __grid_constant__ DzArgs a) {
    using V = Pairs<T, VB>;
    using Raw = typename V::Raw;
    constexpr int N = V::N, P = V::P, U = 4;
    __shared__ float part[4][64 * N];
    const int tx = threadIdx.x & 63, ty = threadIdx.x >> 6;
    const int64_t c = ((int64_t)blockIdx.x * 64 + tx) * N;
    const int64_t r0 = (int64_t)blockIdx.y * a.rows, r1 = r0 + a.rows < a.m ? r0 + a.rows : a.m;
    float2 sum[P] = {};
    if (c < a.n) {
        const T *delta = static_cast<const T *>(a.delta) + c, *y = static_cast<const T *>(a.y) + c;
        T *dz = static_cast<T *>(a.dz), *copy = static_cast<T *>(a.copy);
        for (int64_t r = r0 + ty; r < r1; r += 4 * U) {
            Raw rd[U] = {}, ry[U] = {};
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (r + 4 * u >= r1) break;
                rd[u] = *reinterpret_cast<const Raw *>(delta + (r + 4 * u) * a.ldd);
                if constexpr (A != DNB_ACT_LINEAR) ry[u] = *reinterpret_cast<const Raw *>(y + (r + 4 * u) * a.ldy);
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (r + 4 * u >= r1) break;
                float2 d[P];
                V::unpack(rd[u], d);
                if constexpr (A != DNB_ACT_LINEAR) {
                    float2 f[P];
                    V::unpack(ry[u], f);
#pragma unroll
                    for (int i = 0; i < P; ++i)
                        d[i] = __fmul2_rn(d[i], make_float2(act_grad<A>(f[i].x, a.act), act_grad<A>(f[i].y, a.act)));
                }
                const Raw raw = V::pack(d);
                if (dz) *reinterpret_cast<Raw *>(dz + (r + 4 * u) * a.lddz + c) = raw;
                if (copy) *reinterpret_cast<Raw *>(copy + (r + 4 * u) * a.ld_copy + c) = raw;
#pragma unroll
                for (int i = 0; i < P; ++i) sum[i] = __fadd2_rn(sum[i], d[i]);
            }
        }
    }
    if (!a.part) return;
#pragma unroll
    for (int j = 0; j < N; ++j) part[ty][tx * N + j] = j & 1 ? sum[j / 2].y : sum[j / 2].x;
    __syncthreads();
    for (int i = threadIdx.x; i < 64 * N; i += 256) {
        const int64_t col = (int64_t)blockIdx.x * (64 * N) + i;
        if (col < a.n) a.part[(int64_t)blockIdx.y * a.n + col] = part[0][i] + part[1][i] + part[2][i] + part[3][i];
    }
}

constexpr int kDzRows = 64;

// Rows up to which k_rows is used: [1 | 2 | 4,4096]x[4096,4096]^T 5.9, 7.7, 13.6 us; k_gemm takes 8.2 for all three.
constexpr int64_t kFewRows = 2;

struct FwdSpace {
    void *x, *w;
    size_t total;
};
FwdSpace fwd_space(void *ws, const void *x, int64_t ldx, const void *w, int64_t ldw, int64_t m, int64_t k, int64_t n) {
    Carver c(ws);
    FwdSpace f{};
    if (m > kFewRows && k > 0) {
        if (!tma_ready(x, m > 1 ? ldx : 8)) f.x = c.take(packed_bytes(m, k));
        if (!tma_ready(w, n > 1 ? ldw : 8)) f.w = c.take(packed_bytes(n, k));
    }
    f.total = c.used;
    return f;
}

struct BwdSpace {
    void *x, *w, *dz;
    float *part;
    size_t total;
};
BwdSpace bwd_space(void *ws, const void *x, int64_t ldx, const void *w, int64_t ldw, const void *dz, int64_t lddz,
                   int64_t m, int64_t k, int64_t n) {
    Carver c(ws);
    BwdSpace b{};
    if (!tma_ready(x, m > 1 ? ldx : 8)) b.x = c.take(packed_bytes(m, k));
    if (!tma_ready(w, n > 1 ? ldw : 8)) b.w = c.take(packed_bytes(n, k));
    if (!tma_ready(dz, m > 1 ? lddz : 8)) b.dz = c.take(packed_bytes(m, n));
    b.part = static_cast<float *>(c.take((m + kDzRows - 1) / kDzRows * n * 4));
    b.total = c.used;
    return b;
}

}  // namespace
}  // namespace dnb

using namespace dnb;

extern "C" {

dnb_status dnb_connected_act_forward_workspace(const void *x, int64_t ldx, const void *w, int64_t ldw, int dtype,
                                               int64_t batch, int64_t inputs, int64_t outputs, size_t *bytes) {
    const char *what = "connected_act_forward_workspace";
    if (!bytes) return fail(DNB_ERR_INVALID, "%s: bytes is null", what);
    DNB_TRY(product_shape_check(dtype, batch, inputs, outputs, what));
    *bytes = fwd_space(nullptr, x, ldx, w, ldw, batch, inputs, outputs).total;
    return DNB_OK;
}

dnb_status dnb_connected_act_forward(const void *x, int64_t ldx, const void *w, int64_t ldw, const float *biases,
                                     const void *residual, int64_t ldr, void *y, int64_t ldy, int dtype,
                                     int64_t batch, int64_t inputs, int64_t outputs, int act, void *workspace,
                                     size_t workspace_bytes, dnb_stream stream) {
    const char *what = "connected_act_forward";
    DNB_TRY(product_shape_check(dtype, batch, inputs, outputs, what));
    if (!valid_act(act)) return fail(DNB_ERR_INVALID, "%s: unknown activation %d", what, act);
    if (batch == 0 || outputs == 0) return DNB_OK;
    if (!y || (inputs > 0 && (!x || !w))) return fail(DNB_ERR_INVALID, "%s: null pointer", what);
    if (!matrix_ok(x, batch, inputs, ldx, dtype) || !matrix_ok(w, outputs, inputs, ldw, dtype) ||
        !matrix_ok(y, batch, outputs, ldy, dtype) || (residual && !matrix_ok(residual, batch, outputs, ldr, dtype)) ||
        reinterpret_cast<uintptr_t>(biases) % 4)
        return fail(DNB_ERR_INVALID, "%s: a row stride is shorter than its row, too large, or a pointer is misaligned",
                    what);
    const int64_t sx = matrix_span(batch, inputs, ldx, 2), sw = matrix_span(outputs, inputs, ldw, 2);
    const int64_t sy = matrix_span(batch, outputs, ldy, 2), sr = residual ? matrix_span(batch, outputs, ldr, 2) : 0;
    if (overlaps(y, sy, x, sx) || overlaps(y, sy, w, sw) || overlaps(y, sy, biases, outputs * 4) ||
        (!(residual == y && (ldr == ldy || batch == 1)) && overlaps(y, sy, residual, sr)))
        return fail(DNB_ERR_INVALID, "%s: overlapping tensors", what);
    const FwdSpace f = fwd_space(workspace, x, ldx, w, ldw, batch, inputs, outputs);
    DNB_TRY(workspace_check(workspace, workspace_bytes, f.total, what));
    DeviceState *ds = nullptr;
    DNB_TRY(current_device(&ds));
    const cudaStream_t s = as_stream(stream);
    if (batch <= kFewRows || inputs == 0) {
        RowsArgs a{x, w, residual, y, biases, ldx, ldw, ldr, ldy, batch, outputs, inputs, act, dtype};
        a.n = outputs;
        a.k = inputs;
        if (batch > 2 * 65535) return fail(DNB_ERR_UNSUPPORTED, "%s: too many rows without inputs", what);
        const uintptr_t al = reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(w) |
                             (batch > 1 ? (uintptr_t)ldx * 2 : 0) | (outputs > 1 ? (uintptr_t)ldw * 2 : 0);
        return dispatch_dtype16(dtype, [&]<class T>() {
            if (al % 16 == 0) return run_rows<T, 16>(a, s, what);
            if (al % 4 == 0) return run_rows<T, 4>(a, s, what);
            return run_rows<T, 2>(a, s, what);
        });
    }
    Operand a{x, ldx}, b{w, ldw};
    DNB_TRY(pack_rows({x, ldx, f.x, batch, inputs}, {w, ldw, f.w, outputs, inputs}, dtype, {}, ds, s, what));
    if (f.x) a = {f.x, packed_ld(inputs)};
    if (f.w) b = {f.w, packed_ld(inputs)};
    EpiOut e = epilogue(y, ldy, dtype, batch, outputs);
    e.bias = biases;
    e.act = act;
    if (residual) add_to(e, residual, ldr, dtype);
    return product(false, false, a, b, dtype, batch, outputs, inputs, e, ds, s, what);
}

dnb_status dnb_connected_act_backward_workspace(const void *x, int64_t ldx, const void *w, int64_t ldw,
                                                const void *delta, int64_t ldd, const void *dz, int64_t lddz,
                                                int dtype, int64_t batch, int64_t inputs, int64_t outputs, int act,
                                                size_t *bytes) {
    const char *what = "connected_act_backward_workspace";
    if (!bytes) return fail(DNB_ERR_INVALID, "%s: bytes is null", what);
    DNB_TRY(product_shape_check(dtype, batch, inputs, outputs, what));
    const bool linear = act == DNB_ACT_LINEAR;
    *bytes = bwd_space(nullptr, x, ldx, w, ldw, linear ? delta : dz, linear ? ldd : lddz, batch, inputs, outputs).total;
    return DNB_OK;
}

dnb_status dnb_connected_act_backward(const void *x, int64_t ldx, const void *w, int64_t ldw, const void *y,
                                      int64_t ldy, const void *delta, int64_t ldd, void *dz, int64_t lddz, void *dx,
                                      int64_t lddx, float *bias_updates, void *weight_updates, int64_t lddw,
                                      int updates_dtype, int dtype, int64_t batch, int64_t inputs, int64_t outputs,
                                      int act, int accumulate, void *workspace, size_t workspace_bytes,
                                      dnb_stream stream) {
    const char *what = "connected_act_backward";
    DNB_TRY(product_shape_check(dtype, batch, inputs, outputs, what));
    if (!valid_act(act)) return fail(DNB_ERR_INVALID, "%s: unknown activation %d", what, act);
    if (accumulate & ~(DNB_ACC_UPDATES | DNB_ACC_DELTA)) return fail(DNB_ERR_INVALID, "%s: unknown accumulate bits", what);
    if (weight_updates && updates_dtype != dtype && updates_dtype != DNB_F32)
        return fail(DNB_ERR_INVALID, "%s: updates_dtype must be dtype or f32", what);
    const bool linear = act == DNB_ACT_LINEAR;
    const int64_t mn = batch * outputs;
    if (mn > 0 && (!delta || (!linear && (!y || !dz)))) return fail(DNB_ERR_INVALID, "%s: null pointer", what);
    if (mn > 0 && inputs > 0 && ((dx && !w) || (weight_updates && !x)))
        return fail(DNB_ERR_INVALID, "%s: null pointer", what);
    if (!matrix_ok(x, batch, inputs, ldx, dtype) || !matrix_ok(w, outputs, inputs, ldw, dtype) ||
        !matrix_ok(delta, batch, outputs, ldd, dtype) ||
        (!linear && (!matrix_ok(y, batch, outputs, ldy, dtype) || !matrix_ok(dz, batch, outputs, lddz, dtype))) ||
        (dx && !matrix_ok(dx, batch, inputs, lddx, dtype)) ||
        (weight_updates && !matrix_ok(weight_updates, outputs, inputs, lddw, updates_dtype)) ||
        reinterpret_cast<uintptr_t>(bias_updates) % 4)
        return fail(DNB_ERR_INVALID, "%s: a row stride is shorter than its row, too large, or a pointer is misaligned",
                    what);
    struct Span {
        const void *p;
        int64_t n;
    };
    const Span in[4] = {{x, matrix_span(batch, inputs, ldx, 2)},
                        {w, matrix_span(outputs, inputs, ldw, 2)},
                        {linear ? nullptr : y, matrix_span(batch, outputs, ldy, 2)},
                        {delta, matrix_span(batch, outputs, ldd, 2)}};
    const Span out[4] = {{linear ? nullptr : dz, matrix_span(batch, outputs, lddz, 2)},
                         {dx, matrix_span(batch, inputs, lddx, 2)},
                         {weight_updates, matrix_span(outputs, inputs, lddw, dtype_size(updates_dtype))},
                         {bias_updates, outputs * 4}};
    const bool in_place = !linear && dz == delta && (lddz == ldd || batch == 1);
    for (int o = 0; o < 4; ++o) {
        for (int i = 0; i < 4; ++i)
            if (!(o == 0 && i == 3 && in_place) && overlaps(out[o].p, out[o].n, in[i].p, in[i].n))
                return fail(DNB_ERR_INVALID, "%s: overlapping tensors", what);
        for (int q = 0; q < o; ++q)
            if (overlaps(out[o].p, out[o].n, out[q].p, out[q].n))
                return fail(DNB_ERR_INVALID, "%s: overlapping tensors", what);
    }
    const BwdSpace f = bwd_space(workspace, x, ldx, w, ldw, linear ? delta : dz, linear ? ldd : lddz, batch, inputs,
                                 outputs);
    if (mn > 0) DNB_TRY(workspace_check(workspace, workspace_bytes, f.total, what));
    DeviceState *ds = nullptr;
    const cudaStream_t s = as_stream(stream);
    const bool add_w = accumulate & DNB_ACC_UPDATES, add_x = accumulate & DNB_ACC_DELTA;
    DNB_TRY(current_device(&ds));
    if (mn == 0 || inputs == 0) {  // products over nothing, or with nothing
        if (dx && batch > 0 && inputs > 0 && !add_x) DNB_TRY(zero_rows(dx, batch, inputs, lddx, 2, ds, s, what));
        if (weight_updates && outputs > 0 && inputs > 0 && !add_w)
            DNB_TRY(zero_rows(weight_updates, outputs, inputs, lddw, dtype_size(updates_dtype), ds, s, what));
        if (mn == 0) {
            if (bias_updates && outputs > 0 && !add_w) DNB_TRY(zero_rows(bias_updates, 1, outputs, outputs, 4, ds, s, what));
            return DNB_OK;
        }
    }
    if (!linear || bias_updates || f.dz) {
        DzArgs a{};
        a.y = y;
        a.delta = delta;
        a.dz = linear ? nullptr : dz;
        a.copy = f.dz;
        a.part = bias_updates ? f.part : nullptr;
        a.ldy = ldy;
        a.ldd = ldd;
        a.lddz = lddz;
        a.ld_copy = packed_ld(outputs);
        a.m = batch;
        a.n = outputs;
        a.act = act;
        a.rows = kDzRows;
        const int64_t chunks = (batch + kDzRows - 1) / kDzRows;
        if (chunks > 65535) return fail(DNB_ERR_UNSUPPORTED, "%s: more than 65535 * %d rows", what, kDzRows);
        uintptr_t al = reinterpret_cast<uintptr_t>(delta) | (uintptr_t)(ldd * 2) | (uintptr_t)(outputs * 2);
        if (!linear)
            al |= reinterpret_cast<uintptr_t>(y) | reinterpret_cast<uintptr_t>(dz) | (uintptr_t)(ldy * 2) |
                  (uintptr_t)(lddz * 2);
        const dnb_status st = dispatch_dtype16(dtype, [&]<class T>() {
            return dispatch_act(act, [&]<int A>() {
                const int n = al % 16 == 0 ? 8 : 1;
                const dim3 grid((unsigned)((outputs + 64 * n - 1) / (64 * n)), (unsigned)chunks);
                if (n == 8) k_dz<T, 16, A><<<grid, 256, 0, s>>>(a);
                else k_dz<T, 2, A><<<grid, 256, 0, s>>>(a);
                return after_launch(s, what);
            });
        });
        DNB_TRY(st);
        if (bias_updates) {
            DNB_TRY(column_sums(f.part, chunks, outputs, outputs, bias_updates, add_w, s, what));
        }
    }
    if (inputs == 0) return DNB_OK;
    Operand d{linear ? delta : dz, linear ? ldd : lddz};
    if (f.dz) d = {f.dz, packed_ld(outputs)};
    DNB_TRY(pack_rows({x, ldx, weight_updates ? f.x : nullptr, batch, inputs},
                      {w, ldw, dx ? f.w : nullptr, outputs, inputs}, dtype, {}, ds, s, what));
    if (dx) {
        Operand b{w, ldw};
        if (f.w) b = {f.w, packed_ld(inputs)};
        EpiOut e = epilogue(dx, lddx, dtype, batch, inputs);
        if (add_x) add_to(e, dx, lddx, dtype);
        const dnb_status st = product(false, true, d, b, dtype, batch, inputs, outputs, e, ds, s, what);
        DNB_TRY(st);
    }
    if (weight_updates) {
        Operand b{x, ldx};
        if (f.x) b = {f.x, packed_ld(inputs)};
        EpiOut e = epilogue(weight_updates, lddw, updates_dtype, outputs, inputs);
        if (add_w) add_to(e, weight_updates, lddw, updates_dtype);
        const dnb_status st = product(true, true, d, b, dtype, outputs, inputs, batch, e, ds, s, what);
        DNB_TRY(st);
    }
    return DNB_OK;
}

}  // extern "C"
