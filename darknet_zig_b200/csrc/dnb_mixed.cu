// SGD with momentum and decay on fp32 weights, 16-bit gradients in and a 16-bit copy of the weights
// out: convolutional.zig:330-334's update (dnb_sgd_momentum) with the gradient's addition before it and
// the rounding to the products' type after it, so that a mixed-precision step reads and writes every
// weight once.
//
//   wu += g;  wu = fma(-decay*batch, w, wu);  w = fma(lr/batch, wu, w);  wu *= momentum;  w16 = rn(w)
//
// Bound by memory: 20 bytes an element (g 2, w and wu read and written 16, w16 2), one pass. A thread
// takes 8 elements with 16-byte accesses (two float4 of w and of wu, one vector of g and of w16), the
// widest all four tensors share; rows that cannot (an odd number of columns puts the fp32 rows off their
// boundaries) take single elements, four in flight a thread. A 64M-element vector in bf16: 225 us, 5.96 TB/s.
#include "dnb_types.cuh"

namespace dnb {
namespace {

constexpr int kThreads = 256;

template <class T>
struct SgdArgs {
    float *w, *wu;
    const T *g;
    T *w16;
    int64_t rows, cols, ldg, ld16;
    FastDiv per_row;  // vectors (or elements) of a row; used while their total is below 2^32
    bool flat;        // the 16-bit rows follow one another: no row arithmetic
    float a_decay, a_lr, mom;
};

__device__ __forceinline__ void sgd_one(float &w, float &wu, float g, float a_decay, float a_lr, float mom) {
    wu = wu + g;
    wu = __fmaf_rn(a_decay, w, wu);
    w = __fmaf_rn(a_lr, wu, w);
    wu = wu * mom;
}

// Row and offset of item i when a row has `n` of them.
template <class T>
__device__ __forceinline__ void row_of(const SgdArgs<T> &a, int64_t i, int64_t n, int64_t total, int64_t &r,
                                       int64_t &c) {
    if (a.flat) {
        r = 0;
        c = i;
    } else if (total <= 0xffffffffll) {
        uint32_t q, m;
        a.per_row.divmod((uint32_t)i, q, m);
        r = q;
        c = m;
    } else {
        r = i / n;
        c = i - r * n;
    }
}

template <class T>
__global__ void __launch_bounds__(kThreads) k_sgd_mixed_vec(SgdArgs<T> a) {
    using V = Vec<T, 16>;
    const int64_t n = a.cols / 8, total = a.rows * n;
    for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < total; i += (int64_t)gridDim.x * kThreads) {
        int64_t r, c;
        row_of(a, i, n, total, r, c);
        float4 w0 = ld4(a.w + 8 * i), w1 = ld4(a.w + 8 * i + 4);
        float4 u0 = ld4(a.wu + 8 * i), u1 = ld4(a.wu + 8 * i + 4);
        float g[8] = {};
        if (a.g) V::unpack(*reinterpret_cast<const uint4 *>(a.g + r * a.ldg + 8 * c), g);
        float w[8] = {w0.x, w0.y, w0.z, w0.w, w1.x, w1.y, w1.z, w1.w};
        float u[8] = {u0.x, u0.y, u0.z, u0.w, u1.x, u1.y, u1.z, u1.w};
#pragma unroll
        for (int j = 0; j < 8; ++j) sgd_one(w[j], u[j], g[j], a.a_decay, a.a_lr, a.mom);
        st4(a.w + 8 * i, make_float4(w[0], w[1], w[2], w[3]));
        st4(a.w + 8 * i + 4, make_float4(w[4], w[5], w[6], w[7]));
        st4(a.wu + 8 * i, make_float4(u[0], u[1], u[2], u[3]));
        st4(a.wu + 8 * i + 4, make_float4(u[4], u[5], u[6], u[7]));
        *reinterpret_cast<uint4 *>(a.w16 + r * a.ld16 + 8 * c) = V::pack(w);
    }
}

template <class T>
__global__ void __launch_bounds__(kThreads) k_sgd_mixed(SgdArgs<T> a) {
    const int64_t total = a.rows * a.cols;
    for (int64_t base = (int64_t)blockIdx.x * (4 * kThreads) + threadIdx.x; base < total;
         base += (int64_t)gridDim.x * (4 * kThreads)) {
        float w[4], u[4], g[4];
        int64_t at16[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int64_t i = base + j * kThreads;
            w[j] = u[j] = g[j] = 0.0f;
            if (i >= total) continue;
            int64_t r, c;
            row_of(a, i, a.cols, total, r, c);
            w[j] = a.w[i];
            u[j] = a.wu[i];
            if (a.g) g[j] = Elem<T>::to(a.g[r * a.ldg + c]);
            at16[j] = r * a.ld16 + c;
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int64_t i = base + j * kThreads;
            if (i >= total) continue;
            sgd_one(w[j], u[j], g[j], a.a_decay, a.a_lr, a.mom);
            a.w[i] = w[j];
            a.wu[i] = u[j];
            a.w16[at16[j]] = Elem<T>::from(w[j]);
        }
    }
}

}  // namespace
}  // namespace dnb

using namespace dnb;

extern "C" {

dnb_status dnb_sgd_momentum_mixed(int64_t rows, int64_t cols, float *weights, float *weight_updates,
                                  const void *gradients, int64_t ldg, void *weights16, int64_t ld16, int dtype,
                                  float learning_rate, float momentum, float decay, int64_t batch,
                                  dnb_stream stream) {
    const char *what = "sgd_momentum_mixed";
    if (rows < 0 || cols < 0) return fail(DNB_ERR_INVALID, "%s: negative size", what);
    if (!valid_dtype16(dtype)) return fail(DNB_ERR_INVALID, "%s: dtype must be bf16 or f16", what);
    if (batch <= 0) return fail(DNB_ERR_INVALID, "%s: batch must be positive", what);
    if (rows == 0 || cols == 0) return DNB_OK;
    if (!weights || !weight_updates || !weights16) return fail(DNB_ERR_INVALID, "%s: null pointer", what);
    if (!matrix_ok(weights, rows, cols, cols, DNB_F32) || !matrix_ok(weight_updates, rows, cols, cols, DNB_F32) ||
        !matrix_ok(weights16, rows, cols, ld16, dtype) || (gradients && !matrix_ok(gradients, rows, cols, ldg, dtype)))
        return fail(DNB_ERR_INVALID, "%s: a row stride is shorter than its row, too large, or a pointer is misaligned",
                    what);
    const int64_t n4 = rows * cols * 4, s16 = matrix_span(rows, cols, ld16, 2);
    const int64_t sg = gradients ? matrix_span(rows, cols, ldg, 2) : 0;
    const bool same = gradients == weights16 && ldg == ld16;
    if (overlaps(weights, n4, weight_updates, n4) || overlaps(weights, n4, weights16, s16) ||
        overlaps(weight_updates, n4, weights16, s16) || overlaps(gradients, sg, weights, n4) ||
        overlaps(gradients, sg, weight_updates, n4) || (!same && overlaps(gradients, sg, weights16, s16)))
        return fail(DNB_ERR_INVALID, "%s: overlapping tensors", what);
    DeviceState *ds = nullptr;
    DNB_TRY(current_device(&ds));
    const cudaStream_t s = as_stream(stream);
    const float b = (float)batch;  // convolutional.zig:219
    return dispatch_dtype16(dtype, [&]<class T>() {
        SgdArgs<T> a;
        a.w = weights;
        a.wu = weight_updates;
        a.g = static_cast<const T *>(gradients);
        a.w16 = static_cast<T *>(weights16);
        a.rows = rows;
        a.cols = cols;
        a.ldg = gradients ? ldg : cols;
        a.ld16 = ld16;
        a.a_decay = -decay * b;
        a.a_lr = learning_rate / b;
        a.mom = momentum;
        a.flat = (rows == 1 || (a.ldg == cols && ld16 == cols));
        const bool base = aligned16(weights) && aligned16(weight_updates) && aligned16(weights16) &&
                          (!gradients || aligned16(gradients));
        if (a.flat) {  // one long row; its last columns % 8 elements go by themselves
            const int64_t n = rows * cols, head = base ? n / 8 * 8 : 0;
            a.rows = 1;
            if (head) {
                a.cols = head;
                k_sgd_mixed_vec<T><<<grid_for(head / 8, kThreads, ds), kThreads, 0, s>>>(a);
                DNB_TRY(after_launch(s, what));
            }
            if (head < n) {
                a.cols = n - head;
                a.w += head;
                a.wu += head;
                if (a.g) a.g += head;
                a.w16 += head;
                k_sgd_mixed<T><<<grid_for((n - head + 3) / 4, kThreads, ds), kThreads, 0, s>>>(a);
                DNB_TRY(after_launch(s, what));
            }
            return (dnb_status)DNB_OK;
        }
        const bool vec = base && cols % 8 == 0 && ld16 % 8 == 0 && a.ldg % 8 == 0;
        const int64_t per = vec ? cols / 8 : cols;
        if (per <= 0x7fffffffll) a.per_row = FastDiv((uint32_t)per);
        if (vec)
            k_sgd_mixed_vec<T><<<grid_for(rows * per, kThreads, ds), kThreads, 0, s>>>(a);
        else
            k_sgd_mixed<T><<<grid_for((rows * per + 3) / 4, kThreads, ds), kThreads, 0, s>>>(a);
        return after_launch(s, what);
    });
}

}  // extern "C"
