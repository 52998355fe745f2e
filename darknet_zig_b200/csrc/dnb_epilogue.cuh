// The epilogue of a product whose result is stored: scale, bias, addition, activation, one rounding.
#pragma once

#include "dnb_gemm.cuh"

namespace dnb {

// out = act(alpha * acc + bias[n] + add[m][n]), out and add of out_type (add may be out). A thread holds 32
// columns of a row: 64 contiguous bytes of 16-bit output, 128 of fp32, so its accesses fill whole sectors.
struct EpiOut {
    void *out = nullptr;
    int64_t ld = 0;
    int out_type = DNB_BF16;
    const void *add = nullptr;
    int64_t ld_add = 0;
    const float *bias = nullptr;
    const float *alpha = nullptr;  // device scalar; NULL = 1
    int act = DNB_ACT_LINEAR;
    int64_t m = 0, n = 0;
    bool vec_out = false, vec_add = false;  // rows start on 16-byte boundaries

    struct State {};
    __device__ __forceinline__ void begin(State &, int64_t, int64_t) const {}
    __device__ __forceinline__ void end(State &, int64_t, int64_t) const {}

    template <class T>
    __device__ __forceinline__ void load_add(float (&v)[32], int64_t row, int64_t col, int cols) const {
        const T *p = static_cast<const T *>(add) + row * ld_add + col;
        constexpr int N = 16 / (int)sizeof(T);
        if (vec_add && cols == 32) {
#pragma unroll
            for (int j = 0; j < 32; j += N) {
                float f[N];
                Vec<T, 16>::unpack(*reinterpret_cast<const uint4 *>(p + j), f);
#pragma unroll
                for (int i = 0; i < N; ++i) v[j + i] += f[i];
            }
        } else {
#pragma unroll
            for (int j = 0; j < 32; ++j)
                if (j < cols) v[j] += Elem<T>::to(p[j]);
        }
    }
    template <class T>
    __device__ __forceinline__ void store(const float (&v)[32], int64_t row, int64_t col, int cols) const {
        T *p = static_cast<T *>(out) + row * ld + col;
        constexpr int N = 16 / (int)sizeof(T);
        if (vec_out && cols == 32) {
#pragma unroll
            for (int j = 0; j < 32; j += N) {
                float f[N];
#pragma unroll
                for (int i = 0; i < N; ++i) f[i] = v[j + i];
                *reinterpret_cast<uint4 *>(p + j) = Vec<T, 16>::pack(f);
            }
        } else {
#pragma unroll
            for (int j = 0; j < 32; ++j)
                if (j < cols) p[j] = Elem<T>::from(v[j]);
        }
    }
    __device__ __forceinline__ void columns(State &, float (&v)[32], int64_t row, int64_t col) const {
        if (row >= m) return;
        const int cols = (int)(n - col < 32 ? n - col : 32);
        if (alpha) {
            const float a = *alpha;
#pragma unroll
            for (int j = 0; j < 32; ++j) v[j] *= a;
        }
        if (bias) {
#pragma unroll
            for (int j = 0; j < 32; ++j)
                if (j < cols) v[j] += __ldg(bias + col + j);
        }
        if (add) {
            if (out_type == DNB_F32) load_add<float>(v, row, col, cols);
            else if (out_type == DNB_BF16) load_add<__nv_bfloat16>(v, row, col, cols);
            else load_add<__half>(v, row, col, cols);
        }
        switch (act) {
        case DNB_ACT_LINEAR: break;
        case DNB_ACT_LEAKY:
#pragma unroll
            for (int j = 0; j < 32; ++j) v[j] = act_fwd<DNB_ACT_LEAKY>(v[j], act);
            break;
        case DNB_ACT_RELU:
#pragma unroll
            for (int j = 0; j < 32; ++j) v[j] = act_fwd<DNB_ACT_RELU>(v[j], act);
            break;
        case DNB_ACT_LOGISTIC:
#pragma unroll
            for (int j = 0; j < 32; ++j) v[j] = act_fwd<DNB_ACT_LOGISTIC>(v[j], act);
            break;
        default: activate_any(v, act);
        }
        if (out_type == DNB_F32) store<float>(v, row, col, cols);
        else if (out_type == DNB_BF16) store<__nv_bfloat16>(v, row, col, cols);
        else store<__half>(v, row, col, cols);
    }
    static __device__ __noinline__ float activate_one(float v, int a) { return act_fwd_any(v, a); }
    static __device__ __forceinline__ void activate_any(float (&v)[32], int a) {
#pragma unroll
        for (int j = 0; j < 32; ++j) v[j] = activate_one(v[j], a);
    }
};

}  // namespace dnb
