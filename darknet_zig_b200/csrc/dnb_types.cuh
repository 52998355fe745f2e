// Element types of the 16-bit entries: conversions, packed vectors of 16, 4 or one element's
// bytes, and the host-side checks they share. Every 16-bit value is widened to fp32 exactly and
// every result is rounded to nearest even once.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "dnb_common.cuh"

namespace dnb {

inline bool valid_dtype(int t) { return t == DNB_F32 || t == DNB_BF16 || t == DNB_F16; }
inline bool valid_dtype16(int t) { return t == DNB_BF16 || t == DNB_F16; }
inline int64_t dtype_size(int t) { return t == DNB_F32 ? 4 : 2; }

// A matrix argument: `rows` rows of `cols` elements, `ld` elements apart. True if its size fits the
// kernels' 63-bit byte arithmetic and its pointer is aligned to the element.
inline bool matrix_ok(const void *p, int64_t rows, int64_t cols, int64_t ld, int dtype) {
    const int64_t e = dtype_size(dtype);
    if (reinterpret_cast<uintptr_t>(p) % (uintptr_t)e) return false;
    if (rows <= 1) return rows <= 0 || (ld >= cols && cols <= (int64_t(1) << 60) / e);
    return ld >= cols && ld <= (int64_t(1) << 60) / e / rows;
}
// Bytes from the matrix's first element to its last.
inline int64_t matrix_span(int64_t rows, int64_t cols, int64_t ld, int64_t e) {
    return rows <= 0 || cols <= 0 ? 0 : ((rows - 1) * ld + cols) * e;
}
inline bool overlaps(const void *a, int64_t an, const void *b, int64_t bn) {
    if (!a || !b || an <= 0 || bn <= 0) return false;
    const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
    return x < y + (uintptr_t)bn && y < x + (uintptr_t)an;
}

template <class T>
struct Elem;
template <>
struct Elem<float> {
    static __device__ __forceinline__ float to(float v) { return v; }
    static __device__ __forceinline__ float from(float v) { return v; }
};
template <>
struct Elem<__nv_bfloat16> {
    static __device__ __forceinline__ float to(__nv_bfloat16 v) { return __bfloat162float(v); }
    static __device__ __forceinline__ __nv_bfloat16 from(float v) { return __float2bfloat16_rn(v); }
};
template <>
struct Elem<__half> {
    static __device__ __forceinline__ float to(__half v) { return __half2float(v); }
    static __device__ __forceinline__ __half from(float v) { return __float2half_rn(v); }
};

// VB bytes of elements moved by one access.
template <int VB>
struct RawVec;
template <>
struct RawVec<16> { using type = uint4; };
template <>
struct RawVec<8> { using type = uint2; };
template <>
struct RawVec<4> { using type = uint32_t; };
template <>
struct RawVec<2> { using type = uint16_t; };

template <class T, int VB>
struct Vec {
    static constexpr int N = VB / (int)sizeof(T);
    using Raw = typename RawVec<VB>::type;
    union U {
        Raw raw;
        T e[N];
        __device__ U() {}
    };
    static __device__ __forceinline__ void unpack(const Raw &r, float (&f)[N]) {
        U u;
        u.raw = r;
#pragma unroll
        for (int i = 0; i < N; ++i) f[i] = Elem<T>::to(u.e[i]);
    }
    static __device__ __forceinline__ Raw pack(const float (&f)[N]) {
        U u;
#pragma unroll
        for (int i = 0; i < N; ++i) u.e[i] = Elem<T>::from(f[i]);
        return u.raw;
    }
};

// The same vector as pairs of floats, for the two-wide fp32 instructions (add, multiply and fused
// multiply-add of a pair in one issue). A single element is a pair whose second half is 0.
template <class T, int VB>
struct Pairs {
    static constexpr int N = VB / (int)sizeof(T), P = (N + 1) / 2;
    using Raw = typename RawVec<VB>::type;
    // by value: a reference would be read word by word from where it points to
    static __device__ __forceinline__ void unpack(Raw raw, float2 (&f)[P]) {
        if constexpr (N == 1) {
            float v[1];
            Vec<T, VB>::unpack(raw, v);
            f[0] = make_float2(v[0], 0.0f);
        } else if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int i = 0; i < P; ++i)
                f[i] = make_float2(__uint_as_float(word_of(raw, 2 * i)), __uint_as_float(word_of(raw, 2 * i + 1)));
        } else {
#pragma unroll
            for (int i = 0; i < P; ++i) f[i] = pair(word_of(raw, i), static_cast<T *>(nullptr));
        }
    }
    static __device__ __forceinline__ Raw pack(const float2 (&f)[P]) {
        float v[N];
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = i & 1 ? f[i / 2].y : f[i / 2].x;
        if constexpr (N == 1 || sizeof(T) == 4) {
            return Vec<T, VB>::pack(v);
        } else {
            uint32_t w[P];
#pragma unroll
            for (int i = 0; i < P; ++i) w[i] = word(f[i], static_cast<T *>(nullptr));
            if constexpr (P == 4) return make_uint4(w[0], w[1], w[2], w[3]);
            else if constexpr (P == 2) return make_uint2(w[0], w[1]);
            else return w[0];
        }
    }
    static __device__ __forceinline__ uint32_t word_of(uint4 r, int i) {
        return i == 0 ? r.x : i == 1 ? r.y : i == 2 ? r.z : r.w;
    }
    static __device__ __forceinline__ uint32_t word_of(uint2 r, int i) { return i == 0 ? r.x : r.y; }
    static __device__ __forceinline__ uint32_t word_of(uint32_t r, int) { return r; }
    static __device__ __forceinline__ uint32_t word_of(uint16_t r, int) { return r; }
    static __device__ __forceinline__ float2 pair(uint32_t w, __nv_bfloat16 *) {
        return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
    }
    static __device__ __forceinline__ float2 pair(uint32_t w, __half *) {
        return __half22float2(*reinterpret_cast<const __half2 *>(&w));
    }
    static __device__ __forceinline__ float2 pair(uint32_t, float *) { return make_float2(0.0f, 0.0f); }
    static __device__ __forceinline__ uint32_t word(float2 f, __nv_bfloat16 *) {
        const __nv_bfloat162 h = __float22bfloat162_rn(f);
        return *reinterpret_cast<const uint32_t *>(&h);
    }
    static __device__ __forceinline__ uint32_t word(float2 f, __half *) {
        const __half2 h = __float22half2_rn(f);
        return *reinterpret_cast<const uint32_t *>(&h);
    }
    static __device__ __forceinline__ uint32_t word(float2, float *) { return 0u; }
};
__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }
__device__ __forceinline__ float2 neg(float2 v) { return make_float2(-v.x, -v.y); }

// The special-function unit's exponential and reciprocal, subnormals flushed (no scaling around them).
__device__ __forceinline__ float quick_exp(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x * 1.4426950408889634f));
    return y;
}
__device__ __forceinline__ float quick_rcp(float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// An activation of the 16-bit entries: the fp32 entries' (dnb_common.cuh), but for the logistic, whose
// exponential and reciprocal are the special-function unit's (2 ulp each; a division and an exponential to
// the last bit cost a third of a group norm's time and vanish in the rounding to 16 bits).
template <int A>
__device__ __forceinline__ float act_quick(float x, int a) {
    if constexpr (A == DNB_ACT_LOGISTIC) return quick_rcp(1.0f + quick_exp(-x));
    else return act_fwd<A>(x, a);
}
template <int A>
__device__ __forceinline__ float2 act_pair(float2 x, int a) {
    if constexpr (A == DNB_ACT_LEAKY) {  // the larger of x and 0.1 x (fmaxf of two NaNs is NaN)
        const float2 t = __fmul2_rn(x, both(0.1f));
        return make_float2(fmaxf(x.x, t.x), fmaxf(x.y, t.y));
    }
    return make_float2(act_quick<A>(x.x, a), act_quick<A>(x.y, a));
}

// Calls f.template operator()<T>() with the element type.
template <class F>
auto dispatch_dtype(int dtype, F &&f) {
    switch (dtype) {
    case DNB_BF16: return f.template operator()<__nv_bfloat16>();
    case DNB_F16: return f.template operator()<__half>();
    default: return f.template operator()<float>();
    }
}
template <class F>
auto dispatch_dtype16(int dtype, F &&f) {
    if (dtype == DNB_BF16) return f.template operator()<__nv_bfloat16>();
    return f.template operator()<__half>();
}

}  // namespace dnb
