// The epilogue of a product whose result is stored: scale, bias, addition, activation, one rounding.
#pragma once

#include "dnb_gemm.cuh"

namespace dnb {

__device__ __forceinline__ void store32(uint4 *p, uint4 a, uint4 b) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(a.x), "r"(a.y), "r"(a.z),
                 "r"(a.w), "r"(b.x), "r"(b.y), "r"(b.z), "r"(b.w)
                 : "memory");
}
// A tile's biases from shared memory (the same address in every lane).
__device__ __forceinline__ void add_bias32(float2 (&v)[16], const float *bias) {
#pragma unroll
    for (int j = 0; j < 16; j += 2) {
        const float4 b = *reinterpret_cast<const float4 *>(bias + 2 * j);
        v[j] = __fadd2_rn(v[j], make_float2(b.x, b.y));
        v[j + 1] = __fadd2_rn(v[j + 1], make_float2(b.z, b.w));
    }
}
template <int A>
__device__ __forceinline__ void act32(float2 (&v)[16], int a) {
#pragma unroll
    for (int j = 0; j < 16; ++j) v[j] = act_pair<A>(v[j], a);
}

// out = act(f * acc + bias[n] + add[m][n]) (add may be out), f = alpha * *alpha_dev * row_factor[row].
// With a row map, row r of the product is row rows[r] of out, add and row_factor. A thread holds 32 columns
// of a row: 64 contiguous bytes of 16-bit output, 128 of fp32, so its accesses fill whole sectors.
struct EpiOut {
    void *out = nullptr;
    int64_t ld = 0;
    int out_type = DNB_BF16;
    int add_type = DNB_BF16;
    const void *add = nullptr;
    int64_t ld_add = 0;
    const float *bias = nullptr;
    float alpha = 1.0f;
    const float *alpha_dev = nullptr, *row_factor = nullptr;  // NULL = 1
    const int *rows = nullptr, *m_dev = nullptr;
    int act = DNB_ACT_LINEAR;
    int64_t m = 0, n = 0;
    bool vec_out = false, vec_add = false;  // rows start on 16-byte boundaries
    bool wide_out = false;                  // and out's on 32-byte ones: whole sectors a store
    bool early = false;                     // the addend is 16-bit and vec_add

    struct State {
        int64_t row;  // of out; -1: none
        float f;
    };
    __device__ __forceinline__ void begin(State &s, int64_t row, int64_t) const {
        s.row = -1;
        s.f = 1.0f;
        if (row >= (m_dev ? *m_dev : m)) return;
        s.row = rows ? rows[row] : row;
        s.f = alpha;
        if (alpha_dev) s.f *= *alpha_dev;
        if (row_factor) s.f *= row_factor[s.row];
    }
    __device__ __forceinline__ void end(State &, int64_t, int64_t) const {}

    // the addend of 32 columns, fetched early where it is 16-bit and aligned
    struct Ahead {
        uint4 a[4];
    };
    __device__ __forceinline__ void fetch(const State &s, Ahead &h, int64_t col) const {
        if (!early || s.row < 0 || col + 32 > n) return;
        const uint4 *p = reinterpret_cast<const uint4 *>(static_cast<const uint16_t *>(add) + s.row * ld_add + col);
#pragma unroll
        for (int i = 0; i < 4; ++i) h.a[i] = p[i];
    }

    template <class T>
    __device__ __forceinline__ void add_fetched(float2 (&v)[16], const Ahead &h) const {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            float2 f[4];
            Pairs<T, 16>::unpack(h.a[j], f);
#pragma unroll
            for (int i = 0; i < 4; ++i) v[4 * j + i] = __fadd2_rn(v[4 * j + i], f[i]);
        }
    }
    // The first n elements of a vector at the row's end.
    template <class T>
    static __device__ __forceinline__ uint4 some(const T *p, int n) {
        typename Vec<T, 16>::U u;
        u.raw = make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
        for (int i = 0; i < Vec<T, 16>::N; ++i)
            if (i < n) u.e[i] = p[i];
        return u.raw;
    }
    template <class T>
    __device__ __forceinline__ void load_add(float2 (&v)[16], int64_t row, int64_t col, int cols) const {
        const T *p = static_cast<const T *>(add) + row * ld_add + col;
        constexpr int N = 16 / (int)sizeof(T);
        uint4 raw[32 / N];
#pragma unroll
        for (int j = 0; j < 32 / N; ++j) {
            raw[j] = make_uint4(0u, 0u, 0u, 0u);
            if (j * N + N <= cols) raw[j] = reinterpret_cast<const uint4 *>(p)[j];
            else if (j * N < cols) raw[j] = some(p + j * N, cols - j * N);
        }
#pragma unroll
        for (int j = 0; j < 32 / N; ++j) {
            float2 f[N / 2];
            Pairs<T, 16>::unpack(raw[j], f);
#pragma unroll
            for (int i = 0; i < N / 2; ++i) v[j * N / 2 + i] = __fadd2_rn(v[j * N / 2 + i], f[i]);
        }
    }
    template <class T>
    __device__ __forceinline__ void store(const float2 (&v)[16], int64_t row, int64_t col, int cols) const {
        T *p = static_cast<T *>(out) + row * ld + col;
        constexpr int N = 16 / (int)sizeof(T);
        uint4 raw[32 / N];
#pragma unroll
        for (int j = 0; j < 32 / N; ++j) {
            float2 f[N / 2];
#pragma unroll
            for (int i = 0; i < N / 2; ++i) f[i] = v[j * N / 2 + i];
            raw[j] = Pairs<T, 16>::pack(f);
        }
        if (wide_out && cols == 32) {
#pragma unroll
            for (int j = 0; j < 32 / N; j += 2) store32(reinterpret_cast<uint4 *>(p) + j, raw[j], raw[j + 1]);
        } else {
#pragma unroll
            for (int j = 0; j < 32 / N; ++j) {
                if (j * N + N <= cols) {
                    reinterpret_cast<uint4 *>(p)[j] = raw[j];
                } else if (j * N < cols) {
                    typename Vec<T, 16>::U u;
                    u.raw = raw[j];
#pragma unroll
                    for (int i = 0; i < N; ++i)
                        if (j * N + i < cols) p[j * N + i] = u.e[i];
                }
            }
        }
    }
    __device__ __forceinline__ void activate(float2 (&v)[16]) const {
        switch (act) {
        case DNB_ACT_LINEAR: break;
        case DNB_ACT_LEAKY: act32<DNB_ACT_LEAKY>(v, act); break;
        case DNB_ACT_RELU: act32<DNB_ACT_RELU>(v, act); break;
        case DNB_ACT_LOGISTIC: act32<DNB_ACT_LOGISTIC>(v, act); break;
        default: activate_any(v, act);
        }
    }
    // The addend's elements of a column in the warp's 32 rows (row: lane i's is row i's index, or -1): all on their way
    // before the first is needed.
    template <class T>
    __device__ __forceinline__ void add_rows(float (&u)[32], int64_t row, int64_t col, bool in) const {
        const T *p = static_cast<const T *>(add) + col;
        T got[32];
#pragma unroll
        for (int i = 0; i < 32; ++i) {
            const int64_t at = __shfl_sync(0xffffffffu, row, i);
            got[i] = in && at >= 0 ? p[at * ld_add] : Elem<T>::from(0.0f);
        }
#pragma unroll
        for (int i = 0; i < 32; ++i) u[i] += Elem<T>::to(got[i]);
    }
    template <class T>
    __device__ __forceinline__ void store_rows(const float2 (&v)[16], int64_t row, int64_t col, bool in) const {
        T *p = static_cast<T *>(out) + col;
#pragma unroll
        for (int i = 0; i < 32; ++i) {
            const int64_t at = __shfl_sync(0xffffffffu, row, i);
            if (in && at >= 0) p[at * ld] = Elem<T>::from(i & 1 ? v[i / 2].y : v[i / 2].x);
        }
    }
    // Rows off the 16-byte boundaries: the warp turns its 32 x 32 values over, so that its lanes
    // hold neighbouring columns of a row, and reads and writes a row at a time. (A lane's own row element by element
    // touches 32 sectors an access: 157 us against 85 at a backward of [900,8183]x[316,8183].)
    __device__ __forceinline__ void ragged(int64_t row, float2 (&v)[16], int64_t col, int cols) const {
        const int lane = threadIdx.x & 31;
        float u[32];
#pragma unroll
        for (int j = 0; j < 16; ++j) {
            u[2 * j] = v[j].x;
            u[2 * j + 1] = v[j].y;
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            const bool up = lane & o;
#pragma unroll
            for (int j = 0; j < 32; ++j) {
                if (j & o) continue;
                const float got = __shfl_xor_sync(0xffffffffu, up ? u[j] : u[j + o], o);
                if (up) u[j] = got;
                else u[j + o] = got;
            }
        }
        // u[i]: row i of the warp's, column `lane`
        const bool in = lane < cols;
        if (add) {
            if (add_type == DNB_F32) add_rows<float>(u, row, col + lane, in);
            else if (add_type == DNB_BF16) add_rows<__nv_bfloat16>(u, row, col + lane, in);
            else add_rows<__half>(u, row, col + lane, in);
        }
#pragma unroll
        for (int j = 0; j < 16; ++j) v[j] = make_float2(u[2 * j], u[2 * j + 1]);
        activate(v);
        if (out_type == DNB_F32) store_rows<float>(v, row, col + lane, in);
        else if (out_type == DNB_BF16) store_rows<__nv_bfloat16>(v, row, col + lane, in);
        else store_rows<__half>(v, row, col + lane, in);
    }
    __device__ __forceinline__ void columns(State &s, float2 (&v)[16], const float *tile_bias, const Ahead &h, int64_t,
                                            int64_t col) const {
        const int cols = (int)(n - col < 32 ? n - col : 32);
        const bool whole = vec_out && (!add || vec_add);  // the same in every lane
        if (whole && s.row < 0) return;
        const int64_t row = s.row;
        if (s.f != 1.0f) {
#pragma unroll
            for (int j = 0; j < 16; ++j) v[j] = __fmul2_rn(v[j], both(s.f));
        }
        if (bias) add_bias32(v, tile_bias);
        if (!whole) {
            ragged(row, v, col, cols);
            return;
        }
        if (add) {
            if (early && cols == 32) {
                if (add_type == DNB_BF16) add_fetched<__nv_bfloat16>(v, h);
                else add_fetched<__half>(v, h);
            } else if (add_type == DNB_F32) load_add<float>(v, row, col, cols);
            else if (add_type == DNB_BF16) load_add<__nv_bfloat16>(v, row, col, cols);
            else load_add<__half>(v, row, col, cols);
        }
        activate(v);
        if (out_type == DNB_F32) store<float>(v, row, col, cols);
        else if (out_type == DNB_BF16) store<__nv_bfloat16>(v, row, col, cols);
        else store<__half>(v, row, col, cols);
    }
    static __device__ __noinline__ float activate_one(float v, int a) { return act_fwd_any(v, a); }
    static __device__ __forceinline__ void activate_any(float2 (&v)[16], int a) {
#pragma unroll
        for (int j = 0; j < 16; ++j) v[j] = make_float2(activate_one(v[j].x, a), activate_one(v[j].y, a));
    }
};

inline EpiOut epilogue(void *out, int64_t ld, int type, int64_t m, int64_t n) {
    EpiOut e;
    e.out = out;
    e.ld = ld;
    e.out_type = type;
    e.m = m;
    e.n = n;
    e.vec_out = aligned16(out) && ld * dtype_size(type) % 16 == 0;
    e.wide_out = reinterpret_cast<uintptr_t>(out) % 32 == 0 && ld * dtype_size(type) % 32 == 0;
    return e;
}
inline void add_to(EpiOut &e, const void *add, int64_t ld, int type) {
    e.add = add;
    e.ld_add = ld;
    e.add_type = type;
    e.vec_add = aligned16(add) && ld * dtype_size(type) % 16 == 0;
    e.early = e.vec_add && type != DNB_F32;
}

// The product with this epilogue, in the tiles that pick_tiles names; a_mn / b_mn: MN-major operands. With
// m_dev / k_dev, m and k are what they may reach. dnb_product.cu.
dnb_status product(bool a_mn, bool b_mn, const Operand &a, const Operand &b, int dtype, int64_t m, int64_t n, int64_t k,
                   const EpiOut &e, const DeviceState *ds, cudaStream_t s, const char *what,
                   const int *m_dev = nullptr, const int *k_dev = nullptr);

}  // namespace dnb
