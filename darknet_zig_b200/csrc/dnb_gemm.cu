// Tensor maps and aligned copies for the tensor-core products (dnb_gemm.cuh).
#include "dnb_gemm.cuh"
#include "dnb_pack.cuh"

namespace dnb {

namespace {

using EncodeFn = CUresult (*)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *,
                              const cuuint64_t *, const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave,
                              CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

// The driver's encoder, looked up once: the library links no driver stub.
EncodeFn encoder() {
    static const EncodeFn fn = [] {
        void *p = nullptr;
        cudaDriverEntryPointQueryResult found = cudaDriverEntryPointSymbolNotFound;
        if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &found) !=
                cudaSuccess ||
            found != cudaDriverEntryPointSuccess)
            p = nullptr;
        return reinterpret_cast<EncodeFn>(p);
    }();
    return fn;
}

// Eight elements a thread: 16-byte stores whatever the source's alignment. Vectors [0, split) are job 0's, the
// rest job 1's, so that a product's two operands take one launch.
template <class T>
struct PackArgs {
    const T *src[2];
    T *dst[2];
    int64_t lds[2], ldd[2], rows[2], cols[2], per[2], split;
    FastDiv div[2];  // by per, where the job's vectors are below 2^32
    Gather g;        // job 0's
};
template <class T>
__global__ void __launch_bounds__(256) k_pack(const __grid_constant__ PackArgs<T> a) {
    const int64_t kept = a.g.count ? *a.g.count : a.rows[0], end = a.g.count ? (kept + 63) / 64 * 64 : a.rows[0];
    const int64_t total = a.split + a.rows[1] * a.per[1];
    for (int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x; at < total; at += (int64_t)gridDim.x * 256) {
        const int job = at >= a.split;
        const int64_t i = job ? at - a.split : at, per = a.per[job];
        int64_t r, c;
        if (a.rows[job] * per <= 0xffffffc0ll) {
            uint32_t q, m;
            a.div[job].divmod((uint32_t)i, q, m);
            r = q;
            c = (int64_t)m * 8;
        } else {
            r = i / per;
            c = (i - r * per) * 8;
        }
        typename Vec<T, 16>::U u;
        u.raw = make_uint4(0u, 0u, 0u, 0u);
        if (job == 0 && r >= end) continue;
        if (job == 1 || r < kept) {
            const int64_t from = job == 0 && a.g.rows ? a.g.rows[r] : r, cols = a.cols[job];
            const T *p = a.src[job] + from * a.lds[job] + c;
            if (c + 8 <= cols && (reinterpret_cast<uintptr_t>(p) & 15) == 0) {
                u.raw = *reinterpret_cast<const uint4 *>(p);
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (c + j < cols) u.e[j] = p[j];
            }
            if (job == 0 && a.g.factor) {
                float f[8];
                Vec<T, 16>::unpack(u.raw, f);
                const float by = a.g.factor[from] * *a.g.norm;
#pragma unroll
                for (int j = 0; j < 8; ++j) f[j] *= by;
                u.raw = Vec<T, 16>::pack(f);
            }
        }
        *reinterpret_cast<uint4 *>(a.dst[job] + r * a.ldd[job] + c) = u.raw;
    }
}

// Adds the chunks' column sums in fp64, 8 slices of them in order, then the slices.
__global__ void __launch_bounds__(256) k_column_sums(const float *part, int64_t chunks, int64_t n, int64_t ld,
                                                     float *out, int add) {
    __shared__ double red[8][32];
    const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
    const int64_t c = (int64_t)blockIdx.x * 32 + tx;
    double s = 0.0;
    if (c < n)
#pragma unroll 4
        for (int64_t q = ty; q < chunks; q += 8) s += (double)part[q * ld + c];
    red[ty][tx] = s;
    __syncthreads();
    if (ty == 0 && c < n) {
        for (int i = 1; i < 8; ++i) s += red[i][tx];
        out[c] = (float)(add ? (double)out[c] + s : s);
    }
}

// A block per row; 16-byte stores where every row starts on that boundary, else 2-byte ones.
__global__ void __launch_bounds__(256) k_zero_rows(unsigned char *p, int64_t rows, int64_t row_bytes, int64_t stride,
                                                   const int32_t *labels, int64_t classes, bool wide) {
    for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
        if (labels && labels[r] >= 0 && labels[r] < classes) continue;
        unsigned char *q = p + r * stride;
        const int64_t head = wide ? row_bytes / 16 * 16 : 0;
        for (int64_t i = threadIdx.x * 16; i < head; i += 256 * 16)
            *reinterpret_cast<uint4 *>(q + i) = make_uint4(0u, 0u, 0u, 0u);
        for (int64_t i = head + threadIdx.x * 2; i < row_bytes; i += 256 * 2) *reinterpret_cast<uint16_t *>(q + i) = 0;
    }
}

}  // namespace

dnb_status make_map(CUtensorMap *map, const void *p, int64_t inner, int64_t outer, int64_t stride, int box_outer,
                    int dtype, const char *what) {
    const EncodeFn fn = encoder();
    if (!fn) return fail(DNB_ERR_CUDA, "%s: the driver has no cuTensorMapEncodeTiled", what);
    if (inner <= 0 || outer <= 0 || inner > 0x7fffffffll || outer > 0x7fffffffll || stride > (int64_t(1) << 38))
        return fail(DNB_ERR_UNSUPPORTED, "%s: a matrix of %lld x %lld is beyond the tensor maps", what,
                    (long long)outer, (long long)inner);
    const cuuint64_t dims[2] = {(cuuint64_t)inner, (cuuint64_t)outer};
    // a single row's stride is never used, but must be a valid one
    const cuuint64_t strides[1] = {(cuuint64_t)(outer == 1 ? (inner + 7) / 8 * 8 : stride) * 2};
    const cuuint32_t box[2] = {64u, (cuuint32_t)box_outer}, elem[2] = {1u, 1u};
    const CUresult r = fn(map, dtype == DNB_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2u,
                          const_cast<void *>(p), dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE,
                          CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                          CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return fail(DNB_ERR_CUDA, "%s: cuTensorMapEncodeTiled failed (%d)", what, (int)r);
    return DNB_OK;
}

dnb_status pack_rows(const PackJob &x, const PackJob &w, int dtype, const Gather &g, const DeviceState *ds,
                     cudaStream_t s, const char *what) {
    return dispatch_dtype16(dtype, [&]<class T>() -> dnb_status {
        PackArgs<T> a{};
        const PackJob *jobs[2] = {&x, &w};
        int64_t vectors[2];
        for (int k = 0; k < 2; ++k) {
            const PackJob &q = *jobs[k];
            a.src[k] = static_cast<const T *>(q.src);
            a.dst[k] = static_cast<T *>(q.dst);
            a.lds[k] = q.ld;
            a.ldd[k] = packed_ld(q.cols);
            a.rows[k] = q.dst ? q.rows : 0;
            if (k == 0 && g.count) a.rows[k] = (a.rows[k] + 63) / 64 * 64;
            a.cols[k] = q.cols;
            a.per[k] = q.dst ? (q.cols + 7) / 8 : 1;
            a.div[k] = FastDiv((uint32_t)a.per[k]);
            vectors[k] = a.rows[k] * a.per[k];
        }
        if (vectors[0] + vectors[1] == 0) return DNB_OK;
        a.split = vectors[0];
        a.g = g;
        k_pack<T><<<grid_for(vectors[0] + vectors[1], 256, ds), 256, 0, s>>>(a);
        return after_launch(s, what);
    });
}

dnb_status column_sums(const float *part, int64_t chunks, int64_t n, int64_t ld, float *out, bool add, cudaStream_t s,
                       const char *what) {
    k_column_sums<<<(unsigned)((n + 31) / 32), 256, 0, s>>>(part, chunks, n, ld, out, add);
    return after_launch(s, what);
}

dnb_status zero_rows(void *p, int64_t rows, int64_t cols, int64_t ld, int64_t e, const DeviceState *ds, cudaStream_t s,
                     const char *what, const int32_t *labels, int64_t classes) {
    k_zero_rows<<<grid_for(rows, 1, ds), 256, 0, s>>>(static_cast<unsigned char *>(p), rows, cols * e, ld * e, labels,
                                                      classes, aligned16(p) && ld * e % 16 == 0);
    return after_launch(s, what);
}

}  // namespace dnb
