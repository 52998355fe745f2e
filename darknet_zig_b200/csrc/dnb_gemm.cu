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

// Eight elements a thread: 16-byte stores whatever the source's alignment. Rows whose label is outside
// [0, classes) become zeros and are not read.
__global__ void __launch_bounds__(256) k_pack(const uint16_t *src, int64_t lds, uint16_t *dst, int64_t ldd,
                                              int64_t rows, int64_t cols, int64_t per, const int32_t *labels,
                                              int64_t classes) {
    const int64_t total = rows * per;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
        const int64_t r = i / per, c = (i - r * per) * 8;
        const bool keep = !labels || (labels[r] >= 0 && labels[r] < classes);
        uint16_t v[8] = {};
        if (keep) {
            const uint16_t *p = src + r * lds + c;
            if (c + 8 <= cols && (reinterpret_cast<uintptr_t>(p) & 15) == 0) {
                *reinterpret_cast<uint4 *>(v) = *reinterpret_cast<const uint4 *>(p);
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (c + j < cols) v[j] = p[j];
            }
        }
        *reinterpret_cast<uint4 *>(dst + r * ldd + c) =
            make_uint4(v[0] | (uint32_t)v[1] << 16, v[2] | (uint32_t)v[3] << 16, v[4] | (uint32_t)v[5] << 16,
                       v[6] | (uint32_t)v[7] << 16);
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

dnb_status pack_rows(const void *src, int64_t lds, void *dst, int64_t rows, int64_t cols, const int32_t *labels,
                     int64_t classes, const DeviceState *ds, cudaStream_t s, const char *what) {
    const int64_t per = (cols + 7) / 8;
    k_pack<<<grid_for(rows * per, 256, ds), 256, 0, s>>>(static_cast<const uint16_t *>(src), lds,
                                                         static_cast<uint16_t *>(dst), packed_ld(cols), rows, cols,
                                                         per, labels, classes);
    return after_launch(s, what);
}

}  // namespace dnb
