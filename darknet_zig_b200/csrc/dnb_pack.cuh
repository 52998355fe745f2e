// Aligned copies of 16-bit matrices for TMA, and how a call cuts up the caller's workspace.
#pragma once

#include "dnb_types.cuh"

namespace dnb {

inline int64_t packed_ld(int64_t cols) { return (cols + 7) / 8 * 8; }
inline int64_t packed_bytes(int64_t rows, int64_t cols) { return rows * packed_ld(cols) * 2; }

// Copies up to two matrices to rows packed_ld(cols) apart at 16-byte aligned dst, in one launch (dst NULL: none).
// With a row map, the first matrix's rows are the map's first *count, gathered, with zero rows after them up to
// a multiple of 64. With factors, row r of it is multiplied by factor[r] * *norm and rounded again. dnb_gemm.cu.
struct PackJob {
    const void *src = nullptr;
    int64_t ld = 0;
    void *dst = nullptr;
    int64_t rows = 0, cols = 0;
};
struct Gather {
    const int *rows = nullptr, *count = nullptr;
    const float *factor = nullptr, *norm = nullptr;
};
dnb_status pack_rows(const PackJob &x, const PackJob &w, int dtype, const Gather &g, const DeviceState *ds,
                     cudaStream_t s, const char *what);

inline dnb_status product_shape_check(int dtype, int64_t m, int64_t k, int64_t n, const char *what) {
    if (!valid_dtype16(dtype)) return fail(DNB_ERR_INVALID, "%s: dtype must be bf16 or f16", what);
    if (m < 0 || k < 0 || n < 0) return fail(DNB_ERR_INVALID, "%s: negative size", what);
    if (m > 0x7fffffffll || k > 0x7fffffffll || n > 0x7fffffffll)
        return fail(DNB_ERR_UNSUPPORTED, "%s: a size beyond 2^31 - 1", what);
    return DNB_OK;
}

inline dnb_status workspace_check(void *ws, size_t have, size_t need, const char *what) {
    if (need && (!ws || have < need || !aligned16(ws)))
        return fail(DNB_ERR_INVALID, "%s: needs a 16-byte aligned workspace of %zu bytes, got %zu", what, need,
                    ws ? have : (size_t)0);
    return DNB_OK;
}

// out[c] (+)= the sum of part[q][c] over the chunks q, rows of `part` ld apart; in fp64, in a fixed order.
dnb_status column_sums(const float *part, int64_t chunks, int64_t n, int64_t ld, float *out, bool add, cudaStream_t s,
                       const char *what);
// Fills a matrix's rows with zeros; with labels, only the rows whose label is outside [0, classes).
dnb_status zero_rows(void *p, int64_t rows, int64_t cols, int64_t ld, int64_t e, const DeviceState *ds, cudaStream_t s,
                     const char *what, const int32_t *labels = nullptr, int64_t classes = 0);

// Hands out 256-byte aligned pieces of a workspace (of nothing: only their sum).
struct Carver {
    char *base;
    size_t used = 0;
    explicit Carver(void *p) : base(static_cast<char *>(p)) {}
    void *take(int64_t bytes) {
        void *p = base ? base + used : nullptr;
        used += ((size_t)bytes + 255) / 256 * 256;
        return p;
    }
};

}  // namespace dnb
