// Aligned copies of 16-bit matrices for TMA, and how a call cuts up the caller's workspace.
#pragma once

#include "dnb_types.cuh"

namespace dnb {

inline int64_t packed_ld(int64_t cols) { return (cols + 7) / 8 * 8; }
inline int64_t packed_bytes(int64_t rows, int64_t cols) { return rows * packed_ld(cols) * 2; }

// Copies a matrix to rows packed_ld(cols) apart at a 16-byte aligned dst; with labels, rows whose label is
// outside [0, classes) become zeros without being read. dnb_gemm.cu.
dnb_status pack_rows(const void *src, int64_t lds, void *dst, int64_t rows, int64_t cols, const int32_t *labels,
                     int64_t classes, const DeviceState *ds, cudaStream_t s, const char *what);

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
