// The products whose results are stored (dnb_epilogue.cuh), for each pair of operand layouts and tile shape.
#include "dnb_epilogue.cuh"

namespace dnb {
namespace {

template <bool A_MN, bool B_MN>
dnb_status run(const Operand &a, const Operand &b, int dtype, int64_t m, int64_t n, int64_t k, const EpiOut &e,
               const DeviceState *ds, cudaStream_t s, const char *what, const int *m_dev, const int *k_dev) {
    const Tiles t = pick_tiles(m, n, k);
    if (t.ctas == 2)
        return launch_gemm<GemmCfg<2, 256, A_MN, B_MN>>(a, b, dtype, m, n, k, e, ds, s, what, 1, m_dev, k_dev);
    if (t.split > 1)
        return launch_gemm<GemmCfg<1, 128, A_MN, B_MN, true>>(a, b, dtype, m, n, k, e, ds, s, what, t.split, m_dev, k_dev);
    return launch_gemm<GemmCfg<1, 128, A_MN, B_MN>>(a, b, dtype, m, n, k, e, ds, s, what, 1, m_dev, k_dev);
}

}  // namespace

dnb_status product(bool a_mn, bool b_mn, const Operand &a, const Operand &b, int dtype, int64_t m, int64_t n, int64_t k,
                   const EpiOut &e, const DeviceState *ds, cudaStream_t s, const char *what, const int *m_dev,
                   const int *k_dev) {
    if (a_mn) return run<true, true>(a, b, dtype, m, n, k, e, ds, s, what, m_dev, k_dev);
    if (b_mn) return run<false, true>(a, b, dtype, m, n, k, e, ds, s, what, m_dev, k_dev);
    return run<false, false>(a, b, dtype, m, n, k, e, ds, s, what, m_dev, k_dev);
}

}  // namespace dnb
