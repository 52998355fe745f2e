// The matrix product behind the connected layer and the cross entropy: C[m][n] = sum_k A(m,k) B(n,k) with
// 16-bit operands and fp32 accumulators on the 5th-generation tensor cores, persistent, with the epilogue
// as a template argument.
//
// An operand is K-major (its rows run along k: x and w of a forward product) or MN-major (its rows run
// along m or n: the transposed operands of a backward product); both are brought in by TMA with the
// 128-byte swizzle and described to the tensor core where they lie, so no product needs a transposed copy.
//
// A CTA (CTAS = 1) or a pair on neighbouring SMs (CTAS = 2, cta_group::2) owns one output tile of
// 128*CTAS x BN at a time. Warp 0 issues the loads into a ring of stages (64 k each), warp 1 of the pair's
// first CTA issues the products into one of two accumulators in tensor memory, warps 4-11 take the other
// accumulator through the epilogue meanwhile (two warps a scheduler, each half of the columns: one alone
// leaves its latencies bare and took 7 us for a tile that two finish in 3). A pair halves the operand traffic per
// SM: each CTA holds its own 128 rows of A and half of B's rows, and the products read both CTAs' shared memory.
// Where tiles are few, a cluster of CTAs shares a tile's k (SPLIT).
//
// Bound by the tensor cores from some 256 rows and columns a side on: [2048,4096]x[4096,4096]^T bf16 48 us, 1430
// TFLOP/s; [8192,16384]x[4096,16384]^T with residual 730 us (1506) in a single launch, 850 us (1290) back to back
// under the power cap.
//
// Every wait is bounded (dnb_set_wait_limit_ms): a role whose wait gives up sets the error word and
// leaves its loop; the others' waits then end the same way, the CTA (pair) meets at its last barrier and
// frees its tensor memory.
#pragma once

#include <cuda.h>

#include <atomic>

#include "dnb_types.cuh"

namespace dnb {

// ---- host side: tensor maps ----

// A 2-D tensor map of 16-bit elements: `inner` contiguous elements, `outer` rows `stride` elements apart,
// boxes of 64 x box_outer elements with the 128-byte swizzle, zeros outside. dnb_gemm.cu.
dnb_status make_map(CUtensorMap *map, const void *p, int64_t inner, int64_t outer, int64_t stride, int box_outer,
                    int dtype, const char *what);

// An operand as the tensor core wants it: 16-byte aligned rows. `mn` rows of length k (K-major), or k rows
// of length mn (MN-major).
struct Operand {
    const void *p = nullptr;
    int64_t ld = 0;
};
inline bool tma_ready(const void *p, int64_t ld) { return aligned16(p) && ld % 8 == 0; }

// ---- the product's description ----

struct GemmArgs {
    int64_t m, n, k;
    int m_tiles, n_tiles, k_blocks;
    int band;       // output tiles are taken in bands of this many row tiles, down the rows first
    unsigned idesc; // the tensor core's instruction descriptor
    unsigned stage_bytes;  // what a CTA's loads of a stage bring
    int split;             // CTAs that share a tile (SPLIT)
    const int *m_dev, *k_dev;  // the rows / the reduction's length where the device knows them (NULL: as above)
    unsigned long long wait_ns;
    unsigned *error_word;
};

constexpr int kGemmThreads = 384;  // 4 warps of roles, 8 of epilogue
constexpr int kEpilogueWarps = 8;
constexpr int kBlockK = 64;
constexpr int kMaxSplit = 4;  // CTAs that may share a tile's k
constexpr unsigned DEVERR_WAIT_GEMM = 8u;  // a role of a product gave up waiting

template <int CTAS_, int BN_, bool A_MN_, bool B_MN_, bool SPLIT_ = false>
struct GemmCfg {
    static constexpr int CTAS = CTAS_, BN = BN_;
    static constexpr bool A_MN = A_MN_, B_MN = B_MN_;
    static constexpr bool SPLIT = SPLIT_;      // a cluster of CTAs shares one tile's k
    static constexpr int BM = 128;             // rows of one CTA
    static constexpr int TM = BM * CTAS;       // rows of a tile
    static constexpr int BROWS = BN / CTAS;    // B rows one CTA holds
    static constexpr int A_BYTES = BM * kBlockK * 2, B_BYTES = BROWS * kBlockK * 2;
    static constexpr int STAGE = A_BYTES + B_BYTES;
    static constexpr int STAGES = 6;
    static constexpr int TMEM_COLS = 2 * BN;
    static constexpr int EW = BN / 2;          // columns of an epilogue thread: two share a row
    static constexpr size_t SMEM = 1024 + (size_t)STAGES * STAGE + 16 * STAGES + 64 + 8 * BN;
    static_assert(EW % 64 == 0 && BN <= 256 && (TMEM_COLS & (TMEM_COLS - 1)) == 0, "tile");
    static_assert(!SPLIT || (CTAS == 1 && BN == 128), "four runs of 32 columns are shared out");
    static_assert(!B_MN || BROWS % 64 == 0, "an MN-major box is 64 wide");
};

// ---- device side ----

namespace gemm {

__device__ __forceinline__ uint32_t smem_u32(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }

__device__ __forceinline__ void mbar_init(uint32_t bar, uint32_t count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void mbar_expect(uint32_t bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
// Arrives at a shared::cluster address for reads of tensor memory, which the wait for them and the tcgen05 fence
// before it order: relaxed, for a release would wait for the epilogue's stores too (0.7 us a tile).
__device__ __forceinline__ void mbar_arrive_relaxed(uint32_t bar) {
    asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ bool mbar_try(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, 0x989680;\n\t"
        "selp.b32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(bar), "r"(parity)
        : "memory");
    return ok != 0;
}
// One lane of the (converged) warp.
__device__ __forceinline__ bool elect_one() {
    uint32_t one;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.b32 %0, 1, 0, p;\n\t}" : "=r"(one));
    return one != 0;
}
// Waits for the phase of `parity` to end. False: the limit passed or another role gave up.
__device__ __forceinline__ bool mbar_wait(uint32_t bar, uint32_t parity, const GemmArgs &g, volatile unsigned *gave_up) {
    if (mbar_try(bar, parity)) return true;
    const unsigned long long start = global_ns();
    while (!mbar_try(bar, parity)) {
        if (*gave_up) return false;
        if (global_ns() - start > g.wait_ns) {
            *gave_up = 1u;
            atomicOr(g.error_word, DEVERR_WAIT_GEMM);
            return false;
        }
    }
    return true;
}

// The same, without telling: a wait that passes the limit sets the flag (a shared-memory address) and the error
// word and returns; once the flag is set, every wait returns after one try.
__device__ __forceinline__ void mbar_wait_or_flag(uint32_t bar, uint32_t parity, const GemmArgs &g, uint32_t flag) {
    asm volatile(
        "{\n\t"
        ".reg .pred p;\n\t.reg .u64 t0, t;\n\t.reg .u32 f;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%0], %1;\n\t"
        "@p bra DONE;\n\t"
        "mov.u64 t0, %%globaltimer;\n\t"
        "AGAIN:\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%0], %1, 0x989680;\n\t"
        "@p bra DONE;\n\t"
        "ld.volatile.shared.u32 f, [%3];\n\t"
        "setp.ne.u32 p, f, 0;\n\t"
        "@p bra DONE;\n\t"
        "mov.u64 t, %%globaltimer;\n\t"
        "sub.u64 t, t, t0;\n\t"
        "setp.le.u64 p, t, %2;\n\t"
        "@p bra AGAIN;\n\t"
        "mov.u32 f, 1;\n\t"
        "st.volatile.shared.u32 [%3], f;\n\t"
        "red.global.or.b32 [%4], %5;\n\t"
        "DONE:\n\t"
        "}" ::"r"(bar),
        "r"(parity), "l"(g.wait_ns), "r"(flag), "l"(g.error_word), "r"(DEVERR_WAIT_GEMM)
        : "memory");
}

__device__ __forceinline__ uint32_t map_rank(uint32_t addr, uint32_t rank) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
    return r;
}
__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// One box of a tensor map into this CTA's shared memory; `bar` (a shared::cluster address) counts its bytes.
template <int CTAS>
__device__ __forceinline__ void tma_load(uint32_t dst, const CUtensorMap *map, int x, int y, uint32_t bar) {
    if constexpr (CTAS == 2)
        asm volatile(
            "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 [%0], "
            "[%1, {%2, %3}], [%4];" ::"r"(dst),
            "l"(map), "r"(x), "r"(y), "r"(bar)
            : "memory");
    else
        asm volatile(
            "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], "
            "[%4];" ::"r"(dst),
            "l"(map), "r"(x), "r"(y), "r"(bar)
            : "memory");
}

// Shared-memory matrix descriptor, 128-byte swizzle. K-major: rows of 128 bytes, 8-row groups 1024 bytes
// apart (stride offset); the leading offset is unused. MN-major: 64-element runs along mn, 8-k groups 1024
// bytes apart (stride offset), 64-wide column blocks `leading` bytes apart.
__device__ __forceinline__ uint64_t smem_desc(uint32_t addr, uint32_t leading) {
    return (uint64_t)((addr & 0x3ffff) >> 4) | ((uint64_t)(leading >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) |
           ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}

template <int CTAS>
__device__ __forceinline__ void mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t add) {
    if constexpr (CTAS == 2)
        asm volatile(
            "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
            "l"(a), "l"(b), "r"(idesc), "r"(add)
            : "memory");
    else
        asm volatile(
            "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
            "l"(a), "l"(b), "r"(idesc), "r"(add)
            : "memory");
}
// Arrives on `bar` (in both CTAs of a pair) when the products issued so far are done.
template <int CTAS>
__device__ __forceinline__ void commit(uint32_t bar) {
    if constexpr (CTAS == 2)
        asm volatile(
            "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
                bar),
            "h"((uint16_t)3)
            : "memory");
    else
        asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar)
                     : "memory");
}
template <int CTAS>
__device__ __forceinline__ void tmem_alloc(uint32_t dst, uint32_t cols) {
    if constexpr (CTAS == 2) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(dst), "r"(cols)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
    } else {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(dst), "r"(cols)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
}
template <int CTAS>
__device__ __forceinline__ void tmem_free(uint32_t base, uint32_t cols) {
    if constexpr (CTAS == 2)
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(base), "r"(cols));
    else
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(base), "r"(cols));
}
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// 32 columns of this warp's 32 lanes: r[j] is (lane, column j), there after tmem_wait().
__device__ __forceinline__ void tmem_load32(uint32_t addr, uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
        "%15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
          "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
          "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(addr));
}
// The registers pass through the wait, so that nothing that reads them moves above it.
__device__ __forceinline__ void tmem_wait(uint32_t (&r)[32]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                   "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]),
                   "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]),
                   "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]),
                   "+r"(r[30]), "+r"(r[31])::"memory");
}
// The epilogue warps meet.
__device__ __forceinline__ void epilogue_sync() { asm volatile("bar.sync 1, 256;" ::: "memory"); }

// The row tile and column tile of the t-th tile.
__device__ __forceinline__ void tile_at(const GemmArgs &g, int m_tiles, int t, int &mt, int &nt) {
    const int per = g.band * g.n_tiles, b = t / per, in = t - b * per;
    const int rows = min(g.band, m_tiles - b * g.band);
    nt = in / rows;
    mt = b * g.band + (in - nt * rows);
}

}  // namespace gemm

// Epi: a struct passed by value to the kernel, with
//   const float *bias;                                     a value per column, or NULL
//   struct State;                                          a thread's row, kept over a tile's columns
//   struct Ahead;                                          what 32 columns read from global memory
//   void begin(State &, int64_t row, int64_t col0) const;
//   void fetch(const State &, Ahead &, int64_t col) const; ahead of the accumulators
//   void columns(State &, float2 (&v)[16], const float *bias, const Ahead &, int64_t row, int64_t col) const;
//                                                          32 columns from `col`; bias: theirs, in shared memory
//                                                          (row's columns are seen in two halves of the tile, by
//                                                          two threads)
//   void end(State &, int64_t row, int64_t col0) const;
// All 32 lanes call each of them (rows beyond m included: the functions check). The bias of a tile and the
// first columns' reads are on their way while the accumulators fill; read one by one when needed, 32 biases
// cost 1.5 us a chunk of 32 columns, more than the product of a short k.
template <class C, class Epi>
__global__ void __launch_bounds__(kGemmThreads, 1)
    k_gemm(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
           const __grid_constant__ GemmArgs g, const __grid_constant__ Epi epi) {
    using namespace gemm;
    constexpr int CTAS = C::CTAS, S = C::STAGES;
    extern __shared__ unsigned char raw[];
    const uint32_t base = (smem_u32(raw) + 1023u) & ~1023u;
    unsigned char *tail = raw + (base - smem_u32(raw)) + S * C::STAGE;
    // barriers after the stages: full[S], empty[S], accumulator full[2], accumulator empty[2]; then the
    // tensor memory's address and the give-up flag
    const uint32_t bars = base + S * C::STAGE;
    const uint32_t full = bars, empty = bars + 8 * S, acc_full = bars + 16 * S, acc_empty = acc_full + 16;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(tail + 16 * S + 32);
    volatile unsigned *gave_up = reinterpret_cast<volatile unsigned *>(tail + 16 * S + 36);
    const uint32_t flag = bars + 16 * S + 36;  // gave_up's address
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = CTAS == 2 ? cluster_rank() : 0u;

    if (threadIdx.x == 0) {
        for (int s = 0; s < S; ++s) {
            mbar_init(full + 8 * s, 1);
            mbar_init(empty + 8 * s, 1);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(acc_full + 8 * b, 1);
            mbar_init(acc_empty + 8 * b, kEpilogueWarps * CTAS);
        }
        *gave_up = 0u;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async;" ::: "memory");
    }
    if (warp == 2) tmem_alloc<CTAS>(smem_u32(tmem_slot), C::TMEM_COLS);
    fence_before();
    __syncthreads();
    if constexpr (CTAS == 2) cluster_sync();
    fence_after();
    const uint32_t tmem = *tmem_slot;
    const int m_tiles = g.m_dev ? (*g.m_dev + C::TM - 1) / C::TM : g.m_tiles;
    const int k_all = g.k_dev ? (*g.k_dev + kBlockK - 1) / kBlockK : g.k_blocks;
    const int tiles = m_tiles * g.n_tiles;
    // SPLIT: a tile a cluster, this CTA's share of its k blocks; else every step-th tile, all of them
    const int share = C::SPLIT ? g.split : 1, q = C::SPLIT ? (int)cluster_rank() : 0;
    const int step = C::SPLIT ? 0x3fffffff : (int)gridDim.x / CTAS, first = (int)blockIdx.x / (C::SPLIT ? share : CTAS);
    const int kb0 = C::SPLIT ? k_all * q / share : 0, k_blocks = C::SPLIT ? k_all * (q + 1) / share - kb0 : k_all;

    if (warp == 0 && lane == 0) {
        // loads
        int s = 0, it = 0;
        uint32_t phase = 1;
        bool ok = true;
        for (int t = first; ok && t < tiles; t += step) {
            int mt, nt;
            tile_at(g, m_tiles, t, mt, nt);
            const int am = mt * C::TM + (int)rank * C::BM, bn = nt * C::BN + (int)rank * C::BROWS;
            for (int kb = 0; kb < k_blocks; ++kb, ++it) {
                if (!mbar_wait(empty + 8 * s, phase, g, gave_up)) {
                    ok = false;
                    break;
                }
                const uint32_t a_at = base + s * C::STAGE, b_at = a_at + C::A_BYTES;
                const uint32_t bar = CTAS == 2 ? map_rank(full + 8 * s, 0) : full + 8 * s;
                const int k0 = (kb0 + kb) * kBlockK;
                if (rank == 0) mbar_expect(full + 8 * s, g.stage_bytes * CTAS);
                if constexpr (C::A_MN) {
#pragma unroll
                    for (int c = 0; c < C::BM / 64; ++c) tma_load<CTAS>(a_at + c * 8192, &map_a, am + c * 64, k0, bar);
                } else {
                    tma_load<CTAS>(a_at, &map_a, k0, am, bar);
                }
                if constexpr (C::B_MN) {
#pragma unroll
                    for (int c = 0; c < C::BROWS / 64; ++c)
                        tma_load<CTAS>(b_at + c * 8192, &map_b, bn + c * 64, k0, bar);
                } else {
                    tma_load<CTAS>(b_at, &map_b, k0, bn, bar);
                }
                if (++s == S) {
                    s = 0;
                    phase ^= 1;
                }
            }
        }
        // the last products still read (and their commits still arrive at) these stages
        for (int j = it > S ? it - S : 0; ok && j < it; ++j)
            if (!mbar_wait(empty + 8 * (j % S), (j / S) & 1, g, gave_up)) ok = false;
        // giving up: the copies in flight still land in this pair's shared memory (bounded: 2^20 tries each)
        if (!ok && rank == 0)
            for (int j = it > S ? it - S : 0; j < it; ++j)
                for (int tries = 0; tries < (1 << 20) && !mbar_try(full + 8 * (j % S), (j / S) & 1); ++tries) {}
    } else if (warp == 1 && rank == 0) {
        // Products. The warp runs the loop whole, with waits that return nothing, so that what the instructions take
        // stays in uniform registers; one lane issues (a commit covers what its own thread issued). After a wait
        // that gave up the loop runs to its end on whatever the stages hold.
        const bool issues = elect_one();
        int s = 0, n = 0;
        uint32_t phase = 0;
        for (int t = first; t < tiles; t += step, ++n) {
            const int b = n & 1;
            mbar_wait_or_flag(acc_empty + 8 * b, ((n >> 1) & 1) ^ 1, g, flag);
            fence_after();
            const uint32_t d = tmem + b * C::BN;
            for (int kb = 0; kb < k_blocks; ++kb) {
                mbar_wait_or_flag(full + 8 * s, phase, g, flag);
                fence_after();
                const uint32_t a_at = base + s * C::STAGE, b_at = a_at + C::A_BYTES;
                const uint64_t da = smem_desc(a_at, C::A_MN ? 8192u : 16u), db = smem_desc(b_at, C::B_MN ? 8192u : 16u);
                if (issues) {
#pragma unroll
                    for (int k = 0; k < kBlockK / 16; ++k)  // 16 k: 32 bytes of a K-major row, 16 rows MN-major
                        mma<CTAS>(d, da + (uint64_t)(k * (C::A_MN ? 2048 : 32) >> 4),
                                  db + (uint64_t)(k * (C::B_MN ? 2048 : 32) >> 4), g.idesc, (kb | k) != 0);
                    commit<CTAS>(empty + 8 * s);
                }
                if (++s == S) {
                    s = 0;
                    phase ^= 1;
                }
            }
            if (issues) commit<CTAS>(acc_full + 8 * b);
        }
    }

    // Epilogue: a warp reads its quarter of the tensor memory's lanes (a lane a row) and half of the columns.
    constexpr int EW = C::EW;
    const int w = warp & 3, half = (warp - 4) >> 2;
    float *bias = reinterpret_cast<float *>(tail + 16 * S + 64);  // [2][BN]
    bool failed = false;
    // The n-th tile of this CTA.
    auto take_tile = [&](int t, int n) {
        const int b = n & 1;
        int mt, nt;
        tile_at(g, m_tiles, t, mt, nt);
        const int64_t row = (int64_t)mt * C::TM + (int64_t)rank * C::BM + w * 32 + lane, tile0 = (int64_t)nt * C::BN,
                      col0 = tile0 + half * EW;
        typename Epi::State st;
        epi.begin(st, row, col0);
        typename Epi::Ahead ahead[2];
        epi.fetch(st, ahead[0], col0);
        if (epi.bias) {  // the buffer's last readers, two tiles ago, have met at the last tile's barrier
            const int c = threadIdx.x - 128;
            if (c < C::BN) bias[b * C::BN + c] = tile0 + c < g.n ? epi.bias[tile0 + c] : 0.0f;
            epilogue_sync();
        }
        const float *tile_bias = bias + b * C::BN + half * EW;
        // a warp that gave up goes on to the barriers, which the other warps may still wait at
        if (!failed) failed = !__all_sync(0xffffffffu, mbar_wait(acc_full + 8 * b, (n >> 1) & 1, g, gave_up));
        if (failed) return;
        fence_after();
        const uint32_t at = tmem + ((uint32_t)(w * 32) << 16) + b * C::BN + half * EW;
#pragma unroll 1
        for (int c = 0; c < EW; c += 64) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int64_t col = col0 + c + 32 * h;
                uint32_t r[32];
                __syncwarp();  // the loads are the whole warp's
                if (k_blocks > 0) tmem_load32(at + c + 32 * h, r);
                if (c + 32 * (h + 1) < EW && col + 32 < g.n) epi.fetch(st, ahead[h ^ 1], col + 32);
                if (k_blocks > 0) {
                    tmem_wait(r);
                } else {  // a sum over nothing
#pragma unroll
                    for (int j = 0; j < 32; ++j) r[j] = 0u;
                }
                if (c + 32 * (h + 1) >= EW) {  // all read: the next products may overwrite the accumulators
                    fence_before();
                    __syncwarp();
                    if (lane == 0)
                        mbar_arrive_relaxed(CTAS == 2 ? map_rank(acc_empty + 8 * b, 0) : acc_empty + 8 * b);
                }
                float2 v[16];
#pragma unroll
                for (int j = 0; j < 16; ++j) v[j] = make_float2(__uint_as_float(r[2 * j]), __uint_as_float(r[2 * j + 1]));
                if (col < g.n) epi.columns(st, v, tile_bias + c + 32 * h, ahead[h], row, col);
            }
        }
        if (col0 < g.n) epi.end(st, row, col0);
    };

    if constexpr (!C::SPLIT) {
        if (warp >= 4) {
            int n = 0;
            for (int t = first; t < tiles; t += step, ++n) take_tile(t, n);
        }
    } else {
        // The tile's four runs of 32 columns are shared out among the CTAs of the cluster (two or four): each sends its
        // sums of the other CTAs' columns to them, into shared memory where the stages were (once every CTA's
        // products have read theirs), and takes its own columns through the epilogue. A column's 128 rows lie
        // together, so that a warp's lanes write and read 32 neighbours. One CTA taking the whole tile cost 5 us:
        // 192 KB into one SM.
        const bool mine = first < tiles && warp >= 4;
        const int per = 4 / share;                    // runs of a CTA
        const int own = per == 2 ? 2 * q + half : q;  // this warp's, if it has one
        const bool takes = mine && (per == 2 || half == (q & 1));
        float *partial = reinterpret_cast<float *>(tail - S * C::STAGE);  // [share - 1][per][32 columns][128 rows]
        int mt = 0, nt = 0;
        if (mine) tile_at(g, m_tiles, first, mt, nt);
        const int64_t row = (int64_t)mt * C::TM + w * 32 + lane, tile0 = (int64_t)nt * C::BN, col = tile0 + own * 32;
        typename Epi::State st;
        typename Epi::Ahead ahead;
        __syncwarp();
        if (mine) {
            epi.begin(st, row, col);
            if (takes && col < g.n) epi.fetch(st, ahead, col);
            if (epi.bias) {
                const int c = threadIdx.x - 128;
                if (c < C::BN) bias[c] = tile0 + c < g.n ? epi.bias[tile0 + c] : 0.0f;
                epilogue_sync();
            }
            failed = !__all_sync(0xffffffffu, mbar_wait(acc_full, 0, g, gave_up));
        }
        cluster_sync();
        const uint32_t at = tmem + ((uint32_t)(w * 32) << 16);
        uint32_t r[32];
        if (mine && !failed) {
            fence_after();
            const bool row_ok = row < (g.m_dev ? (int64_t)*g.m_dev : g.m);
#pragma unroll 1
            for (int i = half; i < 4; i += 2) {
                const int to = i / per;
                if (to == q) continue;
                __syncwarp();
                if (k_blocks > 0) {
                    tmem_load32(at + 32 * i, r);
                    tmem_wait(r);
                } else {  // a sum over nothing
#pragma unroll
                    for (int j = 0; j < 32; ++j) r[j] = 0u;
                }
                const int slot = (q < to ? q : q - 1) * per + (i - to * per);
                const uint32_t p = map_rank(smem_u32(partial), to) + 4u * (slot * 32 * C::BM + w * 32 + lane);
                if (row_ok)
#pragma unroll
                    for (int j = 0; j < 32; ++j)
                        asm volatile("st.shared::cluster.b32 [%0], %1;" ::"r"(p + 4u * j * C::BM), "r"(r[j]) : "memory");
            }
        }
        __syncwarp();
        cluster_sync();
        if (takes && !failed && col < g.n) {
            if (k_blocks > 0) {
                tmem_load32(at + 32 * own, r);
                tmem_wait(r);
            } else {
#pragma unroll
                for (int j = 0; j < 32; ++j) r[j] = 0u;
            }
            float2 v[16];
#pragma unroll
            for (int j = 0; j < 16; ++j) v[j] = make_float2(__uint_as_float(r[2 * j]), __uint_as_float(r[2 * j + 1]));
            for (int o = 0; o < share - 1; ++o) {
                const float *p = partial + ((o * per + own - q * per) * 32 * C::BM + w * 32 + lane);
#pragma unroll
                for (int j = 0; j < 16; ++j)
                    v[j] = __fadd2_rn(v[j], make_float2(p[2 * j * C::BM], p[(2 * j + 1) * C::BM]));
            }
            epi.columns(st, v, bias + own * 32, ahead, row, col);
            epi.end(st, row, col);
        }
    }
    __syncwarp();
    fence_before();
    __syncthreads();
    if constexpr (CTAS == 2) cluster_sync();
    fence_after();
    if (warp == 2) tmem_free<CTAS>(tmem, C::TMEM_COLS);
}

// Which tiles a product takes: pairs of 256 x 256, single CTAs of 128 x 128, or clusters of 2 or 4 CTAs that share a
// 128 x 128 tile's k. A block of 64 k costs a pair about 320 ns (its products) and a CTA 175 ns (bringing in the
// operands and issuing; narrower tiles cost as much), 220 where all SMs bring theirs in for long; handing sums over
// 1.5 us. The cheapest by waves * blocks wins:
// few large tiles leave SMs idle, small ones bring the operands in more often. Measured: [1024,4096]x[4096,4096]^T
// pairs 27 us, single CTAs 37; [4096,8192]x[8192,4096] pairs 187, single CTAs 205; [8 | 64 | 256,4096]x[4096,4096]^T single CTAs 13 to 18 us, clusters 8.2, 9.0, 12.3.
struct Tiles {
    int ctas, bn, ew, split;  // ew: columns of an epilogue thread
};
inline Tiles pick_tiles(int64_t m, int64_t n, int64_t k) {
    constexpr int sms = 148;  // a B200's: workspaces depend on the choice, which must not depend on the current device
    const int64_t blocks = (k + kBlockK - 1) / kBlockK;
    auto tiles_of = [&](int64_t tm, int64_t tn) { return (m + tm - 1) / tm * ((n + tn - 1) / tn); };
    auto waves = [](int64_t tiles, int64_t slots) { return (tiles + slots - 1) / slots; };
    const int64_t singles = tiles_of(128, 128);
    Tiles best{1, 128, 64, 1};
    const int64_t single_waves = waves(singles, sms);
    int64_t least = single_waves * blocks * (single_waves > 1 ? 220 : 175) + 1800;
    if (m > 128) {  // else half of each pair's rows would be empty
        const int64_t cost = waves(tiles_of(256, 256), sms / 2) * blocks * 320 + 2500;
        if (cost < least) {
            least = cost;
            best = {2, 256, 128, 1};
        }
    }
    for (int q = 2; q <= kMaxSplit; q *= 2) {
        if (singles * q > sms - 12 || blocks < 2 * q) continue;  // one wave: some SMs are left over by the clusters
        const int64_t cost = (blocks + q - 1) / q * 175 + 1800 + 1500;
        if (cost < least) {
            least = cost;
            best = {1, 128, 32, q};
        }
    }
    return best;
}

// Launches the product of a and b (already TMA-ready). With m_dev / k_dev, m and k are what they may reach.
template <class C, class Epi>
dnb_status launch_gemm(const Operand &a, const Operand &b, int dtype, int64_t m, int64_t n, int64_t k, const Epi &epi,
                       const DeviceState *ds, cudaStream_t s, const char *what, int split = 1,
                       const int *m_dev = nullptr, const int *k_dev = nullptr) {
    static std::atomic<int> opted[kMaxDevices];
    auto kernel = k_gemm<C, Epi>;
    if (!opted[ds->device].load(std::memory_order_acquire)) {
        DNB_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)C::SMEM));
        opted[ds->device].store(1, std::memory_order_release);
    }
    CUtensorMap ma, mb;
    // few rows: no more of A is brought in than there is (the tile's other rows hold what the memory held: their
    // products are never looked at)
    const int a_rows = !C::A_MN && C::CTAS == 1 && m < C::BM ? (int)((m + 7) / 8 * 8) : C::BM;
    if (C::A_MN) DNB_TRY(make_map(&ma, a.p, m, k, a.ld, 64, dtype, what));
    else DNB_TRY(make_map(&ma, a.p, k, m, a.ld, a_rows, dtype, what));
    if (C::B_MN) DNB_TRY(make_map(&mb, b.p, n, k, b.ld, 64, dtype, what));
    else DNB_TRY(make_map(&mb, b.p, k, n, b.ld, C::BROWS, dtype, what));
    GemmArgs g;
    g.m = m;
    g.n = n;
    g.k = k;
    const int64_t mt = (m + C::TM - 1) / C::TM, nt = (n + C::BN - 1) / C::BN;
    if (mt * nt > 0x3fffffffll) return fail(DNB_ERR_UNSUPPORTED, "%s: too many output tiles", what);
    g.m_tiles = (int)mt;
    g.n_tiles = (int)nt;
    g.k_blocks = (int)((k + kBlockK - 1) / kBlockK);
    g.band = 8;
    g.split = split;
    g.stage_bytes = (unsigned)(a_rows * kBlockK * 2 + C::B_BYTES);
    g.m_dev = m_dev;
    g.k_dev = k_dev;
    // fp32 accumulators; operand type; majors; n / 8; m / 16
    const unsigned t = dtype == DNB_BF16 ? 1u : 0u;
    g.idesc = (1u << 4) | (t << 7) | (t << 10) | ((C::A_MN ? 1u : 0u) << 15) | ((C::B_MN ? 1u : 0u) << 16) |
              ((unsigned)(C::BN / 8) << 17) | ((unsigned)(C::TM / 16) << 24);
    g.wait_ns = wait_limit_ns();
    g.error_word = ds->error_word;
    const int64_t slots = ds->sm_count / C::CTAS, tiles = mt * nt;
    cudaLaunchConfig_t cfg = {};
    const int cluster = C::SPLIT ? split : C::CTAS;
    cfg.gridDim = dim3((unsigned)(C::SPLIT ? tiles * split : (tiles < slots ? tiles : slots) * C::CTAS));
    cfg.blockDim = dim3(kGemmThreads);
    cfg.dynamicSmemBytes = C::SMEM;
    cfg.stream = s;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = (unsigned)cluster;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = cluster > 1 ? 1 : 0;
    DNB_CUDA(cudaLaunchKernelEx(&cfg, kernel, ma, mb, g, epi));
    return after_launch(s, what);
}

}  // namespace dnb
