/*
 * Thin wrappers over the fifth-generation tensor cores: tensor memory, the asynchronous matrix
 * product that one thread issues, the tiled form of the bulk copy that feeds it, and the
 * descriptors of all three.  Everything is for 16-bit operands (both binary16 or both bfloat16)
 * with binary32 accumulators, operands staged in shared memory with the 128-byte swizzle.
 *
 * A pair of CTAs (a cluster of two) may work on one tile: each holds its own 128 rows of the
 * left operand and half of the right one, CTA 0 issues the products, and each CTA finds the
 * accumulators of its own rows in its own tensor memory.
 *
 * Shared-memory layouts, as the tiled copy writes them with CU_TENSOR_MAP_SWIZZLE_128B:
 *   operand whose contraction index is contiguous: boxes of 64 contraction elements (128 bytes) by
 *     R rows; groups of eight rows are 1024 bytes apart; the next 16 contraction elements
 *     start 32 bytes further.
 *   operand whose row (or column) index is contiguous: boxes of 64 of those by 64 contraction
 *     elements, 8192 bytes each; groups of eight contraction elements are 1024 bytes apart, so the
 *     next 16 start 2048 bytes further; the next 64 rows are the next box.
 */
#ifndef MSHADOW_GPU_TCGEN05_CUH_
#define MSHADOW_GPU_TCGEN05_CUH_

#include <cuda.h>

#include <cstdint>

#include "./runtime.h"
#include "./tma.cuh"

namespace mshadow {
namespace cuda {
namespace tc5 {

const uint32_t kBoxBytes = 64 * 64 * 2;  // a 64 x 64 box of 16-bit elements

// ---- descriptors ---------------------------------------------------------------------------

/*! \brief shared-memory descriptor, contraction index contiguous */
__device__ __forceinline__ uint64_t DescAlongK(uint32_t saddr) {
  return static_cast<uint64_t>((saddr >> 4) & 0x3fffu) | (uint64_t(1) << 16) | (uint64_t(1024 >> 4) << 32) |
         (uint64_t(1) << 46) | (uint64_t(2) << 61);
}
/*! \brief shared-memory descriptor, row (column) index contiguous, boxes of 64 x 64 one after the other */
__device__ __forceinline__ uint64_t DescAcrossK(uint32_t saddr) {
  return static_cast<uint64_t>((saddr >> 4) & 0x3fffu) | (uint64_t(kBoxBytes >> 4) << 16) |
         (uint64_t(1024 >> 4) << 32) | (uint64_t(1) << 46) | (uint64_t(2) << 61);
}
/*! \brief instruction descriptor: binary32 accumulators, `rows` x `cols` tile */
inline uint32_t InstrDesc(bool bf16, bool a_across, bool b_across, int rows, int cols) {
  const uint32_t t = bf16 ? 1u : 0u;
  return (1u << 4) | (t << 7) | (t << 10) | ((a_across ? 1u : 0u) << 15) | ((b_across ? 1u : 0u) << 16) |
         (static_cast<uint32_t>(cols >> 3) << 17) | (static_cast<uint32_t>(rows >> 4) << 24);
}

typedef CUresult (*EncodeTiledFn)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *,
                                  const cuuint64_t *, const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave,
                                  CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

/*! \brief cuTensorMapEncodeTiled, found through the runtime (the library does not link the driver) */
inline EncodeTiledFn EncodeTiled() {
  static EncodeTiledFn fn = [] {
    void *p = nullptr;
    cudaDriverEntryPointQueryResult found;
    MSHADOW_CUDA_CALL(cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &found));
    CHECK(p != nullptr && found == cudaDriverEntryPointSuccess) << "CUDA driver without cuTensorMapEncodeTiled";
    return reinterpret_cast<EncodeTiledFn>(p);
  }();
  return fn;
}

/*!
 * \brief map of a row-major matrix (`type`: kFloat32, kFloat16 or kBfloat16) whose copies move boxes of 128 bytes by
 *  `box_rows` rows; elements outside the matrix read as zero and are not written.  base and row pitch
 *  16-byte aligned.
 */
inline CUtensorMap MatrixMap(const void *base, int type, int64_t rows, int64_t cols, int64_t ld, int box_rows) {
  CUtensorMap map;
  const int elem = type == kFloat32 ? 4 : 2;
  const cuuint64_t extent[2] = {static_cast<cuuint64_t>(cols), static_cast<cuuint64_t>(rows)};
  const cuuint64_t pitch[1] = {static_cast<cuuint64_t>(ld) * elem};
  const cuuint32_t box[2] = {static_cast<cuuint32_t>(128 / elem), static_cast<cuuint32_t>(box_rows)};
  const cuuint32_t step[2] = {1, 1};
  const CUresult rc =
      EncodeTiled()(&map, type == kFloat32    ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                          : type == kBfloat16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                              : CU_TENSOR_MAP_DATA_TYPE_FLOAT16,
                    2, const_cast<void *>(base), extent, pitch, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                    CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  CHECK_EQ(static_cast<int>(rc), 0) << "CUDA: cuTensorMapEncodeTiled refused a matrix";
  return map;
}

// ---- cluster ---------------------------------------------------------------------------------

__device__ __forceinline__ uint32_t ClusterRank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void ClusterSync() {
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
/*! \brief address of the same shared-memory location in CTA `rank` of the cluster */
__device__ __forceinline__ uint32_t MapToRank(uint32_t saddr, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(saddr), "r"(rank));
  return r;
}
/*!
 * \brief one arrival on a barrier of any CTA of the cluster, without ordering memory: for handing back accumulators whose
 *  loads have completed (a releasing arrival waits for the warp's stores to global memory first)
 */
__device__ __forceinline__ void ArriveCluster(uint32_t cluster_addr) {
  asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}

// ---- tiled copies ----------------------------------------------------------------------------

__device__ __forceinline__ void PrefetchMap(const CUtensorMap *map) {
  asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory");
}
/*! \brief box at column x (a multiple of 8), row y; kCtas == 2: `bar` may be the other CTA's barrier */
template <int kCtas>
__device__ __forceinline__ void LoadBox(uint32_t dst, const CUtensorMap *map, int x, int y, uint32_t bar) {
  if (kCtas == 2) {
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, "
        "{%2, %3}], [%4];" ::"r"(dst),
        "l"(map), "r"(x), "r"(y), "r"(bar)
        : "memory");
  } else {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], "
        "[%4];" ::"r"(dst),
        "l"(map), "r"(x), "r"(y), "r"(bar)
        : "memory");
  }
}

/*! \brief box of shared memory to column x, row y of a matrix (parts outside it are left out); kAdd: added to what is there */
template <bool kAdd>
__device__ __forceinline__ void StoreBox(const CUtensorMap *map, int x, int y, uint32_t src) {
  if (kAdd) {
    asm volatile("cp.reduce.async.bulk.tensor.2d.global.shared::cta.add.tile.bulk_group [%0, {%1, %2}], [%3];" ::"l"(map),
                 "r"(x), "r"(y), "r"(src)
                 : "memory");
  } else {
    asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.tile.bulk_group [%0, {%1, %2}], [%3];" ::"l"(map), "r"(x),
                 "r"(y), "r"(src)
                 : "memory");
  }
  asm volatile("cp.async.bulk.commit_group;" ::: "memory");
}
/*! \brief this thread's stores have read their shared memory */
__device__ __forceinline__ void WaitStoresRead() { asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory"); }
/*! \brief this thread's stores have been written */
__device__ __forceinline__ void WaitStores() { asm volatile("cp.async.bulk.wait_group 0;" ::: "memory"); }

/*! \brief barrier of `threads` threads (whole warps), number `id` of 1 .. 15 */
__device__ __forceinline__ void NamedBarrier(int id, int threads) {
  asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory");
}
// ---- tensor memory and products ---------------------------------------------------------------

/*! \brief all 512 columns; executed by one whole warp (of both CTAs of a pair) */
template <int kCtas>
__device__ __forceinline__ void AllocTensorMemory(uint32_t *slot) {
  if (kCtas == 2) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(tma::SharedAddr(slot)) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
  } else {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(tma::SharedAddr(slot)) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
}
template <int kCtas>
__device__ __forceinline__ void FreeTensorMemory(uint32_t base) {
  if (kCtas == 2) {
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;" ::"r"(base));
  } else {
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(base));
  }
}
/*! \brief accumulators (+)= A . B over 16 contraction elements; issued by one thread */
template <int kCtas>
__device__ __forceinline__ void Multiply(uint32_t acc, uint64_t a, uint64_t b, uint32_t instr, bool add) {
  const uint32_t p = add ? 1u : 0u;
  if (kCtas == 2) {
    asm volatile(
        "{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\ntcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(acc),
        "l"(a), "l"(b), "r"(instr), "r"(p)
        : "memory");
  } else {
    asm volatile(
        "{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\ntcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(acc),
        "l"(a), "l"(b), "r"(instr), "r"(p)
        : "memory");
  }
}
/*! \brief one arrival on `bar` (of every CTA of the pair) when all products issued so far are done */
template <int kCtas>
__device__ __forceinline__ void CommitTo(uint64_t *bar) {
  if (kCtas == 2) {
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
            tma::SharedAddr(bar)),
        "h"(static_cast<uint16_t>(3))
        : "memory");
  } else {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(tma::SharedAddr(bar))
                 : "memory");
  }
}
__device__ __forceinline__ void FenceBefore() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void FenceAfter() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

/*! \brief starts reading 32 columns of the thread's own row (lane of its warp's quarter of tensor memory) */
__device__ __forceinline__ void LoadColumns(uint32_t addr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
        "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]),
        "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]),
        "=r"(r[30]), "=r"(r[31])
      : "r"(addr));
}
/*! \brief the same, 16 columns */
__device__ __forceinline__ void LoadColumns(uint32_t addr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(addr));
}
/*! \brief the loads above have arrived; `r` passes through so that no use of it moves above the wait */
__device__ __forceinline__ void WaitColumns(uint32_t (&r)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                 "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]),
                 "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]),
                 "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]),
                 "+r"(r[30]), "+r"(r[31])
               :
               : "memory");
}

__device__ __forceinline__ void WaitColumns(uint32_t (&r)[16]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                 "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])
               :
               : "memory");
}

// ---- two binary32 at a time --------------------------------------------------------------------

__device__ __forceinline__ uint64_t Pair(float lo, float hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ void Unpair(uint64_t p, float *lo, float *hi) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(*lo), "=f"(*hi) : "l"(p));
}
/*! \brief both sums, both products plus a third: each rounded as __fadd_rn and __fmaf_rn do, at twice their rate */
__device__ __forceinline__ uint64_t AddPair(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t FmaPair(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}

}  // namespace tc5
}  // namespace cuda
}  // namespace mshadow
#endif  // MSHADOW_GPU_TCGEN05_CUH_
