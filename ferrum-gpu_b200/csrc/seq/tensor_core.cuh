// Fifth-generation tensor cores (tcgen05) for pairs of CTAs: descriptors, TMEM,
// tensor copies that complete on the leader's barriers, and the host's tensor
// maps. Every wait is bounded (tma_util.cuh); no copy uses cluster multicast.
#pragma once

#include <cuda.h>

#include "../tma_util.cuh"
#include "cross_entropy.cuh"

namespace ferrum {
namespace seq {

// ---------------------------------------------------------------- descriptors
// Shared-memory operand in 128-byte swizzled atoms of 8 rows of 128 bytes (1024
// bytes, so aligned).
// K-major: a row is 64 values of depth; the next 8 rows follow 1024 bytes on.
// MN-major: an atom's rows are 8 steps of depth, each of 64 values along M or
// N; the next 8 steps follow 1024 bytes on, the next 64 values `block` bytes on.
__device__ __forceinline__ uint64_t operand_desc(uint32_t addr, uint32_t block) {
  constexpr uint64_t kVersion = 1ull << 46, kSwizzle128 = 2ull << 61;
  return (uint64_t)((addr >> 4) & 0x3fff) | ((uint64_t)(block >> 4) << 16) |
         ((uint64_t)(1024 >> 4) << 32) | kVersion | kSwizzle128;
}

// Instruction: float32 accumulators, A and B of one 16-bit type, M x N.
template <class T>
constexpr uint32_t instruction_desc(int m, int n, bool a_mn, bool b_mn) {
  const uint32_t type = std::is_same<T, __nv_bfloat16>::value ? 1 : 0;
  return (1u << 4) | (type << 7) | (type << 10) | ((uint32_t)a_mn << 15) | ((uint32_t)b_mn << 16) |
         ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}

// ---------------------------------------------------------------- CTA pair
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::
                   : "memory");
}
__device__ __forceinline__ void fence_barrier_init() {
  asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
}
// The address of this CTA's shared variable in CTA `rank` of the cluster.
__device__ __forceinline__ uint32_t map_to_rank(const void* p, uint32_t rank) {
  uint32_t a;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(p)), "r"(rank));
  return a;
}
// Arrives on a barrier of either CTA. It orders no memory: what it announces are
// reads of TMEM, complete and fenced before it. (Released, it would wait for the
// warp's stores: 2 of 9 stalls an issue.)
__device__ __forceinline__ void arrive_at(uint32_t bar) {
  asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}

// Box (x, y) of a tensor map into this CTA's shared memory, its bytes counted by
// a barrier that may be the peer's.
__device__ __forceinline__ void pair_load(void* dst, const CUtensorMap* map, int32_t x, int32_t y,
                                          uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%2, %3}], [%4];" ::"r"(smem_u32(dst)),
      "l"(map), "r"(x), "r"(y), "r"(bar)
      : "memory");
}

__device__ __forceinline__ void map_prefetch(const CUtensorMap* map) {
  asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory");
}

// ---------------------------------------------------------------- TMEM
// All 512 columns of both CTAs; called by one whole warp of each.
__device__ __forceinline__ void tmem_alloc_pair(uint32_t* at) {
  asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(at))
               : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
}
__device__ __forceinline__ void tmem_free_pair(uint32_t base) {
  asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;" ::"r"(base));
}
__device__ __forceinline__ void tc_fence_before() {
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
}
__device__ __forceinline__ void tc_fence_after() {
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
}
// D (+)= A B over 16 steps of depth, both CTAs' halves.
__device__ __forceinline__ void mma_pair(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc,
                                         bool add) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)add)
      : "memory");
}
// Arrives on the barrier at this address in both CTAs when the products issued
// so far are done.
__device__ __forceinline__ void commit_pair(uint64_t* bar) {
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64"
      " [%0], %1;" ::"r"(smem_u32(bar)),
      "h"((uint16_t)3)
      : "memory");
}
// The same for one CTA alone: `COLS` columns of TMEM, a power of two from 32 on.
template <int COLS>
__device__ __forceinline__ void tmem_alloc(uint32_t* at) {
  asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(at)),
               "n"(COLS)
               : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
}
template <int COLS>
__device__ __forceinline__ void tmem_free(uint32_t base) {
  asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(base), "n"(COLS));
}
__device__ __forceinline__ void mma_one(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool add) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)add)
      : "memory");
}
__device__ __forceinline__ void commit_one(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(
                   smem_u32(bar))
               : "memory");
}
__device__ __forceinline__ void mbar_arrive(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}

// 32 columns from `at` on of this warp's 32 lanes, a lane a row. The warp is
// brought together first.
__device__ __forceinline__ void tmem_load32(uint32_t at, float (&v)[32]) {
  uint32_t* r = (uint32_t*)v;
  __syncwarp();
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
        "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]),
        "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]),
        "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(at));
}
// The same for 16 columns.
__device__ __forceinline__ void tmem_load16(uint32_t at, float (&v)[16]) {
  uint32_t* r = (uint32_t*)v;
  __syncwarp();
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
        "=r"(r[14]), "=r"(r[15])
      : "r"(at));
}
__device__ __forceinline__ void tmem_load_wait() {
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}

// ---------------------------------------------------------------- host
// Map of `rows` rows of `cols` 16-bit values, `ld` values apart, for boxes of 64
// values (128 bytes, swizzled) by `box_rows`.
cudaError_t tensor_map(CUtensorMap* map, bool bf16, const void* base, int64_t cols, int64_t rows,
                       int64_t ld, int box_rows);
// What a tensor map needs of an array: 16-byte rows.
inline bool mappable(const void* p, int64_t ld, int64_t cols) {
  return aligned(p, 16) && ld % 8 == 0 && ld >= cols && ld < ((int64_t)1 << 38);
}

}  // namespace seq
}  // namespace ferrum
