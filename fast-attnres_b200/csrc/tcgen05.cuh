// PTX wrappers of the fifth-generation tensor cores: tensor memory, shared-memory matrix
// descriptors, MMA issue, and the tiled TMA copies that feed them.
#pragma once

#include <cuda.h>

#include "tma_common.cuh"

namespace attnres_b200 {

// Loads a box into this CTA's shared memory.  In a pair (cta_group::2) the bytes may be counted on
// the other CTA's barrier, so `bar` is a cluster address there.
template <bool PAIR>
__device__ __forceinline__ void tensor_load_2d(uint32_t smem_dst, const CUtensorMap* map, int x,
                                               int y, uint32_t bar) {
  if constexpr (PAIR) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 "
        "[%0], [%1, {%2, %3}], [%4];" ::"r"(smem_dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(bar)
        : "memory");
  } else {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes "
        "[%0], [%1, {%2, %3}], [%4];" ::"r"(smem_dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(bar)
        : "memory");
  }
}

// The address that `smem` of this CTA has in CTA `rank` of the cluster.
__device__ __forceinline__ uint32_t cluster_address(uint32_t smem, uint32_t rank) {
  uint32_t address;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(address) : "r"(smem), "r"(rank));
  return address;
}

__device__ __forceinline__ void mbar_arrive_cluster(uint32_t bar) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}

__device__ __forceinline__ void cluster_barrier() {
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

__device__ __forceinline__ void tensor_store_2d(const CUtensorMap* map, int x, int y,
                                                uint32_t smem_src) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%1, %2}], [%3];" ::"l"(
                   reinterpret_cast<uint64_t>(map)),
               "r"(x), "r"(y), "r"(smem_src)
               : "memory");
  asm volatile("cp.async.bulk.commit_group;" ::: "memory");
}

// The issuing thread's stores have read their shared memory.
__device__ __forceinline__ void tensor_store_wait_read() {
  asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
}

__device__ __forceinline__ void prefetch_tensor_map(const CUtensorMap* map) {
  asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(map)) : "memory");
}

// All 512 columns of the SM's tensor memory, by one whole warp (of each CTA of a pair).
template <bool PAIR>
__device__ __forceinline__ void tmem_alloc_512(uint32_t* smem_slot) {
  if constexpr (PAIR) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(
                     smem_addr(smem_slot))
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  } else {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(
                     smem_addr(smem_slot))
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
}

template <bool PAIR>
__device__ __forceinline__ void tmem_dealloc_512(uint32_t tmem) {
  if constexpr (PAIR)
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
  else
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
}

__device__ __forceinline__ void tcgen05_fence_before() {
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
}
__device__ __forceinline__ void tcgen05_fence_after() {
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
}

// Arrives on `bar` (of both CTAs of a pair) once every MMA this thread issued before has finished.
template <bool PAIR>
__device__ __forceinline__ void tcgen05_commit(uint64_t* bar) {
  if constexpr (PAIR) {
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 "
        "[%0], %1;" ::"r"(smem_addr(bar)),
        "h"((unsigned short)3)
        : "memory");
  } else {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(
                     smem_addr(bar))
                 : "memory");
  }
}

// D[M x N] (+)= A[M x 16] B[N x 16]^T, operands 16-bit in shared memory, D FP32 in tensor memory.
// A CTA alone: M = 128.  A pair: M = 256, each CTA holds 128 rows of A and of D and half of B's.
template <bool PAIR>
__device__ __forceinline__ void tcgen05_mma_f16(uint32_t tmem_d, uint64_t desc_a, uint64_t desc_b,
                                                uint32_t instruction, bool accumulate) {
  if constexpr (PAIR) {
    asm volatile(
        "{\n"
        ".reg .pred p;\n"
        "setp.ne.b32 p, %4, 0;\n"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n"
        "}\n" ::"r"(tmem_d),
        "l"(desc_a), "l"(desc_b), "r"(instruction), "r"((uint32_t)accumulate)
        : "memory");
  } else {
    asm volatile(
        "{\n"
        ".reg .pred p;\n"
        "setp.ne.b32 p, %4, 0;\n"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n"
        "}\n" ::"r"(tmem_d),
        "l"(desc_a), "l"(desc_b), "r"(instruction), "r"((uint32_t)accumulate)
        : "memory");
  }
}

// Instruction descriptor of kind::f16: FP32 accumulator, both operands BF16 or both FP16, either
// of them with its M / N axis contiguous in shared memory instead of its K axis.
__host__ __device__ constexpr uint32_t mma_instruction(bool bf16, bool a_mn_major, bool b_mn_major, int m, int n) {
  return (1u << 4) | ((bf16 ? 1u : 0u) << 7) | ((bf16 ? 1u : 0u) << 10) |
         ((a_mn_major ? 1u : 0u) << 15) | ((b_mn_major ? 1u : 0u) << 16) |
         ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}

// Matrix descriptor of a 128-byte-swizzled operand built from 64 x 64-element boxes (8 KB each,
// rows of 128 bytes, eight-row groups of 1 KB).  K-major: rows are M / N, boxes follow one another
// along M / N, so the eight-row groups are 1 KB apart throughout.  MN-major: rows are K, the
// next 64 elements of M / N are the next box (the leading offset, 8 KB).
__device__ __forceinline__ uint64_t operand_descriptor(uint32_t smem) {
  constexpr uint64_t leading = 8192 >> 4, stride = 1024 >> 4, version = 1, swizzle_128b = 2;
  return (uint64_t)((smem >> 4) & 0x3fffu) | (leading << 16) | (stride << 32) | (version << 46) |
         (swizzle_128b << 61);
}

// 32 lanes x 32 columns: register i of a lane is column i of the lane's row.  The wait is part of
// the statement, so no use of the registers can move in front of it.
__device__ __forceinline__ void tmem_load_32(uint32_t tmem, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];\n"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
        "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]),
        "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]),
        "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(tmem)
      : "memory");
}

__device__ __forceinline__ void tmem_load_16(uint32_t tmem, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];\n"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
        "=r"(r[14]), "=r"(r[15])
      : "r"(tmem)
      : "memory");
}

}  // namespace attnres_b200
