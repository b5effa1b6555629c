// PTX wrappers of the 5th-generation tensor cores (tcgen05, TMEM), their
// shared-memory operands and CTA pairs, shared by the kernels that use them.
#pragma once

#include <cuda.h>

#include <type_traits>

#include "async_copy.cuh"
#include "common.cuh"

namespace mb {

__device__ __forceinline__ void tma_store_3d(const CUtensorMap* map, const void* src, int c0,
                                             int c1, int c2) {
  asm volatile(
      "cp.async.bulk.tensor.3d.global.shared::cta.bulk_group [%0, {%1, %2, %3}], [%4];" ::"l"(
          reinterpret_cast<uint64_t>(map)),
      "r"(c0), "r"(c1), "r"(c2), "r"(smem_addr(src))
      : "memory");
  asm volatile("cp.async.bulk.commit_group;" ::: "memory");
}

__device__ __forceinline__ void tma_store_2d(const CUtensorMap* map, const void* src, int c0,
                                             int c1) {
  asm volatile(
      "cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%1, %2}], [%3];" ::"l"(
          reinterpret_cast<uint64_t>(map)),
      "r"(c0), "r"(c1), "r"(smem_addr(src))
      : "memory");
  asm volatile("cp.async.bulk.commit_group;" ::: "memory");
}

// Wait until at most N of this thread's bulk stores still read shared memory.
template <int N>
__device__ __forceinline__ void tma_store_wait_read() {
  asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(N) : "memory");
}

__device__ __forceinline__ void tma_store_wait_all() {
  asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
}

// 3-D tiled loads: {inner, outer, part} coordinates over an operand stored as
// [parts, outer, ld] (the part dimension has extent 1 for plain operands).
__device__ __forceinline__ void tma_load_3d(void* dst, const CUtensorMap* map, int c0, int c1,
                                            int c2, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(
          smem_addr(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(c2), "r"(smem_addr(bar))
      : "memory");
}

// Shared-memory matrix descriptor: K-major operand, 128-byte swizzle, rows of
// 128 bytes, 8-row groups 1024 bytes apart (the layout the TMA copy writes).
__device__ __forceinline__ uint64_t sw128_kmajor_desc(uint32_t saddr) {
  uint64_t d = 0;
  d |= uint64_t((saddr >> 4) & 0x3fffu);  // start address
  d |= uint64_t(1) << 16;                  // leading byte offset (16 B; unused for this layout)
  d |= uint64_t(1024 >> 4) << 32;          // stride byte offset: 8 rows x 128 B
  d |= uint64_t(1) << 46;                  // descriptor version
  d |= uint64_t(2) << 61;                  // 128-byte swizzle
  return d;
}

__device__ __forceinline__ void mma_f16(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc,
                                        uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d_tmem),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate));
}

// Arrive on `bar` once every MMA issued so far by this thread has completed.
__device__ __forceinline__ void mma_commit(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(
                   smem_addr(bar))
               : "memory");
}

__device__ __forceinline__ void tc_fence_before() {
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
}
__device__ __forceinline__ void tc_fence_after() {
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
}

// Issue a 32-column TMEM load of this warp's 32 lanes; complete it with tmem_wait_ld().
__device__ __forceinline__ void tmem_ld32_issue(uint32_t taddr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]),
        "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]),
        "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]),
        "=r"(r[31])
      : "r"(taddr));
}

__device__ __forceinline__ void tmem_wait_ld() {
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}

template <typename TOut>
__device__ __forceinline__ void store_row32(TOut* dst, const float (&v)[32], int valid,
                                            bool vec_ok) {
  if (vec_ok && valid == 32) {
    if constexpr (std::is_same<TOut, float>::value) {
#pragma unroll
      for (int q = 0; q < 8; ++q) {
        reinterpret_cast<float4*>(dst)[q] = make_float4(v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]);
      }
    } else {
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        uint32_t w[4];
#pragma unroll
        for (int h = 0; h < 4; ++h) {
          const float a = v[8 * q + 2 * h], b = v[8 * q + 2 * h + 1];
          if constexpr (std::is_same<TOut, __nv_bfloat16>::value) {
            const __nv_bfloat162 p = __floats2bfloat162_rn(a, b);
            w[h] = *reinterpret_cast<const uint32_t*>(&p);
          } else {
            const __half2 p = __floats2half2_rn(a, b);
            w[h] = *reinterpret_cast<const uint32_t*>(&p);
          }
        }
        reinterpret_cast<uint4*>(dst)[q] = make_uint4(w[0], w[1], w[2], w[3]);
      }
    }
    return;
  }
  // unrolled with a predicate per element: a loop bounded by `valid` would
  // index v at run time and move it (and every chunk's values) to local memory
#pragma unroll
  for (int j = 0; j < 32; ++j) {
    if (j < valid) {
      if constexpr (std::is_same<TOut, float>::value) dst[j] = v[j];
      else if constexpr (std::is_same<TOut, __nv_bfloat16>::value) dst[j] = __float2bfloat16_rn(v[j]);
      else dst[j] = __float2half_rn(v[j]);
    }
  }
}

// One lane's 32 values of output row r (a 32-column chunk) into a staging slot
// of 32 rows x 128 bytes laid out as the bulk tensor store expects with the
// 128-byte swizzle: 16-byte chunk q of row r sits at chunk q ^ (r & 7), so the
// 32 lanes of a warp writing their rows hit distinct banks. fp32 chunks fill a
// row; 16-bit chunks fill half `h` of it (two chunks per store, so every
// store writes whole 128-byte lines).
template <typename TOut>
__device__ __forceinline__ void stage_row32(uint8_t* slot, int r, int h, const float (&v)[32]) {
  if constexpr (std::is_same<TOut, float>::value) {
#pragma unroll
    for (int q = 0; q < 8; ++q) {
      const int pq = q ^ (r & 7);
      *reinterpret_cast<float4*>(slot + r * 128 + pq * 16) =
          make_float4(v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]);
    }
  } else {
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      uint32_t w[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float a = v[8 * q + 2 * e], b = v[8 * q + 2 * e + 1];
        if constexpr (std::is_same<TOut, __nv_bfloat16>::value) {
          const __nv_bfloat162 p = __floats2bfloat162_rn(a, b);
          w[e] = *reinterpret_cast<const uint32_t*>(&p);
        } else {
          const __half2 p = __floats2half2_rn(a, b);
          w[e] = *reinterpret_cast<const uint32_t*>(&p);
        }
      }
      const int pq = (4 * h + q) ^ (r & 7);
      *reinterpret_cast<uint4*>(slot + r * 128 + pq * 16) = make_uint4(w[0], w[1], w[2], w[3]);
    }
  }
}

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}

// Address in the cluster's shared window of `local` (a shared::cta address)
// as seen in CTA `rank` of the cluster.
__device__ __forceinline__ uint32_t cluster_addr(uint32_t local, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(local), "r"(rank));
  return r;
}

__device__ __forceinline__ void cluster_sync_all() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::
                   : "memory");
}

// Arrive once on the barrier at shared offset `bar` in both CTAs of the pair
// (one multicast commit) when every pair MMA issued so far by this thread has
// completed.
__device__ __forceinline__ void mma_commit_pair_both(uint64_t* bar) {
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64"
      " [%0], %1;" ::"r"(smem_addr(bar)),
      "h"(static_cast<uint16_t>(0x3))
      : "memory");
}

// Arrive once on the barrier at cluster address `bar_cluster` when every
// pair MMA issued so far by this thread has completed.
__device__ __forceinline__ void mma_commit_pair(uint32_t bar_cluster) {
  asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(
                   bar_cluster)
               : "memory");
}

__device__ __forceinline__ void mbar_arrive_cluster(uint32_t bar_cluster) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar_cluster)
               : "memory");
}

}  // namespace mb
