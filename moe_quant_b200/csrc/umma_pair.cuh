// What kernels on the fifth-generation tensor cores share: fences, descriptors, and the pair of CTAs (cta_group::2) whose
// tensor cores work on one tile.
#pragma once

#include <cuda.h>

#include "common.cuh"
#include "mbarrier.cuh"

namespace mq {

// the driver's cuTensorMapEncodeTiled
typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                  const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                  CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
int get_encoder(EncodeTiledFn* out);

__device__ __forceinline__ void mbar_expect_tx(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ void fence_async_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// true in one lane of a converged warp, which the compiler then knows to be one: what it issues to the tensor core takes its operands from uniform
// registers as they are
__device__ __forceinline__ bool elect_one() {
  uint32_t yes;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(yes));
  return yes != 0;
}

// Matrix descriptor of a K-major tile with the 128-byte swizzle: rows of 128 bytes,
// groups of 8 rows 1024 bytes apart (stride byte offset), descriptor version 1.
__device__ __forceinline__ uint64_t kmajor_sw128_desc(uint32_t smem_addr) {
  uint64_t d = (uint64_t)((smem_addr & 0x3FFFFu) >> 4);
  d |= (uint64_t)1 << 16;            // leading byte offset: unused with a swizzle
  d |= (uint64_t)(1024 >> 4) << 32;  // stride byte offset
  d |= (uint64_t)1 << 46;            // version
  d |= (uint64_t)2 << 61;            // SWIZZLE_128B
  return d;
}

__device__ __forceinline__ uint32_t leader_addr(uint32_t local) {   // the same shared-memory location in the cluster's CTA 0
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(r) : "r"(local));
  return r;
}
__device__ __forceinline__ void set_in_cta(int* local, int rank, int v) {   // *local of the cluster's CTA `rank`
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem_u32(local)), "r"(rank));
  asm volatile("st.shared::cluster.s32 [%0], %1;" ::"r"(r), "r"(v) : "memory");
}
__device__ __forceinline__ void mbar_arrive_cluster(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// arrives on this barrier of both CTAs once the MMAs issued so far have completed
__device__ __forceinline__ void umma_commit_pair(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;"
               ::"r"(bar), "h"((uint16_t)3) : "memory");
}
// A wait that only the clock ends (a fault elsewhere does not): for what is still under way after a wait was given up.
__device__ __forceinline__ void mbar_drain(uint32_t bar, uint32_t parity) {
  const uint64_t t0 = global_ns();
  while (!mbar_try(bar, parity))
    if (global_ns() - t0 > 100000000ull) return;
}

__device__ __forceinline__ void tmem_alloc_pair(uint32_t dst_smem) {   // all 512 columns of both CTAs
  asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(dst_smem) : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_dealloc_pair(uint32_t taddr) {
  asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;" ::"r"(taddr) : "memory");
}

// What the two CTAs must know of each other before they leave: a wait of either was given up, slabs multiplied and accumulators handed over (set in
// both), slabs whose copies either producer has issued (the leader's).  With every wait satisfied nothing is under way at the end: the
// producers have seen the last commits on `empty` (await_stages), the epilogue warps all of those on `acc_full`, and the cluster barrier orders
// the arrivals on the leader's `acc_empty`.  After a wait that was given up what is under way comes to its end first (drain): the MMAs through
// their commits, of which the last use of every barrier is known, the copies through the leader's `full` (a stage that one
// producer alone has filled never completes; the copy lands long before that wait runs out).
struct PairEnd {
  int given_up, n_multiplied, n_accs, n_copied[2];
  __device__ __forceinline__ void reset() { given_up = n_multiplied = n_accs = n_copied[0] = n_copied[1] = 0; }
  __device__ __forceinline__ void give_up() {
    set_in_cta(&given_up, 0, 1);
    set_in_cta(&given_up, 1, 1);
  }
  __device__ __forceinline__ void multiplied(int slabs, int accs) {
    for (int c = 0; c < 2; ++c) {
      set_in_cta(&n_multiplied, c, slabs);
      set_in_cta(&n_accs, c, accs);
    }
  }
  __device__ __forceinline__ void copied_by(int rank, int slabs) { set_in_cta(&n_copied[rank], 0, slabs); }
  // by the producers' warps: the last use of every stage has been read (so its copies had landed) and its commit has arrived in this CTA
  static __device__ __forceinline__ bool await_stages(int stages, uint32_t empty0, int slabs, bool ok, int* fault, int code) {
    for (int j = slabs > stages ? slabs - stages : 0; j < slabs && ok; ++j) ok = mbar_wait(empty0 + 8 * (j % stages), (j / stages) & 1, fault, code);
    return ok;
  }
  __device__ __forceinline__ void drain(int stages, int rank, uint32_t full0, uint32_t empty0, uint32_t acc_full) const {
    for (int j = n_multiplied > stages ? n_multiplied - stages : 0; j < n_multiplied; ++j) mbar_drain(empty0 + 8 * (j % stages), (j / stages) & 1);
    for (int j = n_accs > 2 ? n_accs - 2 : 0; j < n_accs; ++j) mbar_drain(acc_full + 8 * (j & 1), (j >> 1) & 1);
    if (rank != 0) return;
    const int c = n_copied[0] > n_copied[1] ? n_copied[0] : n_copied[1];
    for (int j = c > stages ? c - stages : 0; j < c; ++j) mbar_drain(full0 + 8 * (j % stages), (j / stages) & 1);
  }
  template <int NST>
  static __device__ __forceinline__ bool await_stages(uint32_t empty0, int slabs, bool ok, int* fault, int code) {
    return await_stages(NST, empty0, slabs, ok, fault, code);
  }
  template <int NST>
  __device__ __forceinline__ void drain(int rank, uint32_t full0, uint32_t empty0, uint32_t acc_full) const {
    drain(NST, rank, full0, empty0, acc_full);
  }
};

}  // namespace mq
