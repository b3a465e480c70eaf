// PTX wrappers of the dense kernels beyond moe_ptx.cuh: CTA pairs
// (cta_group::2), distributed shared memory, the 16-bit and block-scaled
// 4-bit MMA kinds, and 32-byte global accesses. Waits are those of
// moe_ptx.cuh: bounded, reporting through a status word.
#pragma once

#include <cstdint>
#include <cuda_runtime.h>

#include "moe_ptx.cuh"

namespace moe {

// ------------------------------------------------------------- clusters
__device__ __forceinline__ uint32_t cluster_cta_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}

__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// Only keeps the CTAs together (before one leaves that others may still
// reach): orders no memory, so it does not wait for the CTA's stores.
__device__ __forceinline__ void cluster_sync_relaxed() {
  asm volatile("barrier.cluster.arrive.relaxed.aligned;\n\tbarrier.cluster.wait.aligned;" ::: "memory");
}

// The address, in the cluster's shared window, of `addr` in CTA `rank`.
__device__ __forceinline__ uint32_t map_to_cta(uint32_t addr, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}

__device__ __forceinline__ float4 ld_cluster_f32x4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(addr)
               : "memory");
  return v;
}

// Arrives on a barrier of another CTA of the cluster, for the tensor memory
// that this warp has read (its loads are complete). Relaxed: a release would
// wait for the warp's stores to global memory, which nobody there reads
// (gradients at 128 tokens, H = 7168, I = 2048, 70 -> 57 us; 4-bit block at
// 4096 tokens 91 -> 84). Not for handing over anything that was stored.
__device__ __forceinline__ void mbar_arrive_cluster(uint32_t cluster_bar) {
  asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_bar) : "memory");
}

// mbar_wait for barriers that another CTA of the cluster arrives on.
__device__ __forceinline__ bool mbar_wait_cluster(uint32_t bar, uint32_t parity, volatile int* abort,
                                                  uint32_t* status, uint32_t why) {
  const uint64_t t0 = globaltimer_ns();
  uint32_t spins = 0;
  while (true) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(bar), "r"(parity)
        : "memory");
    if (ok) return true;
    if ((++spins & 31u) == 0u) {
      if (*abort) return false;
      if (globaltimer_ns() - t0 > kWaitBudgetNs) {
        atomicOr(status, why);
        *abort = 1;
        return false;
      }
    }
  }
}

// One lane of a converged warp, the same one every time.
__device__ __forceinline__ bool elect_lane() {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(r));
  return r != 0;
}

// mbar_wait by a whole warp, with one answer for all lanes. The producer and
// MMA warps run their loops with all lanes and let one lane issue, so loop
// counters, addresses and descriptors stay in uniform registers, from which
// the instructions take them: with one lane in the loop an iteration cost
// 540 cycles of issue whatever the tile.
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity, volatile int* abort, uint32_t* status,
                                          uint32_t why) {
  return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort, status, why));
}

// After a wait that gave up: let this thread's own copies land before the
// CTA's shared memory goes away (they take microseconds; 2 ms bound).
__device__ __forceinline__ void drain_copies() {
  const uint64_t t0 = globaltimer_ns();
  while (globaltimer_ns() - t0 < 2000000ull) __nanosleep(1000);
}

// TMA load into this CTA whose completion counts on a barrier of either CTA
// of the pair (cluster address).
__device__ __forceinline__ void tma_load_2d_pair(uint32_t dst, const void* tmap, uint32_t cluster_bar, int x, int y) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2"
      " [%0], [%1, {%3, %4}], [%2];" ::"r"(dst),
      "l"(tmap), "r"(cluster_bar), "r"(x), "r"(y)
      : "memory");
}

// ------------------------------------------------------- tcgen05, CTA pair
__device__ __forceinline__ void tmem_alloc_pair(uint32_t dst_smem, uint32_t ncols) {
  asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(dst_smem), "r"(ncols)
               : "memory");
}

__device__ __forceinline__ void tmem_relinquish_pair() {
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
}

__device__ __forceinline__ void tmem_dealloc_pair(uint32_t taddr, uint32_t ncols) {
  asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(ncols) : "memory");
}

// Arrives on the barrier at this offset in the CTAs of `mask` once every
// tcgen05 operation this thread issued so far is done.
__device__ __forceinline__ void umma_commit_pair(uint32_t bar, uint32_t mask) {
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar),
      "h"(static_cast<uint16_t>(mask))
      : "memory");
}

// D[tmem] (+)= A * B^T, 16-bit operands (both bf16 or both fp16), fp32 sums.
template <int kCtas>
__device__ __forceinline__ void umma_f16(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc,
                                         uint32_t accumulate) {
  if constexpr (kCtas == 2)
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
        "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
        "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
        : "memory");
}

// D[tmem] (+)= (A, exponents sfa) * (B, exponents sfb)^T: e2m1 operands, one
// power-of-two exponent byte per 32 K elements, K = 64 per instruction.
template <int kCtas>
__device__ __forceinline__ void umma_mxf4(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc,
                                          uint32_t sfa, uint32_t sfb, uint32_t accumulate) {
  if constexpr (kCtas == 2)
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(
            d_tmem),
        "l"(adesc), "l"(bdesc), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(
            d_tmem),
        "l"(adesc), "l"(bdesc), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)
        : "memory");
}

// 512 bytes of shared memory (32 rows of 16 bytes) into four TMEM columns,
// repeated in the four 32-lane quarters; with a pair, in each CTA from its
// own shared memory.
template <int kCtas>
__device__ __forceinline__ void tmem_copy_scales(uint32_t taddr, uint64_t desc) {
  if constexpr (kCtas == 2)
    asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
  else
    asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
}

// ------------------------------------------------------------ descriptors
// Shared-memory matrix descriptors as a constant high word and a low word
// that holds the address: the issuing thread only adds to the low word (16
// bytes per count; addresses stay below 2^18, so no carry reaches the field
// above). Building each descriptor from its fields instead made the issuing
// thread the bound of the 4-bit GEMM (96 against 75 us of issue at 8192 x
// 4096 x 7168).
//   K-major, 128-byte swizzle: rows of 128 bytes, eight-row groups 1024 bytes
//     apart; a K step of 32 bytes is +2.
//   MN-major, 128-byte swizzle: 64 M (or N) elements of 16 bits are the 128
//     contiguous bytes, one K element per row, groups of eight K rows 1024
//     bytes apart, the next 64 elements 8192 bytes further on; a K step of 16
//     rows is +128.
//   Scale copy: 32 unswizzled rows of 16 bytes, eight-row groups of 128.
constexpr uint32_t kDescHiSw128 = (1024u >> 4) | (1u << 14) | (2u << 29);
constexpr uint32_t kDescHiPlain = (128u >> 4) | (1u << 14);

// An address in a cluster carries the CTA's rank above its offset, which is all
// that a descriptor takes; what is above would land in the next field, the
// distance to the next 64 elements.
__device__ __forceinline__ uint32_t desc_address(uint32_t addr) { return (addr & 0x3ffffu) >> 4; }
__device__ __forceinline__ uint32_t desc_lo_kmajor(uint32_t addr) { return desc_address(addr) | (1u << 16); }
__device__ __forceinline__ uint32_t desc_lo_mnmajor(uint32_t addr) {
  return desc_address(addr) | ((8192u >> 4) << 16);
}
__device__ __forceinline__ uint32_t desc_lo_scale(uint32_t addr) { return desc_address(addr) | ((128u >> 4) << 16); }

__device__ __forceinline__ uint64_t desc_of(uint32_t hi, uint32_t lo) {
  return (static_cast<uint64_t>(hi) << 32) | lo;
}

// Instruction descriptors. fp32 accumulator; operand type 1 = bf16, 0 = fp16;
// a set major bit means MN-major. N is a run-time value.
__host__ __device__ constexpr uint32_t idesc_f16(int m, int n, bool fp16, bool a_mn, bool b_mn) {
  const uint32_t type = fp16 ? 0u : 1u;
  return (1u << 4) | (type << 7) | (type << 10) | ((a_mn ? 1u : 0u) << 15) | ((b_mn ? 1u : 0u) << 16) |
         (static_cast<uint32_t>(n >> 3) << 17) | (static_cast<uint32_t>(m >> 4) << 24);
}

// e2m1 operands with power-of-two scales; `sf` is the byte (0 or 2) of each
// 32-bit scale word that the instruction's first 32 K elements use.
__host__ __device__ constexpr uint32_t idesc_mxf4(int m, int n, int sf) {
  return (static_cast<uint32_t>(sf) << 4) | (1u << 7) | (1u << 10) | (static_cast<uint32_t>(n >> 3) << 17) |
         (1u << 23) | (static_cast<uint32_t>(m >> 4) << 24) | (static_cast<uint32_t>(sf) << 29);
}

// ------------------------------------------------------- global accesses
__device__ __forceinline__ void st_global_32(void* p, const uint32_t* r) {
  asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "r"(r[0]), "r"(r[1]), "r"(r[2]),
               "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}

__device__ __forceinline__ void ld_global_32(uint32_t* r, const void* p) {
  asm volatile("ld.global.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
               : "l"(p)
               : "memory");
}

}  // namespace moe
