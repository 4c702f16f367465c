// tcgen05 pieces of the 4-bit block-scaled products: instruction descriptor, mma, scale copies, bulk loads.
#pragma once
#include "fp4.cuh"
#include "tc05.cuh"

namespace g53 {
namespace fp4 {

// One thread of a converged warp, by elect.sync.  The roles that issue tcgen05 and bulk copies branch on this and not on a
// lane number: their operands are then known to be warp-uniform, where behind `lane == 0` each instruction carries code that
// makes them so (8 scale copies and 4 mma of N = 128: 953 clocks, 326 this way).
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}\n" : "=r"(p));
  return p != 0;
}

// instruction descriptor of the 4-bit block-scaled kinds: A, B e2m1, K-major; scale type (0 e4m3, 1 E8M0); M; N; scale
// data ids (which half of a 32-bit scale column the mma uses: 2X only)
__device__ __forceinline__ uint32_t idesc4(int m, int n, bool ue8m0, uint32_t sf_id) {
  return (sf_id << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(n >> 3) << 17) | ((ue8m0 ? 1u : 0u) << 23) |
         ((uint32_t)(m >> 7) << 27) | (sf_id << 29);
}

// G: CTAs that share the mma (cta_group)
template <bool NV, int G = 1>
__device__ __forceinline__ void mma4(uint32_t d, uint64_t a, uint64_t b, uint32_t id, uint32_t sfa, uint32_t sfb,
                                     uint32_t acc) {
  if constexpr (NV && G == 1) {
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.u32 p, %6, 0;\n"
        " tcgen05.mma.cta_group::1.kind::mxf4nvf4.block_scale.scale_vec::4X [%0], %1, %2, %3, [%4], [%5], p;\n}\n"
        ::"r"(d), "l"(a), "l"(b), "r"(id), "r"(sfa), "r"(sfb), "r"(acc));
  } else if constexpr (NV) {
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.u32 p, %6, 0;\n"
        " tcgen05.mma.cta_group::2.kind::mxf4nvf4.block_scale.scale_vec::4X [%0], %1, %2, %3, [%4], [%5], p;\n}\n"
        ::"r"(d), "l"(a), "l"(b), "r"(id), "r"(sfa), "r"(sfb), "r"(acc));
  } else if constexpr (G == 1) {
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.u32 p, %6, 0;\n"
        " tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n}\n"
        ::"r"(d), "l"(a), "l"(b), "r"(id), "r"(sfa), "r"(sfb), "r"(acc));
  } else {
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.u32 p, %6, 0;\n"
        " tcgen05.mma.cta_group::2.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n}\n"
        ::"r"(d), "l"(a), "l"(b), "r"(id), "r"(sfa), "r"(sfb), "r"(acc));
  }
}

// one scale atom (32 rows x 16 bytes) -> 4 TMEM columns, repeated in the four lane quadrants.  Descriptor: no swizzle,
// 8-row groups 128 bytes apart
template <int G = 1>
__device__ __forceinline__ void copy_scales(uint32_t tmem, uint32_t smem) {
  uint64_t d = (uint64_t)((smem >> 4) & 0x3FFF);
  d |= (uint64_t)1 << 16;
  d |= (uint64_t)(128 >> 4) << 32;
  d |= (uint64_t)1 << 46;
  if constexpr (G == 1) asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(tmem), "l"(d));
  else asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(tmem), "l"(d));
}

// ---- a pair of CTAs that share the mma: rank 0 issues, completions arrive on the same barrier of both
// (`both`: the two CTAs of the cluster)
__device__ __forceinline__ void commit_pair(uint64_t* b, uint16_t both = 3) {
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;"
      ::"r"(tc::saddr(b)), "h"(both) : "memory");
}
__device__ __forceinline__ void tmem_alloc_pair(uint32_t* dst, uint32_t cols) {
  asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(tc::saddr(dst)), "r"(cols));
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
}
__device__ __forceinline__ void tmem_free_pair(uint32_t base, uint32_t cols) {
  asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(base), "r"(cols));
}
// ---- barriers of a cluster
// arrival on the barrier of a CTA of the cluster by a thread that has written nothing itself (it passes on what a barrier
// told it): a cluster-scope release would cost it about 1000 clocks
__device__ __forceinline__ void signal_at(uint64_t* b, uint32_t rank) {
  uint32_t remote;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(tc::saddr(b)), "r"(rank));
  asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(remote) : "memory");
}
// tc::bar_wait with cluster-scope acquire, for barriers that another CTA arrives on (fail null: never cut short)
__device__ __forceinline__ bool bar_wait_cluster(uint64_t* b, uint32_t ph, volatile int* fail, int* err, int code) {
  for (uint32_t n = 0;; ++n) {
    uint32_t ok;
    asm volatile(
        "{\n .reg .pred p;\n mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n"
        " selp.u32 %0,1,0,p;\n}\n" : "=r"(ok) : "r"(tc::saddr(b)), "r"(ph) : "memory");
    if (ok) return true;
    if (fail && *fail) return false;
    if (n > (1u << 22)) {
      if (fail) *fail = 1;
      atomicExch(err, code);
      return false;
    }
  }
}
// (relaxed: what it orders is mbarrier initialisation, which has its own fence)
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }

__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
               ::"r"(tc::saddr(dst)), "l"(src), "r"(bytes), "r"(tc::saddr(bar)) : "memory");
}
// the same for data that is read once: first to leave L2
__device__ __forceinline__ void bulk_load_hint(void* dst, const void* src, uint32_t bytes, uint64_t* bar, uint64_t pol) {
  asm volatile(
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint [%0], [%1], %2, [%3], %4;"
      ::"r"(tc::saddr(dst)), "l"(src), "r"(bytes), "r"(tc::saddr(bar)), "l"(pol) : "memory");
}
__device__ __forceinline__ void bulk_expect(uint64_t* b, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(tc::saddr(b)), "r"(bytes) : "memory");
}

// an error word of the current device to *code behind the work on `st`, or (null) cleared
inline cudaError_t copy_error(const int& word, int* code, cudaStream_t st) {
  if (code) return cudaMemcpyFromSymbolAsync(code, word, sizeof(int), 0, cudaMemcpyDeviceToHost, st);
  static const int z = 0;
  return cudaMemcpyToSymbolAsync(word, &z, sizeof(int), 0, cudaMemcpyHostToDevice, st);
}

}  // namespace fp4
}  // namespace g53
