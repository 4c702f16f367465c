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

template <bool NV>
__device__ __forceinline__ void mma4(uint32_t d, uint64_t a, uint64_t b, uint32_t id, uint32_t sfa, uint32_t sfb,
                                     uint32_t acc) {
  if constexpr (NV) {
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.u32 p, %6, 0;\n"
        " tcgen05.mma.cta_group::1.kind::mxf4nvf4.block_scale.scale_vec::4X [%0], %1, %2, %3, [%4], [%5], p;\n}\n"
        ::"r"(d), "l"(a), "l"(b), "r"(id), "r"(sfa), "r"(sfb), "r"(acc));
  } else {
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.u32 p, %6, 0;\n"
        " tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n}\n"
        ::"r"(d), "l"(a), "l"(b), "r"(id), "r"(sfa), "r"(sfb), "r"(acc));
  }
}

// one scale atom (32 rows x 16 bytes) -> 4 TMEM columns, repeated in the four lane quadrants.  Descriptor: no swizzle,
// 8-row groups 128 bytes apart
__device__ __forceinline__ void copy_scales(uint32_t tmem, uint32_t smem) {
  uint64_t d = (uint64_t)((smem >> 4) & 0x3FFF);
  d |= (uint64_t)1 << 16;
  d |= (uint64_t)(128 >> 4) << 32;
  d |= (uint64_t)1 << 46;
  asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(tmem), "l"(d));
}

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

}  // namespace fp4
}  // namespace g53
