// Small-M product with 4-bit weights: Y[M, N] = X[M, K] @ W4[N, K]^T for M <= 16 rows (decode windows), W4A16.
//
// A decode projection reads every weight byte once, so HBM is the floor: 9/16 (17/32) byte per weight.  What stands in
// the way at 4 bits is the decode: 2 weights per byte have to become f16 operands, so at 6.5 TB/s an SM has to turn
// out 46 weights per clock.  e2m1 -> f16 is one cvt per two weights (measured 50 cvt per clock and SM on a B200, 23
// needed); the tensor core then multiplies (mma.m16n8k16, the weights as the 16-row operand).
//
// CTA: one 128-row block and one slice of the K tiles (a cluster of `CL` CTAs shares the block, each its own slice);
// persistent over row blocks.  Warp 8 streams the tile images (one cp.async.bulk of 16 KB of codes and one of 2 KB (1 KB)
// of scales per stage) into a ring, and before griddepcontrol.wait pulls its first tiles into L2.  Eight consumer warps: warp (rw, kh) takes rows 16 rw + {0..15} and the same + 64, and half kh of the tile's
// K, so each activation fragment it reads from shared memory serves two weight tiles.
//
// Activations.  bf16 does not fit f16's range, so each row is scaled by a power of two that puts the slice's largest
// magnitude into [2^14, 2^15); a value 2^-29 or more of the largest keeps all its bits, one below is off by at most
// 2^-39 of the largest (f16's subnormal step), 2^15 times less than the rounding of the fp32 sums it enters.  Converted once
// per CTA into shared memory in fragment order, and the row's power is put back on the fp32 sums.  The reduction
// dimension is permuted inside a tile in the same way for both operands.
//
// Scales.  nvfp4: a lane's 16 consecutive codes share one block, so the e4m3 scale multiplies the f16 weights (exact:
// 4 + 2 significant bits, within f16's range).  mxfp4's E8M0 scales exceed f16's range: there the four lanes of a row
// split one block of 32, two mma cover it, and the fp32 result is scaled as it is added to the sum.
//
// Sums of the two K halves meet in shared memory; the slices of a cluster are sent to the rank that owns the rows
// (distributed shared memory, one arrival per sender) and added in rank order: the result does not depend on timing.
// Two receive buffers alternate: a rank can only send block b + 2 after it received every rank's b + 1, which each sent
// after it had finished reading b.  Waits are bounded; one that runs out sets the error word and the CTA goes on without
// waiting, so every barrier is still reached.
#include <algorithm>
#include <cooperative_groups.h>
#include "fp4.cuh"
#include "launchers.h"
#include "tc05.cuh"

namespace cg = cooperative_groups;

namespace g53 {
namespace fp4 {

__device__ int g_gemv_err = 0;

constexpr int kCons = 8;                              // consumer warps
constexpr int kGemvThreads = (kCons + 1) * 32;
constexpr int kMaxSlice = 8;                          // K tiles whose activations a CTA holds at a time
constexpr uint32_t kGemvSpin = 1u << 22;
constexpr int kGemvErr = 0x6b41;

template <bool NV, int NT>
struct GemvSmem {
  static constexpr int kStage = kTileBytes + Fmt<NV>::kScaleBytes;
  static constexpr int kXTile = NT * 4096;            // activations of one K tile, f16 in fragment order
  static constexpr int kSum = 128 * NT * 8 * 4;       // fp32 sums of a block
  static constexpr int kRecv = 2 * 72 * NT * 8 * 4;   // receive buffer: CL x ceil(64 / CL) <= 70 row pairs
  static constexpr int kFixed = kSum + 2 * kRecv;     // sums of the upper K halves, two receive buffers
  // bytes for a slice of `slice` tiles and `stages` ring stages
  static constexpr int bytes(int slice, int stages) { return kFixed + slice * kXTile + stages * kStage + 128; }
};

__device__ __forceinline__ bool gv_wait(uint64_t* b, uint32_t ph, volatile int* stop, bool drain = false) {
  uint32_t n = 0;
  while (!tc::bar_try(b, ph)) {
    if (!drain && *stop) return false;
    if (++n > kGemvSpin) {
      *stop = 1;
      atomicExch(&g_gemv_err, kGemvErr);
      return false;
    }
    if (n > 64) __nanosleep(32);
  }
  return true;
}
// wait on a barrier that other CTAs of the cluster arrive on, with cluster-scope acquire
__device__ __forceinline__ bool gv_wait_cluster(uint64_t* b, uint32_t ph, volatile int* stop) {
  for (uint32_t n = 0;; ++n) {
    uint32_t ok;
    asm volatile(
        "{\n .reg .pred p;\n mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n"
        " selp.u32 %0,1,0,p;\n}\n" : "=r"(ok) : "r"(tc::saddr(b)), "r"(ph) : "memory");
    if (ok) return true;
    if (*stop) return false;
    if (n > kGemvSpin) {
      *stop = 1;
      atomicExch(&g_gemv_err, kGemvErr + 1);
      return false;
    }
  }
}
__device__ __forceinline__ void gv_bulk(void* dst, const void* src, uint32_t bytes, uint64_t* bar, uint64_t pol) {
  asm volatile(
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint [%0], [%1], %2, [%3], %4;"
      ::"r"(tc::saddr(dst)), "l"(src), "r"(bytes), "r"(tc::saddr(bar)), "l"(pol) : "memory");
}
__device__ __forceinline__ void gv_prefetch(const void* src, uint32_t bytes) {
  asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void gv_expect(uint64_t* b, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(tc::saddr(b)), "r"(bytes) : "memory");
}
__device__ __forceinline__ void gv_sync() { asm volatile("bar.sync 1, 256;" ::: "memory"); }   // the consumer warps

// f16 mma without an accumulator input
__device__ __forceinline__ void mma_f16_zero(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};\n"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
}

__device__ __forceinline__ uint32_t hmul2u(uint32_t a, uint32_t s) {
  const __half2 r = __hmul2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&s));
  return *reinterpret_cast<const uint32_t*>(&r);
}

// blocks: row blocks; per: K tiles of a slice; stages: ring depth; clusters: persistent clusters
struct GemvPlan {
  int blocks, KT, per, pass, stages, clusters, CL;
};

template <bool NV, int NT>
__global__ void __launch_bounds__(kGemvThreads, 2) fp4_gemv_kernel(Fp4GemvArgs p, GemvPlan pl) {
  using SM = GemvSmem<NV, NT>;
  constexpr int kStage = SM::kStage;
  extern __shared__ __align__(128) uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t full[8], empty[8], recv_bar[2];
  __shared__ float xpow[16];
  __shared__ int stop_s;
  volatile int* stop = &stop_s;
  uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 127) & ~uintptr_t(127));
  uint8_t* xs = ring + pl.stages * kStage;
  float* upper = reinterpret_cast<float*>(xs + pl.pass * SM::kXTile);   // [NT][128][8] sums of the upper K halves
  float* recv = upper + SM::kSum / 4;                                   // [2][kRecv]

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int CL = pl.CL;
  const int rank = CL > 1 ? (int)blockIdx.x % CL : 0, cid = (int)blockIdx.x / CL;
  const int t_lo = rank * pl.per, t_hi = min(pl.KT, t_lo + pl.per);
  const int nt_k = max(0, t_hi - t_lo);               // K tiles of this CTA
  // rows of a block that this rank finishes: pairs (j, j + 64), j in [j_lo, j_hi)
  const int j_per = (64 + CL - 1) / CL;
  const int j_lo = min(64, rank * j_per), j_hi = min(64, j_lo + j_per);

  if (threadIdx.x == 0) {
    for (int s = 0; s < pl.stages; ++s) {
      tc::bar_init(&full[s], 1);
      tc::bar_init(&empty[s], kCons);
    }
    tc::bar_init(&recv_bar[0], CL > 1 ? CL - 1 : 1);
    tc::bar_init(&recv_bar[1], CL > 1 ? CL - 1 : 1);
    stop_s = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (CL > 1) cg::this_cluster().sync();
  else __syncthreads();
  pdl_trigger();

  if (warp == kCons) {
    if (lane == 0) {
      const uint64_t pol = l2_evict_first_policy();
      uint32_t it = 0;
      bool ok = true;
      // before the wait for the previous kernel only a prefetch into L2: these weights may be what it is writing
      for (int t = t_lo; t < t_hi && t < t_lo + 8 && cid < pl.blocks; ++t) {
        const int64_t tile = (int64_t)cid * pl.KT + t;
        gv_prefetch(p.codes + tile * kTileBytes, kTileBytes);
        gv_prefetch(p.scales + tile * Fmt<NV>::kScaleBytes, Fmt<NV>::kScaleBytes);
      }
      pdl_wait();
      for (int nb = cid; nb < pl.blocks && ok; nb += pl.clusters) {
        const int64_t base = (int64_t)nb * pl.KT;
        for (int t = t_lo; t < t_hi; ++t, ++it) {
          const int s = it % pl.stages;
          const uint32_t round = it / pl.stages;
          if (round > 0 && !gv_wait(&empty[s], (round - 1) & 1, stop)) { ok = false; break; }
          gv_expect(&full[s], kStage);
          uint8_t* dst = ring + s * kStage;
          gv_bulk(dst, p.codes + (base + t) * kTileBytes, kTileBytes, &full[s], pol);
          gv_bulk(dst + kTileBytes, p.scales + (base + t) * Fmt<NV>::kScaleBytes, Fmt<NV>::kScaleBytes, &full[s], pol);
        }
      }
      if (!ok) {
        // stopped: the copies in flight have to land before the CTA ends (bounded)
        const uint32_t first = it > (uint32_t)pl.stages ? it - pl.stages : 0;
        for (uint32_t j = first; j < it; ++j) gv_wait(&full[j % pl.stages], (j / pl.stages) & 1, stop, true);
      }
    }
    __syncwarp();
  } else {
    const int g = lane >> 2, q = lane & 3;
    const int rw = warp & 3, kh = warp >> 2;
    pdl_wait();

    // activations of `n` tiles from tile t0 on -> xs: warp w converts rows w, w + 8
    auto load_x = [&](int t0, int n) {
#pragma unroll
      for (int i = 0; i < NT; ++i) {
        const int m = warp + i * 8;
        if (m >= p.M) break;
        const __nv_bfloat16* xr = p.x + (int64_t)m * p.ldx;
        uint4 v[kMaxSlice];
        uint32_t amax = 0;
#pragma unroll
        for (int t = 0; t < kMaxSlice; ++t) {
          v[t] = make_uint4(0, 0, 0, 0);
          const int k = (t0 + t) * kTileK + lane * 8;
          if (t < n && k < p.K) {
            if (p.xvec) {
              v[t] = *reinterpret_cast<const uint4*>(xr + k);
            } else {
              uint32_t u[4];
#pragma unroll
              for (int e = 0; e < 4; ++e)
                u[e] = (uint32_t)reinterpret_cast<const uint16_t*>(xr)[k + 2 * e] |
                       ((uint32_t)reinterpret_cast<const uint16_t*>(xr)[k + 2 * e + 1] << 16);
              v[t] = make_uint4(u[0], u[1], u[2], u[3]);
            }
          }
          const uint32_t u[4] = {v[t].x, v[t].y, v[t].z, v[t].w};
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const uint32_t a = (u[e] & 0x7fffu) << 16, b = u[e] & 0x7fff0000u;
            amax = max(amax, max(a < kInfBits ? a : 0u, b < kInfBits ? b : 0u));
          }
        }
        amax = __reduce_max_sync(0xffffffffu, amax);
        // exponent to take out: largest finite magnitude -> [2^14, 2^15); infinities and NaN pass through f16 as such
        const int e = max((int)(amax >> 23) - 127 - 14, -112);
        const float dn = pow2i(-e);
        if (lane == 0) xpow[m] = pow2i(e);
#pragma unroll
        for (int t = 0; t < kMaxSlice; ++t) {
          if (t >= n) break;
          const uint32_t u[4] = {v[t].x, v[t].y, v[t].z, v[t].w};
          uint32_t o[4];
#pragma unroll
          for (int c = 0; c < 4; ++c)
            o[c] = f32x2_to_f16x2(__uint_as_float(u[c] << 16) * dn, __uint_as_float(u[c] & 0xffff0000u) * dn);
          // lane holds k = 8 * lane .. + 7 of the tile: 32-chunk c = lane / 4, word w = lane % 4
          const int c = lane >> 2, w = lane & 3;
          // nvfp4: fragment (kh = c & 1, word w) of lane q = c / 2;  mxfp4: fragment c of lane q = w
          const int frag = NV ? (c & 1) * 4 + w : c;
          const int fq = NV ? c >> 1 : w;
          *reinterpret_cast<uint4*>(xs + t * SM::kXTile + (i * 8 + frag) * 512 + (warp * 4 + fq) * 16) =
              make_uint4(o[0], o[1], o[2], o[3]);
        }
      }
    };

    if (nt_k <= pl.pass) {
      load_x(t_lo, nt_k);
      gv_sync();
    }
    uint32_t it = 0, blk = 0;
    bool dead = false;
    for (int nb = cid; nb < pl.blocks; nb += pl.clusters, ++blk) {
      float sum[2][NT][4];
#pragma unroll
      for (int a = 0; a < 2; ++a)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) sum[a][n][e] = 0.f;

      for (int t0 = 0; t0 < nt_k; t0 += pl.pass) {
        const int n_t = min(pl.pass, nt_k - t0);
        if (nt_k > pl.pass) {                          // activations do not fit at once: the next part
          gv_sync();
          load_x(t_lo + t0, n_t);
          gv_sync();
        }
        float acc[2][NT][4];
#pragma unroll
        for (int a = 0; a < 2; ++a)
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[a][n][e] = 0.f;
        for (int t = 0; t < n_t; ++t, ++it) {
          const int s = it % pl.stages;
          if (!dead) {
            const bool ok = gv_wait(&full[s], (it / pl.stages) & 1, stop);
            dead = !__all_sync(0xffffffffu, ok);
          }
          if (!dead) {
            const uint8_t* cs = ring + s * kStage;
            const uint8_t* ss = cs + kTileBytes;
            const uint8_t* xt = xs + t * SM::kXTile + kh * 4 * 512 + lane * 16;
            const int R0 = rw * 16 + g;                // rows R0, R0 + 64, R0 + 8, R0 + 72
            if constexpr (NV) {
              // lane q: 16-byte chunk 2q + kh of each row = blocks (2 kh, 2 kh + 1) of atom q
              uint4 w4[4];
              uint32_t sc[4];
#pragma unroll
              for (int a = 0; a < 2; ++a) {
                const int R = R0 + a * 8;
                w4[2 * a] = *reinterpret_cast<const uint4*>(cs + chunk_off(R, 2 * q + kh));
                w4[2 * a + 1] = *reinterpret_cast<const uint4*>(cs + chunk_off(R + 64, 2 * q + kh));
                const uint8_t* sp = ss + q * 512 + (R & 31) * 16 + (R >> 5) * 4 + kh * 2;
                sc[2 * a] = e4m3x2_to_f16x2(*reinterpret_cast<const uint16_t*>(sp));
                sc[2 * a + 1] = e4m3x2_to_f16x2(*reinterpret_cast<const uint16_t*>(sp + 8));
              }
#pragma unroll
              for (int w = 0; w < 4; ++w) {
                uint4 xb[NT];
#pragma unroll
                for (int n = 0; n < NT; ++n) xb[n] = *reinterpret_cast<const uint4*>(xt + n * 4096 + w * 512);
#pragma unroll
                for (int a = 0; a < 2; ++a) {
                  uint32_t lo[4], hi[4];
                  const uint32_t wl = w == 0 ? w4[2 * a].x : w == 1 ? w4[2 * a].y : w == 2 ? w4[2 * a].z : w4[2 * a].w;
                  const uint32_t wh = w == 0 ? w4[2 * a + 1].x
                                             : w == 1 ? w4[2 * a + 1].y : w == 2 ? w4[2 * a + 1].z : w4[2 * a + 1].w;
                  e2m1x8_to_f16(wl, lo);
                  e2m1x8_to_f16(wh, hi);
                  const uint32_t sl = __byte_perm(sc[2 * a], 0, w < 2 ? 0x1010 : 0x3232);
                  const uint32_t sh = __byte_perm(sc[2 * a + 1], 0, w < 2 ? 0x1010 : 0x3232);
#pragma unroll
                  for (int e = 0; e < 4; ++e) {
                    lo[e] = hmul2u(lo[e], sl);
                    hi[e] = hmul2u(hi[e], sh);
                  }
                  const uint32_t a0[4] = {lo[0], hi[0], lo[1], hi[1]}, a1[4] = {lo[2], hi[2], lo[3], hi[3]};
#pragma unroll
                  for (int n = 0; n < NT; ++n) {
                    mma_f16_16816(acc[a][n], a0, xb[n].x, xb[n].y);
                    mma_f16_16816(acc[a][n], a1, xb[n].z, xb[n].w);
                  }
                }
              }
            } else {
              // chunks 4 kh .. 4 kh + 3 (one block each): lane q takes word q of the chunk
              uint32_t sc[4];
#pragma unroll
              for (int a = 0; a < 2; ++a) {
                const int R = R0 + a * 8;
                const uint8_t* sp = ss + kh * 512 + (R & 31) * 16 + (R >> 5) * 4;
                sc[2 * a] = *reinterpret_cast<const uint32_t*>(sp);
                sc[2 * a + 1] = *reinterpret_cast<const uint32_t*>(sp + 8);
              }
#pragma unroll
              for (int w = 0; w < 4; ++w) {
                uint4 xb[NT];
#pragma unroll
                for (int n = 0; n < NT; ++n) xb[n] = *reinterpret_cast<const uint4*>(xt + n * 4096 + w * 512);
#pragma unroll
                for (int a = 0; a < 2; ++a) {
                  const int R = R0 + a * 8, c = 4 * kh + w;
                  uint32_t lo[4], hi[4];
                  e2m1x8_to_f16(*reinterpret_cast<const uint32_t*>(cs + chunk_off(R, c) + q * 4), lo);
                  e2m1x8_to_f16(*reinterpret_cast<const uint32_t*>(cs + chunk_off(R + 64, c) + q * 4), hi);
                  const float sl = e8m0_to_f32((sc[2 * a] >> (8 * w)) & 0xffu);
                  const float sh = e8m0_to_f32((sc[2 * a + 1] >> (8 * w)) & 0xffu);
                  const uint32_t a0[4] = {lo[0], hi[0], lo[1], hi[1]}, a1[4] = {lo[2], hi[2], lo[3], hi[3]};
#pragma unroll
                  for (int n = 0; n < NT; ++n) {
                    float d[4];
                    mma_f16_zero(d, a0, xb[n].x, xb[n].y);
                    mma_f16_16816(d, a1, xb[n].z, xb[n].w);
                    acc[a][n][0] = fmaf(sl, d[0], acc[a][n][0]);
                    acc[a][n][1] = fmaf(sl, d[1], acc[a][n][1]);
                    acc[a][n][2] = fmaf(sh, d[2], acc[a][n][2]);
                    acc[a][n][3] = fmaf(sh, d[3], acc[a][n][3]);
                  }
                }
              }
            }
          }
          __syncwarp();
          if (lane == 0 && !dead) tc::bar_arrive(&empty[s]);
        }
        // the rows' powers of two back on (columns 2q, 2q + 1 are tokens)
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          const float f0 = xpow[n * 8 + 2 * q], f1 = xpow[n * 8 + 2 * q + 1];
#pragma unroll
          for (int a = 0; a < 2; ++a) {
            sum[a][n][0] = fmaf(acc[a][n][0], f0, sum[a][n][0]);
            sum[a][n][1] = fmaf(acc[a][n][1], f1, sum[a][n][1]);
            sum[a][n][2] = fmaf(acc[a][n][2], f0, sum[a][n][2]);
            sum[a][n][3] = fmaf(acc[a][n][3], f1, sum[a][n][3]);
          }
        }
      }

      // ---- upper K halves -> shared memory; the lower halves add them and hand the rows to their ranks
      auto slot = [&](int n, int r) { return (n * 128 + r) * 8 + 2 * q; };
      if (kh == 1) {
#pragma unroll
        for (int a = 0; a < 2; ++a)
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            const int r = rw * 16 + a * 8 + g;
            *reinterpret_cast<float2*>(upper + slot(n, r)) = make_float2(sum[a][n][0], sum[a][n][1]);
            *reinterpret_cast<float2*>(upper + slot(n, r + 64)) = make_float2(sum[a][n][2], sum[a][n][3]);
          }
      }
      gv_sync();
      float* rb = recv + (blk & 1) * (SM::kRecv / 4);
      if (kh == 0) {
#pragma unroll
        for (int a = 0; a < 2; ++a)
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            const int r = rw * 16 + a * 8 + g;         // 0..63
            const float2 u0 = *reinterpret_cast<const float2*>(upper + slot(n, r));
            const float2 u1 = *reinterpret_cast<const float2*>(upper + slot(n, r + 64));
            const float2 v0 = make_float2(sum[a][n][0] + u0.x, sum[a][n][1] + u0.y);
            const float2 v1 = make_float2(sum[a][n][2] + u1.x, sum[a][n][3] + u1.y);
            // receive buffer of the owner: [sender][pair row][half][NT][8]
            const int owner = r / j_per, jl = r - owner * j_per;
            float* dst = rb + ((rank * j_per + jl) * 2) * (NT * 8) + n * 8 + 2 * q;
            if (CL > 1 && owner != rank) dst = cg::this_cluster().map_shared_rank(dst, owner);
            *reinterpret_cast<float2*>(dst) = v0;
            *reinterpret_cast<float2*>(dst + NT * 8) = v1;
          }
      }
      if (CL > 1) {
        gv_sync();                                     // every row of this CTA is on its way
        if (warp == 0 && lane < CL && lane != rank) {
          // release at cluster scope orders the CTA's stores (seen through the barrier above) before the arrival
          asm volatile("fence.acq_rel.cluster;" ::: "memory");
          uint32_t remote;
          asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote)
                       : "r"(tc::saddr(&recv_bar[blk & 1])), "r"(lane));
          asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(remote) : "memory");
        }
        if (!dead) {
          const bool ok = gv_wait_cluster(&recv_bar[blk & 1], (blk >> 1) & 1, stop);
          dead = !__all_sync(0xffffffffu, ok);
        }
      } else {
        gv_sync();
      }

      // ---- finish rows j_lo..j_hi and + 64: element (row, token), consecutive threads on consecutive rows
      const int rows = j_hi - j_lo;
      const bool swi = p.mode == GEMV_SWIGLU;
      for (int e = threadIdx.x; e < rows * NT * 8 * (swi ? 1 : 2); e += kCons * 32) {
        const int jl = e % rows, rest = e / rows;
        const int tok = rest % (NT * 8), half = rest / (NT * 8);
        if (tok >= p.M) continue;
        float v = 0.f, u = 0.f;
        for (int c = 0; c < CL; ++c) {
          const float* src = rb + ((c * j_per + jl) * 2) * (NT * 8) + tok;
          v += src[half * NT * 8];
          if (swi) u += src[NT * 8];
        }
        const int r = nb * 128 + j_lo + jl + half * 64;
        if (swi) {
          const int col = nb * 64 + j_lo + jl;
          if (col >= p.width) continue;
          if (NV) {
            v *= p.row_scale[r];
            u *= p.row_scale[r + 64];
          }
          // written so that a NaN stays one
          v = v > p.limit ? p.limit : v;
          u = u > p.limit ? p.limit : u < -p.limit ? -p.limit : u;
          reinterpret_cast<__nv_bfloat16*>(p.y)[(int64_t)tok * p.ldy + col] = f2bf(siluf_(v) * u);
        } else {
          if (r >= p.N) continue;
          if (NV) v *= p.row_scale[r];
          const int64_t off = (int64_t)tok * p.ldy + r;
          if (p.mode == GEMV_BF16) {
            reinterpret_cast<__nv_bfloat16*>(p.y)[off] = f2bf(v);
          } else {
            float* y = reinterpret_cast<float*>(p.y) + off;
            *y = p.mode == GEMV_F32_ACC ? *y + v : v;
          }
        }
      }
    }
  }
  // no CTA leaves while another of its cluster may still write to it
  if (CL > 1) cg::this_cluster().sync();
}

// Shape of the launch.  Two CTAs per SM (the second hides the first one's start and reductions).  CL, the CTAs that
// share a row block, is the one that needs the fewest tile steps on the busiest CTA; ties go to the smaller, which
// sends less between CTAs.  The activations of a slice have to fit beside at least two ring stages.
template <bool NV, int NT>
static GemvPlan plan(int N, int K, int sms) {
  using SM = GemvSmem<NV, NT>;
  GemvPlan b{};
  b.blocks = (N + 127) / 128;
  b.KT = tiles_k(K);
  const int slots = 2 * sms;
  long best = -1;
  for (int cl = 1; cl <= 8 && cl <= b.KT; ++cl) {
    const int per = (b.KT + cl - 1) / cl;
    if ((b.KT + per - 1) / per != cl) continue;       // a CTA of the cluster would have no tile
    const int clusters = std::min(b.blocks, std::max(1, slots / cl));
    const long steps = (long)((b.blocks + clusters - 1) / clusters) * (per + 1);
    if (best < 0 || steps < best) {
      best = steps;
      b.CL = cl;
      b.per = per;
      b.clusters = clusters;
    }
  }
  b.pass = std::min(b.per, kMaxSlice);
  const int budget = 112 * 1024;
  b.stages = 8;
  while (b.stages > 2 && SM::bytes(b.pass, b.stages) > budget) --b.stages;
  return b;
}

template <bool NV, int NT>
static cudaError_t launch_gemv(const Fp4GemvArgs& p, int sms, cudaStream_t st) {
  const GemvPlan pl = plan<NV, NT>(p.mode == GEMV_SWIGLU ? ((p.width + 63) / 64) * 128 : p.N, p.K, sms);
  auto kern = fp4_gemv_kernel<NV, NT>;
  const int smem = GemvSmem<NV, NT>::bytes(pl.pass, pl.stages);
  cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(pl.clusters * pl.CL);
  cfg.blockDim = dim3(kGemvThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute at[2];
  int na = 0;
  if (pl.CL > 1) {
    at[na].id = cudaLaunchAttributeClusterDimension;
    at[na].val.clusterDim.x = pl.CL;
    at[na].val.clusterDim.y = 1;
    at[na].val.clusterDim.z = 1;
    ++na;
  }
  if (g53_pdl_on()) {
    at[na].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[na].val.programmaticStreamSerializationAllowed = 1;
    ++na;
  }
  cfg.attrs = at;
  cfg.numAttrs = na;
  return cudaLaunchKernelEx(&cfg, kern, p, pl);
}

}  // namespace fp4
}  // namespace g53

using namespace g53;

cudaError_t g53_fp4_gemv(const Fp4GemvArgs& p, cudaStream_t st) {
  if (p.M < 1 || p.M > 16 || p.N < 1 || p.K < 16 || p.K % (p.nv ? 16 : 32)) return cudaErrorInvalidValue;
  int dev = 0, sms = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess) e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  if (e != cudaSuccess) return e;
  if (p.nv) return p.M <= 8 ? fp4::launch_gemv<true, 1>(p, sms, st) : fp4::launch_gemv<true, 2>(p, sms, st);
  return p.M <= 8 ? fp4::launch_gemv<false, 1>(p, sms, st) : fp4::launch_gemv<false, 2>(p, sms, st);
}

cudaError_t g53_fp4_gemv_error(int* code) {
  const int z = 0;
  cudaError_t e = cudaMemcpyFromSymbol(code, fp4::g_gemv_err, sizeof(int));
  if (e == cudaSuccess && *code) e = cudaMemcpyToSymbol(fp4::g_gemv_err, &z, sizeof(int));
  return e;
}
