// Small-M product with 4-bit weights: Y[M, N] = X[M, K] @ W4[N, K]^T for M <= 32 rows of 16-bit activations (W4A16).
//
// A decode projection reads every weight byte once, so HBM is the floor: 9/16 (17/32) byte per weight.  Widening the
// weights to f16 operands on the CUDA cores cannot keep up with that (built first: 390 instructions per warp and 32 x 128
// weights, 2.7 TB/s), so the codes go to the block-scaled tensor cores as they are, as the 128-row operand of
// tcgen05.mma, and the activations are brought to 4 bits without losing them: each row is expanded into kTerms = 8 rows
//     x = sum_t Q(r_t),   r_0 = x,   r_{t+1} = r_t - Q(r_t)
// of the weights' own format, which become 8 of the mma's N columns.  The fp32 columns of a row are summed in the epilogue.
// Every term leaves at most 0.177 (nvfp4) or 1/4 (mxfp4, after the first) of what was there, block by block, so the sum
// of 8 is within 2^-19 (nvfp4) or 2^-15 (mxfp4) of a block's largest magnitude in the worst case; on normal activations
// the residue is 4e-10 of the row's norm, or zero: an element of bf16's 8 bits is used up after 2 bits a term.  The tensor
// core has the time: N = 64 (8 rows) costs 128 clocks per 128 x 256 tile of weights, HBM delivers one in 790 per SM.
//
// fp4_expand writes the expansion as a tile image (fp4.cuh), rows 8 m + t.  nvfp4: one power of two per row of x brings
// the block scales into e4m3's range, term t uses 2^-kOff[t] of it; the epilogue puts both back.
//
// fp4_skinny: a CTA takes a 128-row block of W and a slice of its K tiles; a cluster of CL CTAs shares a block, and
// clusters walk the blocks.  Warp 0 streams tiles of both operands into a ring (contiguous cp.async.bulk), warp 1 copies
// the scales to TMEM and issues the mma, warps 2-5 read the sums (a thread holds one weight row), send them to the rank of
// the cluster that owns the row (distributed shared memory, one arrival per sender) and finish the rows they own, adding
// in rank order: the result does not depend on timing.  Two receive buffers alternate: a rank can only send block b + 2
// after it received every rank's b + 1, which each sent after it had finished reading b.
//
// Before griddepcontrol.wait only prefetches into L2 are issued: the weights may be what the previous kernel writes.
// Waits are bounded; one that runs out sets the error word and the CTA goes on without waiting, so every barrier is
// still reached, copies and mma in flight are waited for (bounded) and the TMEM is freed.
#include <algorithm>
#include <cooperative_groups.h>
#include "fp4.cuh"
#include "fp4_tc.cuh"
#include "launchers.h"

namespace cg = cooperative_groups;

namespace g53 {
namespace fp4 {

__device__ int g_skinny_err = 0;

constexpr int kTerms = 8;
__host__ __device__ constexpr int term_off(int t) { return (5 * t) / 2; }     // 0 2 5 7 10 12 15 17
constexpr int kSkThreads = 192;
constexpr int kErrSk = 0x6b40;

// ------------------------------------------------------------------------------------------------------ expansion
// CTA: 128 blocks of 16 of one row (a thread each); nvfp4 reads the whole row for its maximum first.
template <bool NV>
__global__ void __launch_bounds__(128) fp4_expand_kernel(Fp4ExpandArgs p) {
  __shared__ uint32_t red[4];
  const int m = blockIdx.y, b = blockIdx.x * 128 + threadIdx.x;
  const int KT = tiles_k(p.K);
  const int nb = KT * 16, nk = p.K / 16;
  const uint16_t* x = reinterpret_cast<const uint16_t*>(p.x) + (int64_t)m * p.ldx;
  pdl_trigger();
  pdl_wait();
  uint32_t w[8];
  auto load = [&](int blk) {
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = 0u;
    if (blk < nk) {
      if (p.vec) {
        const uint4 a = *reinterpret_cast<const uint4*>(x + (int64_t)blk * 16);
        const uint4 c = *reinterpret_cast<const uint4*>(x + (int64_t)blk * 16 + 8);
        w[0] = a.x; w[1] = a.y; w[2] = a.z; w[3] = a.w;
        w[4] = c.x; w[5] = c.y; w[6] = c.z; w[7] = c.w;
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          w[i] = (uint32_t)x[(int64_t)blk * 16 + 2 * i] | ((uint32_t)x[(int64_t)blk * 16 + 2 * i + 1] << 16);
      }
    }
  };
  float scale = 1.f;
  if constexpr (NV) {
    uint32_t am = 0;
    for (int blk = threadIdx.x; blk < nk; blk += 128) {
      load(blk);
#pragma unroll
      for (int i = 0; i < 8; ++i) am = max(am, max((w[i] & 0x7fffu) << 16, w[i] & 0x7fff0000u));
    }
    am = __reduce_max_sync(0xffffffffu, am);
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = am;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 4; ++i) am = max(am, red[i]);
    const int k = am >= kInfBits ? 0 : nv_row_exp(am);
    scale = pow2i(-k);
    if (b == 0) p.factor[m] = am >= kInfBits ? __uint_as_float(0x7fc00000u) : pow2i(k);
  } else if (b == 0) {
    p.factor[m] = 1.f;
  }
  load(b);
  float r[16];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    r[2 * i] = __uint_as_float(w[i] << 16) * scale;
    r[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u) * scale;
  }
  const int kt = b >> 4, kb = b & 15;
#pragma unroll
  for (int t = 0; t < kTerms; ++t) {
    const int row = m * kTerms + t;                  // row of the expansion, < 256
    const int rr = row % kTileRows;
    const int64_t tile = (int64_t)(row / kTileRows) * KT + kt;
    if (NV && t > 0) {
      const float up = pow2i(term_off(t) - term_off(t - 1));
#pragma unroll
      for (int i = 0; i < 16; ++i) r[i] *= up;
    }
    uint32_t am = 0;
#pragma unroll
    for (int i = 0; i < 16; ++i) am = max(am, __float_as_uint(r[i]) & 0x7fffffffu);
    uint32_t sc;
    float s, inv;
    if constexpr (NV) {
      const __nv_fp8_e4m3 q(__uint_as_float(am) * 0.16666667f);      // any scale near a sixth does here
      sc = am >= kInfBits ? 0x7fu : q.__x;
      s = e4m3_to_f32(sc);
      inv = s > 0.f ? __frcp_rn(s) : 0.f;
    } else {
      am = max(am, __shfl_xor_sync(0xffffffffu, am, 1));
      sc = mx_scale(am);
      s = e8m0_to_f32(sc);
      inv = sc == 255u ? 0.f : pow2i(127 - (int)sc);
    }
    uint32_t code[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float f[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) f[i] = r[8 * h + i] * inv;
      code[h] = f32x8_to_e2m1(f);
      uint32_t o[4];
      e2m1x8_to_f16(code[h], o);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&o[i]));
        r[8 * h + 2 * i] = fmaf(-v.x, s, r[8 * h + 2 * i]);
        r[8 * h + 2 * i + 1] = fmaf(-v.y, s, r[8 * h + 2 * i + 1]);
      }
    }
    if (b >= nk) sc = 0u;
    constexpr int kStep = NV ? 1 : 2;
    uint32_t s4 = sc;
    s4 |= __shfl_down_sync(0xffffffffu, sc, kStep) << 8;
    s4 |= __shfl_down_sync(0xffffffffu, sc, 2 * kStep) << 16;
    s4 |= __shfl_down_sync(0xffffffffu, sc, 3 * kStep) << 24;
    if (b < nb) {
      *reinterpret_cast<uint2*>(p.codes + tile * kTileBytes + chunk_off(rr, kb >> 1) + (kb & 1) * 8) =
          make_uint2(code[0], code[1]);
      if ((kb & (4 * kStep - 1)) == 0)
        *reinterpret_cast<uint32_t*>(p.scales + tile * Fmt<NV>::kScaleBytes + scale_off(rr, kb / kStep)) = s4;
    }
  }
}

// -------------------------------------------------------------------------------------------------------- product
// per: K tiles of a slice; stages: ring depth; clusters: persistent clusters; ncol: mma N
struct SkPlan {
  int blocks, KT, per, stages, clusters, CL, ncol, stage_bytes, mp;
};

__device__ __forceinline__ bool sk_wait(uint64_t* b, uint32_t ph, volatile int* stop, bool drain = false) {
  uint32_t n = 0;
  while (!tc::bar_try(b, ph)) {
    if (!drain && *stop) return false;
    if (++n > (1u << 22)) {
      *stop = 1;
      atomicExch(&g_skinny_err, kErrSk);
      return false;
    }
  }
  return true;
}
// wait on a barrier that other CTAs of the cluster arrive on, with cluster-scope acquire
__device__ __forceinline__ bool sk_wait_cluster(uint64_t* b, uint32_t ph, volatile int* stop) {
  for (uint32_t n = 0;; ++n) {
    uint32_t ok;
    asm volatile(
        "{\n .reg .pred p;\n mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n"
        " selp.u32 %0,1,0,p;\n}\n" : "=r"(ok) : "r"(tc::saddr(b)), "r"(ph) : "memory");
    if (ok) return true;
    if (*stop) return false;
    if (n > (1u << 22)) {
      *stop = 1;
      atomicExch(&g_skinny_err, kErrSk + 1);
      return false;
    }
  }
}
__device__ __forceinline__ void sk_sync() { asm volatile("bar.sync 1, 128;" ::: "memory"); }   // the epilogue warps
__device__ __forceinline__ void sk_prefetch(const void* src, uint32_t bytes) {
  asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(src), "r"(bytes) : "memory");
}

// WIDE: mma N up to 256 (17..32 rows), one CTA per SM; otherwise N <= 128 and two CTAs per SM
template <bool NV, bool WIDE>
__global__ void __launch_bounds__(kSkThreads, WIDE ? 1 : 2) fp4_skinny_kernel(Fp4SkinnyArgs p, SkPlan pl) {
  constexpr int kSB = Fmt<NV>::kScaleBytes;
  constexpr int kAtoms = kSB / 512;
  constexpr int kXB = WIDE ? 2 : 1;                   // 128-row blocks of the expansion
  constexpr uint32_t kCols = WIDE ? 512 : 256;        // TMEM columns: sums, scales of W, scales of X
  constexpr uint32_t kSfW = WIDE ? 256 : 128, kSfX = kSfW + 16;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t full[8], empty[8], recv_bar[2], tfull, tempty, drain;
  __shared__ uint32_t tmem_s;
  __shared__ int stop_s;
  volatile int* stop = &stop_s;
  uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  float* recv = reinterpret_cast<float*>(ring + pl.stages * pl.stage_bytes);   // [2][CL][mp][2][j_per]

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int CL = pl.CL;
  const int rank = CL > 1 ? (int)blockIdx.x % CL : 0, cid = (int)blockIdx.x / CL;
  const int t_lo = rank * pl.per, t_hi = min(pl.KT, t_lo + pl.per);
  // rows of a block that this rank finishes: pairs (j, j + 64), j in [j_lo, j_lo + rows)
  const int j_per = (64 + CL - 1) / CL;
  const int j_lo = min(64, rank * j_per), rows = min(64, j_lo + j_per) - j_lo;
  const int xrows = pl.ncol;                          // rows of the expansion that are fetched
  const int xb0 = min(xrows, 128) * 128, xb1 = WIDE ? max(0, xrows - 128) * 128 : 0;
  const int off_x = kTileBytes, off_sw = off_x + xrows * 128, off_sx = off_sw + kSB;

  if (threadIdx.x == 0) {
    for (int s = 0; s < pl.stages; ++s) {
      tc::bar_init(&full[s], 1);
      tc::bar_init(&empty[s], 1);
    }
    tc::bar_init(&recv_bar[0], CL > 1 ? CL - 1 : 1);
    tc::bar_init(&recv_bar[1], CL > 1 ? CL - 1 : 1);
    tc::bar_init(&tfull, 1);
    tc::bar_init(&tempty, 4);
    tc::bar_init(&drain, 1);
    stop_s = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) tc::tmem_alloc(&tmem_s, kCols);
  tc::fence_before();
  if (CL > 1) cg::this_cluster().sync();
  else __syncthreads();
  tc::fence_after();
  const uint32_t tmem = tmem_s;
  pdl_trigger();

  if (warp == 0) {
    if (elect_one()) {
      const uint64_t pol = l2_evict_first_policy();
      for (int t = t_lo; t < t_hi && t < t_lo + 8 && cid < pl.blocks; ++t) {
        const int64_t tile = (int64_t)cid * pl.KT + t;
        sk_prefetch(p.codes + tile * kTileBytes, kTileBytes);
        sk_prefetch(p.scales + tile * kSB, kSB);
      }
      pdl_wait();
      uint32_t it = 0;
      bool ok = true;
      for (int nb = cid; nb < pl.blocks && ok; nb += pl.clusters) {
        for (int t = t_lo; t < t_hi; ++t, ++it) {
          const int s = it % pl.stages;
          const uint32_t round = it / pl.stages;
          if (round > 0 && !sk_wait(&empty[s], (round - 1) & 1, stop)) { ok = false; break; }
          uint8_t* dst = ring + s * pl.stage_bytes;
          bulk_expect(&full[s], (uint32_t)(kTileBytes + kSB + xb0 + kSB + (WIDE && xb1 ? xb1 + kSB : 0)));
          const int64_t tw = (int64_t)nb * pl.KT + t;
          bulk_load_hint(dst, p.codes + tw * kTileBytes, kTileBytes, &full[s], pol);
          bulk_load_hint(dst + off_sw, p.scales + tw * kSB, kSB, &full[s], pol);
          bulk_load(dst + off_x, p.x_codes + (int64_t)t * kTileBytes, xb0, &full[s]);
          bulk_load(dst + off_sx, p.x_scales + (int64_t)t * kSB, kSB, &full[s]);
          if (WIDE && xb1) {
            bulk_load(dst + off_x + kTileBytes, p.x_codes + (int64_t)(pl.KT + t) * kTileBytes, xb1, &full[s]);
            bulk_load(dst + off_sx + kSB, p.x_scales + (int64_t)(pl.KT + t) * kSB, kSB, &full[s]);
          }
        }
      }
      if (!ok) {
        // stopped: the copies in flight have to land before the CTA ends
        const uint32_t first = it > (uint32_t)pl.stages ? it - pl.stages : 0;
        for (uint32_t j = first; j < it; ++j) sk_wait(&full[j % pl.stages], (j / pl.stages) & 1, stop, true);
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    if (elect_one()) {
      const int ksteps = (p.K + 63) / 64;
      uint32_t it = 0, blk = 0;
      bool ok = true;
      for (int nb = cid; nb < pl.blocks && ok; nb += pl.clusters, ++blk) {
        if (blk > 0 && !sk_wait(&tempty, (blk - 1) & 1, stop)) break;
        tc::fence_after();
        for (int t = t_lo; t < t_hi; ++t, ++it) {
          const int s = it % pl.stages;
          if (!sk_wait(&full[s], (it / pl.stages) & 1, stop)) { ok = false; break; }
          tc::fence_after();
          const uint32_t a = tc::saddr(ring + s * pl.stage_bytes);
#pragma unroll
          for (int at = 0; at < kAtoms; ++at) {
            copy_scales(tmem + kSfW + at * 4, a + off_sw + at * 512);
#pragma unroll
            for (int xb = 0; xb < kXB; ++xb)
              copy_scales(tmem + kSfX + at * (4 * kXB) + xb * 4, a + off_sx + xb * kSB + at * 512);
          }
          const int n = min(4, ksteps - t * 4);
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            if (k >= n) break;
            const int at = NV ? k : k >> 1;
            const uint32_t sf = NV ? 0u : (uint32_t)(k & 1) * 2;
            mma4<NV>(tmem, tc::desc_sw128(a + k * 32), tc::desc_sw128(a + off_x + k * 32),
                     idesc4(128, pl.ncol, !NV, sf), tmem + kSfW + at * 4, tmem + kSfX + at * (4 * kXB),
                     (t > t_lo || k > 0) ? 1u : 0u);
          }
          tc::commit(&empty[s]);
        }
        if (ok) tc::commit(&tfull);
      }
      if (*stop) {
        tc::commit(&drain);
        sk_wait(&drain, 0, stop, true);
      }
    }
    __syncwarp();
  } else {
    const int quad = warp & 3, et = threadIdx.x - 64;
    const int r = quad * 32 + lane;                   // row of the block
    const int j = r & 63, half = r >> 6;
    const int owner = j / j_per, jl = j - owner * j_per;
    const int buf_floats = CL * pl.mp * 2 * j_per;
    pdl_wait();
    uint32_t blk = 0;
    bool dead = false;
    for (int nb = cid; nb < pl.blocks; nb += pl.clusters, ++blk) {
      if (!dead) {
        int ok = 0;
        if (lane == 0) ok = sk_wait(&tfull, blk & 1, stop) ? 1 : 0;
        dead = __shfl_sync(0xffffffffu, ok, 0) == 0;
      }
      float* rb = recv + (blk & 1) * buf_floats;
      // this rank's sums of row r, token tok -> [rank][tok][half][jl] of the owner
      float* dst = rb + ((int64_t)rank * pl.mp * 2 + half) * j_per + jl;
      if (CL > 1 && owner != rank) dst = cg::this_cluster().map_shared_rank(dst, owner);
      if (!dead) {
        tc::fence_after();
        for (int m0 = 0; m0 < p.M; m0 += 4) {
          float v[32];
          tc::tmem_ld32(tmem + ((uint32_t)(quad * 32) << 16) + m0 * kTerms, v);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            if (m0 + i >= p.M) break;
            float sum = 0.f;
#pragma unroll
            for (int t = kTerms - 1; t >= 0; --t)     // small terms first
              sum = NV ? fmaf(v[i * kTerms + t], 1.f / (float)(1 << term_off(t)), sum) : sum + v[i * kTerms + t];
            dst[(int64_t)(m0 + i) * 2 * j_per] = NV ? sum * p.x_factor[m0 + i] : sum;
          }
        }
        tc::fence_before();
      }
      __syncwarp();
      if (lane == 0 && !dead) tc::bar_arrive(&tempty);
      sk_sync();                                      // every row of this CTA is on its way
      if (CL > 1) {
        if (warp == 2 && lane < CL && lane != rank) {
          // cluster-scope release: the CTA's stores, seen through the barrier above, come before the arrival
          asm volatile("fence.acq_rel.cluster;" ::: "memory");
          uint32_t remote;
          asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote)
                       : "r"(tc::saddr(&recv_bar[blk & 1])), "r"(lane));
          asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(remote) : "memory");
        }
        __syncwarp();
        if (!dead) {
          const bool ok = sk_wait_cluster(&recv_bar[blk & 1], (blk >> 1) & 1, stop);
          dead = !__all_sync(0xffffffffu, ok);
        }
      }
      // ---- finish rows j_lo.. and + 64: consecutive threads on consecutive rows
      const bool swi = p.mode == GEMV_SWIGLU;
      const int halves = swi ? 1 : 2;
      for (int e = et; e < rows * p.M * halves; e += 128) {
        const int q = e / rows, row = e - q * rows;
        const int tok = swi ? q : q >> 1, hf = swi ? 0 : q & 1;
        float v = 0.f, u = 0.f;
        for (int c = 0; c < CL; ++c) {
          const float* src = rb + ((c * pl.mp + tok) * 2 + hf) * j_per + row;
          v += src[0];
          if (swi) u += src[j_per];
        }
        const int n = nb * 128 + j_lo + row + hf * 64;
        if (swi) {
          const int col = nb * 64 + j_lo + row;
          if (col >= p.width) continue;
          if (NV) {
            v *= p.row_scale[n];
            u *= p.row_scale[n + 64];
          }
          // written so that a NaN stays one
          v = v > p.limit ? p.limit : v;
          u = u > p.limit ? p.limit : u < -p.limit ? -p.limit : u;
          reinterpret_cast<__nv_bfloat16*>(p.y)[(int64_t)tok * p.ldy + col] = f2bf(siluf_(v) * u);
        } else {
          if (n >= p.N) continue;
          if (NV) v *= p.row_scale[n];
          const int64_t off = (int64_t)tok * p.ldy + n;
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
  tc::fence_before();
  // no CTA leaves while another of its cluster may still write to it
  if (CL > 1) cg::this_cluster().sync();
  else __syncthreads();
  if (warp == 1) {
    tc::fence_after();
    tc::tmem_free(tmem, kCols);
  }
}

// Shape of the launch.  CL, the CTAs that share a row block, is the one that needs the fewest tile steps on the busiest
// CTA (a block costs about one more step: its reduction and stores); ties go to the smaller, which sends less.
template <bool NV, bool WIDE>
static SkPlan sk_plan(int N, int K, int M, int sms) {
  SkPlan b{};
  b.blocks = (N + 127) / 128;
  b.KT = tiles_k(K);
  b.mp = M;
  b.ncol = std::max(16, (M * kTerms + 15) / 16 * 16);
  const int slots = (WIDE ? 1 : 2) * sms;
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
  constexpr int kSB = Fmt<NV>::kScaleBytes;
  b.stage_bytes = (kTileBytes + b.ncol * 128 + kSB + (b.ncol > 128 ? 2 : 1) * kSB + 1023) / 1024 * 1024;
  return b;
}
static int sk_recv_bytes(const SkPlan& b) { return 2 * b.CL * b.mp * 2 * ((64 + b.CL - 1) / b.CL) * 4; }

template <bool NV, bool WIDE>
static cudaError_t launch_skinny(const Fp4SkinnyArgs& p, int sms, cudaStream_t st) {
  SkPlan pl = sk_plan<NV, WIDE>(p.mode == GEMV_SWIGLU ? (p.width + 63) / 64 * 128 : p.N, p.K, p.M, sms);
  auto kern = fp4_skinny_kernel<NV, WIDE>;
  const int budget = (WIDE ? 225 : 112) * 1024 - 1024 - sk_recv_bytes(pl);
  pl.stages = std::min(8, budget / pl.stage_bytes);
  if (pl.stages < 2) return cudaErrorInvalidConfiguration;
  const int smem = pl.stages * pl.stage_bytes + sk_recv_bytes(pl) + 1024;
  cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(pl.clusters * pl.CL);
  cfg.blockDim = dim3(kSkThreads);
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

int g53_fp4_terms() { return fp4::kTerms; }

cudaError_t g53_fp4_expand(const Fp4ExpandArgs& p, cudaStream_t st) {
  if (p.M < 1 || p.M > 32 || p.K < 16 || p.K % (p.nv ? 16 : 32)) return cudaErrorInvalidValue;
  const dim3 grid((fp4::tiles_k(p.K) * 16 + 127) / 128, p.M);
  return p.nv ? g53_launch_pdl(fp4::fp4_expand_kernel<true>, grid, dim3(128), 0, st, 1, p)
              : g53_launch_pdl(fp4::fp4_expand_kernel<false>, grid, dim3(128), 0, st, 1, p);
}

cudaError_t g53_fp4_skinny(const Fp4SkinnyArgs& p, cudaStream_t st) {
  if (p.M < 1 || p.M > 32 || p.N < 1 || p.K < 16 || p.K % (p.nv ? 16 : 32)) return cudaErrorInvalidValue;
  int dev = 0, sms = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess) e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  if (e != cudaSuccess) return e;
  if (p.nv) return p.M <= 16 ? fp4::launch_skinny<true, false>(p, sms, st) : fp4::launch_skinny<true, true>(p, sms, st);
  return p.M <= 16 ? fp4::launch_skinny<false, false>(p, sms, st) : fp4::launch_skinny<false, true>(p, sms, st);
}

cudaError_t g53_fp4_skinny_error(int* code) {
  const int z = 0;
  cudaError_t e = cudaMemcpyFromSymbol(code, fp4::g_skinny_err, sizeof(int));
  if (e == cudaSuccess && *code) e = cudaMemcpyToSymbol(fp4::g_skinny_err, &z, sizeof(int));
  return e;
}
