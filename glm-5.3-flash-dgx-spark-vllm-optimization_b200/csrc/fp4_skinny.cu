// Small-M product with 4-bit weights: Y[M, N] = X[M, K] @ W4[N, K]^T for up to 96 rows of 16-bit activations (W4A16, in groups of
// 16 or 32) or up to 128 4-bit rows.
//
// A decode projection reads every weight byte once, so HBM is the floor: 9/16 (17/32) byte per weight.  Widening the
// weights to f16 operands on the CUDA cores cannot keep up with that (built first: 390 instructions per warp and 32 x 128
// weights, 2.7 TB/s), so the codes go to the block-scaled tensor cores as they are, as the 128-row operand of
// tcgen05.mma, and the activations are brought to 4 bits without losing them: a block of x with largest magnitude in
// [2^e, 2^(e+1)) is written as integers X = round(x 2^(21-e)), |X| < 2^22, and X in eight balanced base-8 digits,
//     x = sum_t d_t 2^(e-3t),   d_t in -4..3, t = 0..7,
// all of which are e2m1 values.  Term t of a row is a 4-bit row with the block scales 2^(e-3t); the eight of them are 8 of
// the mma's N columns, and the epilogue sums the eight fp32 columns.  What is lost is at most 2^-22 of the block's largest
// magnitude; a bf16 element within 2^-14 of it loses nothing.  The tensor core has the time: N = 64 (8 rows) costs about
// 290 clocks per 128 x 256 tile of weights, HBM delivers one in 790 per SM.
//
// nvfp4's e4m3 scales hold 2^(e-3t) over a power of two of the row and of the term, which the epilogue puts back; they
// reach from 2^8 down to 2^-9, so a block more than 2^17 below the row's largest shares the scale of one at 2^-17 (off by
// at most 2^-39 of the row's largest).
//
// The expansion is formed by each CTA for its own slice of K, in shared memory, when that is little work (INLINE); else
// fp4_expand writes it once as a tile image (fp4.cuh), rows 8 m + t, and it is fetched tile by tile beside the weights.
//
// fp4_skinny: a CTA takes a 128-row block of W and a slice of its K tiles; a cluster of CL CTAs shares a block, and
// clusters walk the blocks.  Warp 0 streams tiles into a ring (contiguous cp.async.bulk), warp 1 copies the scales to TMEM
// and issues the mma, warps 2-9 (form the expansion,) read the sums (a thread holds one weight row), send them to the rank
// of the cluster that owns the row (st.async into its shared memory, counted in bytes on its barrier: stores with a
// cluster-scope release behind them took a microsecond) and finish the rows they own, adding in rank order: the result does
// not depend on timing.  Two receive buffers alternate: a rank can only send block b + 2 after it received every rank's b +
// 1, and no thread of a rank sends of b + 1 before all of its warps have read b (a barrier of theirs: those that hold none of a
// peer's rows send it nothing, so the arrival of b + 1 alone says nothing about them).  No barrier is needed at the end: a CTA
// leaves after it has received all that is sent to it.
//
// Before griddepcontrol.wait only prefetches into L2 are issued: the weights may be what the previous kernel writes.
// Waits are bounded; one that runs out sets the error word, and the CTA goes on without the main loop's waits but sends and
// receives all the same, so that no CTA of the cluster is left waiting or written to after it has gone; copies and mma in
// flight are waited for (bounded) and the TMEM is freed.
#include <algorithm>
#include <atomic>
#include "fp4.cuh"
#include "fp4_tc.cuh"
#include "launchers.h"

namespace g53 {
namespace fp4 {

__device__ int g_skinny_err = 0;

constexpr int kTerms = 8;
constexpr int kEpi = 8;                               // warps of the expansion and the epilogue
constexpr int kSkThreads = 64 + kEpi * 32;
constexpr int kErrSk = 0x6b40;

// ------------------------------------------------------------------------------------------------------ expansion
// 8 elements (bf16 pairs) of a block with exponent e -> per term a word of 8 codes.  X' = X + sum_t 4 * 8^t has the digits
// d_t + 4 as its octal digits; a byte permutation looks up the codes of 4 digits at a time, even elements in the low and
// odd ones in the high nibble.
template <typename F>
__device__ __forceinline__ void expand8(const uint4& w4, int e, F&& emit) {
  const uint32_t w[4] = {w4.x, w4.y, w4.z, w4.w};
  const float s = pow2i(21 - e);
  uint32_t x[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    // 1.5 * 2^23 + X: X in the low bits of the float
    constexpr uint32_t kShift = 044444444u - 0x4b400000u;
    x[2 * i] = __float_as_uint(fmaf(__uint_as_float(w[i] << 16), s, 12582912.f)) + kShift;
    x[2 * i + 1] = __float_as_uint(fmaf(__uint_as_float(w[i] & 0xffff0000u), s, 12582912.f)) + kShift;
  }
#pragma unroll
  for (int t = 0; t < kTerms; ++t) {
    const int sh = 3 * (kTerms - 1 - t);
    uint32_t lo = 0, hi = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t a = x[2 * i], b = x[2 * i + 1];
      lo |= (sh >= 4 * i ? a >> (sh - 4 * i) : a << (4 * i - sh)) & (7u << (4 * i));
      hi |= (sh >= 4 * i ? b >> (sh - 4 * i) : b << (4 * i - sh)) & (7u << (4 * i));
    }
    // codes of the digits -4 -3 -2 -1 0 1 2 3: 14 13 12 10 0 2 4 5
    emit(t, __byte_perm(0x0a0c0d0eu, 0x05040200u, lo) | __byte_perm(0xa0c0d0e0u, 0x50402000u, hi));
  }
}

__device__ __forceinline__ uint32_t amax_bits8(const uint4& w) {
  const uint32_t a = max_u16x2(max_u16x2(w.x & 0x7fff7fffu, w.y & 0x7fff7fffu),
                               max_u16x2(w.z & 0x7fff7fffu, w.w & 0x7fff7fffu));
  return max(a << 16, a & 0xffff0000u);
}
// largest over the threads of a block: two (16 elements) or four (32)
template <bool NV>
__device__ __forceinline__ uint32_t block_amax(uint32_t am) {
  am = max(am, __shfl_xor_sync(0xffffffffu, am, 1));
  return NV ? am : max(am, __shfl_xor_sync(0xffffffffu, am, 2));
}
// (from L2, like everything that an earlier programmatic launch may have written)
__device__ __forceinline__ uint4 load8(const uint16_t* x, bool vec) {
  if (vec) return __ldcg(reinterpret_cast<const uint4*>(x));
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = (uint32_t)__ldcg(x + 2 * i) | ((uint32_t)__ldcg(x + 2 * i + 1) << 16);
  return make_uint4(w[0], w[1], w[2], w[3]);
}
__device__ __forceinline__ int exponent(uint32_t bits) { return (int)(bits >> 23) - 127; }
// nvfp4: exponent of the row, low enough rows share one (2^(21-e) stays in range)
__device__ __forceinline__ int row_exponent(uint32_t amax) { return max(exponent(amax), -85); }
__device__ __forceinline__ float row_factor(uint32_t amax) {
  return amax >= kInfBits ? __uint_as_float(0x7fc00000u) : pow2i(max(row_exponent(amax) - 8, -126));
}

// largest magnitude of a block -> exponent and scale byte(s).  nvfp4: one byte for all terms (the term's 2^-3t is put back later); mxfp4:
// byte of term 0, term t is 3t lower
template <bool NV>
__device__ __forceinline__ int block_exponent(uint32_t amax, int row_e, uint32_t& byte) {
  if constexpr (NV) {
    const int e = max(min(exponent(amax), row_e), row_e - 17);
    const int n = e - row_e + 8;                      // 8 .. -9
    byte = n >= -6 ? (uint32_t)(n + 7) << 3 : 1u << (n + 9);
    return e;
  } else {
    const int e = max(exponent(amax), -105);
    byte = amax >= kInfBits ? 255u : (uint32_t)(e + 127);
    return min(e, 127);
  }
}
template <bool NV>
__device__ __forceinline__ uint32_t term_scales(uint32_t s4, int t) {
  if constexpr (NV) return s4;
  // four E8M0 bytes, each 3t lower unless NaN (byte-wise: no borrow, every byte is >= 22 or 0 for padding)
  uint32_t r = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t b = (s4 >> (8 * i)) & 0xffu;
    r |= (b == 255u ? 255u : b > 3u * t ? b - 3u * t : 0u) << (8 * i);
  }
  return r;
}
// scale bytes of four neighbouring columns in one word (valid in the first of their lanes)
template <bool NV>
__device__ __forceinline__ uint32_t gather_scales(uint32_t sc) {
  constexpr int kStep = NV ? 2 : 4;
  uint32_t s4 = sc;
  s4 |= __shfl_down_sync(0xffffffffu, sc, kStep) << 8;
  s4 |= __shfl_down_sync(0xffffffffu, sc, 2 * kStep) << 16;
  s4 |= __shfl_down_sync(0xffffffffu, sc, 3 * kStep) << 24;
  return s4;
}

// CTA: 256 times 8 elements of one row; nvfp4 reads the whole row for its maximum first
template <bool NV>
__global__ void __launch_bounds__(256) fp4_expand_kernel(Fp4ExpandArgs p) {
  __shared__ uint32_t red[8];
  const int m = blockIdx.y, b = blockIdx.x * 256 + threadIdx.x;
  const int KT = tiles_k(p.K);
  const int nk = p.K / 8;
  const uint16_t* x = reinterpret_cast<const uint16_t*>(p.x) + (int64_t)m * p.ldx;
  pdl_trigger();
  pdl_wait();
  const uint4 w = b < nk ? load8(x + (int64_t)b * 8, p.vec) : make_uint4(0, 0, 0, 0);
  int row_e = 0;
  if constexpr (NV) {
    uint32_t am = 0;
#pragma unroll 4
    for (int i = threadIdx.x; i < nk; i += 256) am = max(am, amax_bits8(load8(x + (int64_t)i * 8, p.vec)));
    am = __reduce_max_sync(0xffffffffu, am);
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = am;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 8; ++i) am = max(am, red[i]);
    row_e = row_exponent(am);
    if (b == 0) p.factor[m] = row_factor(am);
  } else if (b == 0) {
    p.factor[m] = 1.f;
  }
  uint32_t sc;
  const int e = block_exponent<NV>(block_amax<NV>(amax_bits8(w)), row_e, sc);
  const uint32_t s4 = gather_scales<NV>(b < nk ? sc : 0u);
  const int kt = b >> 5, kb = b & 31;
  if (kt < KT)
    expand8(w, e, [&](int t, uint32_t code) {
      const int row = m * kTerms + t, rr = row % kTileRows;
      const int64_t tile = (int64_t)(row / kTileRows) * KT + kt;
      *reinterpret_cast<uint32_t*>(p.codes + tile * kTileBytes + chunk_off(rr, kb >> 2) + (kb & 3) * 4) = code;
      constexpr int kStep = NV ? 2 : 4;
      if ((kb & (4 * kStep - 1)) == 0)
        *reinterpret_cast<uint32_t*>(p.scales + tile * Fmt<NV>::kScaleBytes + scale_off(rr, kb / kStep)) =
            term_scales<NV>(s4, t);
    });
}

// -------------------------------------------------------------------------------------------------------- product
// per: K tiles of a slice; stages: ring depth; clusters: persistent clusters; ncol: mma N; xbytes: resident expansion
// units: row blocks x groups of (at most `group`) rows of x, each served by one pass over a weight tile
struct SkPlan {
  int units, groups, group, KT, per, stages, clusters, CL, ncol, stage_bytes, xbytes;
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
__device__ __forceinline__ void sk_sync() { asm volatile("bar.sync 1, 256;" ::: "memory"); }   // the epilogue warps
__device__ __forceinline__ void sk_prefetch(const void* src, uint32_t bytes) {
  asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(src), "r"(bytes) : "memory");
}

// one output of the modes that write sums
__device__ __forceinline__ void store1(const Fp4SkinnyArgs& p, int tok, int n, float v) {
  const int64_t off = (int64_t)tok * p.ldy + n;
  if (p.mode == GEMV_BF16) {
    reinterpret_cast<__nv_bfloat16*>(p.y)[off] = f2bf(v);
  } else {
    float* y = reinterpret_cast<float*>(p.y) + off;
    *y = p.mode == GEMV_F32_ACC ? __ldcg(y) + v : v;
  }
}
// four values into the shared memory of a CTA of the cluster, counted on its barrier (both addresses mapped to that CTA)
__device__ __forceinline__ void send4(uint32_t dst, uint32_t bar, const float (&v)[4]) {
  asm volatile("st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.v4.b32 [%0], {%1, %2, %3, %4}, [%5];"
               ::"r"(dst), "r"(__float_as_uint(v[0])), "r"(__float_as_uint(v[1])), "r"(__float_as_uint(v[2])),
               "r"(__float_as_uint(v[3])), "r"(bar) : "memory");
}
__device__ __forceinline__ uint32_t map_to(uint32_t addr, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}

// T: terms per row of x: 8 (expanded), or 1 (4-bit rows as they are).  WIDE: mma N up to 256, one CTA per SM; otherwise N
// <= 128 and two CTAs per SM
template <bool NV, int T, bool WIDE, bool INLINE>
__global__ void __launch_bounds__(kSkThreads, WIDE ? 1 : 2) fp4_skinny_kernel(Fp4SkinnyArgs p, SkPlan pl) {
  constexpr int kSB = Fmt<NV>::kScaleBytes;
  constexpr int kAtoms = kSB / 512;
  constexpr int kXB = WIDE && T > 1 ? 2 : 1;          // 128-row blocks of X per group
  constexpr uint32_t kCols = WIDE ? 512 : 256;        // TMEM columns: sums, scales of W, scales of X
  constexpr uint32_t kSfW = WIDE ? 256 : 128, kSfX = kSfW + 16;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t full[8], empty[8], recv_bar[2], tfull, tempty, xready, drain;
  __shared__ uint32_t tmem_s, xmax[32];
  __shared__ float xfac[32];
  __shared__ int stop_s;
  volatile int* stop = &stop_s;
  uint8_t* xs = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* ring = xs + (INLINE ? pl.xbytes : 0);
  float* recv = reinterpret_cast<float*>(ring + pl.stages * pl.stage_bytes);   // [2][CL][2][j_per][Mp]

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int CL = pl.CL;
  const int rank = CL > 1 ? (int)blockIdx.x % CL : 0, cid = (int)blockIdx.x / CL;
  const int t_lo = rank * pl.per, t_hi = min(pl.KT, t_lo + pl.per);
  // rows of a block that this rank finishes: pairs (j, j + 64), j in [j_lo, j_lo + rows)
  const int j_per = (64 + CL - 1) / CL;
  const int j_lo = min(64, rank * j_per), rows = min(64, j_lo + j_per) - j_lo;
  const int xrows = pl.ncol;                          // rows of the expansion
  const int xb0 = min(xrows, 128) * 128, xb1 = kXB == 2 ? max(0, xrows - 128) * 128 : 0;
  const int xtile = xrows * 128;                      // code bytes of the expansion per K tile
  // a stage: codes of W, (codes of X,) scales of W, (scales of X)
  const int off_x = kTileBytes, off_sw = off_x + (INLINE ? 0 : xtile), off_sx = off_sw + kSB;

  if (threadIdx.x == 0) {
    for (int s = 0; s < pl.stages; ++s) {
      tc::bar_init(&full[s], 1);
      tc::bar_init(&empty[s], 1);
    }
    tc::bar_init(&recv_bar[0], 1);
    tc::bar_init(&recv_bar[1], 1);
    tc::bar_init(&tfull, 1);
    tc::bar_init(&tempty, kEpi);
    tc::bar_init(&xready, kEpi);
    tc::bar_init(&drain, 1);
    stop_s = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (threadIdx.x >= 64 && threadIdx.x < 96) xmax[threadIdx.x - 64] = 0;
  if (warp == 1) tc::tmem_alloc(&tmem_s, kCols);
  tc::fence_before();
  __syncthreads();
  // the peers' barriers are first touched by the epilogue, which waits there (mbarrier_init above is the release)
  if (CL > 1) cluster_arrive();
  tc::fence_after();
  const uint32_t tmem = tmem_s;
  pdl_trigger();

  if (warp == 0) {
    if (elect_one()) {
      const uint64_t pol = l2_evict_first_policy();
      for (int t = t_lo; t < t_hi && t < t_lo + 8; ++t) {
        const int64_t tile = (int64_t)(cid / pl.groups) * pl.KT + t;
        sk_prefetch(p.codes + tile * kTileBytes, kTileBytes);
        sk_prefetch(p.scales + tile * kSB, kSB);
      }
      pdl_wait();
      uint32_t it = 0;
      bool ok = true;
      for (int u = cid; u < pl.units && ok; u += pl.clusters) {
        const int nb = u / pl.groups;
        const int xrow = (u - nb * pl.groups) * pl.group * T;                // first image row of X: a multiple of 64
        const int64_t xblk = (int64_t)(xrow / kTileRows) * pl.KT;
        const int xoff = (xrow & 64) * 128;
        for (int t = t_lo; t < t_hi; ++t, ++it) {
          const int s = it % pl.stages;
          const uint32_t round = it / pl.stages;
          if (round > 0 && !sk_wait(&empty[s], (round - 1) & 1, stop)) { ok = false; break; }
          uint8_t* dst = ring + s * pl.stage_bytes;
          bulk_expect(&full[s], (uint32_t)(kTileBytes + kSB + (INLINE ? 0 : xb0 + kSB + (xb1 ? xb1 + kSB : 0))));
          const int64_t tw = (int64_t)nb * pl.KT + t;
          bulk_load_hint(dst, p.codes + tw * kTileBytes, kTileBytes, &full[s], pol);
          bulk_load_hint(dst + off_sw, p.scales + tw * kSB, kSB, &full[s], pol);
          if constexpr (!INLINE) {
            bulk_load(dst + off_x, p.x_codes + (xblk + t) * kTileBytes + xoff, xb0, &full[s]);
            bulk_load(dst + off_sx, p.x_scales + (xblk + t) * kSB, kSB, &full[s]);
            if (kXB == 2 && xb1) {
              bulk_load(dst + off_x + kTileBytes, p.x_codes + (xblk + pl.KT + t) * kTileBytes, xb1, &full[s]);
              bulk_load(dst + off_sx + kSB, p.x_scales + (xblk + pl.KT + t) * kSB, kSB, &full[s]);
            }
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
    if (CL > 1) cluster_wait();
  } else if (warp == 1) {
    if (elect_one()) {
      pdl_wait();                                     // its bounded waits must not run while an earlier kernel does
      const int ksteps = (p.K + 63) / 64;
      uint32_t it = 0, blk = 0;
      bool ok = true;
      for (int u = cid; u < pl.units && ok; u += pl.clusters, ++blk) {
        // rows 64.. of a 128-row block of X: the second half of its scale columns
        const uint32_t sfx = tmem + kSfX + (((u % pl.groups) * pl.group * T) & 64 ? 2 : 0);
        if (blk > 0 && !sk_wait(&tempty, (blk - 1) & 1, stop)) break;
        tc::fence_after();
        for (int t = t_lo; t < t_hi; ++t, ++it) {
          const int s = it % pl.stages;
          if (!sk_wait(&full[s], (it / pl.stages) & 1, stop) || (INLINE && it == 0 && !sk_wait(&xready, 0, stop))) {
            ok = false;
            break;
          }
          tc::fence_after();
          const uint32_t a = tc::saddr(ring + s * pl.stage_bytes);
          const uint32_t xc = INLINE ? tc::saddr(xs + (t - t_lo) * xtile) : a + off_x;
          const uint32_t xsc = INLINE ? tc::saddr(xs + pl.per * xtile + (t - t_lo) * kSB) : a + off_sx;
#pragma unroll
          for (int at = 0; at < kAtoms; ++at) {
            copy_scales(tmem + kSfW + at * 4, a + off_sw + at * 512);
#pragma unroll
            for (int xb = 0; xb < kXB; ++xb)
              copy_scales(tmem + kSfX + at * (4 * kXB) + xb * 4, xsc + xb * kSB + at * 512);
          }
          const int n = min(4, ksteps - t * 4);
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            if (k >= n) break;
            const int at = NV ? k : k >> 1;
            const uint32_t sf = NV ? 0u : (uint32_t)(k & 1) * 2;
            mma4<NV>(tmem, tc::desc_sw128(a + k * 32), tc::desc_sw128(xc + k * 32), idesc4(128, pl.ncol, !NV, sf),
                     tmem + kSfW + at * 4, sfx + at * (4 * kXB), (t > t_lo || k > 0) ? 1u : 0u);
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
    if (CL > 1) cluster_wait();
  } else {
    const int quad = warp & 3, et = threadIdx.x - 64, part = (warp - 2) >> 2;
    const int r = quad * 32 + lane;                   // row of the block
    const int j = r & 63, half = r >> 6;
    const int owner = j / j_per, jl = j - owner * j_per;
    const int Mp = (min(p.M, pl.group) + 3) & ~3;      // rows of x in a group, rounded up to fours
    const int buf_floats = CL * 2 * j_per * Mp;
    const bool swi = p.mode == GEMV_SWIGLU;
    const bool direct = CL == 1 && !swi;              // rows finished where they are read
    // this thread's first share of the finishing: four tokens of one row (of a pair of rows)
    const int f_q = et / rows, f_row = et - f_q * rows;
    pdl_wait();
    if constexpr (INLINE) {
      // a thread per 8 elements of the slice (the plan sees to it that there are no more than threads)
      const int nblk = (t_hi - t_lo) * 32, nk = p.K / 8 - t_lo * 32;        // eights in the slice; those that exist
      const bool in = et < p.M * nblk;
      const int m = in ? et / nblk : 0, b = et - m * nblk;
      uint4 w = make_uint4(0, 0, 0, 0);
      if (in && b < nk)
        w = load8(reinterpret_cast<const uint16_t*>(p.x) + (int64_t)m * p.ldx + (int64_t)t_lo * kTileK + b * 8, p.xvec);
      const uint32_t am = amax_bits8(w);
      if constexpr (NV) {
        // a warp's lanes belong to one row
        const uint32_t wm = __reduce_max_sync(0xffffffffu, am);
        if (in && lane == 0) atomicMax(&xmax[m], wm);
        sk_sync();
        if (et < p.M) xfac[et] = row_factor(xmax[et]);
      }
      uint32_t sc;
      const int e = block_exponent<NV>(block_amax<NV>(am), NV ? row_exponent(xmax[m]) : 0, sc);
      const uint32_t s4 = gather_scales<NV>(b < nk ? sc : 0u);
      if (in) {
        const int kb = b & 31;
        uint8_t* xc = xs + (b >> 5) * xtile;
        uint8_t* xsc = xs + pl.per * xtile + (b >> 5) * kSB;
        expand8(w, e, [&](int t, uint32_t code) {
          const int row = m * kTerms + t;
          *reinterpret_cast<uint32_t*>(xc + chunk_off(row, kb >> 2) + (kb & 3) * 4) = code;
          constexpr int kStep = NV ? 2 : 4;
          if ((kb & (4 * kStep - 1)) == 0)
            *reinterpret_cast<uint32_t*>(xsc + scale_off(row, kb / kStep)) = term_scales<NV>(s4, t);
        });
      }
      tc::fence_async_smem();
      __syncwarp();
      if (lane == 0) tc::bar_arrive(&xready);
    }
    if (CL > 1) cluster_wait();                       // every CTA of the cluster has its barriers
    sk_sync();
    uint32_t blk = 0;
    bool dead = false;
    for (int u = cid; u < pl.units; u += pl.clusters, ++blk) {
      const int nb = u / pl.groups, x0 = (u - nb * pl.groups) * pl.group;  // first row of x
      const int M = min(p.M - x0, pl.group);
      const uint32_t rbar = tc::saddr(&recv_bar[blk & 1]);
      if (CL > 1 && et == 0) bulk_expect(&recv_bar[blk & 1], (uint32_t)((CL - 1) * 2 * rows * ((M + 3) & ~3) * 4));
      // scale of this thread's weight row: loaded under the main loop
      const RowScale ws = split_scale(NV && nb * 128 + r < p.N ? __ldcg(p.row_scale + nb * 128 + r) : 1.f);
      // factors of the rows of x: lane l those of l, l + 32, ..
      constexpr int kXf = T == 1 ? 4 : 1;
      float xf[kXf];
#pragma unroll
      for (int i = 0; i < kXf; ++i) {
        xf[i] = 1.f;
        if (NV && INLINE) xf[i] = xfac[lane];
        if (NV && !INLINE && lane + 32 * i < M)
          xf[i] = p.x_factor ? __ldcg(p.x_factor + x0 + lane + 32 * i) : p.x_const;
      }
      if (!dead) {
        int ok = 0;
        if (lane == 0) ok = sk_wait(&tfull, blk & 1, stop) ? 1 : 0;
        dead = __shfl_sync(0xffffffffu, ok, 0) == 0;
      }
      tc::fence_after();
      float* rb = recv + (blk & 1) * buf_floats;
      // this rank's sums of row r -> [rank][half][jl][token] of the owner
      float* dst = rb + ((rank * 2 + half) * j_per + jl) * Mp;
      const uint32_t rdst = CL > 1 ? map_to(tc::saddr(dst), owner) : 0, rdbar = CL > 1 ? map_to(rbar, owner) : 0;
      constexpr int kTok = 32 / T;                     // rows of x in 32 columns
      for (int c0 = part * kTok; c0 < M; c0 += kTok * (kEpi / 4)) {
        float f = xf[0];                               // of the 32 rows that hold these
#pragma unroll
        for (int i = 1; i < kXf; ++i) f = c0 >= 32 * i ? xf[i] : f;
        float v[32];
        if (!dead) tc::tmem_ld32(tmem + ((uint32_t)(quad * 32) << 16) + c0 * T, v);
#pragma unroll
        for (int j4 = 0; j4 < kTok; j4 += 4) {
          const int m0 = c0 + j4;
          if (m0 >= M) break;
          float sum[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            sum[i] = 0.f;
#pragma unroll
            for (int t = T - 1; t >= 0; --t)           // small terms first
              sum[i] = NV ? fmaf(v[(j4 + i) * T + t], 1.f / (float)(1 << (3 * t)), sum[i]) : sum[i] + v[(j4 + i) * T + t];
            // rows past M: never used
            if (NV) sum[i] = sum[i] * (__shfl_sync(0xffffffffu, f, (m0 + i) & 31) * ws.a) * ws.b;
          }
          if (direct) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
              if (m0 + i < M && nb * 128 + r < p.N) store1(p, x0 + m0 + i, nb * 128 + r, sum[i]);
          } else if (owner == rank) {
            *reinterpret_cast<float4*>(dst + m0) = make_float4(sum[0], sum[1], sum[2], sum[3]);
          } else {
            send4(rdst + m0 * 4, rdbar, sum);
          }
        }
      }
      tc::fence_before();
      __syncwarp();
      if (lane == 0) tc::bar_arrive(&tempty);
      if (direct) continue;
      sk_sync();                                      // this CTA's own rows
      if (CL > 1) {
        const bool ok = bar_wait_cluster(&recv_bar[blk & 1], (blk >> 1) & 1, nullptr, &g_skinny_err, kErrSk + 1);
        if (!ok) *stop = 1;                           // (waited for in a stopped CTA, too)
      }
      // ---- finish rows j_lo.. and + 64, four tokens at a time: consecutive threads on consecutive rows
      const int shares = rows * ((M + 3) / 4) * (swi ? 1 : 2);
      for (int e = et; e < shares; e += kEpi * 32) {
        const bool own = e == et;
        const int q = own ? f_q : e / rows, row = own ? f_row : e - q * rows;
        const int tok = (swi ? q : q >> 1) * 4, hf = swi ? 0 : q & 1;
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f), w = v;
        for (int c = 0; c < CL; ++c) {
          const float* src = rb + ((c * 2 + hf) * j_per + row) * Mp + tok;
          const float4 a = *reinterpret_cast<const float4*>(src);
          v.x += a.x; v.y += a.y; v.z += a.z; v.w += a.w;
          if (swi) {
            const float4 b = *reinterpret_cast<const float4*>(src + j_per * Mp);
            w.x += b.x; w.y += b.y; w.z += b.z; w.w += b.w;
          }
        }
        const int n = nb * 128 + j_lo + row + hf * 64;
        const float vs[4] = {v.x, v.y, v.z, v.w};
        const float us[4] = {w.x, w.y, w.z, w.w};
        if (swi) {
          const int col = nb * 64 + j_lo + row;
          if (col >= p.width) continue;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            if (tok + i >= M) break;
            float g = vs[i], h = us[i];
            // written so that a NaN stays one
            g = g > p.limit ? p.limit : g;
            h = h > p.limit ? p.limit : h < -p.limit ? -p.limit : h;
            reinterpret_cast<__nv_bfloat16*>(p.y)[(int64_t)(x0 + tok + i) * p.ldy + col] = f2bf(siluf_(g) * h);
          }
        } else {
          if (n >= p.N) continue;
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (tok + i < M) store1(p, x0 + tok + i, n, vs[i]);
        }
      }
      if (CL > 1 && u + pl.clusters < pl.units) sk_sync();   // this block is read: its sums of the next may go out
    }
  }
  tc::fence_before();
  __syncthreads();
  if (warp == 1) {
    tc::fence_after();
    tc::tmem_free(tmem, kCols);
  }
}

constexpr int kMaxDev = 64;

static int sk_recv_bytes(int CL, int M, bool swi) {
  return CL == 1 && !swi ? 0 : 2 * CL * ((M + 3) & ~3) * 2 * ((64 + CL - 1) / CL) * 4;
}
static int sk_budget(bool wide) { return (wide ? 225 : 111) * 1024; }

// Stands in for the product in the question below: the runtime answers one CTA per SM for any kernel that uses TMEM
template <bool WIDE>
__global__ void __launch_bounds__(kSkThreads, WIDE ? 1 : 2) sk_shape_kernel() {}

// clusters of CL CTAs that run at once on the current device (one or two CTAs per SM); asked once per device.  Not CTAs / CL:
// a cluster stays inside a GPC (148 SMs: 296 CTAs alone, 93 clusters of 3, 33 of 8), and a cluster that has to wait for
// another doubles the time.
template <bool WIDE>
static cudaError_t sk_active(int dev, int CL, int* out) {
  static std::atomic<int> known[kMaxDev][9];
  if (dev < kMaxDev && (*out = known[dev][CL].load(std::memory_order_relaxed)) > 0) return cudaSuccess;
  auto kern = sk_shape_kernel<WIDE>;
  cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, sk_budget(WIDE));
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(CL);
  cfg.blockDim = dim3(kSkThreads);
  cfg.dynamicSmemBytes = sk_budget(WIDE);
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = CL;
  at[0].val.clusterDim.y = 1;
  at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  e = cudaOccupancyMaxActiveClusters(out, kern, &cfg);
  if (e != cudaSuccess) return e;
  *out = std::max(*out, 1);
  if (dev < kMaxDev) known[dev][CL].store(*out, std::memory_order_relaxed);
  return cudaSuccess;
}

// the dynamic shared memory limit of a kernel, raised once per device
template <bool NV, int T, bool WIDE, bool INLINE>
static cudaError_t sk_prepare(int dev) {
  static std::atomic<bool> done[kMaxDev];
  if (dev < kMaxDev && done[dev].load(std::memory_order_relaxed)) return cudaSuccess;
  const cudaError_t e = cudaFuncSetAttribute(fp4_skinny_kernel<NV, T, WIDE, INLINE>,
                                             cudaFuncAttributeMaxDynamicSharedMemorySize, sk_budget(WIDE));
  if (e == cudaSuccess && dev < kMaxDev) done[dev].store(true, std::memory_order_relaxed);
  return e;
}

// Shape of the launch: CL, the CTAs that share a row block.  Costs in units of a K tile (about 0.37 us), fitted to a sweep
// of CL over 1, 8 and 16 rows and six weight sizes: each round of blocks costs a CTA its tiles, a round after the first 4
// more and 0.08 for each row and CTA of the cluster (its reduction is not hidden), the last reduction 0.047.  A cluster
// launch keeps an eighth of the room free: with all of it in use, a CTA of a neighbouring kernel makes one cluster wait
// (32 clusters of 8 where 33 fit: 9.5 us, or 15.6).
template <bool NV, int T, bool WIDE, bool INLINE>
static cudaError_t sk_plan(int M, int64_t N, int K, int group, bool swi, int dev, SkPlan& b, double& cost) {
  constexpr int kSB = Fmt<NV>::kScaleBytes;
  b = SkPlan{};
  b.group = group;
  b.groups = (M + group - 1) / group;
  M = std::min(M, group);                             // rows of a group
  const int64_t units = (N + 127) / 128 * b.groups;
  if (units >= (int64_t)1 << 31) return cudaErrorInvalidConfiguration;
  b.units = (int)units;
  b.KT = tiles_k(K);
  b.ncol = std::max(16, (M * T + 15) / 16 * 16);
  const int xtile = b.ncol * 128 + (WIDE && T > 1 ? 2 : 1) * kSB;
  b.stage_bytes = (kTileBytes + kSB + (INLINE ? 0 : xtile) + 1023) / 1024 * 1024;
  for (int cl = 1; cl <= 8 && cl <= b.KT; ++cl) {
    const int per = (b.KT + cl - 1) / cl;
    if ((b.KT + per - 1) / per != cl) continue;       // a CTA of the cluster would have no tile
    if (INLINE && M * per * 32 > kEpi * 32) continue;  // a thread per 8 elements
    int active = 0;
    const cudaError_t e = sk_active<WIDE>(dev, cl, &active);
    if (e != cudaSuccess) return e;
    if (cl > 1) active -= active / 8;
    const int xbytes = INLINE ? (per * xtile + 1023) / 1024 * 1024 : 0;
    const int stages = std::min(8, (sk_budget(WIDE) - 1024 - xbytes - sk_recv_bytes(cl, M, swi)) / b.stage_bytes);
    if (stages < (INLINE ? 4 : 2)) continue;           // a resident expansion must leave the ring its depth
    const int clusters = std::min(b.units, active), rounds = (b.units + clusters - 1) / clusters;
    const double c = rounds * per + (rounds - 1) * (4 + 0.08 * M * cl) + 0.047 * M * cl;
    if (b.CL == 0 || c < cost) {
      cost = c;
      b.CL = cl;
      b.per = per;
      b.clusters = clusters;
      b.stages = stages;
      b.xbytes = xbytes;
    }
  }
  return b.CL ? cudaSuccess : cudaErrorInvalidConfiguration;
}

template <bool NV, int T, bool WIDE, bool INLINE>
static cudaError_t launch_skinny(const Fp4SkinnyArgs& p, cudaStream_t st) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  SkPlan b;
  double cost = 0;
  const bool swi = p.mode == GEMV_SWIGLU;
  if (e == cudaSuccess) e = sk_prepare<NV, T, WIDE, INLINE>(dev);
  if (T > 1) {
    if (e == cudaSuccess) e = sk_plan<NV, T, WIDE, INLINE>(p.M, p.N, p.K, WIDE ? 32 : 16, swi, dev, b, cost);
  } else {
    // 4-bit rows: 128 at a time read W fewer times, 64 leave room for the exchange of a cluster
    SkPlan c;
    double wide_cost = 0;
    if (e == cudaSuccess) e = sk_plan<NV, T, WIDE, INLINE>(p.M, p.N, p.K, 64, swi, dev, b, cost);
    if (e == cudaSuccess && p.M > 64 &&
        sk_plan<NV, T, WIDE, INLINE>(p.M, p.N, p.K, 128, swi, dev, c, wide_cost) == cudaSuccess && wide_cost < cost)
      b = c;
  }
  if (e != cudaSuccess) return e;
  const int smem = b.xbytes + b.stages * b.stage_bytes + sk_recv_bytes(b.CL, std::min(p.M, b.group), swi) + 1024;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(b.clusters * b.CL);
  cfg.blockDim = dim3(kSkThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute at[2];
  int na = 0;
  if (b.CL > 1) {
    at[na].id = cudaLaunchAttributeClusterDimension;
    at[na].val.clusterDim.x = b.CL;
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
  return cudaLaunchKernelEx(&cfg, fp4_skinny_kernel<NV, T, WIDE, INLINE>, p, b);
}

// a launch of fp4_expand costs about 3 tiles, so a plan with the expansion in the kernel may be that much worse
template <bool NV>
static bool expand_inline_t(int M, int64_t N, int K, bool swi) {
  int dev = 0;
  SkPlan b;
  double in = 0, sep = 0;
  return M <= 8 && cudaGetDevice(&dev) == cudaSuccess &&
         sk_plan<NV, kTerms, false, true>(M, N, K, 16, swi, dev, b, in) == cudaSuccess &&
         sk_plan<NV, kTerms, false, false>(M, N, K, 16, swi, dev, b, sep) == cudaSuccess && in <= sep + 3;
}

template <bool NV>
static cudaError_t skinny_t(const Fp4SkinnyArgs& p, cudaStream_t st) {
  if (p.x) return launch_skinny<NV, kTerms, false, true>(p, st);
  if (p.terms == 1) return launch_skinny<NV, 1, true, false>(p, st);
  return p.M <= 16 ? launch_skinny<NV, kTerms, false, false>(p, st) : launch_skinny<NV, kTerms, true, false>(p, st);
}

}  // namespace fp4
}  // namespace g53

using namespace g53;

int g53_fp4_terms() { return fp4::kTerms; }

bool g53_fp4_expand_inline(int M, int64_t N, int K, int nv, bool swiglu) {
  return nv ? fp4::expand_inline_t<true>(M, N, K, swiglu) : fp4::expand_inline_t<false>(M, N, K, swiglu);
}

cudaError_t g53_fp4_expand(const Fp4ExpandArgs& p, cudaStream_t st) {
  if (p.M < 1 || p.M > 65535 || p.K < 16 || p.K % (p.nv ? 16 : 32)) return cudaErrorInvalidValue;
  const dim3 grid((fp4::tiles_k(p.K) * 32 + 255) / 256, p.M);
  return p.nv ? g53_launch_pdl(fp4::fp4_expand_kernel<true>, grid, dim3(256), 0, st, 1, p)
              : g53_launch_pdl(fp4::fp4_expand_kernel<false>, grid, dim3(256), 0, st, 1, p);
}

cudaError_t g53_fp4_skinny(const Fp4SkinnyArgs& p, cudaStream_t st) {
  if (p.M < 1 || p.N < 1 || (p.x && p.M > 8) || p.K < 16 || p.K % (p.nv ? 16 : 32)) return cudaErrorInvalidValue;
  return p.nv ? fp4::skinny_t<true>(p, st) : fp4::skinny_t<false>(p, st);
}

cudaError_t g53_fp4_skinny_error(int* code, cudaStream_t st) { return fp4::copy_error(fp4::g_skinny_err, code, st); }
