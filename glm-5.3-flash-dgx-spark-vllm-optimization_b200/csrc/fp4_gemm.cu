// Large-M product of two 4-bit matrices on the block-scaled tensor cores: Y[M, N] = A4[M, K] @ W4[N, K]^T (W4A4).
//
// tcgen05.mma kind::mxf4nvf4 (nvfp4: scale_vec::4X, one e4m3 scale per 16) and kind::mxf4 (mxfp4: scale_vec::2X, one E8M0
// scale per 32): the tensor core multiplies e2m1 codes, applies both block scales and sums in fp32, at four times the
// bf16 rate.  Row scales (nvfp4) are applied to the fp32 result.
//
// Persistent, one CTA per SM.  Both operands are tile images (fp4.cuh), so a K step of 256 is one contiguous cp.async.bulk
// per 128-row block and array, already swizzled.  Two forms:
//   PAIR    256 x 256 tiles by a cluster of two CTAs (cta_group::2): each holds 128 rows of A, half of the tile's rows of W
//           and all of its scales, so a step brings 38 KB into an SM (nvfp4) where a CTA alone with 128 x 256 needs 54 KB;
//           (8192 x 24576 x 4096 mxfp4: 390 us, 460 alone)
//   single  128 x 128 tiles, for fewer tiles than would fill the SMs in pairs
// Tiles go in bands of 8 row blocks (pairs: 8 pairs).  Warp roles:
//   warp 0    producer: fills the ring, continuously across tiles
//   warp 1    allocates TMEM; one thread (of rank 0) copies the block scales of the stage to TMEM (tcgen05.cp, executed in
//             order with the mma of the same thread) and issues the four K = 64 mma of the stage.  Rank 1's thread passes
//             on that its stage has landed (a plain arrival: with a cluster-scope release it took 1000 clocks a stage)
//   warps 2-9 epilogue: tcgen05.ld, row scales, output (four warps, one per scheduler, take longer over the SwiGLU epilogue
//             than the main loop: 700 us instead of 340 for 8192 x 24576 x 4096)
// TMEM (512 columns): scales at 448..495; a pair's two accumulators are columns 0..255 and 192..447.  They share 64
// columns, which the epilogue of a tile reads first and then hands back, so the main loop of the next tile waits for a
// quarter of the epilogue's loads only.
//
// GEMV_SWIGLU: W4 is a gate/up image (per 128-row block 64 gate rows, then their 64 up rows); the epilogue forms
// silu(min(g, L)) * clip(u, -L, L) in fp32 and quantises it in place: a thread holds 32 consecutive activations of one row,
// a whole 16-byte chunk of the 4-bit image that the down projection reads.  The nvfp4 row scale cannot wait for the row's
// maximum (other CTAs hold the rest of the row), so it is the one that fits max(L, 0.2785) * L, which no activation exceeds
// (silu's lowest value is -0.27847); the e4m3 block scales keep their precision down to about 2^-14 of that.
//
// Waits are bounded; a timeout sets the error word, the roles stop issuing, wait for what they have in flight, and the
// TMEM is freed.
#include <algorithm>
#include <atomic>
#include "fp4.cuh"
#include "fp4_tc.cuh"
#include "launchers.h"

namespace g53 {
namespace fp4 {

__device__ int g_gemm_err = 0;

constexpr int kEpiWarps = 8;
constexpr int kGemmThreads = 64 + kEpiWarps * 32;
constexpr int kBandM = 8;
constexpr uint32_t kSfA = 448, kSfB = 464;            // TMEM columns of the scales

template <bool NV, bool PAIR>
struct GemmCfg {
  static constexpr int kBN = PAIR ? 256 : 128;        // columns of a tile
  static constexpr int kNB = kBN / 128;               // 128-row blocks of W per tile
  static constexpr int kSB = Fmt<NV>::kScaleBytes;
  static constexpr int kAtoms = kSB / 512;            // scale atoms per block and stage
  // a stage: codes of A, codes of W (one block each), scales of A, scales of W (all of the tile)
  static constexpr int kOffSA = 2 * kTileBytes, kOffSB = kOffSA + kSB;
  static constexpr int kStage = kOffSB + kNB * kSB;
  static constexpr int kStages = (226 * 1024 - 1024) / kStage > 6 ? 6 : (226 * 1024 - 1024) / kStage;
  static constexpr int kSmem = kStages * kStage + 1024;
  static constexpr uint32_t kBuf = PAIR ? 192 : 128;  // column of the second accumulator
  static_assert(kStage % 1024 == 0, "tiles are 1024-byte aligned");
};

__device__ __forceinline__ void tile_mn(int t, int MT, int NT, int& m, int& n) {
  const int band = t / (kBandM * NT);
  const int gm = min(kBandM, MT - band * kBandM);
  const int idx = t - band * kBandM * NT;
  m = band * kBandM + idx % gm;
  n = idx / gm;
}

// a warp's 32 x 32 block, a row per lane -> a column per lane
__device__ __forceinline__ void transpose32(float (&v)[32]) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int s = 16; s > 0; s >>= 1) {
    const bool up = lane & s;
#pragma unroll
    for (int i = 0; i < 32; ++i) {
      if (i & s) continue;
      const float other = __shfl_xor_sync(0xffffffffu, up ? v[i] : v[i | s], s);
      if (up) v[i] = other;
      else v[i | s] = other;
    }
  }
}

// 32 columns nb.. of the warp's 32 rows, `row` that of this lane.  16-byte aligned rows are stored by their lanes; others go
// out a row at a time, 32 lanes side by side (2786 x 3916 x 1728 in bf16: 53 us, 151 with a lane's own row element by
// element, which only the last columns of aligned rows take).
__device__ __forceinline__ void store32(const Fp4GemmArgs& p, int row, int nb, RowScale rs, float (&v)[32]) {
  const bool full = nb + 32 <= p.N, acc = p.mode == GEMV_F32_ACC;
  if (p.b_row) {
#pragma unroll
    for (int i = 0; i < 32; i += 4) {
      if (full) {
        const float4 t = __ldcg(reinterpret_cast<const float4*>(p.b_row + nb + i));
        v[i] *= rs.a * t.x; v[i + 1] *= rs.a * t.y; v[i + 2] *= rs.a * t.z; v[i + 3] *= rs.a * t.w;
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (nb + i + j < p.N) v[i + j] *= rs.a * __ldcg(p.b_row + nb + i + j);
      }
    }
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] *= rs.b;
  }
  if (!p.vec) {
    transpose32(v);
    const int lane = threadIdx.x & 31, r0 = row - lane, n = nb + lane;
    if (n >= p.N) return;
#pragma unroll
    for (int i = 0; i < 32; ++i) {
      if (r0 + i >= p.M) break;
      const int64_t off = (int64_t)(r0 + i) * p.ldy + n;
      if (p.mode == GEMV_BF16) {
        reinterpret_cast<__nv_bfloat16*>(p.y)[off] = f2bf(v[i]);
      } else {
        float* y = reinterpret_cast<float*>(p.y) + off;
        *y = acc ? __ldcg(y) + v[i] : v[i];
      }
    }
    return;
  }
  if (row >= p.M) return;
  const int64_t off = (int64_t)row * p.ldy + nb;
  if (p.mode == GEMV_BF16) {
    __nv_bfloat16* y = reinterpret_cast<__nv_bfloat16*>(p.y) + off;
    if (!full) {
#pragma unroll
      for (int i = 0; i < 32; ++i)
        if (nb + i < p.N) y[i] = f2bf(v[i]);
      return;
    }
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      uint32_t w[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        __nv_bfloat162 b = __floats2bfloat162_rn(v[c * 8 + 2 * i], v[c * 8 + 2 * i + 1]);
        w[i] = *reinterpret_cast<uint32_t*>(&b);
      }
      reinterpret_cast<uint4*>(y)[c] = make_uint4(w[0], w[1], w[2], w[3]);
    }
    return;
  }
  float* y = reinterpret_cast<float*>(p.y) + off;
  if (!full) {
#pragma unroll
    for (int i = 0; i < 32; ++i)
      if (nb + i < p.N) y[i] = acc ? __ldcg(y + i) + v[i] : v[i];
    return;
  }
#pragma unroll
  for (int c = 0; c < 8; ++c) {
    float4 o = make_float4(v[4 * c], v[4 * c + 1], v[4 * c + 2], v[4 * c + 3]);
    if (acc) {
      const float4 t = __ldcg(reinterpret_cast<const float4*>(y) + c);
      o.x += t.x; o.y += t.y; o.z += t.z; o.w += t.w;
    }
    reinterpret_cast<float4*>(y)[c] = o;
  }
}

// 32 activations j0.. of one row: gate (v) and up (u) sums -> 4-bit chunk and block scales of the output image
template <bool NV>
__device__ __forceinline__ void swiglu32(const Fp4GemmArgs& p, int row, int j0, int r0, float rs, float (&v)[32],
                                         float (&u)[32]) {
  const float L = p.limit;
#pragma unroll
  for (int i = 0; i < 32; i += 4) {
    float4 sg = make_float4(1.f, 1.f, 1.f, 1.f), su = sg;
    if constexpr (NV) {
      sg = __ldcg(reinterpret_cast<const float4*>(p.b_row + r0 + i));
      su = __ldcg(reinterpret_cast<const float4*>(p.b_row + r0 + 64 + i));
    }
    const float gs[4] = {sg.x, sg.y, sg.z, sg.w}, us[4] = {su.x, su.y, su.z, su.w};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      float g = v[i + k], w = u[i + k];
      if constexpr (NV) {
        // one scale after the other: their product may leave fp32 (and 0 * inf is NaN).  In this order a sum overflows on the
        // way only where the weights' scale is above 2^90; RowScale's third product would cost the epilogue 2%
        g = g * gs[k] * rs;
        w = w * us[k] * rs;
      }
      g = g > L ? L : g;                              // written so that a NaN stays one
      w = w > L ? L : w < -L ? -L : w;
      // g <= L; exp(-g) that overflows leaves g / inf = -0, and __fdividef is 0 there too
      v[i + k] = __fdividef(g, 1.f + __expf(-g)) * w;
    }
  }
  const int rr = row % kTileRows, kt = j0 / kTileK, c = (j0 % kTileK) / 32;
  const int64_t tile = (int64_t)(row / kTileRows) * tiles_k(p.width) + kt;
  uint32_t code[4];
  uint32_t sc = 0;
  if constexpr (NV) {
    const float down = pow2i(-p.h_exp);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      uint32_t am = 0;
#pragma unroll
      for (int i = 0; i < 16; ++i) am = max(am, __float_as_uint(v[h * 16 + i]) & 0x7fffffffu);
      const uint32_t b = am >= kInfBits ? 0x7fu : nv_scale(__uint_as_float(am) * down);
      const float s = e4m3_to_f32(b);
      const float inv = s > 0.f ? __frcp_rn(s) * down : 0.f;
      sc |= b << (8 * h);
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        float f[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = v[h * 16 + k * 8 + i] * inv;
        code[h * 2 + k] = f32x8_to_e2m1(f);
      }
    }
    *reinterpret_cast<uint16_t*>(p.out_scales + tile * Fmt<NV>::kScaleBytes + scale_off(rr, 2 * c)) = (uint16_t)sc;
  } else {
    uint32_t am = 0;
#pragma unroll
    for (int i = 0; i < 32; ++i) am = max(am, __float_as_uint(v[i]) & 0x7fffffffu);
    sc = mx_scale(am);
    const float inv = sc == 255u ? 0.f : pow2i(127 - (int)sc);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      float f[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) f[i] = v[k * 8 + i] * inv;
      code[k] = f32x8_to_e2m1(f);
    }
    p.out_scales[tile * Fmt<NV>::kScaleBytes + scale_off(rr, c)] = (uint8_t)sc;
  }
  *reinterpret_cast<uint4*>(p.out_codes + tile * kTileBytes + chunk_off(rr, c)) =
      make_uint4(code[0], code[1], code[2], code[3]);
}

template <bool NV, bool PAIR, bool SWI>
__global__ void __launch_bounds__(kGemmThreads, 1) fp4_gemm_kernel(Fp4GemmArgs p) {
  using C = GemmCfg<NV, PAIR>;
  constexpr int kStages = C::kStages, kG = PAIR ? 2 : 1, BN = C::kBN;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  __shared__ __align__(8) uint64_t full[kStages], empty[kStages], tfull[2], tempty[2], drain;
  __shared__ uint32_t tmem_s;
  __shared__ int fail_s;
  volatile int* fail = &fail_s;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = PAIR ? (int)(blockIdx.x & 1) : 0;
  const int KT = tiles_k(p.K);
  const int ksteps = (p.K + 63) / 64;
  const int MB = (p.M + 127) / 128, NB = (p.N + 127) / 128;
  const int MT = (MB + kG - 1) / kG, NT = (NB + C::kNB - 1) / C::kNB;
  const int tiles = MT * NT;
  const int t0 = (int)blockIdx.x / kG, tstep = (int)gridDim.x / kG;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      // rank 0 of a pair: its own copies, and word from rank 1 that its have landed
      tc::bar_init(&full[s], PAIR && rank == 0 ? 2 : 1);
      tc::bar_init(&empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      tc::bar_init(&tfull[b], 1);
      tc::bar_init(&tempty[b], kG * kEpiWarps);
    }
    tc::bar_init(&drain, 1);
    fail_s = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    if constexpr (PAIR) tmem_alloc_pair(&tmem_s, 512);
    else tc::tmem_alloc(&tmem_s, 512);
  }
  tc::fence_before();
  __syncthreads();
  if constexpr (PAIR) {
    cluster_arrive();
    cluster_wait();
  }
  tc::fence_after();
  const uint32_t tmem = tmem_s;
  pdl_trigger();
  pdl_wait();

  if (warp == 0) {
    if (elect_one()) {
      uint32_t it = 0;
      bool ok = true;
      for (int t = t0; t < tiles && ok; t += tstep) {
        int mt, nt;
        tile_mn(t, MT, NT, mt, nt);
        const int mb = mt * kG + rank;                 // this CTA's rows of A
        const int nb = nt * C::kNB + rank;             // and of W
        const int nsc = min(C::kNB, NB - nt * C::kNB); // blocks of W that exist
        const bool has_a = mb < MB, has_b = nb < NB;
        const uint32_t bytes = (has_a ? kTileBytes + C::kSB : 0) + (has_b ? kTileBytes : 0) + nsc * C::kSB;
        for (int kt = 0; kt < KT; ++kt, ++it) {
          const int s = it % kStages;
          if (it >= kStages && !tc::bar_wait(&empty[s], ((it / kStages) - 1) & 1, fail, &g_gemm_err, 1)) {
            ok = false;
            break;
          }
          uint8_t* st = smem + s * C::kStage;
          bulk_expect(&full[s], bytes);
          if (has_a) {
            const int64_t ta = (int64_t)mb * KT + kt;
            bulk_load(st, p.a_codes + ta * kTileBytes, kTileBytes, &full[s]);
            bulk_load(st + C::kOffSA, p.a_scales + ta * C::kSB, C::kSB, &full[s]);
          }
          if (has_b) bulk_load(st + kTileBytes, p.b_codes + ((int64_t)nb * KT + kt) * kTileBytes, kTileBytes, &full[s]);
          for (int b = 0; b < nsc; ++b)
            bulk_load(st + C::kOffSB + b * C::kSB, p.b_scales + ((int64_t)(nt * C::kNB + b) * KT + kt) * C::kSB, C::kSB,
                      &full[s]);
        }
      }
      if (*fail) {
        const uint32_t first = it > (uint32_t)kStages ? it - kStages : 0;
        int none = 0;
        for (uint32_t j = first; j < it; ++j) tc::bar_wait(&full[j % kStages], (j / kStages) & 1, &none, nullptr, 0);
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    if (elect_one()) {
      uint32_t it = 0, tl = 0;
      bool ok = true;
      for (int t = t0; t < tiles && ok; t += tstep, ++tl) {
        if (PAIR && rank == 1) {
          for (int kt = 0; kt < KT; ++kt, ++it) {
            const int s = it % kStages;
            if (!tc::bar_wait(&full[s], (it / kStages) & 1, fail, &g_gemm_err, 5)) { ok = false; break; }
            signal_at(&full[s], 0);
          }
          continue;
        }
        const uint32_t buf = tl & 1;
        // pairs: the shared columns of the tile before; single: the buffer's last tile
        const uint32_t lag = PAIR ? 1 : 2;
        if (tl >= lag &&
            !tc::bar_wait(&tempty[(tl - lag) & 1], ((tl - lag) >> 1) & 1, fail, &g_gemm_err, 4)) break;
        tc::fence_after();
        const uint32_t d = tmem + buf * C::kBuf;
        for (int kt = 0; kt < KT; ++kt, ++it) {
          const int s = it % kStages;
          if (!tc::bar_wait(&full[s], (it / kStages) & 1, fail, &g_gemm_err, 2)) {
            ok = false;
            break;
          }
          tc::fence_after();
          const uint32_t a = tc::saddr(smem + s * C::kStage), b = a + kTileBytes;
#pragma unroll
          for (int at = 0; at < C::kAtoms; ++at) {
            copy_scales<kG>(tmem + kSfA + at * 4, a + C::kOffSA + at * 512);
#pragma unroll
            for (int nb = 0; nb < C::kNB; ++nb)
              copy_scales<kG>(tmem + kSfB + at * (4 * C::kNB) + nb * 4, a + C::kOffSB + nb * C::kSB + at * 512);
          }
          const int n = min(4, ksteps - kt * 4);
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            if (k >= n) break;
            const int at = NV ? k : k >> 1;
            const uint32_t sf = NV ? 0u : (uint32_t)(k & 1) * 2;
            mma4<NV, kG>(d, tc::desc_sw128(a + k * 32), tc::desc_sw128(b + k * 32), idesc4(128 * kG, BN, !NV, sf),
                         tmem + kSfA + at * 4, tmem + kSfB + at * (4 * C::kNB), (kt > 0 || k > 0) ? 1u : 0u);
          }
          if constexpr (PAIR) commit_pair(&empty[s]);
          else tc::commit(&empty[s]);
        }
        if (ok) {
          if constexpr (PAIR) commit_pair(&tfull[buf]);
          else tc::commit(&tfull[buf]);
        }
      }
      if (*fail && rank == 0) {
        int none = 0;
        if constexpr (PAIR) commit_pair(&drain);
        else tc::commit(&drain);
        tc::bar_wait(&drain, 0, &none, nullptr, 0);
      }
    }
    __syncwarp();
  } else {
    // two warps per TMEM lane quadrant; `part` 0 takes the half of the tile with the shared columns.  Its arrival on
    // tempty says that those are read; that of part 1, that it is done with the tile before
    const int quad = warp & 3, part = (warp - 2) >> 2;
    uint32_t tl = 0;
    for (int t = t0; t < tiles; t += tstep, ++tl) {
      const uint32_t buf = tl & 1;
      int mt, nt;
      tile_mn(t, MT, NT, mt, nt);
      if (!tc::warp_wait(&tfull[buf], (tl >> 1) & 1, fail, &g_gemm_err, 3)) break;
      tc::fence_after();
      const int row = (mt * kG + rank) * 128 + quad * 32 + lane;
      const bool live = row < p.M;
      const float rs = p.a_row && live ? __ldcg(p.a_row + row) : p.a_const;
      const uint32_t base = tmem + ((uint32_t)(quad * 32) << 16) + buf * C::kBuf;
      auto release = [&]() {
        tc::fence_before();
        __syncwarp();
        if (lane == 0) {
          if (PAIR && rank == 1) signal_at(&tempty[buf], 0);
          else tc::bar_arrive(&tempty[buf]);
        }
      };
      if (PAIR && part == 1) release();
      if constexpr (SWI) {
        const int wide = ((p.width + 63) / 64) * 64;
        if constexpr (PAIR) {
          // a block (64 gate, 64 up columns) per part.  The shared columns are the up half of block 1 (buffer 0) or the gate
          // half of block 0 (buffer 1)
          const int blk = buf == 0 ? 1 - part : part;
          const int nblk = nt * 2 + blk;
          const uint32_t first = buf == 0 ? 64u : 0u;
          float x0[32], x1[32], w[32];
          tc::tmem_ld32(base + blk * 128 + first, x0);
          tc::tmem_ld32(base + blk * 128 + first + 32, x1);
          if (part == 0) release();
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            tc::tmem_ld32(base + blk * 128 + (64u - first) + h * 32, w);
            const int j0 = nblk * 64 + h * 32;
            if (live && j0 < wide) {
              const int r0 = nblk * 128 + h * 32;
              if (buf == 0) swiglu32<NV>(p, row, j0, r0, rs, w, h == 0 ? x0 : x1);
              else swiglu32<NV>(p, row, j0, r0, rs, h == 0 ? x0 : x1, w);
            }
          }
        } else {
          float g[32], u[32];
          tc::tmem_ld32(base + part * 32, g);
          tc::tmem_ld32(base + 64 + part * 32, u);
          release();
          const int j0 = nt * 64 + part * 32;
          if (live && j0 < wide) swiglu32<NV>(p, row, j0, nt * 128 + part * 32, rs, g, u);
        }
      } else {
        const int n0 = nt * BN;
        constexpr int kUnits = BN / 128;              // units of 64 columns per part
#pragma unroll 1
        for (int i = 0; i < kUnits; ++i) {
          // buffer 0 of a pair: units 3, 2 and 0, 1
          const int u = PAIR && buf == 0 ? (part == 0 ? 3 - i : i) : part * kUnits + i;
          float x0[32], x1[32];
          tc::tmem_ld32(base + u * 64, x0);
          tc::tmem_ld32(base + u * 64 + 32, x1);
          if (PAIR ? part == 0 && i == 0 : true) release();
          if (n0 + u * 64 < p.N) store32(p, row, n0 + u * 64, split_scale(rs), x0);
          if (n0 + u * 64 + 32 < p.N) store32(p, row, n0 + u * 64 + 32, split_scale(rs), x1);
        }
      }
    }
  }
  tc::fence_before();
  __syncthreads();
  if constexpr (PAIR) {
    // rank 0's mma read rank 1's shared memory and write its TMEM; rank 1 arrives on rank 0's barriers
    cluster_arrive();
    cluster_wait();
  }
  if (warp == 1) {
    tc::fence_after();
    if constexpr (PAIR) tmem_free_pair(tmem, 512);
    else tc::tmem_free(tmem, 512);
  }
}

constexpr int kMaxDev = 64;

// SMs of the current device
static cudaError_t sm_count(int dev, int* out) {
  static std::atomic<int> known[kMaxDev];
  if (dev < kMaxDev && (*out = known[dev].load(std::memory_order_relaxed)) > 0) return cudaSuccess;
  const cudaError_t e = cudaDeviceGetAttribute(out, cudaDevAttrMultiProcessorCount, dev);
  if (e == cudaSuccess && dev < kMaxDev) known[dev].store(*out, std::memory_order_relaxed);
  return e;
}

template <bool NV, bool PAIR, bool SWI>
static cudaError_t launch_gemm(const Fp4GemmArgs& p, int dev, int sms, cudaStream_t st) {
  using C = GemmCfg<NV, PAIR>;
  auto kern = fp4_gemm_kernel<NV, PAIR, SWI>;
  static std::atomic<bool> ready[kMaxDev];            // the shared memory limit, raised once per device
  if (dev >= kMaxDev || !ready[dev].load(std::memory_order_relaxed)) {
    const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem);
    if (e != cudaSuccess) return e;
    if (dev < kMaxDev) ready[dev].store(true, std::memory_order_relaxed);
  }
  constexpr int kG = PAIR ? 2 : 1;
  const int64_t tiles = (((int64_t)p.M + 128 * kG - 1) / (128 * kG)) * (((int64_t)p.N + C::kBN - 1) / C::kBN);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)std::min<int64_t>(tiles, sms / kG) * kG);
  cfg.blockDim = dim3(kGemmThreads);
  cfg.dynamicSmemBytes = C::kSmem;
  cfg.stream = st;
  cudaLaunchAttribute at[2];
  int na = 0;
  if (PAIR) {
    at[na].id = cudaLaunchAttributeClusterDimension;
    at[na].val.clusterDim.x = 2;
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
  return cudaLaunchKernelEx(&cfg, kern, p);
}

template <bool NV>
static cudaError_t gemm_t(const Fp4GemmArgs& p, int dev, int sms, cudaStream_t st) {
  const bool pair = (int64_t)((p.M + 255) / 256) * ((p.N + 255) / 256) >= sms / 2;
  if (p.mode == GEMV_SWIGLU)
    return pair ? launch_gemm<NV, true, true>(p, dev, sms, st) : launch_gemm<NV, false, true>(p, dev, sms, st);
  return pair ? launch_gemm<NV, true, false>(p, dev, sms, st) : launch_gemm<NV, false, false>(p, dev, sms, st);
}

}  // namespace fp4
}  // namespace g53

using namespace g53;

cudaError_t g53_fp4_gemm(const Fp4GemmArgs& p, cudaStream_t st) {
  if (p.M < 1 || p.N < 1 || p.K < 16 || p.K % (p.nv ? 16 : 32)) return cudaErrorInvalidValue;
  int dev = 0, sms = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess) e = fp4::sm_count(dev, &sms);
  if (e != cudaSuccess) return e;
  Fp4GemmArgs q = p;
  const int esz = p.mode == GEMV_BF16 ? 2 : 4;
  q.vec = (reinterpret_cast<uintptr_t>(p.y) & 15) == 0 && ((p.ldy * esz) & 15) == 0 ? 1 : 0;
  return p.nv ? fp4::gemm_t<true>(q, dev, sms, st) : fp4::gemm_t<false>(q, dev, sms, st);
}

cudaError_t g53_fp4_gemm_error(int* code, cudaStream_t st) { return fp4::copy_error(fp4::g_gemm_err, code, st); }
