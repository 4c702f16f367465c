// Quantisation of bf16 / f16 rows to 4-bit floating point (mxfp4, nvfp4) and the read-back, on the tile images of
// fp4.cuh.
//
// fp4_quantize: per block a maximum of magnitudes, a scale from it, 16 codes per thread.  The row (nvfp4 needs its
// maximum first) stays in registers between the two uses, so the input is read once.  Both kernels move 2 + 1/2 + 1/16
// (1/32) bytes per element, and HBM is their floor; 8192 x 8192 in nvfp4 is quantised at 0.73 of the copy rate, with 67 % of
// the issue slots used: a row's load, maxima and stores follow one another.
// Launched programmatically, so what earlier kernels wrote is read from L2 (__ldcg), not through the read-only path.
// Infinities and NaN: an mxfp4 block that holds one reads back as NaN, an nvfp4 row that holds one likewise (its row
// scale is NaN).  Magnitudes are compared as integers, so a NaN counts as the largest.
#include <algorithm>
#include "fp4.cuh"
#include "launchers.h"

namespace g53 {
namespace fp4 {

template <bool F16>
__device__ __forceinline__ void unpack2(uint32_t w, float& lo, float& hi) {
  if constexpr (F16) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w));
    lo = f.x;
    hi = f.y;
  } else {
    lo = __uint_as_float(w << 16);
    hi = __uint_as_float(w & 0xffff0000u);
  }
}

// T threads per row (32, 64, 128 or 256 of the CTA's 256), up to B blocks of 16 elements per thread in registers; rows
// longer than 16 * T * B are walked twice (REREAD: the second walk hits L2).  Few threads per row keep more 16-byte
// loads in flight per thread; the launcher takes the smallest T whose registers hold the row.
template <bool NV, bool F16, int T, int B, bool REREAD>
__global__ void __launch_bounds__(256) fp4_quantize_kernel(Fp4QuantArgs p) {
  constexpr int kRows = 256 / T;
  __shared__ uint32_t red[8];
  const int sub = threadIdx.x / T, t = threadIdx.x % T;
  const int64_t row = (int64_t)blockIdx.x * kRows + sub;
  const bool live = row < p.R;
  const int KT = tiles_k(p.K);
  const int nb = KT * 16;                            // blocks of 16, padding included
  const int nk = (int)(p.K / 16);
  const uint16_t* x = reinterpret_cast<const uint16_t*>(p.x) + (live ? row : 0) * p.ldx;
  pdl_trigger();
  pdl_wait();

  auto load = [&](int b, uint32_t (&w)[8]) {
    if (live && b < nk) {
      if (p.vec) {
        const uint4* v = reinterpret_cast<const uint4*>(x + (int64_t)b * 16);
        const uint4 a = __ldcg(v), c = __ldcg(v + 1);
        w[0] = a.x; w[1] = a.y; w[2] = a.z; w[3] = a.w;
        w[4] = c.x; w[5] = c.y; w[6] = c.z; w[7] = c.w;
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          w[i] = (uint32_t)__ldcg(x + (int64_t)b * 16 + 2 * i) | ((uint32_t)__ldcg(x + (int64_t)b * 16 + 2 * i + 1) << 16);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) w[i] = 0u;
    }
  };
  // bits (fp32) of the block's largest magnitude
  auto amax16 = [&](const uint32_t (&w)[8]) {
    uint32_t a = w[0] & 0x7fff7fffu;
#pragma unroll
    for (int i = 1; i < 8; ++i) a = max_u16x2(a, w[i] & 0x7fff7fffu);
    const uint32_t m = max(a & 0xffffu, a >> 16);
    if constexpr (F16) {
      if (m >= 0x7c00u) return kInfBits;
      return __float_as_uint(__half2float(__ushort_as_half((unsigned short)m)));
    } else {
      return m << 16;
    }
  };

  uint32_t w[B][8];
  uint32_t am[B];
  uint32_t rmax = 0u;
#pragma unroll
  for (int i = 0; i < B; ++i) load(t + i * T, w[i]);
#pragma unroll
  for (int i = 0; i < B; ++i) {
    am[i] = amax16(w[i]);
    rmax = max(rmax, am[i]);
  }
  if constexpr (REREAD) {
    for (int b = t + B * T; b < nk; b += T) {
      uint32_t v[8];
      load(b, v);
      rmax = max(rmax, amax16(v));
    }
  }
  float down = 1.f;                                   // 2^-k of the row
  if constexpr (NV) {
    rmax = __reduce_max_sync(0xffffffffu, rmax);
    if constexpr (T > 32) {
      if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = rmax;
      __syncthreads();
#pragma unroll
      for (int i = 0; i < T / 32; ++i) rmax = max(rmax, red[sub * (T / 32) + i]);
    }
    const int k = rmax >= kInfBits ? 0 : nv_row_exp(rmax);
    down = pow2i(-k);
    if (live && t == 0) p.row_scale[row] = rmax >= kInfBits ? __uint_as_float(0x7fc00000u) : pow2i(k);
  }

  const int64_t tile0 = (row / kTileRows) * KT;
  const int rr = (int)(row % kTileRows);
  auto emit = [&](int b, const uint32_t (&v)[8], uint32_t amax) {
    uint32_t sc;
    float inv;
    if constexpr (NV) {
      const float a = __uint_as_float(amax) * down;
      sc = amax >= kInfBits ? 0x7fu : nv_scale(a);
      const float s = e4m3_to_f32(sc);
      inv = s > 0.f ? __frcp_rn(s) * down : 0.f;      // down >= 2^-117: no underflow of note
    } else {
      amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 1));     // the other half of the 32-block
      sc = mx_scale(amax);
      inv = sc == 255u ? 0.f : pow2i(127 - (int)sc);
    }
    uint32_t code[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float f[8];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float lo, hi;
        unpack2<F16>(v[4 * h + i], lo, hi);
        if constexpr (NV) {
          f[2 * i] = scaled_on_grid(lo, inv);
          f[2 * i + 1] = scaled_on_grid(hi, inv);
        } else {                                       // exact: the scale is a power of two
          f[2 * i] = lo * inv;
          f[2 * i + 1] = hi * inv;
        }
      }
      code[h] = f32x8_to_e2m1(f);
    }
    if (b >= nk) sc = 0u;
    const int kt = b >> 4, kb = b & 15;               // tile, block of 16 inside it
    const int64_t tile = tile0 + kt;
    if (live && b < nb) {
      uint2* dst = reinterpret_cast<uint2*>(p.codes + tile * kTileBytes + chunk_off(rr, kb >> 1) + (kb & 1) * 8);
      *dst = make_uint2(code[0], code[1]);
    }
    // four scale bytes of one atom row -> one 32-bit store
    constexpr int kStep = NV ? 1 : 2;
    uint32_t s4 = sc;
    s4 |= __shfl_down_sync(0xffffffffu, sc, kStep) << 8;
    s4 |= __shfl_down_sync(0xffffffffu, sc, 2 * kStep) << 16;
    s4 |= __shfl_down_sync(0xffffffffu, sc, 3 * kStep) << 24;
    if (live && b < nb && (kb & (4 * kStep - 1)) == 0) {
      uint8_t* sb = p.scales + tile * Fmt<NV>::kScaleBytes + scale_off(rr, kb / kStep);
      *reinterpret_cast<uint32_t*>(sb) = s4;
    }
  };
  // nb is a multiple of 16 and T of 32, so the four (eight) lanes of a scale word are in range together
#pragma unroll
  for (int i = 0; i < B; ++i)
    if ((i * T) < nb) emit(t + i * T, w[i], am[i]);
  if constexpr (REREAD) {
    for (int b0 = B * T; b0 < nb; b0 += T) {
      uint32_t v[8];
      load(b0 + t, v);
      emit(b0 + t, v, amax16(v));
    }
  }
}

// Read-back: a thread turns 8 codes (one word) into 8 outputs; 32 consecutive threads cover one tile row (256 columns),
// so code loads are 128 contiguous bytes per warp and 16-bit stores 512.  Exact in fp32; rounded once to 16 bits.
// CTA: 8 rows (a warp each) x 4 tiles: 777 x 12288 5.6 us (6.1 with 8 tiles, 8.6 with 16, 5.9 with 2); 8192 x 12288 takes 55
// with any of them, 4.7 TB/s of which four fifths are writes.
constexpr int kDqTiles = 4;
template <bool NV, int OUT>                           // OUT 0 bf16, 1 f16, 2 fp32
__global__ void __launch_bounds__(256) fp4_dequant_kernel(Fp4DequantArgs p) {
  const int KT = tiles_k(p.K);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t row = (int64_t)blockIdx.x * 8 + warp;
  pdl_trigger();
  pdl_wait();
  if (row >= p.R) return;
  const int rr = (int)(row % kTileRows);
  const float rs = NV ? __ldcg(p.row_scale + row) : 1.f;
  // (a grid has 65535 CTAs in y: longer rows go round)
  for (int kt0 = blockIdx.y * kDqTiles; kt0 < KT; kt0 += gridDim.y * kDqTiles) {
#pragma unroll
    for (int q = 0; q < kDqTiles; ++q) {
      const int kt = kt0 + q;
      const int64_t tile = (row / kTileRows) * KT + kt;
      const int64_t k0 = (int64_t)kt * kTileK + lane * 8;
      if (k0 >= p.K) continue;
      const uint32_t w =
          __ldcg(reinterpret_cast<const uint32_t*>(p.codes + tile * kTileBytes + chunk_off(rr, lane >> 2) + (lane & 3) * 4));
      const uint32_t sb = __ldcg(p.scales + tile * Fmt<NV>::kScaleBytes + scale_off(rr, NV ? lane >> 1 : lane >> 2));
      const float s = NV ? e4m3_to_f32(sb) * rs : e8m0_to_f32(sb);
      uint32_t h[4];
      e2m1x8_to_f16(w, h);
      float v[8];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h[i]));
        v[2 * i] = f.x * s;
        v[2 * i + 1] = f.y * s;
      }
      const int64_t off = row * p.ldy + k0;
      if constexpr (OUT == 2) {
        float* y = reinterpret_cast<float*>(p.y) + off;
        if (p.vec) {
          reinterpret_cast<float4*>(y)[0] = make_float4(v[0], v[1], v[2], v[3]);
          reinterpret_cast<float4*>(y)[1] = make_float4(v[4], v[5], v[6], v[7]);
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i) y[i] = v[i];
        }
      } else {
        uint32_t o[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if constexpr (OUT == 0) {
            __nv_bfloat162 b = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
            o[i] = *reinterpret_cast<uint32_t*>(&b);
          } else {
            o[i] = f32x2_to_f16x2(v[2 * i], v[2 * i + 1]);
          }
        }
        uint16_t* y = reinterpret_cast<uint16_t*>(p.y) + off;
        if (p.vec) {
          *reinterpret_cast<uint4*>(y) = make_uint4(o[0], o[1], o[2], o[3]);
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            y[2 * i] = (uint16_t)(o[i] & 0xffffu);
            y[2 * i + 1] = (uint16_t)(o[i] >> 16);
          }
        }
      }
    }
  }
}

template <bool NV, bool F16, int T, int B, bool REREAD>
static cudaError_t launch_q(const Fp4QuantArgs& p, cudaStream_t st) {
  constexpr int kRows = 256 / T;
  return g53_launch_pdl(fp4_quantize_kernel<NV, F16, T, B, REREAD>, dim3((unsigned)((p.R + kRows - 1) / kRows)), dim3(256),
                        0, st, 1, p);
}

template <bool NV, bool F16>
static cudaError_t quantize_t(const Fp4QuantArgs& p, cudaStream_t st) {
  const int nb = tiles_k(p.K) * 16;
  if (nb <= 128) return launch_q<NV, F16, 32, 4, false>(p, st);
  if (nb <= 256) return launch_q<NV, F16, 64, 4, false>(p, st);
  if (nb <= 512) return launch_q<NV, F16, 128, 4, false>(p, st);
  if (nb <= 1024) return launch_q<NV, F16, 256, 4, false>(p, st);
  return launch_q<NV, F16, 256, 4, true>(p, st);
}

template <bool NV>
static cudaError_t dequant_t(const Fp4DequantArgs& p, cudaStream_t st) {
  const dim3 grid((unsigned)((p.R + 7) / 8), std::min(65535, (tiles_k(p.K) + kDqTiles - 1) / kDqTiles));
  switch (p.out) {
    case 0: return g53_launch_pdl(fp4_dequant_kernel<NV, 0>, grid, dim3(256), 0, st, 1, p);
    case 1: return g53_launch_pdl(fp4_dequant_kernel<NV, 1>, grid, dim3(256), 0, st, 1, p);
    default: return g53_launch_pdl(fp4_dequant_kernel<NV, 2>, grid, dim3(256), 0, st, 1, p);
  }
}

}  // namespace fp4
}  // namespace g53

using namespace g53;

cudaError_t g53_fp4_quantize(const Fp4QuantArgs& p, cudaStream_t st) {
  if (p.R < 1 || p.K < 16 || p.K % (p.nv ? 16 : 32)) return cudaErrorInvalidValue;
  if (p.nv) return p.f16 ? fp4::quantize_t<true, true>(p, st) : fp4::quantize_t<true, false>(p, st);
  return p.f16 ? fp4::quantize_t<false, true>(p, st) : fp4::quantize_t<false, false>(p, st);
}

cudaError_t g53_fp4_dequant(const Fp4DequantArgs& p, cudaStream_t st) {
  if (p.R < 1 || p.K < 16 || p.K % (p.nv ? 16 : 32)) return cudaErrorInvalidValue;
  return p.nv ? fp4::dequant_t<true>(p, st) : fp4::dequant_t<false>(p, st);
}
