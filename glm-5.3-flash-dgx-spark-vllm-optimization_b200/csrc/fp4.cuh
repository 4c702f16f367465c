// 4-bit floating-point matrices (e2m1 codes with block scales): storage layout and element helpers shared by the
// quantiser (fp4_quant.cu), the small-M product (fp4_skinny.cu), the product that widens the weights (fp4_exact.cu) and the
// product of two 4-bit matrices (fp4_gemm.cu).
//
// Value of an element: e2m1(code) * block scale * row scale.
//   mxfp4   blocks of 32 along K, block scale 2^(b - 127) (one byte b, E8M0; 255 = NaN), no row scale
//   nvfp4   blocks of 16 along K, block scale e4m3 (0x7F = NaN), fp32 row scale (a power of two)
//
// Storage: a matrix [R, K] is kept as shared-memory images, so every product fetches a 128 x 256 tile with one
// contiguous cp.async.bulk per array (no tensor map, full DRAM bursts, any K that is a multiple of the block):
//   codes   [ceil(R / 128)][ceil(K / 256)][128 rows][128 bytes]: a row's 256 codes (low nibble first) in the 128-byte
//           swizzle of the K-major tcgen05 operand: 16-byte chunk c (32 codes) of row r sits at chunk c ^ (r % 8)
//   scales  [ceil(R / 128)][ceil(K / 256)][256 / block / 4][512 bytes]: 512-byte atoms of 128 rows x 4 block columns in
//           the order tcgen05.cp.32x128b.warpx4 carries to TMEM: byte (r % 32) * 16 + (r / 32) * 4 + column % 4
// Columns past K in the last tile hold zero codes and zero scales; rows past R are not written.
#pragma once
#include <cuda_fp4.h>

#include "common.cuh"

namespace g53 {
namespace fp4 {

constexpr int kTileRows = 128;
constexpr int kTileK = 256;
constexpr int kTileBytes = kTileRows * kTileK / 2;      // 16 KB of codes

template <bool NV>
struct Fmt {
  static constexpr int kBlock = NV ? 16 : 32;
  static constexpr int kCols = kTileK / kBlock;         // block scales per row and tile
  static constexpr int kScaleBytes = kTileRows * kCols; // per tile
};

__host__ __device__ __forceinline__ int tiles_k(int64_t K) { return (int)((K + kTileK - 1) / kTileK); }

// byte of 16-byte chunk c of row r inside a code tile
__device__ __forceinline__ int chunk_off(int r, int c) { return r * 128 + ((c ^ (r & 7)) << 4); }
// byte of block column s of row r inside a scale tile
__device__ __forceinline__ int scale_off(int r, int s) { return (s >> 2) * 512 + (r & 31) * 16 + (r >> 5) * 4 + (s & 3); }

// 8 codes (one 32-bit word) -> four f16x2, exact; o[i] holds codes 2i (low half) and 2i + 1.  Each byte goes into its .b8
// register through an explicit conversion: 62 values a clock and SM, 25 through CUDA's function of one byte.  (Unpacking
// the word into four .b8 registers at once came out of the assembler, 12.9, with bytes exchanged or lost, depending on what
// stood before it.)
__device__ __forceinline__ void e2m1x8_to_f16(uint32_t w, uint32_t (&o)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i)
    asm("{\n .reg .b8 a;\n cvt.u8.u32 a, %1;\n cvt.rn.f16x2.e2m1x2 %0, a;\n}\n" : "=r"(o[i]) : "r"(w >> (8 * i)));
}
// 8 values -> 8 codes (nearest, ties to even, saturating at 6)
__device__ __forceinline__ uint32_t f32x8_to_e2m1(const float (&v)[8]) {
  uint32_t r;
  asm("{\n .reg .b8 a, b, c, d;\n"
      " cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n cvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n"
      " cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n cvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n"
      " mov.b32 %0, {a, b, c, d};\n}\n"
      : "=r"(r) : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
  return r;
}

// E8M0 byte -> fp32 (0 is 2^-127, a subnormal; 255 is NaN)
__device__ __forceinline__ float e8m0_to_f32(uint32_t b) {
  const uint32_t bits = b == 0 ? 0x00400000u : b == 255 ? 0x7fc00000u : b << 23;
  return __uint_as_float(bits);
}
__device__ __forceinline__ float e4m3_to_f32(uint32_t b) {
  const uint32_t h = e4m3x2_to_f16x2((uint16_t)b);
  return __half2float(__ushort_as_half((unsigned short)(h & 0xffffu)));
}

// 2^e for -126 <= e <= 127
__device__ __forceinline__ float pow2i(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }

constexpr uint32_t kInfBits = 0x7f800000u;

// mxfp4 block scale from the bits of the block's largest magnitude: the smallest 2^e with amax <= 6 * 2^e = 1.5 *
// 2^(e+2), at least 2^-126; as its E8M0 byte (255 when the block holds an infinity or NaN)
__device__ __forceinline__ uint32_t mx_scale(uint32_t amax_bits) {
  if (amax_bits >= kInfBits) return 255u;
  const int e = (int)(amax_bits >> 23) - 127 - 2 + ((amax_bits & 0x7fffffu) > 0x400000u ? 1 : 0);
  return (uint32_t)(max(e, -126) + 127);
}

// nvfp4 row scale 2^k from the bits of the row's largest magnitude: the smallest with amax <= 448 * 6 * 2^k =
// 1.3125 * 2^(k+11), and not below 2^-100.  The block scale then uses e4m3's full range and the row scale costs no rounding.
__host__ __device__ __forceinline__ int nv_row_exp(uint32_t amax_bits) {
  const int k = (int)(amax_bits >> 23) - 127 - 11 + ((amax_bits & 0x7fffffu) > 0x280000u ? 1 : 0);
  return k < -100 ? -100 : k;
}
// e4m3 block scale: amax * 2^-k / 6, rounded to nearest even.  An IEEE division: amax * 2^-k = 6 * (a tie between two
// e4m3 values) happens with 16-bit inputs, and the quotient is then exact.
__device__ __forceinline__ uint32_t nv_scale(float amax_scaled) {
  const __nv_fp8_e4m3 v(__fdiv_rn(amax_scaled, 6.f));
  return (uint32_t)v.__x;
}

// A row scale rs = a * b for a sum v that another row scale t (2^-100 .. 2^119) applies to, too: v * (a * t) * b is right
// wherever v * rs * t is a value of fp32.  rs * t itself may not be one (2^-76 * 2^-76), nor v * rs (2^30 * 2^107, t = 2^-15).  a is
// kept in [2^-36, 2^8], so a * t is a power of two of fp32, and for |v| < 2^44 nothing overflows that comes back into range, or
// loses bits that the result has.  b is 1 for rows whose largest magnitude lies between 2^-24 and 2^19.  A NaN stays one.
struct RowScale {
  float a, b;
};
__device__ __forceinline__ RowScale split_scale(float rs) {
  if (rs > 0x1p8f) return {0x1p8f, rs * 0x1p-8f};
  if (rs < 0x1p-36f) return {0x1p-36f, rs * 0x1p36f};
  return {rs, 1.f};
}

// x * inv on the grid of 2^-15, for |x * inv| < 8 and inv the rounded reciprocal of a block scale s (times a power of
// two).  For x of at most 11 significant bits (bf16, f16) and s of at most 4, x / s either equals a border between two
// codes (a multiple of 1/4) or is at least 2^-11 of it, so 2^-13, away: the error that the reciprocal adds (below 2^-20) is
// removed, nothing crosses a border, and ties fall as they would with the exact quotient.  Two instructions.
__device__ __forceinline__ float scaled_on_grid(float x, float inv) {
  return __fsub_rn(__fmaf_rn(x, inv, 384.f), 384.f);
}

// largest of the magnitudes of 16-bit floats, in pairs
__device__ __forceinline__ uint32_t max_u16x2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("max.u16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}

}  // namespace fp4
}  // namespace g53
