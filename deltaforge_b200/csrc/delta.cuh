// What the preparation and the scan of the chunked delta rule share: the layout of a chunk's images, and the fp16 halves.
#pragma once

#include <cuda_fp16.h>

#include "common.cuh"
#include "kernels.h"

namespace dfb {
namespace {

constexpr int C = 64;                // tokens per chunk
constexpr int SQ = C * C * 2;        // bytes of one 64 x 64 16-bit image
// Scalars of a (chunk, value head), floats: on V' into the state, on Q S per token; then at 2 C: decay of the state, +4: scales
// of W per 16 rows, +8: scales of P likewise, +12, +13: the largest on V' per 32 tokens, +14, +15: a bit per token that counts.
constexpr int SCAL = 3 * C * 4;
__host__ __device__ constexpr int w_bytes(int dkp) { return dkp / 64 * SQ; }  // of one half of W: per 64 key dims its 64 rows
// of a value head: T (three bf16 parts), P, W (hi, lo), scalars
__host__ __device__ constexpr int head_bytes(int dkp) { return 4 * SQ + 2 * (dkp / 64 * SQ) + SCAL; }
// of a key head: per 64 key dims the 64 rows of k, then those of q
__host__ __device__ constexpr int key_bytes(int dkp) { return dkp / 64 * 2 * C * 128; }

__device__ __forceinline__ uint32_t h2(float a, float b) {
  __half2 v = __floats2half2_rn(a, b);
  return *(uint32_t*)&v;
}
// (a, b) as fp16 pair hi and the remainder as fp16 pair lo: hi + lo carries 22 bits
__device__ __forceinline__ void split2(float a, float b, uint32_t& hi, uint32_t& lo) {
  const __half2 h = __floats2half2_rn(a, b);
  const float2 f = __half22float2(h);
  hi = *(const uint32_t*)&h;
  lo = h2(a - f.x, b - f.y);
}
// Exponent that takes a largest magnitude m to [2^12, 2^13); 0 for m = 0. Clamped so that 2^e and 2^-e are normal numbers.
__device__ __forceinline__ int scale_exp(float m) {
  if (m == 0.f) return 0;
  const int e = (int)((__float_as_uint(m) >> 23) & 255) - 127 - 12;
  return e < -110 ? -110 : e > 110 ? 110 : e;
}
// The same for a row whose sum of squares is ss: no element exceeds its root.
__device__ __forceinline__ int norm_exp(float ss) { return (((int)((__float_as_uint(ss) >> 23) & 255) - 127 + 2) >> 1) - 13; }
// Largest of the lanes' non-negative values, whose bit patterns order like the values
__device__ __forceinline__ float warp_max_abs(float m) { return __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(m))); }
__device__ __forceinline__ float pow2(int e) { return __int_as_float((e + 127) << 23); }

// Rows of W fp16 with 16-byte chunks permuted within 128 bytes: what 8x8 matrix loads and, for W = 64, tcgen05 operands want
template <int W> __device__ __forceinline__ uint32_t img_off(int row, int chunk) {
  return (uint32_t)(row * W * 2 + ((chunk ^ (row & 7)) << 4));
}

}  // namespace
}  // namespace dfb
