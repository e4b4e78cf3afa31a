// rows8.cuh -- rows in 8 bits: e4m3 elements and, for every 32 of a row, a
// power-of-two scale (e8m0: 2^(byte - 127), 255 is NaN).
//
// The scale of a block is the smallest 2^e with max |v| <= 448 * 2^e, 448
// being e4m3's largest value: nothing saturates, and an element is off by at
// most half a step of its three fraction bits (2^-4 of it; below 2^-6 * 2^e
// half of 2^-9 * 2^e).  A power of two makes the division exact, so the only
// rounding is the element's own, to nearest even.  A block with an infinity or
// a NaN has the scale NaN: all of it reads as NaN, and so do the products with
// it.  Blocks under 2^-127 * 448 take 2^-127.
#pragma once

#include <stdint.h>

#include "common.cuh"

namespace senmoe {

constexpr int kBlock8 = 32;  // elements of a scale

// The scale's byte from the bits of the largest |v|: 448 = 1.75 * 2^8, so a
// fraction above 0.75 carries into the exponent.
__device__ __forceinline__ uint32_t scale_byte(uint32_t largest) {
  if (largest >= 0x7f800000u) return 255u;
  const uint32_t e = (largest + 0x1fffffu) >> 23;
  return e > 8 ? e - 8 : 0u;
}
// 1 / scale (NaN for NaN).
__device__ __forceinline__ float scale_inverse(uint32_t byte) {
  return __uint_as_float(byte == 255u ? 0x7fc00000u : (254u - byte) << 23);
}
__device__ __forceinline__ uint32_t magnitude(float v) { return __float_as_uint(v) & 0x7fffffffu; }
// Two elements, lo in the lower byte.
__device__ __forceinline__ uint32_t to_e4m3x2(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}

// 8 consecutive elements a lane, four lanes a block: every lane of the warp
// calls it, lanes without elements with zeros.  Returns the elements; `byte`
// is the block's scale, the same in its four lanes.
__device__ __forceinline__ uint2 pack8_lane(const float (&v)[8], uint32_t& byte) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) m = max(m, magnitude(v[i]));
  m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
  m = max(m, __shfl_xor_sync(0xffffffffu, m, 2));
  byte = scale_byte(m);
  const float inv = scale_inverse(byte);
  uint32_t h[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) h[i] = to_e4m3x2(v[2 * i] * inv, v[2 * i + 1] * inv);
  return make_uint2(h[0] | h[1] << 16, h[2] | h[3] << 16);
}
// One element a lane, a warp a block.
__device__ __forceinline__ uint8_t pack8_warp(float v, uint32_t& byte) {
  byte = scale_byte(__reduce_max_sync(0xffffffffu, magnitude(v)));
  return static_cast<uint8_t>(to_e4m3x2(v * scale_inverse(byte), 0.0f));
}

// N * 4 scale bytes from p on, p anywhere, in aligned words: begin and end are
// those of all scales, outside of which nothing is read.  `have` bytes belong to
// the row; what lies behind them is of no meaning.
template <int N> __device__ __forceinline__ void scale_words(const uint8_t* p, int have, const uint8_t* begin,
                                                             const uint8_t* end, uint32_t (&w)[N]) {
  const int skew = static_cast<int>(reinterpret_cast<uintptr_t>(p) & 3);
  const uint8_t* a = p - skew;
  if (a >= begin && a + 4 * (N + 1) <= end) {
    uint32_t v[N + 1];
#pragma unroll
    for (int i = 0; i <= N; ++i) v[i] = reinterpret_cast<const uint32_t*>(a)[i];
#pragma unroll
    for (int i = 0; i < N; ++i) w[i] = __funnelshift_r(v[i], v[i + 1], 8 * skew);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) w[i] = 0;
#pragma unroll
    for (int i = 0; i < 4 * N; ++i)
      if (i < have) w[i >> 2] |= static_cast<uint32_t>(p[i]) << 8 * (i & 3);
  }
}

}  // namespace senmoe
