// Row pieces of the block-scaled e4m3 quantizers: 16-bit element types, the 16-lane reductions of
// a 128-element block, and the encoding of eight fp32 values with their block's (or row's) scale.
//
// A lane holds eight consecutive elements (16 bytes of a 16-bit input, 8 bytes of codes), so a
// block of 128 is one aligned row of 16 lanes: its absmax is four DPP steps, without LDS.
#pragma once

#include "fp8.h"
#include "norm_row.h"
#include "tf_common.h"

namespace tf {

struct F16 {  // IEEE binary16
  static constexpr bool kWide = false;  // fp32's exponent range
  static __device__ __forceinline__ float lo(uint32_t pair) { return (float)as_h2(pair)[0]; }
  static __device__ __forceinline__ float hi(uint32_t pair) { return (float)as_h2(pair)[1]; }
  static __device__ __forceinline__ uint32_t round(float v) { return __builtin_bit_cast(uint16_t, (_Float16)v); }
};

struct BF16 {  // the upper half of an fp32
  static constexpr bool kWide = true;
  static __device__ __forceinline__ float lo(uint32_t pair) { return as_f32(pair << 16); }
  static __device__ __forceinline__ float hi(uint32_t pair) { return as_f32(pair & 0xFFFF0000u); }
  static __device__ __forceinline__ uint32_t round(float v) {  // to nearest, ties to even; NaN kept
    return __builtin_bit_cast(uint16_t, (__bf16)v);
  }
};

template <typename T>
__device__ __forceinline__ uint32_t round_pair(float a, float b) {
  return T::round(a) | (T::round(b) << 16);
}

template <typename T>
__device__ __forceinline__ void unpack8(const u4& r, float (&v)[8]) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    v[2 * j] = T::lo(r[j]);
    v[2 * j + 1] = T::hi(r[j]);
  }
}

// Absmax bit pattern of eight values: non-negative floats order as their bit patterns, and every
// NaN lies above infinity, so an unsigned max keeps a NaN, as torch's amax does.
__device__ __forceinline__ uint32_t absmax8(const float (&v)[8]) {
  uint32_t m = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) m = __builtin_elementwise_max(m, as_u32(v[j]) & 0x7FFFFFFFu);
  return m;
}

// Max over an aligned row of 16 lanes (all active), in each of them.
__device__ __forceinline__ uint32_t max16_u32(uint32_t v) {
  v = __builtin_elementwise_max(v, dpp_u32<kDppQuadXor1>(v));
  v = __builtin_elementwise_max(v, dpp_u32<kDppQuadXor2>(v));
  v = __builtin_elementwise_max(v, dpp_u32<kDppHalfRowMirror>(v));
  return __builtin_elementwise_max(v, dpp_u32<kDppRowMirror>(v));
}

// Sum of a wave's 64 lanes (all active) in fp32, wave-uniform, pairwise over the lane index.
__device__ __forceinline__ float wave_sum_f32(float v) {
  v += as_f32(dpp_u32<kDppQuadXor1>(as_u32(v)));
  v += as_f32(dpp_u32<kDppQuadXor2>(as_u32(v)));
  v += as_f32(dpp_u32<kDppHalfRowMirror>(as_u32(v)));
  v += as_f32(dpp_u32<kDppRowMirror>(as_u32(v)));
  const auto at = [&](int l) { return as_f32((uint32_t)__builtin_amdgcn_readlane((int)as_u32(v), l)); };
  return (at(0) + at(16)) + (at(32) + at(48));
}

// e4m3 codes of y[0..8) / s, s = dynamic_scale(amax) of a block or row that holds them.
//
// amax finite: |y / s| <= 448 (1 + 2^-23), which rounds to at most 448 without a clamp; the quotient
// is y * r with r = fp32(1 / s) and one residual correction: the IEEE quotient, or within an ulp
// of it, and exact where the true quotient lies on a tie of two codes, so ties go to even as they
// do after an IEEE division. (s lies in [2^-18, 2^120], so neither r nor a quotient that
// matters under- or overflows.) amax infinite or NaN (rare, uniform over the block): a plain
// division, clamped with compares that keep NaN, as torch's expression gives it.
__device__ __forceinline__ u2 encode8(const float (&y)[8], float s, uint32_t amax_bits) {
  if (amax_bits < 0x7F800000u) {
    const float r = 1.0f / s;
    float q[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float q0 = y[j] * r;
      const float e = __builtin_fmaf(q0, s, -y[j]);
      q[j] = __builtin_fmaf(-e, r, q0);
    }
    return u2{encode4_clamped(q[0], q[1], q[2], q[3]), encode4_clamped(q[4], q[5], q[6], q[7])};
  }
  u2 w = {0u, 0u};
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    float v = y[j] / s;
    v = (v < -kFp8Max) ? -kFp8Max : v;
    v = (v > kFp8Max) ? kFp8Max : v;
    w[j >> 2] |= (uint32_t)e4m3_encode(v) << (8 * (j & 3));
  }
  return w;
}

}  // namespace tf
