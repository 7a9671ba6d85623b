// The block-scaled e4m3 linear: argument bundle, epilogue and launch functions.
//   y[m][n] = sum_b xs[m][b] * ws[n / 128][b] * sum_{k in block b} e4m3(x8[m][k]) * e4m3(w[n][k])
//             (+ bias[n]) (+ residual[m][n]),   block b = K 128 b .. 128 b + 127 (the last may be shorter)
//
// The sum over a block is the MFMA's, the sum over blocks fp32. gfx950's fp8 MFMAs (both the
// 16x16x32 and the block-scaled 16x16x128 form) add products in groups of eight consecutive k in a
// window: each product is cut toward zero at 2^-13 of the power of two below the largest of its group
// (next to 2^16 one of 2^3 is kept and 2^2 is lost); between groups they keep fp32's 24 bits. So the
// cuts take less than 7 x 2^-13 = 8.5e-4 of the sum of an output's products' magnitudes, whatever the codes.
// Measured at K = 3584 (norm of the error over that of the result, without the output's own rounding of 2.1e-4
// in fp16, 1.7e-3 in bf16): normal codes 1.5e-5, one channel of x in eight 20 times the others 4.8e-5,
// that without signs 2.9e-5. What it cannot keep is a sum of small products next to large ones that cancel
// in the same eight: 0.41, where only 2e-4 of the magnitudes is left as the result. The codes' own
// rounding (2^-4 each) moves such a sum by far more, so the codes go to the MFMA as they are; fp16
// MFMAs on decoded codes would keep the bits at half the rate.
#pragma once

#include "tf_common.h"

namespace tf {

typedef int v8i __attribute__((ext_vector_type(8)));

constexpr int kBlockK = 128;        // K per scale block, and per MFMA
constexpr int kUnitScale = 127;     // E8M0 2^0: the MFMA's own block scales leave the product as is

// v of the lane N below, cyclic in each row of 16 lanes.
template <int N>
__device__ __forceinline__ uint32_t dpp_ror(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x120 + N, 0xF, 0xF, false);
}

struct BlockArgs {
  const uint8_t* x8;  // [m, k] codes, row stride ldx bytes (16-byte aligned rows)
  int64_t ldx;
  const float* xs;  // [m, nkb], row stride ldxs
  int64_t ldxs;
  const uint8_t* w;  // [n, k] codes, row stride ldw bytes (16-byte aligned rows)
  int64_t ldw;
  const float* ws;  // [ceil(n / 128), nkb], row stride ldws
  int64_t ldws;
  const uint16_t* bias;      // [n] or nullptr
  const uint16_t* residual;  // [m, n], row stride ldr, or nullptr
  int64_t ldr;
  uint16_t* out;  // [m, n], row stride ldo
  int64_t ldo;
  int m;
  int n;
  int k;
  int nkb;   // ceil(k / 128)
  int bf16;  // type of bias, residual and out (else fp16)
};

__device__ __forceinline__ float from_16(const BlockArgs& a, uint16_t b) {
  return a.bf16 ? as_f32((uint32_t)b << 16) : half_bits_to_float(b);
}
__device__ __forceinline__ uint16_t to_16(const BlockArgs& a, float v) {
  return a.bf16 ? __builtin_bit_cast(uint16_t, (__bf16)v) : __builtin_bit_cast(uint16_t, (_Float16)v);
}

// Whether a run of four consecutive columns (4-aligned) of out (and residual) is one 8-byte access.
__device__ __forceinline__ bool runs_aligned(const BlockArgs& a) {
  return ((a.n | a.ldo) & 3) == 0 && (reinterpret_cast<uintptr_t>(a.out) & 7) == 0 &&
         (a.residual == nullptr || ((a.ldr & 3) == 0 && (reinterpret_cast<uintptr_t>(a.residual) & 7) == 0));
}

// Columns n .. n + 3 of row m from their fp32 sums: bias and residual added in fp32, one rounding.
__device__ __forceinline__ void store_block4(const BlockArgs& a, int m, int n, const f4& sum, bool vec) {
  uint16_t* const o = a.out + (int64_t)m * a.ldo + n;
  const uint16_t* const r = a.residual ? a.residual + (int64_t)m * a.ldr + n : nullptr;
  if (vec) {
    u2 res = {0u, 0u};
    if (r) res = *reinterpret_cast<const u2*>(r);
    uint32_t h[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float v = sum[j];
      if (a.bias) v += from_16(a, a.bias[n + j]);
      if (r) v += from_16(a, (uint16_t)(res[j >> 1] >> (16 * (j & 1))));
      h[j] = to_16(a, v);
    }
    *reinterpret_cast<u2*>(o) = u2{h[0] | (h[1] << 16), h[2] | (h[3] << 16)};
    return;
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if (n + j >= a.n) break;
    float v = sum[j];
    if (a.bias) v += from_16(a, a.bias[n + j]);
    if (r) v += from_16(a, r[j]);
    o[j] = to_16(a, v);
  }
}

// Whether runs of eight columns (8-aligned) of out (and residual) are one 16-byte access.
__device__ __forceinline__ bool wide_rows(const BlockArgs& a) {
  return (a.ldo & 7) == 0 && (reinterpret_cast<uintptr_t>(a.out) & 15) == 0 &&
         (a.residual == nullptr || ((a.ldr & 7) == 0 && (reinterpret_cast<uintptr_t>(a.residual) & 15) == 0));
}

// Columns n .. n + 7 of row m, as store_block4 (n % 8 == 0, N % 8 == 0 and wide_rows hold). STREAM: a
// non-temporal store.
template <bool STREAM>
__device__ __forceinline__ void store_block8(const BlockArgs& a, int m, int n, const f4& lo, const f4& hi) {
  float v[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = j < 4 ? lo[j & 3] : hi[j & 3];
  if (a.bias) {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] += from_16(a, a.bias[n + j]);
  }
  if (a.residual) {
    const u4 r = *reinterpret_cast<const u4*>(a.residual + (int64_t)m * a.ldr + n);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] += from_16(a, (uint16_t)(r[j >> 1] >> (16 * (j & 1))));
  }
  u4 h;
#pragma unroll
  for (int j = 0; j < 4; ++j) h[j] = (uint32_t)to_16(a, v[2 * j]) | ((uint32_t)to_16(a, v[2 * j + 1]) << 16);
  u4* const o = reinterpret_cast<u4*>(a.out + (int64_t)m * a.ldo + n);
  if (STREAM)
    __builtin_nontemporal_store(h, o);
  else
    *o = h;
}

// Row strides (bytes of codes, elements of scales) below which a tile's offsets stay in 31 bits.
constexpr int64_t kMaxCodeStride = 1 << 22;
constexpr int64_t kMaxScaleStride = 1 << 20;

bool block_gemv_known(const tf_gemm_config& cfg);
int launch_block_gemv(const BlockArgs& a, const tf_gemm_config& cfg, hipStream_t stream);

bool block_gemm_known(const tf_gemm_config& cfg);
int block_split(const tf_gemm_config& cfg, int64_t nkb);  // K slices that hold a block
int launch_block_gemm(const BlockArgs& a, const tf_gemm_config& cfg, float* part, hipStream_t stream);

}  // namespace tf
