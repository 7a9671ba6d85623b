// e4m3 codes with a scale per 128 elements of a row, or per row, of three 16-bit producers:
//   quant  y = x
//   silu   y = silu(x[:, :k]) * x[:, k:],  silu(v) = v / (1 + exp(-v))
//   norm   h = round16(x + residual) (or x), y = h * rsqrt(mean(h^2) + eps) * w
// each y in fp32 without a 16-bit rounding on the way (h is rounded because it is an output: the
// next residual), then s = max(amax|y| / 448, 1 / (448 * 512)) and q = e4m3(y / s).
//
// All three read and write each element once: 3 (quant), 5 (silu) or 7 (norm with its residual)
// bytes per element, memory bound from a few hundred rows on, launch bound below. On MI355X (a copy
// of 1 GiB: 5.2 TB/s), bf16, us: quant 4095 x 3584 8.9 (4.9 TB/s), silu 2048 x 18944 38.9 (5.0), norm 4095 x
// 3584 18.9 (5.4); with one scale per row 8.7, 50.7 (a CU holds one row of four chunks a thread), 19.1.
// Rows that 16 bytes do not divide, or that start off them, go by elements: 25, 108 and 63. Loads and
// stores take the caches' default policy: the inputs were just written and the codes are read next
// (non-temporal loads: norm 23.4 us).
#include "fp8_rows.h"

namespace tf {
namespace {

enum Mode { kQuant = 0, kSilu = 1, kNorm = 2 };

struct RowsArgs {
  const uint16_t* x;  // [t, k] (silu: [t, 2k]), row stride ldx
  int64_t ldx;
  const uint16_t* residual;  // norm: [t, k], row stride ldr, or nullptr
  int64_t ldr;
  const uint16_t* w;  // norm: [k]
  uint16_t* hidden;   // norm with a residual: [t, k] contiguous
  uint8_t* q;         // [t, k] contiguous
  float* scale;       // [t, ceil(k / 128)] contiguous, or [t] (by_row)
  int64_t t;
  int k;
  int blocks;   // ceil(k / 128)
  int by_row;   // one scale per row
  float eps;
  float inv_k;  // norm
};

// silu(g) * u = g / (1 + 2^(-g log2 e)) * u through v_exp_f32 and v_rcp_f32 (an ulp each): within
// (7 + 1.23 |g|) 2^-24 of the exact value (the argument is rounded, and the constant off by 0.23 2^-24),
// where an IEEE division and expf cost three times the instructions (2048 x 18944 on MI355X: 48 us against
// 43). g = -inf gives NaN, as the expression does.
//
// From g = -87.3 down its denominator passes 2^126 and the reciprocal fp32's normal range: silu_far8.
__device__ __forceinline__ float silu_mul(float g, float u) {
  const float e = __builtin_amdgcn_exp2f(g * -1.44269504f);
  return g * __builtin_amdgcn_rcpf(1.0f + e) * u;
}

typedef uint16_t us2 __attribute__((ext_vector_type(2)));

// y = silu(g) * u again where g < -80, of a lane's eight bf16 gates and values: an `up` of bf16's size (to
// 3.4e38; fp16 ends at 65504) brings a gate's sigmoid of down to e^-112 back above the smallest scale. There
// the 1 is below 2^-115 of 1 + e^-g, and g e^(g/2) u e^(g/2) stays in range, within the bound above.
// Taken behind one comparison of the eight (negative bf16 order as their bits; below -80.0 = 0xC2A0): as a
// selection in silu_mul it cost every call 11% (2048 x 18944 on MI355X 42.5 us against 38.3).
__device__ __forceinline__ void silu_far8(const u4& gates, const u4& ups, float (&y)[8]) {
  us2 m = __builtin_bit_cast(us2, gates[0]);
#pragma unroll
  for (int j = 1; j < 4; ++j) m = __builtin_elementwise_max(m, __builtin_bit_cast(us2, gates[j]));
  if (m[0] <= 0xC2A0u && m[1] <= 0xC2A0u) return;
  float g[8], u[8];
  unpack8<BF16>(gates, g);
  unpack8<BF16>(ups, u);
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float e = __builtin_amdgcn_exp2f(g[j] * 0.72134752f);
    if (g[j] < -80.0f) y[j] = g[j] * e * u[j] * e;
  }
}

// Eight elements of a row at e0 (zeros past k). VEC: one 16-byte load (k % 8 == 0, aligned rows).
template <bool VEC>
__device__ __forceinline__ u4 load8(const uint16_t* __restrict__ row, int e0, int k) {
  u4 r = {0u, 0u, 0u, 0u};
  if (VEC) {
    if (e0 < k) r = *reinterpret_cast<const u4*>(row + e0);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (e0 + j < k) r[j >> 1] |= (uint32_t)row[e0 + j] << (16 * (j & 1));
  }
  return r;
}

template <bool VEC>
__device__ __forceinline__ void store8(uint8_t* __restrict__ row, int e0, int k, u2 codes) {
  if (VEC) {
    if (e0 < k) *reinterpret_cast<u2*>(row + e0) = codes;
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (e0 + j < k) row[e0 + j] = (uint8_t)(codes[j >> 2] >> (8 * (j & 3)));
  }
}

// ------------------------------------------------------------------ blocks of 128, quant and silu
//
// No step crosses a block, so the launch is flat over the blocks of all rows: 16 lanes a block, each
// thread kBlocksEach of them, all loaded before the first is reduced.
constexpr int kBlocksEach = 2;

template <int MODE, typename T, bool VEC>
__global__ __launch_bounds__(256) void quant_blocks_kernel(RowsArgs a) {
  // Block x of the workgroup is block b0 + x of row0 onward (row0, b0 uniform; b0 + x passes few rows).
  const uint32_t g0 = blockIdx.x * (16u * kBlocksEach);
  const uint32_t row0 = g0 / (uint32_t)a.blocks, b0 = g0 - row0 * (uint32_t)a.blocks;
  const int sub = threadIdx.x & 15;
  int64_t row[kBlocksEach];
  int e0[kBlocksEach], left[kBlocksEach];
  u4 v[kBlocksEach], w[kBlocksEach];
#pragma unroll
  for (int i = 0; i < kBlocksEach; ++i) {
    const uint32_t x = b0 + 16u * i + (threadIdx.x >> 4);
    const uint32_t q = a.blocks >= 16 * kBlocksEach ? (x >= (uint32_t)a.blocks ? 1u : 0u) : x / (uint32_t)a.blocks;
    row[i] = (int64_t)row0 + q;
    e0[i] = (int)(x - q * (uint32_t)a.blocks) * 128 + sub * 8;
    left[i] = row[i] < a.t ? a.k : 0;  // past the last row: nothing is read or written
    const uint16_t* const p = a.x + (left[i] ? row[i] : 0) * a.ldx;
    v[i] = load8<VEC>(p, e0[i], left[i]);
    if (MODE == kSilu) w[i] = load8<VEC>(p + a.k, e0[i], left[i]);
  }
#pragma unroll
  for (int i = 0; i < kBlocksEach; ++i) {
    float y[8];
    unpack8<T>(v[i], y);
    if (MODE == kSilu) {
      float u[8];
      unpack8<T>(w[i], u);
#pragma unroll
      for (int j = 0; j < 8; ++j) y[j] = silu_mul(y[j], u[j]);
      if (T::kWide) silu_far8(v[i], w[i], y);
    }
    const uint32_t amax = max16_u32(absmax8(y));
    const float s = dynamic_scale(as_f32(amax));
    store8<VEC>(a.q + row[i] * a.k, e0[i], left[i], encode8(y, s, amax));
    if (sub == 0 && left[i]) a.scale[row[i] * a.blocks + (e0[i] >> 7)] = s;
  }
}

// ------------------------------------------------------------------ whole rows
//
// A workgroup per row: the norm, whose mean crosses the row, and every producer with one scale per
// row. Thread tid holds the row's 8-element chunks tid + i * threads, so 16 lanes hold a block.
//
// Sum of squares: a chunk's eight in fp32 pairwise, then each 64 consecutive chunks (one wave, one
// i) pairwise over the lane index, then those sums in order. The order depends on k alone, not
// on the launch, so a row's result does not depend on the batch it came in.
template <int MODE, typename T, int CPT, bool VEC>
__global__ __launch_bounds__(1024) void quant_rows_kernel(RowsArgs a) {
  __shared__ float part[16 * CPT];
  __shared__ uint32_t red[16];
  const int tid = threadIdx.x, threads = blockDim.x;
  const int wave = tid >> 6, waves = threads >> 6;
  const int64_t row = blockIdx.x;
  const uint16_t* const x = a.x + row * a.ldx;

  u4 v[CPT], w[CPT];
#pragma unroll
  for (int i = 0; i < CPT; ++i) v[i] = load8<VEC>(x, (tid + i * threads) * 8, a.k);
  if (MODE == kSilu) {
#pragma unroll
    for (int i = 0; i < CPT; ++i) w[i] = load8<VEC>(x + a.k, (tid + i * threads) * 8, a.k);
  }
  float rstd = 0.0f;
  if (MODE == kNorm) {
#pragma unroll
    for (int i = 0; i < CPT; ++i) w[i] = load8<VEC>(a.w, (tid + i * threads) * 8, a.k);
    if (a.residual != nullptr) {
#pragma unroll
      for (int i = 0; i < CPT; ++i) {
        const int e0 = (tid + i * threads) * 8;
        const u4 r = load8<VEC>(a.residual + row * a.ldr, e0, a.k);
#pragma unroll
        for (int j = 0; j < 4; ++j)
          v[i][j] = round_pair<T>(T::lo(v[i][j]) + T::lo(r[j]), T::hi(v[i][j]) + T::hi(r[j]));
        uint16_t* const h = a.hidden + row * a.k;
        if (VEC) {
          if (e0 < a.k) *reinterpret_cast<u4*>(h + e0) = v[i];
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j)
            if (e0 + j < a.k) h[e0 + j] = (uint16_t)(v[i][j >> 1] >> (16 * (j & 1)));
        }
      }
    }
#pragma unroll
    for (int i = 0; i < CPT; ++i) {
      float f[8];
      unpack8<T>(v[i], f);
      const float s = ((f[0] * f[0] + f[1] * f[1]) + (f[2] * f[2] + f[3] * f[3])) +
                      ((f[4] * f[4] + f[5] * f[5]) + (f[6] * f[6] + f[7] * f[7]));
      const float p = wave_sum_f32(s);
      if ((tid & 63) == 0) part[i * waves + wave] = p;
    }
    __syncthreads();
    float total = 0.0f;
    for (int i = 0; i < CPT * waves; ++i) total += part[i];
    rstd = 1.0f / __builtin_sqrtf(total * a.inv_k + a.eps);
  }
  auto values = [&](int i, float(&y)[8]) {
    unpack8<T>(v[i], y);
    if (MODE == kQuant) return;
    float u[8];
    unpack8<T>(w[i], u);
#pragma unroll
    for (int j = 0; j < 8; ++j) y[j] = MODE == kSilu ? silu_mul(y[j], u[j]) : y[j] * rstd * u[j];
    if (MODE == kSilu && T::kWide) silu_far8(v[i], w[i], y);
    if (MODE == kNorm) {
      // Past k the loads are zeros, and 0 * rstd is NaN where rstd is not finite.
      const int e0 = (tid + i * threads) * 8;
#pragma unroll
      for (int j = 0; j < 8; ++j) y[j] = e0 + j < a.k ? y[j] : 0.0f;
    }
  };
  uint8_t* const q = a.q + row * a.k;
  if (a.by_row) {
    float y[CPT][8];
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < CPT; ++i) {
      values(i, y[i]);
      m = __builtin_elementwise_max(m, absmax8(y[i]));
    }
    m = wave_max_u32(m);
    if ((tid & 63) == 0) red[wave] = m;
    __syncthreads();
    for (int i = 0; i < waves; ++i) m = __builtin_elementwise_max(m, red[i]);
    const float s = dynamic_scale(as_f32(m));
    if (tid == 0) a.scale[row] = s;
#pragma unroll
    for (int i = 0; i < CPT; ++i) store8<VEC>(q, (tid + i * threads) * 8, a.k, encode8(y[i], s, m));
    return;
  }
#pragma unroll
  for (int i = 0; i < CPT; ++i) {
    const int e0 = (tid + i * threads) * 8;
    float y[8];
    values(i, y);
    const uint32_t m = max16_u32(absmax8(y));
    const float s = dynamic_scale(as_f32(m));
    store8<VEC>(q, e0, a.k, encode8(y, s, m));
    if ((tid & 15) == 0 && e0 < a.k) a.scale[row * a.blocks + (e0 >> 7)] = s;
  }
}

template <int MODE, typename T, bool VEC>
int launch_rows(const RowsArgs& a, hipStream_t stream) {
  const int chunks = (int)cdiv(a.k, 8);
  // A chunk a thread shortens a row's chain of steps; over many long rows two a thread cost fewer
  // reductions (MI355X: 512 x 3584 norm 4.8 us against 5.1, 4095 x 8192 42.6 against 41.5; one scale per
  // row 4095 x 3584 21.7 against 19.8). Rows past 16 waves take more either way.
  const bool two = a.t >= 1024 && chunks > (a.by_row ? 128 : 512);
  int waves = (int)cdiv(chunks, two ? 128 : 64);
  waves = waves < 16 ? waves : 16;
  const int cpt = (int)cdiv(chunks, 64 * waves);
  const unsigned grid = (unsigned)a.t;
  if (cpt <= 1)
    quant_rows_kernel<MODE, T, 1, VEC><<<grid, 64 * waves, 0, stream>>>(a);
  else if (cpt <= 2)
    quant_rows_kernel<MODE, T, 2, VEC><<<grid, 64 * waves, 0, stream>>>(a);
  else
    quant_rows_kernel<MODE, T, 4, VEC><<<grid, 64 * waves, 0, stream>>>(a);
  return TF_OK;
}

template <int MODE, typename T, bool VEC>
int launch_vec(const RowsArgs& a, hipStream_t stream) {
  // quant rows of up to one chunk a thread are faster a workgroup each (4095 x 3584 on MI355X: 9.0 us
  // against 10.3), longer ones flat (300 x 18944: 5.6 us against 7.3).
  if (MODE == kNorm || a.by_row || (MODE == kQuant && a.k <= 8192)) return launch_rows<MODE, T, VEC>(a, stream);
  quant_blocks_kernel<MODE == kNorm ? kQuant : MODE, T, VEC>
      <<<(unsigned)cdiv(a.t * a.blocks, 16 * kBlocksEach), 256, 0, stream>>>(a);
  return TF_OK;
}

// A row's length, before it is held in 32 bits.
int check_length(int64_t k, const char* name) {
  if (k <= 0) return fail(TF_EINVAL, std::string(name) + ": need k > 0");
  if (k > 0x3FFFFFFF) return fail(TF_EINVAL, std::string(name) + ": row too long");
  return TF_OK;
}

bool multiple(const void* p, uintptr_t a) { return (reinterpret_cast<uintptr_t>(p) % a) == 0; }

template <int MODE>
int run_rows(RowsArgs a, int32_t dtype, int32_t group_size, const char* name, hipStream_t stream) {
  const std::string who(name);
  if (dtype != TF_DTYPE_FP16 && dtype != TF_DTYPE_BF16) return fail(TF_EINVAL, who + ": unknown dtype");
  if (!a.x || !a.q || !a.scale) return fail(TF_EINVAL, who + ": null pointer");
  if (a.t < 0) return fail(TF_EINVAL, who + ": need t >= 0");
  if (group_size != 0 && group_size != 128)
    return fail(TF_EINVAL, who + ": group_size must be 128, or 0 for one scale per row");
  if (a.ldx < (MODE == kSilu ? 2 : 1) * (int64_t)a.k || (a.residual && a.ldr < a.k))
    return fail(TF_EINVAL, who + ": row stride smaller than the row");
  a.blocks = (int)cdiv(a.k, 128);
  a.by_row = group_size == 0;
  if ((MODE == kNorm || a.by_row) && a.k > TF_FP8_MAX_ROW)
    return fail(TF_EINVAL, who + ": rows above " + std::to_string(TF_FP8_MAX_ROW) + " are not supported");
  if (a.t > 0x7FFFFFFF || a.t * a.blocks > 0x7FFFFF00) return fail(TF_EINVAL, who + ": too many rows");
  if (a.t == 0) return TF_OK;
  const bool vec = a.k % 8 == 0 && a.ldx % 8 == 0 && multiple(a.x, 16) && multiple(a.q, 8) &&
                   (MODE != kNorm || multiple(a.w, 16)) &&
                   (!a.residual || (a.ldr % 8 == 0 && multiple(a.residual, 16) && multiple(a.hidden, 16)));
  // A launch takes fewer than 2^32 threads (2^21 rows of up to 1024, or 16 a block).
  const int64_t all = a.t, rows = (int64_t(1) << 27) / a.blocks < (1 << 21) ? (int64_t(1) << 27) / a.blocks : 1 << 21;
  for (int64_t t0 = 0; t0 < all; t0 += rows) {
    RowsArgs b = a;
    b.t = all - t0 < rows ? all - t0 : rows;
    b.x = a.x + t0 * a.ldx;
    b.residual = a.residual ? a.residual + t0 * a.ldr : nullptr;
    b.hidden = a.hidden ? a.hidden + t0 * a.k : nullptr;
    b.q = a.q + t0 * a.k;
    b.scale = a.scale + t0 * (a.by_row ? 1 : a.blocks);
    int rc;
    if (dtype == TF_DTYPE_FP16)
      rc = vec ? launch_vec<MODE, F16, true>(b, stream) : launch_vec<MODE, F16, false>(b, stream);
    else
      rc = vec ? launch_vec<MODE, BF16, true>(b, stream) : launch_vec<MODE, BF16, false>(b, stream);
    if (rc || (rc = check_launch(name))) return rc;
  }
  return TF_OK;
}

}  // namespace
}  // namespace tf

using namespace tf;

extern "C" int tf_fp8_quant(const uint16_t* x, int64_t ldx, int32_t dtype, uint8_t* q, float* scale, int64_t t,
                            int64_t k, int32_t group_size, void* stream) {
  if (int rc = check_length(k, "tf_fp8_quant")) return rc;
  RowsArgs a{};
  a.x = x, a.ldx = ldx, a.q = q, a.scale = scale, a.t = t, a.k = (int)k;
  return run_rows<kQuant>(a, dtype, group_size, "tf_fp8_quant", (hipStream_t)stream);
}

extern "C" int tf_silu_mul_fp8_quant(const uint16_t* x, int64_t ldx, int32_t dtype, uint8_t* q, float* scale,
                                     int64_t t, int64_t k, int32_t group_size, void* stream) {
  if (int rc = check_length(k, "tf_silu_mul_fp8_quant")) return rc;
  RowsArgs a{};
  a.x = x, a.ldx = ldx, a.q = q, a.scale = scale, a.t = t, a.k = (int)k;
  return run_rows<kSilu>(a, dtype, group_size, "tf_silu_mul_fp8_quant", (hipStream_t)stream);
}

extern "C" int tf_add_rmsnorm_fp8_quant(const uint16_t* x, int64_t ldx, const uint16_t* residual, int64_t ldr,
                                        const uint16_t* weight, int32_t dtype, uint8_t* q, float* scale,
                                        uint16_t* hidden, int64_t t, int64_t k, float eps, int32_t group_size,
                                        void* stream) {
  if (int rc = check_length(k, "tf_add_rmsnorm_fp8_quant")) return rc;
  if (!weight || (residual && !hidden)) return fail(TF_EINVAL, "tf_add_rmsnorm_fp8_quant: null pointer");
  RowsArgs a{};
  a.x = x, a.ldx = ldx, a.residual = residual, a.ldr = ldr, a.w = weight, a.hidden = hidden;
  a.q = q, a.scale = scale, a.t = t, a.k = (int)k, a.eps = eps, a.inv_k = 1.0f / (float)k;
  return run_rows<kNorm>(a, dtype, group_size, "tf_add_rmsnorm_fp8_quant", (hipStream_t)stream);
}
