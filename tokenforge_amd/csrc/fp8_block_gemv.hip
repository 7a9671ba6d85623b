// Block-scaled e4m3 linear, few rows: weights straight from HBM into the MFMA's registers.
//
// A workgroup owns 16 columns and 16 TM rows; its waves share the K blocks (wave v takes blocks
// v, v + waves, ...) and their sums meet in LDS in wave order. Per block of K = 128 a wave loads
// the 16 x 128 weight bytes (two 16-byte loads a lane, whole cache lines) and the rows' codes and
// runs one v_mfma_scale_f32_16x16x128_f8f6f4 per 16 rows, unit MFMA scales, from a zero
// accumulator; then acc += (xs * ws) * that in fp32. The weight fragment is the first operand, so
// a lane holds four consecutive columns of one row.
#include "fp8_block.h"
#include "tf_common.h"

namespace tf {
namespace {

template <int TM, int WAVES>
__global__ __launch_bounds__(64 * WAVES) void block_gemv_kernel(BlockArgs a) {
  __shared__ f4 red[WAVES][TM][64];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int c = lane & 15, g = lane >> 4;
  const int n0 = blockIdx.x * 16, m0 = blockIdx.y * 16 * TM;

  const int col = n0 + c;
  const uint8_t* const wp = a.w + (int64_t)(col < a.n ? col : 0) * a.ldw;
  const float* const wsp = a.ws + (int64_t)(n0 >> 7) * a.ldws;
  auto chunk = [&](const uint8_t* row, bool ok, int k) {
    u4 r = {0u, 0u, 0u, 0u};
    if (ok && k < a.k) r = *reinterpret_cast<const u4*>(row + k);
    return r;
  };
  auto frag = [&](const uint8_t* row, bool ok, int kb) {
    const u4 lo = chunk(row, ok, kb * kBlockK + 32 * g), hi = chunk(row, ok, kb * kBlockK + 32 * g + 16);
    return v8i{(int)lo[0], (int)lo[1], (int)lo[2], (int)lo[3], (int)hi[0], (int)hi[1], (int)hi[2], (int)hi[3]};
  };
  f4 acc[TM];
#pragma unroll
  for (int t = 0; t < TM; ++t) acc[t] = f4{0.0f, 0.0f, 0.0f, 0.0f};
  for (int kb = wave; kb < a.nkb; kb += WAVES) {
    const v8i wf = frag(wp, col < a.n, kb);
    const float s = wsp[kb];
#pragma unroll
    for (int t = 0; t < TM; ++t) {
      const int m = m0 + 16 * t + c;
      const bool ok = m < a.m;
      const v8i xf = frag(a.x8 + (int64_t)(ok ? m : 0) * a.ldx, ok, kb);
      const float sc = s * (ok ? a.xs[(int64_t)m * a.ldxs + kb] : 0.0f);
      const f4 d = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wf, xf, f4{0.0f, 0.0f, 0.0f, 0.0f}, 0, 0, 0,
                                                                    kUnitScale, 0, kUnitScale);
#pragma unroll
      for (int q = 0; q < 4; ++q) acc[t][q] = __builtin_fmaf(sc, d[q], acc[t][q]);
    }
  }
#pragma unroll
  for (int t = 0; t < TM; ++t) red[wave][t][lane] = acc[t];
  __syncthreads();
  const bool vec = runs_aligned(a);
  for (int t = wave; t < TM; t += WAVES) {
    const int m = m0 + 16 * t + c, n = n0 + 4 * g;
    f4 sum = red[0][t][lane];
#pragma unroll
    for (int v = 1; v < WAVES; ++v) {
      const f4 p = red[v][t][lane];
#pragma unroll
      for (int q = 0; q < 4; ++q) sum[q] += p[q];
    }
    if (m < a.m && n < a.n) store_block4(a, m, n, sum, vec);
  }
}

template <int TM, int WAVES>
int launch(const BlockArgs& a, hipStream_t stream) {
  const dim3 grid((unsigned)cdiv(a.n, 16), (unsigned)cdiv(a.m, 16 * TM));
  if (grid.y > 65535) return fail(TF_EINVAL, "tf_fp8_block_linear: too many rows for the gemv form");
  block_gemv_kernel<TM, WAVES><<<grid, 64 * WAVES, 0, stream>>>(a);
  return check_launch("tf_fp8_block_linear(gemv)");
}

}  // namespace

bool block_gemv_known(const tf_gemm_config& cfg) {
  return (cfg.block_m == 16 && cfg.num_warps == 8) || (cfg.block_m == 64 && cfg.num_warps == 4);
}

int launch_block_gemv(const BlockArgs& a, const tf_gemm_config& cfg, hipStream_t stream) {
  return cfg.block_m == 16 ? launch<1, 8>(a, stream) : launch<4, 4>(a, stream);
}

}  // namespace tf
