// Block-scaled e4m3 linear, few rows: weights straight from memory into the MFMA's registers.
//
// A workgroup owns 16 columns and TM tiles of up to 16 rows; its KS waves take every KS-th K block each,
// and their sums meet in LDS in wave order. Per block of K = 128 a wave loads the 16 x 128 weight bytes
// (two 16-byte loads a lane, whole cache lines), D blocks ahead in a register ring, and runs one
// v_mfma_scale_f32_16x16x128_f8f6f4 (unit MFMA scales) from a zero accumulator; then acc += (xs * ws) *
// that in fp32. The weight fragment is the first operand, so a lane holds four consecutive columns
// of one row of x.
//
// With few rows most of the MFMA's 16 are free: G K blocks share one x fragment (up to 16 / G rows),
// lane c holding row c % (16 / G) of block c / (16 / G). The product with the weights of block j is
// then right in the lanes of block j, and the others take the scale zero, so x and its scales cost one
// load for G blocks; the lanes of a row are added at the end.
//
// Bound by the weight's bytes from a few MB on. On MI355X, weights from HBM: 37888 x 3584 M = 1 25.2 us
// (5.4 TB/s, the card's copy rate), 3584 x 18944 15.0 us (4.5 TB/s: 224 workgroups), 4608 x 3584 7.6 us,
// of which 3 us are a launch. G = 4 took the first from 31 to 29 us, loads that go through the caches
// from 29 to 26.
#include "fp8_block.h"

namespace tf {
namespace {

template <int N>
__device__ __forceinline__ float rotate16(float v) {  // of the lane N below, in each row of 16 lanes
  return as_f32(dpp_ror<N>(as_u32(v)));
}

template <int KS, int D, int G, int TM>
__global__ __launch_bounds__(64 * KS) void block_gemv_kernel(BlockArgs a) {
  constexpr int MP = 16 / G, NG = D / G;
  static_assert(D % G == 0 && 64 % D == 0, "ring");
  static_assert(TM == 1 || G == 1, "row tiles or shared fragments");
  __shared__ f4 red[KS][TM][64];
  const int lane = threadIdx.x & 63;
  const int ks = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int c = lane & 15, g = lane >> 4;
  const int n0 = (int)blockIdx.x * 16, m0 = (int)blockIdx.y * MP * TM;

  f4 acc[TM];
#pragma unroll
  for (int t = 0; t < TM; ++t) acc[t] = f4{0.0f, 0.0f, 0.0f, 0.0f};

  const int blocks = ks < a.nkb ? (a.nkb - ks + KS - 1) / KS : 0;  // this wave's: ks, ks + KS, ...
  if (blocks > 0) {
    const int ncols = a.n - n0 < 16 ? a.n - n0 : 16;
    const int mrows = a.m - m0 < MP * TM ? a.m - m0 : MP * TM;
    const __amdgpu_buffer_rsrc_t rw =
        make_rsrc(a.w + (int64_t)n0 * a.ldw, (uint32_t)((ncols - 1) * (int)a.ldw + a.k));
    const __amdgpu_buffer_rsrc_t rx =
        make_rsrc(a.x8 + (int64_t)m0 * a.ldx, (uint32_t)((mrows - 1) * (int)a.ldx + a.k));
    const __amdgpu_buffer_rsrc_t rs =
        make_rsrc(a.xs + (int64_t)m0 * a.ldxs, (uint32_t)((mrows - 1) * (int)a.ldxs + a.nkb) * 4u);
    const uint32_t w_off = c < ncols ? (uint32_t)(c * (int)a.ldw + 32 * g) : kOutOfRange;
    const int row = c % MP, member = c / MP;  // this lane's row and place in a group of G blocks
    uint32_t x_off[TM], s_off[TM];
#pragma unroll
    for (int t = 0; t < TM; ++t) {
      const int r = 16 * t + row;
      x_off[t] = r < mrows ? (uint32_t)(r * (int)a.ldx + 32 * g + member * KS * kBlockK) : kOutOfRange;
      s_off[t] = r < mrows ? (uint32_t)(r * (int)a.ldxs + member * KS) * 4u : kOutOfRange;
    }
    const float* const wsp = a.ws + (int64_t)(n0 >> 7) * a.ldws;  // 16 columns lie in one scale block
    // Lane l holds the weight scale of the wave's block l of the current 64.
    auto load_ws = [&](int i) { return wsp[ks + KS * (i + lane < blocks ? i + lane : blocks - 1)]; };

    u4 w[D][2], x[NG][TM][2];
    float xs[NG][TM];
    // Blocks i .. i + G - 1 of the wave into group slot s. Past the last block, and past K inside it,
    // every load gives zeros.
    auto load = [&](int i, int s) __attribute__((always_inline)) {
      const int kb = ks + KS * i;
      const int base = i < blocks ? kb : 0;
      const int x_left = i + member < blocks ? a.k - (kb + member * KS) * kBlockK - 32 * g : 0;
#pragma unroll
      for (int t = 0; t < TM; ++t) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
          x[s][t][h] = __builtin_amdgcn_raw_buffer_load_b128(rx, (int)(16 * h < x_left ? x_off[t] : kOutOfRange),
                                                             base * kBlockK + 16 * h, 0);
        xs[s][t] = as_f32(
            __builtin_amdgcn_raw_buffer_load_b32(rs, (int)(i + member < blocks ? s_off[t] : kOutOfRange), base * 4, 0));
      }
#pragma unroll
      for (int j = 0; j < G; ++j) {
        const bool ok = i + j < blocks;
        const int left = ok ? a.k - (kb + j * KS) * kBlockK - 32 * g : 0;
#pragma unroll
        for (int h = 0; h < 2; ++h)
          w[s * G + j][h] = __builtin_amdgcn_raw_buffer_load_b128(
              rw, (int)(16 * h < left ? w_off : kOutOfRange), (ok ? kb + j * KS : 0) * kBlockK + 16 * h, 0);
      }
    };
    auto wide = [](const u4(&v)[2]) {
      return v8i{(int)v[0][0], (int)v[0][1], (int)v[0][2], (int)v[0][3],
                 (int)v[1][0], (int)v[1][1], (int)v[1][2], (int)v[1][3]};
    };
    float ws64 = load_ws(0);
#pragma unroll
    for (int s = 0; s < NG; ++s) load(G * s, s);
    for (int i0 = 0; i0 < blocks; i0 += D) {
      if ((i0 & 63) == 0 && i0 > 0) ws64 = load_ws(i0);
#pragma unroll
      for (int s = 0; s < NG; ++s) {
#pragma unroll
        for (int j = 0; j < G; ++j) {
          const int i = i0 + s * G + j;
          const float ws = as_f32((uint32_t)__builtin_amdgcn_readlane((int)as_u32(ws64), i & 63));
#pragma unroll
          for (int t = 0; t < TM; ++t) {
            // Past the last block ws is another block's: nothing may be added.
            const float sc = (G == 1 || member == j) && i < blocks ? ws * xs[s][t] : 0.0f;
            const f4 d = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(
                wide(w[s * G + j]), wide(x[s][t]), f4{0.0f, 0.0f, 0.0f, 0.0f}, 0, 0, 0, kUnitScale, 0, kUnitScale);
#pragma unroll
            for (int q = 0; q < 4; ++q) acc[t][q] = __builtin_fmaf(sc, d[q], acc[t][q]);
          }
        }
        load(i0 + D + s * G, s);
      }
    }
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      if (G >= 4) acc[0][q] += rotate16<4>(acc[0][q]);
      if (G >= 2) acc[0][q] += rotate16<8>(acc[0][q]);
    }
  }
#pragma unroll
  for (int t = 0; t < TM; ++t) red[ks][t][lane] = acc[t];
  __syncthreads();
  const int n = n0 + 4 * g;
  const bool vec = runs_aligned(a);
#pragma unroll
  for (int t = 0; t < TM; ++t) {
    const int m = m0 + 16 * t + c;
    if (ks != t % KS || c >= MP || m >= a.m || n >= a.n) continue;
    f4 sum = red[0][t][lane];
#pragma unroll
    for (int v = 1; v < KS; ++v) {
      const f4 p = red[v][t][lane];
#pragma unroll
      for (int q = 0; q < 4; ++q) sum[q] += p[q];
    }
    store_block4(a, m, n, sum, vec);
  }
}

template <int KS, int D, int G, int TM>
int launch(const BlockArgs& a, hipStream_t stream) {
  if (cdiv(a.n, 16) * (64 * KS) > 0xFFFFFFFF) return fail(TF_EINVAL, "tf_fp8_block_linear: too many columns");
  const dim3 grid((unsigned)cdiv(a.n, 16), (unsigned)cdiv(a.m, 16 / G * TM));
  block_gemv_kernel<KS, D, G, TM><<<grid, 64 * KS, 0, stream>>>(a);
  return check_launch("tf_fp8_block_linear(gemv)");
}

struct Entry {
  int bm, bn, warps, stages;
  int (*run)(const BlockArgs&, hipStream_t);
};

#define TF_GEMV(KS, D, G, TM) {16 / G * TM, 16, KS, D, launch<KS, D, G, TM>}
const Entry kEntries[] = {
    TF_GEMV(8, 4, 4, 1), TF_GEMV(4, 4, 4, 1), TF_GEMV(4, 4, 2, 1), TF_GEMV(4, 4, 1, 1), TF_GEMV(4, 2, 1, 2),
};

const Entry* find(const tf_gemm_config& cfg) {
  for (const Entry& e : kEntries)
    if (e.bm == cfg.block_m && e.bn == cfg.block_n && e.warps == cfg.num_warps && e.stages == cfg.num_stages) return &e;
  return nullptr;
}

}  // namespace

bool block_gemv_known(const tf_gemm_config& cfg) { return find(cfg) != nullptr; }

int launch_block_gemv(const BlockArgs& a, const tf_gemm_config& cfg, hipStream_t stream) {
  if (cdiv(a.m, cfg.block_m) > 65535) return fail(TF_EINVAL, "tf_fp8_block_linear: too many rows for the gemv form");
  return find(cfg)->run(a, stream);
}

}  // namespace tf
