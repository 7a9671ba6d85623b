// Block-scaled e4m3 linear, many rows: BM x BN tiles through LDS.
//
// A group of WM x WN waves streams 128-wide K blocks of x and the weight, and the rows' scales of
// the block, into S LDS stages by buffer->LDS loads issued up to S blocks ahead, one barrier a block.
// A wave computes a (16 TM) x (16 TN) sub-tile: per block one v_mfma_scale_f32_16x16x128_f8f6f4
// (unit MFMA scales) per 16 x 16 from a zero accumulator, then acc += (xs[m] * ws) * that in fp32.
// The weight fragment is the first operand: lane l holds row l % 16 and columns 4 (l / 16) + q, so a
// lane's four results share one scale, and the wave's columns lie in one 128-wide scale block.
//
// A block's scale needs its own sum, so four VALU multiply-adds go with each MFMA of 32 cycles: with both
// interleaved in registers alone, random codes reach 3.5 PFLOP/s on MI355X (MFMAs alone 4.0 to 4.4; the
// nominal peak 5.0). The 256 x 256 tile reaches 2.06 (gate_up, N = 37888, K = 3584, M = 4096: 539 us a call
// among others; the library's fp8 product of that size with one scale per tensor 504 us). Without its
// loads it takes 416 us, the loads alone 417, both 500: a stage of 64 KB is one block ahead (LDS holds two),
// so its latency is covered by one block's MFMAs only. Of 9.25 rounds of tiles the last is a quarter full.
// The smaller tiles serve fewer rows, where the weight's bytes bind: gate_up M = 48 33.7 us (4.1 TB/s) on 64 x 256.
//
// Farthest from the floor are 64 to 2500 rows (1.4 to 5 times the bytes or products alone): a tile count just
// past the CUs' costs a round more, each row tile reads the weight again, and with one workgroup a CU its
// first loads and its epilogue stand alone.
//
// WK: K groups of a workgroup, each with waves and stages of its own over a share of the K blocks; the
// sums of the others go to the first through LDS. For tiles so few that a CU has one: it then has WK times
// the waves and loads in flight, and needs neither a second kernel nor partial sums in memory. Best of the
// tiles with WK > 1 against best of those without, us on MI355X: 3584 x 3584 M = 48 9.4 (32 x 64, WK 4)
// against 11.5, M = 333 15.6 (64 x 128, WK 2) against 21.5; 896 x 4864 M = 333 11.2 against 14.7.
//
// What did not help: w refilled half a block earlier behind a second barrier (602 us against 584), lines
// asked for ahead into L2 (620 against 600), wave priorities (no change), bands of 4 or 16 rows (552, 568
// against 553).
//
// LDS rows are 128 bytes, 16-byte chunk c of row r in slot c ^ s(r), s(r) = 2 (r % 4) ^ ((r / 4) % 2):
// with lane l at row l % 16 and chunks 2 (l / 16) + {0, 1} the reads are free of bank conflicts.
#include "fp8_block.h"

namespace tf {
namespace {

__device__ __forceinline__ int slot_xor(int row) { return ((row & 3) << 1) ^ ((row >> 2) & 1); }

template <int BM, int BN, int WM, int WN, int S, int WK>
struct Tile {
  static constexpr int kWaves = WM * WN;  // of one K group
  static constexpr int TM = BM / WM / 16;
  static constexpr int TN = BN / WN / 16;
  static constexpr int kXBytes = BM * kBlockK;
  static constexpr int kWBytes = BN * kBlockK;
  static constexpr int kStage = kXBytes + kWBytes;
  // Row scales: four K blocks of every row at a time, [BM][4] fp32, in a ring of its own. A wave's
  // load brings 16 rows x 4 blocks, so a row's line is read once for four blocks.
  static constexpr int kScaleRows = 16 * kWaves < BM ? 16 * kWaves : BM;  // rows the waves bring in one step
  static constexpr int kScaleSteps = BM / kScaleRows;
  static constexpr int kScaleRing = S <= 3 ? 2 : 4;
  static constexpr int kScaleBuf = BM * 16;
  static constexpr int kGroup = S * kStage + kScaleRing * kScaleBuf + 256;
  static constexpr int kOut = kWaves * 16 * (16 * TN * 4 + 16);        // the epilogue's transposition
  static constexpr int kSums = (WK - 1) * kWaves * TM * TN * 64 * 16;  // the other K groups' sums
  static constexpr int kLds = WK * kGroup > kOut + kSums ? WK * kGroup : kOut + kSums;
  static constexpr int kXLoads = BM / 8 / kWaves;  // 1 KB loads per wave and stage
  static constexpr int kWLoads = BN / 8 / kWaves;
  static constexpr int kLoads = kXLoads + kWLoads + 1;
  static_assert(BM % (8 * kWaves) == 0 && BN % (8 * kWaves) == 0, "a stage splits evenly over the waves");
  static_assert(BM % (16 * WM) == 0 && BN % (16 * WN) == 0, "wave tile");
  static_assert(128 % (16 * TN) == 0, "a wave's columns lie in one scale block");
  static_assert(TN == 2 || TN == 4, "the epilogue's rows take whole waves");
  static_assert(TM % 2 == 0, "the pipeline's two register sets alternate over whole blocks");
  static_assert(kScaleSteps == 1 || kScaleSteps == 2, "a group's scales come with two stages at most");
  static_assert(kLds <= 160 * 1024, "LDS");
};

constexpr int64_t kL2Bytes = 4 << 20;  // of one XCD

template <int N>
__device__ __forceinline__ void stage_barrier() {
  static_assert(N >= 0 && N < 64, "vmcnt range");
  __builtin_amdgcn_sched_barrier(0);
  __builtin_amdgcn_s_waitcnt((N & 0xF) | (0x7 << 4) | (0x0 << 8) | ((N >> 4) << 14));
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_sched_barrier(0);
}

typedef __attribute__((address_space(3))) void* lds_ptr;

// 64 lanes x 16 bytes to the 1 KB at base + 1024 j, lane l's at 16 l.
__device__ __forceinline__ void load16(__amdgpu_buffer_rsrc_t r, uint8_t* base, int j, uint32_t off, int soff) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lds_ptr)(base + j * 1024), 16, off, soff, 0, 0);
}

// STREAM: the output, larger than the XCDs' L2s, goes past them and leaves them to the panels (gate_up M =
// 4096 on MI355X: 532 us, and 548 through them).
template <int BM, int BN, int WM, int WN, int S, int WK, bool STREAM>
__global__ __launch_bounds__(64 * WM * WN * WK) void block_gemm_kernel(BlockArgs a, float* __restrict__ part,
                                                                       int split_k, int tiles_m, int tiles_n) {
  using C = Tile<BM, BN, WM, WN, S, WK>;
  constexpr int TM = C::TM, TN = C::TN;
  extern __shared__ __attribute__((aligned(16))) uint8_t all_smem[];

  const int lane = threadIdx.x & 63;
  const int wave_of_all = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int group = wave_of_all / C::kWaves, wave = wave_of_all % C::kWaves;
  uint8_t* const smem = all_smem + group * C::kGroup;  // the group's stages
  uint8_t* const s_lds = smem + S * C::kStage;
  const int wm = wave / WN, wn = wave % WN;

  // Tiles in bands of 8 tile rows, the rows of a band innermost: the 32 tiles an XCD has in flight
  // then read about 8 + 4 panels.
  const int t = xcd_tile(blockIdx.x, gridDim.x);
  const int plane = tiles_m * tiles_n;
  const int z = t / plane;
  const int r0 = t - z * plane;
  const int band = r0 / (8 * tiles_n);
  const int in_band = r0 - band * 8 * tiles_n;
  const int rows = tiles_m - band * 8 < 8 ? tiles_m - band * 8 : 8;
  const int m0 = (band * 8 + in_band % rows) * BM;
  const int n0 = (in_band / rows) * BN;

  // The slice's K blocks, and this group's share of them; every group takes as many steps as the longest.
  const int slice0 = (int)(((int64_t)z * a.nkb) / split_k);
  const int slice1 = (int)(((int64_t)(z + 1) * a.nkb) / split_k);
  const int steps = (slice1 - slice0 + WK - 1) / WK;
  const int kb0 = slice0 + group * steps;
  const int kb1 = kb0 + steps < slice1 ? kb0 + steps : (kb0 < slice1 ? slice1 : kb0);

  const int mrows = a.m - m0 < BM ? a.m - m0 : BM;
  const int ncols = a.n - n0 < BN ? a.n - n0 : BN;
  const uint8_t* const xp = a.x8 + (int64_t)m0 * a.ldx;
  const uint8_t* const wp = a.w + (int64_t)n0 * a.ldw;
  const float* const sp = a.xs + (int64_t)m0 * a.ldxs;
  const uint32_t x_bytes = (uint32_t)((mrows - 1) * (int)a.ldx + a.k);
  const uint32_t w_bytes = (uint32_t)((ncols - 1) * (int)a.ldw + a.k);
  const uint32_t s_bytes = (uint32_t)((mrows - 1) * (int)a.ldxs + a.nkb) * 4u;

  // Load i of a wave fills 64 consecutive 16-byte slots: slot 64 (wave + waves i) + lane of a stage's x
  // (then w), row (8 (wave + waves i) + lane / 8). A lane's chunk is the same in all of them.
  uint32_t x_off[C::kXLoads], w_off[C::kWLoads];
  const int chunk = ((lane & 7) ^ slot_xor(lane >> 3)) * 16;
#pragma unroll
  for (int i = 0; i < C::kXLoads; ++i) {
    const int row = (wave + C::kWaves * i) * 8 + (lane >> 3);
    x_off[i] = row < mrows ? (uint32_t)(row * (int)a.ldx + chunk) : kOutOfRange;
  }
#pragma unroll
  for (int i = 0; i < C::kWLoads; ++i) {
    const int row = (wave + C::kWaves * i) * 8 + (lane >> 3);
    w_off[i] = row < ncols ? (uint32_t)(row * (int)a.ldw + chunk) : kOutOfRange;
  }
  // Scales of K blocks kb0 + 4 G .. + 3 (group G): lane l brings row l / 4, block l % 4. Group G + 1
  // comes with the last stages of group G (the second of them where kScaleSteps is 1), after
  // every wave has read the group whose buffer it takes, and before its own first block.
  const int s_row = (wave * 16) % C::kScaleRows;
  auto issue_scales = [&](int g, int part, bool real) __attribute__((always_inline)) {
    const __amdgpu_buffer_rsrc_t rs = make_rsrc(sp, real ? s_bytes : 0u);
    const int row0 = part * C::kScaleRows + s_row, row = row0 + (lane >> 2);
    const uint32_t off = row < mrows ? (uint32_t)(row * (int)a.ldxs + (lane & 3)) * 4u : kOutOfRange;
    // An empty load writes zeros: past the ring, where nothing is read.
    uint8_t* const to = s_lds + (real ? (g % C::kScaleRing) * C::kScaleBuf + row0 * 16 : C::kScaleRing * C::kScaleBuf);
    __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (lds_ptr)to, 4, off, real ? (kb0 + 4 * g) * 4 : 0, 0, 0);
  };

  // Load l of a wave for block kb into stage st: x, w, then the scales that come along. A block past
  // the slice is loaded through an empty resource: zeros, without touching memory.
  auto issue = [&](int kb, int st, int l) __attribute__((always_inline)) {
    const bool ok = kb < kb1;
    const int soff = ok ? kb * kBlockK : 0;
    uint8_t* const base = smem + st * C::kStage;
    if (l < C::kXLoads) {
      load16(make_rsrc(xp, ok ? x_bytes : 0u), base, wave + C::kWaves * l, x_off[l < C::kXLoads ? l : 0], soff);
    } else if (l < C::kXLoads + C::kWLoads) {
      const int i = l < C::kXLoads || l >= C::kXLoads + C::kWLoads ? 0 : l - C::kXLoads;
      load16(make_rsrc(wp, ok ? w_bytes : 0u), base + C::kXBytes, wave + C::kWaves * i, w_off[i], soff);
    } else {
      const int in_group = (kb - kb0) & 3, g = ((kb - kb0) >> 2) + 1;
      const int part = in_group - (4 - C::kScaleSteps);
      issue_scales(g, part < 0 ? 0 : part, part >= 0 && kb0 + 4 * g < kb1);
    }
  };
  // Before a block's first load: where K ends inside it, the last one, chunks past it are zeros on both
  // sides, from there on (only empty blocks follow).
  auto mask_tail = [&](int kb) __attribute__((always_inline)) {
    if (kb < kb1 && a.k - kb * kBlockK <= chunk) {
#pragma unroll
      for (int i = 0; i < C::kXLoads; ++i) x_off[i] = kOutOfRange;
#pragma unroll
      for (int i = 0; i < C::kWLoads; ++i) w_off[i] = kOutOfRange;
    }
  };

  f4 acc[TM][TN];
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j) acc[i][j] = f4{0.0f, 0.0f, 0.0f, 0.0f};

  // Fragment reads: rows 16 apart keep their slots, so a fragment is two chunks at a constant offset.
  const int c16 = lane & 15;
  const int slot = (2 * (lane >> 4)) ^ slot_xor(c16);
  const int x_row = wm * TM * 16 + c16;
  const uint32_t x_at = (uint32_t)(x_row * 8 + slot) * 16u;
  const uint32_t w_at = C::kXBytes + (uint32_t)((wn * TN * 16 + c16) * 8 + slot) * 16u;
  auto frag = [&](const uint8_t* stage, uint32_t at, int i) {
    const u4 lo = *reinterpret_cast<const u4*>(stage + at + i * 16 * kBlockK);
    const u4 hi = *reinterpret_cast<const u4*>(stage + (at ^ 16u) + i * 16 * kBlockK);
    return v8i{(int)lo[0], (int)lo[1], (int)lo[2], (int)lo[3], (int)hi[0], (int)hi[1], (int)hi[2], (int)hi[3]};
  };
  // The wave's columns share one scale per block; lane l holds that of block kb0 + l of the current 64, read
  // by lane number, as neither a scalar load (it shares the LDS reads' counter, and waiting for it
  // waits for all of them) nor a vector load (it would wait for the stage loads) then stands in the loop.
  // Columns past N are never stored.
  int nb = (n0 + wn * TN * 16) >> 7;
  nb = nb <= ((a.n - 1) >> 7) ? nb : (a.n - 1) >> 7;
  const float* const wsp = a.ws + (int64_t)nb * a.ldws;
  const int kb_last = (kb1 <= a.nkb ? kb1 : a.nkb) - 1;  // a K group without a block may start past the last
  auto load_ws = [&](int kb) { return wsp[kb + lane < kb1 ? kb + lane : kb_last]; };
  float ws64 = load_ws(kb0);

#pragma unroll
  for (int i = 0; i < C::kScaleSteps; ++i) issue_scales(0, i, kb0 < kb1);
#pragma unroll
  for (int s = 0; s < S; ++s) {
    mask_tail(kb0 + s);
#pragma unroll
    for (int l = 0; l < C::kLoads; ++l)
      if (s < S - 1 || l < TN) issue(kb0 + s, s, l);  // the last stage's others go out in the first block
  }
  stage_barrier<(S - 2) * C::kLoads + (TN < C::kLoads ? TN : C::kLoads)>();
  // Software pipeline: the fragments of a step are read one step ahead, its results are scaled one
  // step after its MFMAs, and the barrier to the next block stands before a block's last step: by
  // then a wave has read all of its stage, so the stage is refilled and the next block's first
  // fragments are read beside that step's MFMAs. The refill's loads go out one after each of these
  // MFMAs and two after each of the next step's: together, ahead of them, they hold the wave up
  // (gate_up M = 4096 on MI355X: 584 us against 555; later ones arrive late: 592 to 608).
  v8i bf[TN], af[2];
  float xs[2], sc[2] = {0.0f, 0.0f};
  f4 d[2][TN];
#pragma unroll
  for (int j = 0; j < TN; ++j) {
    bf[j] = frag(smem, w_at, j);
    d[(TM - 1) & 1][j] = f4{0.0f, 0.0f, 0.0f, 0.0f};
  }
  af[0] = frag(smem, x_at, 0);
  auto scale = [&](int step, int i) {  // of row x_row + 16 i, K block kb0 + step
    return *reinterpret_cast<const float*>(s_lds + ((step >> 2) % C::kScaleRing) * C::kScaleBuf + (step & 3) * 4 +
                                           (x_row + 16 * i) * 16);
  };
  xs[0] = scale(0, 0);
  int st = 0;
  for (int kb = kb0; kb < kb0 + steps; ++kb) {
    const uint8_t* const stage = smem + st * C::kStage;
    const int next = st + 1 == S ? 0 : st + 1;
    const uint8_t* const stage2 = smem + next * C::kStage;
    const int at = (kb - kb0) & 63;
    if (at == 0 && kb > kb0) {
      ws64 = load_ws(kb);
      __asm__ volatile("" : "+v"(ws64));  // waits for it here, not at its uses
    }
    const float ws = as_f32((uint32_t)__builtin_amdgcn_readlane((int)as_u32(ws64), at));
#pragma unroll
    for (int i = 0; i < TM; ++i) {
      if (i + 1 < TM) {
        af[(i + 1) & 1] = frag(stage, x_at, i + 1);
        xs[(i + 1) & 1] = scale(kb - kb0, i + 1);
      } else {
        stage_barrier<(S - 2) * C::kLoads>();
        mask_tail(kb + S);
        af[(i + 1) & 1] = frag(stage2, x_at, 0);
        xs[(i + 1) & 1] = scale(kb + 1 - kb0, 0);
      }
      // Past a shorter group's last block the codes are zeros and the scales anything.
      sc[i & 1] = WK == 1 || kb < kb1 ? xs[i & 1] * ws : 0.0f;
      constexpr int kLast = TM - 1;
      const int p = i == 0 ? kLast : i - 1;  // the step whose results are scaled here
#pragma unroll
      for (int j = 0; j < TN; ++j) {
        d[i & 1][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(bf[j], af[i & 1], f4{0.0f, 0.0f, 0.0f, 0.0f}, 0,
                                                                       0, 0, kUnitScale, 0, kUnitScale);
#pragma unroll
        for (int q = 0; q < 4; ++q)
          acc[p][j][q] = __builtin_fmaf(sc[(i + 1) & 1], d[(i + 1) & 1][j][q], acc[p][j][q]);
        // Holds the MFMA and the scaling here: without a use in order they are moved to their results' uses.
        __asm__ volatile("" : "+v"(d[i & 1][j]), "+v"(acc[p][j]));
        if (i + 1 == TM) {
          bf[j] = frag(stage2, w_at, j);  // in place, its last MFMA issued
          if (j < C::kLoads) issue(kb + S, st, j);
        }
        if (i == 0) {
#pragma unroll
          for (int l = TN; l < C::kLoads; ++l)
            if ((l - TN) / 2 == j || (j + 1 == TN && (l - TN) / 2 > j)) issue(kb + S - 1, st == 0 ? S - 1 : st - 1, l);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    st = next;
  }
#pragma unroll
  for (int j = 0; j < TN; ++j)
#pragma unroll
    for (int q = 0; q < 4; ++q)
      acc[TM - 1][j][q] = __builtin_fmaf(sc[(TM - 1) & 1], d[(TM - 1) & 1][j][q], acc[TM - 1][j][q]);

  // ---- epilogue. A lane holds runs of four columns of 16 rows, 32 bytes of each line; each wave
  // turns 16 rows x 16 TN columns at a time over through LDS (its own part of the stages, free once every
  // wave's last, empty loads have ended), so that a store covers whole 128-byte pieces (TN 4) of its
  // rows.
  const bool partial = split_k > 1;
  const bool wide = (a.n & 7) == 0 && (partial || wide_rows(a));
  const int n_wave = n0 + wn * TN * 16;
  const int g4 = 4 * (lane >> 4);
  stage_barrier<0>();
  if (WK > 1) {  // the groups' sums, added in group order
    f4* const sums = reinterpret_cast<f4*>(all_smem + C::kOut) + wave * TM * TN * 64 + lane;
#pragma unroll
    for (int i = 0; i < TM * TN; ++i)
      if (group > 0) sums[((group - 1) * C::kWaves * TM * TN + i) * 64] = acc[i / TN][i % TN];
    __syncthreads();
    if (group > 0) return;
#pragma unroll
    for (int v = 0; v < WK - 1; ++v)
#pragma unroll
      for (int i = 0; i < TM * TN; ++i) {
        const f4 p = sums[(v * C::kWaves * TM * TN + i) * 64];
#pragma unroll
        for (int q = 0; q < 4; ++q) acc[i / TN][i % TN][q] += p[q];
      }
  }
  if (wide) {
    constexpr int kCols = 16 * TN, kRow = kCols * 4 + 16;  // LDS row in bytes, padded off the banks of the next
    constexpr int kLanes = kCols / 8;                      // lanes per row, eight columns each
    uint8_t* const mine = all_smem + wave * 16 * kRow;
#pragma unroll
    for (int i = 0; i < TM; ++i) {
#pragma unroll
      for (int j = 0; j < TN; ++j) *reinterpret_cast<f4*>(mine + c16 * kRow + (16 * j + g4) * 4) = acc[i][j];
      __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "wavefront");
#pragma unroll
      for (int h = 0; h < 16 * kLanes / 64; ++h) {
        const int row = h * (64 / kLanes) + lane / kLanes, col = (lane % kLanes) * 8;
        const f4 lo = *reinterpret_cast<const f4*>(mine + row * kRow + col * 4);
        const f4 hi = *reinterpret_cast<const f4*>(mine + row * kRow + col * 4 + 16);
        const int m = m0 + (wm * TM + i) * 16 + row, n = n_wave + col;
        if (m >= a.m || n >= a.n) continue;
        if (partial) {
          f4* const p = reinterpret_cast<f4*>(part + ((int64_t)z * a.m + m) * a.n + n);
          p[0] = lo;
          p[1] = hi;
        } else {
          store_block8<STREAM>(a, m, n, lo, hi);
        }
      }
      __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "wavefront");
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < TM; ++i) {
    const int m = m0 + x_row + 16 * i;
    if (m >= a.m) continue;
#pragma unroll
    for (int j = 0; j < TN; ++j) {
      const int n = n_wave + 16 * j + g4;
      if (n >= a.n) continue;
      if (partial) {
        float* const p = part + ((int64_t)z * a.m + m) * a.n + n;
#pragma unroll
        for (int q = 0; q < 4; ++q)
          if (n + q < a.n) p[q] = acc[i][j][q];
      } else {
        store_block4(a, m, n, acc[i][j], false);
      }
    }
  }
}

// Sum of the K slices in slice order, then the epilogue; four columns a thread.
__global__ __launch_bounds__(256) void block_reduce_kernel(BlockArgs a, const float* __restrict__ part, int split_k,
                                                           int runs) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t m = i / runs;
  if (m >= a.m) return;
  const int n = (int)(i - m * runs) * 4;
  const int64_t plane = (int64_t)a.m * a.n;
  const float* const p = part + m * a.n + n;
  f4 sum = {0.0f, 0.0f, 0.0f, 0.0f};
  if ((a.n & 3) == 0) {
    for (int z0 = 0; z0 < split_k; z0 += 4) {  // four slices' loads in flight
      f4 v[4];
#pragma unroll
      for (int z = 0; z < 4; ++z)
        v[z] = z0 + z < split_k ? *reinterpret_cast<const f4*>(p + (z0 + z) * plane) : f4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int z = 0; z < 4; ++z)
#pragma unroll
        for (int q = 0; q < 4; ++q) sum[q] += v[z][q];
    }
  } else {
    for (int z = 0; z < split_k; ++z)
#pragma unroll
      for (int q = 0; q < 4; ++q)
        if (n + q < a.n) sum[q] += p[z * plane + q];
  }
  store_block4(a, (int)m, n, sum, runs_aligned(a));
}

template <int BM, int BN, int WM, int WN, int S, int WK>
int launch(const BlockArgs& a, int split, float* part, hipStream_t stream) {
  using C = Tile<BM, BN, WM, WN, S, WK>;
  const int tiles_m = (int)cdiv(a.m, BM), tiles_n = (int)cdiv(a.n, BN);
  const int64_t grid = (int64_t)tiles_m * tiles_n * split;
  if (grid * (64 * C::kWaves * WK) > 0xFFFFFFFF) return fail(TF_EINVAL, "tf_fp8_block_linear: too many tiles");
  constexpr bool kMayStream = BM == 256;  // the tile of large outputs
  const bool stream_out = kMayStream && split == 1 && (int64_t)a.m * a.n * 2 > (int64_t)kXcds * kL2Bytes;
  auto kernel =
      stream_out ? block_gemm_kernel<BM, BN, WM, WN, S, WK, kMayStream> : block_gemm_kernel<BM, BN, WM, WN, S, WK, false>;
  if (C::kLds > 64 * 1024 &&
      hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize,
                          C::kLds) != hipSuccess)
    return fail(TF_ELAUNCH, "tf_fp8_block_linear: cannot reserve LDS");
  kernel<<<(unsigned)grid, 64 * C::kWaves * WK, C::kLds, stream>>>(a, part, split, tiles_m, tiles_n);
  if (int rc = check_launch("tf_fp8_block_linear(gemm)")) return rc;
  if (split == 1) return TF_OK;
  const int runs = (int)cdiv(a.n, 4);
  const int64_t groups = cdiv((int64_t)a.m * runs, 256);
  block_reduce_kernel<<<(unsigned)groups, 256, 0, stream>>>(a, part, split, runs);
  return check_launch("tf_fp8_block_linear(reduce)");
}

struct Entry {
  int bm, bn, warps, stages;
  int (*run)(const BlockArgs&, int, float*, hipStream_t);
};

#define TF_BLOCK(BM, BN, WM, WN, S, WK) {BM, BN, WM * WN * WK, S, launch<BM, BN, WM, WN, S, WK>}
const Entry kEntries[] = {
    TF_BLOCK(256, 256, 2, 4, 2, 1), TF_BLOCK(128, 256, 2, 4, 3, 1), TF_BLOCK(128, 128, 2, 4, 4, 1),
    TF_BLOCK(64, 256, 2, 4, 3, 1),  TF_BLOCK(64, 128, 2, 2, 3, 2),  TF_BLOCK(64, 64, 2, 2, 4, 2),
    TF_BLOCK(32, 128, 1, 4, 4, 1),  TF_BLOCK(32, 64, 1, 2, 3, 4),
};

const Entry* find(const tf_gemm_config& cfg) {
  for (const Entry& e : kEntries)
    if (e.bm == cfg.block_m && e.bn == cfg.block_n && e.warps == cfg.num_warps && e.stages == cfg.num_stages) return &e;
  return nullptr;
}

}  // namespace

bool block_gemm_known(const tf_gemm_config& cfg) { return cfg.split_k >= 1 && find(cfg) != nullptr; }

int block_split(const tf_gemm_config& cfg, int64_t nkb) {
  return (int)(cfg.split_k < nkb ? cfg.split_k : (nkb > 0 ? nkb : 1));
}

int launch_block_gemm(const BlockArgs& a, const tf_gemm_config& cfg, float* part, hipStream_t stream) {
  return find(cfg)->run(a, block_split(cfg, a.nkb), part, stream);
}

}  // namespace tf
