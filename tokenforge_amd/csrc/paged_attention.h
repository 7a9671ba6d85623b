// Attention of one new token per sequence over a paged cache: the kernel template, instantiated by head length
// in paged_attention_d*.hip, launched and joined by paged_attention.hip.
//
// Work. Items are (sequence, key-value head, 16 or 32 of its query heads); an item is a run of steps of 16 NT tokens.
// All items' steps form one line, and workgroup w takes the steps [w share, (w + 1) share) of it: parts that end with
// their item where the grid is enough for those, else equal ones across items, whatever the sequences' lengths are.
// Lengths are read on the device; the host knows none. Items that lie in one workgroup are finished by it, the others
// leave (maximum, sum, accumulator) in the workspace for the join. Where the table's rows are short, a workgroup takes an
// item and there is no line.
//
// Memory bound: every cached byte is read once (counters: 1.004 to 1.02 times the cache's bytes), 4 q_heads d flops a
// token are 3% of the matrix rate at that speed. On MI355X (copy of 1 GiB 5.14 TB/s), head length 128, 28 query on 4
// key-value heads, us: 64 sequences of 2000 to 16384 tokens in bf16 (929 MB) 147 and 5 for the join, 32 of up to 4096
// (69 MB) 15.6 and 3.9, 128 of up to 2048 in e4m3 (90 MB) 24.8 in one launch, one of 32749 in e4m3 (35 MB) 11.8 and
// 4.9. Beside the bytes a call takes some 5.5 (a launch; lengths, table and keys wait for each other; the
// last join in LDS).
//
// A wave takes every fourth step. S^T = K Q^T by v_mfma_f32_16x16x32 with 16 tokens as rows and 16 query heads as
// columns: lane 16g + c then holds head c's scores of tokens 4g .. 4g + 3 of each tile, which is, for the second
// product O^T = V^T P^T, the operand P^T of two tiles (its 8 consecutive k of lane 16g + c are those tokens):
// probabilities never leave their lane. V^T's operand wants 8 tokens of one channel; a lane loads the same 8
// tokens' CS consecutive channels (whole rows, 16 lanes a row) and turns them over in registers, one v_perm_b32
// for 4 bytes. No step goes through LDS. Running maximum, sum and accumulator are fp32; the waves' are joined in
// LDS when an item ends.
//
// Probabilities go into the second product as two 16-bit halves, 16 bits together in bf16, 21 in fp16 (fewer below 2^-19
// of the row's largest, split2): the product is memory bound, and with one half alone a bf16 result is off by 1.4 times
// its own rounding. The lower half is not zero where the upper is not, so that an infinite value times it is infinite and
// not NaN. Scales of e4m3 values go into the probabilities before the split, e4m3 codes into bf16 (exact).
#pragma once

#include "kv_cache.h"

namespace tf {

struct AttnArgs {
  const uint16_t* q;
  int64_t q_row, q_head;  // elements
  const uint8_t* k;
  const uint8_t* v;
  int64_t k_page, k_head, v_page, v_head;  // bytes
  uint32_t k_token, v_token;               // bytes
  const float* ks;
  const float* vs;
  int64_t ks_page, ks_head, vs_page, vs_head;  // elements
  uint32_t ks_token, vs_token;
  const int32_t* table;
  int64_t table_row;
  const int32_t* lens;
  uint16_t* out;
  float* part;  // [2 grid] pieces of part_rows rows
  int2* ends;   // [items] first and last workgroup of an item
  int64_t pages;
  PageDiv page;
  int m, heads, group, row_groups, part_rows, d;
  int cap;     // tokens a row of the table covers
  int window;
  float scale_log2;
  int direct;  // a workgroup takes a whole item; else the items' steps lie on one line
};

// Tokens of a step. Two tiles make the second product's k; four where a tile is 2 KB or less (heads up to 64), whose
// steps would end before the next one's loads are back.
constexpr int attention_step(int dp) { return dp == 64 ? 64 : 32; }

// Workgroups a CU holds, and the grid of the shared line: two by their 167 to 256 registers, one for heads past 128
// (320 to 420, and 134 KB of LDS).
constexpr int attention_resident(int dp) { return dp > 128 ? 1 : 2; }
constexpr int attention_grid(int dp) { return 256 * attention_resident(dp); }

// Floats of a piece: the rows' accumulators, then their (maximum, sum), up to 16 bytes.
__host__ __device__ constexpr int64_t piece_floats(int rows, int dp) { return rows * dp + (2 * rows + 3) / 4 * 4; }

// Bytes of keys and values from which a call's loads are nontemporal, by what its line holds or, where a workgroup takes
// a whole item and none knows the others' lengths, by what the table covers. Each byte is read once; a call that fills
// a good part of the 256 MB last-level cache only pushes out of it what other kernels left. MI355X, three caches in
// turn, us without and with: 64 sequences of 2000 to 16384 tokens (929 MB) 169 and 150, 8 of 8192 (134 MB) 31.7 and
// 28.5; 32 of up to 4096 (69 MB), where three caches stay in it, 19.2 and 21.4. Whole items: 512 sequences of up to 512
// tokens (table 537 MB) 97.4 and 92.1, 128 of up to 2048 in e4m3 (table 268 MB) 24.1 and 26.3. Only the form of whole
// tiles and exact head lengths has such a loop.
constexpr int64_t kStreamLine = 100 << 20, kStreamTable = 384 << 20;

// Where a workgroup leaves its part of an item: it has at most two such, of an item that began before it and of one
// that begins in it and goes on behind it.
__host__ __device__ __forceinline__ int64_t piece_of(int workgroup, bool begins) {
  return 2 * (int64_t)workgroup + (begins ? 1 : 0);
}

// Tokens [begin, end) of sequence b, and its steps of KS tokens.
template <int KS>
struct Span {
  int begin, end;
  uint32_t first, count;
  __device__ __forceinline__ Span(int b, int e, uint32_t f, uint32_t c) : begin(b), end(e), first(f), count(c) {}
  __device__ __forceinline__ Span(const AttnArgs& a, int b) {
    int n = a.lens[b];
    n = n < 0 ? 0 : n > a.cap ? a.cap : n;
    end = n;
    begin = a.window > 0 && n > a.window ? n - a.window : 0;
    first = (uint32_t)begin / KS;
    count = n > 0 ? ((uint32_t)n + KS - 1) / KS - first : 0u;
  }
};

typedef __bf16 b8 __attribute__((ext_vector_type(8)));
typedef __bf16 b2 __attribute__((ext_vector_type(2)));

template <bool WIDE>
__device__ __forceinline__ f4 mfma16(u4 a, u4 b, f4 c) {
  if (WIDE)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b8, a), __builtin_bit_cast(b8, b), c, 0, 0, 0);
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, a), __builtin_bit_cast(h8, b), c, 0, 0, 0);
}

// Two codes (the low or high half of a word) as a pair of 16-bit values, exactly.
template <bool WIDE, bool HI>
__device__ __forceinline__ uint32_t codes2(uint32_t w) {
  if (WIDE) return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, HI));
  return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, HI));
}

// Max (sum) over lanes c, c + 16, c + 32, c + 48, in each of them.
__device__ __forceinline__ float max4(float v) {
  auto s = __builtin_amdgcn_permlane16_swap(as_u32(v), as_u32(v), false, false);
  v = __builtin_fmaxf(as_f32(s[0]), as_f32(s[1]));
  s = __builtin_amdgcn_permlane32_swap(as_u32(v), as_u32(v), false, false);
  return __builtin_fmaxf(as_f32(s[0]), as_f32(s[1]));
}
__device__ __forceinline__ float sum4(float v) {
  auto s = __builtin_amdgcn_permlane16_swap(as_u32(v), as_u32(v), false, false);
  v = as_f32(s[0]) + as_f32(s[1]);
  s = __builtin_amdgcn_permlane32_swap(as_u32(v), as_u32(v), false, false);
  return as_f32(s[0]) + as_f32(s[1]);
}

// Probabilities p0, p1 as two pairs that add up to them (see the top). bf16: truncated, and what is left. fp16, of
// probabilities times kUp: a little less than truncated, and what is left, rounded.
//
// fp16 pairs end on the subnormals' step of 2^-24, 2^-39 of the row's largest: a probability is off by half of that,
// or by 2^-21 of itself if that is more, to either side, so 16 bits hold down to 2^-24 of the largest (16.6 in the
// scores), 12 at 2^-28. kUp is the most that the largest may be multiplied by. What is left is 2^-24 or more wherever
// the upper half is not 0 (the product with 1 - 2^-12 and the 2^-24 taken off see to it for values that fp16 holds
// exactly), so that an infinite value stays one for probabilities from 2^-37 of the largest on; far below, and in bf16
// below 2^-106, it gives NaN, as in fp32 below 2^-149.
constexpr float kUp = 0x1p15f;

template <bool WIDE>
__device__ __forceinline__ void split2(float p0, float p1, uint32_t& hi, uint32_t& lo) {
  if (WIDE) {
    hi = __builtin_amdgcn_perm(as_u32(p1), as_u32(p0), 0x07060302u);
    const float r0 = p0 - as_f32(as_u32(p0) & 0xFFFF0000u), r1 = p1 - as_f32(as_u32(p1) & 0xFFFF0000u);
    lo = round_pair<BF16>(r0 != 0.0f ? r0 : p0 * 0x1p-20f, r1 != 0.0f ? r1 : p1 * 0x1p-20f);
  } else {
    constexpr float kLess = kUp * (1.0f - 0x1p-12f);
    const auto h = __builtin_amdgcn_cvt_pkrtz(__builtin_fmaxf(__builtin_fmaf(p0, kLess, -0x1p-24f), 0.0f),
                                              __builtin_fmaxf(__builtin_fmaf(p1, kLess, -0x1p-24f), 0.0f));
    hi = __builtin_bit_cast(uint32_t, h);
    lo = round_pair<F16>(__builtin_fmaf(p0, kUp, -(float)h[0]), __builtin_fmaf(p1, kUp, -(float)h[1]));
  }
}

// T: type of q, out and 16-bit caches. DP: head length the tiles hold (d <= DP). PAGED: pages hold whole tiles of
// 16 tokens (and scales go by 16-byte loads), so a tile's place is one scalar; else every token is looked up. FULL:
// d == DP. MT: 16s of query heads that share the loads of an item.
template <typename T, bool FP8, int DP, int MT, bool PAGED, bool FULL>
struct Attn {
  static constexpr int kWaves = 4;
  static constexpr int NT = attention_step(DP) / 16;  // tiles of 16 tokens a step
  static constexpr int KS = 16 * NT;
  static constexpr int NK = DP / 32;                  // MFMAs over the channels
  static constexpr int NSUB = DP > 128 ? DP / 128 : 1;
  static constexpr int CS = DP / NSUB / 16;           // channels of a lane's V load: 8, or 4 (DP 64)
  static constexpr int KW = FP8 ? DP / 64 : DP / 32;  // 16-byte words of a lane's K row part
  static constexpr int VW = FP8 ? CS / 4 : CS / 2;    // words of a lane's V load
  static constexpr bool PW = FP8 || T::kWide;         // the second product in bf16
  static constexpr int ROW = DP + 4;                  // floats of a row in LDS
  static constexpr int kAhead = PAGED ? 64 / NT : 1;  // steps whose places one lookup holds
  static constexpr int E = FP8 ? 1 : 2;               // bytes of an element

  u4 k[NT][KW];
  uint32_t v[NT][4][NSUB][VW];
  f4 ks[NT], vs[NT];  // PAGED: scales of tokens 4g .. 4g + 3
  float ks1, vs1;     // else: of the lane's own token

  f4 acc[MT][NSUB * CS];
  float top[MT], sum[MT];
  u4 q[MT][NK];

  // Channels of MFMA j of the first product in lane group g: 8 from
  static __device__ __forceinline__ int k_at(int j, int g) {
    return FP8 ? 64 * (j >> 1) + 16 * g + 8 * (j & 1) : 32 * j + 8 * g;
  }
};

// ------------------------------------------------------------------ places
//
// Where tiles (PAGED: 64 / NT steps of the wave, a tile a lane) or a step's tokens (else: a token a lane) lie, each
// lane looking up its own: byte offsets in the caches, element offsets in the scales, and one bit whether there is
// such a page.
struct Places {
  uint64_t k, v, ks, vs;
  uint64_t there;
};

// First token of the lane's tile, or its token, in the lookup that begins with `step`.
template <typename A, bool PAGED>
__device__ __forceinline__ uint32_t own_key(uint32_t step, int lane) {
  if (!PAGED) return step * A::KS + (uint32_t)lane;
  return ((step + 4u * (uint32_t)(lane / A::NT)) * A::NT + (uint32_t)(lane % A::NT)) * 16u;
}

// Its entry in the table, of tokens below `limit`. Where that is the table's own end, the lookup does not depend on
// the sequence's length, and both are on their way at once.
template <typename A, bool PAGED>
__device__ __forceinline__ int look_up(const AttnArgs& a, const int32_t* table, uint32_t step, uint32_t limit,
                                       int lane) {
  const uint32_t key = own_key<A, PAGED>(step, lane);
  return key < limit ? table[div_page(key, a.page)] : -1;
}

template <typename A, bool PAGED, bool FP8>
__device__ __forceinline__ Places places_of(const AttnArgs& a, int entry, uint32_t step, int end, int lane) {
  const uint32_t key = own_key<A, PAGED>(step, lane);
  const bool ok = key < (uint32_t)end && (uint64_t)(uint32_t)entry < (uint64_t)a.pages && (PAGED || lane < A::KS);
  const uint64_t page = ok ? (uint32_t)entry : 0u;
  const uint32_t off = ok ? key - div_page(key, a.page) * a.page.page : 0u;
  Places p{};
  p.there = __builtin_amdgcn_ballot_w64(ok);
  p.k = page * (uint64_t)a.k_page + (uint64_t)off * a.k_token;
  p.v = page * (uint64_t)a.v_page + (uint64_t)off * a.v_token;
  if (FP8) {
    p.ks = page * (uint64_t)a.ks_page + (uint64_t)off * a.ks_token;
    p.vs = page * (uint64_t)a.vs_page + (uint64_t)off * a.vs_token;
  }
  return p;
}

__device__ __forceinline__ uint64_t of_lane(uint64_t v, int lane) {
  const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)v, lane);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(v >> 32), lane);
  return lo | (uint64_t)hi << 32;
}
__device__ __forceinline__ uint64_t from_lane(uint64_t v, int lane) {
  const uint32_t lo = (uint32_t)__builtin_amdgcn_ds_bpermute(lane * 4, (int)(uint32_t)v);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_ds_bpermute(lane * 4, (int)(uint32_t)(v >> 32));
  return lo | (uint64_t)hi << 32;
}

__device__ __forceinline__ uint32_t from_lane32(uint32_t v, int lane) {
  return (uint32_t)__builtin_amdgcn_ds_bpermute(lane * 4, (int)v);
}

// The step's bits of `there`: one a tile (PAGED) or a token.
template <typename A, bool PAGED>
__device__ __forceinline__ uint64_t step_bits(const Places& p, int slot) {
  return PAGED ? (p.there >> (slot * A::NT)) & ((1u << A::NT) - 1u) : p.there;
}

// ------------------------------------------------------------------ loads

template <bool STREAM, typename V>
__device__ __forceinline__ V load_as(const uint8_t* p) {
  return STREAM ? __builtin_nontemporal_load(reinterpret_cast<const V*>(p)) : *reinterpret_cast<const V*>(p);
}

template <bool STREAM, typename T, bool FP8, int DP, int MT, bool PAGED, bool FULL>
__device__ __forceinline__ void load_k(const AttnArgs& a, Attn<T, FP8, DP, MT, PAGED, FULL>& s, const uint8_t* kh,
                                       const float* ksh, const Places& at, int slot, int lane) {
  using A = Attn<T, FP8, DP, MT, PAGED, FULL>;
  const int c = lane & 15, g = lane >> 4;
  if (FP8 && !PAGED) s.ks1 = ksh[at.ks];
#pragma unroll
  for (int i = 0; i < A::NT; ++i) {
    const uint8_t* base;
    if (PAGED) {
      base = kh + of_lane(at.k, slot * A::NT + i) + (uint32_t)c * a.k_token;
      if (FP8) s.ks[i] = *reinterpret_cast<const f4*>(ksh + of_lane(at.ks, slot * A::NT + i) + 4 * g);
    } else {
      base = kh + from_lane(at.k, 16 * i + c);
    }
#pragma unroll
    for (int w = 0; w < A::KW; ++w) {
      const int d0 = FP8 ? 64 * w + 16 * g : 32 * w + 8 * g;
      if (FULL) {
        s.k[i][w] = load_as<STREAM, u4>(base + d0 * A::E);
      } else if (FP8) {  // rows of 8-byte alignment; channels past d from the row's start, cleared in scores()
        const u2 lo = load_as<STREAM, u2>(base + (d0 < a.d ? d0 : 0));
        const u2 hi = load_as<STREAM, u2>(base + (d0 + 8 < a.d ? d0 + 8 : 0));
        s.k[i][w] = u4{lo[0], lo[1], hi[0], hi[1]};
      } else {
        s.k[i][w] = load_as<STREAM, u4>(base + (d0 < a.d ? d0 : 0) * A::E);
      }
    }
  }
}

template <bool STREAM, typename T, bool FP8, int DP, int MT, bool PAGED, bool FULL>
__device__ __forceinline__ void load_v(const AttnArgs& a, Attn<T, FP8, DP, MT, PAGED, FULL>& s, const uint8_t* vh,
                                       const float* vsh, const Places& at, int slot, int lane) {
  using A = Attn<T, FP8, DP, MT, PAGED, FULL>;
  const int c = lane & 15, g = lane >> 4;
  if (FP8 && !PAGED) s.vs1 = vsh[at.vs];
#pragma unroll
  for (int i = 0; i < A::NT; ++i) {
    const uint8_t* tile = nullptr;
    if (PAGED) {
      tile = vh + of_lane(at.v, slot * A::NT + i);
      if (FP8) s.vs[i] = *reinterpret_cast<const f4*>(vsh + of_lane(at.vs, slot * A::NT + i) + 4 * g);
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const uint8_t* const base =
          PAGED ? tile + (uint32_t)(4 * g + r) * a.v_token : vh + from_lane(at.v, 16 * i + 4 * g + r);
#pragma unroll
      for (int n = 0; n < A::NSUB; ++n) {
        const int d0 = 128 * n + A::CS * c;
        const uint8_t* const p = base + (FULL || d0 < a.d ? d0 : 0) * A::E;
        if (A::VW == 4) {
          const u4 w = load_as<STREAM, u4>(p);
#pragma unroll
          for (int x = 0; x < A::VW; ++x) s.v[i][r][n][x] = w[x & 3];
        } else if (A::VW == 2) {
          const u2 w = load_as<STREAM, u2>(p);
#pragma unroll
          for (int x = 0; x < A::VW; ++x) s.v[i][r][n][x] = w[x & 1];
        } else {
          s.v[i][r][n][0] = load_as<STREAM, uint32_t>(p);
        }
      }
    }
  }
}

// ------------------------------------------------------------------ one step

// The maximum of a part whose tokens all score -infinity: 0 / 0 in the end, NaN, if the others' do too, where a maximum
// of -infinity says that no token takes part, and gives zeros.
constexpr float kLeast = -3.402823466e38f;

// Whether token 4g + r of tile i of the step takes part.
template <typename A, bool PAGED>
__device__ __forceinline__ bool takes_part(uint32_t step, int i, int r, int g, int begin, int end, uint64_t bits) {
  const int key = (int)(step * A::KS + 16u * i + 4u * g + r);
  return key >= begin && key < end && ((bits >> (PAGED ? i : 16 * i + 4 * g + r)) & 1u);
}

// Whether all tokens of the step take part (uniform).
template <typename A, bool PAGED>
__device__ __forceinline__ bool all_take_part(uint32_t step, int begin, int end, uint64_t bits) {
  constexpr uint64_t kAll = PAGED || A::KS < 64 ? (uint64_t(1) << (PAGED ? A::NT : A::KS % 64)) - 1 : ~uint64_t(0);
  return (int)(step * A::KS) >= begin && (int)(step * A::KS) + A::KS <= end && bits == kAll;
}

// Scores of the step's tokens, in units of log2, -inf where a token takes no part: x[tile][r] of head c, token
// 4g + r. Returns whether any takes part (uniform).
template <typename T, bool FP8, int DP, int MT, bool PAGED, bool FULL>
__device__ __forceinline__ bool scores(const AttnArgs& a, Attn<T, FP8, DP, MT, PAGED, FULL>& s, uint32_t step, int begin,
                                       int end, uint64_t bits, int lane,
                                       float (&x)[MT][Attn<T, FP8, DP, MT, PAGED, FULL>::NT][4]) {
  using A = Attn<T, FP8, DP, MT, PAGED, FULL>;
  const int g = lane >> 4;
#pragma unroll
  for (int i = 0; i < A::NT; ++i) {
    f4 t[MT];
#pragma unroll
    for (int m = 0; m < MT; ++m) t[m] = f4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int j = 0; j < A::NK; ++j) {
      u4 f;
      if (FP8) {
        const u4 w = s.k[i][j >> 1];
        const uint32_t w0 = j & 1 ? w[2] : w[0], w1 = j & 1 ? w[3] : w[1];
        f = u4{codes2<T::kWide, false>(w0), codes2<T::kWide, true>(w0), codes2<T::kWide, false>(w1),
               codes2<T::kWide, true>(w1)};
      } else {
        f = s.k[i][j];
      }
      if (!FULL && A::k_at(j, g) >= a.d) f = u4{0u, 0u, 0u, 0u};
#pragma unroll
      for (int m = 0; m < MT; ++m) t[m] = mfma16<T::kWide>(f, s.q[m][j], t[m]);
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      float ks = 1.0f;
      if (FP8) ks = PAGED ? s.ks[i][r] : as_f32(from_lane32(as_u32(s.ks1), 16 * i + 4 * g + r));
#pragma unroll
      for (int m = 0; m < MT; ++m) x[m][i][r] = FP8 ? t[m][r] * a.scale_log2 * ks : t[m][r] * a.scale_log2;
    }
  }
  if (all_take_part<A, PAGED>(step, begin, end, bits)) return true;
  bool some = false;
#pragma unroll
  for (int i = 0; i < A::NT; ++i)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const bool in = takes_part<A, PAGED>(step, i, r, g, begin, end, bits);
      some |= in;
#pragma unroll
      for (int m = 0; m < MT; ++m) x[m][i][r] = in ? x[m][i][r] : -__builtin_inff();
    }
  return __builtin_amdgcn_ballot_w64(some) != 0;
}

// Scores -> probabilities: the running maximum, the accumulators' rescaling, the sum.
template <typename T, bool FP8, int DP, int MT, bool PAGED, bool FULL>
__device__ __forceinline__ void softmax(Attn<T, FP8, DP, MT, PAGED, FULL>& s,
                                        float (&x)[MT][Attn<T, FP8, DP, MT, PAGED, FULL>::NT][4]) {
  using A = Attn<T, FP8, DP, MT, PAGED, FULL>;
#pragma unroll
  for (int t = 0; t < MT; ++t) {
    float m = x[t][0][0];
#pragma unroll
    for (int i = 0; i < A::NT; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) m = __builtin_fmaxf(m, x[t][i][r]);
    m = __builtin_fmaxf(s.top[t], max4(m));
    if (__builtin_amdgcn_ballot_w64(m > s.top[t])) {
      // -inf -> anything: nothing is there to rescale
      const float f = s.top[t] == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(s.top[t] - m);
      s.sum[t] *= f;
#pragma unroll
      for (int j = 0; j < A::NSUB * A::CS; ++j)
#pragma unroll
        for (int r = 0; r < 4; ++r) s.acc[t][j][r] *= f;
      s.top[t] = m;
    }
    const float ref = m == -__builtin_inff() ? 0.0f : m;
#pragma unroll
    for (int i = 0; i < A::NT; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        x[t][i][r] = __builtin_amdgcn_exp2f(x[t][i][r] - ref);
        s.sum[t] += x[t][i][r];
      }
  }
}

template <typename T, bool FP8, int DP, int MT, bool PAGED, bool FULL>
__device__ __forceinline__ void accumulate(Attn<T, FP8, DP, MT, PAGED, FULL>& s, uint32_t step, int begin, int end,
                                           uint64_t bits, int lane,
                                           float (&p)[MT][Attn<T, FP8, DP, MT, PAGED, FULL>::NT][4]) {
  using A = Attn<T, FP8, DP, MT, PAGED, FULL>;
  const int g = lane >> 4;
  if (FP8 && !PAGED) {
#pragma unroll
    for (int i = 0; i < A::NT; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) s.vs[i][r] = as_f32(from_lane32(as_u32(s.vs1), 16 * i + 4 * g + r));
  }
  // Values (and scales) of tokens that take no part may be anything: NaN times a probability of zero is NaN.
  if (!all_take_part<A, PAGED>(step, begin, end, bits)) {
#pragma unroll
    for (int i = 0; i < A::NT; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const bool in = takes_part<A, PAGED>(step, i, r, g, begin, end, bits);
        if (FP8) s.vs[i][r] = in ? s.vs[i][r] : 0.0f;
#pragma unroll
        for (int n = 0; n < A::NSUB; ++n)
#pragma unroll
          for (int w = 0; w < A::VW; ++w) s.v[i][r][n][w] = in ? s.v[i][r][n][w] : 0u;
      }
  }
#pragma unroll
  for (int u = 0; u < A::NT; u += 2) {
    u4 hi[MT], lo[MT];
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const int i = u + (x >> 1), r = 2 * (x & 1);
        const float p0 = FP8 ? p[m][i][r] * s.vs[i][r] : p[m][i][r];
        const float p1 = FP8 ? p[m][i][r + 1] * s.vs[i][r + 1] : p[m][i][r + 1];
        uint32_t h, l;
        split2<A::PW>(p0, p1, h, l);
        hi[m][x] = h, lo[m][x] = l;
      }
#pragma unroll
    for (int n = 0; n < A::NSUB; ++n)
#pragma unroll
      for (int w = 0; w < A::VW; ++w) {
        // word w of eight tokens (tile u: r = 0..3, tile u + 1: r = 0..3) turned over to channels
        u4 f[FP8 ? 4 : 2];
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const int i = u + (x >> 1), r = 2 * (x & 1);
          const uint32_t a0 = s.v[i][r][n][w], a1 = s.v[i][r + 1][n][w];
          if (FP8) {
            const uint32_t e = __builtin_amdgcn_perm(a1, a0, 0x05010400u);  // channels 0 and 1 of both tokens
            const uint32_t o = __builtin_amdgcn_perm(a1, a0, 0x07030602u);
            f[0][x] = codes2<true, false>(e), f[1][x] = codes2<true, true>(e);
            f[FP8 ? 2 : 0][x] = codes2<true, false>(o), f[FP8 ? 3 : 1][x] = codes2<true, true>(o);
          } else {
            f[0][x] = __builtin_amdgcn_perm(a1, a0, 0x05040100u);
            f[1][x] = __builtin_amdgcn_perm(a1, a0, 0x07060302u);
          }
        }
#pragma unroll
        for (int y = 0; y < (FP8 ? 4 : 2); ++y)
#pragma unroll
          for (int m = 0; m < MT; ++m) {
            f4& t = s.acc[m][n * A::CS + (FP8 ? 4 : 2) * w + y];
            t = mfma16<A::PW>(f[y], hi[m], t);
            t = mfma16<A::PW>(f[y], lo[m], t);
          }
      }
  }
}

// ------------------------------------------------------------------ the kernel

template <typename T>
__device__ __forceinline__ void store4(uint16_t* p, const f4& y) {
  *reinterpret_cast<u2*>(p) = u2{round_pair<T>(y[0], y[1]), round_pair<T>(y[2], y[3])};
}

template <int N>
struct template_int {
  static constexpr int value = N;
};

// Inclusive sums over a wave's lanes (all active): inside rows of 16, then each row's last lane into the rows behind.
__device__ __forceinline__ uint32_t wave_scan_u32(uint32_t v) {
  const auto shifted = [](uint32_t x, auto ctrl, auto rows) {
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, decltype(ctrl)::value, decltype(rows)::value, 0xF, false);
  };
  const template_int<0xF> all;
  v += shifted(v, template_int<0x111>{}, all);  // row_shr 1, 2, 4, 8
  v += shifted(v, template_int<0x112>{}, all);
  v += shifted(v, template_int<0x114>{}, all);
  v += shifted(v, template_int<0x118>{}, all);
  v += shifted(v, template_int<0x142>{}, template_int<0xA>{});  // row_bcast 15 into rows 1 and 3
  v += shifted(v, template_int<0x143>{}, template_int<0xC>{});  // row_bcast 31 into rows 2 and 3
  return v;
}

__device__ __forceinline__ uint32_t wave_total_u32(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_readlane((int)wave_scan_u32(v), 63);
}

__device__ __forceinline__ uint32_t scalar(uint32_t v) {
  return (uint32_t)__builtin_amdgcn_readfirstlane((int)v);
}

// (share a constant wherever this is inlined)
__device__ __forceinline__ uint32_t parts_of(uint32_t count, uint32_t share) { return (count + share - 1) / share; }

// An item's part of a workgroup: steps [at, stop) of sequence b's item `item`.
struct Item {
  int b, begin, end, head, row;  // row: first of its query heads in the group
  uint32_t item, first, count, at, stop;
};

// The item's steps that `left` allow, from its step `at`.
template <int MT, typename S>
__device__ __forceinline__ Item item_of(const AttnArgs& a, const S& span, int b, uint32_t item, uint32_t at,
                                        uint32_t left) {
  const uint32_t stop = span.count - at < left ? span.count : at + left;
  const int head = (int)(item / (uint32_t)a.row_groups), row = 16 * MT * (int)(item - (uint32_t)head * a.row_groups);
  return Item{b, span.begin, span.end, head, row, item, span.first, span.count, at, stop};
}

// How the line of all items' steps is cut: into parts of `share`, none across two items (`apart`, the line's items
// rounded up to whole parts) if the grid is enough for parts of s0, s1 or s2, else into as many equal ones as the grid.
struct Cut {
  uint32_t total, share;
  bool apart;
};

template <typename S>
__device__ __forceinline__ Cut cut_line(const AttnArgs& a, uint32_t count, int lane, uint32_t per, uint32_t s0,
                                        uint32_t s1, uint32_t s2) {
  uint32_t n = count, p0 = parts_of(n, s0), p1 = parts_of(n, s1), p2 = parts_of(n, s2);
  for (int i = lane + 64; i < a.m; i += 64) {
    const uint32_t more = S(a, i).count;
    n += more, p0 += parts_of(more, s0), p1 += parts_of(more, s1), p2 += parts_of(more, s2);
  }
  const uint32_t n0 = wave_total_u32(p0) * per, n1 = wave_total_u32(p1) * per, n2 = wave_total_u32(p2) * per;
  if (n0 <= gridDim.x) return Cut{n0 * s0, s0, true};
  if (n1 <= gridDim.x) return Cut{n1 * s1, s1, true};
  if (n2 <= gridDim.x) return Cut{n2 * s2, s2, true};
  const uint32_t total = wave_total_u32(n) * per;
  return Cut{total, (total + gridDim.x - 1) / gridDim.x, false};
}

// A workgroup's items from `it` on, `left` steps behind it.
template <typename A, bool STREAM, typename T, bool FP8, int DP, int MT, bool PAGED, bool FULL>
__device__ __forceinline__ void run_items(const AttnArgs& a, Item it, uint32_t left, uint32_t share,
                                          float (&rows)[2][A::kWaves][16][A::ROW],
                                          float2 (&ends)[2][A::kWaves][16]) {
  using S = Span<A::KS>;
  int half = 0;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int c = lane & 15, g = lane >> 4;
  const uint32_t per = (uint32_t)(a.heads * a.row_groups);  // items of a sequence
  Attn<T, FP8, DP, MT, PAGED, FULL> s;
  const auto rows_of = [&](const Item& i) { return a.group - i.row < 16 * MT ? a.group - i.row : 16 * MT; };
  const auto table_of = [&](const Item& i) { return a.table + (int64_t)i.b * a.table_row; };
  // Entries behind the workgroup's part are not fetched where its end is known: 64 of them are 32 lines of memory.
  const auto limit_of = [&](const Item& i) {
    const uint32_t end = (i.first + i.stop) * A::KS;
    return a.direct || end > (uint32_t)a.cap ? (uint32_t)a.cap : end;
  };
  const auto load_q = [&](const Item& i) {  // rows past the group's end repeat its first and are not written
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      const int row = i.row + (16 * m + c < rows_of(i) ? 16 * m + c : 0);
      const uint16_t* const qp = a.q + (int64_t)i.b * a.q_row + (int64_t)(i.head * a.group + row) * a.q_head;
#pragma unroll
      for (int j = 0; j < A::NK; ++j) {
        const int d0 = A::k_at(j, g);
        s.q[m][j] = *reinterpret_cast<const u4*>(qp + (FULL || d0 < a.d ? d0 : 0));
      }
    }
  };
  const auto get_k = [&](const Item& i, const Places& at, int slot) {
    load_k<STREAM>(a, s, a.k + i.head * a.k_head, FP8 ? a.ks + i.head * a.ks_head : nullptr, at, slot, lane);
  };
  const auto get_v = [&](const Item& i, const Places& at, int slot) {
    load_v<STREAM>(a, s, a.v + i.head * a.v_head, FP8 ? a.vs + i.head * a.vs_head : nullptr, at, slot, lane);
  };

  // The first step's loads; then each item's, while the item before it ends.
  uint32_t step = (a.window ? it.first : 0u) + it.at + (uint32_t)wave;
  int entry = look_up<A, PAGED>(a, table_of(it), step, limit_of(it), lane), slot = 0;
  load_q(it);
  bool has = step < it.first + it.stop;  // whether the wave has a step of the item
  Places at = places_of<A, PAGED, FP8>(a, entry, step, it.end, lane);
  if (has) {
    get_k(it, at, slot);
    get_v(it, at, slot);
  }
  for (;;) {
    // The item behind this one, and its first entry of the table.
    bool more = left != 0;
    Item next = it;
    if (more) {
      uint32_t item = it.item + 1;
      int b = it.b;
      S span{it.begin, it.end, it.first, it.count};
      if (item == per) {
        item = 0;
        do
          if (++b < a.m) span = S(a, b);
        while (b < a.m && span.count == 0);
      }
      more = b < a.m;  // (always, but where lengths change under the call)
      next = more ? item_of<MT>(a, span, b, item, 0, left) : it;
      left -= more ? next.stop : 0;
    }
    const uint32_t next_step = next.first + next.at + (uint32_t)wave;
    const bool next_has = more && next_step < next.first + next.stop;
    int next_entry = -1;
    if (next_has) next_entry = look_up<A, PAGED>(a, table_of(next), next_step, limit_of(next), lane);

#pragma unroll
    for (int m = 0; m < MT; ++m) {
      s.top[m] = -__builtin_inff(), s.sum[m] = 0.0f;
#pragma unroll
      for (int j = 0; j < A::NSUB * A::CS; ++j) s.acc[m][j] = f4{0.0f, 0.0f, 0.0f, 0.0f};
    }
    const uint32_t last = it.first + it.stop;
    bool any = false;  // whether a token of the wave's steps takes part
    if (has) {
      float x[MT][A::NT][4];
      if (!FULL) {
#pragma unroll
        for (int j = 0; j < A::NK; ++j)
          if (A::k_at(j, g) >= a.d) {
#pragma unroll
            for (int m = 0; m < MT; ++m) s.q[m][j] = u4{0u, 0u, 0u, 0u};
          }
      }
      if (step + 4 * A::kAhead < last) entry = look_up<A, PAGED>(a, table_of(it), step + 4 * A::kAhead, limit_of(it), lane);
      for (; step + 4 < last; step += 4) {
        const uint64_t bits = step_bits<A, PAGED>(at, slot);
        any |= scores(a, s, step, it.begin, it.end, bits, lane, x);
        if (++slot == A::kAhead) {
          slot = 0;
          at = places_of<A, PAGED, FP8>(a, entry, step + 4, it.end, lane);
          entry = look_up<A, PAGED>(a, table_of(it), step + 4 + 4 * A::kAhead, limit_of(it), lane);
        }
        get_k(it, at, slot);
        softmax(s, x);
        accumulate(s, step, it.begin, it.end, bits, lane, x);
        get_v(it, at, slot);
      }
      const uint64_t bits = step_bits<A, PAGED>(at, slot);
      any |= scores(a, s, step, it.begin, it.end, bits, lane, x);
      softmax(s, x);
      accumulate(s, step, it.begin, it.end, bits, lane, x);
    }
    if (next_has) {
      slot = 0;
      at = places_of<A, PAGED, FP8>(a, next_entry, next_step, next.end, lane);
      load_q(next);
      get_k(next, at, slot);
      get_v(next, at, slot);
    }

    // The waves' parts of 16 heads side by side in one half of the LDS; the next 16's go to the other, so that one
    // barrier each is enough: past it, every wave has read what it needs of the half before.
    const bool starts = it.at == 0, whole = starts && it.stop == it.count;
    float* const piece = whole ? nullptr : a.part + piece_of((int)blockIdx.x, starts) * piece_floats(a.part_rows, DP);
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      const int nrows = rows_of(it) - 16 * m < 16 ? rows_of(it) - 16 * m : 16;  // none of the last 16, maybe
      const float own = sum4(s.sum[m]) * (A::PW ? 1.0f : kUp);  // as the products are
      if (c < nrows) {
        if (g == 0) ends[half][wave][c] = float2{any ? __builtin_fmaxf(s.top[m], kLeast) : s.top[m], own};
#pragma unroll
        for (int n = 0; n < A::NSUB; ++n)
#pragma unroll
          for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int j = 0; j < A::CS; j += 4) {
              f4 y;
#pragma unroll
              for (int x = 0; x < 4; ++x) y[x] = s.acc[m][n * A::CS + j + x][r];
              *reinterpret_cast<f4*>(&rows[half][wave][c][128 * n + (4 * g + r) * A::CS + j]) = y;
            }
      }
      __syncthreads();
      for (int e = tid; e < nrows * (DP / 4); e += 256) {
        const int row = e / (DP / 4), d0 = (e - row * (DP / 4)) * 4;
        float2 tl[A::kWaves];
        f4 part[A::kWaves];
#pragma unroll
        for (int w = 0; w < A::kWaves; ++w) {
          tl[w] = ends[half][w][row];
          part[w] = *reinterpret_cast<const f4*>(&rows[half][w][row][d0]);
        }
        const float t = __builtin_fmaxf(__builtin_fmaxf(tl[0].x, tl[1].x), __builtin_fmaxf(tl[2].x, tl[3].x));
        float l = 0.0f;
        f4 y = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int w = 0; w < A::kWaves; ++w) {
          const float f = tl[w].x == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(tl[w].x - t);
          l += tl[w].y * f;
          y += part[w] * f;
        }
        if (whole) {
          const float inv = t == -__builtin_inff() ? 0.0f : 1.0f / l;
          if (FULL || d0 < a.d)
            store4<T>(a.out + (((int64_t)it.b * a.heads + it.head) * a.group + it.row + 16 * m + row) * a.d + d0,
                      y * inv);
        } else {
          *reinterpret_cast<f4*>(piece + (16 * m + row) * DP + d0) = y;
          if (d0 == 0) *reinterpret_cast<float2*>(piece + a.part_rows * DP + 2 * (16 * m + row)) = float2{t, l};
        }
      }
      half ^= 1;
    }
    if (starts && tid == 0 && !a.direct) {
      // an item's last workgroup: `rest` steps of it lie behind this workgroup's
      const uint32_t rest = it.count - it.stop;
      a.ends[(int64_t)it.b * per + it.item] = int2{(int)blockIdx.x, (int)(blockIdx.x + (rest + share - 1) / share)};
    }
    if (!more) return;
    it = next, step = next_step, has = next_has;
  }
}

// STREAM: the call may be one for nontemporal loads. (Of two loops where one is run, the other's code costs the small
// calls some 0.3 us.)
template <bool STREAM, typename T, bool FP8, int DP, int MT, bool PAGED, bool FULL>
__global__ __launch_bounds__(256, attention_resident(DP)) void attention_kernel(AttnArgs a) {
  using A = Attn<T, FP8, DP, MT, PAGED, FULL>;
  using S = Span<A::KS>;
  __shared__ float rows[2][A::kWaves][16][A::ROW];
  __shared__ float2 ends[2][A::kWaves][16];  // (maximum, sum)
  const int lane = threadIdx.x & 63;
  const uint32_t per = (uint32_t)(a.heads * a.row_groups);  // items of a sequence

  Item it;
  bool stream = STREAM;
  uint32_t left = ~0u, share = 0;  // steps of this workgroup behind the item, and of every workgroup
  if (a.direct) {
    const int b = (int)(blockIdx.x / per);
    it = item_of<MT>(a, S(a, b), b, blockIdx.x - (uint32_t)b * per, 0, ~0u);
    left = 0;
  } else {
    // Every wave for itself, a sequence a lane: the line's length, then the sequence that holds the workgroup's first
    // step. Parts of one item where the grid allows it: the end of an item costs a workgroup some us.
    S own(a, lane < a.m ? lane : a.m - 1);
    if (lane >= a.m) own.count = 0;
    Cut line = cut_line<S>(a, own.count, lane, per, 4, 8, 12);
    if (!line.apart && line.share <= 32) line = cut_line<S>(a, own.count, lane, per, 16, 24, 32);
    const bool apart = line.apart;
    const uint32_t total = line.total;
    share = line.share;
    stream = STREAM && (uint64_t)total * (A::KS * 2 * DP * A::E) >= (uint64_t)kStreamLine * (uint32_t)a.row_groups;
    const auto room = [&](uint32_t count) { return apart ? (count + share - 1) / share * share : count; };
    const uint64_t start = (uint64_t)blockIdx.x * share;
    if (start >= total) return;
    left = total - (uint32_t)start < share ? total - (uint32_t)start : share;
    const uint32_t want = (uint32_t)start / per;
    uint32_t before = 0;
    for (int i0 = 0;; i0 += 64) {
      if (i0 >= a.m) return;  // (only where lengths change under the call)
      if (i0) {
        own = S(a, i0 + lane < a.m ? i0 + lane : a.m - 1);
        if (i0 + lane >= a.m) own.count = 0;
      }
      const uint32_t incl = before + wave_scan_u32(room(own.count));
      const int at = (int)__builtin_popcountll(__builtin_amdgcn_ballot_w64(incl <= want));
      if (at < 64) {
        const auto of = [&](uint32_t v) { return (uint32_t)__builtin_amdgcn_readlane((int)v, at); };
        own.begin = (int)of((uint32_t)own.begin), own.end = (int)of((uint32_t)own.end);
        own.first = of(own.first), own.count = of(own.count);
        const uint32_t size = room(own.count), rest = (uint32_t)start - (of(incl) - size) * per, item = rest / size;
        it = item_of<MT>(a, own, i0 + at, item, rest - item * size, left);
        break;
      }
      before = (uint32_t)__builtin_amdgcn_readlane((int)incl, 63);
    }
    left = apart ? 0 : left - (it.stop - it.at);
  }
  it = Item{(int)scalar(it.b), (int)scalar(it.begin), (int)scalar(it.end), (int)scalar(it.head), (int)scalar(it.row),
            scalar(it.item), scalar(it.first), scalar(it.count), scalar(it.at), scalar(it.stop)};
  left = scalar(left), share = scalar(share);

  if (STREAM && stream)
    run_items<A, true, T, FP8, DP, MT, PAGED, FULL>(a, it, left, share, rows, ends);
  else
    run_items<A, false, T, FP8, DP, MT, PAGED, FULL>(a, it, left, share, rows, ends);
}

struct AttnKind {
  bool bf16, fp8, paged, full, stream;
};

template <typename T, bool FP8, int DP, int MT>
int launch_attention_as(const AttnArgs& a, const AttnKind& k, unsigned grid, hipStream_t stream) {
  if (k.paged && k.full && k.stream)
    attention_kernel<true, T, FP8, DP, MT, true, true><<<grid, 256, 0, stream>>>(a);
  else if (k.paged && k.full)
    attention_kernel<false, T, FP8, DP, MT, true, true><<<grid, 256, 0, stream>>>(a);
  else if (k.paged)
    attention_kernel<false, T, FP8, DP, MT, true, false><<<grid, 256, 0, stream>>>(a);
  else
    attention_kernel<false, T, FP8, DP, MT, false, false><<<grid, 256, 0, stream>>>(a);
  return check_launch("tf_paged_attention");
}

template <int DP, int MT>
int launch_attention(const AttnArgs& a, const AttnKind& k, unsigned grid, hipStream_t stream) {
  if (k.bf16)
    return k.fp8 ? launch_attention_as<BF16, true, DP, MT>(a, k, grid, stream)
                 : launch_attention_as<BF16, false, DP, MT>(a, k, grid, stream);
  return k.fp8 ? launch_attention_as<F16, true, DP, MT>(a, k, grid, stream)
               : launch_attention_as<F16, false, DP, MT>(a, k, grid, stream);
}

// By head length and 16s of query heads, each head length in a file of its own.
int launch_attention_d64(const AttnArgs& a, const AttnKind& k, int tiles, unsigned grid, hipStream_t stream);
int launch_attention_d128(const AttnArgs& a, const AttnKind& k, int tiles, unsigned grid, hipStream_t stream);
int launch_attention_d256(const AttnArgs& a, const AttnKind& k, unsigned grid, hipStream_t stream);

}  // namespace tf
