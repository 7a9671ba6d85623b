// C entry of the paged attention: checks, the choice of the compiled kernel, and the join of items that several
// workgroups share.
#include "paged_attention.h"

namespace tf {
namespace {

struct JoinArgs {
  const float* part;
  const int2* ends;
  const int32_t* lens;
  uint16_t* out;
  int heads, group, row_groups, part_rows, d, dp, tiles;
  uint32_t count;  // sequences * query heads
  int grid;        // workgroups of the attention
};

// Part of a row: its channels y of a lane, in units of 2^top, and the sum l of the probabilities.
struct Part {
  float top, l;
  f4 y;
};

__device__ __forceinline__ void merge(Part& a, float top, float l, const f4& y) {
  const float t = __builtin_fmaxf(a.top, top);
  const float fa = a.top == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(a.top - t);
  const float fb = top == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(top - t);
  a.l = a.l * fa + l * fb;
  a.y = a.y * fa + y * fb;
  a.top = t;
}

// out = sum_p acc_p 2^(top_p - top) / sum_p sum_p 2^(top_p - top) of a sequence's query head over the pieces p that
// the attention's workgroups left, by one wave (WAVES 1) or a workgroup of 4 or 8. dp / 4 lanes take a piece; a wave takes
// 64 / (dp / 4) side by side, four of each at once, and the parts are merged in an order that depends on the number
// of pieces alone. Items that one workgroup held are done already; sequences without tokens get zeros here.
template <typename T, int WAVES>
__global__ __launch_bounds__(WAVES == 1 ? 256 : 64 * WAVES) void join_kernel(JoinArgs a) {
  __shared__ Part parts[WAVES][64];
  constexpr int kOnce = 4;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const uint32_t q_heads = (uint32_t)(a.heads * a.group);
  const uint32_t at = WAVES == 1 ? blockIdx.x * 4 + (uint32_t)wave : blockIdx.x;
  if (at >= a.count) return;
  const int b = (int)(at / q_heads), qh = (int)(at - (uint32_t)b * q_heads);
  const int head = qh / a.group, in = qh - head * a.group, rg = in / (16 * a.tiles), row = in - rg * 16 * a.tiles;
  const int n = a.lens[b];
  const int2 found = a.ends[((int64_t)b * a.heads + head) * a.row_groups + rg];
  // (within the pieces, also where lengths change under the call and an item was left out)
  const int2 ends{found.x > 0 ? found.x : 0, found.y < a.grid ? found.y : a.grid - 1};
  const int lanes = a.dp >> 2, side = 64 / lanes, part = lane / lanes, e = (lane & (lanes - 1)) * 4;
  uint16_t* const out = a.out + (int64_t)at * a.d;
  const bool writes = (WAVES == 1 || wave == 0) && part == 0 && e < a.d;
  if (n <= 0) {
    if (writes) *reinterpret_cast<u2*>(out + e) = u2{0u, 0u};
    return;
  }
  if (ends.x >= ends.y) return;
  const int64_t size = piece_floats(a.part_rows, a.dp);
  Part mine{-__builtin_inff(), 0.0f, f4{0.0f, 0.0f, 0.0f, 0.0f}};
  const int each = WAVES * side;
  for (int p0 = ends.x + (WAVES == 1 ? 0 : wave) * side + part; p0 <= ends.y; p0 += each * kOnce) {
    float2 tl[kOnce];
    f4 y[kOnce];
#pragma unroll
    for (int i = 0; i < kOnce; ++i) {
      const int p = p0 + i * each <= ends.y ? p0 + i * each : p0;
      const float* const piece = a.part + piece_of(p, p == ends.x) * size;
      tl[i] = *reinterpret_cast<const float2*>(piece + a.part_rows * a.dp + 2 * row);
      y[i] = *reinterpret_cast<const f4*>(piece + row * a.dp + e);
    }
#pragma unroll
    for (int i = 0; i < kOnce; ++i)
      if (p0 + i * each <= ends.y) merge(mine, tl[i].x, tl[i].y, y[i]);
  }
  for (int o = lanes; o < 64; o <<= 1) {
    const float t = __shfl_xor(mine.top, o), l = __shfl_xor(mine.l, o);
    f4 y;
#pragma unroll
    for (int j = 0; j < 4; ++j) y[j] = __shfl_xor(mine.y[j], o);
    merge(mine, t, l, y);
  }
  if (WAVES > 1) {
    parts[wave % WAVES][lane] = mine;
    __syncthreads();
    if (wave != 0) return;
#pragma unroll
    for (int w = 1; w < WAVES; ++w) merge(mine, parts[w][lane].top, parts[w][lane].l, parts[w][lane].y);
  }
  if (writes) store4<T>(out + e, mine.y * (mine.top == -__builtin_inff() ? 0.0f : 1.0f / mine.l));
}

// Rows from which a wave each fills the CUs in the join; below, few items get 8 waves a row where the table has room for
// long ones (the host knows no lengths): of 8 items that fill the line one has 64 pieces, past heads of 128 32 (MI355X,
// one sequence of 32749 tokens in e4m3: 16.6 us with 8 waves, 17.9 with 4 and 16.7 with 16, which cost one of
// 4096 0.5 and 1.3 us).
constexpr uint32_t kJoinByWave = 1024;
constexpr int64_t kFewItems = 8, kLongItems = 8192;

// Bytes of an item up to which a workgroup takes it whole, by what the table's row holds, and the same from kManyItems
// items on. MI355X, heads of 128 in e4m3, us whole and on the line; lengths that fill the row, then lengths spread over
// the logarithm from a twentieth of it:
//   items     256 KB                     384 KB                     512 KB                     1 MB
//     400   24.3  28.0   13.6  18.1   35.7  38.4   17.4  21.4   45.6  46.8   21.5  27.4    84.3  82.2   47.8  39.4
//     512   28.0  29.9   14.1  19.5   40.0  40.2   18.3  28.3   51.8  51.0   24.2  33.5    91.3  94.6   49.8  47.1
//     520   35.3  36.0   14.8  28.4   50.3  47.6   18.4  28.7   65.3  59.0   24.6  35.2   120.1 103.9   49.8  47.9
//     768   40.9  46.0   22.7  32.8   63.5  70.8   31.7  39.1   70.0  80.0   44.6  46.4   134.7 144.5   78.0  63.9
//    1024   53.0  66.4   27.0  40.3   73.4  87.6   38.9  46.8   92.9 110.4   48.4  56.2   177.7 238.8   91.5  82.6
// In bf16 512 items of 512 KB take 48.2, 47.5, 20.4 and 28.5, of 1 MB 88.8, 92.1, 44.7 and 42.6; 4 items of 256 KB 10.7 and
// 8.1 in e4m3, 8.0 and 8.1 in bf16. So whole items gain up to the limits, but for a few items in e4m3 and just past a round of
// the grid's places (520 equal ones); from 400 items on they would gain past 256 KB as well.
constexpr int64_t kDirect = 256 << 10, kDirectMany = 512 << 10, kManyItems = 512;

bool multiple(const void* p, uintptr_t a) { return (reinterpret_cast<uintptr_t>(p) % a) == 0; }

// Sizes of a call, and "" or what is wrong with them.
struct Plan {
  int dp, group, tiles, row_groups, part_rows;
  int64_t items, cap, part_floats, bytes;
  uint32_t grid;
  bool fp8, direct, stream;
};

std::string plan_of(const tf_kv_cache& c, int64_t m, int32_t q_heads, int64_t width, int64_t window, Plan& p) {
  if (m < 0 || width < 0 || m > 0x7FFFFFFF) return "bad size";
  if (window < 0) return "need window >= 0";
  if (q_heads <= 0 || q_heads > 0xFFFF || q_heads % c.heads) return "q_heads must be a multiple of the cache's heads";
  p.fp8 = c.dtype == TF_DTYPE_E4M3;
  p.dp = c.head_dim <= 64 ? 64 : c.head_dim <= 128 ? 128 : 256;
  p.group = q_heads / c.heads;
  // Past 16 query heads a key-value head, 32 share its loads; past heads of 128 the registers hold no second tile. With
  // whole tiles of exact lengths they hold both, and 161 sequences of up to 4096 with 20 query heads on each of 2 take
  // 54 us against 82 in 16 bits, 44 against 57 in e4m3 (32 sequences: 19.5 against 21.9, 18.1 against 17.7). The forms that
  // look each token up keep 10 to 42 registers a lane in scratch, the 16-bit one of odd lengths 2 or 3: 161 sequences with
  // pages of 24 73.8 against 77.0 in bf16 and 52.6 against 59.3 in e4m3, 32 of them 23.1 against 21.5 and alike.
  p.tiles = p.group > 16 && p.dp <= 128 ? 2 : 1;
  p.row_groups = (int)cdiv(p.group, 16 * p.tiles);
  p.part_rows = p.group < 16 * p.tiles ? p.group : 16 * p.tiles;
  p.items = m * c.heads * p.row_groups;
  if (width > 0x7FFFFF00 / c.page_size) return "block_table covers 2^31 - 256 tokens or more";
  p.cap = width * c.page_size;
  if (m * q_heads > 0x7FFFFF || p.items * cdiv(p.cap, 16) > 0x7FFFFFFF)
    return "more sequences, heads and tokens of block_table than 2^31 steps of 16";
  // An item's steps are at most those of its row of the table. Where they are few, or not many and the items enough
  // to fill the CUs, a workgroup takes a whole item: no second launch, and no search for the workgroup's place. The
  // longest item then sets the time.
  const int step = attention_step(p.dp);
  int64_t most = cdiv(p.cap, step);
  if (window > 0) most = most < cdiv(window, step) + 1 ? most : cdiv(window, step) + 1;
  const int64_t bytes = most * step * 2 * p.dp * (p.fp8 ? 1 : 2);
  p.direct = bytes <= (p.items >= kManyItems ? kDirectMany : kDirect);
  p.stream = m * c.heads * bytes >= (p.direct ? kStreamTable : kStreamLine);
  p.grid = p.direct ? (uint32_t)p.items : (uint32_t)attention_grid(p.dp);
  p.part_floats = p.direct ? 0 : 2 * (int64_t)p.grid * piece_floats(p.part_rows, p.dp);
  p.bytes = p.direct ? 0 : p.part_floats * 4 + p.items * 8;
  return "";
}

}  // namespace
}  // namespace tf

using namespace tf;

extern "C" int64_t tf_paged_attention_workspace_bytes(const tf_kv_cache* cache, int64_t m, int32_t q_heads,
                                                      int64_t width, int32_t window) {
  Plan p;
  if (!cache || !kv_cache_error(cache, cache->dtype == TF_DTYPE_E4M3 ? TF_DTYPE_FP16 : cache->dtype).empty()) return -1;
  if (!plan_of(*cache, m, q_heads, width, window, p).empty()) return -1;
  return p.bytes;
}

extern "C" int tf_paged_attention(const tf_kv_cache* cache, const uint16_t* q, int64_t q_row, int64_t q_head,
                                  int32_t q_heads, int32_t dtype, const int32_t* block_table, int64_t table_stride,
                                  int64_t width, const int32_t* seq_lens, int64_t m, float scale, int32_t window,
                                  uint16_t* out, float* workspace, int64_t workspace_bytes, void* stream) {
  const auto bad = [](const std::string& what) { return fail(TF_EINVAL, "tf_paged_attention: " + what); };
  const std::string e = kv_cache_error(cache, dtype);
  if (!e.empty()) return bad(e);
  const tf_kv_cache& c = *cache;
  if (!q || !out || (!block_table && width) || !seq_lens) return bad("null pointer");
  if (!multiple(q, 16) || q_row % 8 || q_head % 8 || !multiple(out, 16))
    return bad("rows of q and out must be 16-byte aligned");
  if (q_row < 0 || q_head < 0 || table_stride < 0) return bad("negative stride");
  Plan p;
  const std::string wrong = plan_of(c, m, q_heads, width, window, p);
  if (!wrong.empty()) return bad(wrong);
  if (p.bytes > 0 && (!workspace || workspace_bytes < p.bytes))
    return bad("workspace too small (" + std::to_string(workspace_bytes) + " < " + std::to_string(p.bytes) + ")");
  if (p.bytes > 0 && !multiple(workspace, 16)) return bad("workspace not 16-byte aligned");
  if (m == 0) return TF_OK;
  const int size = p.fp8 ? 1 : 2;
  AttnArgs a{};
  a.q = q, a.q_row = q_row, a.q_head = q_head;
  a.k = (const uint8_t*)c.k, a.v = (const uint8_t*)c.v;
  a.k_page = c.k_strides[0] * size, a.k_head = c.k_strides[1] * size, a.k_token = (uint32_t)c.k_strides[2] * size;
  a.v_page = c.v_strides[0] * size, a.v_head = c.v_strides[1] * size, a.v_token = (uint32_t)c.v_strides[2] * size;
  a.ks = c.k_scale, a.vs = c.v_scale;
  a.ks_page = c.k_scale_strides[0], a.ks_head = c.k_scale_strides[1], a.ks_token = (uint32_t)c.k_scale_strides[2];
  a.vs_page = c.v_scale_strides[0], a.vs_head = c.v_scale_strides[1], a.vs_token = (uint32_t)c.v_scale_strides[2];
  a.table = block_table, a.table_row = table_stride, a.lens = seq_lens, a.out = out;
  a.part = workspace, a.ends = reinterpret_cast<int2*>(workspace + p.part_floats);
  a.pages = c.pages, a.page = page_div((uint32_t)c.page_size);
  a.m = (int)m, a.heads = c.heads, a.group = p.group, a.row_groups = p.row_groups, a.part_rows = p.part_rows;
  a.d = c.head_dim, a.cap = (int)p.cap, a.window = window, a.scale_log2 = scale * 1.44269504088896341f;
  a.direct = p.direct;
  bool paged = c.page_size % 16 == 0;
  if (p.fp8) {  // a tile's scales go by 16-byte loads
    paged = paged && multiple(c.k_scale, 16) && multiple(c.v_scale, 16);
    for (const int64_t* st : {c.k_scale_strides, c.v_scale_strides})
      paged = paged && st[0] % 4 == 0 && st[1] % 4 == 0 && st[2] == 1;
  }
  bool full = c.head_dim == p.dp;
  if (p.fp8) {  // whole rows go by 16-byte loads
    full = full && multiple(c.k, 16);
    for (int i = 0; i < 3; ++i) full = full && c.k_strides[i] % 16 == 0;
  }
  const bool bf16 = dtype == TF_DTYPE_BF16;
  const AttnKind kind{bf16, p.fp8, paged, full, p.stream};
  const auto s = (hipStream_t)stream;
  const int rc = p.dp == 64    ? launch_attention_d64(a, kind, p.tiles, p.grid, s)
                 : p.dp == 128 ? launch_attention_d128(a, kind, p.tiles, p.grid, s)
                               : launch_attention_d256(a, kind, p.grid, s);
  if (rc) return rc;
  if (p.direct) return TF_OK;
  const auto count = (uint32_t)(m * q_heads);
  const JoinArgs j{a.part,       a.ends,      seq_lens, out,  c.heads, p.group,
                   p.row_groups, p.part_rows, a.d,      p.dp, p.tiles, count,   (int)p.grid};
  if (count >= kJoinByWave)
    bf16 ? join_kernel<BF16, 1><<<(unsigned)cdiv(count, 4), 256, 0, s>>>(j)
         : join_kernel<F16, 1><<<(unsigned)cdiv(count, 4), 256, 0, s>>>(j);
  else if (p.items <= kFewItems && p.cap >= kLongItems)
    bf16 ? join_kernel<BF16, 8><<<count, 512, 0, s>>>(j) : join_kernel<F16, 8><<<count, 512, 0, s>>>(j);
  else
    bf16 ? join_kernel<BF16, 4><<<count, 256, 0, s>>>(j) : join_kernel<F16, 4><<<count, 256, 0, s>>>(j);
  return check_launch("tf_paged_attention");
}
