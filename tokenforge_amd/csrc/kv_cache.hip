// Writing a paged key-value cache, with or without the rotation of queries and keys in front, and reading it
// back by slots.
//
// A row (one head of one token) lies on 4, 8 or 16 lanes, two chunks of eight elements a lane, so its absmax is 2 to
// 4 lane exchanges and nothing crosses a row. A lane group takes EACH consecutive rows of a token (its keys, its
// values, then the queries): their loads are on their way together, and the token's slot, position and angles are
// read once. In the rotation by halves a lane's two chunks are each other's partners. Every byte is read and written
// once; memory bound from some thousand tokens on, latency below. On MI355X (copy of 1 GiB 5.14 TB/s), heads of 128, us:
// 8191 tokens of 36 rows rotated into bf16 (155 MB) 32.2, 4095 of 8 rows written in e4m3 (13 MB) 5.5, 32767 read from
// e4m3 slots in no order (102 MB, and a line of memory for each of 262136 scales) 21.5; one token 2.8.
#include "kv_cache.h"
#include "overlap.h"

namespace tf {
namespace {

struct KvArgs {
  const uint16_t* src[3];  // k, v, q
  int64_t src_token[3], src_head[3];
  uint8_t* cache[2];
  int64_t page_stride[2], head_stride[2], token_stride[2];  // elements
  float* scale[2];
  int64_t scale_page[2], scale_head[2], scale_token[2];
  uint16_t* out[3];  // read: k, v; rope: [2] = q
  const int64_t* slots;
  const int64_t* positions;
  const float* cos_sin;
  int64_t max_positions;
  int64_t capacity;  // pages * page_size
  int64_t groups;    // lane groups of the launch
  PageDiv page;
  PageDiv per_token;  // lane groups of a token
  int rows;           // of a token: 2 * heads (+ q_heads)
  int heads, q_heads, d, rot;
};

// The largest of v over the row's LANES lanes (4, 8 or 16; all active), in each of them.
template <int LANES>
__device__ __forceinline__ uint32_t row_max_u32(uint32_t v) {
  v = __builtin_elementwise_max(v, dpp_u32<kDppQuadXor1>(v));
  v = __builtin_elementwise_max(v, dpp_u32<kDppQuadXor2>(v));
  if (LANES > 4) v = __builtin_elementwise_max(v, dpp_u32<kDppHalfRowMirror>(v));
  if (LANES > 8) v = __builtin_elementwise_max(v, dpp_u32<kDppRowMirror>(v));
  return v;
}

struct Row {
  int part, head;  // 0 (k), 1 (v) or 2 (q)
};

__device__ __forceinline__ Row row_of(const KvArgs& a, int r) {
  if (r < a.heads) return Row{0, r};
  if (r < 2 * a.heads) return Row{1, r - a.heads};
  return Row{2, r - 2 * a.heads};
}

// Where a slot lies; page < 0 where there is none.
struct Place {
  int64_t page, off;
};

__device__ __forceinline__ Place place_of(const KvArgs& a, int64_t slot) {
  if (slot < 0 || slot >= a.capacity) return Place{-1, 0};
  if (slot < (int64_t(1) << 31)) {
    const uint32_t page = div_page((uint32_t)slot, a.page);
    return Place{page, (uint32_t)slot - page * a.page.page};
  }
  const int64_t page = slot / a.page.page;
  return Place{page, slot - page * a.page.page};
}

enum Rope { kNone = 0, kHalves = 1, kOther = 2, kPairs = 3 };

// Elements of a lane's two chunks. By halves (rot a multiple of 16): partners in the rotated part, neighbours behind.
template <int ROPE, int LANES>
__device__ __forceinline__ void chunks_of(const KvArgs& a, int lane, int (&e)[2]) {
  if (ROPE == kHalves) {
    const int half = a.rot >> 1, turned = half >> 3;
    e[0] = lane < turned ? 8 * lane : a.rot + 16 * (lane - turned);
    e[1] = e[0] + (lane < turned ? half : 8);
  } else {
    e[0] = 8 * lane, e[1] = 8 * (lane + LANES);
  }
}

// The angles of a lane's elements. By halves: both chunks'; in pairs: four of each chunk.
struct Turn {
  f4 c[2], s[2];
};

template <int ROPE>
__device__ __forceinline__ Turn turn_of(const KvArgs& a, const int (&e)[2], int64_t token) {
  Turn t{};
  const int half = a.rot >> 1;
  const int64_t pos = a.positions[token];
  const bool known = pos >= 0 && pos < a.max_positions;
  const float* const cs = a.cos_sin + (known ? pos : 0) * a.rot;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    if (ROPE == kHalves) {
      if (e[0] < half) {
        t.c[i] = *reinterpret_cast<const f4*>(cs + e[0] + 4 * i);
        t.s[i] = *reinterpret_cast<const f4*>(cs + half + e[0] + 4 * i);
      }
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (e[i] + 2 * j < a.rot) t.c[i][j] = cs[e[i] / 2 + j], t.s[i][j] = cs[half + e[i] / 2 + j];
    }
  }
  if (!known) {
#pragma unroll
    for (int j = 0; j < 8; ++j) t.c[j >> 2][j & 3] = __builtin_nanf("");
  }
  return t;
}

// The lane's elements y of the row x, rotated in fp32.
template <typename T, int ROPE>
__device__ __forceinline__ void rotate(const KvArgs& a, const uint16_t* x, const int (&e)[2], const Turn& t,
                                       int64_t token, float (&y)[2][8]) {
  const int half = a.rot >> 1;
  if (ROPE == kHalves) {
    if (e[0] >= half) return;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float c = t.c[j >> 2][j & 3], s = t.s[j >> 2][j & 3], u = y[0][j], w = y[1][j];
      y[0][j] = u * c - w * s;
      y[1][j] = w * c + u * s;
    }
    return;
  }
  if (ROPE == kPairs) {
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (e[i] + 2 * j < a.rot) {
          const float c = t.c[i][j], s = t.s[i][j], u = y[i][2 * j], w = y[i][2 * j + 1];
          y[i][2 * j] = u * c - w * s;
          y[i][2 * j + 1] = w * c + u * s;
        }
    return;
  }
  // Halves that eight does not divide: an element at a time.
  const int64_t pos = a.positions[token];
  const bool known = pos >= 0 && pos < a.max_positions;
  const float* const cs = a.cos_sin + (known ? pos : 0) * a.rot;
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int at = e[i] + j;
      if (at >= a.rot) continue;
      const int k = at < half ? at : at - half;
      const float w = T::lo(x[at < half ? at + half : at - half]), c = cs[k], s = cs[half + k];
      const float r = at < half ? y[i][j] * c - w * s : y[i][j] * c + w * s;
      y[i][j] = known ? r : __builtin_nanf("");
    }
}

template <typename T, bool FP8, int ROPE, int LANES, int EACH>
__global__ __launch_bounds__(256) void kv_write_kernel(KvArgs a) {
  const int64_t group = (int64_t)blockIdx.x * (256 / LANES) + threadIdx.x / LANES;
  const bool live = group < a.groups;
  const uint32_t gi = live ? (uint32_t)group : 0u, token = div_page(gi, a.per_token);
  const int r0 = (int)(gi - token * a.per_token.page) * EACH;
  int e[2];
  chunks_of<ROPE, LANES>(a, threadIdx.x % LANES, e);
  u4 v[EACH][2];
  const uint16_t* x[EACH];
#pragma unroll
  for (int n = 0; n < EACH; ++n) {
    const Row r = row_of(a, r0 + n < a.rows ? r0 + n : a.rows - 1);
    x[n] = a.src[r.part] + (int64_t)token * a.src_token[r.part] + r.head * a.src_head[r.part];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      v[n][i] = u4{0u, 0u, 0u, 0u};
      if (live && r0 + n < a.rows && e[i] < a.d) v[n][i] = *reinterpret_cast<const u4*>(x[n] + e[i]);
    }
  }
  const Place at = place_of(a, a.slots[token]);
  Turn turn{};
  if (ROPE == kHalves || ROPE == kPairs) turn = turn_of<ROPE>(a, e, token);
#pragma unroll
  for (int n = 0; n < EACH; ++n) {
    const bool mine = live && r0 + n < a.rows;
    const Row r = row_of(a, mine ? r0 + n : a.rows - 1);
    float y[2][8];
    unpack8<T>(v[n][0], y[0]);
    unpack8<T>(v[n][1], y[1]);
    if (ROPE != kNone && r.part != 1) {
      rotate<T, ROPE>(a, x[n], e, turn, token, y);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[n][j >> 2][j & 3] = round_pair<T>(y[j >> 2][2 * (j & 3)], y[j >> 2][2 * (j & 3) + 1]);
      if (r.part == 2) {
        uint16_t* const q = a.out[2] + ((int64_t)token * a.q_heads + r.head) * a.d;
#pragma unroll
        for (int i = 0; i < 2; ++i)
          if (mine && e[i] < a.d) *reinterpret_cast<u4*>(q + e[i]) = v[n][i];
      }
    }
    const bool kept = mine && r.part < 2 && at.page >= 0;
    const int p = r.part & 1;
    const int64_t to = at.page * a.page_stride[p] + r.head * a.head_stride[p] + at.off * a.token_stride[p];
    if (ROPE != kNone && r.part == 2) continue;  // (a lane group's rows are of one part, each with all its lanes)
    if (FP8) {
      if (e[0] >= a.d) {
#pragma unroll
        for (int j = 0; j < 8; ++j) y[0][j] = 0.0f;
      }
      if (e[1] >= a.d) {
#pragma unroll
        for (int j = 0; j < 8; ++j) y[1][j] = 0.0f;
      }
      const uint32_t amax = row_max_u32<LANES>(__builtin_elementwise_max(absmax8(y[0]), absmax8(y[1])));
      const float s = dynamic_scale(as_f32(amax));
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const u2 codes = encode8(y[i], s, amax);
        if (kept && e[i] < a.d) *reinterpret_cast<u2*>(a.cache[p] + to + e[i]) = codes;
      }
      if (kept && e[0] == 0)
        a.scale[p][at.page * a.scale_page[p] + r.head * a.scale_head[p] + at.off * a.scale_token[p]] = s;
    } else {
#pragma unroll
      for (int i = 0; i < 2; ++i)
        if (kept && e[i] < a.d) *reinterpret_cast<u4*>(reinterpret_cast<uint16_t*>(a.cache[p]) + to + e[i]) = v[n][i];
    }
  }
}

// code * scale of eight codes, rounded once.
template <typename T>
__device__ __forceinline__ u4 decode8(u2 codes, float s) {
  u4 r;
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)codes[w], false);
    const auto hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)codes[w], true);
    float p[4] = {lo[0] * s, lo[1] * s, hi[0] * s, hi[1] * s};
    // fp32 products first, as the torch expression rounds them (a fused multiply and conversion would not)
#pragma unroll
    for (int j = 0; j < 4; ++j) __asm__ volatile("" : "+v"(p[j]));
    r[2 * w] = round_pair<T>(p[0], p[1]);
    r[2 * w + 1] = round_pair<T>(p[2], p[3]);
  }
  return r;
}

template <typename T, bool FP8, int LANES, int EACH>
__global__ __launch_bounds__(256) void kv_read_kernel(KvArgs a) {
  const int64_t group = (int64_t)blockIdx.x * (256 / LANES) + threadIdx.x / LANES;
  if (group >= a.groups) return;
  const uint32_t token = div_page((uint32_t)group, a.per_token);
  const int r0 = (int)((uint32_t)group - token * a.per_token.page) * EACH;
  int e[2];
  chunks_of<kNone, LANES>(a, threadIdx.x % LANES, e);
  const Place at = place_of(a, a.slots[token]);
  u4 v[EACH][2];
  u2 codes[EACH][2];
  float s[EACH];
#pragma unroll
  for (int n = 0; n < EACH; ++n) {
    const Row r = row_of(a, r0 + n < a.rows ? r0 + n : a.rows - 1);
    const int p = r.part;
    const bool there = at.page >= 0;
    const int64_t from = at.page * a.page_stride[p] + r.head * a.head_stride[p] + at.off * a.token_stride[p];
    s[n] = 0.0f;
    if (FP8 && there)
      s[n] = a.scale[p][at.page * a.scale_page[p] + r.head * a.scale_head[p] + at.off * a.scale_token[p]];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      codes[n][i] = u2{0u, 0u}, v[n][i] = u4{0u, 0u, 0u, 0u};
      if (there && e[i] < a.d) {
        if (FP8)
          codes[n][i] = *reinterpret_cast<const u2*>(a.cache[p] + from + e[i]);
        else
          v[n][i] = *reinterpret_cast<const u4*>(reinterpret_cast<const uint16_t*>(a.cache[p]) + from + e[i]);
      }
    }
  }
#pragma unroll
  for (int n = 0; n < EACH; ++n) {
    if (r0 + n >= a.rows) break;
    const Row r = row_of(a, r0 + n);
    uint16_t* const out = a.out[r.part] + ((int64_t)token * a.heads + r.head) * a.d;
#pragma unroll
    for (int i = 0; i < 2; ++i)
      if (e[i] < a.d) *reinterpret_cast<u4*>(out + e[i]) = FP8 ? decode8<T>(codes[n][i], s[n]) : v[n][i];
  }
}

template <typename T, bool FP8, int ROPE, bool READ, int LANES, int EACH>
void launch_each(KvArgs a, int64_t t, hipStream_t stream) {
  a.per_token = page_div((uint32_t)cdiv(a.rows, EACH));
  a.groups = t * a.per_token.page;
  const unsigned grid = (unsigned)cdiv(a.groups, 256 / LANES);
  if (READ)
    kv_read_kernel<T, FP8, LANES, EACH><<<grid, 256, 0, stream>>>(a);
  else
    kv_write_kernel<T, FP8, ROPE, LANES, EACH><<<grid, 256, 0, stream>>>(a);
}

// Two rows a lane group share the angles once the rows fill the CUs (MI355X, 8191 tokens of 36 rows of 128: 35.9 us
// against 39.1 with one, 39.0 with four); without angles one is faster (32767 tokens read: 26.0 us against 28.9).
template <typename T, bool FP8, int ROPE, bool READ, int LANES>
void launch_lanes(const KvArgs& a, int64_t t, hipStream_t stream) {
  if (ROPE != kNone && t * a.rows >= 16384)
    launch_each<T, FP8, ROPE, READ, LANES, ROPE == kNone ? 1 : 2>(a, t, stream);
  else
    launch_each<T, FP8, ROPE, READ, LANES, 1>(a, t, stream);
}

template <typename T, bool FP8, int ROPE, bool READ>
void launch_row(const KvArgs& a, int64_t t, hipStream_t stream) {
  if (a.d <= 64)
    launch_lanes<T, FP8, ROPE, READ, 4>(a, t, stream);
  else if (a.d <= 128)
    launch_lanes<T, FP8, ROPE, READ, 8>(a, t, stream);
  else
    launch_lanes<T, FP8, ROPE, READ, 16>(a, t, stream);
}

template <int ROPE, bool READ>
void launch_type(const KvArgs& a, int64_t t, bool bf16, bool fp8, hipStream_t stream) {
  if (bf16)
    fp8 ? launch_row<BF16, true, ROPE, READ>(a, t, stream) : launch_row<BF16, false, ROPE, READ>(a, t, stream);
  else
    fp8 ? launch_row<F16, true, ROPE, READ>(a, t, stream) : launch_row<F16, false, ROPE, READ>(a, t, stream);
}

bool multiple(const void* p, uintptr_t a) { return (reinterpret_cast<uintptr_t>(p) % a) == 0; }

KvArgs cache_args(const tf_kv_cache& c) {
  KvArgs a{};
  a.cache[0] = (uint8_t*)c.k, a.cache[1] = (uint8_t*)c.v;
  a.scale[0] = c.k_scale, a.scale[1] = c.v_scale;
  a.page_stride[0] = c.k_strides[0], a.head_stride[0] = c.k_strides[1], a.token_stride[0] = c.k_strides[2];
  a.page_stride[1] = c.v_strides[0], a.head_stride[1] = c.v_strides[1], a.token_stride[1] = c.v_strides[2];
  a.scale_page[0] = c.k_scale_strides[0], a.scale_head[0] = c.k_scale_strides[1];
  a.scale_token[0] = c.k_scale_strides[2];
  a.scale_page[1] = c.v_scale_strides[0], a.scale_head[1] = c.v_scale_strides[1];
  a.scale_token[1] = c.v_scale_strides[2];
  a.capacity = c.pages * c.page_size;
  a.heads = c.heads, a.d = c.head_dim, a.page = page_div((uint32_t)c.page_size);
  a.rows = 2 * c.heads;
  return a;
}

std::string written_error(const tf_kv_cache& c) {
  if (c.k == c.v) return "keys and values are written to one place";
  if (c.dtype == TF_DTYPE_E4M3 && c.k_scale == c.v_scale) return "scales of keys and values are written to one place";
  const bool fp8 = c.dtype == TF_DTYPE_E4M3;
  const int64_t size[3] = {c.pages, c.heads, c.page_size};
  const auto placed = [&](const void* p, const int64_t (&stride)[3], int64_t bytes, int64_t run) {
    Runs r(p, run);
    for (int i = 0; i < 3; ++i) r.add(stride[i] * bytes, size[i]);
    return r;
  };
  const int e = fp8 ? 1 : 2;
  const Runs all[4] = {placed(c.k, c.k_strides, e, e * c.head_dim), placed(c.v, c.v_strides, e, e * c.head_dim),
                       placed(c.k_scale, c.k_scale_strides, 4, 4), placed(c.v_scale, c.v_scale_strides, 4, 4)};
  const char* const names[4] = {"k", "v", "k_scale", "v_scale"};
  for (int i = 0; i < (fp8 ? 4 : 2); ++i)
    for (int j = 0; j < i; ++j)
      if (overlap(all[j], all[i])) return std::string(names[j]) + " and " + names[i] + " of the cache overlap";
  return "";
}

std::string rows_error(const void* p, int64_t token, int64_t head, const char* name) {
  if (!p) return std::string(name) + " is a null pointer";
  if (!multiple(p, 16) || token % 8 || head % 8) return std::string("rows of ") + name + " must be 16-byte aligned";
  return "";
}

// A launch takes fewer than 2^32 threads (16 a row at most): tokens in parts.
template <typename F>
int in_parts(KvArgs a, int64_t t, const char* name, F&& launch) {
  const int64_t most = (int64_t(1) << 26) / a.rows;
  for (int64_t t0 = 0; t0 < t; t0 += most) {
    const int64_t n = t - t0 < most ? t - t0 : most;
    KvArgs b = a;
    b.slots = a.slots + t0;
    b.positions = a.positions ? a.positions + t0 : nullptr;
    for (int p = 0; p < 3; ++p) {
      b.src[p] = a.src[p] ? a.src[p] + t0 * a.src_token[p] : nullptr;
      b.out[p] = a.out[p] ? a.out[p] + t0 * (p == 2 ? a.q_heads : a.heads) * a.d : nullptr;
    }
    launch(b, n);
    if (int rc = check_launch(name)) return rc;
  }
  return TF_OK;
}

}  // namespace

std::string kv_cache_error(const tf_kv_cache* c, int32_t dtype) {
  if (!c) return "null pointer";
  if (dtype != TF_DTYPE_FP16 && dtype != TF_DTYPE_BF16) return "unknown dtype";
  if (c->dtype != dtype && c->dtype != TF_DTYPE_E4M3) return "the cache's type is neither the rows' nor e4m3";
  if (!c->k || !c->v) return "null pointer";
  if (c->pages <= 0 || c->heads <= 0 || c->page_size <= 0) return "need pages, heads and page_size above 0";
  if (c->heads > 0xFFFF || c->page_size > (1 << 24) || c->pages > (int64_t(1) << 31))
    return "heads above 65535, pages of more than 2^24 tokens or more than 2^31 pages";
  if (c->head_dim <= 0 || c->head_dim % 8 || c->head_dim > TF_KV_MAX_HEAD_DIM)
    return "head_dim must be a multiple of 8 up to " + std::to_string(TF_KV_MAX_HEAD_DIM);
  const bool fp8 = c->dtype == TF_DTYPE_E4M3;
  if (!multiple(c->k, fp8 ? 8 : 16) || !multiple(c->v, fp8 ? 8 : 16)) return "unaligned cache";
  for (const int64_t* s : {c->k_strides, c->v_strides}) {
    if (s[0] % 8 || s[1] % 8 || s[2] % 8) return "unaligned rows of the cache";
    if (s[0] < 0 || s[1] < 0 || s[2] < 0) return "negative stride";
    if (s[2] >= kMaxTokenStride) return "tokens of a page 2^24 elements or more apart";
  }
  if (!fp8) return "";
  if (!c->k_scale || !c->v_scale) return "null pointer";
  for (const int64_t* s : {c->k_scale_strides, c->v_scale_strides}) {
    if (s[0] < 0 || s[1] < 0 || s[2] < 0) return "negative stride";
    if (s[2] >= kMaxTokenStride) return "scales of a page 2^24 elements or more apart";
  }
  return "";
}

}  // namespace tf

using namespace tf;

extern "C" int tf_kv_cache_write(const tf_kv_cache* cache, const uint16_t* k, int64_t k_token, int64_t k_head,
                                 const uint16_t* v, int64_t v_token, int64_t v_head, int32_t dtype,
                                 const int64_t* slots, int64_t t, void* stream) {
  const auto bad = [](const std::string& what) { return fail(TF_EINVAL, "tf_kv_cache_write: " + what); };
  std::string e = kv_cache_error(cache, dtype);
  if (e.empty()) e = written_error(*cache);
  if (e.empty()) e = rows_error(k, k_token, k_head, "k");
  if (e.empty()) e = rows_error(v, v_token, v_head, "v");
  if (!e.empty()) return bad(e);
  if (!slots) return bad("null pointer");
  if (t < 0) return bad("need t >= 0");
  KvArgs a = cache_args(*cache);
  a.src[0] = k, a.src_token[0] = k_token, a.src_head[0] = k_head;
  a.src[1] = v, a.src_token[1] = v_token, a.src_head[1] = v_head;
  a.slots = slots;
  return in_parts(a, t, "tf_kv_cache_write", [&](const KvArgs& b, int64_t n) {
    launch_type<kNone, false>(b, n, dtype == TF_DTYPE_BF16, cache->dtype == TF_DTYPE_E4M3, (hipStream_t)stream);
  });
}

extern "C" int tf_rope_kv_cache_write(const tf_kv_cache* cache, const uint16_t* q, int64_t q_token, int64_t q_head,
                                      int32_t q_heads, const uint16_t* k, int64_t k_token, int64_t k_head,
                                      const uint16_t* v, int64_t v_token, int64_t v_head, int32_t dtype,
                                      const float* cos_sin, int64_t max_positions, int32_t rot, int32_t interleaved,
                                      const int64_t* positions, const int64_t* slots, uint16_t* q_out, int64_t t,
                                      void* stream) {
  const auto bad = [](const std::string& what) { return fail(TF_EINVAL, "tf_rope_kv_cache_write: " + what); };
  std::string e = kv_cache_error(cache, dtype);
  if (e.empty()) e = written_error(*cache);
  if (e.empty()) e = rows_error(q, q_token, q_head, "q");
  if (e.empty()) e = rows_error(k, k_token, k_head, "k");
  if (e.empty()) e = rows_error(v, v_token, v_head, "v");
  if (e.empty()) e = rows_error(q_out, 0, 0, "q_out");
  if (!e.empty()) return bad(e);
  if (!slots || !positions || !cos_sin) return bad("null pointer");
  if (!multiple(cos_sin, 16)) return bad("cos_sin must be 16-byte aligned");
  if (q_heads <= 0 || q_heads > 0xFFFF) return bad("need q_heads from 1 to 65535");
  if (rot <= 0 || rot % 2 || rot > cache->head_dim) return bad("rot must be even, above 0 and at most head_dim");
  if (t < 0 || max_positions <= 0) return bad("need t >= 0 and max_positions above 0");
  KvArgs a = cache_args(*cache);
  a.src[0] = k, a.src_token[0] = k_token, a.src_head[0] = k_head;
  a.src[1] = v, a.src_token[1] = v_token, a.src_head[1] = v_head;
  a.src[2] = q, a.src_token[2] = q_token, a.src_head[2] = q_head;
  a.out[2] = q_out, a.q_heads = q_heads, a.rows += q_heads;
  a.slots = slots, a.positions = positions, a.cos_sin = cos_sin, a.max_positions = max_positions, a.rot = rot;
  const bool bf16 = dtype == TF_DTYPE_BF16, fp8 = cache->dtype == TF_DTYPE_E4M3;
  return in_parts(a, t, "tf_rope_kv_cache_write", [&](const KvArgs& b, int64_t n) {
    if (interleaved)
      launch_type<kPairs, false>(b, n, bf16, fp8, (hipStream_t)stream);
    else if (rot % 16 == 0)
      launch_type<kHalves, false>(b, n, bf16, fp8, (hipStream_t)stream);
    else
      launch_type<kOther, false>(b, n, bf16, fp8, (hipStream_t)stream);
  });
}

extern "C" int tf_kv_cache_read(const tf_kv_cache* cache, const int64_t* slots, uint16_t* k_out, uint16_t* v_out,
                                int32_t dtype, int64_t t, void* stream) {
  const auto bad = [](const std::string& what) { return fail(TF_EINVAL, "tf_kv_cache_read: " + what); };
  std::string e = kv_cache_error(cache, dtype);
  if (e.empty()) e = rows_error(k_out, 0, 0, "k_out");
  if (e.empty()) e = rows_error(v_out, 0, 0, "v_out");
  if (!e.empty()) return bad(e);
  if (!slots) return bad("null pointer");
  if (t < 0) return bad("need t >= 0");
  KvArgs a = cache_args(*cache);
  a.out[0] = k_out, a.out[1] = v_out, a.slots = slots;
  return in_parts(a, t, "tf_kv_cache_read", [&](const KvArgs& b, int64_t n) {
    launch_type<kNone, true>(b, n, dtype == TF_DTYPE_BF16, cache->dtype == TF_DTYPE_E4M3, (hipStream_t)stream);
  });
}
