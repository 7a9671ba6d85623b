// Writing a paged key-value cache, with or without the rotation of queries and keys in front, and reading it
// back by slots.
//
// A row (one head of one token) lies on 8, 16 or 32 lanes, eight elements a lane, so its absmax is 3 to 5 lane
// exchanges and nothing crosses a row. The launch is flat over the rows of all tokens: a token's keys, its
// values, then (rope) its queries. Every byte is read and written once; memory bound from some thousand
// tokens on, latency below.
#include "kv_cache.h"

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
  int64_t rows;
  uint32_t per_token;  // rows of a token: 2 * heads (+ q_heads)
  int heads, q_heads, d, rot, page_size;
};

// The largest of v over the row's LANES lanes (8, 16 or 32; all active), in each of them.
template <int LANES>
__device__ __forceinline__ uint32_t row_max_u32(uint32_t v) {
  v = __builtin_elementwise_max(v, dpp_u32<kDppQuadXor1>(v));
  v = __builtin_elementwise_max(v, dpp_u32<kDppQuadXor2>(v));
  v = __builtin_elementwise_max(v, dpp_u32<kDppHalfRowMirror>(v));
  if (LANES > 8) v = __builtin_elementwise_max(v, dpp_u32<kDppRowMirror>(v));
  if (LANES > 16) {
    const auto s = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    v = __builtin_elementwise_max((uint32_t)s[0], (uint32_t)s[1]);
  }
  return v;
}

// Where row `row` belongs: its token, 0 (k), 1 (v) or 2 (q), and its head.
struct Row {
  int64_t token;
  int part, head;
};

__device__ __forceinline__ Row row_of(const KvArgs& a, uint32_t row) {
  const uint32_t t = row / a.per_token;
  const int r = (int)(row - t * a.per_token);
  if (r < a.heads) return Row{t, 0, r};
  if (r < 2 * a.heads) return Row{t, 1, r - a.heads};
  return Row{t, 2, r - 2 * a.heads};
}

// y of the row's elements e0 .. e0 + 7 (own values in y), rotated in fp32. `x` is the row.
template <typename T, bool INTERLEAVED>
__device__ __forceinline__ void rotate8(const KvArgs& a, const uint16_t* x, int64_t token, int e0, float (&y)[8]) {
  const int half = a.rot >> 1;
  if (e0 >= a.rot) return;
  const int64_t pos = a.positions[token];
  const bool known = pos >= 0 && pos < a.max_positions;
  const float* const cs = a.cos_sin + (known ? pos : 0) * a.rot;
  if (INTERLEAVED) {
#pragma unroll
    for (int j = 0; j < 8; j += 2) {
      if (e0 + j >= a.rot) break;
      const float c = cs[(e0 + j) >> 1], s = cs[half + ((e0 + j) >> 1)];
      const float u = y[j], w = y[j + 1];
      y[j] = known ? u * c - w * s : __builtin_nanf("");
      y[j + 1] = known ? w * c + u * s : __builtin_nanf("");
    }
    return;
  }
  if ((half & 7) == 0) {  // the partners are eight consecutive elements, in the row's other half
    const bool first = e0 < half;
    const int i0 = first ? e0 : e0 - half;
    float w[8];
    unpack8<T>(*reinterpret_cast<const u4*>(x + (first ? e0 + half : e0 - half)), w);
    const f4 c0 = *reinterpret_cast<const f4*>(cs + i0), c1 = *reinterpret_cast<const f4*>(cs + i0 + 4);
    const f4 s0 = *reinterpret_cast<const f4*>(cs + half + i0), s1 = *reinterpret_cast<const f4*>(cs + half + i0 + 4);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float c = j < 4 ? c0[j & 3] : c1[j & 3], s = j < 4 ? s0[j & 3] : s1[j & 3];
      const float r = first ? y[j] * c - w[j] * s : y[j] * c + w[j] * s;
      y[j] = known ? r : __builtin_nanf("");
    }
    return;
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const int e = e0 + j;
    if (e >= a.rot) break;
    const int i = e < half ? e : e - half;
    const uint32_t o = x[e < half ? e + half : e - half];
    const float w = T::lo(o), c = cs[i], s = cs[half + i];
    const float r = e < half ? y[j] * c - w * s : y[j] * c + w * s;
    y[j] = known ? r : __builtin_nanf("");
  }
}

enum Rope { kNone = 0, kHalves = 1, kPairs = 2 };

template <typename T, bool FP8, int ROPE, int LANES>
__global__ __launch_bounds__(256) void kv_write_kernel(KvArgs a) {
  const int64_t row = (int64_t)blockIdx.x * (256 / LANES) + threadIdx.x / LANES;
  const int e0 = (threadIdx.x % LANES) * 8;
  const bool live = row < a.rows, mine = live && e0 < a.d;
  const Row r = row_of(a, live ? (uint32_t)row : 0u);
  const uint16_t* const x = a.src[r.part] + r.token * a.src_token[r.part] + r.head * a.src_head[r.part];
  u4 v = {0u, 0u, 0u, 0u};
  if (mine) v = *reinterpret_cast<const u4*>(x + e0);
  const int64_t slot = r.part < 2 ? a.slots[r.token] : 0;
  float y[8];
  unpack8<T>(v, y);
  if (ROPE != kNone && mine && r.part != 1) rotate8<T, ROPE == kPairs>(a, x, r.token, e0, y);
  if (ROPE != kNone && (!FP8 || r.part == 2) && r.part != 1) {
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = round_pair<T>(y[2 * j], y[2 * j + 1]);
  }
  if (ROPE != kNone && r.part == 2) {
    if (mine) *reinterpret_cast<u4*>(a.out[2] + (r.token * a.q_heads + r.head) * a.d + e0) = v;
  }
  const bool kept = mine && r.part < 2 && slot >= 0 && slot < a.capacity;
  const int p = r.part & 1;
  const int64_t page = kept ? slot / a.page_size : 0, off = kept ? slot - page * a.page_size : 0;
  const int64_t at = page * a.page_stride[p] + r.head * a.head_stride[p] + off * a.token_stride[p] + e0;
  if (FP8) {
    const uint32_t amax = row_max_u32<LANES>(absmax8(y));
    const float s = dynamic_scale(as_f32(amax));
    const u2 codes = encode8(y, s, amax);
    if (kept) {
      *reinterpret_cast<u2*>(a.cache[p] + at) = codes;
      if (e0 == 0) a.scale[p][page * a.scale_page[p] + r.head * a.scale_head[p] + off * a.scale_token[p]] = s;
    }
  } else if (kept) {
    *reinterpret_cast<u4*>(reinterpret_cast<uint16_t*>(a.cache[p]) + at) = v;
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

template <typename T, bool FP8, int LANES>
__global__ __launch_bounds__(256) void kv_read_kernel(KvArgs a) {
  const int64_t row = (int64_t)blockIdx.x * (256 / LANES) + threadIdx.x / LANES;
  const int e0 = (threadIdx.x % LANES) * 8;
  if (row >= a.rows || e0 >= a.d) return;
  const Row r = row_of(a, (uint32_t)row);
  const int64_t slot = a.slots[r.token];
  u4 v = {0u, 0u, 0u, 0u};
  if (slot >= 0 && slot < a.capacity) {
    const int64_t page = slot / a.page_size, off = slot - page * a.page_size;
    const int p = r.part;
    const int64_t at = page * a.page_stride[p] + r.head * a.head_stride[p] + off * a.token_stride[p] + e0;
    if (FP8) {
      const float s = a.scale[p][page * a.scale_page[p] + r.head * a.scale_head[p] + off * a.scale_token[p]];
      v = decode8<T>(*reinterpret_cast<const u2*>(a.cache[p] + at), s);
    } else {
      v = *reinterpret_cast<const u4*>(reinterpret_cast<const uint16_t*>(a.cache[p]) + at);
    }
  }
  *reinterpret_cast<u4*>(a.out[r.part] + (r.token * a.heads + r.head) * a.d + e0) = v;
}

template <typename T, bool FP8, int ROPE, bool READ, int LANES>
void launch_lanes(const KvArgs& a, hipStream_t stream) {
  const unsigned grid = (unsigned)cdiv(a.rows, 256 / LANES);
  if (READ)
    kv_read_kernel<T, FP8, LANES><<<grid, 256, 0, stream>>>(a);
  else
    kv_write_kernel<T, FP8, ROPE, LANES><<<grid, 256, 0, stream>>>(a);
}

template <typename T, bool FP8, int ROPE, bool READ>
void launch_row(const KvArgs& a, hipStream_t stream) {
  if (a.d <= 64)
    launch_lanes<T, FP8, ROPE, READ, 8>(a, stream);
  else if (a.d <= 128)
    launch_lanes<T, FP8, ROPE, READ, 16>(a, stream);
  else
    launch_lanes<T, FP8, ROPE, READ, 32>(a, stream);
}

template <int ROPE, bool READ>
void launch_type(const KvArgs& a, bool bf16, bool fp8, hipStream_t stream) {
  if (bf16)
    fp8 ? launch_row<BF16, true, ROPE, READ>(a, stream) : launch_row<BF16, false, ROPE, READ>(a, stream);
  else
    fp8 ? launch_row<F16, true, ROPE, READ>(a, stream) : launch_row<F16, false, ROPE, READ>(a, stream);
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
  a.heads = c.heads, a.d = c.head_dim, a.page_size = c.page_size;
  a.per_token = 2u * (uint32_t)c.heads;
  return a;
}

std::string rows_error(const void* p, int64_t token, int64_t head, const char* name) {
  if (!p) return std::string(name) + " is a null pointer";
  if (!multiple(p, 16) || token % 8 || head % 8) return std::string("rows of ") + name + " must be 16-byte aligned";
  return "";
}

// A launch takes fewer than 2^32 threads and 2^31 rows: tokens in parts.
template <typename F>
int in_parts(KvArgs a, int64_t t, const char* name, F&& launch) {
  const int64_t most = (int64_t(1) << 26) / a.per_token > 0 ? (int64_t(1) << 26) / a.per_token : 1;
  for (int64_t t0 = 0; t0 < t; t0 += most) {
    const int64_t n = t - t0 < most ? t - t0 : most;
    KvArgs b = a;
    b.rows = n * a.per_token;
    b.slots = a.slots + t0;
    b.positions = a.positions ? a.positions + t0 : nullptr;
    for (int p = 0; p < 3; ++p) {
      b.src[p] = a.src[p] ? a.src[p] + t0 * a.src_token[p] : nullptr;
      b.out[p] = a.out[p] ? a.out[p] + t0 * (p == 2 ? a.q_heads : a.heads) * a.d : nullptr;
    }
    launch(b);
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
  if (e.empty()) e = rows_error(k, k_token, k_head, "k");
  if (e.empty()) e = rows_error(v, v_token, v_head, "v");
  if (!e.empty()) return bad(e);
  if (!slots) return bad("null pointer");
  if (t < 0) return bad("need t >= 0");
  KvArgs a = cache_args(*cache);
  a.src[0] = k, a.src_token[0] = k_token, a.src_head[0] = k_head;
  a.src[1] = v, a.src_token[1] = v_token, a.src_head[1] = v_head;
  a.slots = slots;
  return in_parts(a, t, "tf_kv_cache_write", [&](const KvArgs& b) {
    launch_type<kNone, false>(b, dtype == TF_DTYPE_BF16, cache->dtype == TF_DTYPE_E4M3, (hipStream_t)stream);
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
  a.out[2] = q_out, a.q_heads = q_heads, a.per_token += (uint32_t)q_heads;
  a.slots = slots, a.positions = positions, a.cos_sin = cos_sin, a.max_positions = max_positions, a.rot = rot;
  const bool bf16 = dtype == TF_DTYPE_BF16, fp8 = cache->dtype == TF_DTYPE_E4M3;
  return in_parts(a, t, "tf_rope_kv_cache_write", [&](const KvArgs& b) {
    if (interleaved)
      launch_type<kPairs, false>(b, bf16, fp8, (hipStream_t)stream);
    else
      launch_type<kHalves, false>(b, bf16, fp8, (hipStream_t)stream);
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
  return in_parts(a, t, "tf_kv_cache_read", [&](const KvArgs& b) {
    launch_type<kNone, true>(b, dtype == TF_DTYPE_BF16, cache->dtype == TF_DTYPE_E4M3, (hipStream_t)stream);
  });
}
