// C entry of the block-scaled e4m3 linear: checks and the choice of the compiled kernel.
#include "fp8_block.h"

namespace tf {
namespace {

bool multiple(const void* p, uintptr_t a) { return (reinterpret_cast<uintptr_t>(p) % a) == 0; }

bool sizes_known(int64_t m, int64_t n, int64_t k) {
  return m >= 0 && n >= 0 && k >= 0 && m <= 0x7FFFFFFF && n <= 0x7FFFFF00 && k <= 0x7FFFFF00;
}

}  // namespace
}  // namespace tf

using namespace tf;

extern "C" int64_t tf_fp8_block_workspace_bytes(int64_t m, int64_t n, int64_t k, const tf_gemm_config* cfg) {
  if (!cfg || !sizes_known(m, n, k) || cfg->block_k != kBlockK) return -1;
  if (cfg->kernel == TF_KERNEL_FP8_BLOCK_GEMV) return block_gemv_known(*cfg) ? 0 : -1;
  if (cfg->kernel != TF_KERNEL_FP8_BLOCK_GEMM || !block_gemm_known(*cfg)) return -1;
  const int split = block_split(*cfg, cdiv(k, kBlockK));
  if (split <= 1) return 0;
  int64_t bytes = 0;
  if (__builtin_mul_overflow(m * n, split * (int64_t)sizeof(float), &bytes)) return -1;  // m * n < 2^62
  return bytes;
}

extern "C" int tf_fp8_block_linear(const uint8_t* x8, int64_t ldx8, const float* xscale, int64_t ldxs,
                                   const uint8_t* weight, int64_t ldw, const float* wscale, int64_t ldws,
                                   const uint16_t* bias, const uint16_t* residual, int64_t ldr, uint16_t* out,
                                   int64_t ldo, int32_t dtype, int64_t m, int64_t n, int64_t k,
                                   const tf_gemm_config* cfg, float* workspace, int64_t workspace_bytes,
                                   void* stream) {
  const auto bad = [](const std::string& what) { return fail(TF_EINVAL, "tf_fp8_block_linear: " + what); };
  if (!x8 || !xscale || !weight || !wscale || !out || !cfg) return bad("null pointer");
  if (dtype != TF_DTYPE_FP16 && dtype != TF_DTYPE_BF16) return bad("unknown dtype");
  if (!sizes_known(m, n, k) || k == 0) return bad("bad size");
  if (k % 16) return bad("k must be a multiple of 16");
  const int64_t nkb = cdiv(k, kBlockK);
  if (ldx8 < k || ldw < k || ldxs < nkb || ldws < nkb || ldo < n || (residual && ldr < n))
    return bad("row stride smaller than the row");
  if (ldx8 % 16 || ldw % 16 || !multiple(x8, 16) || !multiple(weight, 16))
    return bad("rows of x8 and weight must be 16-byte aligned");
  if (ldx8 >= kMaxCodeStride || ldw >= kMaxCodeStride || ldxs >= kMaxScaleStride)
    return bad("rows further apart than 4 MiB (codes) or 2^20 elements (scales)");
  const int64_t need = tf_fp8_block_workspace_bytes(m, n, k, cfg);
  if (need < 0) return bad("not a compiled config, or partial sums of 2^63 bytes");
  if (need > 0 && (!workspace || workspace_bytes < need))
    return bad("workspace too small (" + std::to_string(workspace_bytes) + " < " + std::to_string(need) + ")");
  if (need > 0 && !multiple(workspace, 16)) return bad("workspace not 16-byte aligned");
  if (m == 0 || n == 0) return TF_OK;
  BlockArgs a{};
  a.x8 = x8, a.ldx = ldx8, a.xs = xscale, a.ldxs = ldxs;
  a.w = weight, a.ldw = ldw, a.ws = wscale, a.ldws = ldws;
  a.bias = bias, a.residual = residual, a.ldr = ldr, a.out = out, a.ldo = ldo;
  a.m = (int)m, a.n = (int)n, a.k = (int)k, a.nkb = (int)nkb, a.bf16 = dtype == TF_DTYPE_BF16;
  if (cfg->kernel == TF_KERNEL_FP8_BLOCK_GEMV) return launch_block_gemv(a, *cfg, (hipStream_t)stream);
  return launch_block_gemm(a, *cfg, workspace, (hipStream_t)stream);
}
