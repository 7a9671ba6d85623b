// The attention kernels of heads up to 64.
#include "paged_attention.h"

namespace tf {

int launch_attention_d64(const AttnArgs& a, bool bf16, bool fp8, bool paged, bool full, unsigned grid,
                         hipStream_t stream) {
  return launch_attention<64>(a, bf16, fp8, paged, full, grid, stream);
}

}  // namespace tf
