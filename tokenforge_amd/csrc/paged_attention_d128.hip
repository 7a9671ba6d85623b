// The attention kernels of heads up to 128.
#include "paged_attention.h"

namespace tf {

int launch_attention_d128(const AttnArgs& a, bool bf16, bool fp8, bool paged, bool full, unsigned grid,
                         hipStream_t stream) {
  return launch_attention<128>(a, bf16, fp8, paged, full, grid, stream);
}

}  // namespace tf
