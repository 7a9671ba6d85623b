// The attention kernels of heads up to 128.
#include "paged_attention.h"

namespace tf {

int launch_attention_d128(const AttnArgs& a, const AttnKind& k, int tiles, unsigned grid, hipStream_t stream) {
  return tiles == 1 ? launch_attention<128, 1>(a, k, grid, stream) : launch_attention<128, 2>(a, k, grid, stream);
}

}  // namespace tf
