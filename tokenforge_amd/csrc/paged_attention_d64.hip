// The attention kernels of heads up to 64.
#include "paged_attention.h"

namespace tf {

int launch_attention_d64(const AttnArgs& a, const AttnKind& k, int tiles, unsigned grid, hipStream_t stream) {
  return tiles == 1 ? launch_attention<64, 1>(a, k, grid, stream) : launch_attention<64, 2>(a, k, grid, stream);
}

}  // namespace tf
