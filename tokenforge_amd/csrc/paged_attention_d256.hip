// The attention kernels of heads up to 256.
#include "paged_attention.h"

namespace tf {

int launch_attention_d256(const AttnArgs& a, const AttnKind& k, unsigned grid, hipStream_t stream) {
  return launch_attention<256, 1>(a, k, grid, stream);
}

}  // namespace tf
