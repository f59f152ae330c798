// The tile kernels with a gate in their store for bf16 operands.
#include "gemm_tile_launch.h"

namespace sd {
SD_TILE_GATED_INSTANCES(BF16)
}  // namespace sd
