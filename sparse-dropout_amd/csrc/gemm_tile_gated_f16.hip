// The tile kernels with a gate in their store for fp16 operands.
#include "gemm_tile_launch.h"

namespace sd {
SD_TILE_GATED_INSTANCES(F16)
}  // namespace sd
