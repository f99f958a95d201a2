// The grouped products of float16.
#include "gemm_grouped_tile.h"

namespace convrot {
template hipError_t launch_grouped_tile<kF16>(int tile, int kind, const GroupedOperands& p, hipStream_t stream);
}
