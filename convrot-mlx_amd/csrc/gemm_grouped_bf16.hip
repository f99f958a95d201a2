// The grouped products of bfloat16.
#include "gemm_grouped_tile.h"

namespace convrot {
template hipError_t launch_grouped_tile<kBF16>(int tile, int kind, const GroupedOperands& p, hipStream_t stream);
}
