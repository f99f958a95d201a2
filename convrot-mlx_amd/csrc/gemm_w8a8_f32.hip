// The tiled W8A8 kernels with float32 outputs.
#include "gemm_w8a8_tile.h"

namespace convrot {
template hipError_t launch_w8a8_tile<kF32>(int tile, const W8a8Operands& p, const W8a8Split& split, hipStream_t stream);
}
