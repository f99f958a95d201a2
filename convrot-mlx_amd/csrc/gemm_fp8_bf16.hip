// The tiled products of 8-bit floating point with bfloat16 outputs.
#include "gemm_fp8_tile.h"

namespace convrot {
template hipError_t launch_fp8_tile<kBF16>(int tile, const Fp8Operands& p, const W8a8Split& split, hipStream_t stream);
}
