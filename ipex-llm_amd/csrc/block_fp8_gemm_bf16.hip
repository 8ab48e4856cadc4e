// The tiled products (block_fp8_gemm.h) with results in bf16; a file of their own for the build's sake.
#include "block_fp8_tiled.h"

namespace lowbit {

void launch_tiled_bf16(const TiledArgs &p, int form, hipStream_t st) { launch_tiled_form<__bf16, false, TILED_PLAIN>(p, form, st); }

}  // namespace lowbit
