// The tiled products (block_fp8_gemm.h) with results in f16; a file of their own for the build's sake.
#include "block_fp8_tiled.h"

namespace lowbit {

void launch_tiled_f16(const TiledArgs &p, int form, hipStream_t st) { launch_tiled_form<_Float16, false, TILED_PLAIN>(p, form, st); }
void launch_tiled_part(const TiledArgs &p, int form, hipStream_t st) { launch_tiled_form<float, false, TILED_PART>(p, form, st); }

}  // namespace lowbit
