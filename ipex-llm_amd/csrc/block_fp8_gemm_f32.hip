// The tiled products (block_fp8_gemm.h) with results in f32; a file of their own for the build's sake.
#include "block_fp8_tiled.h"

namespace lowbit {

void launch_tiled_f32(const TiledArgs &p, int form, hipStream_t st) { launch_tiled_form<float, true, TILED_PLAIN>(p, form, st); }
void launch_tiled_part_exact(const TiledArgs &p, int form, hipStream_t st) { launch_tiled_form<float, true, TILED_PART>(p, form, st); }

}  // namespace lowbit
