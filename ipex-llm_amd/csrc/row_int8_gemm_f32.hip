// The tiled product with results in float32, and the integer sums of a split.
#include "row_int8_tiled.h"

namespace lowbit {

void launch_int8_f32(const Int8Args &p, int form, hipStream_t st) { launch_int8_form<float, INT8_PLAIN>(p, form, st); }
void launch_int8_part(const Int8Args &p, int form, hipStream_t st) { launch_int8_form<float, INT8_PART>(p, form, st); }

}  // namespace lowbit
