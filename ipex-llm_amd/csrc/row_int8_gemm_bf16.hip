// The tiled product with results in bfloat16.
#include "row_int8_tiled.h"

namespace lowbit {

void launch_int8_bf16(const Int8Args &p, int form, hipStream_t st) { launch_int8_form<__bf16, INT8_PLAIN>(p, form, st); }

}  // namespace lowbit
