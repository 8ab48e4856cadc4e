// The forms of the tiled product that launches choose from.
#pragma once
#include "block_fp8_gemm.h"

namespace lowbit {

// rows and weight rows of a tile, workgroups that a CU holds, groups of waves that share its blocks, and a step's time (us): with the GPU
// full, with one workgroup on a CU; the same with float32 results, whose codes go through the bfloat16 MFMA (0: no such form; waves of 64 x
// 64 on a tile of 128 x 128 take 2.8 us there, and no size would choose them)
struct TiledForm {
    int rows, cols, per_cu, groups;
    float step_us, alone_us, exact_us, exact_alone_us;
};
enum { TILED_256, TILED_192_256, TILED_128_256, TILED_128, TILED_64, TILED_32, TILED_64_SHARED, TILED_64_64_SHARED, TILED_COUNT };
static const TiledForm TILED_FORMS[TILED_COUNT] = {
    {256, 256, 1, 1, 1.73f, 1.48f, 0.0f, 0.0f},
    {192, 256, 1, 1, 1.40f, 1.11f, 0.0f, 0.0f},
    {128, 256, 1, 1, 1.03f, 0.83f, 1.82f, 1.43f},
    {128, 128, 2, 1, 0.99f, 0.54f, 0.0f, 0.0f},
    {64, 128, 2, 1, 0.68f, 0.37f, 1.00f, 0.60f},
    {32, 128, 2, 1, 0.70f, 0.34f, 0.91f, 0.48f},
    {64, 128, 1, 2, 0.86f, 0.65f, 1.16f, 1.05f},
    {64, 64, 1, 2, 0.70f, 0.43f, 0.97f, 0.66f},
};

struct TiledPlan {
    int form, splits;
    float us;
};

// One launch per form; the wave tiles are 64 x 128, 96 x 64, 64 x 64, 64 x 64, 32 x 64, 32 x 32, 32 x 64 and 32 x 32.
template <typename OT, bool EXACT, TiledMode MODE, bool BY_EXPERT = false> void launch_tiled_form(const TiledArgs &p, int form, hipStream_t st) {
    if (form == TILED_256) {
        // (the operands of a 64 x 128 wave tile in bfloat16 do not fit its registers: no plan asks for it)
        if constexpr (!EXACT) launch_tiled<OT, EXACT, MODE, BY_EXPERT, false, 4, 8, 4, 2, 2, 2>(p, st);
    } else if (form == TILED_192_256) {
        // (rows of x in bfloat16 do not fit LDS twice)
        if constexpr (!EXACT) launch_tiled<OT, EXACT, MODE, BY_EXPERT, false, 6, 4, 2, 4, 2, 2>(p, st);
    } else if (form == TILED_128_256) launch_tiled<OT, EXACT, MODE, BY_EXPERT, false, 4, 4, 2, 4, EXACT ? 2 : 3, 2>(p, st);
    else if (form == TILED_128) {
        if constexpr (!EXACT) launch_tiled<OT, EXACT, MODE, BY_EXPERT, false, 4, 4, 2, 2, 2, 2>(p, st);
    } else if (form == TILED_64) launch_tiled<OT, EXACT, MODE, BY_EXPERT, false, 2, 4, 2, 2, EXACT ? 2 : 3, 2>(p, st);
    else if (form == TILED_32) launch_tiled<OT, EXACT, MODE, BY_EXPERT, false, 2, 2, 1, 4, 3, 2>(p, st);
    else if constexpr (!BY_EXPERT) {
        if (form == TILED_64_SHARED) launch_tiled<OT, EXACT, MODE, BY_EXPERT, false, 2, 4, 2, 2, EXACT ? 2 : 3, 2, 2>(p, st);
        else launch_tiled<OT, EXACT, MODE, BY_EXPERT, false, 2, 2, 2, 2, 3, 2, 2>(p, st);
    }
}

void launch_tiled_f16(const TiledArgs &p, int form, hipStream_t st);
void launch_tiled_bf16(const TiledArgs &p, int form, hipStream_t st);
void launch_tiled_f32(const TiledArgs &p, int form, hipStream_t st);
void launch_tiled_part(const TiledArgs &p, int form, hipStream_t st);
void launch_tiled_part_exact(const TiledArgs &p, int form, hipStream_t st);

// Estimated time (us) of `units` tiles of a form that walk `steps` blocks each
float tiled_walk_us(float step_us, float alone_us, int per_cu, int64_t units, int steps);
TiledPlan block_fp8_tiled_plan(bool exact, int M, int N, int K);
size_t block_fp8_tiled_part_bytes(const TiledPlan &plan, int M, int N);
int launch_block_fp8_tiled(TiledArgs p, int dtype, const TiledPlan &plan, hipStream_t st);

}  // namespace lowbit
