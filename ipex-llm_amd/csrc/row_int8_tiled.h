// The forms of the tiled product that launches choose from.
#pragma once
#include "row_int8_gemm.h"

namespace lowbit {

// rows and weight rows of a tile, workgroups that a CU holds, groups of waves that share its blocks, and a step's time (us): with the GPU
// full, with one workgroup on a CU, and what the latter takes longer where the weight comes from memory
struct Int8Form {
    int rows, cols, per_cu, groups;
    float step_us, alone_us, far_us;
};
enum { INT8_256, INT8_192_256, INT8_128_256, INT8_128, INT8_32, INT8_128_WIDE, INT8_64_WIDE, INT8_64_SHARED, INT8_32_SHARED, INT8_COUNT };
static const Int8Form INT8_FORMS[INT8_COUNT] = {
    {256, 256, 1, 1, 1.26f, 0.95f, 0.10f},
    {192, 256, 1, 1, 1.025f, 0.76f, 0.17f},
    {128, 256, 1, 1, 0.764f, 0.606f, 0.19f},
    {128, 128, 2, 1, 0.888f, 0.426f, 0.107f},
    {32, 128, 2, 1, 0.507f, 0.214f, 0.161f},
    {128, 128, 1, 1, 0.486f, 0.344f, 0.132f},
    {64, 128, 1, 1, 0.368f, 0.248f, 0.146f},
    {64, 64, 1, 2, 0.686f, 0.419f, 0.113f},
    {64, 32, 1, 4, 0.911f, 0.527f, 0.116f},
};

// What a product of codes runs as: a form of tiles, or (waves > 0) the streaming kernel of row_int8_stream.h
struct Int8Plan {
    int form, splits, waves;
    float us;
};

// One launch per form; the wave tiles are 64 x 128, 96 x 64, 64 x 64, 64 x 64, 32 x 32, 32 x 64 and three times 32 x 32.  Forms of one workgroup on a CU
// fill its LDS with as many buffers as there is room for.
//
// Weights from memory: 512 rows by [4096 x 4096] take 18.7 us in tiles of 64 x 128 of four waves, two workgroups on a CU, and 16.7 in those of eight
// waves; 150 by [13824 x 5120] 28.0 and 25.6 in tiles of 128 x 128; 64 by [4096 x 11008] 30.4 in tiles of 64 x 64 shared by two groups, and 23.0
// in tiles of 64 x 32 shared by four, which put twice the CUs to work.
template <typename OT, Int8Mode MODE> void launch_int8_form(const Int8Args &p, int form, hipStream_t st) {
    if (form == INT8_256) launch_int8_tile<OT, MODE, false, false, 4, 8, 4, 2, 2, 2>(p, st);
    else if (form == INT8_192_256) launch_int8_tile<OT, MODE, false, false, 6, 4, 2, 4, 2, 2>(p, st);
    else if (form == INT8_128_256) launch_int8_tile<OT, MODE, false, false, 4, 4, 2, 4, 3, 2>(p, st);
    else if (form == INT8_128) launch_int8_tile<OT, MODE, false, false, 4, 4, 2, 2, 2, 2>(p, st);
    else if (form == INT8_32) launch_int8_tile<OT, MODE, false, false, 2, 2, 1, 4, 3, 2>(p, st);
    else if (form == INT8_128_WIDE) launch_int8_tile<OT, MODE, false, false, 2, 4, 4, 2, 4, 2>(p, st);
    else if (form == INT8_64_WIDE) launch_int8_tile<OT, MODE, false, false, 2, 2, 2, 4, 4, 2>(p, st);
    else if (form == INT8_64_SHARED) launch_int8_tile<OT, MODE, false, false, 2, 2, 2, 2, 4, 2, 2>(p, st);
    else launch_int8_tile<OT, MODE, false, false, 2, 2, 2, 1, 3, 2, 4>(p, st);
}

void launch_int8_f16(const Int8Args &p, int form, hipStream_t st);
void launch_int8_bf16(const Int8Args &p, int form, hipStream_t st);
void launch_int8_f32(const Int8Args &p, int form, hipStream_t st);
void launch_int8_part(const Int8Args &p, int form, hipStream_t st);

// Estimated time (us) of `units` tiles of a form that walk `steps` blocks each (block_fp8_gemm.hip)
float tiled_walk_us(float step_us, float alone_us, int per_cu, int64_t units, int steps);
Int8Plan row_int8_product_plan(int M, int N, int K);
size_t row_int8_part_bytes(const Int8Plan &plan, int M, int N);
int launch_row_int8_codes(Int8Args p, int dtype, const Int8Plan &plan, hipStream_t st);
int launch_row_int8_quantize(const void *x, int dtype, int64_t rows, int K, uint8_t *codes, int ldc, float *scale, const int32_t *limit, hipStream_t st);

}  // namespace lowbit
