// Products of many rows in tiles (row_int8_gemm.h): which tiles, how many splits of K, and the sum of the splits.
#include "row_int8_stream.h"

namespace lowbit {

// y = xs * ws * sum of the splits' sums (+ bias), rounded once; four columns per thread.  Whole numbers: exact in any order, and in float32 rounded once.
template <typename OT>
__global__ __launch_bounds__(256) void row_int8_reduce_kernel(const i32x4 *__restrict__ part, const float *__restrict__ xs, const float *__restrict__ ws,
                                                              const OT *__restrict__ bias, OT *__restrict__ y, int M, int N, int quads, int splits, int64_t first) {
    const int64_t id = first + (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (id >= (int64_t)M * quads) return;
    const int m = (int)(id / quads), n = (int)(id - (int64_t)m * quads) * 4;
    const int64_t stride = (int64_t)M * quads;
    const i32x4 *at = part + id;
    int64_t v[4] = {};                                       // (64 bits: given_codes_plan in row_int8_rows.hip)
    for (int s = 0; s < splits; s++) {
        const i32x4 one = at[s * stride];
#pragma unroll
        for (int j = 0; j < 4; j++) v[j] += one[j];
    }
    const float by = xs[m];
    OT *const to = y + (int64_t)m * N + n;
    typedef OT out4 __attribute__((ext_vector_type(4)));
    out4 o;
#pragma unroll
    for (int j = 0; j < 4; j++) o[j] = n + j < N ? Stored<OT>::of((float)v[j] * by * ws[n + j] + (bias ? (float)bias[n + j] : 0.0f)) : OT{};
    if (n + 4 <= N) {
        __builtin_memcpy(to, &o, sizeof(o));                 // (rows may start at odd places)
        return;
    }
#pragma unroll
    for (int j = 0; j < 4; j++)
        if (n + j < N) to[j] = o[j];
}

static int cdiv(int a, int b) { return (a + b - 1) / b; }

template <typename OT, bool PART> static void launch_stream(const Int8Args &p, int waves, hipStream_t st) {
    const dim3 grid((p.N + 15) / 16, p.splits);
    if (p.M > 16) {
        if (waves == 4) hipLaunchKernelGGL((row_int8_stream_kernel<OT, PART, 2, 4>), grid, dim3(256), 0, st, p);
        else hipLaunchKernelGGL((row_int8_stream_kernel<OT, PART, 2, 8>), grid, dim3(512), 0, st, p);
    } else if (waves == 4) hipLaunchKernelGGL((row_int8_stream_kernel<OT, PART, 1, 4>), grid, dim3(256), 0, st, p);
    else hipLaunchKernelGGL((row_int8_stream_kernel<OT, PART, 1, 8>), grid, dim3(512), 0, st, p);
}

// Estimated times in us, fitted to timed launches with weights from memory.
//
// Tiles: rounds of workgroups over the GPU, each a walk of blocks; a step with one workgroup on a CU is longer where the weight comes from memory, which one
// of 2 MB starts to and one of 16 MB does; what a launch, its first loads and its stores take, and again the first loads of each further round; the
// results, which forms of two workgroups on a CU write while the other one multiplies; the sums of groups; with splits the sums written and read.
// 233 sizes, 5 to 8192 rows by 64 to 28672 by 128 to 16384, forms and splits of each: the pick is 1.7 % above the fastest on average.
static float tiled_us(int form, int M, int N, int KB, int splits) {
    const Int8Form &f = INT8_FORMS[form];
    const int64_t units = (int64_t)cdiv(M, f.rows) * cdiv(N, f.cols) * splits, further = (units - 1) / (256 * f.per_cu);
    const float megabytes = (float)N * KB * INT8_BLOCK * 1e-6f, far = megabytes <= 2.0f ? 0.0f : megabytes >= 16.0f ? 1.0f : log2f(megabytes * 0.5f) / 3.0f;
    float us = tiled_walk_us(f.step_us, f.alone_us + far * f.far_us, f.per_cu, units, cdiv(cdiv(KB, splits), f.groups)) + 3.24f + 0.11f * far + 0.83f * further;
    us += (f.per_cu == 1 ? 0.38e-6f : 0.28e-6f) * 2.0f * M * N;
    if (f.groups > 1) us += 0.5f;
    if (splits > 1) us += 1.16f + 0.76f * log2f((float)splits) + (float)splits * M * N * 8.0f / 3.6e6f;
    return us;
}
// The streaming kernel: blocks of K that a CU walks, each with x, and what the other CUs leave it of the memory; 518 launches of 1 to 32 rows, within 9 %
// at rms.  Eight waves per workgroup while there are no more than three workgroups for two CUs, with twelve blocks or more to walk: the pick of the
// two is 1.1 % above the shorter on average.
static int stream_waves(int N, int KB, int splits) { return cdiv(N, 16) * splits <= 384 && cdiv(KB, splits) >= 12 ? 8 : 4; }
static float stream_us(int M, int N, int KB, int splits) {
    const float units = (float)cdiv(N, 16) * splits / 256, load = units > 1.0f ? units : 1.0f, shared = units < 1.0f ? units : 1.0f;
    float us = 2.7f + 0.07f * (load - 1.0f) + cdiv(KB, splits) * (load * (0.084f + 0.0025f * M) + shared * 0.032f);
    if (splits > 1) us += 2.4f + (float)splits * M * N * 8.0f / 3.6e6f;
    return us;
}

Int8Plan row_int8_product_plan(int M, int N, int K) {
    static const int tried[] = {1, 2, 3, 4, 6, 8};
    const int KB = int8_blocks(K);
    Int8Plan best = {INT8_128_256, 1, 0, 0.0f};
    auto take = [&](const Int8Plan &p) {
        if (best.us == 0.0f || p.us < best.us) best = p;
    };
    for (int form = 0; form < INT8_COUNT; form++)
        for (int splits : tried) {
            if (splits > 1 && (KB < 2 * splits || (int64_t)cdiv(M, INT8_FORMS[form].rows) * cdiv(N, INT8_FORMS[form].cols) >= 512)) break;
            if (splits > 1 && (size_t)splits * M * ((N + 3) / 4 * 4) * 4 > (size_t)256 << 20) break;
            take({form, splits, 0, tiled_us(form, M, N, KB, splits)});
        }
    if (M <= STREAM_ROWS)
        for (int splits : tried) {
            if (splits > 1 && KB < 2 * splits) break;
            take({0, splits, 1, stream_us(M, N, KB, splits)});
        }
    best.splits = cdiv(KB, cdiv(KB, best.splits));           // (every split has a block)
    if (best.waves) best.waves = stream_waves(N, KB, best.splits);
    return best;
}

size_t row_int8_part_bytes(const Int8Plan &plan, int M, int N) {
    return plan.splits > 1 ? (size_t)plan.splits * M * ((N + 3) / 4 * 4) * 4 : 0;
}

template <typename OT> static void launch_reduce(const Int8Args &p, hipStream_t st) {
    const int quads = (p.N + 3) / 4;
    constexpr int64_t most = (int64_t)1 << 31;               // threads of a launch
    for (int64_t first = 0, all = (int64_t)p.M * quads; first < all; first += most)
        hipLaunchKernelGGL((row_int8_reduce_kernel<OT>), dim3((uint32_t)(((all - first < most ? all - first : most) + 255) / 256)), dim3(256), 0, st,
                           (const i32x4 *)p.part, p.xs, p.ws, (const OT *)p.bias, (OT *)p.y, p.M, p.N, quads, p.splits, first);
}

// p: x (codes in rows of ldx bytes, zeros past K up to whole blocks), xs, w, ws, bias, y, M, N, K and, for splits, part
int launch_row_int8_codes(Int8Args p, int dtype, const Int8Plan &plan, hipStream_t st) {
    p.KB = int8_blocks(p.K);
    p.pitch = (p.N + 3) / 4 * 4;
    p.splits = plan.splits;
    p.split_blocks = cdiv(p.KB, plan.splits);
    const Int8Form &f = INT8_FORMS[plan.form];
    if ((int64_t)cdiv(p.M, plan.waves ? STREAM_ROWS : f.rows) * cdiv(p.N, plan.waves ? 16 : f.cols) * plan.splits > most_groups(512)) return -3;
    if (plan.splits > 1) {
        if (plan.waves) launch_stream<float, true>(p, plan.waves, st);
        else launch_int8_part(p, plan.form, st);
        if (dtype == DT_F16) launch_reduce<_Float16>(p, st);
        else if (dtype == DT_BF16) launch_reduce<__bf16>(p, st);
        else launch_reduce<float>(p, st);
    } else if (dtype == DT_F16) {
        if (plan.waves) launch_stream<_Float16, false>(p, plan.waves, st);
        else launch_int8_f16(p, plan.form, st);
    } else if (dtype == DT_BF16) {
        if (plan.waves) launch_stream<__bf16, false>(p, plan.waves, st);
        else launch_int8_bf16(p, plan.form, st);
    } else if (plan.waves) launch_stream<float, false>(p, plan.waves, st);
    else launch_int8_f32(p, plan.form, st);
    return 0;
}

}  // namespace lowbit
