// Products of many rows in tiles (row_int8_gemm.h): which tiles, how many splits of K, and the sum of the splits.
#include "row_int8_tiled.h"

namespace lowbit {

// y = xs * ws * sum of the splits' sums (+ bias), rounded once; four columns per thread.  Whole numbers: exact in any order.
template <typename OT>
__global__ __launch_bounds__(256) void row_int8_reduce_kernel(const i32x4 *__restrict__ part, const float *__restrict__ xs, const float *__restrict__ ws,
                                                              const OT *__restrict__ bias, OT *__restrict__ y, int M, int N, int quads, int splits) {
    const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (id >= (int64_t)M * quads) return;
    const int m = (int)(id / quads), n = (int)(id - (int64_t)m * quads) * 4;
    const int64_t stride = (int64_t)M * quads;
    const i32x4 *at = part + id;
    i32x4 v = *at;
    for (int s = 1; s < splits; s++) v += at[s * stride];
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

// Estimated time in us: rounds of workgroups over the GPU, each a walk of blocks; what a launch, its first loads and its stores take, and
// again the first loads of each further round; the sums of two groups; with splits the sums written and read.
static float tiled_us(int form, int M, int N, int KB, int splits) {
    const Int8Form &f = INT8_FORMS[form];
    const int64_t units = (int64_t)cdiv(M, f.rows) * cdiv(N, f.cols) * splits, further = (units - 1) / (256 * f.per_cu);
    float us = tiled_walk_us(f.step_us, f.alone_us, f.per_cu, units, cdiv(cdiv(KB, splits), f.groups)) + 4.6f + 0.9f * further;
    if (f.groups > 1) us += 0.45f;
    if (splits > 1) us += 2.0f + (float)splits * M * N * 8.0f / 5.0e6f;
    return us;
}

Int8Plan row_int8_tiled_plan(int M, int N, int K) {
    const int KB = int8_blocks(K);
    Int8Plan best = {INT8_128_256, 1, 0.0f};
    for (int form = 0; form < INT8_COUNT; form++) {
        static const int tried[] = {1, 2, 3, 4, 6, 8};
        for (int splits : tried) {
            if (splits > 1 && (KB < 2 * splits || (int64_t)cdiv(M, INT8_FORMS[form].rows) * cdiv(N, INT8_FORMS[form].cols) >= 512)) break;
            if (splits > 1 && (size_t)splits * M * ((N + 3) / 4 * 4) * 4 > (size_t)256 << 20) break;
            const float us = tiled_us(form, M, N, KB, splits);
            if (best.us == 0.0f || us < best.us) best = {form, splits, us};
        }
    }
    best.splits = cdiv(KB, cdiv(KB, best.splits));           // (every split has a block)
    return best;
}

size_t row_int8_part_bytes(const Int8Plan &plan, int M, int N) {
    return plan.splits > 1 ? (size_t)plan.splits * M * ((N + 3) / 4 * 4) * 4 : 0;
}

template <typename OT> static void launch_reduce(const Int8Args &p, hipStream_t st) {
    const int quads = (p.N + 3) / 4;
    hipLaunchKernelGGL((row_int8_reduce_kernel<OT>), dim3((uint32_t)(((int64_t)p.M * quads + 255) / 256)), dim3(256), 0, st, (const i32x4 *)p.part, p.xs,
                       p.ws, (const OT *)p.bias, (OT *)p.y, p.M, p.N, quads, p.splits);
}

// p: x (codes in rows of ldx bytes, zeros past K up to whole blocks), xs, w, ws, bias, y, M, N, K and, for splits, part
int launch_row_int8_tiled(Int8Args p, int dtype, const Int8Plan &plan, hipStream_t st) {
    p.KB = int8_blocks(p.K);
    p.pitch = (p.N + 3) / 4 * 4;
    p.splits = plan.splits;
    p.split_blocks = cdiv(p.KB, plan.splits);
    const Int8Form &f = INT8_FORMS[plan.form];
    if ((int64_t)cdiv(p.M, f.rows) * cdiv(p.N, f.cols) * plan.splits > most_groups(512)) return -3;
    if (plan.splits > 1) {
        launch_int8_part(p, plan.form, st);
        if (dtype == DT_F16) launch_reduce<_Float16>(p, st);
        else if (dtype == DT_BF16) launch_reduce<__bf16>(p, st);
        else launch_reduce<float>(p, st);
    } else if (dtype == DT_F16) launch_int8_f16(p, plan.form, st);
    else if (dtype == DT_BF16) launch_int8_bf16(p, plan.form, st);
    else launch_int8_f32(p, plan.form, st);
    return 0;
}

}  // namespace lowbit
