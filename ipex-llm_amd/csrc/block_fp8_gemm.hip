// Products of many rows in tiles (block_fp8_gemm.h): which tiles, how many splits of K, and the sum of the splits.
#include "block_fp8_tiled.h"
#include "lowbit_splits.h"

namespace lowbit {

// y = sum of the splits' float32 sums (+ bias), rounded once; four columns per thread.
template <typename OT>
__global__ __launch_bounds__(256) void block_fp8_reduce_kernel(const f32x4 *__restrict__ part, const OT *__restrict__ bias, OT *__restrict__ y,
                                                               int M, int N, int quads, int splits) {
    const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (id >= (int64_t)M * quads) return;
    const int m = (int)(id / quads), n = (int)(id - (int64_t)m * quads) * 4;
    const f32x4 v = sum_splits(part + id, (int64_t)M * quads, splits);
    OT *const to = y + (int64_t)m * N + n;
    typedef OT out4 __attribute__((ext_vector_type(4)));
    out4 o;
#pragma unroll
    for (int j = 0; j < 4; j++) o[j] = Stored<OT>::of(v[j] + (bias && n + j < N ? (float)bias[n + j] : 0.0f));
    if (n + 4 <= N) {
        __builtin_memcpy(to, &o, sizeof(o));                 // (rows may start at odd places)
        return;
    }
#pragma unroll
    for (int j = 0; j < 4; j++)
        if (n + j < N) to[j] = o[j];
}

static int cdiv(int a, int b) { return (a + b - 1) / b; }

// Rounds of workgroups over the GPU, each a walk of `steps` blocks.  A step is shorter on a CU that runs one workgroup where two fit, and
// while few CUs share the memory.
float tiled_walk_us(float step_us, float alone_us, int per_cu, int64_t units, int steps) {
    const int slots = 256 * per_cu;
    const int64_t rounds = units / slots, rest = units - rounds * slots;
    return steps * (rounds * step_us + (!rest ? 0.0f : rest <= 256 ? alone_us : step_us));
}

// Estimated time in us: the walks; what a launch, its first loads and its stores take, and again the first loads of each further round; the
// sums of two groups; with splits the sums written and read in float32.  The constants are fitted to timed launches of 705 sizes (float32:
// 462), weights from memory, 5 to 8192 rows by 256 to 28672 by 512 to 16384; on as many others the pick is 0.9 % (0.6 %) above the
// fastest of the forms and splits on average, 24 % at worst.
static float tiled_us(int form, int M, int N, int KB, int splits, bool exact) {
    const TiledForm &f = TILED_FORMS[form];
    const int64_t units = (int64_t)cdiv(M, f.rows) * cdiv(N, f.cols) * splits, further = (units - 1) / (256 * f.per_cu);
    float us = tiled_walk_us(exact ? f.exact_us : f.step_us, exact ? f.exact_alone_us : f.alone_us, f.per_cu, units, cdiv(cdiv(KB, splits), f.groups));
    us += (exact ? 4.1f : 4.6f) + 0.9f * further;
    if (f.groups > 1) us += 0.45f;
    if (splits > 1) us += 2.0f + (float)splits * M * N * 8.0f / (exact ? 3.9e6f : 5.0e6f);
    return us;
}

TiledPlan block_fp8_tiled_plan(bool exact, int M, int N, int K) {
    const int KB = fp8_blocks(K);
    TiledPlan best = {TILED_128_256, 1, 0.0f};
    for (int form = 0; form < TILED_COUNT; form++) {
        if (exact && TILED_FORMS[form].exact_us == 0.0f) continue;
        static const int tried[] = {1, 2, 3, 4, 6, 8};
        for (int splits : tried) {
            if (splits > 1 && (KB < 2 * splits || (int64_t)cdiv(M, TILED_FORMS[form].rows) * cdiv(N, TILED_FORMS[form].cols) >= 512)) break;
            if (splits > 1 && (size_t)splits * M * ((N + 3) / 4 * 4) * 4 > (size_t)256 << 20) break;
            const float us = tiled_us(form, M, N, KB, splits, exact);
            if (best.us == 0.0f || us < best.us) best = {form, splits, us};
        }
    }
    best.splits = cdiv(KB, cdiv(KB, best.splits));           // (every split has a block)
    return best;
}

size_t block_fp8_tiled_part_bytes(const TiledPlan &plan, int M, int N) {
    return plan.splits > 1 ? (size_t)plan.splits * M * ((N + 3) / 4 * 4) * 4 : 0;
}

void launch_block_fp8_reduce(const float *part, const void *bias, void *y, int dtype, int M, int N, int splits, hipStream_t st) {
    const int quads = (N + 3) / 4;
    const dim3 grid((uint32_t)(((int64_t)M * quads + 255) / 256));
    if (dtype == DT_F16)
        hipLaunchKernelGGL((block_fp8_reduce_kernel<_Float16>), grid, dim3(256), 0, st, (const f32x4 *)part, (const _Float16 *)bias, (_Float16 *)y, M, N, quads, splits);
    else if (dtype == DT_BF16)
        hipLaunchKernelGGL((block_fp8_reduce_kernel<__bf16>), grid, dim3(256), 0, st, (const f32x4 *)part, (const __bf16 *)bias, (__bf16 *)y, M, N, quads, splits);
    else
        hipLaunchKernelGGL((block_fp8_reduce_kernel<float>), grid, dim3(256), 0, st, (const f32x4 *)part, (const float *)bias, (float *)y, M, N, quads, splits);
}

// p: x (codes), xs, w, ws, bias, y, M, N, K and, for splits, part
int launch_block_fp8_tiled(TiledArgs p, int dtype, const TiledPlan &plan, hipStream_t st) {
    p.KB = fp8_blocks(p.K);
    p.ldx = (int64_t)p.KB * FP8_BLOCK * (dtype == DT_F32 ? 2 : 1);
    p.ldxs = p.M;
    p.pitch = (p.N + 3) / 4 * 4;
    p.splits = plan.splits;
    p.split_blocks = cdiv(p.KB, plan.splits);
    const TiledForm &f = TILED_FORMS[plan.form];
    if ((int64_t)cdiv(p.M, f.rows) * cdiv(p.N, f.cols) * plan.splits > most_groups(512)) return -3;
    if (plan.splits > 1) {
        if (dtype == DT_F32) launch_tiled_part_exact(p, plan.form, st);
        else launch_tiled_part(p, plan.form, st);
        launch_block_fp8_reduce(p.part, p.bias, p.y, dtype, p.M, p.N, plan.splits, st);
    } else if (dtype == DT_F16) launch_tiled_f16(p, plan.form, st);
    else if (dtype == DT_BF16) launch_tiled_bf16(p, plan.form, st);
    else launch_tiled_f32(p, plan.form, st);
    return 0;
}

}  // namespace lowbit
