// The gradient that flows on below a product with a weight in e4m3 and a scale for each block of 128 (block_fp8.h):
//     gx[m, k] = sum_nb ws[nb, k / 128] * sum_{n in nb} g[m, n] * wc[n, k]
//
// g stays in 16 bits: codes are exact in either 16-bit type, so the products are exact, the sums float32 and the result is rounded once.
// The sum runs along N, across the rows of the weight: its tile is turned over on the way into LDS.
#include "block_fp8.h"

namespace lowbit {

template <typename AT>
__global__ __launch_bounds__(256) void block_fp8_back_kernel(const AT *__restrict__ grad, const uint8_t *__restrict__ w, const float *__restrict__ ws,
                                                             AT *__restrict__ gx, int M, int N, int K) {
    using V8 = typename Vec8<AT>::type;
    constexpr int PITCH = 40;                                // 32 values of n and 8 to spread the rows over the banks
    __shared__ __attribute__((aligned(16))) AT wt[64 * PITCH], gt[64 * PITCH];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 15, g = lane >> 4;
    const int k0 = blockIdx.x * 64, m0 = blockIdx.y * 64, KB = fp8_blocks(K);
    f32x4 acc[4] = {};
    for (int nb = 0; nb < N; nb += FP8_BLOCK) {
        f32x4 part[4] = {};
        for (int n0 = nb; n0 < nb + FP8_BLOCK && n0 < N; n0 += 32) {
            __syncthreads();
            for (int i = threadIdx.x; i < 64 * 32; i += 256) {
                const int n = i >> 6, k = i & 63;
                const int code = n0 + n < N && k0 + k < K ? w[(int64_t)(n0 + n) * K + k0 + k] : 0;
                wt[k * PITCH + n] = to_at<AT>(__builtin_amdgcn_cvt_pk_f32_fp8(code, false)[0]);
                const int m = i >> 5, gn = i & 31;
                gt[m * PITCH + gn] = m0 + m < M && n0 + gn < N ? grad[(int64_t)(m0 + m) * N + n0 + gn] : to_at<AT>(0.0f);
            }
            __syncthreads();
            const V8 a = *(const V8 *)(wt + (wave * 16 + r) * PITCH + g * 8);
#pragma unroll
            for (int i = 0; i < 4; i++) part[i] = mfma16(a, *(const V8 *)(gt + (i * 16 + r) * PITCH + g * 8), part[i]);
        }
        const float s = ws[(int64_t)(nb / FP8_BLOCK) * KB + k0 / FP8_BLOCK];
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
            for (int j = 0; j < 4; j++) acc[i][j] = fmaf(s, part[i][j], acc[i][j]);
    }
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const int m = m0 + i * 16 + r;
        if (m >= M) continue;
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const int k = k0 + wave * 16 + g * 4 + j;
            if (k < K) gx[(int64_t)m * K + k] = to_at<AT>(acc[i][j]);
        }
    }
}

size_t block_fp8_back_workspace_bytes(int dtype, int M, int N, int K) { return 0; }

int launch_block_fp8_back(const void *grad, const uint8_t *w, const float *ws, void *gx, int dtype, int M, int N, int K, uint8_t *space,
                          hipStream_t st) {
    const dim3 grid((K + 63) / 64, (M + 63) / 64);
    if (dtype == DT_F16)
        hipLaunchKernelGGL((block_fp8_back_kernel<_Float16>), grid, dim3(256), 0, st, (const _Float16 *)grad, w, ws, (_Float16 *)gx, M, N, K);
    else if (dtype == DT_BF16)
        hipLaunchKernelGGL((block_fp8_back_kernel<__bf16>), grid, dim3(256), 0, st, (const __bf16 *)grad, w, ws, (__bf16 *)gx, M, N, K);
    else return -4;
    return 0;
}

}  // namespace lowbit
