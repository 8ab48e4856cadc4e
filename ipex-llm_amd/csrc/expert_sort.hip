// The launch that places counted pairs (expert_sort.h).
#include "expert_sort.h"

namespace lowbit {

// Places the pairs of a chunk per wave behind those of lower experts and of earlier chunks, in their order.  Every workgroup sums the chunks'
// counts for itself; four waves each, since with sixteen the ranks of 64 pairs, 300 instructions, wait for one another (10 and 18 us).  6726
// pairs over 4 experts 6.6 us, 32768 over 128 16.
__global__ __launch_bounds__(256) void expert_place_kernel(const int64_t *__restrict__ ids, const int32_t *__restrict__ counts,
                                                           int32_t *__restrict__ offsets, int32_t *__restrict__ order,
                                                           int32_t *__restrict__ pos, int pairs, int n_exp, int chunks, int chunk) {
    constexpr int U = 16;                                    // counts on their way together
    extern __shared__ int32_t at[];                          // [n_exp] pairs of earlier chunks, [n_exp + 1] offsets, [waves][n_exp] next places
    const int threads = blockDim.x, waves = threads >> 6, t = threadIdx.x, lane = t & 63, wave = t >> 6, c0 = blockIdx.x * waves;
    int32_t *const before = at, *const total = at + n_exp, *const next = total + n_exp + 1;
    for (int e = t; e < 2 * n_exp; e += threads) at[e] = 0;
    __syncthreads();
    const int parts = threads > n_exp ? threads / n_exp : 1, step = threads > n_exp ? n_exp : threads, part = t / step;
    if (part < parts)
        for (int e = t - part * step; e < n_exp; e += step) {
            int earlier = 0, all = 0;
            for (int c = part; c < chunks; c += parts * U) {
                int n[U];
#pragma unroll
                for (int u = 0; u < U; u++) n[u] = c + u * parts < chunks ? counts[(int64_t)(c + u * parts) * n_exp + e] : 0;
#pragma unroll
                for (int u = 0; u < U; u++) {
                    all += n[u];
                    earlier += c + u * parts < c0 ? n[u] : 0;
                }
            }
            atomicAdd(&before[e], earlier);
            atomicAdd(&total[e], all);
        }
    __syncthreads();
    if (wave == 0) {                                         // total: from sums to offsets
        int sum = 0;
        for (int e0 = 0; e0 < n_exp; e0 += 64) {
            const int own = e0 + lane < n_exp ? total[e0 + lane] : 0;
            int upto = own;
#pragma unroll
            for (int d = 1; d < 64; d <<= 1) {
                const int up = __shfl_up(upto, d);
                if (lane >= d) upto += up;
            }
            if (e0 + lane < n_exp) total[e0 + lane] = sum + upto - own;
            sum += __builtin_amdgcn_readlane(upto, 63);
        }
        if (lane == 0) total[n_exp] = sum;
    }
    __syncthreads();
    if (blockIdx.x == 0)
        for (int e = t; e <= n_exp; e += threads) offsets[e] = total[e];
    for (int e = t; e < n_exp; e += threads) {
        int place = total[e] + before[e];
        for (int w = 0; w < waves; w += U) {
            int n[U];
#pragma unroll
            for (int u = 0; u < U; u++) n[u] = c0 + w + u < chunks ? counts[(int64_t)(c0 + w + u) * n_exp + e] : 0;
#pragma unroll
            for (int u = 0; u < U; u++) {
                if (w + u < waves) next[(w + u) * n_exp + e] = place;
                place += n[u];
            }
        }
    }
    __syncthreads();
    const int first = (c0 + wave) * chunk;                   // (a chunk past the last one starts behind the pairs)
    for (int i = 0; i < chunk; i += 64) {
        const int b = first + i + lane;
        const int64_t id = b < pairs ? ids[b] : -1;
        const int e = id >= 0 && id < n_exp ? (int)id : -1;
        int rank = 0, same = 0;                              // among the 64 pairs of the same expert
#pragma unroll
        for (int l = 0; l < 64; l++) {
            const bool equal = __builtin_amdgcn_readlane(e, l) == e;
            same += equal;
            rank += equal && l < lane;
        }
        const int place = e >= 0 ? next[wave * n_exp + e] + rank : -1;
        __syncthreads();                                     // (places are read ahead of their update, and after the last one's)
        if (e >= 0 && rank == same - 1) next[wave * n_exp + e] += same;
        __syncthreads();
        if (b < pairs) pos[b] = place;
        if (e >= 0) order[place] = b;
    }
}

void launch_expert_place(const int64_t *ids, const int32_t *counts, int32_t *offsets, int32_t *order, int32_t *pos, int pairs, int n_exp, hipStream_t st) {
    const int chunk = sort_chunk(pairs), chunks = (pairs + chunk - 1) / chunk;
    const int waves = n_exp <= 2048 ? 4 : 1;                 // at most 48 KiB
    hipLaunchKernelGGL(expert_place_kernel, dim3((chunks + waves - 1) / waves), dim3(64 * waves), ((size_t)n_exp * (waves + 2) + 1) * 4, st, ids, counts,
                       offsets, order, pos, pairs, n_exp, chunks, chunk);
}

}  // namespace lowbit
