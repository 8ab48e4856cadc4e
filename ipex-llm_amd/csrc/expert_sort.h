// The pairs of a mixture-of-experts block sorted by expert: offsets[e] .. offsets[e + 1] - 1 are the places of expert e's pairs, in their
// order; order[place] is the pair there, pos[pair] its place (-1: an id that names no expert).
//
// Up to EXPERTS_SORT_PAIRS pairs one launch places them, whose first workgroups may do other work.  More: its workgroups count a chunk of pairs
// each, and a second launch places them.
#pragma once
#include "lowbit_formats.h"

namespace lowbit {

constexpr int EXPERTS_SORT_PAIRS = 3200, EXPERTS_CHUNKS = 256;

// pairs of a chunk, whole waves of them
__host__ __device__ inline int sort_chunk(int pairs) { return ((pairs + EXPERTS_CHUNKS - 1) / EXPERTS_CHUNKS + 63) / 64 * 64; }

// Workgroup `at` of 256 places four pairs: a wave counts the pairs that come before its own - those of lower experts, and the earlier ones of its
// expert -, and waves pairs + e write offsets[e].  (pairs + n_exp + 4) / 4 workgroups.
__device__ inline void place_pairs(const int64_t *__restrict__ ids, int32_t *__restrict__ offsets, int32_t *__restrict__ order, int32_t *__restrict__ pos,
                                   int pairs, int n_exp, int at) {
    const int lane = threadIdx.x & 63, b = at * 4 + (threadIdx.x >> 6);
    if (b > pairs + n_exp) return;
    const bool is_pair = b < pairs;
    const int64_t own = is_pair ? ids[b] : b - pairs;
    int before = 0;
    for (int j0 = lane; j0 - lane < pairs; j0 += 512) {
        int64_t e[8];
#pragma unroll
        for (int i = 0; i < 8; i++) e[i] = j0 + i * 64 < pairs ? ids[j0 + i * 64] : -1;
#pragma unroll
        for (int i = 0; i < 8; i++)
            before += __popcll(__ballot(e[i] >= 0 && e[i] < n_exp && (e[i] < own || (is_pair && e[i] == own && j0 + i * 64 < b))));
    }
    if (lane != 0) return;
    if (!is_pair) {
        offsets[own] = before;
        return;
    }
    const bool valid = own >= 0 && own < n_exp;
    pos[b] = valid ? before : -1;
    if (valid) order[before] = b;
}

// Workgroup `at` of 256 counts its chunk's pairs by expert, counts[at][e], in n_exp words of dynamic LDS.
__device__ inline void count_pairs(const int64_t *__restrict__ ids, int32_t *__restrict__ counts, int pairs, int n_exp, int chunk, int at) {
    extern __shared__ int32_t seen[];
    const int first = at * chunk, last = first + chunk < pairs ? first + chunk : pairs;
    for (int e = threadIdx.x; e < n_exp; e += 256) seen[e] = 0;
    __syncthreads();
    for (int b = first + threadIdx.x; b < last; b += 256) {
        const int64_t e = ids[b];
        if (e >= 0 && e < n_exp) atomicAdd(&seen[e], 1);
    }
    __syncthreads();
    for (int e = threadIdx.x; e < n_exp; e += 256) counts[(int64_t)at * n_exp + e] = seen[e];
}

// the second launch
void launch_expert_place(const int64_t *ids, const int32_t *counts, int32_t *offsets, int32_t *order, int32_t *pos, int pairs, int n_exp, hipStream_t st);

}  // namespace lowbit
