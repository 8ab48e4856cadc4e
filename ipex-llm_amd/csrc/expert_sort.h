// The pairs of a mixture-of-experts block sorted by expert: offsets[e] .. offsets[e + 1] - 1 are the places of expert e's pairs, in their
// order; order[place] is the pair there, pos[pair] its place (-1: an id that names no expert).
//
// Up to EXPERTS_SORT_PAIRS pairs one workgroup sorts them, beside others of its launch that do other work.  More, or more than EXPERTS_SORT_EXPERTS:
// workgroups of that launch count a chunk of pairs each, and a second launch places them.  A whole block in int8, 4096 pairs over 64 experts of [512 x 1024]
// 51.4 us with one workgroup and 55.7 with a second launch, 3300 over 8 of [256 x 512] 31 and 37.
//
// The block-scaled experts have a third way, counted_by_each: a wave for each pair and each expert counts what comes before it.
#pragma once
#include "lowbit_formats.h"

namespace lowbit {

constexpr int EXPERTS_SORT_PAIRS = 4096, EXPERTS_SORT_EXPERTS = 2048, EXPERTS_CHUNKS = 256;

inline bool one_sorts(int64_t pairs, int n_exp) { return pairs <= EXPERTS_SORT_PAIRS && n_exp <= EXPERTS_SORT_EXPERTS; }

// Few pairs for the experts there are: each counted by a wave of its own.  That grows with pairs * pairs but not with the experts, of which one workgroup has
// counts to clear, to sum and to find: a whole block-scaled block of [128 x 256] with 1600 pairs over 160 experts 27.4 us this way and 28.5 with one workgroup, over
// 16 25.9 and 25.5; 1920 over 64 26.1 and 26.4; 2400 over 128 29.1 and 28.5, over 1024 114 and 118, over 2100, which one workgroup does not take, 255 and 362; 3000
// over 8 34.8 and 31.3.
inline bool counted_by_each(int64_t pairs, int n_exp) { return pairs <= 3200 && 5 * (int64_t)n_exp >= pairs - 1600; }
inline size_t sort_lds(int n_exp) { return (size_t)n_exp * 4 * sizeof(int32_t); }

// pairs of a chunk, whole waves of them
__host__ __device__ inline int sort_chunk(int pairs) { return ((pairs + EXPERTS_CHUNKS - 1) / EXPERTS_CHUNKS + 63) / 64 * 64; }

// The 256 threads of a workgroup sort the pairs.  Each wave has a run of them, 64 at a time: it counts them by expert, the counts become first
// places, and a second pass over the ids, which are in registers, places them.  Lanes of the same expert find one another by a ballot for each
// bit of its number.  sort_lds(n_exp) bytes of dynamic LDS.
__device__ __forceinline__ void sort_pairs(const int64_t *__restrict__ ids, int32_t *__restrict__ offsets, int32_t *__restrict__ order, int32_t *__restrict__ pos,
                                  int pairs, int n_exp) {
    constexpr int HELD = EXPERTS_SORT_PAIRS / 256;
    extern __shared__ int32_t places[];                      // [4][n_exp]: pairs of each wave, then their next places
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
    const int run = (pairs + 255) / 256 * 64, first = wave * run;
    int e[HELD];
#pragma unroll
    for (int i = 0; i < HELD; i++) {
        const int b = first + i * 64 + lane;
        const int64_t id = i * 64 < run && b < pairs ? ids[b] : -1;
        e[i] = id >= 0 && id < n_exp ? (int)id : -1;
    }
    for (int i = t; i < 4 * n_exp; i += 256) places[i] = 0;
    __syncthreads();
    const int own = wave * n_exp;
#pragma unroll
    for (int i = 0; i < HELD; i++)
        if (e[i] >= 0) atomicAdd(&places[own + e[i]], 1);
    __syncthreads();
    if (wave == 0) {
        int before = 0;
        for (int e0 = 0; e0 < n_exp; e0 += 64) {
            const int at = e0 + lane;
            int n[4] = {}, all = 0;
            if (at < n_exp)
#pragma unroll
                for (int w = 0; w < 4; w++) all += n[w] = places[w * n_exp + at];
            int upto = all;
#pragma unroll
            for (int d = 1; d < 64; d <<= 1) {
                const int up = __shfl_up(upto, d);
                if (lane >= d) upto += up;
            }
            int place = before + upto - all;
            if (at < n_exp) {
                offsets[at] = place;
#pragma unroll
                for (int w = 0; w < 4; w++) {
                    places[w * n_exp + at] = place;
                    place += n[w];
                }
            }
            before += __builtin_amdgcn_readlane(upto, 63);
        }
        if (lane == 0) offsets[n_exp] = before;
    }
    __syncthreads();
    const int bits = 32 - __builtin_clz(n_exp);              // (every number below n_exp, and the -1 of no expert is not among them)
#pragma unroll
    for (int i = 0; i < HELD; i++) {
        if (i * 64 >= run) break;
        uint64_t same = __ballot(e[i] >= 0);
        for (int bit = 0; bit < bits; bit++) {
            const uint64_t set = __ballot(e[i] >> bit & 1);
            same &= e[i] >> bit & 1 ? set : ~set;
        }
        const int b = first + i * 64 + lane;
        int place = -1;
        if (e[i] >= 0) {
            const int rank = __popcll(same & ((1ull << lane) - 1));
            // (LDS accesses of a wave keep their order, among the lanes and from turn to turn)
            asm volatile("" ::: "memory");
            place = places[own + e[i]] + rank;
            order[place] = b;
            asm volatile("" ::: "memory");
            if (rank == 0) places[own + e[i]] = place + __popcll(same);
        }
        if (b < pairs) pos[b] = place;
    }
}

// Workgroup `at` of (pairs + n_exp + 4) / 4 places four: a wave counts the pairs that come before its own - those of lower experts, and the earlier ones of its
// expert -, and waves pairs + e write offsets[e].
__device__ __forceinline__ void count_for_each(const int64_t *__restrict__ ids, int32_t *__restrict__ offsets, int32_t *__restrict__ order, int32_t *__restrict__ pos,
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
__device__ __forceinline__ void count_pairs(const int64_t *__restrict__ ids, int32_t *__restrict__ counts, int pairs, int n_exp, int chunk, int at) {
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
