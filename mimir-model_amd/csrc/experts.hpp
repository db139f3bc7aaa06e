// What the kernels of a mixture of experts share: the plan that puts the
// (token, choice) pairs of a call in order by expert (include/mimg.h).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace mimg {

constexpr int EXPERTS_MAX = 512;    // experts of a layer
constexpr int EXPERTS_MAX_TOP = 32; // choices of a token

// The int32 entries of a plan: first[experts + 1] (the place of each expert's
// first pair in the order; the last entry is the number of pairs that have an
// expert), then from a multiple of 64 on the order (pairs by expert, those
// of an expert in rising order, pairs without one behind all), then likewise
// each pair's expert (-1 without one).
struct PlanLayout {
    int64_t order, expert, total;
};
__host__ __device__ __forceinline__ PlanLayout plan_layout(int64_t pairs, int experts) {
    PlanLayout l;
    l.order = (experts + 1 + 63) / 64 * 64;
    l.expert = l.order + (pairs + 63) / 64 * 64;
    l.total = l.expert + pairs;
    return l;
}

// Whether a workgroup of 256 for every four rows of an expert, `groups` times
// over, is a grid (less than 2^32 threads).
inline bool experts_gemv_grid(int64_t n, int64_t groups) { return (n + 3) / 4 * groups < (1ll << 24); }

// A pair's expert as the plan has it, held to the call's own experts: a plan of
// another call gives wrong results, and no access elsewhere.
__device__ __forceinline__ int plan_expert(const int32_t* expert, int64_t pair, int experts) {
    const int e = expert[pair];
    return e < experts ? e : -1;
}

}  // namespace mimg
