// paged_shares.h -- what the attention kernels over paged caches share: steps shared out to workgroups, and
// the joining of a row's parts.
#pragma once

#include "common.h"

namespace inf {

// `all` steps in `groups` shares, the first ones a step longer where they do not come out even.
struct Shares {
    int q, r;
    __device__ __forceinline__ Shares(int all, int groups) : q(all / groups), r(all - q * groups) {}
    __device__ __forceinline__ int start(int g) const { return g * q + min(g, r); }
    __device__ __forceinline__ int of(int step) const {
        const int big = r * (q + 1);
        return step < big ? step / (q + 1) : r + (step - big) / q;
    }
};

// The parts of a row: their number, and the first one's place in `part` and `stats` (in steps of Hq).
struct RowParts {
    int n;
    int64_t at;
};

// (M, L), a maximum and a sum of exponentials below it, with another such pair.
__device__ __forceinline__ void join_part(float& M, float& L, float m, float l) {
    const float top = fmaxf(M, m), ref = top == -INFINITY ? 0.f : top;
    L = L * fast_exp2(M - ref) + l * fast_exp2(m - ref);
    M = top;
}

}  // namespace inf
