// What every form of the loss over a vocabulary makes of a row: which class is its own, and its loss.
#pragma once

#include "elem_types.cuh"

namespace
{

struct xe_rows {
    const int32_t* target;
    const float* weight;   // NULL: ones
    int64_t vocab;
    // the row's class, -1 if it has none
    __device__ __forceinline__ int64_t its(int64_t i) const
    {
        const int64_t t = target[i];
        return t < 0 || t >= vocab ? -1 : t;
    }
    __device__ __forceinline__ bool counts(int64_t i) const { return !weight || weight[i] != 0.0f; }
    // the row's class, -1 if it is left out
    __device__ __forceinline__ int64_t own(int64_t i) const { return counts(i) ? its(i) : -1; }
};

// A row's loss and what is kept of it, from the largest logit m and l = sum exp(z - m) of the other classes and the own one's logit:
// log(1 + l exp(m - z_t)), from whichever side is the larger; alone in the vocabulary a class loses nothing.  An own logit of +infinity has no loss (infinity less
// infinity), although the others are nothing beside it; one of -infinity loses everything, and the others' sum is what it is.  What is kept has nothing to do with the row's weight, which the gradient's call brings along: a weight of 0 here need not be 0 there.
__device__ __forceinline__ void xe_finish(const xe_rows& rows, int64_t i, float m, float l, float mine, float* loss, float2* stats)
{
    const double d = (double)m - (double)mine;
    double one, lse;
    if ((m == -INFINITY && l == 0.0f) || mine == INFINITY) one = (double)(mine - mine), lse = one + (double)mine;
    else if (d > 0) {
        const double beside = log((double)l + exp(-d));   // the sum of all relative to m
        one = d + beside, lse = (double)m + beside;
    } else one = log1p((double)l * exp(d)), lse = one + (double)mine;
    loss[i] = !rows.counts(i) ? 0.0f : (float)(one * (rows.weight ? (double)rows.weight[i] : 1.0));
    if (stats) stats[i] = make_float2((float)lse, (float)expm1(-one));
}

}  // namespace
