// What s2v_linear_i8_grad (linear_i8_grad.cu) hands to the kernel for layers of few outputs over many rows (linear_i8_direct.cu).
#pragma once

#include "mm16.cuh"

struct linear_i8_grad_args {
    int64_t m, n, k, lddy, ldq, lddw;
    int dy_type;
    const void* dy;
    const int8_t* q;
    const float* scale;
    const float* factor;   // of columns of dy before they are rounded to fp16, or NULL
    const float* alpha;    // their inverses
    void* dW;
};
// whether the matrices lie as it needs them: rows on 16-byte boundaries
bool linear_i8_direct_lies(int64_t m, int dy_type, const void* dy, int64_t lddy, const int8_t* q, int64_t ldq);
bool linear_i8_direct_takes(int64_t m, int64_t n, int64_t k, int dy_type);
size_t linear_i8_direct_floats(int64_t m, int64_t n, int64_t k);   // of `part`; `columns`: [148][n] sums of dy, or NULL
int linear_i8_direct(s2v_ctx* ctx, cudaStream_t st, const linear_i8_grad_args& g, float* part, float* columns, int* shares);
