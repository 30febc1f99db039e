// What the entry points of linear_i8.cu launch for the product of 8-bit matrices (gemm_i8.cu).
#pragma once

#include "elem_types.cuh"

struct s2v_gemm_i8_args {
    int64_t m, n, k, lda, ldb, ldc;
    const int8_t* A;
    const int8_t* B;
    const float* a_scale;
    const float* b_scale;
    const float* bias;
    int relu, c_type;
    void* C;
};
int s2v_launch_gemm_i8(s2v_ctx* ctx, cudaStream_t st, const s2v_gemm_i8_args& a);
