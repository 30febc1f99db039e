// What the entry points of linear_i8.cu launch for the product of 8-bit matrices (gemm_i8.cu).
#pragma once

#include "elem_types.cuh"

struct s2v_gemm_i8_args {
    int64_t m, n, k, lda, ldb, ldc;
    const void* A;   // 8-bit, but for s2v_launch_gemv_i8 with an x_type
    const int8_t* B;
    const float* a_scale;
    const float* b_scale;
    const float* bias;
    int relu, c_type;
    void* C;
};
// `dependent`: the kernel in front writes A and a_scale and has told the next launch to start (griddepcontrol.launch_dependents)
int s2v_launch_gemm_i8(s2v_ctx* ctx, cudaStream_t st, const s2v_gemm_i8_args& a, bool dependent);
// gemm_i8_few.cu: one or two tokens that fit shared memory as 8-bit integers; x_type < 0: A is 8-bit with scales, else it is quantised on the way
bool s2v_gemv_i8_takes(int64_t m, int64_t n, int64_t k);
int s2v_launch_gemv_i8(s2v_ctx* ctx, cudaStream_t st, int x_type, const s2v_gemm_i8_args& a);
// gemm_i8_few.cu: outputs of few tiles, k > 0
float s2v_gemm_i8_split_cost(const s2v_ctx* ctx, const s2v_gemm_i8_args& a);   // us, about
int s2v_launch_gemm_i8_split(s2v_ctx* ctx, cudaStream_t st, const s2v_gemm_i8_args& a, bool dependent);
