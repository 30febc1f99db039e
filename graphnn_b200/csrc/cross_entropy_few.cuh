// The loss over a few classes for a mini-batch (cross_entropy_few.cu): launches are what such calls take.
#pragma once

#include "elem_types.cuh"

bool xe_few_takes(int64_t rows, int64_t vocab, int64_t k);
size_t xe_few_bytes(int64_t rows, int64_t vocab);   // of the gradient's workspace
int xe_few_loss(s2v_ctx* ctx, cudaStream_t st, int64_t rows, int64_t vocab, int64_t k, int type, const void* x, int64_t ldx, const void* W, int64_t ldw, const int32_t* target,
                const float* row_weight, float* loss, float* stats);
int xe_few_grad(s2v_ctx* ctx, cudaStream_t st, int64_t rows, int64_t vocab, int64_t k, int type, const void* x, int64_t ldx, const void* W, int64_t ldw, const int32_t* target,
                const float* row_weight, const float* stats, void* workspace, void* dx, int64_t lddx, void* dW, int64_t lddw);
