// Products of 16-bit matrices on the tensor cores (mm16.cu) for the loss over a vocabulary and for weight gradients.
//
// fp32 operands come as three bf16 matrices ("parts") whose sum they are, x = x0 + x1 + x2 with |x1| <= 2^-9 |x| and |x2| <= 2^-18 |x|, and
// sum x y = x0 y0 + x0 y1 + x1 y0 + x1 y1 + x0 y2 + x2 y0, leaving out terms of 2^-26 and less: six products at the rate of 16-bit ones, each exact in
// fp32 accumulators, where the fp32 units would take thirty.
#pragma once

#include "elem_types.cuh"

// One operand: `parts` matrices [rows x cols] of 16-bit numbers, rows `ld` numbers apart (a multiple of 8, 16-byte aligned), parts `part` numbers apart.
struct mm16_operand {
    const void* p = nullptr;
    int64_t rows = 0, cols = 0, ld = 0, part = 0;
    int parts = 1;
};

struct mm16_args {
    int type = S2V_BF16;      // of both operands: S2V_F16 or S2V_BF16
    mm16_operand a, b;        // along k: [m x k], [n x k];  across: [k x m], [k x n]
    int64_t m = 0, n = 0, k = 0;
    // rows' classes (loss): a target outside [0, vocab), or a weight of 0, leaves the row out
    const int32_t* target = nullptr;
    const float* weight = nullptr;
    int64_t vocab = 0, first = 0;       // the n columns are the classes from `first` on
    // MM16_SUMS: for each row and half tile of columns, the largest output m and sum exp(. - m) of the columns other than the row's own; the own one's output
    float2* part = nullptr;             // [mm16_sum_lines(...)][m]
    float* mine = nullptr;              // [m]
    // MM16_SOFTMAX_GRAD: row_scale (exp(. - stats.x), in the row's own column stats.y), as 16-bit numbers (one part of S2V_F16, one or three of S2V_BF16)
    const float2* stats = nullptr;
    const float* row_scale = nullptr;   // [m]; 0: zeros, whatever the outputs are
    void* g = nullptr;
    int64_t ldg = 0, g_part = 0;        // rows of a multiple of 64 numbers
    int g_parts = 1;
    // MM16_OUT and the others: out = alpha * product (+ what `sum` holds); alpha: one number, or one for each row, or NULL
    const float* alpha = nullptr;
    int alpha_rows = 0;
    float* sum = nullptr;               // [m x mm16_pitch(n)] fp32; outputs of the products before this one, and of this one where `out` is NULL
    bool add = false;                   // whether sum holds something
    const float* fix = nullptr;         // [m] or NULL: out gets fix_i times row target_i of fix_w ([vocab x n], of out_type) too
    const void* fix_w = nullptr;
    int64_t fix_ld = 0;
    float* lines = nullptr;             // mm16_lines_bytes(): sums of shares of k
    int out_type = S2V_F32;
    void* out = nullptr;
    int64_t ldo = 0;
};
enum mm16_kind { MM16_SUMS, MM16_SOFTMAX_GRAD, MM16_OUT, MM16_OUT_ACROSS, MM16_OUT_ALONG };   // outputs with B across; with A and B across; with both along k

// Places in a workspace are 256 bytes apart, from its first such boundary on (outputs leave 32 bytes at a time; callers promise 16): what to add to its size.
constexpr size_t MM16_SLACK = 240;
inline unsigned char* mm16_space(void* workspace) { return reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(workspace) + 255) & ~(uintptr_t)255); }
// whether the bytes of a matrix of 16 or fewer bytes a number are far from passing 64 bits
inline bool mm16_size_ok(int64_t rows, int64_t cols) { return cols == 0 || rows <= ((int64_t)1 << 56) / cols; }
inline int64_t mm16_pitch(int64_t n) { return (n + 7) / 8 * 8; }
int mm16_sum_lines(const s2v_ctx* ctx, int64_t m, int64_t n);                     // as the launch will write them
int64_t mm16_sum_lines_most(int64_t n);                                           // the most of any launch
size_t mm16_lines_bytes(int64_t k, int products);                                 // of `lines`; products: of parts, 1, 3 or 6
int mm16_launch(s2v_ctx* ctx, cudaStream_t st, mm16_kind kind, const mm16_args& a);

// Rows of x as 16-bit parts (1 or 3), zeros where a target leaves the row out (target NULL: none); columns up to the next multiple of 8 are filled with zeros.
int mm16_pack(s2v_ctx* ctx, cudaStream_t st, int64_t rows, int64_t cols, int x_type, const void* x, int64_t ldx, const int32_t* target, const float* weight, int64_t vocab, void* out,
              int64_t ldo, int64_t part);

#ifdef __CUDACC__
namespace
{

// The nearest bf16 numbers to two of fp32, the first in the low half; finite ones that lie nearer to infinity than to the type's largest number are cut instead.
__device__ __forceinline__ uint32_t mm16_head(float x, float y)
{
    uint32_t h = pack_16bit<__nv_bfloat16>(x, y);
    if ((h & 0x7fffu) == 0x7f80u && fabsf(x) < INFINITY) h = (h & 0xffff0000u) | __float_as_uint(x) >> 16;
    if ((h & 0x7fff0000u) == 0x7f800000u && fabsf(y) < INFINITY) h = (h & 0xffffu) | (__float_as_uint(y) & 0xffff0000u);
    return h;
}

}  // namespace
#endif
