// linear_loss.cuh — the projection to the vocabulary with its cross entropy: what its kernels share.
//
// hidden H [n, D] and weight W [V, D] give logits z = H W^T, never kept as such. With lse_r = log sum_v exp(z_rv / T)
//     row_loss_r = lse_r - z_rt / T + c lse_r^2,      loss = sum_r w_r row_loss_r
//     G_rv = w_r / T (p_rv (1 + 2 c lse_r) - 1[v = t]),   dH = G W,   dW = G^T H
// so a step is three products of 2 n V D operations each. The rows that count (w_r != 0) are put together first,
// so rows that do not are neither computed nor read, and taken in blocks: for the rows of a block the exponentials of
// every piece of the vocabulary (a tile's columns) are held between the first product and the other two.
#pragma once

#include "rows.cuh"

namespace ctb {

enum LinearRow : int { kLnHidden = 0, kLnGrad, kLnTarget, kLnWeight, kLnRowLoss, kLnLse, kLnViews };

// Device-side facts of a call, written by linear_order (or known before it).
struct LinearFacts {
    int32_t count;   // rows that count
    float wmax;      // the largest finite |weight| among them, 0 without any
};

struct LinearRowFactor {  // what turns a row's held exponentials into its G (bfloat16)
    float m, c, at_target;
    int32_t target;
};

struct Matrix2 {  // a matrix of a call's own, or an operand: element (i, j) at ptr[i * row + j * col]
    void* ptr;
    int64_t row, col;
    int32_t dtype;
};

struct LinearArgs {
    RowViews<kLnViews> v;  // rows and cols (D) of hidden
    int64_t vocab;
    Matrix2 weight, grad_weight;
    double scale, inv_temp, z_coef;
    float c2;  // log2(e) / T
    // scratch
    LinearFacts* facts;
    int32_t* order;    // [rows] the rows that count in their order, then the others
    double* weighted;  // [rows] w_r row_loss_r, by row
    float* target_z;   // [block] z_rt
    float2* stats;     // [block][tiles] bfloat16: (maximum, sum of exponentials) of every 128 columns
    void* held;        // [block][held_pitch] float32 logits or 16-bit exponentials of a block, then G
    int64_t held_pitch;
    int64_t tiles;     // pieces of 128 columns
    LinearRowFactor* factors;  // [block]
    float* partial;    // [splits][part_rows][part_pitch]
    int64_t part_rows, part_pitch;
    float* acc;        // [V][acc_pitch] dW over the blocks so far, where there are several
    int64_t acc_pitch;
    Matrix2 h, w;      // what the products read: the operands, or packed copies
    int64_t block;     // rows a block
    int splits;
    int32_t* status;
    unsigned long long* timeouts;
};

// The rows of block `b` that count.
__device__ __forceinline__ int64_t linear_block_rows(const LinearArgs& a, int64_t first) {
    const int64_t n = static_cast<int64_t>(a.facts->count) - first;
    return n < 0 ? 0 : n < a.block ? n : a.block;
}

// What G is divided by so that the usual weights (one value, or 0) leave its target entries at exactly -1: bfloat16
// keeps 8 bits of them, and the same rounding in every row would not average out. The float32 path uses it too.
__device__ __forceinline__ double linear_factor(const LinearArgs& a) {
    const float w = a.order ? a.facts->wmax : 1.0f;
    return a.scale * a.inv_temp * (w == 0.0f ? 1.0 : static_cast<double>(w));
}

// The products of rows [first, first + rows) of those that count: z, dH (in splits), dW.
int linear_logits_f32(const LinearArgs& a, int64_t first, int64_t rows, cudaStream_t st);             // linear_loss_f32.cu
int linear_grad_hidden_f32(const LinearArgs& a, int64_t first, int64_t rows, cudaStream_t st);        // linear_loss_f32.cu
int linear_grad_weight_f32(const LinearArgs& a, int64_t first, int64_t rows, bool last, cudaStream_t st);  // linear_loss_f32.cu

int linear_logits_tc(const LinearArgs& a, int64_t first, int64_t rows, bool hold, cudaStream_t st);      // linear_loss_tc.cu
int linear_grad_hidden_tc(const LinearArgs& a, int64_t first, int64_t rows, cudaStream_t st);         // linear_loss_tc.cu
int linear_grad_weight_tc(const LinearArgs& a, int64_t first, int64_t rows, bool last, cudaStream_t st);  // linear_loss_tc.cu

constexpr int kLinearPiece = 128;  // columns of logits that share a maximum in bfloat16's held exponentials

}  // namespace ctb
