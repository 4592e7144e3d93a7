// wm_products.h -- internal interface between the C-ABI of the 16-bit
// operators (wm_products_capi.hip) and their kernels.  Not part of the public
// ABI.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace wm {

// A product of 16-bit matrices, one per group.  All three directions write
// out[q][p], contiguous along p, summed over a contraction index c:
//   FWD  z[r][n]  = sum_k W_e[n][k] x[r][k]     p = n, q = r, c = k
//   DX   dx[r][k] = sum_n W_e[n][k] dz[r][n]    p = k, q = r, c = n
//   DW   dW[n][k] = sum_r x[r][k] dz[r][n]      p = k, q = n, c = r
// r runs over the rows of group e: offsets[e] <= r < offsets[e + 1].
enum Dir : int { FWD = 0, DX = 1, DW = 2 };

struct ProductArgs {
    int bf16;                   // 16-bit type of every operand: 1 bf16, 0 fp16
    int rows, in, out, E;       // out: rows of one W_e
    int x_rows;                 // rows of x (bound of token[])
    const int32_t* offsets;     // [E + 1], NULL: one group of all rows
    const int32_t* token;       // [rows] row of x of each grouped row, NULL: the row itself
    const uint16_t* x;
    int64_t ldx;
    const uint16_t* w;
    int64_t ldw, w_stride;
    // forward
    int act;
    const uint16_t* bias;       // [E][out]
    const uint16_t* res;
    int64_t ldres;
    void* y;
    int64_t ldy;
    int y_f32;
    uint16_t* pre;
    int64_t ldpre;
    // backward
    const uint16_t* dz;
    int64_t lddz;
    uint16_t* dx;
    int64_t lddx;
    void* dw;                   // [E][out][in], dense
    int dw_f32;
    float* db;                  // [E][out]
    // parts of the contraction: each leaves fp32 sums [split][row][column] (and
    // [split][E * out] of db), which a second kernel adds in order
    int split;                  // 1: none
    float *part, *part_db;
};

// Bytes of workspace that a direction (backward: DX and DW together) uses.
int64_t product_workspace(const ProductArgs& a, bool backward);
// The kernel of a direction (index of WM_PRODUCT_KERNELS) and its parts.
int product_plan(const ProductArgs& a, int dir, int* parts);
// ws holds product_workspace() bytes, 256-byte aligned.
int launch_product(const ProductArgs& a, uint8_t* ws, hipStream_t s);
int launch_product_backward(const ProductArgs& a, uint8_t* ws, hipStream_t s);     // dx, dw, db: those not NULL

int launch_group(const int32_t* ids, int T, int K, int E, int32_t* offsets, int32_t* token, int32_t* row,
                 hipStream_t s);

struct ActArgs {
    int bf16, act;
    int64_t rows;
    int out;                    // outputs per row (SwiGLU: half the columns of pre and dz)
    const uint16_t* dy;
    int64_t lddy;
    const uint16_t* pre;
    int64_t ldpre;
    uint16_t* dz;
    int64_t lddz;
};
int launch_act_backward(const ActArgs& a, hipStream_t s);

struct CombineRowsArgs {
    int bf16;
    int T, K, H;
    int rows;                   // rows of y (bound of row[])
    const int32_t* row;         // [T][K]
    const float* w;             // [T][K], NULL: ones
    const uint16_t* y;
    int64_t ldy;
    const void* res;            // type of out, NULL
    int64_t ldres;
    void* out;
    int64_t ldout;
    int out_f32;
    // backward: out is dout (read)
    uint16_t* dy;
    int64_t lddy;
    float* dw;
};
int launch_combine_rows(const CombineRowsArgs& a, hipStream_t s);
int launch_combine_rows_backward(const CombineRowsArgs& a, hipStream_t s);

}  // namespace wm
