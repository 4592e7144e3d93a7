// wm_products_capi.hip -- the extern "C" surface of the operators on 16-bit
// weights: argument checks, then the launchers of wm_products.h.  Host code
// only; nothing allocates, waits or keeps state.
#include <hip/hip_runtime.h>
#include <stdint.h>
#include <stdio.h>

#include "../../include/winmoe_hip.h"
#include "wm_host.h"
#include "wm_products.h"

using namespace wm;

namespace {
inline hipStream_t S(void* s) { return (hipStream_t)s; }
inline bool al(const void* p, uintptr_t a) { return (uintptr_t)p % a == 0; }
inline bool dtype_ok(int t) { return t == WM_F16 || t == WM_BF16; }
inline int64_t size_of(int t) { return t == WM_F32 ? 4 : 2; }

// Sizes are bounded so that row and column indexes stay in 32 bits; element
// offsets are 64-bit throughout.
constexpr int kMaxRows = 1 << 30, kMaxDim = 1 << 26, kMaxGroups = 65535;
constexpr int kMaxTokens = (1 << 24) - 1;      // 256 threads for each in one launch
constexpr int64_t kMaxStride = 1ll << 40, kMaxWeights = 1ll << 48;

// What both directions need; 0 when the descriptor is sound.
int check_desc(const wm_product_desc* d) {
    WM_CHECK_ARG(d);
    WM_CHECK_ARG(dtype_ok(d->dtype));
    WM_CHECK_ARG(d->rows >= 0 && d->rows <= kMaxRows && d->x_rows >= 0);
    WM_CHECK_ARG(d->in >= 1 && d->in <= kMaxDim && d->out >= 1 && d->out <= kMaxDim);
    WM_CHECK_ARG(d->n_groups >= 1 && d->n_groups <= kMaxGroups);
    WM_CHECK_ARG(d->offsets || d->n_groups == 1);
    WM_CHECK_ARG(al(d->offsets, 4) && al(d->token, 4));
    WM_CHECK_ARG(d->token || d->x_rows >= d->rows);
    WM_CHECK_ARG(d->ldx >= d->in && d->ldw >= d->in && d->ldx <= kMaxStride && d->ldw <= kMaxStride);
    WM_CHECK_ARG((int64_t)d->in * d->out <= kMaxWeights / d->n_groups);
    WM_CHECK_ARG(d->n_groups == 1 || d->w_stride >= (int64_t)(d->out - 1) * d->ldw + d->in);
    WM_CHECK_ARG(d->act >= WM_ACT_NONE && d->act <= WM_ACT_SIGMOID);
    return WM_OK;
}

// Forward: the operands and the epilogue; 0 when all of it is sound.
int check_forward(const wm_product_desc* d) {
    const bool gated = d->act == WM_ACT_SWIGLU;
    WM_CHECK_ARG(!gated || d->out % 2 == 0);
    WM_CHECK_ARG(d->y_type == d->dtype || d->y_type == WM_F32);
    WM_CHECK_ARG(al(d->x, 2) && al(d->w, 2) && al(d->bias, 2) && al(d->residual, 2) && al(d->pre, 2));
    WM_CHECK_ARG(al(d->y, size_of(d->y_type)));
    const int cols = gated ? d->out / 2 : d->out;
    WM_CHECK_ARG(d->rows == 0 || d->ldy >= cols);
    WM_CHECK_ARG(!d->residual || d->ld_residual >= cols);
    WM_CHECK_ARG(!d->pre || d->ld_pre >= d->out);
    return WM_OK;
}
int check_backward(const wm_product_desc* d) {
    WM_CHECK_ARG(d->act == WM_ACT_NONE);
    WM_CHECK_ARG(al(d->x, 2) && al(d->w, 2) && al(d->dz, 2));
    WM_CHECK_ARG(d->rows == 0 || d->ld_dz >= d->out);
    return WM_OK;
}

ProductArgs arguments(const wm_product_desc* d) {
    ProductArgs a = {};
    a.bf16 = d->dtype == WM_BF16;
    a.rows = d->rows;
    a.in = d->in;
    a.out = d->out;
    a.E = d->n_groups;
    a.x_rows = d->x_rows;
    a.offsets = d->offsets;
    a.token = d->token;
    a.x = (const uint16_t*)d->x;
    a.ldx = d->ldx;
    a.w = (const uint16_t*)d->w;
    a.ldw = d->ldw;
    a.w_stride = d->n_groups > 1 ? d->w_stride : 0;
    a.act = d->act;
    a.bias = (const uint16_t*)d->bias;
    a.res = (const uint16_t*)d->residual;
    a.ldres = d->ld_residual;
    a.y = d->y;
    a.ldy = d->ldy;
    a.y_f32 = d->y_type == WM_F32;
    a.pre = (uint16_t*)d->pre;
    a.ldpre = d->ld_pre;
    a.dz = (const uint16_t*)d->dz;
    a.lddz = d->ld_dz;
    a.split = 1;
    return a;
}
}  // namespace

extern "C" int64_t wm_product_workspace_size(const wm_product_desc* d, int backward) {
    if (int rc = check_desc(d)) return rc;
    if (int rc = backward ? check_backward(d) : check_forward(d)) return rc;
    return product_workspace(arguments(d), backward != 0);
}

extern "C" int wm_product_plan(const wm_product_desc* d, int direction, int* parts) {
    if (int rc = check_desc(d)) return rc;
    WM_CHECK_ARG(direction >= FWD && direction <= DW && parts && d->rows > 0);
    if (int rc = direction == FWD ? check_forward(d) : check_backward(d)) return rc;
    return product_plan(arguments(d), direction, parts);
}

extern "C" int wm_product(const wm_product_desc* d, void* ws, int64_t ws_bytes, void* stream) {
    if (int rc = check_desc(d)) return rc;
    if (int rc = check_forward(d)) return rc;
    if (d->rows == 0) return WM_OK;
    WM_CHECK_ARG(d->x && d->w && d->y);
    const ProductArgs a = arguments(d);
    const int64_t need = product_workspace(a, false);
    WM_CHECK_ARG(need == 0 || (ws && al(ws, 256) && ws_bytes >= need));
    if (wm_init()) return WM_ERR;
    WM_FAIL_HIP(launch_product(a, (uint8_t*)ws, S(stream)));
    return WM_OK;
}

extern "C" int wm_product_backward(const wm_product_desc* d, void* dx, int64_t ld_dx, void* dw, int dw_type, float* db,
                                   void* ws, int64_t ws_bytes, void* stream) {
    if (int rc = check_desc(d)) return rc;
    if (int rc = check_backward(d)) return rc;
    WM_CHECK_ARG(!dw || dw_type == d->dtype || dw_type == WM_F32);
    WM_CHECK_ARG(d->rows == 0 || d->dz);
    WM_CHECK_ARG(!dx || (al(dx, 2) && ld_dx >= d->in && d->w));
    WM_CHECK_ARG((!dw && !db) || d->rows == 0 || d->x);
    WM_CHECK_ARG(al(dw, size_of(dw_type)) && al(db, 4));
    ProductArgs a = arguments(d);
    const int64_t need = product_workspace(a, true);
    WM_CHECK_ARG(need == 0 || (ws && al(ws, 256) && ws_bytes >= need));
    if (wm_init()) return WM_ERR;
    a.dx = (uint16_t*)dx;
    a.lddx = ld_dx;
    a.dw = dw;
    a.dw_f32 = dw_type == WM_F32;
    a.db = db;
    WM_FAIL_HIP(launch_product_backward(a, (uint8_t*)ws, S(stream)));
    return WM_OK;
}

extern "C" int wm_act_backward(int dtype, int act, int64_t rows, int cols, const void* dy, int64_t ld_dy,
                               const void* pre, int64_t ld_pre, void* dz, int64_t ld_dz, void* stream) {
    WM_CHECK_ARG(dtype_ok(dtype));
    WM_CHECK_ARG(act >= WM_ACT_NONE && act <= WM_ACT_SIGMOID);
    WM_CHECK_ARG(rows >= 0 && rows <= kMaxRows && cols >= 1 && cols <= kMaxDim);
    if (rows == 0) return WM_OK;
    const int64_t wide = act == WM_ACT_SWIGLU ? 2 * (int64_t)cols : cols;
    WM_CHECK_ARG(dy && pre && dz && al(dy, 2) && al(pre, 2) && al(dz, 2));
    WM_CHECK_ARG(ld_dy >= cols && ld_pre >= wide && ld_dz >= wide);
    if (wm_init()) return WM_ERR;
    ActArgs a = {};
    a.bf16 = dtype == WM_BF16;
    a.act = act;
    a.rows = rows;
    a.out = cols;
    a.dy = (const uint16_t*)dy;
    a.lddy = ld_dy;
    a.pre = (const uint16_t*)pre;
    a.ldpre = ld_pre;
    a.dz = (uint16_t*)dz;
    a.lddz = ld_dz;
    WM_FAIL_HIP(launch_act_backward(a, S(stream)));
    return WM_OK;
}

extern "C" int wm_group_by_expert(const int32_t* ids, int T, int K, int E, int32_t* offsets, int32_t* token,
                                  int32_t* row, void* stream) {
    WM_CHECK_ARG(T >= 0 && K >= 1 && E >= 1 && E <= kMaxGroups);
    WM_CHECK_ARG((int64_t)T * K < 0x7FFFFFFF - 0xFFFF);
    WM_CHECK_ARG(offsets && al(offsets, 4));
    WM_CHECK_ARG(T == 0 || (ids && token && row && al(ids, 4) && al(token, 4) && al(row, 4)));
    if (wm_init()) return WM_ERR;
    WM_FAIL_HIP(launch_group(ids, T, K, E, offsets, token, row, S(stream)));
    return WM_OK;
}

extern "C" int wm_combine_rows(int dtype, const void* y, int64_t ld_y, int rows, const int32_t* row, const float* w,
                               int T, int K, int H, const void* residual, int64_t ld_residual, void* out,
                               int64_t ld_out, int out_type, void* stream) {
    WM_CHECK_ARG(dtype_ok(dtype) && (out_type == dtype || out_type == WM_F32));
    WM_CHECK_ARG(T >= 0 && T <= kMaxTokens && K >= 0 && rows >= 0 && H >= 1 && H <= kMaxDim && (int64_t)T * K <= 0x7FFFFFFF);
    if (T == 0) return WM_OK;
    WM_CHECK_ARG(out && al(out, size_of(out_type)) && ld_out >= H);
    WM_CHECK_ARG(K == 0 || (row && al(row, 4) && al(w, 4)));
    WM_CHECK_ARG(K == 0 || rows == 0 || (y && al(y, 2) && ld_y >= H));
    WM_CHECK_ARG(!residual || (al(residual, size_of(out_type)) && ld_residual >= H));
    if (wm_init()) return WM_ERR;
    CombineRowsArgs a = {};
    a.bf16 = dtype == WM_BF16;
    a.T = T;
    a.K = K;
    a.H = H;
    a.rows = rows;
    a.row = row;
    a.w = w;
    a.y = (const uint16_t*)y;
    a.ldy = ld_y;
    a.res = residual;
    a.ldres = ld_residual;
    a.out = out;
    a.ldout = ld_out;
    a.out_f32 = out_type == WM_F32;
    WM_FAIL_HIP(launch_combine_rows(a, S(stream)));
    return WM_OK;
}

extern "C" int wm_combine_rows_backward(int dtype, const void* dout, int64_t ld_dout, int dout_type, const void* y,
                                        int64_t ld_y, int rows, const int32_t* row, const float* w, int T, int K,
                                        int H, void* dy, int64_t ld_dy, float* dw, void* stream) {
    WM_CHECK_ARG(dtype_ok(dtype) && (dout_type == dtype || dout_type == WM_F32));
    WM_CHECK_ARG(T >= 0 && K >= 0 && rows >= 0 && H >= 1 && H <= kMaxDim && (int64_t)T * K <= 0x7FFFFFFF);
    WM_CHECK_ARG((int64_t)T * ((K + 4ll) / 5) <= kMaxTokens / 2);
    if (T == 0 || K == 0 || (!dy && !dw)) return WM_OK;
    WM_CHECK_ARG(dout && al(dout, size_of(dout_type)) && ld_dout >= H);
    WM_CHECK_ARG(row && al(row, 4) && al(w, 4) && al(dw, 4));
    WM_CHECK_ARG(!dw || rows == 0 || (y && al(y, 2) && ld_y >= H));
    WM_CHECK_ARG(!dy || (al(dy, 2) && ld_dy >= H));
    if (wm_init()) return WM_ERR;
    CombineRowsArgs a = {};
    a.bf16 = dtype == WM_BF16;
    a.T = T;
    a.K = K;
    a.H = H;
    a.rows = rows;
    a.row = row;
    a.w = w;
    a.y = (const uint16_t*)y;
    a.ldy = ld_y;
    a.out = (void*)dout;
    a.ldout = ld_dout;
    a.out_f32 = dout_type == WM_F32;
    a.dy = (uint16_t*)dy;
    a.lddy = ld_dy;
    a.dw = dw;
    WM_FAIL_HIP(launch_combine_rows_backward(a, S(stream)));
    return WM_OK;
}
