// wm_pairs.hip -- the (token, pick) pairs around the grouped products: sorting
// them by expert, the weighted sum over a token's picks with its gradients,
// and the gradient of an activation.  All are bound by memory or by latency;
// values are 16 bits in memory and fp32 in registers, each result rounded once.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "wm_act.h"
#include "wm_products.h"

namespace wm {

// ------------------------------------------------------------------ grouping

// Stable counting sort of n = T * K ids, one workgroup per expert and no
// workspace: expert e's rows begin at the number of valid ids below e, which
// the workgroup counts itself.  The ids are a few hundred KB at most and are
// read from the caches.  Each of the 16 waves owns a contiguous part of the
// ids; it counts ids below e and equal to e, the waves exchange their counts
// once, and a second pass writes the places of the equal ones in order.
// Workgroup E takes the ids outside [0, E): their rows follow the last group.
constexpr int GRP_WAVES = 16;
__global__ __launch_bounds__(64 * GRP_WAVES) void k_group(const int32_t* __restrict__ ids, int n, int K, int E,
                                                          int32_t* __restrict__ offsets, int32_t* __restrict__ token,
                                                          int32_t* __restrict__ row) {
    __shared__ int cnt[2][GRP_WAVES];
    const int e = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int seg = (n + GRP_WAVES - 1) / GRP_WAVES, i0 = min(wave * seg, n), i1 = min(i0 + seg, n);
    int below = 0, equal = 0;
    for (int i = i0 + lane; i < i1; i += 64) {
        const int v = ids[i];
        const int id = (uint32_t)v < (uint32_t)E ? v : E;
        below += id < e;
        equal += id == e;
    }
#pragma unroll
    for (int d = 32; d; d >>= 1) {
        below += __shfl_xor(below, d);
        equal += __shfl_xor(equal, d);
    }
    if (lane == 0) {
        cnt[0][wave] = below;
        cnt[1][wave] = equal;
    }
    __syncthreads();
    int at = 0, all = 0;
    for (int w = 0; w < GRP_WAVES; w++) {
        at += cnt[0][w] + (w < wave ? cnt[1][w] : 0);
        all += cnt[0][w];
    }
    if (threadIdx.x == 0) offsets[e] = all;
    for (int i = i0; i < i1; i += 64) {
        const int v = i + lane < i1 ? ids[i + lane] : 0;
        const bool mine = i + lane < i1 && ((uint32_t)v < (uint32_t)E ? v : E) == e;
        const uint64_t m = __ballot(mine);
        if (mine) {
            const int r = at + __popcll(m & ((1ull << lane) - 1));
            row[i + lane] = e < E ? r : -1;
            token[r] = e < E ? (i + lane) / K : -1;
        }
        at += __popcll(m);
    }
}

int launch_group(const int32_t* ids, int T, int K, int E, int32_t* offsets, int32_t* token, int32_t* row,
                 hipStream_t s) {
    hipLaunchKernelGGL(k_group, dim3(E + 1), dim3(64 * GRP_WAVES), 0, s, ids, T * K, K, E, offsets, token, row);
    return (int)hipGetLastError();
}

// ------------------------------------------------------------------ activation

// dz = act'(pre) * dy; SwiGLU's pre and dz hold the gate half, then the up
// half: dg = dy u silu'(g), du = dy silu(g).  One thread per 8 outputs.
template <bool BF> __global__ __launch_bounds__(256) void k_act_backward(const ActArgs a) {
    const uint32_t per = (a.out + 7) / 8;
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, r = i / per;
    if (r >= a.rows) return;
    const int c = (int)(i - r * per) * 8, n = a.out - c;
    float dy[8], z[8], dz[8];
    get8<BF>(a.dy + r * a.lddy + c, n, dy);
    get8<BF>(a.pre + r * a.ldpre + c, n, z);
    if (a.act == WM_ACT_SWIGLU) {
        float u[8], du[8];
        get8<BF>(a.pre + r * a.ldpre + a.out + c, n, u);
#pragma unroll
        for (int k = 0; k < 8; k++) {
            dz[k] = dy[k] * u[k] * act_slope(WM_ACT_SILU, z[k]);
            du[k] = dy[k] * act_value(WM_ACT_SILU, z[k], 1.0f);
        }
        put8<BF>(a.dz + r * a.lddz + a.out + c, n, du);
    } else {
#pragma unroll
        for (int k = 0; k < 8; k++) dz[k] = dy[k] * act_slope(a.act, z[k]);
    }
    put8<BF>(a.dz + r * a.lddz + c, n, dz);
}

int launch_act_backward(const ActArgs& a, hipStream_t s) {
    const int64_t blocks = (a.rows * ((a.out + 7) / 8) + 255) / 256;
    if (blocks == 0) return 0;
    if (blocks > 0x7FFFFFFF) return (int)hipErrorInvalidConfiguration;
    if (a.bf16) hipLaunchKernelGGL(HIP_KERNEL_NAME(k_act_backward<true>), dim3((uint32_t)blocks), dim3(256), 0, s, a);
    else hipLaunchKernelGGL(HIP_KERNEL_NAME(k_act_backward<false>), dim3((uint32_t)blocks), dim3(256), 0, s, a);
    return (int)hipGetLastError();
}

// ------------------------------------------------------------------ combine

// out[t] = sum_k w[t][k] * y[row[t][k]] + res[t], k in order; a row outside
// [0, rows) counts as zeros.  One thread per 8 columns of a token.
template <bool BF> __global__ __launch_bounds__(256) void k_combine_rows(const CombineRowsArgs a) {
    const int t = blockIdx.x, c = (blockIdx.y * 256 + threadIdx.x) * 8, n = a.H - c;
    if (n <= 0) return;
    float s[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    if (a.res) {
        const int64_t at = (int64_t)t * a.ldres + c;
        if (a.out_f32) getf8((const float*)a.res + at, n, s);
        else get8<BF>((const uint16_t*)a.res + at, n, s);
    }
    for (int k = 0; k < a.K; k++) {
        const int r = a.row[(int64_t)t * a.K + k];
        if ((uint32_t)r >= (uint32_t)a.rows) continue;
        const float w = a.w ? a.w[(int64_t)t * a.K + k] : 1.0f;
        float v[8];
        get8<BF>(a.y + (int64_t)r * a.ldy + c, n, v);
#pragma unroll
        for (int i = 0; i < 8; i++) s[i] = fmaf(w, v[i], s[i]);
    }
    const int64_t at = (int64_t)t * a.ldout + c;
    if (a.out_f32) putf8((float*)a.out + at, n, s);
    else put8<BF>((uint16_t*)a.out + at, n, s);
}

int launch_combine_rows(const CombineRowsArgs& a, hipStream_t s) {
    if (a.T == 0 || a.H == 0) return 0;
    const dim3 grid(a.T, (a.H + 2047) / 2048);
    if (a.bf16) hipLaunchKernelGGL(HIP_KERNEL_NAME(k_combine_rows<true>), grid, dim3(256), 0, s, a);
    else hipLaunchKernelGGL(HIP_KERNEL_NAME(k_combine_rows<false>), grid, dim3(256), 0, s, a);
    return (int)hipGetLastError();
}

// dy[row[t][k]] = w[t][k] * dout[t] and dw[t][k] = <dout[t], y[row[t][k]]>:
// one wave per pair.  Rows that no pair names are not written.
template <bool BF> __global__ __launch_bounds__(256) void k_combine_rows_backward(const CombineRowsArgs a) {
    const int64_t pair = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    const int lane = threadIdx.x & 63;
    if (pair >= (int64_t)a.T * a.K) return;
    const int t = (int)(pair / a.K), r = a.row[pair];
    if ((uint32_t)r >= (uint32_t)a.rows) {
        if (a.dw && lane == 0) a.dw[pair] = 0.0f;
        return;
    }
    const float w = a.w ? a.w[pair] : 1.0f;
    float dot = 0.0f;
    for (int c = lane * 8; c < a.H; c += 512) {
        const int n = a.H - c;
        const int64_t at = (int64_t)t * a.ldout + c;
        float g[8], v[8];
        if (a.out_f32) getf8((const float*)a.out + at, n, g);
        else get8<BF>((const uint16_t*)a.out + at, n, g);
        if (a.dw) {
            get8<BF>(a.y + (int64_t)r * a.ldy + c, n, v);
#pragma unroll
            for (int i = 0; i < 8; i++) dot = fmaf(g[i], v[i], dot);
        }
        if (a.dy) {
#pragma unroll
            for (int i = 0; i < 8; i++) g[i] *= w;
            put8<BF>(a.dy + (int64_t)r * a.lddy + c, n, g);
        }
    }
    if (a.dw) {
#pragma unroll
        for (int d = 32; d; d >>= 1) dot += __shfl_xor(dot, d);
        if (lane == 0) a.dw[pair] = dot;
    }
}

int launch_combine_rows_backward(const CombineRowsArgs& a, hipStream_t s) {
    const int64_t blocks = ((int64_t)a.T * a.K + 3) / 4;
    if (blocks == 0) return 0;
    if (a.bf16) hipLaunchKernelGGL(HIP_KERNEL_NAME(k_combine_rows_backward<true>), dim3((uint32_t)blocks), dim3(256), 0, s, a);
    else hipLaunchKernelGGL(HIP_KERNEL_NAME(k_combine_rows_backward<false>), dim3((uint32_t)blocks), dim3(256), 0, s, a);
    return (int)hipGetLastError();
}

}  // namespace wm
