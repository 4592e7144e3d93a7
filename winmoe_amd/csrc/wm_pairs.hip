// wm_pairs.hip -- the (token, pick) pairs around the grouped products: sorting
// them by expert, the weighted sum over a token's picks with its gradients,
// and the gradient of an activation.  All are bound by memory or by latency;
// values are 16 bits in memory and fp32 in registers, each result rounded once.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <type_traits>

#include "wm_act.h"
#include "wm_products.h"

namespace wm {

// ------------------------------------------------------------------ grouping

// Stable counting sort of n = T * K ids in one launch and without workspace or
// atomics: a workgroup takes EP neighbouring experts, whose rows begin at the
// number of valid ids below the first, which it counts itself.  The ids are
// read from the caches, twice by every workgroup; each of its 16 waves owns a
// contiguous part of them, counts, exchanges its counts once and then writes
// the places of its experts' ids in order.  The experts are 0 .. E, the last
// one standing for the ids outside [0, E): their rows follow the last group.
//
// Bound by latency: two rounds of loads, one exchange.  512 experts: 10 ids
// 3.9 us, 5120 ids 5.9 us, 40960 ids 12.9 us in a graph, of which about 2.4 us
// is the launch; one id per lane and load and one expert per workgroup took
// 4.7, 7.6 and 29.6 us.
constexpr int GRP_WAVES = 16;
template <int EP> __global__ __launch_bounds__(64 * GRP_WAVES) void k_group(const int32_t* __restrict__ ids, int n, int K, int E,
                                                                            int32_t* __restrict__ offsets, int32_t* __restrict__ token,
                                                                            int32_t* __restrict__ row) {
    __shared__ int cnt[1 + EP][GRP_WAVES];
    const int e0 = blockIdx.x * EP, lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    // parts are multiples of 4 ids, so that only the last one ends within 4
    const int seg = (n + 4 * GRP_WAVES - 1) / (4 * GRP_WAVES) * 4, i0 = min(wave * seg, n), i1 = min(i0 + seg, n);
    typedef int ids4 __attribute__((ext_vector_type(4), aligned(4)));
    // the wave's ids in order, 4 per lane and 256 at a time, up to 4 loads in
    // flight; -1 behind the end, which no expert has
    auto each = [&](auto use) __attribute__((always_inline)) {
        auto group = [&](int i, auto count) __attribute__((always_inline)) {
            constexpr int N = decltype(count)::value;
            ids4 v[N];
#pragma unroll
            for (int b = 0; b < N; b++) v[b] = *(const ids4*)(ids + i + 256 * b + 4 * lane);
#pragma unroll
            for (int b = 0; b < N; b++) {
#pragma unroll
                for (int c = 0; c < 4; c++) v[b][c] = (uint32_t)v[b][c] < (uint32_t)E ? v[b][c] : E;
                use(v[b], i + 256 * b + 4 * lane);
            }
        };
        int i = i0;
        for (; i + 1024 <= i1; i += 1024) group(i, std::integral_constant<int, 4>());
        for (; i + 256 <= i1; i += 256) group(i, std::integral_constant<int, 1>());
        if (i < i1) {
            ids4 v;
#pragma unroll
            for (int c = 0; c < 4; c++) {
                const int p = i + 4 * lane + c, id = p < i1 ? ids[p] : -1;
                v[c] = (uint32_t)id < (uint32_t)E ? id : p < i1 ? E : -1;
            }
            use(v, i + 4 * lane);
        }
    };
    int below = 0, equal[EP];
#pragma unroll
    for (int k = 0; k < EP; k++) equal[k] = 0;
    each([&](const ids4& v, int) __attribute__((always_inline)) {
#pragma unroll
        for (int c = 0; c < 4; c++) {
            below += (uint32_t)v[c] < (uint32_t)e0;
#pragma unroll
            for (int k = 0; k < EP; k++) equal[k] += v[c] == e0 + k;
        }
    });
#pragma unroll
    for (int d = 32; d; d >>= 1) {
        below += __shfl_xor(below, d);
#pragma unroll
        for (int k = 0; k < EP; k++) equal[k] += __shfl_xor(equal[k], d);
    }
    if (lane == 0) {
        cnt[0][wave] = below;
#pragma unroll
        for (int k = 0; k < EP; k++) cnt[1 + k][wave] = equal[k];
    }
    __syncthreads();
    int at[EP], start = 0, any = 0;
    for (int w = 0; w < GRP_WAVES; w++) start += cnt[0][w];
#pragma unroll
    for (int k = 0; k < EP; k++) {
        if (threadIdx.x == 0 && e0 + k <= E) offsets[e0 + k] = start;
        at[k] = start;
        for (int w = 0; w < GRP_WAVES; w++) {
            at[k] += w < wave ? cnt[1 + k][w] : 0;
            start += cnt[1 + k][w];
        }
        any += cnt[1 + k][wave];
    }
    if (any == 0) return;
    const uint64_t lower = (1ull << lane) - 1;
    each([&](const ids4& v, int i) __attribute__((always_inline)) {
#pragma unroll
        for (int k = 0; k < EP; k++) {
            if (!__ballot(v[0] == e0 + k || v[1] == e0 + k || v[2] == e0 + k || v[3] == e0 + k)) continue;
            uint64_t m[4];
            int before = 0;             // of the lower lanes
#pragma unroll
            for (int c = 0; c < 4; c++) {
                m[c] = __ballot(v[c] == e0 + k);
                before += __popcll(m[c] & lower);
            }
#pragma unroll
            for (int c = 0; c < 4; c++)
                if (v[c] == e0 + k) {
                    const int r = at[k] + before++, p = i + c;
                    row[p] = e0 + k < E ? r : -1;
                    token[r] = e0 + k < E ? p / K : -1;
                }
            at[k] += __popcll(m[0]) + __popcll(m[1]) + __popcll(m[2]) + __popcll(m[3]);
        }
    });
}

int launch_group(const int32_t* ids, int T, int K, int E, int32_t* offsets, int32_t* token, int32_t* row,
                 hipStream_t s) {
    // with many ids for many experts, half as many workgroups read half as much
    const int n = T * K, per = n >= 1024 && E >= 384 ? 2 : 1;
    const auto k = per == 2 ? k_group<2> : k_group<1>;
    hipLaunchKernelGGL(k, dim3((E + per) / per), dim3(64 * GRP_WAVES), 0, s, ids, n, K, E, offsets, token, row);
    return (int)hipGetLastError();
}

// ------------------------------------------------------------------ activation

// dz = act'(pre) * dy; SwiGLU's pre and dz hold the gate half, then the up
// half: dg = dy u silu'(g), du = dy silu(g).  One thread per 8 outputs, one pass:
// bound by memory, SwiGLU over 16384 x 1024 31.0 us, 5.4 TB/s.
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
    if (blocks > 0xFFFFFFFFll / 256) return (int)hipErrorInvalidConfiguration;       // a launch holds fewer than 2^32 threads
    if (a.bf16) hipLaunchKernelGGL(HIP_KERNEL_NAME(k_act_backward<true>), dim3((uint32_t)blocks), dim3(256), 0, s, a);
    else hipLaunchKernelGGL(HIP_KERNEL_NAME(k_act_backward<false>), dim3((uint32_t)blocks), dim3(256), 0, s, a);
    return (int)hipGetLastError();
}

// ------------------------------------------------------------------ combine

// out[t] = sum_k w[t][k] * y[row[t][k]] + res[t], k in order; a row outside
// [0, rows) counts as zeros.  One thread per 8 columns of a token, the rows of
// CR picks in flight.  Bound by memory: 512 x 10 x 4096 with an fp32 residual
// 10.4 us; 4096 x 10 x 4096 80 us, 103 us where rows were converted as they came.
constexpr int CR = 5;
template <bool BF> __global__ __launch_bounds__(256) void k_combine_rows(const CombineRowsArgs a) {
    const int t = blockIdx.x, c = (blockIdx.y * 256 + threadIdx.x) * 8, n = a.H - c;
    if (n <= 0) return;
    const int32_t* rows = a.row + (int64_t)t * a.K;
    const float* ws = a.w ? a.w + (int64_t)t * a.K : nullptr;
    float s[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    if (a.res) {
        const int64_t at = (int64_t)t * a.ldres + c;
        if (a.out_f32) getf8((const float*)a.res + at, n, s);
        else get8<BF>((const uint16_t*)a.res + at, n, s);
    }
    for (int k0 = 0; k0 < a.K; k0 += CR) {
        uint4 raw[CR];                  // converted behind all loads
        float w[CR], v[8];
        bool live[CR];
#pragma unroll
        for (int j = 0; j < CR; j++) {
            const int r = k0 + j < a.K ? rows[k0 + j] : -1;
            live[j] = (uint32_t)r < (uint32_t)a.rows;
            w[j] = live[j] && ws ? ws[k0 + j] : 1.0f;
            if (live[j]) raw[j] = load8(a.y + (int64_t)r * a.ldy + c, n);
        }
#pragma unroll
        for (int j = 0; j < CR; j++)
            if (live[j]) {
                unpack8<BF>(raw[j], v);
#pragma unroll
                for (int i = 0; i < 8; i++) s[i] = fmaf(w[j], v[i], s[i]);
            }
    }
    const int64_t at = (int64_t)t * a.ldout + c;
    if (a.out_f32) putf8((float*)a.out + at, n, s);
    else put8<BF>((uint16_t*)a.out + at, n, s);
}

int launch_combine_rows(const CombineRowsArgs& a, hipStream_t s) {
    if (a.T == 0 || a.H == 0) return 0;
    if (a.T > 0xFFFFFFFFll / 256) return (int)hipErrorInvalidConfiguration;
    const dim3 grid(a.T, (a.H + 2047) / 2048);
    if (a.bf16) hipLaunchKernelGGL(HIP_KERNEL_NAME(k_combine_rows<true>), grid, dim3(256), 0, s, a);
    else hipLaunchKernelGGL(HIP_KERNEL_NAME(k_combine_rows<false>), grid, dim3(256), 0, s, a);
    return (int)hipGetLastError();
}

// dy[row[t][k]] = w[t][k] * dout[t] and dw[t][k] = <dout[t], y[row[t][k]]>: a
// workgroup takes CB picks of a token, so that dout[t] is read once for them
// and their rows are in flight together.  Rows that no pick names are not
// written.  Bound by memory: 4096 x 10 x 4096 158 us, 4.4 TB/s; one pick per
// workgroup took 235 us.
constexpr int CB = 5;
template <bool BF> __global__ __launch_bounds__(512) void k_combine_rows_backward(const CombineRowsArgs a, int per) {
    __shared__ float sums[8][CB];
    const int t = blockIdx.x / per, k0 = (int)(blockIdx.x % per) * CB, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t pair = (int64_t)t * a.K + k0;
    int r[CB];
    bool live[CB];
    float w[CB], dot[CB];
#pragma unroll
    for (int j = 0; j < CB; j++) {
        r[j] = k0 + j < a.K ? a.row[pair + j] : -1;
        live[j] = (uint32_t)r[j] < (uint32_t)a.rows;
        w[j] = live[j] && a.w ? a.w[pair + j] : 1.0f;
        dot[j] = 0.0f;
    }
    for (int c = threadIdx.x * 8; c < a.H; c += blockDim.x * 8) {
        const int n = a.H - c;
        const int64_t at = (int64_t)t * a.ldout + c;
        float g[8], v[8];
        uint4 raw[CB];                  // converted behind all loads
        if (a.dw)
#pragma unroll
            for (int j = 0; j < CB; j++)
                if (live[j]) raw[j] = load8(a.y + (int64_t)r[j] * a.ldy + c, n);
        if (a.out_f32) getf8((const float*)a.out + at, n, g);
        else get8<BF>((const uint16_t*)a.out + at, n, g);
        if (a.dw)
#pragma unroll
            for (int j = 0; j < CB; j++)
                if (live[j]) {
                    unpack8<BF>(raw[j], v);
#pragma unroll
                    for (int i = 0; i < 8; i++) dot[j] = fmaf(g[i], v[i], dot[j]);
                }
        if (a.dy)
#pragma unroll
            for (int j = 0; j < CB; j++)
                if (live[j]) {
                    float d[8];
#pragma unroll
                    for (int i = 0; i < 8; i++) d[i] = w[j] * g[i];
                    put8<BF>(a.dy + (int64_t)r[j] * a.lddy + c, n, d);
                }
    }
    if (!a.dw) return;
#pragma unroll
    for (int j = 0; j < CB; j++) {
        float v = dot[j];
        v += dpp_f32<DPP_XOR1>(v);
        v += dpp_f32<DPP_XOR2>(v);
        v += dpp_f32<DPP_HALF_MIRROR>(v);
        v += dpp_f32<DPP_MIRROR>(v);
        v += __shfl_xor(v, 16);
        v += __shfl_xor(v, 32);
        if (lane == 0) sums[wave][j] = v;
    }
    __syncthreads();
    const int j = threadIdx.x;
    if (j < CB && k0 + j < a.K) {
        float v = 0.0f;
        for (int i = 0; i < (int)blockDim.x / 64; i++) v += sums[i][j];
        a.dw[pair + j] = v;
    }
}

int launch_combine_rows_backward(const CombineRowsArgs& a, hipStream_t s) {
    const int per = (a.K + CB - 1) / CB;
    const int64_t blocks = (int64_t)a.T * per;
    if (blocks == 0) return 0;
    if (blocks > 0xFFFFFFFFll / 512) return (int)hipErrorInvalidConfiguration;
    const auto k = a.bf16 ? k_combine_rows_backward<true> : k_combine_rows_backward<false>;
    // 8 columns per thread: a row of up to 4096 in one go
    hipLaunchKernelGGL(k, dim3((uint32_t)blocks), dim3(a.H > 2048 ? 512 : 256), 0, s, a, per);
    return (int)hipGetLastError();
}

}  // namespace wm
