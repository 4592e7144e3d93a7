// wm_products.hip -- products of 16-bit matrices, plain and grouped by expert:
// forward (bias, activation and residual in the epilogue), gradient of the
// input and gradient of the matrices.
//
// One tile kernel serves the three directions (wm_products.h).  A workgroup
// sums a BP x BQ tile of out[q][p] over the contraction index with
// v_mfma_f32_16x16x32: the p operand gives the rows of the result, so a lane
// holds 4 consecutive outputs of one row.  Products of 16-bit values are exact
// in fp32 and every sum is kept in fp32; a result is rounded once, when it is
// stored.
//
// An operand whose memory rows run along the contraction (x and W forward, dz
// for dx) is kept in LDS as [index][64], the others (W for dx, x and dz for
// dW: rows are contraction steps) as [64][index] and read through the
// transposing LDS load.  16-byte chunks are permuted within a row so that the
// lanes of a read fall on different banks.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "../../include/winmoe_hip.h"
#include "wm_act.h"
#include "wm_device.h"
#include "wm_products.h"

namespace wm {

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

constexpr int BK = 64;          // contraction steps staged at once

template <bool BF> WM_DEV f32x4 mfma(s16x8 a, s16x8 b, f32x4 c) {
    if constexpr (BF) return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// 8 values at p, of which the first n exist; the others are zero.  p needs no
// alignment beyond its type's.
WM_DEV uint4 load8(const uint16_t* p, int n) {
    uint4 v = {0, 0, 0, 0};
    if (n >= 8) {
        __builtin_memcpy(&v, p, 16);
    } else {
        uint16_t e[8];
#pragma unroll
        for (int i = 0; i < 8; i++) e[i] = i < n ? p[i] : 0;
        __builtin_memcpy(&v, e, 16);
    }
    return v;
}

// Workgroup's group: `qt` counts the tiles of BQ rows over all groups.
// Offsets are clamped to [0, rows], so whatever they hold no row outside is
// touched.  Every wave looks it up by itself.
struct GroupTile {
    int e, start, n, tile;      // e < 0: past the last tile
};
WM_DEV GroupTile find_tile(const int32_t* __restrict__ offsets, int E, int rows, int bq, int qt) {
    GroupTile g{-1, 0, 0, 0};
    if (!offsets) {
        g.e = qt * bq < rows ? 0 : -1;
        g.n = rows;
        g.tile = qt;
        return g;
    }
    const int lane = threadIdx.x & 63;
    int before = 0;
    for (int e0 = 0; e0 < E; e0 += 64) {
        const int e = e0 + lane;
        const int a = e < E ? min(max(offsets[e], 0), rows) : 0;
        const int b = e < E ? min(max(offsets[e + 1], a), rows) : 0;
        const int t = (b - a + bq - 1) / bq;
        int sum = t;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const int v = __shfl_up(sum, d);
            if (lane >= d) sum += v;
        }
        const uint64_t hit = __ballot(before + sum > qt);
        if (hit) {
            const int l = __builtin_ctzll(hit);
            g.e = e0 + l;
            g.start = __builtin_amdgcn_readlane(a, l);
            g.n = __builtin_amdgcn_readlane(b, l) - g.start;
            g.tile = qt - (before + __builtin_amdgcn_readlane(sum, l) - __builtin_amdgcn_readlane(t, l));
            return g;
        }
        before += __builtin_amdgcn_readlane(sum, 63);
    }
    return g;
}

// ------------------------------------------------------------------ LDS tiles

// [TILE][64], memory rows along the contraction.  Slot s (16 bytes) holds
// chunk (s & 7) ^ (index & 7) of row index = s >> 3.
template <int TILE> struct AlongC {
    WM_DEV static void slot(int s, int& index, int& c) {
        index = s >> 3;
        c = 8 * ((s & 7) ^ (index & 7));
    }
    // operand of 16 indices from `base` on, 32 contraction steps from 32 * ks on
    WM_DEV static s16x8 frag(const lds8_t* t, int base, int ks, int lane) {
        const int i = base + (lane & 15), ch = (4 * ks + (lane >> 4)) ^ (lane & 7);
        return *(const __attribute__((address_space(3))) s16x8*)(t + 128 * i + 16 * ch);
    }
};

// [64][TILE], memory rows are contraction steps.  Units of 16 values are
// permuted within a row by the row's bits 0, 1 and 3, which the 16 rows of a
// transposing read run through.
template <int TILE> struct AcrossC {
    static constexpr int CH = TILE / 8, U = TILE / 16;
    WM_DEV static int perm(int c) { return ((c & 3) | ((c >> 1) & 4)) & (U - 1); }
    WM_DEV static void slot(int s, int& index, int& c) {
        c = s / CH;
        const int pos = s % CH;
        index = 16 * ((pos >> 1) ^ perm(c)) + 8 * (pos & 1);
    }
    WM_DEV static s16x8 frag(const lds8_t* t, int base, int ks, int lane) {
        const int g = lane >> 4, j = lane & 15, c = 32 * ks + 8 * g + (j >> 2);
        const lds8_t* p = t + 2 * TILE * c + 32 * ((base >> 4) ^ perm(c)) + 8 * (j & 3);
        typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
        const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)p);
        const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(p + 8 * TILE));
        return (s16x8){lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
    }
};

// ------------------------------------------------------------------ epilogue

template <bool BF> WM_DEV void store4(void* base, int64_t at, int f32, bool vec, int n, f32x4 v) {
    if (f32) {
        float* p = (float*)base + at;
        if (vec && n >= 4) *(f32x4*)p = v;
        else
#pragma unroll
            for (int i = 0; i < 4; i++)
                if (i < n) p[i] = v[i];
    } else {
        uint16_t* p = (uint16_t*)base + at;
        if (vec && n >= 4) {
            *(uint2*)p = (uint2){to16<BF>(v[0]) | (uint32_t)to16<BF>(v[1]) << 16, to16<BF>(v[2]) | (uint32_t)to16<BF>(v[3]) << 16};
        } else {
#pragma unroll
            for (int i = 0; i < 4; i++)
                if (i < n) p[i] = to16<BF>(v[i]);
        }
    }
}

template <bool BF> WM_DEV f32x4 load4(const uint16_t* p, int n) {
    f32x4 v;
#pragma unroll
    for (int i = 0; i < 4; i++) v[i] = i < n ? from16<BF>(p[i]) : 0.0f;
    return v;
}

// z (and for SwiGLU the up half u) of outputs [p, p + 4) of row q.
template <bool BF> WM_DEV void store_forward(const ProductArgs& a, int e, int q, int p, int outs, bool vec, f32x4 z, f32x4 u) {
    const int n = outs - p;
    if (n <= 0) return;
    const bool gated = a.act == WM_ACT_SWIGLU;
    if (a.bias) {
        const uint16_t* b = a.bias + (int64_t)e * a.out;
        z += load4<BF>(b + p, n);
        if (gated) u += load4<BF>(b + outs + p, n);
    }
    if (a.pre) {
        store4<BF>(a.pre, (int64_t)q * a.ldpre + p, 0, false, n, z);
        if (gated) store4<BF>(a.pre, (int64_t)q * a.ldpre + outs + p, 0, false, n, u);
    }
#pragma unroll
    for (int i = 0; i < 4; i++) z[i] = act_value(a.act, z[i], u[i]);
    if (a.res) z += load4<BF>((const uint16_t*)a.res + (int64_t)q * a.ldres + p, n);
    store4<BF>(a.y, (int64_t)q * a.ldy + p, a.y_f32, vec, n, z);
}

// ------------------------------------------------------------------ the tile kernel

// WP x WQ waves, each a (BP / WP) x (BQ / WQ) part of the tile.  Two LDS
// buffers: the chunks of the next 64 steps are loaded into registers while
// this buffer's products run, then stored into the other one.
template <bool BF, int DIR, int BP, int BQ, int WP, int WQ>
__global__ __launch_bounds__(64 * WP * WQ) void k_product(const ProductArgs a) {
    constexpr int NT = 64 * WP * WQ, FP = BP / WP / 16, FQ = BQ / WQ / 16;
    constexpr bool PC = DIR == FWD, QC = DIR != DW;         // operand's rows run along the contraction
    using PT = typename std::conditional<PC, AlongC<BP>, AcrossC<BP>>::type;
    using QT = typename std::conditional<QC, AlongC<BQ>, AcrossC<BQ>>::type;
    constexpr int PS = BP * 8, QS = BQ * 8, NP = (PS + NT - 1) / NT, NQ = (QS + NT - 1) / NT;
    __shared__ __attribute__((aligned(16))) uint8_t lds[2][(BP + BQ) * 2 * BK];

    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wp = wave % WP, wq = wave / WP;
    const bool gated = DIR == FWD && a.act == WM_ACT_SWIGLU;
    const int outs = DIR == FWD ? (gated ? a.out / 2 : a.out) : a.in;       // extent of p in the result
    const int cols = gated ? BP / 2 : BP;
    const int nP = (outs + cols - 1) / cols;
    const int p0 = (int)(blockIdx.x % nP) * cols;
    int e, q0, qn, c0 = 0, cn;
    const uint16_t* w;
    if (DIR == DW) {
        const int nQ = (a.out + BQ - 1) / BQ, t = blockIdx.x / nP;
        e = t / nQ;
        q0 = (t % nQ) * BQ;
        qn = a.out;
        c0 = a.offsets ? min(max(a.offsets[e], 0), a.rows) : 0;
        cn = a.offsets ? min(max(a.offsets[e + 1], c0), a.rows) : a.rows;       // contraction [c0, cn)
        w = nullptr;
    } else {
        const GroupTile g = find_tile(a.offsets, a.E, a.rows, BQ, blockIdx.x / nP);
        if (g.e < 0) return;
        e = g.e;
        q0 = g.start + g.tile * BQ;
        qn = g.start + g.n;
        cn = DIR == FWD ? a.in : a.out;
        w = a.w + (int64_t)e * a.w_stride;
    }
    // row of x of grouped row r, or none
    auto xrow = [&](int r) __attribute__((always_inline)) -> const uint16_t* {
        const int t = a.token ? a.token[r] : r;
        return (uint32_t)t < (uint32_t)a.x_rows ? a.x + (int64_t)t * a.ldx : nullptr;
    };

    // what each of the thread's chunks holds: memory row (AlongC) and index
    const uint16_t *prow[NP], *qrow[NQ];
    int pi[NP], pc[NP], qi[NQ], qc[NQ];
#pragma unroll
    for (int i = 0; i < NP; i++) {
        PT::slot(tid + i * NT, pi[i], pc[i]);
        prow[i] = nullptr;
        if (PC) {
            // SwiGLU: 16 gate rows, then the 16 up rows of the same outputs
            const int o = gated ? p0 + (pi[i] >> 5) * 16 + (pi[i] & 15) : p0 + pi[i];
            if (o < outs && tid + i * NT < PS) prow[i] = w + (int64_t)(gated && (pi[i] & 16) ? outs + o : o) * a.ldw;
        }
    }
#pragma unroll
    for (int i = 0; i < NQ; i++) {
        QT::slot(tid + i * NT, qi[i], qc[i]);
        qrow[i] = nullptr;
        if (QC && tid + i * NT < QS && q0 + qi[i] < qn) {
            const int r = q0 + qi[i];
            qrow[i] = DIR == FWD ? xrow(r) : a.dz + (int64_t)r * a.lddz;
        }
    }
    uint4 pv[NP], qv[NQ];
    auto load = [&](int c) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < NP; i++) {
            if (PC) {
                pv[i] = load8(prow[i] + c + pc[i], prow[i] ? cn - c - pc[i] : 0);
            } else {
                const int r = c + pc[i];
                const bool live = r < cn && tid + i * NT < PS;
                const uint16_t* row = !live ? nullptr : DIR == DW ? xrow(r) : w + (int64_t)r * a.ldw;
                pv[i] = load8(row + p0 + pi[i], row ? outs - p0 - pi[i] : 0);
            }
        }
#pragma unroll
        for (int i = 0; i < NQ; i++) {
            if (QC) {
                qv[i] = load8(qrow[i] + c + qc[i], qrow[i] ? cn - c - qc[i] : 0);
            } else {
                const int r = c + qc[i];
                const bool live = r < cn && tid + i * NT < QS;
                qv[i] = load8(a.dz + (int64_t)r * a.lddz + q0 + qi[i], live ? a.out - q0 - qi[i] : 0);
            }
        }
    };
    auto stage = [&](int b) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < NP; i++)
            if (PS % NT == 0 || tid + i * NT < PS) *(uint4*)(lds[b] + 16 * (tid + i * NT)) = pv[i];
#pragma unroll
        for (int i = 0; i < NQ; i++)
            if (QS % NT == 0 || tid + i * NT < QS) *(uint4*)(lds[b] + 16 * (PS + tid + i * NT)) = qv[i];
    };

    f32x4 acc[FP][FQ], accb[FQ];
#pragma unroll
    for (int i = 0; i < FP; i++)
#pragma unroll
        for (int j = 0; j < FQ; j++) acc[i][j] = (f32x4)0.0f;
#pragma unroll
    for (int j = 0; j < FQ; j++) accb[j] = (f32x4)0.0f;
    // db: one more p operand, all ones, in the first tile of p
    const bool sums = DIR == DW && a.db && p0 == 0 && wp == 0;
    const short one = BF ? 0x3F80 : 0x3C00;
    const s16x8 ones = {one, one, one, one, one, one, one, one};

    if (c0 < cn) {
        load(c0);
        stage(0);
        __syncthreads();
    }
    int b = 0;
    for (int c = c0; c < cn; c += BK, b ^= 1) {
        const bool more = c + BK < cn;
        if (more) load(c + BK);
        const lds8_t* pt = (const lds8_t*)lds[b];
        const lds8_t* qt = pt + BP * 2 * BK;
#pragma unroll
        for (int ks = 0; ks < BK / 32; ks++) {
            s16x8 pf[FP], qf[FQ];
#pragma unroll
            for (int i = 0; i < FP; i++) pf[i] = PT::frag(pt, wp * (BP / WP) + 16 * i, ks, lane);
#pragma unroll
            for (int j = 0; j < FQ; j++) qf[j] = QT::frag(qt, wq * (BQ / WQ) + 16 * j, ks, lane);
#pragma unroll
            for (int i = 0; i < FP; i++)
#pragma unroll
                for (int j = 0; j < FQ; j++) acc[i][j] = mfma<BF>(pf[i], qf[j], acc[i][j]);
            if (sums)
#pragma unroll
                for (int j = 0; j < FQ; j++) accb[j] = mfma<BF>(ones, qf[j], accb[j]);
        }
        if (more) stage(b ^ 1);
        __syncthreads();
    }

    const int pl = 4 * (lane >> 4);
#pragma unroll
    for (int j = 0; j < FQ; j++) {
        const int q = q0 + wq * (BQ / WQ) + 16 * j + (lane & 15);
        if (q >= qn) continue;
        if (DIR == FWD) {
            const bool vec = a.y_f32 ? (a.ldy % 4 == 0 && (uintptr_t)a.y % 16 == 0) : (a.ldy % 4 == 0 && (uintptr_t)a.y % 8 == 0);
            if (gated) {
#pragma unroll
                for (int i = 0; i + 1 < FP; i += 2)
                    store_forward<BF>(a, e, q, p0 + wp * (BP / WP / 2) + 8 * i + pl, outs, vec, acc[i][j], acc[i + 1][j]);
            } else {
#pragma unroll
                for (int i = 0; i < FP; i++)
                    store_forward<BF>(a, e, q, p0 + wp * (BP / WP) + 16 * i + pl, outs, vec, acc[i][j], acc[i][j]);
            }
        } else if (DIR == DX) {
            const bool vec = a.lddx % 4 == 0 && (uintptr_t)a.dx % 8 == 0;
#pragma unroll
            for (int i = 0; i < FP; i++) {
                const int p = p0 + wp * (BP / WP) + 16 * i + pl;
                store4<BF>(a.dx, (int64_t)q * a.lddx + p, 0, vec, outs - p, acc[i][j]);
            }
        } else {
            const bool vec = a.in % 4 == 0 && (uintptr_t)a.dw % 16 == 0;
            const int64_t at = ((int64_t)e * a.out + q) * a.in;
#pragma unroll
            for (int i = 0; i < FP; i++) {
                const int p = p0 + wp * (BP / WP) + 16 * i + pl;
                if (a.dw) store4<BF>(a.dw, at + p, a.dw_f32, vec, outs - p, acc[i][j]);
            }
            if (sums && lane < 16) a.db[(int64_t)e * a.out + q] = accb[j][0];
        }
    }
}

// ------------------------------------------------------------------ launch

// Upper bound of the tiles of bq rows that `rows` rows in E groups can make.
static int64_t row_tiles(int64_t rows, int64_t E, int bq, bool grouped) {
    if (!grouped) return (rows + bq - 1) / bq;
    return std::min(rows, rows / bq + E);
}

template <int DIR, int BP, int BQ, int WP, int WQ> static int run(const ProductArgs& a, int64_t qtiles, hipStream_t s) {
    const bool gated = DIR == FWD && a.act == WM_ACT_SWIGLU;
    const int outs = DIR == FWD ? (gated ? a.out / 2 : a.out) : a.in, cols = gated ? BP / 2 : BP;
    const int64_t blocks = qtiles * ((outs + cols - 1) / cols);
    if (blocks == 0) return 0;
    if (blocks > 0x7FFFFFFF) return (int)hipErrorInvalidConfiguration;
    if (a.bf16) hipLaunchKernelGGL(HIP_KERNEL_NAME(k_product<true, DIR, BP, BQ, WP, WQ>), dim3((uint32_t)blocks), dim3(64 * WP * WQ), 0, s, a);
    else hipLaunchKernelGGL(HIP_KERNEL_NAME(k_product<false, DIR, BP, BQ, WP, WQ>), dim3((uint32_t)blocks), dim3(64 * WP * WQ), 0, s, a);
    return (int)hipGetLastError();
}

template <int DIR> static int run_rows(const ProductArgs& a, hipStream_t s) {
    const bool grouped = a.offsets != nullptr;
    if (a.rows / std::max(a.E, 1) <= 32) return run<DIR, 128, 32, 4, 1>(a, row_tiles(a.rows, a.E, 32, grouped), s);
    return run<DIR, 128, 128, 2, 2>(a, row_tiles(a.rows, a.E, 128, grouped), s);
}

int launch_product(const ProductArgs& a, hipStream_t s) { return run_rows<FWD>(a, s); }
int launch_product_dx(const ProductArgs& a, hipStream_t s) { return run_rows<DX>(a, s); }
int launch_product_dw(const ProductArgs& args, hipStream_t s) {
    ProductArgs a = args;
    if (!a.dw) a.in = 1;        // db alone: one tile of p
    return run<DW, 128, 128, 2, 2>(a, (int64_t)a.E * ((a.out + 127) / 128), s);
}

}  // namespace wm
