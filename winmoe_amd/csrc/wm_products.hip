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

// Workgroup -> tile.  Workgroups go round the 8 XCDs, so each XCD takes a
// contiguous run of tiles, in blocks of 8 row tiles times all column tiles:
// what runs on an XCD at once shares rows and columns in its L2.
struct TileId {
    int p, q;
};
WM_DEV TileId tile_id(int block, int blocks, int nP) {
    const int per = blocks / 8, rest = blocks % 8, xcd = block % 8;
    const int t = xcd * per + min(xcd, rest) + block / 8;
    const int q8 = t / (8 * nP), nq = min(8, blocks / nP - 8 * q8), in = t - q8 * 8 * nP;
    return {in / nq, 8 * q8 + in % nq};
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

// A wave's FP x FQ fragments go through LDS, PH parts one after another, so
// that a lane then holds 8 consecutive outputs of one row: one 16-byte store
// (and bias or residual load) per row and lane instead of two of 8 bytes that
// jump between rows, and the epilogue's code once instead of once per
// fragment.  LDS rows are 4 floats longer than the fragments': the 16 rows
// that a store touches fall on different banks.
template <int FP, int FQ, int PH> constexpr int epilogue_floats() { return FQ / PH * 16 * (FP * 16 + 4); }

// Outputs from p0 on (contiguous) of rows from q0 on, below qn.  lds: the wave's own.
template <bool BF, int DIR, int FP, int FQ, int PH>
WM_DEV void store_tile(const ProductArgs& a, int e, int p0, int q0, int qn, int outs, int lane, const f32x4 (&acc)[FP][FQ],
                       lf32_t* lds) {
    constexpr int ROW = FP * 16 + 4;
    typedef __attribute__((address_space(3))) f32x4 lf32x4;
    const bool gated = DIR == FWD && a.act == WM_ACT_SWIGLU;
    const int units = gated ? FP : 2 * FP;
#pragma unroll
    for (int ph = 0; ph < PH; ph++) {
        wave_lds_sync();
#pragma unroll
        for (int j = 0; j < FQ / PH; j++)
#pragma unroll
            for (int i = 0; i < FP; i++)
                *(lf32x4*)(lds + (16 * j + (lane & 15)) * ROW + 16 * i + 4 * (lane >> 4)) = acc[i][ph * (FQ / PH) + j];
        wave_lds_sync();
#pragma unroll 1
        for (int k = lane; k < FQ / PH * 16 * units; k += 64) {
            const int r = k / units, u = k % units, q = q0 + ph * (FQ / PH) * 16 + r, p = p0 + 8 * u, n = outs - p;
            if (q >= qn || n <= 0) continue;
            // SwiGLU: 16 gate values, then the up values of the same outputs
            const lf32_t* src = lds + r * ROW + (gated ? 32 * (u >> 1) + 8 * (u & 1) : 8 * u);
            float z[8];
#pragma unroll
            for (int i = 0; i < 8; i++) z[i] = src[i];
            if constexpr (DIR == FWD) {
                float up[8] = {0, 0, 0, 0, 0, 0, 0, 0}, v[8];
                if (gated)
#pragma unroll
                    for (int i = 0; i < 8; i++) up[i] = src[16 + i];
                if (a.bias) {
                    const uint16_t* b = a.bias + (int64_t)e * a.out + p;
                    get8<BF>(b, n, v);
#pragma unroll
                    for (int i = 0; i < 8; i++) z[i] += v[i];
                    if (gated) {
                        get8<BF>(b + outs, n, v);
#pragma unroll
                        for (int i = 0; i < 8; i++) up[i] += v[i];
                    }
                }
                if (a.pre) {
                    uint16_t* pre = a.pre + (int64_t)q * a.ldpre + p;
                    put8<BF>(pre, n, z);
                    if (gated) put8<BF>(pre + outs, n, up);
                }
                if (a.act != WM_ACT_NONE)
#pragma unroll
                    for (int i = 0; i < 8; i++) z[i] = act_value(a.act, z[i], up[i]);
                if (a.res) {
                    get8<BF>(a.res + (int64_t)q * a.ldres + p, n, v);
#pragma unroll
                    for (int i = 0; i < 8; i++) z[i] += v[i];
                }
                if (a.y_f32) putf8((float*)a.y + (int64_t)q * a.ldy + p, n, z);
                else put8<BF>((uint16_t*)a.y + (int64_t)q * a.ldy + p, n, z);
            } else if constexpr (DIR == DX) {
                put8<BF>(a.dx + (int64_t)q * a.lddx + p, n, z);
            } else {
                const int64_t at = ((int64_t)e * a.out + q) * a.in + p;
                if (a.dw_f32) putf8((float*)a.dw + at, n, z);
                else put8<BF>((uint16_t*)a.dw + at, n, z);
            }
        }
    }
}

// Sum of an operand's 8 values of one column, added to s.
template <bool BF> WM_DEV float add8(s16x8 v, float s) {
#pragma unroll
    for (int i = 0; i < 8; i++) s += from16<BF>((uint16_t)v[i]);
    return s;
}

// db of the wave's columns: lane l summed the steps of its quarter for column l % 16.
template <int FQ> WM_DEV void store_db(const ProductArgs& a, int e, int q0, int lane, const float (&sum)[FQ]) {
#pragma unroll
    for (int j = 0; j < FQ; j++) {
        float s = sum[j];
        s += __shfl_xor(s, 16);
        s += __shfl_xor(s, 32);
        const int q = q0 + 16 * j + lane;
        if (lane < 16 && q < a.out) a.db[(int64_t)e * a.out + q] = s;
    }
}

// ------------------------------------------------------------------ tile kernel for any alignment

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
    constexpr int STAGE = (BP + BQ) * 2 * BK, PH = 1, EPI = WP * WQ * 4 * epilogue_floats<FP, FQ, PH>();
    __shared__ __attribute__((aligned(16))) uint8_t lds[2 * STAGE > EPI ? 2 * STAGE : EPI];

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
            if (PS % NT == 0 || tid + i * NT < PS) *(uint4*)(lds + b * STAGE + 16 * (tid + i * NT)) = pv[i];
#pragma unroll
        for (int i = 0; i < NQ; i++)
            if (QS % NT == 0 || tid + i * NT < QS) *(uint4*)(lds + b * STAGE + 16 * (PS + tid + i * NT)) = qv[i];
    };

    f32x4 acc[FP][FQ];
    float sum[FQ];
#pragma unroll
    for (int i = 0; i < FP; i++)
#pragma unroll
        for (int j = 0; j < FQ; j++) acc[i][j] = (f32x4)0.0f;
#pragma unroll
    for (int j = 0; j < FQ; j++) sum[j] = 0.0f;
    // db: the first tile of p sums the operand that it reads anyway
    const bool sums = DIR == DW && a.db && p0 == 0 && wp == 0;

    if (c0 < cn) {
        load(c0);
        stage(0);
        __syncthreads();
    }
    int b = 0;
    for (int c = c0; c < cn; c += BK, b ^= 1) {
        const bool more = c + BK < cn;
        if (more) load(c + BK);
        const lds8_t* pt = (const lds8_t*)lds + b * STAGE;
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
                for (int j = 0; j < FQ; j++) sum[j] = add8<BF>(qf[j], sum[j]);
        }
        if (more) stage(b ^ 1);
        __syncthreads();
    }

    if (sums) store_db<FQ>(a, e, q0 + wq * (BQ / WQ), lane, sum);
    if (DIR == DW && !a.dw) return;
    store_tile<BF, DIR, FP, FQ, PH>(a, e, p0 + (gated ? wp * (BP / WP / 2) : wp * (BP / WP)), q0 + wq * (BQ / WQ), qn, outs, lane, acc,
                                    (lf32_t*)lds + wave * epilogue_floats<FP, FQ, PH>());
}

// ------------------------------------------------------------------ tile kernel for whole 16-byte chunks

// 16 bytes per lane from src to dst (the wave's, lane order).  In assembly, as
// the compiler would wait for every such load before any later LDS read; the
// kernel waits itself (WM_WAIT_VMCNT) before the barrier that hands a stage over.
WM_DEV void lds_dma16(const void* src, lds8_t* dst) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"((uint32_t)(uintptr_t)dst), "v"(src) : "memory");
}

// Read in place of chunks that do not exist.
static __device__ __attribute__((aligned(16))) uint16_t zero_chunk[8];

// The same tile with LDS-DMA: two stages of 64 contraction steps, filled while
// the other one is used.  The operands of a half stage (32 steps) are read
// into registers while the products of the half before run, across the stage
// boundary too: at the middle of stage k every wave waits for its part of
// stage k + 1 and its last reads of stage k, and after the barrier fills stage
// k + 2 into the buffer just left.  One barrier per stage.
//
// Every chunk of 8 values exists whole or not at all (operand_rules()); rows
// and columns past the matrix repeat valid ones, as their results are not
// stored, and steps past the end of the contraction are zeros in both operands.
template <bool BF, int DIR, int BP, int BQ, int WP, int WQ>
__global__ __launch_bounds__(64 * WP * WQ) void k_product_dma(const ProductArgs a) {
    constexpr int NT = 64 * WP * WQ, FP = BP / WP / 16, FQ = BQ / WQ / 16;
    constexpr bool PC = DIR == FWD, QC = DIR != DW;
    using PT = typename std::conditional<PC, AlongC<BP>, AcrossC<BP>>::type;
    using QT = typename std::conditional<QC, AlongC<BQ>, AcrossC<BQ>>::type;
    constexpr int PS = BP * 8, QS = BQ * 8, NP = PS / NT, NQ = QS / NT, STAGE = (BP + BQ) * 2 * BK;
    static_assert(PS % NT == 0 && QS % NT == 0, "whole chunks per thread");
    constexpr int PH = WP * WQ * 4 * epilogue_floats<FP, FQ, 1>() > 160 * 1024 ? 2 : 1, EPI = WP * WQ * 4 * epilogue_floats<FP, FQ, PH>();
    __shared__ __attribute__((aligned(1024))) uint8_t lds[2 * STAGE > EPI ? 2 * STAGE : EPI];

    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wp = wave % WP, wq = wave / WP;
    const bool gated = DIR == FWD && a.act == WM_ACT_SWIGLU;
    const int outs = DIR == FWD ? (gated ? a.out / 2 : a.out) : a.in;
    const int cols = gated ? BP / 2 : BP;
    const int nP = (outs + cols - 1) / cols;
    const TileId id = tile_id(blockIdx.x, gridDim.x, nP);
    const int p0 = id.p * cols;
    int e, q0, qn, c0 = 0, cn;
    const uint16_t* w = nullptr;
    if (DIR == DW) {
        const int nQ = (a.out + BQ - 1) / BQ;
        e = id.q / nQ;
        q0 = (id.q % nQ) * BQ;
        qn = a.out;
        c0 = a.offsets ? min(max(a.offsets[e], 0), a.rows) : 0;
        cn = a.offsets ? min(max(a.offsets[e + 1], c0), a.rows) : a.rows;
    } else {
        const GroupTile g = find_tile(a.offsets, a.E, a.rows, BQ, id.q);
        if (g.e < 0) return;
        e = g.e;
        q0 = g.start + g.tile * BQ;
        qn = g.start + g.n;
        cn = DIR == FWD ? a.in : a.out;
        w = a.w + (int64_t)e * a.w_stride;
    }

    // AlongC: src = the chunk's row at its column, lim = where the row ends.
    // AcrossC: src = column of row 0, pc = the chunk's row in the stage.
    const uint16_t *psrc[NP], *qsrc[NQ];
    int pc[NP], qc[NQ], plim[NP], qlim[NQ];
#pragma unroll
    for (int i = 0; i < NP; i++) {
        int ix;
        PT::slot(tid + i * NT, ix, pc[i]);
        plim[i] = cn;
        if (PC) {
            const int o = min(gated ? p0 + (ix >> 5) * 16 + (ix & 15) : p0 + ix, outs - 1);
            psrc[i] = w + (int64_t)(gated && (ix & 16) ? outs + o : o) * a.ldw;
        } else {
            const int o = p0 + ix < outs ? p0 + ix : p0;
            psrc[i] = (DIR == DW ? a.x : w) + o;
        }
    }
#pragma unroll
    for (int i = 0; i < NQ; i++) {
        int ix;
        QT::slot(tid + i * NT, ix, qc[i]);
        qlim[i] = cn;
        if (QC) {
            const int r = min(q0 + ix, qn - 1);
            if (DIR == FWD) {
                const int t = a.token ? a.token[r] : r;
                const bool live = (uint32_t)t < (uint32_t)a.x_rows;
                qlim[i] = live ? cn : 0;
                qsrc[i] = a.x + (int64_t)(live ? t : 0) * a.ldx;
            } else {
                qsrc[i] = a.dz + (int64_t)r * a.lddz;
            }
        } else {
            qsrc[i] = a.dz + (q0 + ix < qn ? q0 + ix : q0);
        }
    }
    // DW gathers rows of x: the tokens of a stage are loaded one stage ahead
    int tok[NP];
    auto tokens = [&](int c) __attribute__((always_inline)) {
        if (DIR == DW && a.token)
#pragma unroll
            for (int i = 0; i < NP; i++) tok[i] = c + pc[i] < cn ? a.token[c + pc[i]] : -1;
    };
    auto fill = [&](int c, int b) __attribute__((always_inline)) {
        lds8_t* dst = (lds8_t*)lds + b * STAGE + 1024 * wave;
#pragma unroll
        for (int i = 0; i < NP; i++) {
            const int at = c + pc[i];
            const uint16_t* src;
            if (PC) {
                src = at < plim[i] ? psrc[i] + at : zero_chunk;
            } else if (DIR == DW) {
                const int t = a.token ? tok[i] : at;
                src = at < cn && (uint32_t)t < (uint32_t)a.x_rows ? psrc[i] + (int64_t)t * a.ldx : zero_chunk;
            } else {
                src = at < cn ? psrc[i] + (int64_t)at * a.ldw : zero_chunk;
            }
            lds_dma16(src, dst + i * NT * 16);
        }
#pragma unroll
        for (int i = 0; i < NQ; i++) {
            const int at = c + qc[i];
            const uint16_t* src;
            if (QC) src = at < qlim[i] ? qsrc[i] + at : zero_chunk;
            else src = at < cn ? qsrc[i] + (int64_t)at * a.lddz : zero_chunk;
            lds_dma16(src, dst + (PS + i * NT) * 16);
        }
    };

    f32x4 acc[FP][FQ];
    float sum[FQ];
#pragma unroll
    for (int i = 0; i < FP; i++)
#pragma unroll
        for (int j = 0; j < FQ; j++) acc[i][j] = (f32x4)0.0f;
#pragma unroll
    for (int j = 0; j < FQ; j++) sum[j] = 0.0f;
    const bool sums = DIR == DW && a.db && p0 == 0 && wp == 0;

    s16x8 pf[FP], qf[FQ];
    auto read = [&](int h, int b) __attribute__((always_inline)) {
        const lds8_t* pt = (const lds8_t*)lds + b * STAGE;
        const lds8_t* qt = pt + PS * 16;
#pragma unroll
        for (int i = 0; i < FP; i++) pf[i] = PT::frag(pt, wp * (BP / WP) + 16 * i, h, lane);
#pragma unroll
        for (int j = 0; j < FQ; j++) qf[j] = QT::frag(qt, wq * (BQ / WQ) + 16 * j, h, lane);
    };
    auto multiply = [&]() __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < FP; i++)
#pragma unroll
            for (int j = 0; j < FQ; j++) acc[i][j] = mfma<BF>(pf[i], qf[j], acc[i][j]);
        if (sums)
#pragma unroll
            for (int j = 0; j < FQ; j++) sum[j] = add8<BF>(qf[j], sum[j]);
    };

    if (c0 < cn) {
        tokens(c0);
        fill(c0, 0);
        if (c0 + BK < cn) {
            tokens(c0 + BK);
            fill(c0 + BK, 1);
            tokens(c0 + 2 * BK);
        }
        WM_WAIT_VMCNT(0);
        __syncthreads();
        int b = 0;
        for (int c = c0; c < cn; c += BK, b ^= 1) {
            read(0, b);
            multiply();
            read(1, b);
            multiply();
            WM_WAIT_VMCNT(0);                   // this wave's part of the next stage
            __syncthreads();                    // and its last reads of this one
            if (c + 2 * BK < cn) {
                fill(c + 2 * BK, b);
                tokens(c + 3 * BK);
            }
        }
    }
    if (sums) store_db<FQ>(a, e, q0 + wq * (BQ / WQ), lane, sum);
    if (DIR == DW && !a.dw) return;
    store_tile<BF, DIR, FP, FQ, PH>(a, e, p0 + (gated ? wp * (BP / WP / 2) : wp * (BP / WP)), q0 + wq * (BQ / WQ), qn, outs, lane, acc,
                                    (lf32_t*)lds + wave * epilogue_floats<FP, FQ, PH>());
}

// ------------------------------------------------------------------ launch

// Upper bound of the tiles of bq rows that `rows` rows in E groups can make.
static int64_t row_tiles(int64_t rows, int64_t E, int bq, bool grouped) {
    if (!grouped) return (rows + bq - 1) / bq;
    return std::min(rows, rows / bq + E);
}

template <int DIR, int BP, int BQ, int WP, int WQ, bool DMA> static int run(const ProductArgs& a, int64_t qtiles, hipStream_t s) {
    const bool gated = DIR == FWD && a.act == WM_ACT_SWIGLU;
    const int outs = DIR == FWD ? (gated ? a.out / 2 : a.out) : a.in, cols = gated ? BP / 2 : BP;
    const int64_t blocks = qtiles * ((outs + cols - 1) / cols);
    if (blocks == 0) return 0;
    if (blocks > 0x7FFFFFFF) return (int)hipErrorInvalidConfiguration;
    void (*k)(const ProductArgs);
    if constexpr (DMA) k = a.bf16 ? k_product_dma<true, DIR, BP, BQ, WP, WQ> : k_product_dma<false, DIR, BP, BQ, WP, WQ>;
    else k = a.bf16 ? k_product<true, DIR, BP, BQ, WP, WQ> : k_product<false, DIR, BP, BQ, WP, WQ>;
    hipLaunchKernelGGL(k, dim3((uint32_t)blocks), dim3(64 * WP * WQ), 0, s, a);
    return (int)hipGetLastError();
}

// Whether every 16-byte chunk of the operands is aligned and whole.
static bool rows16(const void* p, int64_t ld) { return (uintptr_t)p % 16 == 0 && ld % 8 == 0; }
template <int DIR> static bool whole_chunks(const ProductArgs& a) {
    if (a.in % 8 || (DIR != FWD && (a.out % 8 || !rows16(a.dz, a.lddz)))) return false;
    if (DIR != DX && !rows16(a.x, a.ldx)) return false;
    return DIR == DW || (rows16(a.w, a.ldw) && a.w_stride % 8 == 0);
}

template <int DIR> static int run_rows(const ProductArgs& a, hipStream_t s) {
    const bool grouped = a.offsets != nullptr;
    const int64_t per = a.rows / std::max(a.E, 1);
    if (!whole_chunks<DIR>(a)) {
        if (per <= 32) return run<DIR, 128, 32, 4, 1, false>(a, row_tiles(a.rows, a.E, 32, grouped), s);
        return run<DIR, 128, 128, 2, 2, false>(a, row_tiles(a.rows, a.E, 128, grouped), s);
    }
    if (per <= 32) return run<DIR, 128, 32, 4, 1, true>(a, row_tiles(a.rows, a.E, 32, grouped), s);
    if (per <= 128) return run<DIR, 128, 128, 2, 2, true>(a, row_tiles(a.rows, a.E, 128, grouped), s);
    return run<DIR, 256, 256, 2, 4, true>(a, row_tiles(a.rows, a.E, 256, grouped), s);
}

int launch_product(const ProductArgs& a, hipStream_t s) { return run_rows<FWD>(a, s); }
int launch_product_dx(const ProductArgs& a, hipStream_t s) { return run_rows<DX>(a, s); }
int launch_product_dw(const ProductArgs& args, hipStream_t s) {
    ProductArgs a = args;
    if (!a.dw) a.in = 1;        // db alone: one tile of p
    if (!whole_chunks<DW>(a)) return run<DW, 128, 128, 2, 2, false>(a, (int64_t)a.E * ((a.out + 127) / 128), s);
    return run<DW, 256, 256, 2, 4, true>(a, (int64_t)a.E * ((a.out + 255) / 256), s);
}

}  // namespace wm
