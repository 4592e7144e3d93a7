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
#include <cmath>
#include <type_traits>

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

// Workgroup's group: `qt` counts the tiles of BQ rows over all groups.
// Offsets are clamped to [0, rows], so whatever they hold no row outside is
// touched.  Every wave looks it up by itself.
struct GroupTile {
    int e, start, n, tile;      // e < 0: past the last tile
};
WM_DEV int wave_scan(int v) {
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, false);     // row_shr:1, 2, 4, 8
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false);     // lane 15 of a row into the next, then of both
    v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false);
    return v;
}
// 512 groups at a time, 8 per lane, all loads in flight together.
WM_DEV GroupTile find_tile(const int32_t* __restrict__ offsets, int E, int rows, int bq, int qt) {
    GroupTile g{-1, 0, 0, 0};
    if (!offsets) {
        g.e = (int64_t)qt * bq < rows ? 0 : -1;
        g.n = rows;
        g.tile = qt;
        return g;
    }
    const int lane = threadIdx.x & 63, shift = __builtin_ctz(bq);      // bq is a power of two
    int before = 0;
    for (int e0 = 0; e0 < E; e0 += 512) {
        const int base = e0 + 8 * lane;
        int off[9], sum = 0;
#pragma unroll
        for (int i = 0; i < 9; i++) off[i] = offsets[min(base + i, E)];
        off[0] = min(max(off[0], 0), rows);
#pragma unroll
        for (int i = 1; i < 9; i++) {
            const int v = min(max(off[i], 0), rows);
            off[i] = v;
            sum += (max(v - off[i - 1], 0) + bq - 1) >> shift;
        }
        const int end = before + wave_scan(sum);
        const uint64_t hit = __ballot(end > qt);
        if (hit) {
            const int l = __builtin_ctzll(hit);
            int at = end - sum, e = base, start = off[0], n = 0;
            bool found = false;
#pragma unroll
            for (int i = 1; i < 9; i++) {
                const int m = max(off[i] - off[i - 1], 0), t = (m + bq - 1) >> shift;
                if (!found) {
                    e = base + i - 1;
                    start = off[i - 1];
                    n = m;
                    found = at + t > qt;
                    at += found ? 0 : t;
                }
            }
            g.e = __builtin_amdgcn_readlane(e, l);
            g.start = __builtin_amdgcn_readlane(start, l);
            g.n = __builtin_amdgcn_readlane(n, l);
            g.tile = qt - __builtin_amdgcn_readlane(at, l);
            return g;
        }
        before = __builtin_amdgcn_readlane(end, 63);
    }
    return g;
}

// Workgroup -> tile.  Workgroups go round the 8 XCDs, so each XCD takes a
// contiguous run of tiles, in blocks of 4 row tiles times all column tiles:
// what runs on an XCD at once shares rows and columns in its L2.
struct TileId {
    int p, q;
};
constexpr int TILE_ROWS = 4;
WM_DEV TileId tile_id(int block, int blocks, int nP) {
    const int per = blocks / 8, rest = blocks % 8, xcd = block % 8;
    const int t = xcd * per + min(xcd, rest) + block / 8;
    const int qb = t / (TILE_ROWS * nP), nq = min(TILE_ROWS, blocks / nP - TILE_ROWS * qb), in = t - qb * TILE_ROWS * nP;
    return {in / nq, TILE_ROWS * qb + in % nq};
}
// Grouped products: how much work a row tile holds is not known on the host (the
// last ones hold none, an expert's dW takes as long as its rows), so blocks of
// `g` row tiles times all column tiles go round the XCDs in turn, the rest in
// blocks of one, then in runs as above.  16384 rows of 64 experts' 1024 x 2048,
// the popular experts first, in runs and in turn: dx 157 and 125 us (256 x 256
// tiles), dW 242 and 186 us; 4004 rows forward 72 and 60 us.
WM_DEV TileId tile_id_grouped(int block, int blocks, int nP, int g) {
    int q0 = 0;
#pragma unroll
    for (int level = 0; level < 2; level++) {
        const int n = level ? 1 : g, per = n * nP, rounds = blocks / (8 * per), full = rounds * 8 * per;
        if (block < full) {
            const int i = block / 8, in = i % per;
            return {in / n, q0 + n * (i / per * 8 + block % 8) + in % n};
        }
        block -= full;
        blocks -= full;
        q0 += rounds * 8 * n;
    }
    const TileId t = tile_id(block, blocks, nP);
    return {t.p, q0 + t.q};
}

// ------------------------------------------------------------------ LDS tiles

// [TILE][BK], memory rows along the contraction.  A row's 16-byte chunks are
// permuted by its index, so that the 16 rows of a read fall on all banks.
template <int TILE> struct AlongC {
    static constexpr int CH = BK / 8;
    WM_DEV static int perm(int index) { return index & 7; }
    // what slot s (16 bytes) holds
    WM_DEV static void slot(int s, int& index, int& c) {
        index = s / CH;
        c = 8 * ((s % CH) ^ perm(index));
    }
    // operand of 16 indices from `base` on, 32 contraction steps from 32 * ks on
    WM_DEV static s16x8 frag(const lds8_t* t, int base, int ks, int lane) {
        const int i = base + (lane & 15), ch = (4 * ks + (lane >> 4)) ^ perm(lane & 15);
        return *(const __attribute__((address_space(3))) s16x8*)(t + 2 * BK * i + 16 * ch);
    }
};

// [BK][TILE], memory rows are contraction steps.  Units of 16 values are
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

// 8 outputs of row q from column p on, from their sums (up: SwiGLU's up half).
template <bool BF, int DIR> WM_DEV void store8(const ProductArgs& a, int e, int q, int p, int outs, float (&z)[8], float (&up)[8]) {
    const int n = outs - p;
    if constexpr (DIR == FWD) {
        const bool gated = a.act == WM_ACT_SWIGLU;
        float v[8];
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

// A wave's FP x FQ fragments go through LDS, PH parts one after another, so
// that a lane then holds 8 consecutive outputs of one row: one 16-byte store
// (and bias or residual load) per row and lane instead of two of 8 bytes that
// jump between rows, and the epilogue's code once instead of once per
// fragment.  LDS rows are 4 floats longer than the fragments': the 16 rows
// that a store touches fall on different banks.
template <int FP, int FQ, int PH> constexpr int epilogue_floats() { return FQ / PH * 16 * (FP * 16 + 4); }

// Outputs from p0 on (contiguous) of rows from q0 on, below qn.  lds: the wave's own.
template <bool BF, int DIR, int FP, int FQ, int PH>
WM_DEV void store_tile(const ProductArgs& a, int e, int part, int p0, int q0, int qn, int outs, int lane, const f32x4 (&acc)[FP][FQ],
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
            const f32x4 lo = *(const lf32x4*)src, hi = *(const lf32x4*)(src + 4);
            float z[8] = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]}, up[8] = {0, 0, 0, 0, 0, 0, 0, 0};
            if (gated) {
                const f32x4 l = *(const lf32x4*)(src + 16), h = *(const lf32x4*)(src + 20);
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    up[i] = l[i];
                    up[4 + i] = h[i];
                }
            }
            if (a.split > 1) {
                const int64_t at = DIR == DW ? (int64_t)(part * a.E + e) * a.out + q : (int64_t)part * a.rows + q;
                float* d = a.part + at * (DIR == FWD ? a.out : a.in) + p;
                putf8(d, n, z);
                if (gated) putf8(d + outs, n, up);
            } else {
                store8<BF, DIR>(a, e, q, p, outs, z, up);
            }
        }
    }
}

// dW's fragments straight from the registers, 4 outputs per lane and store:
// fp32 always (64 bytes of a row per store; 2047 x 4096 over 1001 rows 40.2 us
// through LDS, 35.6 us so), 16 bits where products take longer than the writes
// (64 experts' 1024 x 2048 over 16384 rows 236 and 226 us, but 512 experts over
// 5120 rows 1482 and 1558 us).
template <bool BF, int FP, int FQ>
WM_DEV void store_direct(const ProductArgs& a, int e, int p0, int q0, int lane, const f32x4 (&acc)[FP][FQ]) {
    const int pl = p0 + 4 * (lane >> 4);
#pragma unroll
    for (int j = 0; j < FQ; j++) {
        const int q = q0 + 16 * j + (lane & 15);
        if (q >= a.out) continue;
        const int64_t at = ((int64_t)e * a.out + q) * a.in + pl;
#pragma unroll
        for (int i = 0; i < FP; i++) {
            if (pl + 16 * i >= a.in) continue;
            const f32x4 v = acc[i][j];
            if (a.dw_f32) *(f32x4*)((float*)a.dw + at + 16 * i) = v;
            else *(uint2*)((uint16_t*)a.dw + at + 16 * i) = (uint2){to16<BF>(v[0]) | (uint32_t)to16<BF>(v[1]) << 16,
                                                                  to16<BF>(v[2]) | (uint32_t)to16<BF>(v[3]) << 16};
        }
    }
}

// One output of the forward product, from its sums.
template <bool BF> WM_DEV void store_one(const ProductArgs& a, int e, int q, int p, int outs, float z, float u) {
    const bool gated = a.act == WM_ACT_SWIGLU;
    if (a.bias) {
        const uint16_t* b = a.bias + (int64_t)e * a.out + p;
        z += from16<BF>(b[0]);
        if (gated) u += from16<BF>(b[outs]);
    }
    if (a.pre) {
        uint16_t* pre = a.pre + (int64_t)q * a.ldpre + p;
        pre[0] = to16<BF>(z);
        if (gated) pre[outs] = to16<BF>(u);
    }
    z = act_value(a.act, z, u);
    if (a.res) z += from16<BF>(a.res[(int64_t)q * a.ldres + p]);
    if (a.y_f32) ((float*)a.y)[(int64_t)q * a.ldy + p] = z;
    else ((uint16_t*)a.y)[(int64_t)q * a.ldy + p] = to16<BF>(z);
}

// Sum of an operand's 8 values of one column, added to s.
template <bool BF> WM_DEV float add8(s16x8 v, float s) {
#pragma unroll
    for (int i = 0; i < 8; i++) s += from16<BF>((uint16_t)v[i]);
    return s;
}

// db of the wave's columns: lane l summed the steps of its quarter for column l % 16.
template <int FQ> WM_DEV void store_db(const ProductArgs& a, int e, int part, int q0, int lane, const float (&sum)[FQ]) {
#pragma unroll
    for (int j = 0; j < FQ; j++) {
        float s = sum[j];
        s += __shfl_xor(s, 16);
        s += __shfl_xor(s, 32);
        const int q = q0 + 16 * j + lane;
        if (lane < 16 && q < a.out) (a.split > 1 ? a.part_db + (int64_t)part * a.E * a.out : a.db)[(int64_t)e * a.out + q] = s;
    }
}

// ------------------------------------------------------------------ tile kernel for any alignment

// WP x WQ waves, each a (BP / WP) x (BQ / WQ) part of the tile.  Two LDS
// buffers: the chunks of the next 64 steps are loaded into registers while
// this buffer's products run, then stored into the other one.
template <bool BF, int DIR, int BP, int BQ, int WP, int WQ>
__global__ __launch_bounds__(64 * WP * WQ) void k_product(const ProductArgs a) {
    constexpr int NT = 64 * WP * WQ, FP = BP / WP / 16, FQ = BQ / WQ / 16;
    static_assert(DIR != FWD || FP % 2 == 0, "SwiGLU's gate and up meet in a wave");
    static_assert(DIR != DW, "dW runs on copies");
    constexpr bool PC = DIR == FWD;         // W's rows run along the contraction; x's and dz's do
    using PT = typename std::conditional<PC, AlongC<BP>, AcrossC<BP>>::type;
    using QT = AlongC<BQ>;
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
    const GroupTile g = find_tile(a.offsets, a.E, a.rows, BQ, blockIdx.x / nP);
    if (g.e < 0) return;
    const int e = g.e, q0 = g.start + g.tile * BQ, qn = g.start + g.n, cn = DIR == FWD ? a.in : a.out;
    const uint16_t* w = a.w + (int64_t)e * a.w_stride;
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
        if (tid + i * NT < QS && q0 + qi[i] < qn) {
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
                pv[i] = load8(w + (int64_t)r * a.ldw + p0 + pi[i], live ? outs - p0 - pi[i] : 0);
            }
        }
#pragma unroll
        for (int i = 0; i < NQ; i++) qv[i] = load8(qrow[i] + c + qc[i], qrow[i] ? cn - c - qc[i] : 0);
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
#pragma unroll
    for (int i = 0; i < FP; i++)
#pragma unroll
        for (int j = 0; j < FQ; j++) acc[i][j] = (f32x4)0.0f;

    load(0);
    stage(0);
    __syncthreads();
    int b = 0;
    for (int c = 0; c < cn; c += BK, b ^= 1) {
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
        }
        if (more) stage(b ^ 1);
        __syncthreads();
    }

    store_tile<BF, DIR, FP, FQ, PH>(a, e, 0, p0 + (gated ? wp * (BP / WP / 2) : wp * (BP / WP)), q0 + wq * (BQ / WQ), qn, outs, lane, acc,
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

// The same tile with LDS-DMA: a ring of S stages of 64 contraction steps, S - 1
// of them in flight or in use at any time.  One barrier per stage: behind it
// every wave's part of the stage has landed and every wave is done with the
// stage before, whose buffer is filled again at once.
//
// Every chunk of 8 values exists whole or not at all (whole_chunks()); rows
// and columns past the matrix repeat valid ones, as their results are not
// stored, and steps past the end of the contraction are zeros in both operands.
//
// A call with too few tiles to fill the chip gives each tile's contraction to
// a.split workgroups (k_join adds their sums).
//
// 128 wide tiles have 8 waves: a wave's loads are issued one behind the other
// before its products, and with 4 waves each issues twice as many (2048 x 2048 x
// 2048: 31.9 and 28.6 us forward, 36.7 and 31.3 us for dW).
//
// Grouped products of few rows per expert are bound by memory: 5120 rows of 512
// experts' 4096 x 1024 take 790 us, 5.5 TB/s.  dx of 16384 rows of 64 experts'
// 1024 x 2048 takes 125 to 132 us (256 x 256 tiles, 520 TFLOP/s), dW 186 to 192 us.
template <bool BF, int DIR, int BP, int BQ, int WP, int WQ, int S>
__global__ __launch_bounds__(64 * WP * WQ) void k_product_dma(const ProductArgs a) {
    constexpr int NT = 64 * WP * WQ, FP = BP / WP / 16, FQ = BQ / WQ / 16;
    static_assert(DIR != FWD || FP % 2 == 0, "SwiGLU's gate and up meet in a wave");
    constexpr bool PC = DIR == FWD, QC = DIR != DW;
    using PT = typename std::conditional<PC, AlongC<BP>, AcrossC<BP>>::type;
    using QT = typename std::conditional<QC, AlongC<BQ>, AcrossC<BQ>>::type;
    constexpr int PS = BP * BK / 8, QS = BQ * BK / 8, NP = PS / NT, NQ = QS / NT, STAGE = (BP + BQ) * 2 * BK;
    static_assert(PS % NT == 0 && QS % NT == 0, "whole chunks per thread");
    static_assert((S - 2) * (NP + NQ) < 64, "loads are counted");
    constexpr int PH = WP * WQ * 4 * epilogue_floats<FP, FQ, 1>() > 160 * 1024 ? 2 : 1, EPI = WP * WQ * 4 * epilogue_floats<FP, FQ, PH>();
    __shared__ __attribute__((aligned(1024))) uint8_t lds[BP == 256 && DIR != DW ? STAGE / 2 * 5 : S * STAGE > EPI ? S * STAGE : EPI];
    static_assert(sizeof(lds) >= EPI, "the epilogue fits");

    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wp = wave % WP, wq = wave / WP;
    const bool gated = DIR == FWD && a.act == WM_ACT_SWIGLU;
    const int outs = DIR == FWD ? (gated ? a.out / 2 : a.out) : a.in;
    const int cols = gated ? BP / 2 : BP;
    const int nP = (outs + cols - 1) / cols;
    const int tiles = gridDim.x / a.split, part = blockIdx.x / tiles;
    const TileId id = a.offsets ? tile_id_grouped(blockIdx.x % tiles, tiles, nP, DIR == DW ? (a.out + BQ - 1) / BQ : TILE_ROWS)
                                : tile_id(blockIdx.x % tiles, tiles, nP);
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

    const int steps = cn - c0;
    if (a.split > 1) {
        const int n = (cn - c0 + BK - 1) / BK, first = c0;
        c0 = first + BK * (int)((int64_t)n * part / a.split);
        cn = min(cn, first + BK * (int)((int64_t)n * (part + 1) / a.split));
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
    // DW gathers rows of x: a load of 64 chunks covers R rows.  Their tokens come
    // through scalar loads (vector loads would wait for the stages in flight
    // before them), one stage ahead (64 experts, 16384 gathered rows: 226 us
    // without, 186 us with).
    constexpr int R = 512 / BP;
    int tok[NP][R] = {};
    auto tokens = [&](int c) __attribute__((always_inline)) {
        if (DIR == DW && a.token)
#pragma unroll
            for (int i = 0; i < NP; i++)
#pragma unroll
                for (int k = 0; k < R; k++) {
                    const int r = c + (64 * wave + i * NT) / (BP / 8) + k;
                    tok[i][k] = r < cn ? ((const __attribute__((address_space(4))) int32_t*)(uintptr_t)a.token)[r] : -1;
                }
    };
    auto token = [&](int i) __attribute__((always_inline)) {
        int v = 0;
#pragma unroll
        for (int k = 0; k < R; k++) v |= tok[i][k] & -(int)(lane / (64 / R) == k);
        return v;
    };
    auto fill_p = [&](int c, int i, lds8_t* dst) __attribute__((always_inline)) {
        const int at = c + pc[i];
        const uint16_t* src;
        if (PC) {
            src = at < plim[i] ? psrc[i] + at : zero_chunk;
        } else if (DIR == DW) {
            const int t = a.token ? token(i) : at;
            src = at < cn && (uint32_t)t < (uint32_t)a.x_rows ? psrc[i] + (int64_t)t * a.ldx : zero_chunk;
        } else {
            src = at < cn ? psrc[i] + (int64_t)at * a.ldw : zero_chunk;
        }
        lds_dma16(src, dst + 1024 * wave + i * NT * 16);
    };
    auto fill_q = [&](int c, int i, lds8_t* dst) __attribute__((always_inline)) {
        const int at = c + qc[i];
        const uint16_t* src;
        if (QC) src = at < qlim[i] ? qsrc[i] + at : zero_chunk;
        else src = at < cn ? qsrc[i] + (int64_t)at * a.lddz : zero_chunk;
        lds_dma16(src, dst + 1024 * wave + i * NT * 16);
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

    s16x8 pf[FP], qf[FQ];
    auto read = [&](int h, const lds8_t* pt, const lds8_t* qt) __attribute__((always_inline)) {
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

    if constexpr (BP == 256 && DIR != DW) {
        // Two groups of 4 waves, one of each group per SIMD, take turns: while
        // one reads its operands of half a stage the other one multiplies.  Time
        // runs in slots that end in a barrier: group 0 reads the halves of stage
        // k in slots 4 k and 4 k + 2 and multiplies in slots 4 k + 1 and 4 k + 3,
        // group 1 does so one slot later.  So stage k is done with after slot
        // 4 k + 3 and stage k + 1 has to be there by then.
        //
        // LDS holds 5 operand tiles: both of stage k, both of stage k + 1 and
        // p of stage k + 2, in turn.  A wave fetches its part of q of stage k + 1,
        // then of p of stage k + 2, along with its reads of the two halves: a
        // load waits for its turn, which would hold up products behind it.
        //
        // 4096 x 16384 x 4096 takes 435 to 470 us (1170 to 1260 TFLOP/s; a library
        // product 1460).  A stage takes 1.5 to 1.6 us; its matrix instructions need
        // 0.9 us, 1.2 at the clock that long products run at, its 192 KB of LDS
        // reads 0.6 at the 315 B/ns that a CU reaches, its 64 KB of loads 0.5 from
        // L2 (120 B/ns).  4 waves of 128 x 128, which read a third less, took 477 us,
        // as their sums move between register files.
        static_assert(S == 2 && BP == BQ && NP == 4 && NQ == 4, "5 tiles of equal size");
        constexpr int TILE = BP * 2 * BK;
        const bool second = wave >= 4;
        const int n = (cn - c0 + BK - 1) / BK;
        lds8_t* const tiles = (lds8_t*)lds;
        auto slot_end = [&]() __attribute__((always_inline)) {
            __builtin_amdgcn_sched_barrier(0);
            asm volatile("s_barrier" ::: "memory");
            __builtin_amdgcn_sched_barrier(0);
        };
        auto fetch_q = [&](int k, int t) __attribute__((always_inline)) {
            if (k < n)
#pragma unroll
                for (int i = 0; i < NQ; i++) fill_q(c0 + k * BK, i, tiles + t * TILE);
        };
        auto fetch_p = [&](int k, int t) __attribute__((always_inline)) {
            if (k < n)
#pragma unroll
                for (int i = 0; i < NP; i++) fill_p(c0 + k * BK, i, tiles + t * TILE);
        };
        auto landed = [&](int k) __attribute__((always_inline)) {       // stage k + 1; p of stage k + 2 may not be
            if (k + 2 < n) WM_WAIT_VMCNT(4);
            else WM_WAIT_VMCNT(0);
        };
        auto products = [&]() __attribute__((always_inline)) {
            __builtin_amdgcn_s_setprio(1);
            multiply();
            __builtin_amdgcn_s_setprio(0);
        };
        if (n > 0) {
            fetch_p(0, 0);
            fetch_q(0, 1);
            fetch_p(1, 2);
            landed(-1);
            slot_end();
            if (second) slot_end();
            int tp = 0;                                     // tile of p of stage k; q's is the next
            for (int k = 0; k < n; k++) {
                const lds8_t *pt = tiles + tp * TILE, *qt = tiles + (tp == 4 ? 0 : tp + 1) * TILE;
                read(0, pt, qt);
                fetch_q(k + 1, tp >= 2 ? tp - 2 : tp + 3);
                asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
                slot_end();
                products();
                slot_end();
                read(1, pt, qt);
                fetch_p(k + 2, tp >= 1 ? tp - 1 : tp + 4);
                if (second) landed(k);
                asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
                slot_end();
                products();
                if (!second) landed(k);
                slot_end();
                tp = tp >= 3 ? tp - 3 : tp + 2;
            }
            if (!second) slot_end();
        }
    } else if (c0 < cn) {
        auto fill = [&](int c, int b) __attribute__((always_inline)) {
            lds8_t* dst = (lds8_t*)lds + b * STAGE;
#pragma unroll
            for (int i = 0; i < NP; i++) fill_p(c, i, dst);
#pragma unroll
            for (int i = 0; i < NQ; i++) fill_q(c, i, dst + PS * 16);
        };
#pragma unroll
        for (int i = 0; i < S - 1; i++) {
            if (i && c0 + i * BK >= cn) break;
            tokens(c0 + i * BK);
            fill(c0 + i * BK, i);
        }
        tokens(c0 + (S - 1) * BK);
        int b = 0;
        for (int c = c0; c < cn; c += BK) {
            // stages c + BK .. c + (S - 2) BK may still be in flight
            if (S > 2 && c + (S - 2) * BK < cn) WM_WAIT_VMCNT((S - 2) * (NP + NQ));
            else WM_WAIT_VMCNT(0);
            asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
            if (c + (S - 1) * BK < cn) fill(c + (S - 1) * BK, b == 0 ? S - 1 : b - 1);
            tokens(c + S * BK);
            const lds8_t* pt = (const lds8_t*)lds + b * STAGE;
#pragma unroll
            for (int h = 0; h < BK / 32; h++) {
                read(h, pt, pt + PS * 16);
                multiply();
            }
            b = b == S - 1 ? 0 : b + 1;
        }
        asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");        // the epilogue writes over the last stage
    }
    if (sums) store_db<FQ>(a, e, part, q0 + wq * (BQ / WQ), lane, sum);
    if (DIR == DW && !a.dw) return;
    if constexpr (DIR == DW) {
        if (a.split == 1 && a.in % 4 == 0 && (uintptr_t)a.dw % 16 == 0 && (a.dw_f32 || steps > 2 * BK)) {
            store_direct<BF, FP, FQ>(a, e, p0 + wp * (BP / WP), q0 + wq * (BQ / WQ), lane, acc);
            return;
        }
    }
    store_tile<BF, DIR, FP, FQ, PH>(a, e, part, p0 + (gated ? wp * (BP / WP / 2) : wp * (BP / WP)), q0 + wq * (BQ / WQ), qn, outs, lane, acc,
                                    (lf32_t*)lds + wave * epilogue_floats<FP, FQ, PH>());
}

// ------------------------------------------------------------------ joining parts

// Adds the parts' sums in order and finishes the outputs: one thread per 8 of
// them.  Rows of no group are left out.
template <bool BF, int DIR> __global__ __launch_bounds__(256) void k_join(const ProductArgs a) {
    const bool gated = DIR == FWD && a.act == WM_ACT_SWIGLU;
    const int width = DIR == FWD ? a.out : a.in, outs = gated ? width / 2 : width;
    const int rows = DIR == DW ? a.E * a.out : a.rows;
    const uint32_t per = (outs + 7) / 8;
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int64_t r = i / per;
    if (r >= rows) return;
    const int p = (int)(i - r * per) * 8, n = outs - p;
    int e = 0, q = (int)r;
    if (DIR == DW) {
        e = q / a.out;
        q -= e * a.out;
        if (a.db && p == 0) {
            float s = 0.0f;
            for (int k = 0; k < a.split; k++) s += a.part_db[(int64_t)k * rows + r];
            a.db[r] = s;
        }
        if (!a.dw) return;
    } else if (a.offsets) {
        if (q < a.offsets[0] || q >= a.offsets[a.E]) return;
        int hi = a.E;                   // offsets[e] <= q < offsets[hi]
        while (hi - e > 1) {
            const int mid = (e + hi) / 2;
            if (a.offsets[mid] <= q) e = mid;
            else hi = mid;
        }
    }
    float z[8] = {0, 0, 0, 0, 0, 0, 0, 0}, up[8] = {0, 0, 0, 0, 0, 0, 0, 0}, v[8];
#pragma unroll 4
    for (int k = 0; k < a.split; k++) {
        const float* s = a.part + ((int64_t)k * rows + r) * width + p;
        getf8(s, n, v);
#pragma unroll
        for (int j = 0; j < 8; j++) z[j] += v[j];
        if (gated) {
            getf8(s + outs, n, v);
#pragma unroll
            for (int j = 0; j < 8; j++) up[j] += v[j];
        }
    }
    store8<BF, DIR>(a, e, q, p, outs, z, up);
}

// ------------------------------------------------------------------ few rows

// Forward product of up to 16 rows per tile, bound by streaming W once.  A
// workgroup takes 16 rows of W (SwiGLU: 8 gate rows and their up rows) and all
// of the contraction, split over its waves in contiguous parts, so enough
// workgroups exist without sums across them.  W goes from memory straight
// into the operand registers, 8 loads of 1 KB in flight per wave; x is read
// from the caches.  The waves' sums meet in LDS, in wave order.  No alignment
// is assumed: only the last step of 32 may be partial.  One row of 4096 x 4096
// takes 8.1 us, 2.4 us of it the launch.
template <bool BF, int NW> __global__ __launch_bounds__(64 * NW) void k_product_few(const ProductArgs a) {
    constexpr int ROW = 20;             // floats per row of sums, 16 used
    __shared__ __attribute__((aligned(16))) float red[NW * 16 * ROW];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), g = lane >> 4, l = lane & 15;
    const bool gated = a.act == WM_ACT_SWIGLU;
    const int outs = gated ? a.out / 2 : a.out, cols = gated ? 8 : 16, nP = (outs + cols - 1) / cols;
    const GroupTile t = find_tile(a.offsets, a.E, a.rows, 16, blockIdx.x / nP);
    if (t.e < 0) return;
    const int p0 = (int)(blockIdx.x % nP) * cols, q0 = t.start + t.tile * 16, qn = t.start + t.n;

    const int o = min(p0 + (gated ? l & 7 : l), outs - 1), q = q0 + l;
    const uint16_t* wrow = a.w + (int64_t)t.e * a.w_stride + (int64_t)(gated && (l & 8) ? outs + o : o) * a.ldw + 8 * g;
    const int r = q < qn ? (a.token ? a.token[q] : q) : -1;
    const bool live = (uint32_t)r < (uint32_t)a.x_rows;
    const uint16_t* xrow = a.x + (int64_t)(live ? r : 0) * a.ldx + 8 * g;
    f32x4 acc[2] = {(f32x4)0.0f, (f32x4)0.0f};
    const int steps = (a.in + 31) / 32, per = (steps + NW - 1) / NW, s1 = min((wave + 1) * per, steps);
    int s = wave * per;
    auto batch = [&](auto n) __attribute__((always_inline)) {
        constexpr int N = decltype(n)::value;
        s16x8 wv[N], xv[N];
#pragma unroll
        for (int i = 0; i < N; i++) __builtin_memcpy(&wv[i], wrow + 32 * (s + i), 16);
#pragma unroll
        for (int i = 0; i < N; i++) xv[i] = (s16x8)0;
        if (live)
#pragma unroll
            for (int i = 0; i < N; i++) __builtin_memcpy(&xv[i], xrow + 32 * (s + i), 16);
#pragma unroll
        for (int i = 0; i < N; i++) acc[i & 1] = mfma<BF>(wv[i], xv[i], acc[i & 1]);
        s += N;
    };
    const int full = min(s1, a.in / 32);
    while (s + 8 <= full) batch(std::integral_constant<int, 8>());
    while (s + 4 <= full) batch(std::integral_constant<int, 4>());
    while (s < full) batch(std::integral_constant<int, 1>());
    if (s < s1) {
        const int c = 32 * s, n = a.in - c - 8 * g;
        const uint4 wt = load8(wrow + c, n), xt = load8(xrow + c, live ? n : 0);
        acc[0] = mfma<BF>(__builtin_bit_cast(s16x8, wt), __builtin_bit_cast(s16x8, xt), acc[0]);
    }
    *(f32x4*)&red[(wave * 16 + l) * ROW + 4 * g] = acc[0] + acc[1];
    __syncthreads();
    for (int k = threadIdx.x; k < 16 * cols; k += 64 * NW) {
        const int row = k / cols, j = k % cols;
        if (q0 + row >= qn || p0 + j >= outs) continue;
        float z = 0.0f, u = 0.0f;
#pragma unroll
        for (int w = 0; w < NW; w++) {
            z += red[(w * 16 + row) * ROW + j];
            if (gated) u += red[(w * 16 + row) * ROW + 8 + j];
        }
        store_one<BF>(a, t.e, q0 + row, p0 + j, outs, z, u);
    }
}

// ------------------------------------------------------------------ repacking

// Copies rows into rows of `ld` values, zeros behind the first `cols`: makes an
// operand whose rows are odd or unaligned fit for 16-byte chunks.
__global__ __launch_bounds__(256) void k_repack(const uint16_t* __restrict__ src, int64_t ld_src, int64_t stride_src, int rows,
                                                int cols, uint16_t* __restrict__ dst, int ld, int64_t stride_dst) {
    const uint32_t per = ld / 8;
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, r = i / per;
    if (r >= rows) return;
    const int c = (int)(i - r * per) * 8;
    const uint4 v = load8(src + blockIdx.y * stride_src + r * ld_src + c, cols - c);
    *(uint4*)(dst + blockIdx.y * stride_dst + r * ld + c) = v;
}

// ------------------------------------------------------------------ launch

// How a product is run.  The kernels' times are estimated from their own
// measurements (bf16): `alone` is what a stage of 64 steps takes with one
// workgroup on a CU, `share` what it adds to a CU that is full, `ends` a tile's
// first loads and its stores, all in us.
enum Kernel : int { ANY128, ANY32, FEW, T256, T128, T128x64, T128x32, T64, T64x32, T64x16 };
struct TileCost {
    Kernel k;
    int bp, bq, resident;
    float alone, share, ends;
};
static constexpr TileCost kTiles[] = {
    {T256, 256, 256, 1, 1.40f, 1.60f, 6.0f},  {T128, 128, 128, 2, 0.73f, 0.52f, 3.0f}, {T128x64, 128, 64, 2, 0.54f, 0.35f, 2.5f},
    {T128x32, 128, 32, 2, 0.42f, 0.33f, 2.0f}, {T64, 64, 64, 2, 0.37f, 0.24f, 2.0f},    {T64x32, 64, 32, 3, 0.34f, 0.20f, 2.0f},
    {T64x16, 64, 16, 4, 0.34f, 0.15f, 2.0f},   {ANY128, 128, 128, 2, 1.00f, 0.69f, 3.0f}, {ANY32, 128, 32, 4, 0.70f, 0.45f, 2.0f},
};
struct Plan {
    Kernel k;
    int split;
};
static bool tiled(const Plan& p) { return p.k >= T256; }

static int columns(const ProductArgs& a, int dir) {      // of the result
    return dir == FWD ? (a.act == WM_ACT_SWIGLU ? a.out / 2 : a.out) : a.in;
}

// Upper bound of the tiles of bq rows that `rows` rows in E groups can make.
static int64_t row_tiles(const ProductArgs& a, int bq) {
    if (!a.offsets) return (a.rows + bq - 1) / bq;
    return std::min((int64_t)a.rows, (int64_t)a.rows / bq + a.E);
}

// Whether every 16-byte chunk of an operand is aligned and whole.
static bool chunks16(const void* p, int64_t ld, int cols) { return (uintptr_t)p % 16 == 0 && ld % 8 == 0 && cols % 8 == 0; }

// What the LDS-DMA tiles need copied first: operands of odd or unaligned rows.
struct Copies {
    bool x, w, dz;
    bool any() const { return x || w || dz; }
};
static Copies copies(const ProductArgs& a, bool fwd, bool dx, bool dw) {
    return {(fwd || dw) && !chunks16(a.x, a.ldx, a.in), (fwd || dx) && !(chunks16(a.w, a.ldw, a.in) && a.w_stride % 8 == 0),
            (dx || dw) && !chunks16(a.dz, a.lddz, a.out)};
}

// The kernel and the number of parts with the least estimated time.  The chip
// is taken as 256 CUs.  The host does not know the groups: rows are taken as
// spread evenly at random over the experts, with some more tiles than that
// makes, as groups are skewed; smaller tiles, which fetch more, share a CU less
// well there than in one group (dx of 32768 rows of 128 experts' 1024 x 1024: 256
// x 256 124 us, 128 x 128 141 us; in one group their estimates hold).
//
// Tiles: reading the weights (writing, for dW) overlaps the products, the worse
// the closer the two are; tiles 64 wide read them in shorter rows.  A split pays a second kernel
// (which has to look groups up) and the parts' way to memory and back: 4 or 7 us
// and 2.5 TB/s.  Copies pay 3 us and 4 TB/s, which the kernels for any alignment
// do not need (dW has none of those).
// Few rows (k_product_few, forward): W once per 16 rows, 5.2 TB/s (grouped 4.6,
// and up to 1024 columns 3.9, where workgroups are short), x from the caches at
// 15 TB/s, or the time of its waves' batches one after another.  In a graph, us: 1 row,
// 4096 x 4096 9.0 (split tiles 12.4); 48 rows 25 (tiles 14.5); 4 of 64 experts'
// 1024 x 2048 7.3 (tiles 18.3); 16 rows, 65536 x 4096 122 (tiles 110).
static Plan plan(const ProductArgs& a, int dir) {
    const double E = a.E, rows = a.rows, groups = a.offsets && E > 1 ? std::max(1.0, E * (1.0 - std::exp(-rows / E))) : 1.0, per = rows / groups;
    const int outs = columns(a, dir);
    const bool gated = dir == FWD && a.act == WM_ACT_SWIGLU;
    const double stages = std::max(1.0, std::ceil((dir == FWD ? a.in : dir == DX ? a.out : per) / BK));
    const double weights = 2.0 * groups * a.in * a.out;
    const double memory = (dir == DW ? 2.0 * E * a.in * a.out * (1.0 + a.dw_f32) : weights) / 5.6e6;        // us
    const double sums = (dir == DW ? E * a.out * a.in : rows * (dir == FWD ? a.out : a.in)) * 8.0;
    const Copies c = copies(a, dir == FWD, dir == DX, dir == DW);
    double copy = 0.0;
    if (c.w) copy += 3.0 + 4.0 * E * a.in * a.out / 4e6;
    if (c.x && dir == FWD) copy += 3.0 + 4.0 * a.x_rows * a.in / 4e6;
    if (c.dz && dir == DX) copy += 3.0 + 4.0 * rows * a.out / 4e6;
    auto row_parts = [&](int bq) { return groups > 1 ? groups * (0.75 + std::max(0.25, per / bq)) : std::ceil(rows / bq); };

    Plan best{T128, 1};
    double least = 1e30;
    for (const TileCost& t : kTiles) {
        const bool any = t.k == ANY128 || t.k == ANY32;
        if ((dir == DW && (any || t.bp != t.bq)) || (any && !c.any())) continue;
        const double p = std::ceil(outs / (double)(gated ? t.bp / 2 : t.bp));
        const double q = dir == DW ? E * std::ceil(a.out / (double)t.bq) : row_parts(t.bq);
        for (int s = 1; s <= (any ? 1 : 16) && s * 2 <= stages + 1; s *= 2) {
            if (s > 1 && s * sums > 512e6) break;
            const double n = std::ceil(p * q * s / 256), turns = std::max(1.0, n / t.resident);
            const double share = groups > 1 && t.resident > 1 ? 1.25 * t.share : t.share;
            const double work = std::ceil(stages / s) * std::max(t.alone * turns, share * n) + t.ends * turns;
            const double stream = t.bp < 128 ? 1.15 * memory : memory;
            const double more = std::max(work, stream), less = std::min(work, stream);
            const double us = 3.0 + more + 0.35 * less * (less / more) * (less / more) + (any ? 0.0 : copy) +
                              (s > 1 ? (a.offsets ? 7.0 : 4.0) + s * sums / 2.5e6 : 0.0);
            if (us < least) {
                least = us;
                best = {t.k, s};
            }
        }
    }
    if (dir == FWD) {
        const double passes = row_parts(16) / groups, x = row_parts(16) * std::min(per, 16.0) * a.in * 2.0 * std::ceil(outs / (gated ? 8.0 : 16.0));
        const double batches = std::ceil(a.in / (a.in <= 2048 ? 4.0 : 8.0) / 64) / 4;           // of 8 loads, per wave
        const double rate = a.in <= 1024 ? 3.9e6 : a.offsets ? 4.6e6 : 5.2e6;
        const double us = (a.offsets ? 5.5 : 3.0) + std::max(passes * weights / rate + x / 15e6, batches * (1.6 + 0.085 * std::min(per, 16.0)));
        if (us < least) best = {FEW, 1};
    }
    return best;
}

struct Layout {
    int64_t x, w, dz, part, total;
};
static int64_t up256(int64_t n) { return (n + 255) & ~(int64_t)255; }
static Layout layout(const ProductArgs& a, const Copies& c, int64_t part) {
    const int64_t in8 = (a.in + 7) / 8 * 8, out8 = (a.out + 7) / 8 * 8;
    Layout l;
    l.x = 0;
    l.w = l.x + (c.x ? up256(2 * in8 * a.x_rows) : 0);
    l.dz = l.w + (c.w ? up256(2 * in8 * a.out * a.E) : 0);
    l.part = l.dz + (c.dz ? up256(2 * out8 * a.rows) : 0);
    l.total = l.part + part;
    return l;
}
static int64_t part_bytes(const ProductArgs& a, int dir, int split) {
    if (split == 1) return 0;
    const int64_t n = dir == DW ? (int64_t)a.E * a.out * (a.in + 1) : (int64_t)a.rows * (dir == FWD ? a.out : a.in);
    return 4 * n * split;
}
// db without dw takes one column of x.
static ProductArgs only_db(const ProductArgs& a) {
    ProductArgs b = a;
    b.in = 1;
    b.dw_f32 = 0;
    return b;
}

int product_plan(const ProductArgs& a, int dir, int* parts) {
    const Plan p = plan(a, dir);
    *parts = p.split;
    return p.k;
}

int64_t product_workspace(const ProductArgs& a, bool backward) {
    if (a.rows == 0) return 0;
    if (!backward) {
        const Plan p = plan(a, FWD);
        return layout(a, tiled(p) ? copies(a, true, false, false) : Copies{}, part_bytes(a, FWD, p.split)).total;
    }
    // whichever of dx, dw and db the call asks for
    ProductArgs b = a;
    int64_t part = 0;
    const Plan px = plan(a, DX);
    part = part_bytes(a, DX, px.split);
    for (int f32 = 0; f32 < 2; f32++) {
        b.dw_f32 = f32;
        part = std::max(part, part_bytes(b, DW, plan(b, DW).split));
    }
    b = only_db(a);
    part = std::max(part, part_bytes(b, DW, plan(b, DW).split));
    return layout(a, copies(a, false, tiled(px), true), part).total;
}

// A launch holds fewer than 2^32 threads.
static bool too_many(int64_t blocks, int threads) { return blocks > 0xFFFFFFFFll / threads; }

template <int DIR, int BP, int BQ, int WP, int WQ, int S> static int run(const ProductArgs& a, hipStream_t s) {
    const bool gated = DIR == FWD && a.act == WM_ACT_SWIGLU;
    const int outs = columns(a, DIR), cols = gated ? BP / 2 : BP;
    const int64_t qtiles = DIR == DW ? (int64_t)a.E * ((a.out + BQ - 1) / BQ) : row_tiles(a, BQ);
    const int64_t blocks = qtiles * ((outs + cols - 1) / cols) * a.split;
    if (too_many(blocks, 64 * WP * WQ)) return (int)hipErrorInvalidConfiguration;
    void (*k)(const ProductArgs);
    if constexpr (S > 0) k = a.bf16 ? k_product_dma<true, DIR, BP, BQ, WP, WQ, S> : k_product_dma<false, DIR, BP, BQ, WP, WQ, S>;
    else k = a.bf16 ? k_product<true, DIR, BP, BQ, WP, WQ> : k_product<false, DIR, BP, BQ, WP, WQ>;
    hipLaunchKernelGGL(k, dim3((uint32_t)blocks), dim3(64 * WP * WQ), 0, s, a);
    if (a.split > 1) {
        const int64_t rows = DIR == DW ? (int64_t)a.E * a.out : a.rows;
        const int64_t joins = (rows * ((outs + 7) / 8) + 255) / 256;
        if (too_many(joins, 256)) return (int)hipErrorInvalidConfiguration;
        hipLaunchKernelGGL(HIP_KERNEL_NAME(a.bf16 ? k_join<true, DIR> : k_join<false, DIR>), dim3((uint32_t)joins), dim3(256), 0, s, a);
    }
    return (int)hipGetLastError();
}

template <int DIR> static int run_tiles(const ProductArgs& a, Kernel k, hipStream_t s) {
    switch (k) {
    case T256: return run<DIR, 256, 256, 2, 4, 2>(a, s);
    case T128: return run<DIR, 128, 128, 2, 4, 2>(a, s);
    case T64: return run<DIR, 64, 64, 2, 2, 4>(a, s);
    default: break;
    }
    if constexpr (DIR != DW) {
        switch (k) {
        case T128x64: return run<DIR, 128, 64, 4, 2, 3>(a, s);
        case T128x32: return run<DIR, 128, 32, 4, 1, 4>(a, s);
        case T64x32: return run<DIR, 64, 32, 2, 2, 4>(a, s);
        case T64x16: return run<DIR, 64, 16, 2, 1, 4>(a, s);
        case ANY128: return run<DIR, 128, 128, 2, 2, 0>(a, s);
        case ANY32: return run<DIR, 128, 32, 4, 1, 0>(a, s);
        default: break;
        }
    }
    return (int)hipErrorInvalidValue;
}

// 4 waves up to 2048 columns, 8 above: 256 to 512 columns per wave.
template <int NW> static int run_few(const ProductArgs& a, hipStream_t s) {
    const bool gated = a.act == WM_ACT_SWIGLU;
    const int outs = columns(a, FWD), cols = gated ? 8 : 16;
    const int64_t blocks = row_tiles(a, 16) * ((outs + cols - 1) / cols);
    if (too_many(blocks, 64 * NW)) return (int)hipErrorInvalidConfiguration;
    const auto k = a.bf16 ? k_product_few<true, NW> : k_product_few<false, NW>;
    hipLaunchKernelGGL(k, dim3((uint32_t)blocks), dim3(64 * NW), 0, s, a);
    return (int)hipGetLastError();
}

static int repack(const uint16_t* src, int64_t ld_src, int64_t stride_src, int n, int rows, int cols, uint16_t* dst, hipStream_t s) {
    const int ld = (cols + 7) / 8 * 8;
    const int64_t blocks = ((int64_t)rows * (ld / 8) + 255) / 256;
    if (blocks == 0) return 0;
    if (too_many(blocks, 256) || n > 65535) return (int)hipErrorInvalidConfiguration;
    hipLaunchKernelGGL(k_repack, dim3((uint32_t)blocks, n), dim3(256), 0, s, src, ld_src, stride_src, rows, cols, dst, ld, (int64_t)rows * ld);
    return (int)hipGetLastError();
}

// Copies what needs it into the workspace and points the arguments there.
static int copy_operands(ProductArgs& a, const Copies& c, const Layout& l, uint8_t* ws, hipStream_t s) {
    const int64_t in8 = (a.in + 7) / 8 * 8, out8 = (a.out + 7) / 8 * 8;
    if (c.x) {
        if (int rc = repack(a.x, a.ldx, 0, 1, a.x_rows, a.in, (uint16_t*)(ws + l.x), s)) return rc;
        a.x = (const uint16_t*)(ws + l.x);
        a.ldx = in8;
    }
    if (c.w) {
        if (int rc = repack(a.w, a.ldw, a.w_stride, a.E, a.out, a.in, (uint16_t*)(ws + l.w), s)) return rc;
        a.w = (const uint16_t*)(ws + l.w);
        a.ldw = in8;
        a.w_stride = in8 * a.out;
    }
    if (c.dz) {
        if (int rc = repack(a.dz, a.lddz, 0, 1, a.rows, a.out, (uint16_t*)(ws + l.dz), s)) return rc;
        a.dz = (const uint16_t*)(ws + l.dz);
        a.lddz = out8;
    }
    return 0;
}

int launch_product(const ProductArgs& args, uint8_t* ws, hipStream_t s) {
    ProductArgs a = args;
    const Plan p = plan(a, FWD);
    a.split = p.split;
    if (p.k == FEW) return a.in <= 2048 ? run_few<4>(a, s) : run_few<8>(a, s);
    const Copies c = tiled(p) ? copies(a, true, false, false) : Copies{};
    const Layout l = layout(a, c, 0);
    if (int rc = copy_operands(a, c, l, ws, s)) return rc;
    a.part = (float*)(ws + l.part);
    return run_tiles<FWD>(a, p.k, s);
}

int launch_product_backward(const ProductArgs& args, uint8_t* ws, hipStream_t s) {
    ProductArgs a = args;
    const bool dx = a.dx && a.rows, dw = a.dw || a.db;
    const Plan px = dx ? plan(a, DX) : Plan{ANY32, 1};
    const Copies c = copies(a, false, tiled(px), dw && a.rows);
    const Layout l = layout(a, c, 0);
    ProductArgs b = a;
    if (int rc = copy_operands(b, c, l, ws, s)) return rc;
    b.part = (float*)(ws + l.part);
    if (dx) {
        ProductArgs& t = tiled(px) ? b : a;
        t.split = px.split;
        if (int rc = run_tiles<DX>(t, px.k, s)) return rc;
    }
    if (dw) {
        ProductArgs t = b.dw ? b : only_db(b);
        const Plan p = a.rows ? plan(t, DW) : Plan{T128, 1};
        t.split = p.split;
        t.part_db = t.part + (int64_t)p.split * t.E * t.out * t.in;
        return run_tiles<DW>(t, p.k, s);
    }
    return 0;
}

}  // namespace wm
