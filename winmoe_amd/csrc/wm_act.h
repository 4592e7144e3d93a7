// wm_act.h -- 16-bit conversions, activations and row accesses of the 16-bit
// operators.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/winmoe_hip.h"
#include "wm_device.h"

namespace wm {

// Round to nearest even, NaN stays NaN.
template <bool BF> WM_DEV uint16_t to16(float v) {
    if constexpr (BF) return __builtin_bit_cast(uint16_t, (__bf16)v);
    else return __builtin_bit_cast(uint16_t, (_Float16)v);
}
template <bool BF> WM_DEV float from16(uint16_t b) {
    if constexpr (BF) return __builtin_bit_cast(float, (uint32_t)b << 16);
    else return (float)__builtin_bit_cast(_Float16, b);
}

WM_DEV float sigmoid(float x) { return 1.0f / (1.0f + expf(-x)); }

// Phi(z), the normal distribution function, and its density.  Phi(-|z|) is
// exp(-z^2 / 2) / 2 times erfcx(|z| / sqrt 2), which falls smoothly from 1: a
// polynomial in t = 1 / (1 + 0.4 x), least squares reweighted towards equal
// relative error on [0, 11], 7e-8 in exact arithmetic and 2.6e-7 in fp32.  So
// it keeps its relative precision in the tail, at one exponential for both
// values (the gradient over 16384 x 4096: 123 us with the library's erfc and
// exp, which bound it, 81 us with this).
WM_DEV void normal(float z, float& cdf, float& pdf) {
    const float a = fminf(fabsf(z), 20.0f), h = 0.5f * a * a;          // exp(-200) is 0
    float e = expf(-h);
    e = fmaf(-fmaf(0.5f * a, a, -h), e, e);                             // what h lost in rounding
    const float t = __builtin_amdgcn_rcpf(fmaf(0.4f * 0.70710678f, a, 1.0f));
    float p = 0.04288169f;
    p = fmaf(p, t, -0.14826289f);
    p = fmaf(p, t, 0.10044732f);
    p = fmaf(p, t, 0.06909195f);
    p = fmaf(p, t, 0.09281324f);
    p = fmaf(p, t, 0.18782872f);
    p = fmaf(p, t, 0.2033099f);
    p = fmaf(p, t, 0.2262443f);
    p = fmaf(p, t, 0.22564584f);
    const float q = 0.5f * (p * t) * e;
    cdf = z > 0.0f ? 1.0f - q : q;
    pdf = 0.39894228f * e;
}

// y = act(z); SwiGLU: silu(z) * u.  GELU is the exact one, z * Phi(z).
WM_DEV float act_value(int act, float z, float u) {
    switch (act) {
    case WM_ACT_RELU: return z < 0.0f ? 0.0f : z;
    case WM_ACT_SILU: return z * sigmoid(z);
    case WM_ACT_GELU: {
        float cdf, pdf;
        normal(z, cdf, pdf);
        return z * cdf;
    }
    case WM_ACT_SWIGLU: return z * sigmoid(z) * u;
    case WM_ACT_SIGMOID: return sigmoid(z);
    default: return z;
    }
}

// d act / dz; for SwiGLU of silu(z) alone.
WM_DEV float act_slope(int act, float z) {
    switch (act) {
    case WM_ACT_RELU: return z > 0.0f ? 1.0f : 0.0f;
    case WM_ACT_GELU: {
        float cdf, pdf;
        normal(z, cdf, pdf);
        return fmaf(z, pdf, cdf);
    }
    case WM_ACT_SILU:
    case WM_ACT_SWIGLU: {
        const float s = sigmoid(z);
        return s * (1.0f + z * (1.0f - s));
    }
    case WM_ACT_SIGMOID: {
        const float s = sigmoid(z);
        return s * (1.0f - s);
    }
    default: return 1.0f;
    }
}

// ------------------------------------------------------------------ 8 values at a time

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

// The same as fp32.
template <bool BF> WM_DEV void unpack8(uint4 raw, float* v) {
    uint16_t e[8];
    __builtin_memcpy(e, &raw, 16);
#pragma unroll
    for (int i = 0; i < 8; i++) v[i] = from16<BF>(e[i]);
}
template <bool BF> WM_DEV void get8(const uint16_t* p, int n, float* v) { unpack8<BF>(load8(p, n), v); }
template <bool BF> WM_DEV void put8(uint16_t* p, int n, const float* v) {
    uint16_t e[8];
#pragma unroll
    for (int i = 0; i < 8; i++) e[i] = to16<BF>(v[i]);
    if (n >= 8) {
        __builtin_memcpy(p, e, 16);
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++)
            if (i < n) p[i] = e[i];
    }
}
WM_DEV void getf8(const float* p, int n, float* v) {
    if (n >= 8) {
        __builtin_memcpy(v, p, 32);
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = i < n ? p[i] : 0.0f;
    }
}
WM_DEV void putf8(float* p, int n, const float* v) {
    if (n >= 8) {
        __builtin_memcpy(p, v, 32);
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++)
            if (i < n) p[i] = v[i];
    }
}

}  // namespace wm
