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

// y = act(z); SwiGLU: silu(z) * u.  GELU is the exact one, z * Phi(z), with
// Phi through erfc so that it keeps its relative precision for z < 0.
WM_DEV float act_value(int act, float z, float u) {
    switch (act) {
    case WM_ACT_RELU: return z < 0.0f ? 0.0f : z;
    case WM_ACT_SILU: return z * sigmoid(z);
    case WM_ACT_GELU: return z * (0.5f * erfcf(-0.70710678f * z));
    case WM_ACT_SWIGLU: return z * sigmoid(z) * u;
    default: return z;
    }
}

// d act / dz; for SwiGLU of silu(z) alone.
WM_DEV float act_slope(int act, float z) {
    switch (act) {
    case WM_ACT_RELU: return z > 0.0f ? 1.0f : 0.0f;
    case WM_ACT_GELU: return 0.5f * erfcf(-0.70710678f * z) + z * (0.39894228f * expf(-0.5f * z * z));
    case WM_ACT_SILU:
    case WM_ACT_SWIGLU: {
        const float s = sigmoid(z);
        return s * (1.0f + z * (1.0f - s));
    }
    default: return 1.0f;
    }
}

// ------------------------------------------------------------------ 8 values at a time

// 8 values at p, of which the first n exist, as fp32; no alignment needed.
template <bool BF> WM_DEV void get8(const uint16_t* p, int n, float* v) {
    uint16_t e[8];
    if (n >= 8) {
        __builtin_memcpy(e, p, 16);
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) e[i] = i < n ? p[i] : 0;
    }
#pragma unroll
    for (int i = 0; i < 8; i++) v[i] = from16<BF>(e[i]);
}
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
