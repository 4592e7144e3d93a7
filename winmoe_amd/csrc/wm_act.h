// wm_act.h -- 16-bit conversions and activations of the 16-bit operators.
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

}  // namespace wm
