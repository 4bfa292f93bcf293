// lm_common.cuh -- pieces shared by the language-model operators: the storage-type
// dispatch without f64, and the gate functions in fp32.
#pragma once

#include "dg_common.cuh"

#define DG_DISPATCH_LM(dtype, T, ...)                      \
    switch (dtype) {                                       \
    case DG_DTYPE_F32: { using T = float; __VA_ARGS__; } break;          \
    case DG_DTYPE_F16: { using T = __half; __VA_ARGS__; } break;         \
    case DG_DTYPE_BF16: { using T = __nv_bfloat16; __VA_ARGS__; } break; \
    case DG_DTYPE_F64: return DG_ERR_UNSUPPORTED;          \
    default: return DG_ERR_INVALID_ARGUMENT;               \
    }

namespace dg {

// one special-function operation each, results below the normal range flushed to 0
__device__ __forceinline__ float exp2_ftz(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ float rcp_ftz(float x) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

// a = sigmoid(z) and 1 - a, each to fp32's relative precision: with e = exp(-z),
// a = 1 / (1 + e) and 1 - a = e a.  z is held above -80, where a is 2e-35 (and e finite).
__device__ __forceinline__ void sigmoid_pair(float z, float& a, float& one_minus_a) {
    const float e = exp2_ftz(fminf(z * -1.4426950408889634f, 115.f));
    a = rcp_ftz(1.f + e);
    one_minus_a = e * a;
}
__device__ __forceinline__ float sigmoid(float z) {
    return rcp_ftz(1.f + exp2_ftz(fminf(z * -1.4426950408889634f, 115.f)));
}

// activations of the feed-forward block and their derivatives
template <int ACT>
__device__ __forceinline__ float act_fn(float z) {
    if (ACT == DG_ACT_SILU) return z * sigmoid(z);
    // z/2 (1 + tanh s) = z sigmoid(2 s)
    return z * sigmoid(1.5957691216057308f * fmaf(0.044715f * z * z, z, z));
}
template <int ACT>
__device__ __forceinline__ void act_grad(float z, float& f, float& df) {
    float s, n;
    if (ACT == DG_ACT_SILU) {
        sigmoid_pair(z, s, n);
        f = z * s;
        df = s * fmaf(z, n, 1.f);
    } else {
        const float z2 = z * z;
        sigmoid_pair(1.5957691216057308f * fmaf(0.044715f * z2, z, z), s, n);
        f = z * s;
        df = s * fmaf(z * n, 1.5957691216057308f * fmaf(0.134145f, z2, 1.f), 1.f);
    }
}

}  // namespace dg
