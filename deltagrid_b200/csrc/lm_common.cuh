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

// Programmatic dependent launch: a kernel lets the next one of its stream start as soon as its own blocks
// leave room, and touches no memory before the kernel in front of it has completed, so that launch
// latency and set-up run under the end of the work before (about 2 us a kernel back to back).  Such a kernel's
// inputs may still be written after it has started, so it loads none by the read-only path (ld.global.nc).
__device__ __forceinline__ void let_next_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void wait_for_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

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

// the smaller and the larger of two; a NaN stays one
__device__ __forceinline__ float min_nan(float a, float b) {
    float r;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

// The recurrence's gate: a = sigmoid(z) = 1 / (1 + e) with e = exp(-z), and 1 - a, as e a where e is small
// and a near 1, else by the difference (e may be infinite: a is 0 there and forgets any state).  A NaN
// stays one in both.  z log2(e) is rounded once, so e and the smaller of the two carry |z| 2^-24 relative.
__device__ __forceinline__ void sigmoid_pair(float z, float& a, float& one_minus_a) {
    const float e = exp2_ftz(z * -1.4426950408889634f);
    a = rcp_ftz(1.f + e);
    one_minus_a = e > 1.f ? 1.f - a : e * a;
}
// sigmoid(z) for z sigmoid(z): 0 for z below -88, where 1 + exp(-z) has no normal inverse, and so the product
__device__ __forceinline__ float sigmoid(float z) { return rcp_ftz(1.f + exp2_ftz(z * -1.4426950408889634f)); }
// s = sigmoid(z) and n = 1 - s for a slope s (1 + z n ...): both are 0 for z below -88, and so the slope
__device__ __forceinline__ void slope_pair(float z, float& s, float& n) {
    const float e = fminf(exp2_ftz(z * -1.4426950408889634f), 3.4e38f);
    s = rcp_ftz(1.f + e);
    n = e * s;
}

// two fp32 values at a time (the two-wide instructions of sm_100)
struct F2 {
    float x, y;
};
__device__ __forceinline__ uint64_t f2_bits(F2 a) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a.x), "f"(a.y));
    return r;
}
__device__ __forceinline__ F2 f2_from(uint64_t a) {
    F2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(a));
    return r;
}
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(f2_bits(a)), "l"(f2_bits(b)), "l"(f2_bits(c)));
    return f2_from(r);
}
__device__ __forceinline__ F2 mul2(F2 a, F2 b) {
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(f2_bits(a)), "l"(f2_bits(b)));
    return f2_from(r);
}
__device__ __forceinline__ F2 add2(F2 a, F2 b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(f2_bits(a)), "l"(f2_bits(b)));
    return f2_from(r);
}
__device__ __forceinline__ F2 both(float a) { return {a, a}; }

// slope_pair of two values
__device__ __forceinline__ void slope_pair2(F2 z, F2& s, F2& n) {
    F2 e = mul2(z, both(-1.4426950408889634f));
    e.x = fminf(exp2_ftz(e.x), 3.4e38f);
    e.y = fminf(exp2_ftz(e.y), 3.4e38f);
    s = add2(e, both(1.f));
    s.x = rcp_ftz(s.x);
    s.y = rcp_ftz(s.y);
    n = mul2(e, s);
}
__device__ __forceinline__ F2 sigmoid2(F2 z) {
    F2 e = mul2(z, both(-1.4426950408889634f));
    e.x = exp2_ftz(e.x);
    e.y = exp2_ftz(e.y);
    e = add2(e, both(1.f));
    return {rcp_ftz(e.x), rcp_ftz(e.y)};
}
// Activations of the feed-forward block and their derivatives.  GELU's tanh form is z sigmoid(2 s), s =
// sqrt(2 / pi) (z + 0.044715 z^3); its slope is formed at z held to +-12, beyond which it is 0 or 1 to
// fp32 (2 s is 142 there) and z^2 may leave fp32.
__device__ __forceinline__ float held(float z) { return min_nan(max_nan(z, -12.f), 12.f); }
template <int ACT>
__device__ __forceinline__ float act_fn(float z) {
    if (ACT == DG_ACT_SILU) return z * sigmoid(z);
    return z * sigmoid(1.5957691216057308f * fmaf(0.044715f * z * z, z, z));
}
template <int ACT>
__device__ __forceinline__ void act_grad(float z, float& f, float& df) {
    float s, n;
    if (ACT == DG_ACT_SILU) {
        slope_pair(z, s, n);
        df = s * fmaf(z, n, 1.f);
    } else {
        const float h = held(z), h2 = h * h;
        slope_pair(1.5957691216057308f * fmaf(0.044715f * h2, h, h), s, n);
        df = s * fmaf(h * n, 1.5957691216057308f * fmaf(0.134145f, h2, 1.f), 1.f);
    }
    f = z * s;
}

template <int ACT> __device__ __forceinline__ F2 act_fn2(F2 z) {
    if (ACT == DG_ACT_SILU) return mul2(z, sigmoid2(z));
    const F2 z2 = mul2(z, z);
    return mul2(z, sigmoid2(mul2(both(1.5957691216057308f), fma2(mul2(both(0.044715f), z2), z, z))));
}
template <int ACT> __device__ __forceinline__ void act_grad2(F2 z, F2& f, F2& df) {
    F2 s, n;
    if (ACT == DG_ACT_SILU) {
        slope_pair2(z, s, n);
        df = mul2(s, fma2(z, n, both(1.f)));
    } else {
        const F2 h{held(z.x), held(z.y)}, h2 = mul2(h, h);
        slope_pair2(mul2(both(1.5957691216057308f), fma2(mul2(both(0.044715f), h2), h, h)), s, n);
        const F2 slope = mul2(both(1.5957691216057308f), fma2(both(0.134145f), h2, both(1.f)));
        df = mul2(s, fma2(mul2(h, n), slope, both(1.f)));
    }
    f = mul2(z, s);
}

}  // namespace dg

namespace dg_host {
// Clusters of 1..16 CTAs that are resident at once on a whole B200 with 1, 2 or 3 such CTAs to an SM
// (cudaOccupancyMaxActiveClusters; a cluster stays inside one group of SMs)
constexpr int kClusters[3][16] = {{148, 74, 45, 33, 26, 22, 15, 15, 15, 11, 7, 7, 7, 7, 7, 7},
                                  {296, 148, 93, 71, 56, 45, 37, 33, 30, 26, 21, 21, 17, 14, 14, 14},
                                  {444, 222, 142, 104, 82, 71, 56, 48, 45, 41, 31, 31, 28, 24, 24, 21}};
// Launches with programmatic dependent launch and, with cluster > 0, that cluster size.  most_smem: the dynamic
// shared memory of the kernel's largest launch; its limit is always set to that, so that another host
// thread's smaller launch does not lower it between this one's setting and launch.
template <typename... P, typename... A>
int launch_lm(void (*kern)(P...), dim3 grid, dim3 block, size_t smem, size_t most_smem, int cluster, cudaStream_t stream,
              A... args) {
    cudaError_t e;
    if (smem > most_smem) return DG_ERR_UNSUPPORTED;
    if (most_smem > 16 * 1024) {               // (static shared memory counts against the 48 KB too)
        e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)most_smem);
        if (e != cudaSuccess) return record_cuda_error(e);
    }
    if (cluster > 8) {
        e = cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
        if (e != cudaSuccess) return record_cuda_error(e);
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = (unsigned)cluster;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = cluster > 0 ? 2 : 1;
    e = cudaLaunchKernelEx(&cfg, kern, static_cast<P>(args)...);
    if (e != cudaSuccess) return record_cuda_error(e);
    return check_launch();
}
}  // namespace dg_host
