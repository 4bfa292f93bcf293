// gated_ffn_few.cu -- the gated feed-forward block for a few tokens (f16 / bf16), up to 32: bound
// by reading the 2 F D weights once and, where they are small, by latency (one token of 768 x 768
// 2.2 us; 8 of 2048 x 5504, 45 MB, 11 us, 0.64 of what HBM allows).
//
// The weights go from global memory straight into matrix fragments (mma.sync m16n8k16): rows
// 0-7 of a fragment are eight gate rows, rows 8-15 the value rows of the same features, and
// the columns are tokens, so a thread ends with gate and value of the same feature and token.
// A sum over k may take k in any order, so lane t of a row's four loads 16 consecutive bytes
// (eight k, two fragments' worth) of each of its two rows and of its token's x, and no
// operand passes through shared memory.
//
// The eight warps of a CTA take the 64-byte pieces of the same 8 G rows in turn, whole
// 512-byte runs together, U pieces in flight each; their sums meet in shared memory, where
// the activation, the product and the one rounding follow.
#include "lm_common.cuh"

namespace {

constexpr int THREADS = 256;
constexpr int WARPS = THREADS / 32;
constexpr int CHUNK = 32;                  // contracted elements per piece

template <typename T>
__device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                    uint32_t b1) {
    if constexpr (std::is_same<T, __half>::value)
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Weights are read once: past L1.  (Not by the read-only path: a kernel in front of this one may write what it
// reads after this one has started.)
__device__ __forceinline__ uint4 load_once(const void* p) {
    uint4 v;
    asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p) : "memory");
    return v;
}

// NT: blocks of eight tokens.  G: groups of eight features per CTA.  U: pieces in flight per warp.
template <typename T, int ACT, int NT, int G, int U>
__global__ void __launch_bounds__(THREADS)
    ffn_few_kernel(int M, int D, int F, const T* x, int64_t ldx, const T* w, const T* bias, T* h) {
    __shared__ float part[WARPS][G][NT][4][32];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, row = lane >> 2, k8 = (lane & 3) * 8;
    const int f0 = blockIdx.x * 8 * G, chunks = (D + CHUNK - 1) / CHUNK;
    const uint4 zero = make_uint4(0, 0, 0, 0);
    float c[G][NT][4] = {};
    dg::let_next_start();
    dg::wait_for_previous();
    const T* wg[G];
#pragma unroll
    for (int i = 0; i < G; ++i) wg[i] = w + (int64_t)min(f0 + 8 * i + row, F - 1) * D + k8;       // (beyond F: not written)
    const int64_t up = (int64_t)F * D;
    for (int base = warp; base < chunks; base += WARPS * U) {
        uint4 ag[U][G], au[U][G], b[U][NT];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int k = (base + u * WARPS) * CHUNK;
            const bool on = k + k8 < D;
#pragma unroll
            for (int i = 0; i < G; ++i) {
                ag[u][i] = on ? load_once(wg[i] + k) : zero;
                au[u][i] = on ? load_once(wg[i] + up + k) : zero;
            }
#pragma unroll
            for (int n = 0; n < NT; ++n)
                b[u][n] = on && 8 * n + row < M ? dg::ld16(x + (8 * n + row) * ldx + k + k8) : zero;
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int i = 0; i < G; ++i)
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    mma<T>(c[i][n], ag[u][i].x, au[u][i].x, ag[u][i].y, au[u][i].y, b[u][n].x, b[u][n].y);
                    mma<T>(c[i][n], ag[u][i].z, au[u][i].z, ag[u][i].w, au[u][i].w, b[u][n].z, b[u][n].w);
                }
    }
#pragma unroll
    for (int i = 0; i < G; ++i)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) part[warp][i][n][e][lane] = c[i][n][e];
    __syncthreads();
    // outputs (group, token block, odd or even token, lane)
    for (int o = threadIdx.x; o < G * NT * 64; o += THREADS) {
        const int l = o & 31, odd = (o >> 5) & 1, n = (o >> 6) % NT, i = (o >> 6) / NT;
        const int f = f0 + 8 * i + (l >> 2), m = 8 * n + 2 * (l & 3) + odd;
        if (m >= M || f >= F) continue;
        float g = 0.f, u = 0.f;
#pragma unroll
        for (int v = 0; v < WARPS; ++v) g += part[v][i][n][odd][l], u += part[v][i][n][2 + odd][l];
        if (bias) g += dg::to_f(bias[f]), u += dg::to_f(bias[F + f]);
        h[(int64_t)m * F + f] = dg::from_f<T>(dg::act_fn<ACT>(g) * u);
    }
}

template <typename T, int NT, int G, int U>
int run(int act, int M, int D, int F, const void* x, int64_t ldx, const void* w, const void* bias, void* h, cudaStream_t s) {
    auto k = act == DG_ACT_SILU ? ffn_few_kernel<T, DG_ACT_SILU, NT, G, U> : ffn_few_kernel<T, DG_ACT_GELU, NT, G, U>;
    return dg_host::launch_lm(k, dim3((unsigned)((F / 8 + G - 1) / G)), dim3(THREADS), 0, 0, 0, s, M, D, F, (const T*)x, ldx,
                              (const T*)w, (const T*)bias, (T*)h);
}

template <typename T>
int by_tokens(int act, int M, int D, int F, const void* x, int64_t ldx, const void* w, const void* bias, void* h,
              cudaStream_t s) {
    // two feature groups share a load of x where that leaves every SM two CTAs
    const bool two = F / 16 >= 2 * 148;
    if (M <= 8) return two ? run<T, 1, 2, 2>(act, M, D, F, x, ldx, w, bias, h, s) : run<T, 1, 1, 4>(act, M, D, F, x, ldx, w, bias, h, s);
    if (M <= 16) return two ? run<T, 2, 2, 2>(act, M, D, F, x, ldx, w, bias, h, s) : run<T, 2, 1, 4>(act, M, D, F, x, ldx, w, bias, h, s);
    return two ? run<T, 4, 2, 2>(act, M, D, F, x, ldx, w, bias, h, s) : run<T, 4, 1, 2>(act, M, D, F, x, ldx, w, bias, h, s);
}

}  // namespace

namespace dg_host {

// Whether this form is taken rather than the split one (16-bit types, D and F multiples of 8, aligned rows).
// It starts faster, but every weight byte meets 1/8 byte of x for each token, from L2, and a CTA's eight
// features take all of D.  Up to 8 tokens it wins below 64 MB of weights (768 x 768: 2.2 us against 4.8;
// 2048 x 5504, 45 MB: 10.6 against 10.9; 4096 x 11008, 180 MB: 36 against 33), up to 16 below 12 MB and up to
// 32 below 8 MB (32 x 768 x 768: 4.0 us against 5.2; 32 x 1536 x 2048: 9.0 against 7.6), D not long (16 x 4096
// x 400: 10.8 against 6.9).
bool ffn_few_supports(int64_t M, int D, int F) {
    const int64_t bytes = (int64_t)4 * F * D;
    return M <= 8 ? bytes <= 64 << 20 : D <= 2048 && ((M <= 16 && bytes <= 12 << 20) || (M <= 32 && bytes <= 8 << 20));
}

int ffn_few_forward(int dtype, int64_t M, int D, int F, int act, const void* x, int64_t ldx, const void* w,
                    const void* bias, void* h, cudaStream_t s) {
    return dtype == DG_DTYPE_F16 ? by_tokens<__half>(act, (int)M, D, F, x, ldx, w, bias, h, s)
                                 : by_tokens<__nv_bfloat16>(act, (int)M, D, F, x, ldx, w, bias, h, s);
}

}  // namespace dg_host
