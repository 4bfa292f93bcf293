// gated_ffn.cu -- the gated feed-forward block h = act(x Wg^T + bg) * (x Wu^T + bu) and its
// backward pass on CUDA cores: 64 x 64 output tiles, 16 of the contracted axis at a time
// through shared memory, 4 x 4 outputs per thread.  These kernels take any storage type, size
// and alignment; 16-bit calls with D and F multiples of 8 and 16-byte aligned rows go to the
// tcgen05 kernel of gated_ffn_tc.cu or, forward with up to 256 tokens, to gated_ffn_few.cu and
// gated_ffn_split.cu.  Bound by shared-memory reads and issue: 16384 x 768 x 768 takes 1.4 ms
// (27 TFLOP/s).
#include "lm_common.cuh"

namespace dg_host {
bool ffn_tc_supports(int dtype, int64_t M, int D, int F);
bool ffn_tc_aligned(const void* a, int64_t lda, const void* b, const void* c, const void* d, int64_t ldd,
                    const void* e, const void* f);
bool ffn_few_supports(int64_t M, int D, int F);
int ffn_few_forward(int dtype, int64_t M, int D, int F, int act, const void* x, int64_t ldx, const void* w,
                    const void* bias, void* h, cudaStream_t s);
int ffn_tc_forward(int dtype, int64_t M, int D, int F, int act, const void* x, int64_t ldx, const void* w,
                   const void* bias, void* h, int32_t* status, cudaStream_t s);
bool ffn_split_supports(int64_t M, int D, int F);
int ffn_split_forward(int dtype, int64_t M, int D, int F, int act, const void* x, int64_t ldx, const void* w,
                      const void* bias, void* h, int32_t* status, cudaStream_t s);
size_t ffn_tc_workspace(int64_t M, int D, int F);
int ffn_tc_backward(int dtype, int64_t M, int D, int F, int act, const void* x, int64_t ldx, const void* w,
                    const void* bias, const void* dh, int64_t ld_dh, void* dx, void* dw, void* db, void* workspace,
                    int32_t* status, cudaStream_t s);
}  // namespace dg_host

namespace {

constexpr int TM = 64, TN = 64, TK = 16, THREADS = 256;

// rows of a tile: value (r, k) of an operand with element strides (rs, ks), zero outside
template <typename T>
__device__ __forceinline__ void load_tile(float (*dst)[TM + 4], const T* p, int64_t rs, int64_t ks, int64_t r0,
                                          int64_t rows, int64_t k0, int64_t K) {
    for (int i = threadIdx.x; i < TM * TK; i += THREADS) {
        // neighbouring threads along the operand's contiguous axis
        const int r = ks == 1 ? i / TK : i % TM, k = ks == 1 ? i % TK : i / TM;
        dst[k][r] = (r0 + r < rows && k0 + k < K) ? dg::to_f(p[(r0 + r) * rs + (k0 + k) * ks]) : 0.f;
    }
}

__device__ __forceinline__ void mac_tile(float (&acc)[4][4], const float (*a)[TM + 4], const float (*b)[TN + 4]) {
    const int tr = (threadIdx.x / 16) * 4, tc = (threadIdx.x % 16) * 4;
#pragma unroll
    for (int k = 0; k < TK; ++k) {
        const float4 av = *reinterpret_cast<const float4*>(&a[k][tr]), bv = *reinterpret_cast<const float4*>(&b[k][tc]);
        const float ar[4] = {av.x, av.y, av.z, av.w}, br[4] = {bv.x, bv.y, bv.z, bv.w};
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(ar[i], br[j], acc[i][j]);
    }
}

// G and U of a tile, then h (dh null) or dG and dU into dz [M,2F] and their column sums over
// the tile's rows into colsum [row tiles, 2F]
template <typename T, int ACT>
__global__ void __launch_bounds__(THREADS)
    ffn_gate_kernel(int64_t M, int D, int F, const T* x, int64_t ldx, const T* w, const T* bias, T* h, const T* dh,
                    int64_t ld_dh, T* dz, float* colsum) {
    __shared__ __align__(16) float sx[TK][TM + 4], sg[TK][TN + 4], su[TK][TN + 4];
    __shared__ float cs[2][16][TN];
    const int64_t m0 = (int64_t)blockIdx.y * TM;
    const int f0 = blockIdx.x * TN;
    float g[4][4] = {}, u[4][4] = {};
    for (int k0 = 0; k0 < D; k0 += TK) {
        load_tile(sx, x, ldx, 1, m0, M, k0, D);
        load_tile(sg, w, D, 1, f0, F, k0, D);
        load_tile(su, w + (int64_t)F * D, D, 1, f0, F, k0, D);
        __syncthreads();
        mac_tile(g, sx, sg);
        mac_tile(u, sx, su);
        __syncthreads();
    }
    const int tr = (threadIdx.x / 16) * 4, tc = (threadIdx.x % 16) * 4;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int f = f0 + tc + j;
        const float bg = bias && f < F ? dg::to_f(bias[f]) : 0.f, bu = bias && f < F ? dg::to_f(bias[F + f]) : 0.f;
        float sum_g = 0.f, sum_u = 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int64_t m = m0 + tr + i;
            const float gv = g[i][j] + bg, uv = u[i][j] + bu;
            if (m >= M || f >= F) continue;
            if (!dh) {
                h[m * F + f] = dg::from_f<T>(dg::act_fn<ACT>(gv) * uv);
            } else {
                float a, da;
                dg::act_grad<ACT>(gv, a, da);
                const float d = dg::to_f(dh[m * ld_dh + f]);
                const float zg = d * uv * da, zu = d * a;      // stored in T, as the tensor-core kernels have to
                dz[m * 2 * F + f] = dg::from_f<T>(zg);
                dz[m * 2 * F + F + f] = dg::from_f<T>(zu);
                sum_g += zg;
                sum_u += zu;
            }
        }
        if (colsum) {
            cs[0][threadIdx.x / 16][tc + j] = sum_g;
            cs[1][threadIdx.x / 16][tc + j] = sum_u;
        }
    }
    if (colsum) {
        __syncthreads();
        if (threadIdx.x < 2 * TN) {
            const int half = threadIdx.x / TN, c = threadIdx.x % TN;
            float s = 0.f;
            for (int r = 0; r < 16; ++r) s += cs[half][r][c];
            if (f0 + c < F) colsum[(int64_t)blockIdx.y * 2 * F + half * F + f0 + c] = s;
        }
    }
}

// C [M,N] = A B with A(m,k) and B(n,k) of any strides
template <typename T>
__global__ void __launch_bounds__(THREADS)
    ffn_product_kernel(int64_t M, int N, int64_t K, const T* a, int64_t a_rs, int64_t a_ks, const T* b, int64_t b_rs,
                       int64_t b_ks, T* c) {
    __shared__ __align__(16) float sa[TK][TM + 4], sb[TK][TN + 4];
    const int64_t m0 = (int64_t)blockIdx.y * TM;
    const int n0 = blockIdx.x * TN;
    float acc[4][4] = {};
    for (int64_t k0 = 0; k0 < K; k0 += TK) {
        load_tile(sa, a, a_rs, a_ks, m0, M, k0, K);
        load_tile(sb, b, b_rs, b_ks, n0, N, k0, K);
        __syncthreads();
        mac_tile(acc, sa, sb);
        __syncthreads();
    }
    const int tr = (threadIdx.x / 16) * 4, tc = (threadIdx.x % 16) * 4;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (m0 + tr + i < M && n0 + tc + j < N) c[(m0 + tr + i) * N + n0 + tc + j] = dg::from_f<T>(acc[i][j]);
}

// dbias[c] = sum over row tiles, in order
template <typename T>
__global__ void ffn_colsum_kernel(int tiles, int cols, const float* part, T* out) {
    const int c = blockIdx.x * blockDim.x + threadIdx.x;
    if (c >= cols) return;
    float s = 0.f;
    for (int t = 0; t < tiles; ++t) s += part[(int64_t)t * cols + c];
    out[c] = dg::from_f<T>(s);
}

size_t round16(size_t n) { return (n + 15) & ~size_t(15); }

int check_args(int dtype, int64_t M, int D, int F, int activation) {
    if (dtype == DG_DTYPE_F64) return DG_ERR_UNSUPPORTED;
    if (dtype < DG_DTYPE_F32 || dtype > DG_DTYPE_BF16 || M < 0 || D <= 0 || F <= 0) return DG_ERR_INVALID_ARGUMENT;
    if (activation != DG_ACT_SILU && activation != DG_ACT_GELU) return DG_ERR_INVALID_ARGUMENT;
    if (M > (int64_t)65535 * TM || F > (1 << 20) || D > (1 << 24)) return DG_ERR_UNSUPPORTED;    // grid limits
    return DG_OK;
}

}  // namespace

extern "C" {

int dg_gated_ffn_forward(int dtype, int64_t M, int D, int F, int activation, const void* x, int64_t ldx,
                         const void* weight, const void* bias, void* h, int32_t* dev_status, void* stream) {
    const int rc = check_args(dtype, M, D, F, activation);
    if (rc != DG_OK) return rc;
    if (M == 0) return DG_OK;
    if (!x || !weight || !h || ldx < D) return DG_ERR_INVALID_ARGUMENT;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (dg_host::ffn_tc_supports(dtype, M, D, F) && dg_host::ffn_tc_aligned(x, ldx, weight, bias, h, 0, h, h)) {
        if (dg_host::ffn_few_supports(M, D, F))
            return dg_host::ffn_few_forward(dtype, M, D, F, activation, x, ldx, weight, bias, h, s);
        if (dg_host::ffn_split_supports(M, D, F))
            return dg_host::ffn_split_forward(dtype, M, D, F, activation, x, ldx, weight, bias, h, dev_status, s);
        return dg_host::ffn_tc_forward(dtype, M, D, F, activation, x, ldx, weight, bias, h, dev_status, s);
    }
    const dim3 grid((F + TN - 1) / TN, (unsigned)((M + TM - 1) / TM));
    DG_DISPATCH_LM(dtype, S, {
        auto k = activation == DG_ACT_SILU ? ffn_gate_kernel<S, DG_ACT_SILU> : ffn_gate_kernel<S, DG_ACT_GELU>;
        k<<<grid, THREADS, 0, s>>>(M, D, F, (const S*)x, ldx, (const S*)weight, (const S*)bias, (S*)h, nullptr, 0,
                                   nullptr, nullptr);
    });
    return dg_host::check_launch();
}

size_t dg_gated_ffn_backward_workspace_size(int dtype, int64_t M, int D, int F) {
    if (check_args(dtype, M, D, F, DG_ACT_SILU) != DG_OK) return 0;
    const size_t simple =
        round16((size_t)M * 2 * F * dg_host::dtype_size(dtype)) + round16((size_t)((M + TM - 1) / TM) * 2 * F * 4);
    const size_t tc = dg_host::ffn_tc_supports(dtype, M, D, F) ? dg_host::ffn_tc_workspace(M, D, F) : 0;
    return simple > tc ? simple : tc;
}

int dg_gated_ffn_backward(int dtype, int64_t M, int D, int F, int activation, const void* x, int64_t ldx,
                          const void* weight, const void* bias, const void* dh, int64_t ld_dh, void* dx,
                          void* dweight, void* dbias, void* workspace, size_t workspace_bytes,
                          int32_t* dev_status, void* stream) {
    const int rc = check_args(dtype, M, D, F, activation);
    if (rc != DG_OK) return rc;
    if (!weight || (M > 0 && (!x || !dh || ldx < D || ld_dh < F))) return DG_ERR_INVALID_ARGUMENT;
    if (M > 0 && (!workspace || workspace_bytes < dg_gated_ffn_backward_workspace_size(dtype, M, D, F) ||
                  (reinterpret_cast<uintptr_t>(workspace) & 15)))
        return DG_ERR_WORKSPACE;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (M > 0 && dg_host::ffn_tc_supports(dtype, M, D, F) &&
        dg_host::ffn_tc_aligned(x, ldx, weight, bias, dh, ld_dh, dx, dweight))
        return dg_host::ffn_tc_backward(dtype, M, D, F, activation, x, ldx, weight, bias, dh, ld_dh, dx, dweight,
                                        dbias, workspace, dev_status, s);
    const unsigned mt = (unsigned)((M + TM - 1) / TM);
    DG_DISPATCH_LM(dtype, S, {
        S* dz = static_cast<S*>(workspace);
        float* part = dbias ? reinterpret_cast<float*>(static_cast<char*>(workspace) +
                                                       round16((size_t)M * 2 * F * sizeof(S))) : nullptr;
        if (M > 0) {
            auto k = activation == DG_ACT_SILU ? ffn_gate_kernel<S, DG_ACT_SILU> : ffn_gate_kernel<S, DG_ACT_GELU>;
            k<<<dim3((F + TN - 1) / TN, mt), THREADS, 0, s>>>(M, D, F, (const S*)x, ldx, (const S*)weight,
                                                              (const S*)bias, nullptr, (const S*)dh, ld_dh, dz, part);
            if (dx)
                ffn_product_kernel<S><<<dim3((D + TN - 1) / TN, mt), THREADS, 0, s>>>(
                    M, D, 2 * (int64_t)F, dz, 2 * (int64_t)F, 1, (const S*)weight, 1, D, (S*)dx);
        }
        if (dweight)
            ffn_product_kernel<S><<<dim3((D + TN - 1) / TN, (2 * F + TM - 1) / TM), THREADS, 0, s>>>(
                2 * F, D, M, dz, 1, 2 * (int64_t)F, (const S*)x, 1, ldx, (S*)dweight);
        if (dbias) ffn_colsum_kernel<S><<<(2 * F + 255) / 256, 256, 0, s>>>((int)mt, 2 * F, part, (S*)dbias);
    });
    return dg_host::check_launch();
}

}  // extern "C"
