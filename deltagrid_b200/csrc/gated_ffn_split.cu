// gated_ffn_split.cu -- the gated feed-forward block for up to 256 tokens on tcgen05 (f16 / bf16):
// bound by reading the 2 F D weights once, so every SM has to read its share of them at once.
//
// The weights are the rows of the product and the tokens its columns: a CTA multiplies 64 gate
// rows and the 64 value rows of the same features (M = 128) with all tokens (N = 16 .. 256) over
// a part of the contracted axis, and the CTAs of a cluster take the parts of the same features.
// The accumulator (TMEM lane = weight row, column = token) goes to shared memory in fp32; then
// each CTA of the cluster takes a share of the tokens, adds the parts in their order through
// distributed shared memory and applies bias, activation and product: one rounding, and the same
// sum on every run.
//
// Roles (256 threads): warp 4 loads stages by TMA, warp 5 issues the MMAs; then all warps read the
// accumulator (half of the columns each) and finish the outputs.  Waits are bounded by the
// library's wait limit.
//
// 13 x 2048 x 5504 (45 MB of weights) takes 11.1 us, 0.63 of what HBM allows; 32 x 4096 x 11008
// (180 MB) 33.5 us, 0.83; launch, first loads and the exchange take the rest (4.6 us where the
// weights are 2 MB).  Per CTA 128 rows of weights, not 256 in a pair: tiles of half the features
// let twice as many SMs load.
#include <cuda.h>

#include "chunk_common.cuh"
#include "lm_common.cuh"

namespace dg_host {
uint32_t wait_limit();
}

namespace {

constexpr int THREADS = 256;
constexpr int FEATURES = 64;               // of a CTA
constexpr int BK = 64;                     // contracted elements per stage: 128 bytes
constexpr uint32_t W_TILE = 2 * FEATURES * BK * 2;
constexpr int MAX_STAGES = 8;
constexpr uint32_t MOST_ROOM = 216 * 1024;  // for stages, of one CTA on an SM

struct SplitParams {
    int M, N, F;                           // N: tokens rounded up to 16
    int blocks, per_split, splits, stages; // stages of the contracted axis, in all and of a CTA
    uint32_t columns;                      // TMEM columns
    const void* bias;
    void* h;
    int32_t* status;
    uint32_t wait_limit;
};

__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ float4 remote_load(const float* p, uint32_t rank) {
    uint32_t a;
    float4 v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(tc::smem_u32(p)), "r"(rank));
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(a) : "memory");
    return v;
}
__device__ __forceinline__ void add(float4& a, const float4& b) { a.x += b.x, a.y += b.y, a.z += b.z, a.w += b.w; }

template <typename T, int ACT>
__global__ void __launch_bounds__(THREADS)
    ffn_split_kernel(const __grid_constant__ CUtensorMap tmw, const __grid_constant__ CUtensorMap tmx, SplitParams p) {
    constexpr bool BF16 = !std::is_same<T, __half>::value;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* sm = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    float* part = reinterpret_cast<float*>(sm);        // [N][128], after the products
    __shared__ uint64_t full[MAX_STAGES], empty[MAX_STAGES], done;
    __shared__ uint32_t tmem_holder;
    __shared__ int aborted;
    const int tid = threadIdx.x, warp = tid >> 5;
    const int rank = p.splits > 1 ? (int)cluster_rank() : 0;
    const int f0 = (int)(blockIdx.x / p.splits) * FEATURES;
    const int kb0 = rank * p.per_split, kb1 = min(kb0 + p.per_split, p.blocks);
    const uint32_t stage = W_TILE + (uint32_t)p.N * BK * 2;

    if (warp == 0) tc::tmem_alloc(&tmem_holder, p.columns);
    if (tid == 32) {
        for (int i = 0; i < p.stages; ++i) {
            tc::mbar_init(full + i, 1);
            tc::mbar_init(empty + i, 1);
        }
        tc::mbar_init(&done, 1);
        aborted = 0;
        tc::fence_barrier_init();
    }
    if (tid == 128) {
        tc::prefetch_tmap(&tmw);
        tc::prefetch_tmap(&tmx);
    }
    tc::tc_fence_before();
    __syncthreads();
    tc::tc_fence_after();
    dg::let_next_start();
    dg::wait_for_previous();
    const uint32_t tmem = tmem_holder;
    bool bad = false;

    if (tid == 128) {
        int s = 0;
        uint32_t ph = 1;                   // the empty barriers' first phase counts as passed
        for (int kb = kb0; kb < kb1; ++kb) {
            if (!tc::mbar_wait(empty + s, ph, p.wait_limit)) { bad = true; break; }
            tc::mbar_expect_tx(full + s, stage);
            uint8_t* w = sm + s * stage;
            tc::tma_load_2d(w, &tmw, full + s, kb * BK, f0);   // (beyond F: value rows, whose outputs are not written)
            tc::tma_load_2d(w + W_TILE / 2, &tmw, full + s, kb * BK, p.F + f0);
            tc::tma_load_2d(w + W_TILE, &tmx, full + s, kb * BK, 0);
            if (++s == p.stages) { s = 0; ph ^= 1; }
        }
    } else if (tid == 160) {
        const uint32_t idesc = tc::make_idesc(128, p.N, BF16 ? 1 : 0, 0, 0);
        int s = 0;
        uint32_t ph = 0;
        for (int kb = kb0; kb < kb1; ++kb) {
            if (!tc::mbar_wait(full + s, ph, p.wait_limit)) { bad = true; break; }
            tc::tc_fence_after();
            const uint32_t w = tc::smem_u32(sm + s * stage), x = w + W_TILE;
#pragma unroll
            for (int kk = 0; kk < BK / 16; ++kk)
                tc::mma_f16(tmem, tc::make_desc(w + kk * 32, 16, 1024), tc::make_desc(x + kk * 32, 16, 1024), idesc,
                            kb != kb0 || kk != 0);
            tc::mma_commit(empty + s);
            if (++s == p.stages) { s = 0; ph ^= 1; }
        }
        if (!bad) tc::mma_commit(&done);
    }
    __syncwarp();
    if (!tc::mbar_wait(&done, 0, p.wait_limit)) bad = true;
    if (!__any_sync(DG_FULL_MASK, bad)) {
        tc::tc_fence_after();
        const uint32_t row = tmem + ((uint32_t)(32 * (warp & 3)) << 16);
        float* out = part + (tid & 127);
#pragma unroll 1
        for (int n = 16 * (warp >> 2); n < p.N; n += 32) {
            uint32_t r[16];
            tc::tmem_ld16(row + n, r);
            tc::tmem_wait_ld();
#pragma unroll
            for (int i = 0; i < 16; ++i) out[(n + i) * 128] = __uint_as_float(r[i]);
        }
        tc::tc_fence_before();
    }
    if (bad) {
        dg::flag_status(p.status, DG_DEVCHK_TIMEOUT);
        aborted = 1;
    }
    __syncwarp();
    __syncthreads();
    if (aborted) {               // loads and products in flight land within microseconds
        const uint64_t t0 = tc::globaltimer_ns();
        for (int i = 0; i < (1 << 20) && tc::globaltimer_ns() - t0 < 2000000; ++i) __nanosleep(1000);
    }
    __syncwarp();
    if (p.splits > 1) cluster_sync();
    // this CTA's share of the tokens, four features to a thread
    const int t0 = (int)((int64_t)p.M * rank / p.splits), t1 = (int)((int64_t)p.M * (rank + 1) / p.splits);
    const T* bias = static_cast<const T*>(p.bias);
    for (int i = tid; i < (t1 - t0) * (FEATURES / 4); i += THREADS) {
        const int m = t0 + i / (FEATURES / 4), f = i % (FEATURES / 4) * 4;
        if (f0 + f >= p.F) continue;       // (F is a multiple of 8)
        const float* src = part + m * 128 + f;
        float4 g = make_float4(0.f, 0.f, 0.f, 0.f), u = g;
        if (p.splits == 1) {
            g = *reinterpret_cast<const float4*>(src);
            u = *reinterpret_cast<const float4*>(src + FEATURES);
        } else {
#pragma unroll 4
            for (int s = 0; s < p.splits; ++s) {
                add(g, remote_load(src, s));
                add(u, remote_load(src + FEATURES, s));
            }
        }
        if (bias) {
            const T *bg = bias + f0 + f, *bu = bg + p.F;
            add(g, make_float4(dg::to_f(bg[0]), dg::to_f(bg[1]), dg::to_f(bg[2]), dg::to_f(bg[3])));
            add(u, make_float4(dg::to_f(bu[0]), dg::to_f(bu[1]), dg::to_f(bu[2]), dg::to_f(bu[3])));
        }
        uint2 o;
        o.x = dgc::Io<T>::pack2(dg::act_fn<ACT>(g.x) * u.x, dg::act_fn<ACT>(g.y) * u.y);
        o.y = dgc::Io<T>::pack2(dg::act_fn<ACT>(g.z) * u.z, dg::act_fn<ACT>(g.w) * u.w);
        *reinterpret_cast<uint2*>(static_cast<T*>(p.h) + (int64_t)m * p.F + f0 + f) = o;
    }
    if (p.splits > 1) {
        __syncwarp();
        cluster_sync();                    // the others have read this CTA's part
    }
    if (warp == 0) {
        tc::tc_fence_after();
        tc::tmem_dealloc(tmem, p.columns);
    }
}

// 16-bit [rows][cols] matrix, box of 64 columns x box_rows, 128B swizzle
bool map_matrix(CUtensorMap* m, const void* base, int64_t rows, int64_t cols, int64_t ld, int box_rows, bool bf16) {
    dgc::EncodeTiledFn fn = dgc::encode_fn();
    if (!fn) return false;
    cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)ld * 2};
    cuuint32_t box[2] = {64, (cuuint32_t)box_rows}, steps[2] = {1, 1};
    return fn(m, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, const_cast<void*>(base),
              dims, strides, box, steps, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
              CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

}  // namespace

namespace dg_host {

// Whether this form is taken rather than the tile kernel: up to 128 tokens (64 x 2048 x 5504: 12.8 us against
// 16.9; 128 x 768 x 768: 7.0 against 7.9), up to 256 where the tile kernel has few tiles with a long axis (200
// x 4096 x 1000: 13 us against 22; but 256 x 4096 x 11008: 65 against 51).
bool ffn_split_supports(int64_t M, int D, int F) { return M <= 128 || (M <= 256 && D >= 1536 && F <= 4096); }

int ffn_split_forward(int dtype, int64_t M, int D, int F, int act, const void* x, int64_t ldx, const void* w,
                      const void* bias, void* h, int32_t* status, cudaStream_t s) {
    const bool bf16 = dtype == DG_DTYPE_BF16;
    SplitParams p{};
    p.M = (int)M, p.N = (int)(M + 15) / 16 * 16, p.F = F;
    p.blocks = (D + BK - 1) / BK;
    const int tiles = (F + FEATURES - 1) / FEATURES, per_sm = p.N <= 128 ? 2 : 1;
    int splits = 1;
    // As many parts as are resident at once, each of 3 stages or, where parts would share SMs, 6: what a part
    // saves in loads it costs in the exchange (13 x 4096 x 1000 in 8 parts 7.9 us, 1 20; 13 x 512 x 8192 in 1
    // 6.4 us, 2 7.2; 128 x 1024 x 1024 in 4 7.3 us, 8 10).
    while (splits < 8 && tiles <= kClusters[per_sm - 1][splits] &&
           p.blocks / (splits + 1) >= (tiles * (splits + 1) > 148 ? 6 : 3))
        ++splits;
    p.per_split = (p.blocks + splits - 1) / splits;
    p.splits = (p.blocks + p.per_split - 1) / p.per_split;             // none empty
    const uint32_t stage = W_TILE + (uint32_t)p.N * BK * 2, room = per_sm == 2 ? MOST_ROOM / 2 : MOST_ROOM;
    p.stages = (int)(room / stage);
    if (p.stages > MAX_STAGES) p.stages = MAX_STAGES;
    uint32_t smem = (uint32_t)p.stages * stage;
    p.columns = 32;
    while (p.columns < (uint32_t)p.N) p.columns *= 2;
    p.bias = bias, p.h = h, p.status = status, p.wait_limit = wait_limit();
    CUtensorMap mw, mx;
    if (!map_matrix(&mw, w, 2 * (int64_t)F, D, D, FEATURES, bf16) || !map_matrix(&mx, x, M, D, ldx, p.N, bf16))
        return DG_ERR_UNSUPPORTED;
    auto kern = bf16 ? (act == DG_ACT_SILU ? ffn_split_kernel<__nv_bfloat16, DG_ACT_SILU> : ffn_split_kernel<__nv_bfloat16, DG_ACT_GELU>)
                     : (act == DG_ACT_SILU ? ffn_split_kernel<__half, DG_ACT_SILU> : ffn_split_kernel<__half, DG_ACT_GELU>);
    return launch_lm(kern, dim3((unsigned)(tiles * p.splits)), dim3(THREADS), smem + 1024, MOST_ROOM + 1024,
                     p.splits > 1 ? p.splits : 0, s, mw, mx, p);
}

}  // namespace dg_host
