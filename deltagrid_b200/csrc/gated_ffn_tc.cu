// gated_ffn_tc.cu -- the products of the gated feed-forward block on tcgen05 (f16 / bf16),
// one persistent kernel in three roles:
//   GATE    G = x Wg^T, U = x Wu^T of one tile side by side in TMEM; epilogue
//           h = act(G + bg) * (U + bu)
//   DGATE   the same products again; epilogue dG = dh U act'(G), dU = dh act(G) and, where
//           the bias gradient is wanted, their sums over 32 rows in fp32
//   PLAIN   C = A B for dx = [dG dU] W and dW = [dG dU]^T x (operands of either major),
//           optionally split along the contracted axis into fp32 partial products
//
// A pair of CTAs (cta_group::2) shares one tile of 256 rows x 256 columns: each CTA holds
// its 128 rows of A and half of B's columns (GATE: the even CTA the 128 gate rows of the
// weights, the odd one the 128 value rows), so each operand byte that enters shared memory
// feeds twice the products it would in a tile of one CTA.  One thread of the even CTA issues
// the MMAs of the pair (M = 256, N = 256, K = 16) into one of two accumulators of 256 TMEM
// columns, so that the epilogue of a tile runs under the products of the next.
//
// Roles per CTA (384 threads): warp 0 loads operand stages by TMA, warp 1 issues the MMAs
// (even CTA only), warp 2 loads DGATE's dh tiles, warps 4-7 and 8-11 are two epilogue groups
// (thread = TMEM lane = row) that take alternate slices of 64 columns.
//
// GATE and DGATE take 128 features a tile, or 64 where there are few tiles: then a tile's
// accumulator has 128 columns, four of them fit, and the epilogue groups take alternate tiles.
//
// What bounds it: the tensor cores.  8192 x 2048 x 5504 in bf16: GATE 227 us (1.63 PFLOP/s, tensor
// pipe 95%), DGATE 255 us (81%: its epilogue reads and writes twice as much), dx 248 us and dW
// 237 us (96% and 95%).  16384 x 768 x 768: 37 us (1.05 PFLOP/s): 384 tiles are 5.2 waves on 74
// pairs and take 6.
//
// Every wait is bounded by the library's wait limit; a role that gives up flags
// DG_DEVCHK_TIMEOUT, the others run into their own limits, and the CTA lets what it has in
// flight land before it frees its TMEM.
#include <cuda.h>

#include "chunk_common.cuh"
#include "lm_common.cuh"

namespace {

enum Role { GATE = 0, DGATE = 1, PLAIN = 2 };

constexpr int BM = 128;                    // rows per CTA (256 per pair)
constexpr int BN = 256;                    // accumulator columns of a tile
constexpr int BK = 64;                     // contracted elements per stage: 128 bytes
constexpr int THREADS = 384;
constexpr uint32_t TILE = BM * BK * 2;     // 16 KB: one operand tile, one staging buffer
constexpr int GROUP_M = 8;                 // tile rows walked together, for L2

// FT: features of a tile (GATE, DGATE; PLAIN tiles have the shape of 128)
template <int ROLE, int FT> struct Cfg {
    static constexpr int STAGES = FT == 64 ? (ROLE == DGATE ? 6 : 8) : (ROLE == DGATE ? 5 : 6);
    static constexpr uint32_t BTILE = FT * BK * 2;                 // this CTA's half of B
    static constexpr uint32_t STAGE = TILE + BTILE;
    static constexpr int ACC = FT == 64 ? 4 : 2, ACCW = 2 * FT;    // accumulators and their columns
    static constexpr uint32_t DH = STAGES * STAGE;                 // DGATE: dh, then dG (one slice per group)
    static constexpr uint32_t OUT = DH + (ROLE == DGATE ? 2 * TILE : 0);
    static constexpr uint32_t BAR = OUT + 2 * TILE;
    static constexpr uint32_t BIAS = BAR + 256;                    // fp32: per group 64 gate and 64 value biases
    static constexpr uint32_t BYTES = BIAS + 1024;
};

struct FfnParams {
    int64_t M;                 // output rows
    int N;                     // output columns (GATE, DGATE: features F)
    int K;                     // contracted elements
    int m_tiles, n_tiles, splits, kb_per_split;
    const void* bias;          // GATE, DGATE: [2F] or null
    float* colsum;             // DGATE: [4 x row tiles of 128][2F] or null
    int32_t* status;
    uint32_t wait_limit;
};

// ---- cluster and cta_group::2 forms -------------------------------------------
__device__ __forceinline__ uint32_t cta_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// address of the same shared-memory location in the even CTA of the pair
__device__ __forceinline__ uint32_t in_leader(const void* p) {
    uint32_t a;
    asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(a) : "r"(tc::smem_u32(p)));
    return a;
}
__device__ __forceinline__ void arrive_at(uint32_t cluster_addr) {
    asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}
__device__ __forceinline__ void tma_load_pair(void* dst, const CUtensorMap* map, uint32_t bar, int c0, int c1) {
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, "
        "%3}], [%4];" ::"r"(tc::smem_u32(dst)),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(bar)
        : "memory");
}
__device__ __forceinline__ void mma_pair(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
        " tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
}
// arrive on this barrier in both CTAs once the MMAs issued so far have completed
__device__ __forceinline__ void commit_pair(uint64_t* bar) {
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
            tc::smem_u32(bar)),
        "h"((uint16_t)3)
        : "memory");
}
__device__ __forceinline__ void tmem_alloc_pair(uint32_t* dst, uint32_t n) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(tc::smem_u32(dst)), "r"(n)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_dealloc_pair(uint32_t t, uint32_t n) {
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(t), "r"(n) : "memory");
}

// work item -> tile row, tile column and split; GROUP_M tile rows at a time, so that the tiles
// in flight share both operands in L2
struct Work {
    int mt, nt, split;
};
__device__ __forceinline__ Work work_of(const FfnParams& p, int64_t i) {
    const int tiles = p.m_tiles * p.n_tiles;
    const int s = (int)(i / tiles), t = (int)(i - (int64_t)s * tiles);
    const int per = GROUP_M * p.n_tiles, g = t / per, r = t - g * per;
    const int rows = min(GROUP_M, p.m_tiles - g * GROUP_M);
    return {g * GROUP_M + r % rows, r / rows, s};
}

// nothing that uses these registers moves above this point (the wait for the loads that fill them)
__device__ __forceinline__ void loaded(uint32_t (&r)[16]) {
    asm volatile("" : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                 "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]));
}

// sums of v[c] over the warp's 32 lanes for c = 0..15: lane l gets column l / 2's
__device__ __forceinline__ float column_sums(float (&v)[16], int lane) {
#pragma unroll
    for (int o = 16; o > 1; o >>= 1) {
        const bool up = lane & o;
#pragma unroll
        for (int i = 0; i < o / 2; ++i) {
            const float send = up ? v[i] : v[i + o / 2], keep = up ? v[i + o / 2] : v[i];
            v[i] = keep + __shfl_xor_sync(DG_FULL_MASK, send, o);
        }
    }
    return v[0] + __shfl_xor_sync(DG_FULL_MASK, v[0], 1);
}

template <typename T, int ROLE, int ACT, bool A_MN, bool B_MN, bool F32_OUT, int FT>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(THREADS, 1)
    ffn_tc_kernel(const __grid_constant__ CUtensorMap tma, const __grid_constant__ CUtensorMap tmb,
                  const __grid_constant__ CUtensorMap tmd, const __grid_constant__ CUtensorMap tmo, FfnParams p) {
    using C = Cfg<ROLE, FT>;
    constexpr bool BF16 = !std::is_same<T, __half>::value;
    constexpr int ST = C::STAGES;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* sm = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint64_t* full = reinterpret_cast<uint64_t*>(sm + C::BAR);      // [ST], counted in the even CTA
    uint64_t* empty = full + ST;                                    // [ST]
    uint64_t* acc_full = empty + ST;                                // [ACC]
    uint64_t* acc_empty = acc_full + C::ACC;                        // [ACC], counted in the even CTA
    uint64_t* dh_full = acc_empty + C::ACC;                         // [2] one per epilogue group
    uint64_t* dh_empty = dh_full + 2;                               // [2]
    uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(dh_empty + 2);
    int* aborted = reinterpret_cast<int*>(tmem_holder + 1);
    const int tid = threadIdx.x, warp = tid >> 5;
    const uint32_t rank = cta_rank();
    const int64_t items = (int64_t)p.m_tiles * p.n_tiles * p.splits;
    const int64_t first = blockIdx.x >> 1, stride = gridDim.x >> 1;
    const int nkb_all = (p.K + BK - 1) / BK;

    if (warp == 0) tmem_alloc_pair(tmem_holder, 512);
    if (tid == 0) {
        for (int i = 0; i < ST; ++i) {
            tc::mbar_init(full + i, 1);
            tc::mbar_init(empty + i, 1);
        }
        for (int i = 0; i < C::ACC; ++i) {
            tc::mbar_init(acc_full + i, 1);
            tc::mbar_init(acc_empty + i, FT == 64 ? 2 : 4);        // epilogue groups of both CTAs that read it
        }
        for (int i = 0; i < 2; ++i) {
            tc::mbar_init(dh_full + i, 1);
            tc::mbar_init(dh_empty + i, 1);
        }
        *aborted = 0;
        tc::fence_barrier_init();
    }
    if (tid == 0) {
        tc::prefetch_tmap(&tma);
        tc::prefetch_tmap(&tmb);
        tc::prefetch_tmap(&tmo);
    }
    tc::tc_fence_before();
    __syncthreads();
    cluster_sync();
    tc::tc_fence_after();
    dg::let_next_start();
    dg::wait_for_previous();
    const uint32_t tmem = *tmem_holder;
    bool bad = false;

    if (warp == 0 && (tid & 31) == 0) {
        // ============================ operand loads ============================
        int s = 0;
        uint32_t ph = 1;                       // the empty barriers' first phase counts as passed
        for (int64_t it = first; it < items && !bad; it += stride) {
            const Work w = work_of(p, it);
            const int row = w.mt * 2 * BM + (int)rank * BM;
            // B's half of this CTA: GATE / DGATE the gate or the value rows, PLAIN columns
            const int col = ROLE == PLAIN ? w.nt * BN + (int)rank * BM : (int)rank * p.N + w.nt * FT;
            const int kb0 = w.split * p.kb_per_split, kb1 = min(kb0 + p.kb_per_split, nkb_all);
            for (int kb = kb0; kb < kb1; ++kb) {
                if (!tc::mbar_wait(empty + s, ph, p.wait_limit)) { bad = true; break; }
                if (rank == 0) tc::mbar_expect_tx(full + s, 2 * C::STAGE);
                const uint32_t bar = in_leader(full + s);
                uint8_t* a = sm + s * C::STAGE;
                uint8_t* b = a + TILE;
                const int k = kb * BK;
                if (A_MN) {
                    tma_load_pair(a, &tma, bar, row, k);
                    tma_load_pair(a + TILE / 2, &tma, bar, row + 64, k);
                } else {
                    tma_load_pair(a, &tma, bar, k, row);
                }
                if (B_MN) {
                    tma_load_pair(b, &tmb, bar, col, k);
                    tma_load_pair(b + TILE / 2, &tmb, bar, col + 64, k);
                } else {
                    tma_load_pair(b, &tmb, bar, k, col);
                }
                if (++s == ST) { s = 0; ph ^= 1; }
            }
        }
    } else if (warp == 1 && rank == 0 && (tid & 31) == 0) {
        // ================================= MMAs =================================
        constexpr uint32_t idesc = tc::make_idesc(2 * BM, C::ACCW, BF16 ? 1 : 0, A_MN ? 1 : 0, B_MN ? 1 : 0);
        int s = 0;
        uint32_t ph = 0, n = 0;
        for (int64_t it = first; it < items && !bad; it += stride, ++n) {
            const uint32_t acc = n % C::ACC;
            const Work w = work_of(p, it);
            const int kb0 = w.split * p.kb_per_split, kb1 = min(kb0 + p.kb_per_split, nkb_all);
            if (!tc::mbar_wait(acc_empty + acc, (n / C::ACC & 1) ^ 1, p.wait_limit)) { bad = true; break; }
            tc::tc_fence_after();
            const uint32_t d = tmem + acc * C::ACCW;
            for (int kb = kb0; kb < kb1; ++kb) {
                if (!tc::mbar_wait(full + s, ph, p.wait_limit)) { bad = true; break; }
                tc::tc_fence_after();
                const uint32_t a = tc::smem_u32(sm + s * C::STAGE), b = a + TILE;
#pragma unroll
                for (int kk = 0; kk < BK / 16; ++kk) {
                    // K-major: 16 elements are 32 bytes of each 128-byte row, 8 rows 1024 bytes apart.
                    // MN-major: 16 k-rows of 128 bytes; the two blocks of 64 are TILE / 2 apart.
                    const uint64_t ad = A_MN ? tc::make_desc(a + kk * 2048, TILE / 2, 1024)
                                             : tc::make_desc(a + kk * 32, 16, 1024);
                    const uint64_t bd = B_MN ? tc::make_desc(b + kk * 2048, TILE / 2, 1024)
                                             : tc::make_desc(b + kk * 32, 16, 1024);
                    mma_pair(d, ad, bd, idesc, kb != kb0 || kk != 0);
                }
                commit_pair(empty + s);
                if (++s == ST) { s = 0; ph ^= 1; }
            }
            if (bad) break;
            commit_pair(acc_full + acc);
        }
    } else if (ROLE == DGATE && warp == 2 && (tid & 31) == 0) {
        // ============================ dh tiles ============================
        uint32_t n = 0;
        for (int64_t it = first; it < items && !bad; it += stride, ++n) {
            const Work w = work_of(p, it);
            for (int g = 0; g < 2; ++g) {
                if (FT == 64 && (int)(n & 1) != g) continue;
                const uint32_t use = FT == 64 ? n >> 1 : n;
                if (!tc::mbar_wait(dh_empty + g, (use & 1) ^ 1, p.wait_limit)) { bad = true; break; }
                tc::mbar_expect_tx(dh_full + g, TILE);
                tc::tma_load_2d(sm + C::DH + g * TILE, &tmd, dh_full + g, w.nt * FT + (FT == 64 ? 0 : 64 * g),
                                w.mt * 2 * BM + (int)rank * BM);
            }
        }
    } else if (warp >= 4) {
        // =============================== epilogue ===============================
        const int g = (warp - 4) >> 2, t = tid - 128 - 128 * g, lane = tid & 31;
        const uint32_t bar_id = 1 + g;
        const uint32_t trow = tmem + ((uint32_t)(32 * (warp & 3)) << 16);
        uint8_t* out = sm + C::OUT + g * TILE;
        uint8_t* dh = sm + C::DH + g * TILE;
        float* bias = reinterpret_cast<float*>(sm + C::BIAS) + 128 * g;
        uint32_t n = 0, acc = 0;
        // the buffer's last TMA store has read it
        auto buffer_free = [&]() {
            if (t == 0) tc::bulk_wait_read0();
            tc::group_sync(bar_id);
        };
        auto release_acc = [&]() {
            tc::tc_fence_before();
            tc::group_sync(bar_id);
            if (t == 0) arrive_at(in_leader(acc_empty + acc));
        };
        for (int64_t it = first; it < items; it += stride, ++n) {
            if (FT == 64 && (int)(n & 1) != g) continue;
            const Work w = work_of(p, it);
            acc = n % C::ACC;
            const int row0 = w.mt * 2 * BM + (int)rank * BM;
            const int c0 = FT == 64 ? 0 : 64 * g;              // this group's columns of the gate
            const int f0 = w.nt * FT + c0;                 // GATE, DGATE: this group's 64 features
            if (ROLE != PLAIN) {                               // (read last before the store's barrier)
                const int f = f0 + (t & 63);
                bias[t] = p.bias && f < p.N
                              ? dg::to_f(static_cast<const T*>(p.bias)[(int64_t)(t >> 6) * p.N + f]) : 0.f;
            }
            bad = !tc::mbar_wait(acc_full + acc, n / C::ACC & 1, p.wait_limit);
            if (ROLE == DGATE && !bad) bad = !tc::mbar_wait(dh_full + g, (FT == 64 ? n >> 1 : n) & 1, p.wait_limit);
            if (tc::group_sync_or(bar_id, bad)) { bad = true; break; }
            tc::tc_fence_after();
            const uint32_t d = trow + acc * C::ACCW;
            if (ROLE != PLAIN) {
                // 16 columns of gate and value at a time, the next ones on their way from TMEM
                uint32_t gr[2][16], ur[2][16];
                tc::tmem_ld16(d + c0, gr[0]);
                tc::tmem_ld16(d + FT + c0, ur[0]);
                float sum_g[4], sum_u[4];
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    tc::tmem_wait_ld();
                    loaded(gr[q & 1]);
                    loaded(ur[q & 1]);
                    if (q < 3) {
                        tc::tmem_ld16(d + c0 + 16 * (q + 1), gr[(q + 1) & 1]);
                        tc::tmem_ld16(d + FT + c0 + 16 * (q + 1), ur[(q + 1) & 1]);
                    } else {
                        release_acc();
                    }
                    if (q == 0) buffer_free();
                    float zg[16], zu[16];
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        const uint32_t at = tc::sw128((uint32_t)t, (uint32_t)(2 * q + c));
                        uint32_t o[4], o2[4], dv[4];
                        if (ROLE == DGATE) *reinterpret_cast<uint4*>(dv) = *reinterpret_cast<const uint4*>(dh + at);
#pragma unroll
                        for (int e = 0; e < 8; e += 2) {
                            const int i = 8 * c + e;
                            const dg::F2 bg = *reinterpret_cast<const dg::F2*>(bias + 16 * q + i);
                            const dg::F2 bu = *reinterpret_cast<const dg::F2*>(bias + 64 + 16 * q + i);
                            const dg::F2 gv = dg::add2({__uint_as_float(gr[q & 1][i]), __uint_as_float(gr[q & 1][i + 1])}, bg);
                            const dg::F2 uv = dg::add2({__uint_as_float(ur[q & 1][i]), __uint_as_float(ur[q & 1][i + 1])}, bu);
                            if (ROLE == GATE) {
                                const dg::F2 h = dg::mul2(dg::act_fn2<ACT>(gv), uv);
                                o[e / 2] = dgc::Io<T>::pack2(h.x, h.y);
                            } else {
                                const float2 dhv = dgc::Io<T>::unpack2(dv[e / 2]);
                                const dg::F2 dd{dhv.x, dhv.y};
                                dg::F2 a, s;
                                dg::act_grad2<ACT>(gv, a, s);
                                // dG and dU go to 16 bits: the tensor cores read no other type for dx and dW,
                                // and a second half of each would double those products.  dbias is summed before
                                const dg::F2 xg = dg::mul2(dg::mul2(dd, uv), s), xu = dg::mul2(dd, a);
                                zg[i] = xg.x, zg[i + 1] = xg.y;
                                zu[i] = xu.x, zu[i + 1] = xu.y;
                                o[e / 2] = dgc::Io<T>::pack2(xg.x, xg.y);
                                o2[e / 2] = dgc::Io<T>::pack2(xu.x, xu.y);
                            }
                        }
                        if (ROLE == GATE) {
                            *reinterpret_cast<uint4*>(out + at) = *reinterpret_cast<const uint4*>(o);
                        } else {      // dG takes dh's place
                            *reinterpret_cast<uint4*>(dh + at) = *reinterpret_cast<const uint4*>(o);
                            *reinterpret_cast<uint4*>(out + at) = *reinterpret_cast<const uint4*>(o2);
                        }
                    }
                    if (ROLE == DGATE && p.colsum) {
                        sum_g[q] = column_sums(zg, lane);
                        sum_u[q] = column_sums(zu, lane);
                    }
                }
                if (ROLE == DGATE && p.colsum) {
                    float* dst = p.colsum + ((int64_t)(w.mt * 2 + (int)rank) * 4 + (warp & 3)) * 2 * p.N;
                    // even lanes write the gate's sums, odd ones the value's
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        const int f = f0 + 16 * q + (lane >> 1);
                        if (f < p.N) dst[(lane & 1 ? p.N : 0) + f] = lane & 1 ? sum_u[q] : sum_g[q];
                    }
                }
                tc::fence_proxy_async();
                tc::group_sync(bar_id);
                if (t == 0) {
                    if (f0 < p.N && row0 < p.M) {
                        if (ROLE == GATE) {
                            tc::tma_store_2d(&tmo, out, f0, row0);
                        } else {
                            tc::tma_store_3d(&tmo, dh, f0, 0, row0);
                            tc::tma_store_3d(&tmo, out, f0, 1, row0);
                        }
                    }
                    tc::bulk_commit_group();
                    if (ROLE == DGATE) {               // dG has been read: the next dh may land there
                        tc::bulk_wait_read0();
                        tc::mbar_arrive(dh_empty + g);
                    }
                }
            } else {
                constexpr int W = F32_OUT ? 32 : 64;   // columns of a slice of 128 bytes
#pragma unroll 1
                for (int j = g; j < BN / W; j += 2) {
                    const int col = w.nt * BN + W * j;
                    uint32_t ra[32], rb[32];
                    tc::tmem_ld32(d + W * j, ra);
                    if (!F32_OUT) tc::tmem_ld32(d + W * j + 32, rb);
                    tc::tmem_wait_ld();
                    if (j + 2 >= BN / W) release_acc();
                    buffer_free();
#pragma unroll
                    for (int c = 0; c < 8; ++c) {
                        uint32_t o[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            if (F32_OUT) {
                                o[e] = ra[4 * c + e];
                            } else {
                                const int i = (8 * c + 2 * e) & 31;
                                o[e] = c < 4 ? dgc::Io<T>::pack2(__uint_as_float(ra[i]), __uint_as_float(ra[i + 1]))
                                             : dgc::Io<T>::pack2(__uint_as_float(rb[i]), __uint_as_float(rb[i + 1]));
                            }
                        }
                        *reinterpret_cast<uint4*>(out + tc::sw128((uint32_t)t, (uint32_t)c)) =
                            *reinterpret_cast<const uint4*>(o);
                    }
                    tc::fence_proxy_async();
                    tc::group_sync(bar_id);
                    if (t == 0) {
                        if (col < p.N && row0 < p.M) tc::tma_store_3d(&tmo, out, col, row0, w.split);
                        tc::bulk_commit_group();
                    }
                }
            }
        }
        if (t == 0) tc::bulk_wait0();
    }
    if (bad) {
        dg::flag_status(p.status, DG_DEVCHK_TIMEOUT);
        *aborted = 1;
    }
    __syncwarp();
    tc::tc_fence_before();
    __syncthreads();
    if (*aborted) {              // loads and products in flight land within microseconds
        const uint64_t t0 = tc::globaltimer_ns();
        for (int i = 0; i < (1 << 20) && tc::globaltimer_ns() - t0 < 2000000; ++i) __nanosleep(1000);
    }
    __syncwarp();
    cluster_sync();
    if (warp == 0) {
        tc::tc_fence_after();
        tmem_dealloc_pair(tmem, 512);
    }
}

// What a backward pass still has to add up, in one launch after its products: the fp32 partial products of a
// split dx or dW, in order of the splits (8 values a thread), and dbias from its sums over 32
// rows, in a fixed order (32 columns a block, warp w takes rows w, w + 32, ...).
struct Join {
    const float4* part;
    uint4* out;
    int64_t n8;                            // outputs / 8
    int splits, blocks;
};
constexpr int kFinish = 1024;
template <typename T>
__global__ void __launch_bounds__(kFinish) finish_kernel(Join dx, Join dw, const float* sums, int rows, int cols, T* dbias) {
    __shared__ float s[32][33];
    dg::let_next_start();
    dg::wait_for_previous();
    int block = (int)blockIdx.x - (dbias ? (cols + 31) / 32 : 0);      // dbias first: its chains are the longest
    if (block >= 0) {
        const Join& q = block < dx.blocks ? dx : dw;
        if (block >= dx.blocks) block -= dx.blocks;
        const int64_t i = (int64_t)block * kFinish + threadIdx.x;
        if (i >= q.n8) return;
        float4 a = q.part[2 * i], b = q.part[2 * i + 1];
#pragma unroll 4
        for (int k = 1; k < q.splits; ++k) {
            const float4 c = q.part[2 * (q.n8 * k + i)], d = q.part[2 * (q.n8 * k + i) + 1];
            a.x += c.x; a.y += c.y; a.z += c.z; a.w += c.w;
            b.x += d.x; b.y += d.y; b.z += d.z; b.w += d.w;
        }
        uint4 v;
        v.x = dgc::Io<T>::pack2(a.x, a.y);
        v.y = dgc::Io<T>::pack2(a.z, a.w);
        v.z = dgc::Io<T>::pack2(b.x, b.y);
        v.w = dgc::Io<T>::pack2(b.z, b.w);
        q.out[i] = v;
        return;
    }
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, c = blockIdx.x * 32 + lane;
    float a = 0.f;
    if (c < cols)
        for (int r = warp; r < rows; r += 32) a += sums[(int64_t)r * cols + c];
    s[warp][lane] = a;
    __syncthreads();
    a = s[lane][warp];                     // column `warp` of the block, partial sum `lane`
#pragma unroll
    for (int o = 16; o; o >>= 1) a += __shfl_xor_sync(DG_FULL_MASK, a, o);
    if (lane == 0 && blockIdx.x * 32 + warp < cols) dbias[blockIdx.x * 32 + warp] = dg::from_f<T>(a);
}

CUtensorMapDataType map_type(bool bf16) {
    return bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
}

// rank-2 or rank-3 map with 128-byte rows in the box, 128B swizzle; strides in bytes
bool make_tmap(CUtensorMap* m, CUtensorMapDataType type, const void* base, int rank, const cuuint64_t* dims,
               const cuuint64_t* strides, const cuuint32_t* box) {
    dgc::EncodeTiledFn fn = dgc::encode_fn();
    if (!fn) return false;
    cuuint32_t estr[3] = {1, 1, 1};
    return fn(m, type, rank, const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
              CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// 16-bit [rows][cols] matrix, box of 64 columns x box_rows
bool map_matrix(CUtensorMap* m, const void* base, int64_t rows, int64_t cols, int64_t ld, int box_rows, bool bf16) {
    cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)ld * 2};
    cuuint32_t box[2] = {64, (cuuint32_t)box_rows};
    return make_tmap(m, map_type(bf16), base, 2, dims, strides, box);
}

}  // namespace

namespace dg_host {

uint32_t wait_limit();
int sm_count(int device, int* out);

namespace {

int pairs(int* out) {
    int dev = 0, nsm = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return record_cuda_error(e);
    const int rc = sm_count(dev, &nsm);
    *out = nsm / 2;
    return rc;
}

template <typename K>
int launch(K kern, uint32_t smem, int64_t items, const CUtensorMap& a, const CUtensorMap& b, const CUtensorMap& d,
           const CUtensorMap& o, const FfnParams& p, cudaStream_t s) {
    int np = 0;
    const int rc = pairs(&np);
    if (rc != DG_OK) return rc;
    // (the cluster size stands at the kernel)
    return launch_lm(kern, dim3((unsigned)(2 * (items < np ? items : np))), dim3(THREADS), smem + 1024, smem + 1024, 0, s, a, b, d,
                     o, p);
}

FfnParams tiles_of(int64_t M, int N, int K, int tile_n, int32_t* status) {
    FfnParams p{};
    p.M = M, p.N = N, p.K = K;
    p.m_tiles = (int)((M + 2 * BM - 1) / (2 * BM));
    p.n_tiles = (N + tile_n - 1) / tile_n;
    p.splits = 1;
    p.kb_per_split = (K + BK - 1) / BK;
    p.status = status;
    p.wait_limit = wait_limit();
    return p;
}

// splits of a PLAIN product whose tiles would not fill the pairs: as many as fit one wave, each
// with at least 8 stages of the contracted axis (below that the pipeline hardly fills)
int splits_of(int64_t M, int N, int64_t K, int np) {
    const int64_t tiles = ((M + 2 * BM - 1) / (2 * BM)) * ((N + BN - 1) / BN);
    const int64_t nkb = (K + BK - 1) / BK;
    int64_t s = np / (tiles > 0 ? tiles : 1);
    if (s > nkb / 8) s = nkb / 8;
    return (int)(s < 1 ? 1 : s);
}

// C [M,N] = A B, contracted length K; A as [M,K] (a_mn: [K,M]), B as [N,K] (b_mn: [K,N]).  Where it is split,
// `join` gets what remains to be added up.
template <typename T, bool A_MN, bool B_MN>
int product(int64_t M, int N, int64_t K, const void* a, int64_t lda, const void* b, int64_t ldb, void* c, float* part,
            int splits, Join* join, int32_t* status, cudaStream_t s) {
    constexpr bool bf16 = !std::is_same<T, __half>::value;
    FfnParams p = tiles_of(M, N, (int)K, BN, status);
    const int nkb = p.kb_per_split;
    p.kb_per_split = (nkb + splits - 1) / splits;
    p.splits = splits = (nkb + p.kb_per_split - 1) / p.kb_per_split;       // none empty
    CUtensorMap ma, mb, mo;
    bool ok = A_MN ? map_matrix(&ma, a, K, M, lda, BK, bf16) : map_matrix(&ma, a, M, K, lda, BM, bf16);
    ok = ok && (B_MN ? map_matrix(&mb, b, K, N, ldb, BK, bf16) : map_matrix(&mb, b, N, K, ldb, BM, bf16));
    const int e = splits > 1 ? 4 : 2;
    cuuint64_t dims[3] = {(cuuint64_t)N, (cuuint64_t)M, (cuuint64_t)splits};
    cuuint64_t strides[2] = {(cuuint64_t)N * e, (cuuint64_t)N * e * (cuuint64_t)M};
    cuuint32_t box[3] = {(cuuint32_t)(128 / e), BM, 1};
    ok = ok && make_tmap(&mo, splits > 1 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : map_type(bf16),
                         splits > 1 ? static_cast<void*>(part) : c, 3, dims, strides, box);
    if (!ok) return DG_ERR_UNSUPPORTED;
    const int64_t items = (int64_t)p.m_tiles * p.n_tiles * p.splits;
    if (splits > 1) {
        const int64_t n8 = M * N / 8;
        *join = {reinterpret_cast<const float4*>(part), static_cast<uint4*>(c), n8, splits, (int)((n8 + kFinish - 1) / kFinish)};
    }
    return splits == 1
               ? launch(ffn_tc_kernel<T, PLAIN, 0, A_MN, B_MN, false, 128>, (Cfg<PLAIN, 128>::BYTES), items, ma, mb, ma, mo, p, s)
               : launch(ffn_tc_kernel<T, PLAIN, 0, A_MN, B_MN, true, 128>, (Cfg<PLAIN, 128>::BYTES), items, ma, mb, ma, mo, p, s);
}

bool aligned(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
size_t round256(size_t n) { return (n + 255) & ~size_t(255); }

struct Spaces {
    size_t dz, colsum, part_dx, part_dw, total;
    int splits_dx, splits_dw;
};
Spaces spaces(int64_t M, int D, int F) {
    int np = 74;
    if (pairs(&np) != DG_OK) np = 74;          // no device here: the size for a whole B200
    Spaces w;
    w.splits_dx = splits_of(M, D, 2 * (int64_t)F, np);
    w.splits_dw = splits_of(2 * (int64_t)F, D, M, np);
    w.dz = round256((size_t)M * 2 * F * 2);
    w.colsum = round256((size_t)((M + 2 * BM - 1) / (2 * BM)) * 8 * 2 * F * 4);
    w.part_dx = round256(w.splits_dx > 1 ? (size_t)w.splits_dx * M * D * 4 : 0);
    w.part_dw = round256(w.splits_dw > 1 ? (size_t)w.splits_dw * 2 * F * D * 4 : 0);
    w.total = w.dz + w.colsum + w.part_dx + w.part_dw;
    return w;
}

}  // namespace

// 16-bit types whose rows TMA can address: D and F multiples of 8, 16-byte aligned tensors
bool ffn_tc_supports(int dtype, int64_t M, int D, int F) {
    return (dtype == DG_DTYPE_F16 || dtype == DG_DTYPE_BF16) && D % 8 == 0 && F % 8 == 0 && M <= (int64_t)1 << 30;
}
bool ffn_tc_aligned(const void* a, int64_t lda, const void* b, const void* c, const void* d, int64_t ldd,
                    const void* e, const void* f) {
    return aligned(a) && aligned(b) && aligned(c) && aligned(d) && aligned(e) && aligned(f) && lda % 8 == 0 &&
           ldd % 8 == 0;
}

// Features per tile.  A tile of 64 takes not half but four fifths of one of 128: its MMAs read A from shared
// memory twice as often (16384 x 768 x 768: 49 us in 11 waves of 64, 37 us in 6 of 128).  So it is taken
// where its tiles need no more waves (129 to 256 x 768 x 768: 8.1 us against 9.8).
static int tile_features(int64_t M, int F, int np) {
    const int64_t rows = (M + 2 * BM - 1) / (2 * BM);
    const int64_t waves128 = (rows * ((F + 127) / 128) + np - 1) / np, waves64 = (rows * ((F + 63) / 64) + np - 1) / np;
    return waves64 * 4 < waves128 * 5 ? 64 : 128;
}

template <typename T, int ROLE, int FT>
static int gate_t(int64_t M, int D, int F, int act, const void* x, int64_t ldx, const void* w, const CUtensorMap& md,
                  const CUtensorMap& mo, FfnParams p, cudaStream_t s) {
    constexpr bool bf16 = !std::is_same<T, __half>::value;
    CUtensorMap mx, mw;
    if (!map_matrix(&mx, x, M, D, ldx, BM, bf16) || !map_matrix(&mw, w, 2 * (int64_t)F, D, D, FT, bf16))
        return DG_ERR_UNSUPPORTED;
    p.n_tiles = (F + FT - 1) / FT;
    const int64_t items = (int64_t)p.m_tiles * p.n_tiles;
    return act == DG_ACT_SILU
               ? launch(ffn_tc_kernel<T, ROLE, DG_ACT_SILU, false, false, false, FT>, Cfg<ROLE, FT>::BYTES, items, mx, mw,
                        md, mo, p, s)
               : launch(ffn_tc_kernel<T, ROLE, DG_ACT_GELU, false, false, false, FT>, Cfg<ROLE, FT>::BYTES, items, mx, mw,
                        md, mo, p, s);
}
template <typename T, int ROLE>
static int gate(int64_t M, int D, int F, int act, const void* x, int64_t ldx, const void* w, const CUtensorMap& md,
                const CUtensorMap& mo, const FfnParams& p, cudaStream_t s) {
    int np = 0;
    const int rc = pairs(&np);
    if (rc != DG_OK) return rc;
    return tile_features(M, F, np) == 64 ? gate_t<T, ROLE, 64>(M, D, F, act, x, ldx, w, md, mo, p, s)
                                         : gate_t<T, ROLE, 128>(M, D, F, act, x, ldx, w, md, mo, p, s);
}

template <typename T>
static int forward_t(int64_t M, int D, int F, int act, const void* x, int64_t ldx, const void* w, const void* bias,
                     void* h, int32_t* status, cudaStream_t s) {
    constexpr bool bf16 = !std::is_same<T, __half>::value;
    FfnParams p = tiles_of(M, F, D, BM, status);
    p.bias = bias;
    CUtensorMap mh;
    if (!map_matrix(&mh, h, M, F, F, BM, bf16)) return DG_ERR_UNSUPPORTED;
    return gate<T, GATE>(M, D, F, act, x, ldx, w, mh, mh, p, s);
}

int ffn_tc_forward(int dtype, int64_t M, int D, int F, int act, const void* x, int64_t ldx, const void* w,
                   const void* bias, void* h, int32_t* status, cudaStream_t s) {
    return dtype == DG_DTYPE_F16 ? forward_t<__half>(M, D, F, act, x, ldx, w, bias, h, status, s)
                                 : forward_t<__nv_bfloat16>(M, D, F, act, x, ldx, w, bias, h, status, s);
}

size_t ffn_tc_workspace(int64_t M, int D, int F) { return spaces(M, D, F).total; }

template <typename T>
static int backward_t(int64_t M, int D, int F, int act, const void* x, int64_t ldx, const void* w, const void* bias,
                      const void* dh, int64_t ld_dh, void* dx, void* dw, void* db, void* workspace, int32_t* status,
                      cudaStream_t s) {
    constexpr bool bf16 = !std::is_same<T, __half>::value;
    const Spaces sp = spaces(M, D, F);
    char* ws = static_cast<char*>(workspace);
    void* dz = ws;
    float* colsum = reinterpret_cast<float*>(ws + sp.dz);
    float* part_dx = reinterpret_cast<float*>(ws + sp.dz + sp.colsum);
    float* part_dw = reinterpret_cast<float*>(ws + sp.dz + sp.colsum + sp.part_dx);
    FfnParams p = tiles_of(M, F, D, BM, status);
    p.bias = bias;
    p.colsum = db ? colsum : nullptr;
    CUtensorMap md, mz;
    cuuint64_t dims[3] = {(cuuint64_t)F, 2, (cuuint64_t)M};
    cuuint64_t strides[2] = {(cuuint64_t)F * 2, (cuuint64_t)F * 4};
    cuuint32_t box[3] = {64, 1, BM};
    if (!map_matrix(&md, dh, M, F, ld_dh, BM, bf16) || !make_tmap(&mz, map_type(bf16), dz, 3, dims, strides, box))
        return DG_ERR_UNSUPPORTED;
    int rc = gate<T, DGATE>(M, D, F, act, x, ldx, w, md, mz, p, s);
    Join join_dx{}, join_dw{};
    if (rc == DG_OK && dx)
        rc = product<T, false, true>(M, D, 2 * (int64_t)F, dz, 2 * (int64_t)F, w, D, dx, part_dx, sp.splits_dx, &join_dx, status, s);
    if (rc == DG_OK && dw)
        rc = product<T, true, true>(2 * (int64_t)F, D, M, dz, 2 * (int64_t)F, x, ldx, dw, part_dw, sp.splits_dw, &join_dw, status, s);
    const int blocks = join_dx.blocks + join_dw.blocks + (db ? (2 * F + 31) / 32 : 0);
    if (rc == DG_OK && blocks > 0)
        rc = launch_lm(finish_kernel<T>, dim3((unsigned)blocks), dim3(kFinish), 0, 0, 0, s, join_dx, join_dw, (const float*)colsum,
                       p.m_tiles * 8, 2 * F, static_cast<T*>(db));
    return rc;
}

int ffn_tc_backward(int dtype, int64_t M, int D, int F, int act, const void* x, int64_t ldx, const void* w,
                    const void* bias, const void* dh, int64_t ld_dh, void* dx, void* dw, void* db, void* workspace,
                    int32_t* status, cudaStream_t s) {
    return dtype == DG_DTYPE_F16
               ? backward_t<__half>(M, D, F, act, x, ldx, w, bias, dh, ld_dh, dx, dw, db, workspace, status, s)
               : backward_t<__nv_bfloat16>(M, D, F, act, x, ldx, w, bias, dh, ld_dh, dx, dw, db, workspace, status, s);
}

}  // namespace dg_host
