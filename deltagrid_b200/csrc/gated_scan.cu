// gated_scan.cu -- the gated linear recurrence h_t = c_t h_{t-1} + (1 - a_t) x_t with
// a = sigmoid(gate): forward, backward and single step.
//
// A run of steps acts on the state as h -> P h + H (P the product of its c, H its end state
// from zero), and such maps compose, so the sequence splits along time:
//   - a thread takes R = 8 consecutive steps of VEC channels; its maps are composed with its
//     neighbours' by shuffles and, through shared memory, with the other warps';
//   - a CTA (256 threads) takes a tile of 256 / LPR x 8 steps by LPR x VEC channels and
//     walks the sequence tile by tile with the state in registers;
//   - where rows and channels give too few CTAs, a cluster of up to 16 takes consecutive
//     tiles and exchanges their maps through distributed shared memory, one cluster barrier
//     per tile.
// Each input is read and each output written once.  The order of every composition is fixed
// by the sizes alone, so results repeat bit for bit.
//
// Inputs come by cp.async into shared memory that only the copying thread reads, one tile
// ahead: no registers are held for data in flight and no barrier waits for it.
//
// The backward pass carries r_t = c_t (d_t + r_{t+1}) (d the gradient that enters at step t)
// the same way in reverse, and forms the states again from the marks that the forward pass
// leaves every DG_SCAN_MARK_STEPS steps: fp32 states, so nothing is lost to the rounding of
// y, for 4 / 64 bytes a step.
#include <type_traits>

#include "lm_common.cuh"

namespace {

constexpr int R = 8;                       // consecutive steps per thread
constexpr int THREADS = 256;
constexpr int WARPS = THREADS / 32;
constexpr int STAGES = 2;                  // tiles of input in shared memory
static_assert(DG_SCAN_MARK_STEPS % R == 0, "a mark falls on a thread's first step");

struct ScanIn {
    const void *x, *g, *o;
    int64_t x_sb, x_st, g_sb, g_st, o_sb, o_st;
    const int32_t* lengths;
    const uint8_t* resets;
    int B, T, D, cluster;
};

struct ScanGrad {
    const float* marks;
    const void* dy;
    int64_t dy_sb, dy_st;
    const float* dh_last;
    void *dx, *dg_, *do_;
    int64_t dx_sb, dx_st, dg_sb, dg_st, do_sb, do_st;
    float* dh0;
};

// ---- cp.async ------------------------------------------------------------------
// copies BYTES (4 or 8), or zeros where !on
template <int BYTES>
__device__ __forceinline__ void copy_async(void* dst, const void* src, bool on) {
    const int n = on ? BYTES : 0;
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(
                     (uint32_t)__cvta_generic_to_shared(dst)),
                 "l"(src), "n"(BYTES), "r"(n)
                 : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void copy_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_barrier() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ void store_remote(float2* p, uint32_t rank, float2 v) {
    uint32_t a;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"((uint32_t)__cvta_generic_to_shared(p)), "r"(rank));
    asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};" ::"r"(a), "f"(v.x), "f"(v.y) : "memory");
}

// VEC storage elements
template <typename T, int VEC> struct alignas(sizeof(T) * VEC) Pack {
    T v[VEC];
};

// maps of a tile, per channel: one per warp, and one per CTA of the cluster
template <int CH> struct Maps {
    float2 warp[2][WARPS][CH];             // (P, H)
    float2 cta[2][16][CH];
};

template <typename T, int VEC, int LPR, int ARRAYS> struct Tile {
    static constexpr int GROUPS = THREADS / LPR, STEPS = GROUPS * R, CH = LPR * VEC;
    typedef Pack<T, VEC> P;
    static constexpr size_t STAGE = (size_t)ARRAYS * R * THREADS * sizeof(P);
};

// one thread's 8 steps of one input into its own column of the stage
template <typename T, int VEC>
__device__ __forceinline__ void fetch(Pack<T, VEC>* st, const T* p, int64_t step, int n, bool on) {
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const bool live = on && r < n;
        if constexpr (sizeof(T) * VEC >= 4) {
            copy_async<sizeof(T) * VEC>(st + r * THREADS, live ? p + r * step : p, live);
        } else {                           // 2 bytes: below what cp.async copies
            T z = dg::from_f<T>(0.f);
            if (live) z = p[r * step];
            st[r * THREADS].v[0] = z;
        }
    }
}

// composes (P, H) maps over the row groups of a warp: in: the thread's own map, out: the map of
// the groups before it; returns the whole warp's map in the last group
template <int LPR>
__device__ __forceinline__ void warp_before(float P, float H, float& Pb, float& Hb, float& Pw, float& Hw, int lane) {
#pragma unroll
    for (int o = LPR; o < 32; o <<= 1) {
        const float p = __shfl_up_sync(DG_FULL_MASK, P, o), h = __shfl_up_sync(DG_FULL_MASK, H, o);
        if (lane >= o) {
            H = fmaf(P, h, H);
            P *= p;
        }
    }
    Pw = P;
    Hw = H;
    Pb = 1.f;
    Hb = 0.f;
    if (LPR < 32) {
        const float p = __shfl_up_sync(DG_FULL_MASK, P, LPR & 31), h = __shfl_up_sync(DG_FULL_MASK, H, LPR & 31);
        if (lane >= LPR) {
            Pb = p;
            Hb = h;
        }
    }
}
// the same from the other end of the warp; the whole warp's map is in the first group
template <int LPR>
__device__ __forceinline__ void warp_after(float P, float Q, float& Pb, float& Qb, float& Pw, float& Qw, int lane) {
#pragma unroll
    for (int o = LPR; o < 32; o <<= 1) {
        const float p = __shfl_down_sync(DG_FULL_MASK, P, o), q = __shfl_down_sync(DG_FULL_MASK, Q, o);
        if (lane + o < 32) {
            Q = fmaf(P, q, Q);
            P *= p;
        }
    }
    Pw = P;
    Qw = Q;
    Pb = 1.f;
    Qb = 0.f;
    if (LPR < 32) {
        const float p = __shfl_down_sync(DG_FULL_MASK, P, LPR & 31), q = __shfl_down_sync(DG_FULL_MASK, Q, LPR & 31);
        if (lane + LPR < 32) {
            Pb = p;
            Qb = q;
        }
    }
}

template <typename T, int VEC, int LPR, bool OG>
__global__ void __launch_bounds__(THREADS, 3)
    scan_forward_kernel(ScanIn in, const float* h0, T* y, float* h_last, float* marks) {
    typedef Tile<T, VEC, LPR, OG ? 3 : 2> Tl;
    typedef Pack<T, VEC> Pk;
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ Maps<Tl::CH> maps;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int S = in.cluster, rank = S > 1 ? (int)cluster_rank() : 0;
    const int blocks = (in.D + Tl::CH - 1) / Tl::CH;
    const int unit = blockIdx.x / S, b = unit / blocks;
    const int lc = tid % LPR, d = (unit % blocks) * Tl::CH + lc * VEC;
    const bool on = d < in.D;
    const int len = in.lengths ? min(max(in.lengths[b], 0), in.T) : in.T;
    const T* x = (const T*)in.x + b * in.x_sb + d;
    const T* g = (const T*)in.g + b * in.g_sb + d;
    const T* o = OG ? (const T*)in.o + b * in.o_sb + d : nullptr;
    const uint8_t* rs = in.resets ? in.resets + (int64_t)b * in.T : nullptr;
    const int nblk = (in.T + DG_SCAN_MARK_STEPS - 1) / DG_SCAN_MARK_STEPS;
    Pk* mine = reinterpret_cast<Pk*>(smem) + tid;
    constexpr int ARR = R * THREADS, STG = (OG ? 3 : 2) * ARR;
    const int span = S * Tl::STEPS, ntiles = (in.T + span - 1) / span;
    const int t_first = rank * Tl::STEPS + (tid / LPR) * R;

    uint8_t next_reset = 0;                // of step lc of this thread's group, for lc < R
    auto prefetch = [&](int it) {
        const int t = it * span + t_first;
        Pk* st = mine + (it & 1) * STG;
        fetch<T, VEC>(st, x + t * in.x_st, in.x_st, len - t, on);
        fetch<T, VEC>(st + ARR, g + t * in.g_st, in.g_st, len - t, on);
        if (OG) fetch<T, VEC>(st + 2 * ARR, o + t * in.o_st, in.o_st, len - t, on);
        copy_commit();
        if (rs) next_reset = (lc < R && t + lc < len) ? rs[t + lc] : 0;
    };

    float state[VEC];
#pragma unroll
    for (int v = 0; v < VEC; ++v) state[v] = (h0 && on) ? h0[(int64_t)b * in.D + d + v] : 0.f;
    if (ntiles > 0) prefetch(0);
    for (int it = 0; it < ntiles; ++it) {
        const int t = it * span + t_first;
        unsigned resets = 0;
        if (rs) resets = __ballot_sync(DG_FULL_MASK, next_reset != 0) >> (lane & ~(LPR - 1));
        if (it + 1 < ntiles) prefetch(it + 1);
        else copy_commit();
        copy_wait<1>();
        const Pk* st = mine + (it & 1) * STG;
        float c[R][VEC], u[R][VEC], P[VEC], H[VEC];
#pragma unroll
        for (int v = 0; v < VEC; ++v) P[v] = 1.f, H[v] = 0.f;
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const Pk xv = st[r * THREADS], gv = st[ARR + r * THREADS];
#pragma unroll
            for (int v = 0; v < VEC; ++v) {
                float a, na;
                dg::sigmoid_pair(dg::to_f(gv.v[v]), a, na);
                c[r][v] = t + r < len ? ((resets >> r) & 1 ? 0.f : a) : 1.f;
                u[r][v] = t + r < len ? na * dg::to_f(xv.v[v]) : 0.f;
                H[v] = fmaf(c[r][v], H[v], u[r][v]);
                P[v] *= c[r][v];
            }
        }
        float Pb[VEC], Hb[VEC];
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
            float Pw, Hw;
            warp_before<LPR>(P[v], H[v], Pb[v], Hb[v], Pw, Hw, lane);
            if (lane >= 32 - LPR) maps.warp[it & 1][warp][lc * VEC + v] = make_float2(Pw, Hw);
        }
        __syncthreads();
        float h[VEC];
        if (S > 1) {
            for (int i = tid; i < S * Tl::CH; i += THREADS) {       // this CTA's map to every CTA
                const int ch = i % Tl::CH;
                float2 m = maps.warp[it & 1][0][ch];
#pragma unroll
                for (int w = 1; w < WARPS; ++w) {
                    const float2 n = maps.warp[it & 1][w][ch];
                    m.y = fmaf(n.x, m.y, n.y);
                    m.x *= n.x;
                }
                store_remote(&maps.cta[it & 1][rank][ch], i / Tl::CH, m);
            }
            __syncwarp();
            cluster_barrier();
        }
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
            const int ch = lc * VEC + v;
            float s = state[v], mine_s = s;
            if (S > 1) {
                for (int k = 0; k < S; ++k) {
                    if (k == rank) mine_s = s;
                    const float2 m = maps.cta[it & 1][k][ch];
                    s = fmaf(m.x, s, m.y);
                }
                state[v] = s;
                s = mine_s;
            }
#pragma unroll
            for (int w = 0; w < WARPS; ++w) {
                if (w == warp) mine_s = s;
                const float2 m = maps.warp[it & 1][w][ch];
                s = fmaf(m.x, s, m.y);
            }
            if (S == 1) state[v] = s;
            h[v] = fmaf(Pb[v], mine_s, Hb[v]);
        }
        if (!on) continue;
        if (marks && t < in.T && t % DG_SCAN_MARK_STEPS == 0)
#pragma unroll
            for (int v = 0; v < VEC; ++v) marks[((int64_t)b * nblk + t / DG_SCAN_MARK_STEPS) * in.D + d + v] = h[v];
        T* yp = y + ((int64_t)b * in.T + t) * in.D + d;
#pragma unroll
        for (int r = 0; r < R; ++r) {
            if (t + r >= in.T) break;
            Pk out;
            Pk ov;
            if (OG) ov = st[2 * ARR + r * THREADS];
#pragma unroll
            for (int v = 0; v < VEC; ++v) {
                h[v] = fmaf(c[r][v], h[v], u[r][v]);
                float w = h[v];
                if (OG) {
                    const float z = dg::to_f(ov.v[v]);
                    w *= z * dg::sigmoid(z);
                }
                out.v[v] = dg::from_f<T>(t + r < len ? w : 0.f);
            }
            *reinterpret_cast<Pk*>(yp + (int64_t)r * in.D) = out;
        }
    }
    if (h_last && on && rank == 0 && tid < LPR)
#pragma unroll
        for (int v = 0; v < VEC; ++v) h_last[(int64_t)b * in.D + d + v] = state[v];
}

template <typename T, int VEC, int LPR, bool OG>
__global__ void __launch_bounds__(THREADS, 2) scan_backward_kernel(ScanIn in, ScanGrad q) {
    typedef Tile<T, VEC, LPR, OG ? 4 : 3> Tl;
    typedef Pack<T, VEC> Pk;
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ Maps<Tl::CH> maps;          // warp: (P, H) forward; cta: (P, Q) reverse
    __shared__ float back[2][WARPS][Tl::CH];        // Q per warp, reverse (its P is the forward one)
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int S = in.cluster, rank = S > 1 ? (int)cluster_rank() : 0;
    const int blocks = (in.D + Tl::CH - 1) / Tl::CH;
    const int unit = blockIdx.x / S, b = unit / blocks;
    const int lc = tid % LPR, d = (unit % blocks) * Tl::CH + lc * VEC;
    const bool on = d < in.D;
    const int len = in.lengths ? min(max(in.lengths[b], 0), in.T) : in.T;
    const T* x = (const T*)in.x + b * in.x_sb + d;
    const T* g = (const T*)in.g + b * in.g_sb + d;
    const T* o = OG ? (const T*)in.o + b * in.o_sb + d : nullptr;
    const T* dy = (const T*)q.dy + b * q.dy_sb + d;
    const uint8_t* rs = in.resets ? in.resets + (int64_t)b * in.T : nullptr;
    const int nblk = (in.T + DG_SCAN_MARK_STEPS - 1) / DG_SCAN_MARK_STEPS;
    Pk* mine = reinterpret_cast<Pk*>(smem) + tid;
    constexpr int ARR = R * THREADS, STG = (OG ? 4 : 3) * ARR;
    const int span = S * Tl::STEPS, ntiles = (in.T + span - 1) / span;
    const int t_first = rank * Tl::STEPS + (tid / LPR) * R;

    uint8_t next_reset = 0;
    float next_mark[VEC];                  // the state before the CTA's tile
    auto prefetch = [&](int it) {
        const int t = it * span + t_first, t0 = it * span + rank * Tl::STEPS;
        Pk* st = mine + (it & 1) * STG;
        fetch<T, VEC>(st, x + t * in.x_st, in.x_st, len - t, on);
        fetch<T, VEC>(st + ARR, g + t * in.g_st, in.g_st, len - t, on);
        fetch<T, VEC>(st + 2 * ARR, dy + t * q.dy_st, q.dy_st, len - t, on);
        if (OG) fetch<T, VEC>(st + 3 * ARR, o + t * in.o_st, in.o_st, len - t, on);
        copy_commit();
        if (rs) next_reset = (lc < R && t + lc < len) ? rs[t + lc] : 0;
#pragma unroll
        for (int v = 0; v < VEC; ++v)
            next_mark[v] = (on && t0 < in.T) ? q.marks[((int64_t)b * nblk + t0 / DG_SCAN_MARK_STEPS) * in.D + d + v] : 0.f;
    };

    float state[VEC];                      // r of the step after the tiles done so far
#pragma unroll
    for (int v = 0; v < VEC; ++v) state[v] = (q.dh_last && on) ? q.dh_last[(int64_t)b * in.D + d + v] : 0.f;
    if (ntiles > 0) prefetch(ntiles - 1);
    for (int it = ntiles - 1; it >= 0; --it) {
        const int t = it * span + t_first;
        unsigned resets = 0;
        if (rs) resets = __ballot_sync(DG_FULL_MASK, next_reset != 0) >> (lane & ~(LPR - 1));
        float mark[VEC];
#pragma unroll
        for (int v = 0; v < VEC; ++v) mark[v] = next_mark[v];
        if (it > 0) prefetch(it - 1);
        else copy_commit();
        copy_wait<1>();
        const Pk* st = mine + (it & 1) * STG;
        // c, u of the forward map and the gradient that enters at each step
        float c[R][VEC], u[R][VEC], na[R][VEC], e[R][VEC], P[VEC], H[VEC], Q[VEC];
#pragma unroll
        for (int v = 0; v < VEC; ++v) P[v] = 1.f, H[v] = 0.f, Q[v] = 0.f;
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const Pk xv = st[r * THREADS], gv = st[ARR + r * THREADS], dv = st[2 * ARR + r * THREADS];
            Pk ov;
            if (OG) ov = st[3 * ARR + r * THREADS];
#pragma unroll
            for (int v = 0; v < VEC; ++v) {
                float a;
                dg::sigmoid_pair(dg::to_f(gv.v[v]), a, na[r][v]);
                c[r][v] = t + r < len ? ((resets >> r) & 1 ? 0.f : a) : 1.f;
                u[r][v] = t + r < len ? na[r][v] * dg::to_f(xv.v[v]) : 0.f;
                float w = dg::to_f(dv.v[v]);
                if (OG) {
                    const float z = dg::to_f(ov.v[v]);
                    w *= z * dg::sigmoid(z);
                }
                e[r][v] = t + r < len ? w : 0.f;
                H[v] = fmaf(c[r][v], H[v], u[r][v]);
                P[v] *= c[r][v];
            }
        }
#pragma unroll
        for (int r = R - 1; r >= 0; --r)
#pragma unroll
            for (int v = 0; v < VEC; ++v) Q[v] = c[r][v] * (Q[v] + e[r][v]);
        float Pb[VEC], Hb[VEC], Pa[VEC], Qa[VEC];
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
            float Pw, Hw, Pv, Qw;
            warp_before<LPR>(P[v], H[v], Pb[v], Hb[v], Pw, Hw, lane);
            warp_after<LPR>(P[v], Q[v], Pa[v], Qa[v], Pv, Qw, lane);
            if (lane >= 32 - LPR) maps.warp[it & 1][warp][lc * VEC + v] = make_float2(Pw, Hw);
            if (lane < LPR) back[it & 1][warp][lc * VEC + v] = Qw;
        }
        __syncthreads();
        if (S > 1) {
            for (int i = tid; i < S * Tl::CH; i += THREADS) {
                const int ch = i % Tl::CH;
                float2 m = make_float2(1.f, 0.f);
#pragma unroll
                for (int w = WARPS - 1; w >= 0; --w) {
                    const float p = maps.warp[it & 1][w][ch].x;
                    m.y = fmaf(p, m.y, back[it & 1][w][ch]);
                    m.x *= p;
                }
                store_remote(&maps.cta[it & 1][rank][ch], i / Tl::CH, m);
            }
            __syncwarp();
            cluster_barrier();
        }
        float rr[VEC], h[VEC];
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
            const int ch = lc * VEC + v;
            float s = state[v], mine_s = s;
            if (S > 1) {
                for (int k = S - 1; k >= 0; --k) {
                    if (k == rank) mine_s = s;
                    const float2 m = maps.cta[it & 1][k][ch];
                    s = fmaf(m.x, s, m.y);
                }
                state[v] = s;
                s = mine_s;
            }
            float f = mark[v], mine_f = f;
#pragma unroll
            for (int w = WARPS - 1; w >= 0; --w) {
                if (w == warp) mine_s = s;
                s = fmaf(maps.warp[it & 1][w][ch].x, s, back[it & 1][w][ch]);
            }
#pragma unroll
            for (int w = 0; w < WARPS; ++w) {
                if (w == warp) mine_f = f;
                const float2 m = maps.warp[it & 1][w][ch];
                f = fmaf(m.x, f, m.y);
            }
            if (S == 1) state[v] = s;
            rr[v] = fmaf(Pa[v], mine_s, Qa[v]);
            h[v] = fmaf(Pb[v], mine_f, Hb[v]);
        }
        if (!on) continue;
        // forward: u becomes the state before each step; then back through the steps
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
            for (int v = 0; v < VEC; ++v) {
                const float before = h[v];
                h[v] = fmaf(c[r][v], before, u[r][v]);
                u[r][v] = (resets >> r) & 1 ? 0.f : before;
            }
#pragma unroll
        for (int r = R - 1; r >= 0; --r) {
            const Pk xv = st[r * THREADS];
            Pk ov, dv, px, pg, po;
            if (OG) {
                dv = st[2 * ARR + r * THREADS];
                ov = st[3 * ARR + r * THREADS];
            }
            const bool live = t + r < len;
#pragma unroll
            for (int v = 0; v < VEC; ++v) {
                const float xt = dg::to_f(xv.v[v]), et = e[r][v] + rr[v], n = na[r][v];
                float a = c[r][v];
                if ((resets >> r) & 1) a = 1.f - n;             // c is 0 there
                px.v[v] = dg::from_f<T>(live ? et * n : 0.f);
                pg.v[v] = dg::from_f<T>(live ? et * (u[r][v] - xt) * (a * n) : 0.f);
                if (OG) {
                    const float z = dg::to_f(ov.v[v]);
                    float sg, sn;
                    dg::sigmoid_pair(z, sg, sn);
                    const float ht = fmaf(a, u[r][v], n * xt);
                    po.v[v] = dg::from_f<T>(live ? dg::to_f(dv.v[v]) * ht * (sg * fmaf(z, sn, 1.f)) : 0.f);
                }
                rr[v] = c[r][v] * et;
            }
            if (t + r < in.T) {
                *reinterpret_cast<Pk*>((T*)q.dx + b * q.dx_sb + (t + r) * q.dx_st + d) = px;
                *reinterpret_cast<Pk*>((T*)q.dg_ + b * q.dg_sb + (t + r) * q.dg_st + d) = pg;
                if (OG) *reinterpret_cast<Pk*>((T*)q.do_ + b * q.do_sb + (t + r) * q.do_st + d) = po;
            }
        }
    }
    if (q.dh0 && on && rank == 0 && tid < LPR)
#pragma unroll
        for (int v = 0; v < VEC; ++v) q.dh0[(int64_t)b * in.D + d + v] = state[v];
}

template <typename T>
__global__ void scan_step_kernel(int D, const T* x, int64_t x_sb, const T* g, int64_t g_sb, const T* o, int64_t o_sb,
                                 float* h, T* y) {
    const int d = blockIdx.x * blockDim.x + threadIdx.x;
    const int64_t b = blockIdx.y;
    if (d >= D) return;
    float a, na;
    dg::sigmoid_pair(dg::to_f(g[b * g_sb + d]), a, na);
    const float hn = fmaf(a, h[b * D + d], na * dg::to_f(x[b * x_sb + d]));
    h[b * D + d] = hn;
    float out = hn;
    if (o) {
        const float z = dg::to_f(o[b * o_sb + d]);
        out = hn * (z * dg::sigmoid(z));
    }
    y[b * D + d] = dg::from_f<T>(out);
}

// ---------------------------------------------------------------------------
// launches
// ---------------------------------------------------------------------------

// whether rows can be read and written VEC elements at a time
struct Row {
    const void* p;
    int64_t sb, st;
};
bool pairs_aligned(int D, size_t elem, std::initializer_list<Row> rows) {
    if (D % 2) return false;
    for (const Row& r : rows)
        if (r.p && ((reinterpret_cast<uintptr_t>(r.p) % (2 * elem)) || r.sb % 2 || r.st % 2)) return false;
    return true;
}

// Channels per CTA (lpr x vec) and cluster size.  Each CTA walks ceil(tiles / cluster) tiles, and
// `occ` of them share an SM, clusters staying inside one of eight groups of about 18 SMs: the
// least waves x walked steps, taking wide channel blocks (whole 128-byte lines) and small
// clusters (cheap barriers) where that is a tie.
struct Shape {
    int lpr, cluster;
};
Shape shape_of(int B, int T, int D, int vec, int occ) {
    Shape best{32, 1};
    int64_t least = -1;
    for (int lpr = 32; lpr >= 8; lpr /= 2) {
        const int64_t units = (int64_t)B * ((D + lpr * vec - 1) / (lpr * vec));
        const int steps = THREADS / lpr * R, tiles = (T + steps - 1) / steps;
        for (int s = 1; s <= 16 && (s == 1 || s <= tiles); ++s) {
            const int64_t slots = s == 1 ? 148 * occ : 8 * (18 * occ / s) * s;
            const int64_t cost = (units * s + slots - 1) / slots * ((tiles + s - 1) / s) * steps;
            if (least < 0 || cost < least) {
                least = cost;
                best = {lpr, s};
            }
        }
    }
    return best;
}

template <typename K, typename... A>
int launch(K kern, unsigned grid, int cluster, size_t smem, cudaStream_t stream, A... args) {
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return dg_host::record_cuda_error(e);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(THREADS);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)cluster;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    if (cluster > 8) {
        e = cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
        if (e != cudaSuccess) return dg_host::record_cuda_error(e);
    }
    e = cudaLaunchKernelEx(&cfg, kern, args...);
    if (e != cudaSuccess) return dg_host::record_cuda_error(e);
    return dg_host::check_launch();
}

template <typename T, int VEC, int LPR, bool OG>
int run_forward(const ScanIn& in, const float* h0, void* y, float* h_last, float* marks, cudaStream_t s) {
    typedef Tile<T, VEC, LPR, OG ? 3 : 2> Tl;
    const int64_t grid = (int64_t)in.B * ((in.D + Tl::CH - 1) / Tl::CH) * in.cluster;
    if (grid > 0x7fffffff) return DG_ERR_UNSUPPORTED;
    return launch(scan_forward_kernel<T, VEC, LPR, OG>, (unsigned)grid, in.cluster, STAGES * Tl::STAGE, s, in, h0, (T*)y,
                  h_last, marks);
}
template <typename T, int VEC, int LPR, bool OG>
int run_backward(const ScanIn& in, const ScanGrad& q, cudaStream_t s) {
    typedef Tile<T, VEC, LPR, OG ? 4 : 3> Tl;
    const int64_t grid = (int64_t)in.B * ((in.D + Tl::CH - 1) / Tl::CH) * in.cluster;
    if (grid > 0x7fffffff) return DG_ERR_UNSUPPORTED;
    return launch(scan_backward_kernel<T, VEC, LPR, OG>, (unsigned)grid, in.cluster, STAGES * Tl::STAGE, s, in, q);
}

// calls F<T, VEC, LPR, OG>(...) for the sizes at hand
#define SCAN_LPR(F, T, VEC, OG, lpr, ...)                                          \
    ((lpr) == 32 ? F<T, VEC, 32, OG>(__VA_ARGS__) : (lpr) == 16 ? F<T, VEC, 16, OG>(__VA_ARGS__) \
                                                                : F<T, VEC, 8, OG>(__VA_ARGS__))
#define SCAN_RUN(F, T, two, og, lpr, ...)                                                       \
    ((two) ? ((og) ? SCAN_LPR(F, T, 2, true, lpr, __VA_ARGS__) : SCAN_LPR(F, T, 2, false, lpr, __VA_ARGS__)) \
           : ((og) ? SCAN_LPR(F, T, 1, true, lpr, __VA_ARGS__) : SCAN_LPR(F, T, 1, false, lpr, __VA_ARGS__)))

// CTAs that share an SM, by shared memory and registers
constexpr int occupancy(bool backward, size_t elem) { return elem == 4 ? 1 : backward ? 2 : 3; }

}  // namespace

extern "C" {

int dg_gated_scan_forward(int dtype, int B, int T, int D, const void* x, int64_t x_sb, int64_t x_st,
                          const void* gate, int64_t gate_sb, int64_t gate_st, const void* out_gate,
                          int64_t out_gate_sb, int64_t out_gate_st, const float* h0, const int32_t* lengths,
                          const uint8_t* resets, void* y, float* h_last, float* marks, void* stream) {
    if (dtype == DG_DTYPE_F64) return DG_ERR_UNSUPPORTED;
    if (dtype < DG_DTYPE_F32 || dtype > DG_DTYPE_BF16 || B < 0 || T < 0 || D < 0) return DG_ERR_INVALID_ARGUMENT;
    if (B == 0 || D == 0) return DG_OK;
    if (T > 0 && (!x || !gate || !y)) return DG_ERR_INVALID_ARGUMENT;
    if (T == 0 && !h_last) return DG_OK;
    if (T > (1 << 30)) return DG_ERR_UNSUPPORTED;
    const size_t elem = dg_host::dtype_size(dtype);
    const bool two = pairs_aligned(D, elem, {{x, x_sb, x_st}, {gate, gate_sb, gate_st}, {out_gate, out_gate_sb, out_gate_st},
                                             {y, 0, 0}});
    const Shape sh = shape_of(B, T, D, two ? 2 : 1, occupancy(false, elem));
    const ScanIn in{x, gate, out_gate, x_sb, x_st, gate_sb, gate_st, out_gate_sb, out_gate_st, lengths, resets, B, T, D,
                    sh.cluster};
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    DG_DISPATCH_LM(dtype, S, {
        return SCAN_RUN(run_forward, S, two, out_gate != nullptr, sh.lpr, in, h0, y, h_last, marks, s);
    });
    return DG_OK;
}

int dg_gated_scan_backward(int dtype, int B, int T, int D, const void* x, int64_t x_sb, int64_t x_st,
                           const void* gate, int64_t gate_sb, int64_t gate_st, const void* out_gate,
                           int64_t out_gate_sb, int64_t out_gate_st, const int32_t* lengths, const uint8_t* resets,
                           const float* marks, const void* dy, int64_t dy_sb, int64_t dy_st, const float* dh_last,
                           void* dx, int64_t dx_sb, int64_t dx_st, void* dgate, int64_t dgate_sb, int64_t dgate_st,
                           void* dout_gate, int64_t dout_gate_sb, int64_t dout_gate_st, float* dh0, void* stream) {
    if (dtype == DG_DTYPE_F64) return DG_ERR_UNSUPPORTED;
    if (dtype < DG_DTYPE_F32 || dtype > DG_DTYPE_BF16 || B < 0 || T < 0 || D < 0) return DG_ERR_INVALID_ARGUMENT;
    if ((out_gate == nullptr) != (dout_gate == nullptr)) return DG_ERR_INVALID_ARGUMENT;
    if (B == 0 || D == 0) return DG_OK;
    if (T > 0 && (!x || !gate || !marks || !dy || !dx || !dgate)) return DG_ERR_INVALID_ARGUMENT;
    if (T == 0 && !dh0) return DG_OK;
    if (T > (1 << 30)) return DG_ERR_UNSUPPORTED;
    const size_t elem = dg_host::dtype_size(dtype);
    const bool two = pairs_aligned(D, elem, {{x, x_sb, x_st}, {gate, gate_sb, gate_st}, {out_gate, out_gate_sb, out_gate_st},
                                             {dy, dy_sb, dy_st}, {dx, dx_sb, dx_st}, {dgate, dgate_sb, dgate_st},
                                             {dout_gate, dout_gate_sb, dout_gate_st}});
    const Shape sh = shape_of(B, T, D, two ? 2 : 1, occupancy(true, elem));
    const ScanIn in{x, gate, out_gate, x_sb, x_st, gate_sb, gate_st, out_gate_sb, out_gate_st, lengths, resets, B, T, D,
                    sh.cluster};
    const ScanGrad q{marks, dy, dy_sb, dy_st, dh_last, dx, dgate, dout_gate, dx_sb, dx_st, dgate_sb, dgate_st,
                     dout_gate_sb, dout_gate_st, dh0};
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    DG_DISPATCH_LM(dtype, S, { return SCAN_RUN(run_backward, S, two, out_gate != nullptr, sh.lpr, in, q, s); });
    return DG_OK;
}

int dg_gated_scan_step(int dtype, int B, int D, const void* x, int64_t x_sb, const void* gate, int64_t gate_sb,
                       const void* out_gate, int64_t out_gate_sb, float* h, void* y, void* stream) {
    if (dtype == DG_DTYPE_F64) return DG_ERR_UNSUPPORTED;
    if (dtype < DG_DTYPE_F32 || dtype > DG_DTYPE_BF16 || B < 0 || D < 0) return DG_ERR_INVALID_ARGUMENT;
    if (B == 0 || D == 0) return DG_OK;
    if (!x || !gate || !h || !y) return DG_ERR_INVALID_ARGUMENT;
    if (B > 65535) return DG_ERR_UNSUPPORTED;
    DG_DISPATCH_LM(dtype, S, {
        scan_step_kernel<S><<<dim3((D + 127) / 128, B), 128, 0, static_cast<cudaStream_t>(stream)>>>(
            D, static_cast<const S*>(x), x_sb, static_cast<const S*>(gate), gate_sb, static_cast<const S*>(out_gate),
            out_gate_sb, h, static_cast<S*>(y));
    });
    return dg_host::check_launch();
}

}  // extern "C"
