// gated_scan.cu -- the gated linear recurrence h_t = c_t h_{t-1} + (1 - a_t) x_t with
// a = sigmoid(gate): forward, backward and single step.
//
// A run of steps acts on the state as h -> P h + H (P the product of its c, H its end state
// from zero), and such maps compose, so the sequence splits along time:
//   - a thread takes R consecutive steps of VEC channels and composes its map with its
//     neighbours' by shuffles;
//   - a CTA (256 threads) takes a tile of 256 / LPR x R steps by LPR x VEC channels: each warp
//     leaves its map in shared memory, one thread per channel carries the state through them,
//     and every thread applies its steps to the state it starts from.  The CTA walks the
//     sequence tile by tile;
//   - where rows and channels give too few CTAs, a cluster of up to 16 takes consecutive
//     tiles and exchanges their maps through distributed shared memory: asynchronous stores
//     that count on the receiver's mbarrier, so that no fence waits for a warp's other stores.
// A reset (c = 0) is a product of -0, which no product of gates is: there a map gives H whatever the
// state before it, infinite or NaN, where 0 h + H would not.
// Each input is read and each output written once.  The order of every composition is fixed
// by the sizes alone, so results repeat bit for bit.
//
// Inputs come one tile ahead by cp.async into shared memory that only the copying warp (or
// thread) reads: no registers are held for data in flight and no CTA barrier waits for it.
//
// The backward pass carries r_t = c_t (d_t + r_{t+1}) (d the gradient that enters at step t)
// the same way in reverse, and forms the states again from the marks that the forward pass
// leaves every DG_SCAN_MARK_STEPS steps: fp32 states, so nothing is lost to the rounding of
// y, for 4 / 32 of a byte a step.
//
// What bounds it: HBM at 8 (forward, 16-bit, with an output gate) to 14 bytes (backward) an
// element, with issue slots and the special-function unit (two operations for each sigmoid)
// at about half of their limits too; pairs of channels use the two-wide fp32 instructions to
// keep issue slots free.  8 x 4096 x 768 in bf16: forward 51 us (3.9 TB/s, 0.61 of the copy
// bandwidth), backward 102 us (3.5 TB/s, 0.54), with resets 52 and 111 us; 1 x 65536 x 768 forward 140 us
// (2.9 TB/s), as its clusters of 15 leave a fifth of the SM's places empty.
#include <type_traits>

#include "lm_common.cuh"
#include "tc_util.cuh"

namespace dg_host {
uint32_t wait_limit();
}

namespace {

constexpr int THREADS = 256;
constexpr int WARPS = THREADS / 32;
constexpr int STAGES = 2;                  // tiles of input in shared memory
constexpr int kForwardSteps = 8, kBackwardSteps = 4;      // steps per thread, by the registers of three CTAs to an SM

struct ScanIn {
    const void *x, *g, *o;
    int64_t x_sb, x_st, g_sb, g_st, o_sb, o_st;
    const int32_t* lengths;
    const uint8_t* resets;
    int B, T, D, cluster;
    int32_t* status;
    uint32_t wait_limit;
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

// ---- cp.async and clusters -------------------------------------------------------
// copies BYTES (4, 8 or 16), or zeros where !on
template <int BYTES>
__device__ __forceinline__ void copy_async(void* dst, const void* src, bool on) {
    const int n = on ? BYTES : 0;
    const uint32_t a = (uint32_t)__cvta_generic_to_shared(dst);
    if constexpr (BYTES == 16)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(a), "l"(src), "r"(n) : "memory");
    else
        asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(a), "l"(src), "n"(BYTES), "r"(n) : "memory");
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
// stores v at p's place in CTA `rank` and counts its 8 bytes on `bar` there
__device__ __forceinline__ void store_remote(float2* p, uint64_t* bar, uint32_t rank, float2 v) {
    uint32_t a, m;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"((uint32_t)__cvta_generic_to_shared(p)), "r"(rank));
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(m) : "r"((uint32_t)__cvta_generic_to_shared(bar)), "r"(rank));
    asm volatile("st.async.shared::cluster.mbarrier::complete_tx::bytes.v2.f32 [%0], {%1, %2}, [%3];" ::"r"(a), "f"(v.x),
                 "f"(v.y), "r"(m)
                 : "memory");
}

// ---- one or two channels at a time ------------------------------------------------
template <int VEC> struct alignas(4 * VEC) Fv {
    float v[VEC];
};
template <int VEC> __device__ __forceinline__ Fv<VEC> all(float x) {
    Fv<VEC> r;
#pragma unroll
    for (int i = 0; i < VEC; ++i) r.v[i] = x;
    return r;
}
__device__ __forceinline__ Fv<1> vfma(Fv<1> a, Fv<1> b, Fv<1> c) { return {fmaf(a.v[0], b.v[0], c.v[0])}; }
__device__ __forceinline__ Fv<1> vmul(Fv<1> a, Fv<1> b) { return {a.v[0] * b.v[0]}; }
__device__ __forceinline__ Fv<1> vadd(Fv<1> a, Fv<1> b) { return {a.v[0] + b.v[0]}; }
__device__ __forceinline__ uint64_t bits(Fv<2> a) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a.v[0]), "f"(a.v[1]));
    return r;
}
__device__ __forceinline__ Fv<2> unbits(uint64_t a) {
    Fv<2> r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.v[0]), "=f"(r.v[1]) : "l"(a));
    return r;
}
__device__ __forceinline__ Fv<2> vfma(Fv<2> a, Fv<2> b, Fv<2> c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(bits(a)), "l"(bits(b)), "l"(bits(c)));
    return unbits(r);
}
__device__ __forceinline__ Fv<2> vmul(Fv<2> a, Fv<2> b) {
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(bits(a)), "l"(bits(b)));
    return unbits(r);
}
__device__ __forceinline__ Fv<2> vadd(Fv<2> a, Fv<2> b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(bits(a)), "l"(bits(b)));
    return unbits(r);
}

// VEC storage elements
template <typename T, int VEC> struct alignas(sizeof(T) * VEC) Pack {
    T v[VEC];
};
template <typename T, int VEC> __device__ __forceinline__ Fv<VEC> widen(const Pack<T, VEC>& p) {
    Fv<VEC> r;
    if constexpr (std::is_same<T, __nv_bfloat16>::value && VEC == 2) {
        const uint32_t u = *reinterpret_cast<const uint32_t*>(&p);
        r.v[0] = __uint_as_float(u << 16);
        r.v[1] = __uint_as_float(u & 0xffff0000u);
    } else {
#pragma unroll
        for (int i = 0; i < VEC; ++i) r.v[i] = dg::to_f(p.v[i]);
    }
    return r;
}
template <typename T, int VEC> __device__ __forceinline__ Pack<T, VEC> narrow(Fv<VEC> a) {
    Pack<T, VEC> p;
    if constexpr (std::is_same<T, __nv_bfloat16>::value && VEC == 2) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(a.v[0], a.v[1]);
        p = *reinterpret_cast<const Pack<T, VEC>*>(&h);
    } else if constexpr (std::is_same<T, __half>::value && VEC == 2) {
        const __half2 h = __floats2half2_rn(a.v[0], a.v[1]);
        p = *reinterpret_cast<const Pack<T, VEC>*>(&h);
    } else {
#pragma unroll
        for (int i = 0; i < VEC; ++i) p.v[i] = dg::from_f<T>(a.v[i]);
    }
    return p;
}

// dg::sigmoid_pair: the recurrence's gate a and na = 1 - a
template <int VEC> __device__ __forceinline__ void gates(Fv<VEC> z, Fv<VEC>& a, Fv<VEC>& na) {
    Fv<VEC> e = vmul(z, all<VEC>(-1.4426950408889634f));
#pragma unroll
    for (int i = 0; i < VEC; ++i) e.v[i] = dg::exp2_ftz(e.v[i]);
    a = vadd(e, all<VEC>(1.f));
#pragma unroll
    for (int i = 0; i < VEC; ++i) a.v[i] = dg::rcp_ftz(a.v[i]);
    const Fv<VEC> small = vmul(e, a), large = vfma(a, all<VEC>(-1.f), all<VEC>(1.f));
#pragma unroll
    for (int i = 0; i < VEC; ++i) na.v[i] = e.v[i] > 1.f ? large.v[i] : small.v[i];
}
// z sigmoid(z) (dg::sigmoid), and dg::slope_pair
template <int VEC> __device__ __forceinline__ Fv<VEC> silu(Fv<VEC> z) {
    Fv<VEC> e = vmul(z, all<VEC>(-1.4426950408889634f));
#pragma unroll
    for (int i = 0; i < VEC; ++i) e.v[i] = dg::exp2_ftz(e.v[i]);
    e = vadd(e, all<VEC>(1.f));
#pragma unroll
    for (int i = 0; i < VEC; ++i) e.v[i] = dg::rcp_ftz(e.v[i]);
    return vmul(z, e);
}
template <int VEC> __device__ __forceinline__ void slope_pair(Fv<VEC> z, Fv<VEC>& s, Fv<VEC>& n) {
    Fv<VEC> e = vmul(z, all<VEC>(-1.4426950408889634f));
#pragma unroll
    for (int i = 0; i < VEC; ++i) e.v[i] = fminf(dg::exp2_ftz(e.v[i]), 3.4e38f);
    s = vadd(e, all<VEC>(1.f));
#pragma unroll
    for (int i = 0; i < VEC; ++i) s.v[i] = dg::rcp_ftz(s.v[i]);
    n = vmul(e, s);
}

// The marked product of a map that holds a reset, whether a product is one, and the state after a map.
// The chains over warps and CTAs compute P s + H and look at their end alone: a state that is not finite
// does not become so again, and then, in calls with resets, the chain is taken once more by after().
// (after() at each link cost up to 18% of a call, 1 x 65536 x 768 backward 299 to 353 us; the look at the
// end 2%, 306 us.  Calls without resets, RS = false, have neither.)
constexpr float kReset = -0.f;
__device__ __forceinline__ bool is_reset(float P) { return __float_as_uint(P) == 0x80000000u; }
__device__ __forceinline__ bool finite(float s) { return fabsf(s) < INFINITY; }
__device__ __forceinline__ float after(float P, float H, float s) { return is_reset(P) ? H : fmaf(P, s, H); }
template <int VEC> __device__ __forceinline__ Fv<VEC> after(Fv<VEC> P, Fv<VEC> H, Fv<VEC> s) {
    s = vfma(P, s, H);
#pragma unroll
    for (int i = 0; i < VEC; ++i) s.v[i] = is_reset(P.v[i]) ? H.v[i] : s.v[i];
    return s;
}

// p, marked where one of the products in `marks` is
__device__ __forceinline__ float marked(float p, uint32_t marks) {
    return __uint_as_float(__float_as_uint(p) | (marks & 0x80000000u));
}
// A thread's chain over its warps' maps (P of `maps`, H of `maps` or `back`) by after(), first to last or last to
// first, from the state s: the states between them into carry (or null), the last returned.
template <bool FORWARD, int CH>
__device__ __forceinline__ float chain_again(const float2 (*maps)[CH], const float (*back)[CH], int tid, float s,
                                             float (*carry)[CH]) {
#pragma unroll 1
    for (int i = 0; i < WARPS; ++i) {
        const int w = FORWARD ? i : WARPS - 1 - i;
        if (carry) carry[w][tid] = s;
        const float2 m = maps[w][tid];
        s = after(m.x, back ? back[w][tid] : m.y, s);
    }
    return s;
}

// What a CTA keeps of its tile, per channel; the maps of the cluster's CTAs (two tiles' worth of
// [cluster][CH]) lie behind the input stages
template <int CH> struct Maps {
    float2 warp[WARPS][CH];                // each warp's (P, H)
    float carry[WARPS][CH];                // the state each warp starts from
    uint64_t received[2];                  // the cluster's maps of even and odd tiles
};
template <int CH> struct MapsBack : Maps<CH> {
    float back[WARPS][CH];                 // each warp's Q of the reverse map
    float carry_back[WARPS][CH];
};

template <typename T, int VEC, int LPR, int R, int ARRAYS> struct Tile {
    static constexpr int STEPS = THREADS / LPR * R, CH = LPR * VEC;
    typedef Pack<T, VEC> P;
    // one input's tile: [warp][row group][step][channel]
    static constexpr int WARP_PACKS = 32 / LPR * (R * LPR + (LPR < 32 ? LPR : 0));
    static constexpr int ARRAY = WARPS * WARP_PACKS;              // packs
    static constexpr size_t STAGE = (size_t)ARRAYS * ARRAY * sizeof(P);
    static constexpr size_t bytes(int cluster) {
        return STAGES * STAGE + (cluster > 1 ? 2 * cluster * CH * sizeof(float2) : 0);
    }
};

// A warp's steps of one input into its part of a stage.  WIDE: 16 bytes a lane, any lane any
// step of the warp.  Otherwise each thread copies the steps it reads itself.  Row groups lie kPad
// packs further apart than their steps need, so that a warp's reads meet 32 different banks.
template <int LPR> constexpr int kPad = LPR < 32 ? LPR : 0;
template <typename T, int VEC, int LPR, int R, bool WIDE>
__device__ __forceinline__ void fetch(Pack<T, VEC>* warp_part, const T* row, int64_t step, int t_warp, int len, int d0,
                                      int D, int lane) {
    constexpr int GROUP = R * LPR + kPad<LPR>;                    // packs from one row group to the next
    if constexpr (WIDE) {
        constexpr int E = 16 / sizeof(T), CPS = LPR * VEC / E, SPC = 32 / CPS, N = 32 / LPR * R / SPC;
        const int col = lane % CPS * E;
        const bool on = d0 + col < D;
        const T* p = on ? row + (int64_t)(t_warp + lane / CPS) * step + d0 + col : row;
        const int64_t advance = on ? SPC * step : 0;
        const int left = on ? len - t_warp - lane / CPS : 0;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int s = lane / CPS + i * SPC;
            T* dst = reinterpret_cast<T*>(warp_part) + (s / R * GROUP + s % R * LPR) * VEC + col;
            copy_async<16>(dst, p, i * SPC < left);                // reads nothing where it is false
            p += advance;
        }
    } else {
        const int lc = lane % LPR, s0 = lane / LPR * R, d = d0 + lc * VEC;
        const T* p = row + (int64_t)(t_warp + s0) * step + d;
        Pack<T, VEC>* dst = warp_part + lane / LPR * GROUP + lc;
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const bool live = d < D && t_warp + s0 + r < len;
            if constexpr (sizeof(T) * VEC >= 4) {
                copy_async<sizeof(T) * VEC>(dst + r * LPR, live ? p : row, live);
            } else {                       // 2 bytes: below what cp.async copies
                T z = dg::from_f<T>(0.f);
                if (live) z = *p;
                dst[r * LPR].v[0] = z;
            }
            p += step;
        }
    }
}

// composes (P, H) maps over the row groups of a warp.  In: the thread's own map; out: the map of
// the groups before it (FORWARD) or after it, and the whole warp's, which the last (first) group has
// (MARKED: some group's map holds a reset)
template <int LPR, int VEC, bool FORWARD, bool MARKED>
__device__ __forceinline__ void warp_maps(Fv<VEC> P, Fv<VEC> H, Fv<VEC>& Pb, Fv<VEC>& Hb, Fv<VEC>& Pw, Fv<VEC>& Hw,
                                          int lane) {
    auto from = [&](float x, int o) {
        return FORWARD ? __shfl_up_sync(DG_FULL_MASK, x, o) : __shfl_down_sync(DG_FULL_MASK, x, o);
    };
#pragma unroll
    for (int v = 0; v < VEC; ++v) {
#pragma unroll
        for (int o = LPR; o < 32; o <<= 1) {
            const float p = from(P.v[v], o), h = from(H.v[v], o);
            if ((FORWARD ? lane >= o : lane + o < 32) && !(MARKED && is_reset(P.v[v]))) {
                H.v[v] = fmaf(P.v[v], h, H.v[v]);
                P.v[v] *= p;
            }
        }
        Pb.v[v] = 1.f;
        Hb.v[v] = 0.f;
        if (LPR < 32) {
            const float p = from(P.v[v], LPR & 31), h = from(H.v[v], LPR & 31);
            if (FORWARD ? lane >= LPR : lane + LPR < 32) {
                Pb.v[v] = p;
                Hb.v[v] = h;
            }
        }
    }
    Pw = P;
    Hw = H;
}

// where a thread stands: shared by both passes
template <int LPR, int VEC, int R> struct Place {
    int warp, lane, lc, rank, b, d0, d, span, ntiles;
    bool on;
    __device__ __forceinline__ Place(const ScanIn& in) {
        constexpr int CH = LPR * VEC, STEPS = THREADS / LPR * R;
        warp = threadIdx.x >> 5, lane = threadIdx.x & 31, lc = lane % LPR;
        rank = in.cluster > 1 ? (int)cluster_rank() : 0;
        const int blocks = (in.D + CH - 1) / CH, unit = blockIdx.x / in.cluster;
        b = unit / blocks;
        d0 = unit % blocks * CH;
        d = d0 + lc * VEC;
        on = d < in.D;
        span = in.cluster * STEPS;
        ntiles = (in.T + span - 1) / span;
    }
    // the first step of this warp in tile `it`, and of this thread
    __device__ __forceinline__ int warp_step(int it) const {
        return it * span + rank * (THREADS / LPR * R) + warp * (32 / LPR * R);
    }
    __device__ __forceinline__ int step(int it) const { return warp_step(it) + lane / LPR * R; }
};

// Where documents start in a warp's steps.  The load was made a tile earlier: lane r of a group holds step
// r, so the group's bits of the vote are its thread's: bit r for step r.
template <int LPR, int R> __device__ __forceinline__ uint8_t load_reset(const uint8_t* rs, int t, int lc, int len) {
    return lc < R && t + lc < len ? rs[t + lc] : 0;
}
template <int LPR, int R> __device__ __forceinline__ unsigned reset_bits(unsigned vote, int lane) {
    static_assert(LPR >= R, "one lane per step");
    return vote >> (lane & ~(LPR - 1)) & ((1u << R) - 1);
}

// the forward map of a thread's steps: c, u and their composition (P, H).  WHOLE: every step is
// valid and none starts a document.
template <bool WHOLE, typename T, int VEC, int LPR, int R>
__device__ __forceinline__ void forward_map(const Pack<T, VEC>* xs, const Pack<T, VEC>* gs, int left, unsigned resets,
                                            Fv<VEC> (&c)[R], Fv<VEC> (&u)[R], Fv<VEC>* nas, Fv<VEC>& P, Fv<VEC>& H) {
#pragma unroll
    for (int r = 0; r < R; ++r) {
        Fv<VEC> na;
        gates(widen(gs[r * LPR]), c[r], na);
        u[r] = vmul(na, widen(xs[r * LPR]));
        const bool reset = !WHOLE && r < left && (resets >> r) & 1;
        if (!WHOLE && r >= left) c[r] = all<VEC>(1.f), u[r] = all<VEC>(0.f);
        if (reset) c[r] = all<VEC>(kReset);
        H = r == 0 || reset ? u[r] : vfma(c[r], H, u[r]);
        P = r == 0 || reset ? c[r] : vmul(P, c[r]);
        if (nas) nas[r] = na;
    }
}

// y of a thread's steps from the state h before them; `left` valid steps, `room` steps inside T
template <bool WHOLE, typename T, int VEC, int LPR, bool OG, int R>
__device__ __forceinline__ void forward_apply(Fv<VEC> h, const Fv<VEC> (&c)[R], const Fv<VEC> (&u)[R],
                                              const Pack<T, VEC>* os, T* y, int D, int left, int room) {
#pragma unroll
    for (int r = 0; r < R; ++r) {
        h = WHOLE ? vfma(c[r], h, u[r]) : after(c[r], u[r], h);
        Fv<VEC> w = h;
        if (OG) w = vmul(w, silu(widen(os[r * LPR])));
        if (!WHOLE && r >= left) w = all<VEC>(0.f);
        if (WHOLE || r < room) *reinterpret_cast<Pack<T, VEC>*>(y + (int64_t)r * D) = narrow<T>(w);
    }
}

// The cluster's part of a tile: this CTA's map to all, then the state before this CTA and (returned
// in `state`) after the whole span.  Called by the threads that carry a channel.
template <int CH, bool FORWARD, bool RS>
__device__ __forceinline__ float through_cluster(float2* maps, uint64_t* received, float2 own, int tid, int rank, int S,
                                                 int n, float& state, uint32_t limit, bool& bad) {
    const int buf = n & 1;
    float2* m = maps + (size_t)buf * S * CH;
    if (tid == 0) tc::mbar_expect_tx(received + buf, S * CH * (uint32_t)sizeof(float2));
    for (int k = 0; k < S; ++k) store_remote(m + rank * CH + tid, received + buf, k, own);
    if (!bad) bad = !tc::mbar_wait(received + buf, (n >> 1) & 1, limit);
    float s = state, before = s;
    for (int i = 0; i < S; ++i) {
        const int k = FORWARD ? i : S - 1 - i;
        if (k == rank) before = s;
        const float2 a = m[k * CH + tid];
        s = fmaf(a.x, s, a.y);
    }
    if (RS && !finite(s)) {
        s = state;
#pragma unroll 1
        for (int i = 0; i < S; ++i) {
            const int k = FORWARD ? i : S - 1 - i;
            if (k == rank) before = s;
            const float2 a = m[k * CH + tid];
            s = after(a.x, a.y, s);
        }
    }
    state = s;
    return before;
}

// Barriers of the cluster exchange: set up before the first tile; at the end, a CTA whose wait gave
// up says so and stays until the others' stores have landed.
__device__ __forceinline__ void open_exchange(uint64_t* received, int S) {
    if (S == 1) return;
    if (threadIdx.x == 0) {
        tc::mbar_init(received, 1);
        tc::mbar_init(received + 1, 1);
        tc::fence_barrier_init();
    }
    __syncthreads();
    cluster_barrier();
}
__device__ __forceinline__ void close_exchange(int S, bool bad, int32_t* status) {
    if (S == 1) return;
    if (bad) dg::flag_status(status, DG_DEVCHK_TIMEOUT);
    if (__syncthreads_or(bad)) {
        const uint64_t t0 = tc::globaltimer_ns();
        for (int i = 0; i < (1 << 20) && tc::globaltimer_ns() - t0 < 2000000; ++i) __nanosleep(1000);
    }
    __syncwarp();
    cluster_barrier();
}

// RS: the call has resets.  Three CTAs share an SM, two where pairs of fp32 channels fill its shared memory.
template <typename T, int VEC, int LPR, bool WIDE, bool OG, bool RS>
__global__ void __launch_bounds__(THREADS, sizeof(T) * VEC == 8 ? 2 : 3)
    scan_forward_kernel(ScanIn in, const float* h0, T* y, float* h_last, float* marks) {
    constexpr int R = kForwardSteps;
    static_assert(DG_SCAN_MARK_STEPS % R == 0, "a mark falls on a thread's first step");
    typedef Tile<T, VEC, LPR, R, OG ? 3 : 2> Tl;
    typedef Pack<T, VEC> Pk;
    typedef Fv<VEC> V;
    extern __shared__ __align__(16) uint8_t smem[];
    float2* cta_maps = reinterpret_cast<float2*>(smem + STAGES * Tl::STAGE);
    __shared__ Maps<Tl::CH> maps;
    const Place<LPR, VEC, R> at(in);
    const int tid = threadIdx.x, S = in.cluster, d = at.d;
    const T* x = (const T*)in.x + at.b * in.x_sb;
    const T* g = (const T*)in.g + at.b * in.g_sb;
    const T* o = OG ? (const T*)in.o + at.b * in.o_sb : nullptr;
    const uint8_t* rs = RS ? in.resets + (int64_t)at.b * in.T : nullptr;
    const int nblk = (in.T + DG_SCAN_MARK_STEPS - 1) / DG_SCAN_MARK_STEPS;
    constexpr int ARR = Tl::ARRAY, STG = (OG ? 3 : 2) * ARR;
    Pk* warp_part = reinterpret_cast<Pk*>(smem) + at.warp * Tl::WARP_PACKS;
    const int own = at.lane / LPR * (R * LPR + kPad<LPR>) + at.lc;              // this thread's first pack in it
    bool bad = false;
    open_exchange(maps.received, S);
    dg::wait_for_previous();
    const int len = in.lengths ? min(max(in.lengths[at.b], 0), in.T) : in.T;

    uint8_t next_reset = 0;
    auto prefetch = [&](int it) {
        const int t = at.warp_step(it);
        Pk* st = warp_part + (it & 1) * STG;
        fetch<T, VEC, LPR, R, WIDE>(st, x, in.x_st, t, len, at.d0, in.D, at.lane);
        fetch<T, VEC, LPR, R, WIDE>(st + ARR, g, in.g_st, t, len, at.d0, in.D, at.lane);
        if (OG) fetch<T, VEC, LPR, R, WIDE>(st + 2 * ARR, o, in.o_st, t, len, at.d0, in.D, at.lane);
        copy_commit();
        if (RS) next_reset = load_reset<LPR, R>(rs, at.step(it), at.lc, len);
    };

    // thread c < CH carries channel d0 + c from tile to tile
    float state = 0.f;
    if (tid < Tl::CH && h0 && at.d0 + tid < in.D) state = h0[(int64_t)at.b * in.D + at.d0 + tid];
    if (at.ntiles > 0) prefetch(0);
    for (int it = 0; it < at.ntiles; ++it) {
        const int t = at.step(it);
        const unsigned vote = RS ? __ballot_sync(DG_FULL_MASK, next_reset != 0) : 0;
        const unsigned resets = reset_bits<LPR, R>(vote, at.lane);
        __syncwarp();                      // the other stage has been read
        if (it + 1 < at.ntiles) prefetch(it + 1);
        else copy_commit();
        copy_wait<1>();
        __syncwarp();
        const Pk* st = warp_part + (it & 1) * STG + own;
        V c[R], u[R], P, H;
        const bool whole = t + R <= len && resets == 0;
        if (whole) forward_map<true, T, VEC, LPR, R>(st, st + ARR, R, 0, c, u, nullptr, P, H);
        else forward_map<false, T, VEC, LPR, R>(st, st + ARR, len - t, resets, c, u, nullptr, P, H);
        V Pb, Hb, Pw, Hw;
        if (vote) warp_maps<LPR, VEC, true, true>(P, H, Pb, Hb, Pw, Hw, at.lane);
        else warp_maps<LPR, VEC, true, false>(P, H, Pb, Hb, Pw, Hw, at.lane);
        if (at.lane >= 32 - LPR)
#pragma unroll
            for (int v = 0; v < VEC; ++v) maps.warp[at.warp][at.lc * VEC + v] = make_float2(Pw.v[v], Hw.v[v]);
        __syncthreads();
        if (tid < Tl::CH) {
            float2 m[WARPS];
#pragma unroll
            for (int w = 0; w < WARPS; ++w) m[w] = maps.warp[w][tid];
            float s = state;
            if (S > 1) {
                float2 a = m[0];
                uint32_t mark = __float_as_uint(a.x);
#pragma unroll
                for (int w = 1; w < WARPS; ++w) {
                    a = make_float2(a.x * m[w].x, fmaf(m[w].x, a.y, m[w].y));
                    mark |= __float_as_uint(m[w].x);
                }
                a.x = marked(a.x, mark);
                if (RS && !finite(a.y)) a.y = chain_again<true, Tl::CH>(maps.warp, nullptr, tid, 0.f, nullptr);
                s = through_cluster<Tl::CH, true, RS>(cta_maps, maps.received, a, tid, at.rank, S, it, state,
                                                      in.wait_limit, bad);
            }
            const float s0 = s;
#pragma unroll
            for (int w = 0; w < WARPS; ++w) {
                maps.carry[w][tid] = s;
                s = fmaf(m[w].x, s, m[w].y);
            }
            if (RS && !finite(s)) s = chain_again<true, Tl::CH>(maps.warp, nullptr, tid, s0, maps.carry);
            if (S == 1) state = s;
        }
        __syncthreads();
        V h = *reinterpret_cast<const V*>(&maps.carry[at.warp][at.lc * VEC]);
        if (LPR < 32) h = vote ? after(Pb, Hb, h) : vfma(Pb, h, Hb);
        if (at.on) {
            if (marks && t < in.T && t % DG_SCAN_MARK_STEPS == 0)
#pragma unroll
                for (int v = 0; v < VEC; ++v)
                    marks[((int64_t)at.b * nblk + t / DG_SCAN_MARK_STEPS) * in.D + d + v] = h.v[v];
            T* yp = y + ((int64_t)at.b * in.T + t) * in.D + d;
            if (whole) forward_apply<true, T, VEC, LPR, OG, R>(h, c, u, st + 2 * ARR, yp, in.D, R, R);
            else forward_apply<false, T, VEC, LPR, OG, R>(h, c, u, st + 2 * ARR, yp, in.D, len - t, in.T - t);
        }
    }
    dg::let_next_start();                  // not before: its CTAs would fill the SMs unevenly (8 us of 162)
    if (h_last && at.rank == 0 && tid < Tl::CH && at.d0 + tid < in.D)
        h_last[(int64_t)at.b * in.D + at.d0 + tid] = state;
    close_exchange(S, bad, in.status);
}

// the gradients of a thread's steps, last to first: u holds the state before each step (0 at a
// reset), rr what comes back from the steps after them
template <bool WHOLE, typename T, int VEC, int LPR, bool OG, int R>
__device__ __forceinline__ void backward_apply(Fv<VEC> rr, const Fv<VEC> (&c)[R], const Fv<VEC> (&u)[R],
                                               const Fv<VEC> (&na)[R], const Fv<VEC> (&e)[R], const Pack<T, VEC>* xs,
                                               const Pack<T, VEC>* dys, const Pack<T, VEC>* os, T* px, int64_t sx, T* pg,
                                               int64_t sg, T* po, int64_t so, int left, int room, unsigned resets) {
#pragma unroll
    for (int r = R - 1; r >= 0; --r) {
        const Fv<VEC> xt = widen(xs[r * LPR]), et = vadd(e[r], rr), n = na[r];
        Fv<VEC> a = c[r];
        if (!WHOLE && ((resets >> r) & 1)) a = vfma(n, all<VEC>(-1.f), all<VEC>(1.f));      // c is 0 there
        const Fv<VEC> en = vmul(et, n);
        Fv<VEC> gx = en, gg = vmul(vmul(en, a), vfma(xt, all<VEC>(-1.f), u[r])), go = all<VEC>(0.f);
        if (OG) {
            const Fv<VEC> z = widen(os[r * LPR]);
            Fv<VEC> sg_, sn;
            slope_pair(z, sg_, sn);
            const Fv<VEC> ht = vfma(a, u[r], vmul(n, xt));
            go = vmul(vmul(widen(dys[r * LPR]), ht), vmul(sg_, vfma(z, sn, all<VEC>(1.f))));
        }
        rr = vmul(c[r], et);
        if (!WHOLE && ((resets >> r) & 1)) rr = all<VEC>(0.f);
        if (!WHOLE && r >= left) gx = gg = go = all<VEC>(0.f);
        if (WHOLE || r < room) {
            *reinterpret_cast<Pack<T, VEC>*>(px + r * sx) = narrow<T>(gx);
            *reinterpret_cast<Pack<T, VEC>*>(pg + r * sg) = narrow<T>(gg);
            if (OG) *reinterpret_cast<Pack<T, VEC>*>(po + r * so) = narrow<T>(go);
        }
    }
}

template <typename T, int VEC, int LPR, bool WIDE, bool OG, bool RS>
__global__ void __launch_bounds__(THREADS, sizeof(T) * VEC == 8 ? 2 : 3) scan_backward_kernel(ScanIn in, ScanGrad q) {
    constexpr int R = kBackwardSteps;
    typedef Tile<T, VEC, LPR, R, OG ? 4 : 3> Tl;
    static_assert(Tl::STEPS % DG_SCAN_MARK_STEPS == 0, "tiles start at marks");
    typedef Pack<T, VEC> Pk;
    typedef Fv<VEC> V;
    extern __shared__ __align__(16) uint8_t smem[];
    float2* cta_maps = reinterpret_cast<float2*>(smem + STAGES * Tl::STAGE);
    __shared__ MapsBack<Tl::CH> maps;
    const Place<LPR, VEC, R> at(in);
    const int tid = threadIdx.x, S = in.cluster, d = at.d;
    const T* x = (const T*)in.x + at.b * in.x_sb;
    const T* g = (const T*)in.g + at.b * in.g_sb;
    const T* o = OG ? (const T*)in.o + at.b * in.o_sb : nullptr;
    const T* dy = (const T*)q.dy + at.b * q.dy_sb;
    const uint8_t* rs = RS ? in.resets + (int64_t)at.b * in.T : nullptr;
    const int nblk = (in.T + DG_SCAN_MARK_STEPS - 1) / DG_SCAN_MARK_STEPS;
    constexpr int ARR = Tl::ARRAY, STG = (OG ? 4 : 3) * ARR;
    Pk* warp_part = reinterpret_cast<Pk*>(smem) + at.warp * Tl::WARP_PACKS;
    const int own = at.lane / LPR * (R * LPR + kPad<LPR>) + at.lc;
    const bool carries = tid < Tl::CH && at.d0 + tid < in.D;      // thread c carries channel d0 + c
    bool bad = false;
    open_exchange(maps.received, S);
    dg::wait_for_previous();
    const int len = in.lengths ? min(max(in.lengths[at.b], 0), in.T) : in.T;

    uint8_t next_reset = 0;
    float next_mark = 0.f;                 // the state before the CTA's tile
    auto prefetch = [&](int it) {
        const int t = at.warp_step(it), t0 = it * at.span + at.rank * Tl::STEPS;
        Pk* st = warp_part + (it & 1) * STG;
        fetch<T, VEC, LPR, R, WIDE>(st, x, in.x_st, t, len, at.d0, in.D, at.lane);
        fetch<T, VEC, LPR, R, WIDE>(st + ARR, g, in.g_st, t, len, at.d0, in.D, at.lane);
        fetch<T, VEC, LPR, R, WIDE>(st + 2 * ARR, dy, q.dy_st, t, len, at.d0, in.D, at.lane);
        if (OG) fetch<T, VEC, LPR, R, WIDE>(st + 3 * ARR, o, in.o_st, t, len, at.d0, in.D, at.lane);
        copy_commit();
        if (RS) next_reset = load_reset<LPR, R>(rs, at.step(it), at.lc, len);
        if (carries && t0 < in.T)
            next_mark = q.marks[((int64_t)at.b * nblk + t0 / DG_SCAN_MARK_STEPS) * in.D + at.d0 + tid];
    };

    float state = 0.f;                     // r of the step after the tiles done so far
    if (carries && q.dh_last) state = q.dh_last[(int64_t)at.b * in.D + at.d0 + tid];
    if (at.ntiles > 0) prefetch(at.ntiles - 1);
    for (int it = at.ntiles - 1; it >= 0; --it) {
        const int t = at.step(it);
        const unsigned vote = RS ? __ballot_sync(DG_FULL_MASK, next_reset != 0) : 0;
        const unsigned resets = reset_bits<LPR, R>(vote, at.lane);
        const float mark = next_mark;
        __syncwarp();
        if (it > 0) prefetch(it - 1);
        else copy_commit();
        copy_wait<1>();
        __syncwarp();
        const Pk* st = warp_part + (it & 1) * STG + own;
        const bool whole = t + R <= len && resets == 0;
        // c and u of the forward map, and the gradient that enters at each step
        V c[R], u[R], na[R], e[R], P, H, Q = all<VEC>(0.f);
        if (whole) forward_map<true, T, VEC, LPR, R>(st, st + ARR, R, 0, c, u, na, P, H);
        else forward_map<false, T, VEC, LPR, R>(st, st + ARR, len - t, resets, c, u, na, P, H);
#pragma unroll
        for (int r = R - 1; r >= 0; --r) {
            e[r] = widen(st[2 * ARR + r * LPR]);
            if (OG) e[r] = vmul(e[r], silu(widen(st[3 * ARR + r * LPR])));
            Q = r == R - 1 ? vmul(c[r], e[r]) : vmul(c[r], vadd(Q, e[r]));       // dy is 0 beyond len
        }
        if (resets) {                      // what comes back stops at a reset, finite or not
#pragma unroll
            for (int r = R - 1; r >= 0; --r)
                Q = (resets >> r) & 1 ? all<VEC>(0.f) : r == R - 1 ? vmul(c[r], e[r]) : vmul(c[r], vadd(Q, e[r]));
        }
        V Pb, Hb, Pa, Qa, Pw, Hw, Pv, Qw;
        if (vote) {
            warp_maps<LPR, VEC, true, true>(P, H, Pb, Hb, Pw, Hw, at.lane);
            warp_maps<LPR, VEC, false, true>(P, Q, Pa, Qa, Pv, Qw, at.lane);
        } else {
            warp_maps<LPR, VEC, true, false>(P, H, Pb, Hb, Pw, Hw, at.lane);
            warp_maps<LPR, VEC, false, false>(P, Q, Pa, Qa, Pv, Qw, at.lane);
        }
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
            if (at.lane >= 32 - LPR) maps.warp[at.warp][at.lc * VEC + v] = make_float2(Pw.v[v], Hw.v[v]);
            if (at.lane < LPR) maps.back[at.warp][at.lc * VEC + v] = Qw.v[v];
        }
        __syncthreads();
        if (tid < Tl::CH) {
            float2 m[WARPS];
            float bk[WARPS];
#pragma unroll
            for (int w = 0; w < WARPS; ++w) m[w] = maps.warp[w][tid], bk[w] = maps.back[w][tid];
            float f = mark, s = state;
#pragma unroll
            for (int w = 0; w < WARPS; ++w) {
                maps.carry[w][tid] = f;
                f = fmaf(m[w].x, f, m[w].y);
            }
            if (RS && !finite(f)) chain_again<true, Tl::CH>(maps.warp, nullptr, tid, mark, maps.carry);
            if (S > 1) {
                float2 a = make_float2(m[WARPS - 1].x, bk[WARPS - 1]);
                uint32_t marks = __float_as_uint(a.x);
#pragma unroll
                for (int w = WARPS - 2; w >= 0; --w) {
                    a = make_float2(a.x * m[w].x, fmaf(m[w].x, a.y, bk[w]));
                    marks |= __float_as_uint(m[w].x);
                }
                a.x = marked(a.x, marks);
                if (RS && !finite(a.y)) a.y = chain_again<false, Tl::CH>(maps.warp, maps.back, tid, 0.f, nullptr);
                s = through_cluster<Tl::CH, false, RS>(cta_maps, maps.received, a, tid, at.rank, S, at.ntiles - 1 - it,
                                                       state, in.wait_limit, bad);
            }
            const float s0 = s;
#pragma unroll
            for (int w = WARPS - 1; w >= 0; --w) {
                maps.carry_back[w][tid] = s;
                s = fmaf(m[w].x, s, bk[w]);
            }
            if (RS && !finite(s)) s = chain_again<false, Tl::CH>(maps.warp, maps.back, tid, s0, maps.carry_back);
            if (S == 1) state = s;
        }
        __syncthreads();
        V h = *reinterpret_cast<const V*>(&maps.carry[at.warp][at.lc * VEC]);
        V rr = *reinterpret_cast<const V*>(&maps.carry_back[at.warp][at.lc * VEC]);
        if (LPR < 32) {
            h = vote ? after(Pb, Hb, h) : vfma(Pb, h, Hb);
            rr = vote ? after(Pa, Qa, rr) : vfma(Pa, rr, Qa);
        }
        if (at.on) {
#pragma unroll
            for (int r = 0; r < R; ++r) {  // u becomes the state before each step
                const V before = h;
                h = vfma(c[r], before, u[r]);
                u[r] = before;
            }
            T* px = (T*)q.dx + at.b * q.dx_sb + t * q.dx_st + d;
            T* pg = (T*)q.dg_ + at.b * q.dg_sb + t * q.dg_st + d;
            T* po = OG ? (T*)q.do_ + at.b * q.do_sb + t * q.do_st + d : nullptr;
            if (whole) {
                backward_apply<true, T, VEC, LPR, OG, R>(rr, c, u, na, e, st, st + 2 * ARR, st + 3 * ARR, px, q.dx_st, pg,
                                                      q.dg_st, po, q.do_st, R, R, 0);
            } else {
                if (resets) {              // 0 at a reset, and what follows it from there on
                    bool started = false;
#pragma unroll
                    for (int r = 0; r < R; ++r) {
                        const bool reset = (resets >> r) & 1;
                        if (reset) u[r] = all<VEC>(0.f);
                        else if (started) u[r] = h;
                        started |= reset;
                        h = vfma(c[r], u[r], vmul(na[r], widen(st[r * LPR])));
                    }
                }
                backward_apply<false, T, VEC, LPR, OG, R>(rr, c, u, na, e, st, st + 2 * ARR, st + 3 * ARR, px, q.dx_st, pg,
                                                       q.dg_st, po, q.do_st, len - t, in.T - t, resets);
            }
        }
    }
    dg::let_next_start();
    if (q.dh0 && at.rank == 0 && carries) q.dh0[(int64_t)at.b * in.D + at.d0 + tid] = state;
    close_exchange(S, bad, in.status);
}

// grid: channels x rows, the rows walked where there are more than a grid has
template <typename T>
__global__ void scan_step_kernel(int B, int D, const T* x, int64_t x_sb, const T* g, int64_t g_sb, const T* o, int64_t o_sb,
                                 float* h, T* y) {
    const int d = blockIdx.x * blockDim.x + threadIdx.x;
    dg::let_next_start();
    dg::wait_for_previous();
    if (d >= D) return;
    for (int64_t b = blockIdx.y; b < B; b += gridDim.y) {
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
}

// ---------------------------------------------------------------------------
// launches
// ---------------------------------------------------------------------------

// How rows can be read and written: 0 one element at a time, 1 two, 2 two with inputs read
// 16 bytes at a time
struct Row {
    const void* p;
    int64_t sb, st;
};
int width_of(int D, size_t elem, std::initializer_list<Row> rows) {
    int64_t units = D;                     // every start and stride in elements, as one set of bits
    uintptr_t bytes = 0;
    for (const Row& r : rows)
        if (r.p) {
            bytes |= reinterpret_cast<uintptr_t>(r.p);
            units |= r.sb | r.st;
        }
    if (units % 2 || bytes % (2 * elem)) return 0;
    return units % (int64_t)(16 / elem) || bytes % 16 ? 1 : 2;
}

// Channels per CTA (lpr x vec) and cluster size, by the work of the busiest SM: CTAs on it x walked steps x
// channels, 1100 more for each tile walked and 24000 for each wave of CTAs.  Clusters fill some SMs before
// others, so their SMs count as full, and 0.3 of a wave more is counted where there are several; an SM with a
// single CTA waits at its barriers (1.6 x its work).  Rows of 32 and 64 bytes cost HBM 38% and 15% more than
// rows of 128.  Fitted to 48 shapes, whose choice takes 1% longer than the best on average and 13% at worst.
// Forward: 2 x 300 x 512 lpr 32 cluster 5 3.4 us, none 7.5; 8 x 4096 x 768 cluster 4 50 us, 2 70, lpr 8 66;
// 32 x 2048 x 1024 cluster 2 109 us, none 114, lpr 8 146.
struct Shape {
    int lpr, cluster;
};
Shape shape_of(int B, int T, int D, int vec, int steps_per_thread, int occ, bool narrow) {
    Shape best{32, 1};
    double least = -1.0;
    for (int lpr = 32; lpr >= 8; lpr /= 2) {
        if (lpr == 16 && !narrow) continue;
        const int64_t units = (int64_t)B * ((D + lpr * vec - 1) / (lpr * vec));
        const int steps = THREADS / lpr * steps_per_thread, tiles = (T + steps - 1) / steps;
        for (int s = 1; s <= 16 && (s == 1 || s <= tiles); ++s) {
            const int64_t slots = dg_host::kClusters[occ - 1][s - 1], n = units * s, per_sm = (n + 147) / 148;
            const double waves = units <= slots ? 1.0 : (double)units / slots + 0.3;
            const double share = waves > 1.0 || (s > 1 && n > 148) ? waves * occ : per_sm > 1 ? (double)per_sm : 1.6;
            const double walked = (double)((tiles + s - 1) / s);
            const double cost = share * walked * steps * lpr * vec * (lpr == 8 ? 1.38 : lpr == 16 ? 1.15 : 1.0) +
                                waves * (1100.0 * walked + 24000.0);
            if (least < 0 || cost < least) {
                least = cost;
                best = {lpr, s};
            }
        }
    }
    return best;
}

template <typename T, int VEC, int LPR, bool WIDE, bool OG, bool RS>
int run_forward(const ScanIn& in, const float* h0, void* y, float* h_last, float* marks, cudaStream_t s) {
    typedef Tile<T, VEC, LPR, kForwardSteps, OG ? 3 : 2> Tl;
    const int64_t grid = (int64_t)in.B * ((in.D + Tl::CH - 1) / Tl::CH) * in.cluster;
    if (grid > 0x7fffffff) return DG_ERR_UNSUPPORTED;
    return dg_host::launch_lm(scan_forward_kernel<T, VEC, LPR, WIDE, OG, RS>, dim3((unsigned)grid), dim3(THREADS),
                              Tl::bytes(in.cluster), Tl::bytes(16), in.cluster, s, in, h0, (T*)y, h_last, marks);
}
template <typename T, int VEC, int LPR, bool WIDE, bool OG, bool RS>
int run_backward(const ScanIn& in, const ScanGrad& q, cudaStream_t s) {
    typedef Tile<T, VEC, LPR, kBackwardSteps, OG ? 4 : 3> Tl;
    const int64_t grid = (int64_t)in.B * ((in.D + Tl::CH - 1) / Tl::CH) * in.cluster;
    if (grid > 0x7fffffff) return DG_ERR_UNSUPPORTED;
    return dg_host::launch_lm(scan_backward_kernel<T, VEC, LPR, WIDE, OG, RS>, dim3((unsigned)grid), dim3(THREADS),
                              Tl::bytes(in.cluster), Tl::bytes(16), in.cluster, s, in, q);
}

// calls F<T, VEC, LPR, WIDE, OG, RS>(...) for the shape at hand
#define SCAN_RS(F, T, VEC, LPR, WIDE, OG, rs, ...) \
    ((rs) ? F<T, VEC, LPR, WIDE, OG, true>(__VA_ARGS__) : F<T, VEC, LPR, WIDE, OG, false>(__VA_ARGS__))
#define SCAN_OG(F, T, VEC, LPR, WIDE, og, rs, ...)                   \
    ((og) ? SCAN_RS(F, T, VEC, LPR, WIDE, true, rs, __VA_ARGS__)     \
          : SCAN_RS(F, T, VEC, LPR, WIDE, false, rs, __VA_ARGS__))
#define SCAN_RUN(F, T, width, lpr, og, rs, ...)                                  \
    ((width) == 2   ? (lpr) == 32   ? SCAN_OG(F, T, 2, 32, true, og, rs, __VA_ARGS__)  \
                      : (lpr) == 16 ? SCAN_OG(F, T, 2, 16, true, og, rs, __VA_ARGS__)  \
                                    : SCAN_OG(F, T, 2, 8, true, og, rs, __VA_ARGS__)   \
     : (width) == 1 ? (lpr) == 32 ? SCAN_OG(F, T, 2, 32, false, og, rs, __VA_ARGS__)   \
                                  : SCAN_OG(F, T, 2, 8, false, og, rs, __VA_ARGS__)    \
     : (lpr) == 32  ? SCAN_OG(F, T, 1, 32, false, og, rs, __VA_ARGS__)                 \
                    : SCAN_OG(F, T, 1, 8, false, og, rs, __VA_ARGS__))

// CTAs that share an SM, by shared memory and registers
constexpr int occupancy(bool backward, size_t elem) { return elem == 4 ? 2 : 3; }

}  // namespace

extern "C" {

int dg_gated_scan_forward(int dtype, int B, int T, int D, const void* x, int64_t x_sb, int64_t x_st,
                          const void* gate, int64_t gate_sb, int64_t gate_st, const void* out_gate,
                          int64_t out_gate_sb, int64_t out_gate_st, const float* h0, const int32_t* lengths,
                          const uint8_t* resets, void* y, float* h_last, float* marks, int32_t* dev_status,
                          void* stream) {
    if (dtype == DG_DTYPE_F64) return DG_ERR_UNSUPPORTED;
    if (dtype < DG_DTYPE_F32 || dtype > DG_DTYPE_BF16 || B < 0 || T < 0 || D < 0) return DG_ERR_INVALID_ARGUMENT;
    if (B == 0 || D == 0) return DG_OK;
    if (T > 0 && (!x || !gate || !y)) return DG_ERR_INVALID_ARGUMENT;
    if (T == 0 && !h_last) return DG_OK;
    if (T > (1 << 30)) return DG_ERR_UNSUPPORTED;
    const size_t elem = dg_host::dtype_size(dtype);
    const int width = width_of(D, elem, {{x, x_sb, x_st}, {gate, gate_sb, gate_st}, {out_gate, out_gate_sb, out_gate_st},
                                         {y, 0, 0}});
    const Shape sh = shape_of(B, T, D, width ? 2 : 1, kForwardSteps, occupancy(false, elem), width == 2);
    const ScanIn in{x, gate, out_gate, x_sb, x_st, gate_sb, gate_st, out_gate_sb, out_gate_st, lengths, resets, B, T, D,
                    sh.cluster, dev_status, dg_host::wait_limit()};
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    DG_DISPATCH_LM(dtype, S, {
        return SCAN_RUN(run_forward, S, width, sh.lpr, out_gate != nullptr, resets != nullptr, in, h0, y, h_last, marks,
                        s);
    });
    return DG_OK;
}

int dg_gated_scan_backward(int dtype, int B, int T, int D, const void* x, int64_t x_sb, int64_t x_st,
                           const void* gate, int64_t gate_sb, int64_t gate_st, const void* out_gate,
                           int64_t out_gate_sb, int64_t out_gate_st, const int32_t* lengths, const uint8_t* resets,
                           const float* marks, const void* dy, int64_t dy_sb, int64_t dy_st, const float* dh_last,
                           void* dx, int64_t dx_sb, int64_t dx_st, void* dgate, int64_t dgate_sb, int64_t dgate_st,
                           void* dout_gate, int64_t dout_gate_sb, int64_t dout_gate_st, float* dh0,
                           int32_t* dev_status, void* stream) {
    if (dtype == DG_DTYPE_F64) return DG_ERR_UNSUPPORTED;
    if (dtype < DG_DTYPE_F32 || dtype > DG_DTYPE_BF16 || B < 0 || T < 0 || D < 0) return DG_ERR_INVALID_ARGUMENT;
    if ((out_gate == nullptr) != (dout_gate == nullptr)) return DG_ERR_INVALID_ARGUMENT;
    if (B == 0 || D == 0) return DG_OK;
    if (T > 0 && (!x || !gate || !marks || !dy || !dx || !dgate)) return DG_ERR_INVALID_ARGUMENT;
    if (T == 0 && !dh0) return DG_OK;
    if (T > (1 << 30)) return DG_ERR_UNSUPPORTED;
    const size_t elem = dg_host::dtype_size(dtype);
    const int width = width_of(D, elem, {{x, x_sb, x_st}, {gate, gate_sb, gate_st}, {out_gate, out_gate_sb, out_gate_st},
                                         {dy, dy_sb, dy_st}, {dx, dx_sb, dx_st}, {dgate, dgate_sb, dgate_st},
                                         {dout_gate, dout_gate_sb, dout_gate_st}});
    const Shape sh = shape_of(B, T, D, width ? 2 : 1, kBackwardSteps, occupancy(true, elem), width == 2);
    const ScanIn in{x, gate, out_gate, x_sb, x_st, gate_sb, gate_st, out_gate_sb, out_gate_st, lengths, resets, B, T, D,
                    sh.cluster, dev_status, dg_host::wait_limit()};
    const ScanGrad q{marks, dy, dy_sb, dy_st, dh_last, dx, dgate, dout_gate, dx_sb, dx_st, dgate_sb, dgate_st,
                     dout_gate_sb, dout_gate_st, dh0};
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    DG_DISPATCH_LM(dtype, S, {
        return SCAN_RUN(run_backward, S, width, sh.lpr, out_gate != nullptr, resets != nullptr, in, q, s);
    });
    return DG_OK;
}

int dg_gated_scan_step(int dtype, int B, int D, const void* x, int64_t x_sb, const void* gate, int64_t gate_sb,
                       const void* out_gate, int64_t out_gate_sb, float* h, void* y, void* stream) {
    if (dtype == DG_DTYPE_F64) return DG_ERR_UNSUPPORTED;
    if (dtype < DG_DTYPE_F32 || dtype > DG_DTYPE_BF16 || B < 0 || D < 0) return DG_ERR_INVALID_ARGUMENT;
    if (B == 0 || D == 0) return DG_OK;
    if (!x || !gate || !h || !y) return DG_ERR_INVALID_ARGUMENT;
    DG_DISPATCH_LM(dtype, S, {
        return dg_host::launch_lm(scan_step_kernel<S>, dim3(D / 128 + (D % 128 != 0), B < 65535 ? B : 65535), dim3(128), 0, 0, 0,
                                  static_cast<cudaStream_t>(stream), B, D, static_cast<const S*>(x), x_sb,
                                  static_cast<const S*>(gate), gate_sb, static_cast<const S*>(out_gate), out_gate_sb, h,
                                  static_cast<S*>(y));
    });
    return DG_OK;
}

}  // extern "C"
