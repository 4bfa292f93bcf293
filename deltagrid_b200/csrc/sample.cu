// sample.cu -- draws one token per row from given uniform numbers, with temperature,
// top-k, top-p and min-p.
//
// Masses are integers: w = floor(2^40 exp((l - max) / T)), summed in 64 bits, so every sum
// is exact and no result depends on the order of a reduction.  The kept set is a prefix of
// the order (logit descending, index ascending).
//
// A row is read once, by one CTA or by a cluster of up to 16 that share its slices, and kept
// in shared memory as integer keys in the order of the values (16 bits for 16-bit logits).
//   1. top_k: the k-th largest of 1024 partial maxima is a bound that at least k tokens reach
//      and few more do.  They are collected in one CTA; up to 256 are ranked by comparing
//      each with all (512 threads share that), more are sorted.  Ranks and the mass before
//      each give the kept ones, the same comparison by index gives the token.  Only collected
//      tokens need an exponential.
//   2. Where that does not do (no top_k, a large one, many equal logits): counts in 255 bins of
//      the distance below the maximum.  For top_p they say nearly where the cut lies: counts
//      times the mass at a bin's middle.  Then only keys near the cut are counted again,
//      finer, with their exact masses, beside the exact mass of all above them; the few tokens
//      of the bin that holds the cut are ranked in one CTA.  Two walks over the keys in index
//      order draw the token.  Where a row has a cluster, what a cut leaves is copied together
//      first, in index order, for the steps after it.  Without a cut (no top_k, no top_p) only
//      the walks are needed.
//
// What bounds it: not the 64 KB of a bf16 row of 32000 (2.5 us for 256 rows) but the latency
// of the steps after it, some fifteen barriers of up to 512 threads; two CTAs share an SM.
// 256 x 32000 with top_k 50 takes 11 us (1.5 TB/s); one row of 131072 fp32 logits with top_p
// alone, in a cluster of 16, 20 us; 33 x 50001 with top_k 4000 and top_p, clusters of 4, 27 us.
#include <type_traits>

#include "lm_common.cuh"

namespace {

constexpr int ST = 512;                    // threads per CTA
constexpr int WARPS = ST / 32;
constexpr size_t MOST_SMEM = 180 * 1024;   // dynamic, of a cluster's CTA
constexpr int CAP = 1024;                  // tokens collected at most
constexpr int RANKED = 256;                // up to here ranked by comparing all, beyond sorted
typedef unsigned long long u64;

struct SampleParams {
    const void* logits;
    int64_t row_stride;
    int V, slice, cluster, room;           // room: tokens that can be copied together
    const float* u;
    const float *temperature, *top_p, *min_p;
    const int32_t* top_k;
    float temperature_v, top_p_v, min_p_v;
    int32_t top_k_v;
    int64_t* token;
    float* logprob;
};

// ---- keys ------------------------------------------------------------------------
// Unsigned, in the order of the values; NaN counts as -inf, -0 equals +0.  0 is no value's key: it
// marks places outside the row.
template <typename T> struct Key {         // 16-bit logits, two to a word
    typedef uint16_t type;
    static constexpr int BITS = 16;
    static constexpr bool BF16 = std::is_same<T, __nv_bfloat16>::value;
    // NaN -> -inf (the larger of the two that is a number), -0 -> +0
    __device__ static __forceinline__ uint32_t clean(uint32_t x) {
        if constexpr (BF16) {
            const uint32_t inf = 0xff80ff80u, zero = 0;
            __nv_bfloat162 v = __hmax2(*reinterpret_cast<const __nv_bfloat162*>(&x), *reinterpret_cast<const __nv_bfloat162*>(&inf));
            v = __hadd2(v, *reinterpret_cast<const __nv_bfloat162*>(&zero));
            return *reinterpret_cast<const uint32_t*>(&v);
        } else {
            const uint32_t inf = 0xfc00fc00u, zero = 0;
            __half2 v = __hmax2(*reinterpret_cast<const __half2*>(&x), *reinterpret_cast<const __half2*>(&inf));
            v = __hadd2(v, *reinterpret_cast<const __half2*>(&zero));
            return *reinterpret_cast<const uint32_t*>(&v);
        }
    }
    __device__ static __forceinline__ uint32_t larger(uint32_t a, uint32_t b) {        // of cleaned values
        if constexpr (BF16) {
            const __nv_bfloat162 v = __hmax2(*reinterpret_cast<const __nv_bfloat162*>(&a), *reinterpret_cast<const __nv_bfloat162*>(&b));
            return *reinterpret_cast<const uint32_t*>(&v);
        } else {
            const __half2 v = __hmax2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
            return *reinterpret_cast<const uint32_t*>(&v);
        }
    }
    __device__ static __forceinline__ uint32_t ordered(uint32_t x) {      // cleaned values -> keys
        uint32_t neg;                                                     // each half's sign in all its bits
        asm("prmt.b32 %0, %1, 0, 0xbb99;" : "=r"(neg) : "r"(x));
        return x ^ (neg | 0x80008000u);
    }
    static constexpr uint32_t NONE = BF16 ? 0xff80ff80u : 0xfc00fc00u;    // -inf
    __device__ static __forceinline__ uint32_t one(T l) { return ordered(clean(*reinterpret_cast<const uint16_t*>(&l))) & 0xffffu; }
    __device__ static __forceinline__ float value(uint32_t k) {
        const uint32_t b = (k ^ ((k & 0x8000u) ? 0x8000u : 0xffffu)) & 0xffffu;
        if (BF16) return __uint_as_float(b << 16);
        const uint16_t h = (uint16_t)b;
        return __half2float(*reinterpret_cast<const __half*>(&h));
    }
    // the larger key of a word
    __device__ static __forceinline__ uint32_t most(uint32_t w) { return max(w >> 16, w & 0xffffu); }
    __device__ static __forceinline__ uint32_t larger_key(uint32_t a, uint32_t b) {       // of both halves
        uint32_t r;
        asm("max.u16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
        return r;
    }
    // whether any key of the vector reaches bound (above 0)
    __device__ static __forceinline__ bool reaches(const uint4& v, uint32_t bound) {
        const uint32_t below = (bound - 1) * 0x10001u;
        const uint32_t m = larger_key(larger_key(v.x, v.y), larger_key(v.z, v.w));
        return larger_key(m, below) != below;
    }
    __device__ static __forceinline__ uint32_t near(float l) { return one(dg::from_f<T>(l)); }
};
template <> struct Key<float> {
    typedef uint32_t type;
    static constexpr int BITS = 32;
    static constexpr uint32_t NONE = 0xff800000u;
    __device__ static __forceinline__ uint32_t clean(uint32_t x) {
        return __float_as_uint(fmaxf(__uint_as_float(x), -INFINITY) + 0.f);
    }
    __device__ static __forceinline__ uint32_t larger(uint32_t a, uint32_t b) {
        return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b)));
    }
    __device__ static __forceinline__ uint32_t ordered(uint32_t b) { return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u); }
    __device__ static __forceinline__ uint32_t one(float l) { return ordered(clean(__float_as_uint(l))); }
    __device__ static __forceinline__ float value(uint32_t k) {
        return __uint_as_float(k ^ ((k >> 31) ? 0x80000000u : 0xffffffffu));
    }
    __device__ static __forceinline__ uint32_t most(uint32_t w) { return w; }
    __device__ static __forceinline__ bool reaches(const uint4& v, uint32_t bound) {
        return max(max(v.x, v.y), max(v.z, v.w)) >= bound;
    }
    __device__ static __forceinline__ uint32_t near(float l) { return one(l); }
};

// The masses of N tokens; the row's maximum m is above -inf.  Below -28 (2^40 e^-28 < 1) a mass is 0, as it
// is for -inf and for the undefined quotients of infinite operands.  (l - m) / T is rounded to 32 bits
// once: times an inverse that is exact (T a power of two), or times the 64-bit inverse, whose error of
// 2^-52 cannot move the rounding, as a quotient of 24-bit numbers stays 2^-49 away from every midpoint.
// Side by side and without branches, for the chain of one is long.
struct Mass {
    float m, inverse;                      // inverse: of a power of two, else 0
    double inverse64;
    __device__ __forceinline__ Mass(float m_, float T) : m(m_), inverse64(1.0 / (double)T) {
        inverse = (__float_as_uint(T) & 0x7fffffu) == 0 && T > 1e-18f && T < 1e18f ? 1.f / T : 0.f;
    }
    template <int N> __device__ __forceinline__ void of(const float (&l)[N], u64 (&w)[N]) const {
        float z[N];
        if (inverse != 0.f) {
#pragma unroll
            for (int i = 0; i < N; ++i) z[i] = (l[i] - m) * inverse;
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i) z[i] = (float)((double)(l[i] - m) * inverse64);
        }
#pragma unroll
        for (int i = 0; i < N; ++i) {
            // floor(2^40 e) from the bits of e = f 2^(E - 150), f of 24 bits, E <= 127
            const uint32_t b = __float_as_uint(expf(fmaxf(z[i], -28.f))), f = (b & 0x7fffffu) | 0x800000u;
            const u64 v = ((u64)f << 17) >> (127 - (b >> 23));
            w[i] = l[i] == m ? 1ull << 40 : z[i] > -28.f ? v : 0;
        }
    }
};
// floor (up = 0) or ceiling of n f / 2^24, f <= 2^24, n < 2^58
__device__ __forceinline__ u64 fraction_of(u64 f, u64 n, bool up) {
    return f * (n >> 24) + ((f * (n & 0xffffff) + (up ? 0xffffff : 0)) >> 24);
}

// ---- clusters ----------------------------------------------------------------------
__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ uint32_t remote(const void* p, uint32_t rank) {
    uint32_t a;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"((uint32_t)__cvta_generic_to_shared(p)), "r"(rank));
    return a;
}
__device__ __forceinline__ uint32_t remote_load32(const uint32_t* p, uint32_t rank) {
    uint32_t v;
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(remote(p, rank)));
    return v;
}
__device__ __forceinline__ void remote_store64(u64* p, uint32_t rank, u64 v) {
    asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(remote(p, rank)), "l"(v) : "memory");
}
__device__ __forceinline__ void remote_store128(void* p, uint32_t rank, uint4 v) {
    asm volatile("st.shared::cluster.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(remote(p, rank)), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}
__device__ __forceinline__ void remote_store32(uint32_t* p, uint32_t rank, uint32_t v) {
    asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(remote(p, rank)), "r"(v) : "memory");
}
__device__ __forceinline__ uint32_t remote_add(uint32_t* p, uint32_t rank, uint32_t v) {
    uint32_t o;
    asm volatile("atom.relaxed.cluster.shared::cluster.add.u32 %0, [%1], %2;" : "=r"(o) : "r"(remote(p, rank)), "r"(v) : "memory");
    return o;
}

struct alignas(16) Shared {
    u64 list[CAP];                         // collected tokens: key << 32 | ~index
    u64 masses[RANKED];                    // theirs
    uint32_t hist[4][256];                 // counts, and the masses' 13 + 13 + 14 bits
    u64 bin_mass[256];                     // what they amount to: every CTA's, this one's part of the bins
    uint32_t bin_count[256];
    u64 all_mass[256];                     // the cluster's
    uint32_t all_count[256], far_count[256];
    u64 warp[WARPS];
    u64 sent[4][16], extra[16];            // values from the cluster's CTAs
    u64 found[2];                          // where a cut lies; the piece that holds the draw
    u64 cross[2];                          // a crossing: its bin, and the running value before it
    uint32_t queue[CAP];                   // vectors that hold a token to collect
    uint32_t vectors, collected[3];
    uint32_t flag;
};

// a barrier of the CTA, or of its cluster
__device__ __forceinline__ void join(int cluster) {
    if (cluster == 1) {
        __syncthreads();
    } else {
        __syncwarp();
        asm volatile("barrier.cluster.arrive.release.aligned;\n barrier.cluster.wait.acquire.aligned;" ::: "memory");
    }
}

__device__ __forceinline__ u64 warp_sum(u64 v) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(DG_FULL_MASK, v, o);
    return v;
}
__device__ __forceinline__ u64 warp_scan(u64 v, int lane) {       // inclusive
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const u64 n = __shfl_up_sync(DG_FULL_MASK, v, o);
        if (lane >= o) v += n;
    }
    return v;
}
// sum over the CTA, in every thread
__device__ __forceinline__ u64 block_sum(u64 v, Shared& s) {
    v = warp_sum(v);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) s.warp[threadIdx.x >> 5] = v;
    __syncthreads();
    v = s.warp[threadIdx.x % WARPS];
#pragma unroll
    for (int o = WARPS / 2; o; o >>= 1) v += __shfl_xor_sync(DG_FULL_MASK, v, o);
    return v;
}
// barrier of the first `threads` threads (whole warps)
__device__ __forceinline__ void part_sync(int threads) {
    if (threads == 32) __syncwarp();
    else asm volatile("bar.sync 1, %0;" ::"r"(threads) : "memory");
}
// exclusive prefix sum over the first `threads` threads; *total in each of them
__device__ __forceinline__ u64 part_before(u64 v, u64* total, int threads, Shared& s) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const u64 inc = warp_scan(v, lane);
    if (threads == 32) {
        *total = __shfl_sync(DG_FULL_MASK, inc, 31);
        return inc - v;
    }
    part_sync(threads);
    if (lane == 31) s.warp[warp] = inc;
    part_sync(threads);
    u64 before = 0, t = 0;
    for (int i = 0; i < threads / 32; ++i) {
        if (i == warp) before = t;
        t += s.warp[i];
    }
    *total = t;
    return before + inc - v;
}
// exclusive prefix sum over the CTA's threads; *total in every thread
__device__ __forceinline__ u64 block_before(u64 v, u64* total, Shared& s) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const u64 inc = warp_scan(v, lane);
    __syncthreads();
    if (lane == 31) s.warp[warp] = inc;
    __syncthreads();
    const u64 all = warp_scan(lane < WARPS ? s.warp[lane] : 0, lane);
    *total = __shfl_sync(DG_FULL_MASK, all, 31);
    u64 before = __shfl_sync(DG_FULL_MASK, all, (warp - 1) & 31);
    if (warp == 0) before = 0;
    return before + inc - v;
}
// One value per CTA of the cluster, in lane r the value of CTA r (0 beyond).  Values are sent, not fetched: after
// the barrier they are here, and no CTA's memory is read from outside.  Each slot is used once.
__device__ __forceinline__ u64 over_cluster(u64 v, int slot, int cluster, int rank, Shared& s) {
    if (threadIdx.x < cluster) remote_store64(&s.sent[slot][rank], threadIdx.x, v);
    join(cluster);
    const int lane = threadIdx.x & 31;
    return lane < cluster ? s.sent[slot][lane] : 0;
}

// sorts list[0, n2) (n2 a power of two, 64 to 1024) by the first n2 / 2 threads, one exchange per thread
// and stage; exchanges inside 64 elements stay within a warp
__device__ __forceinline__ void sort_list(u64* list, int n2, bool descending) {
    const int t = threadIdx.x;
#pragma unroll 1
    for (int size = 2; size <= n2; size *= 2)
#pragma unroll 1
        for (int j = size / 2; j; j /= 2) {
            const int i = 2 * t - (t & (j - 1)), k = i + j;
            const u64 a = list[i], b = list[k];
            const bool down = ((i & size) == 0) == descending;
            if (down ? a < b : a > b) {
                list[i] = b;
                list[k] = a;
            }
            if (j > 32 || (j == 1 && size >= 64)) part_sync(n2 / 2);
            else __syncwarp();
        }
}

// MANY: a row has a CTA of its own and two share an SM; else a cluster's CTAs have an SM each, and twice the
// registers for independent chains.
template <typename T, bool MANY>
__global__ void __launch_bounds__(ST, MANY ? 2 : 1) sample_kernel(SampleParams p) {
    constexpr int GROUP = MANY ? 4 : 8;
    typedef Key<T> K;
    typedef typename K::type key_t;
    constexpr int E = 16 / sizeof(T);
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ Shared s;
    uint4* vecs = reinterpret_cast<uint4*>(smem);
    key_t* keys = reinterpret_cast<key_t*>(smem);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int C = p.cluster, rank = C > 1 ? (int)cluster_rank() : 0, row = blockIdx.x / C;
    const int V = p.V, s0 = min(rank * p.slice, V), n = min(p.slice, V - s0);
    const T* src = static_cast<const T*>(p.logits) + (int64_t)row * p.row_stride + s0;

    if (C > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");       // (waited for before the first sending)
    dg::let_next_start();
    dg::wait_for_previous();
    // ---- parameters
    const float temp = p.temperature ? p.temperature[row] : p.temperature_v;
    int k = p.top_k ? p.top_k[row] : p.top_k_v;
    const float top_p = p.top_p ? p.top_p[row] : p.top_p_v, min_p = p.min_p ? p.min_p[row] : p.min_p_v, u = p.u[row];

    // ---- the slice as keys: element i at keys[off + i], whole 16-byte vectors of the row on whole
    // vectors of the table, zeros around the slice
    const int head = min((int)((16 - (reinterpret_cast<uintptr_t>(src) & 15)) & 15) / (int)sizeof(T), n);
    const int off = (E - head % E) % E, nv = (off + n + E - 1) / E, body = (n - head) / E, v0 = (off + head) / E;
    uint32_t top0 = K::NONE, top1 = K::NONE;       // largest values of this thread's even and odd vectors
    if (tid < 4 * 256) (&s.hist[0][0])[tid] = (&s.hist[0][0])[tid + ST] = 0;
    if (tid == 0) s.vectors = s.collected[0] = s.collected[1] = s.collected[2] = 0;
    if (tid < off) keys[tid] = 0;
    if (tid < nv * E - off - n) keys[off + n + tid] = 0;
    uint32_t most0 = 0, most1 = 0;
    if (tid < head) {
        most0 = K::one(src[tid]);
        keys[off + tid] = (key_t)most0;
    }
    if (tid < n - head - body * E) {
        most1 = K::one(src[head + body * E + tid]);
        keys[off + head + body * E + tid] = (key_t)most1;
    }
    const uint4* vsrc = reinterpret_cast<const uint4*>(src + head);
#pragma unroll 1
    for (int i = tid; i < body; i += 4 * ST) {
        uint4 v[4];
#pragma unroll
        for (int q = 0; q < 4; ++q)
            if (i + q * ST < body) v[q] = dg::ld16(vsrc + i + q * ST);
#pragma unroll
        for (int q = 0; q < 4; ++q)
            if (i + q * ST < body) {
                v[q] = make_uint4(K::clean(v[q].x), K::clean(v[q].y), K::clean(v[q].z), K::clean(v[q].w));
                const uint32_t t = K::larger(K::larger(v[q].x, v[q].y), K::larger(v[q].z, v[q].w));
                if (q & 1) top1 = K::larger(top1, t);
                else top0 = K::larger(top0, t);
                vecs[v0 + i + q * ST] =
                    make_uint4(K::ordered(v[q].x), K::ordered(v[q].y), K::ordered(v[q].z), K::ordered(v[q].w));
            }
    }
    if (tid < body) most0 = max(most0, K::most(K::ordered(top0)));
    if (tid + ST < body) most1 = max(most1, K::most(K::ordered(top1)));

    const bool greedy = !(temp > 0.f);
    const float tdiv = greedy ? 1.f : temp;
    if (k <= 0 || k > V) k = V;
    if (greedy) k = 1;
    const u64 P = (u64)(fminf(fmaxf(top_p, 0.f), 1.f) * 16777216.f);
    const u64 least = (u64)(fminf(fmaxf(min_p, 0.f), 1.f) * 1099511627776.f);
    const u64 U = (u64)(fminf(fmaxf(u, 0.f), 1.f - 1.f / 16777216.f) * 16777216.f);
    const bool cut_k = k < V, cut_p = P < (1u << 24);

    // ---- the row's maximum, and the bound
    const int j = (k + C - 1) / C;         // this CTA's share
    const bool collect = cut_k && j <= 512;
    uint32_t bound = 0;
    u64 mx = __reduce_max_sync(DG_FULL_MASK, max(most0, most1));
    if (lane == 0) s.warp[warp] = mx;
    __syncthreads();
    mx = __reduce_max_sync(DG_FULL_MASK, (uint32_t)s.warp[lane % WARPS]);
    if (collect) {
        // counts of the partial maxima by their keys' distance below the largest (bf16's resolution
        // for 32-bit keys); the bound is the first key of the bin in which the j-th lies
        constexpr int low = K::BITS - 16;
        auto bin_of = [&](uint32_t key) { return min(((uint32_t)mx - key) >> low, 255u); };
        if (most0) atomicAdd(&s.hist[0][bin_of(most0)], 1u);
        if (most1) atomicAdd(&s.hist[0][bin_of(most1)], 1u);
        __syncthreads();
        if (warp == 0) {
            uint32_t v[8], sum = 0;
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = s.hist[0][8 * lane + i], sum += v[i];
            uint32_t run = sum;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const uint32_t x = __shfl_up_sync(DG_FULL_MASK, run, o);
                if (lane >= o) run += x;
            }
            const unsigned hit = __ballot_sync(DG_FULL_MASK, run >= (uint32_t)j);
            if (lane == (hit ? __ffs(hit) - 1 : 31)) {
                run -= sum;
                uint32_t b = 8 * lane;
#pragma unroll
                for (int i = 0; i < 7; ++i)
                    if (run + v[i] < (uint32_t)j && b == 8 * lane + i) run += v[i], ++b;
                s.cross[0] = b;
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) s.hist[0][8 * lane + i] = 0;
        }
        __syncthreads();
        const uint32_t bin = (uint32_t)s.cross[0];
        if (bin < 255 && (uint64_t)mx >= ((uint64_t)(bin + 1) << low)) {
            bound = (uint32_t)mx - (((bin + 1) << low) - 1);
        } else {
            // further down: bit by bit, to the same resolution
            for (int bit = K::BITS - 1; bit >= low; --bit) {
                const uint32_t c = bound | (1u << bit);
                const int reach = __syncthreads_count(most0 >= c) + __syncthreads_count(most1 >= c);
                if (reach >= j) bound = c;
            }
        }
    }
    if (C > 1) {
        // j tokens of each CTA reach its bound, so C j reach the smallest
        __syncwarp();
        asm volatile("barrier.cluster.wait.aligned;" ::: "memory");        // all CTAs have started
        const u64 v = over_cluster(mx << 32 | (0xffffffffu - bound), 0, C, rank, s);
        mx = __reduce_max_sync(DG_FULL_MASK, (uint32_t)(v >> 32));
        bound = 0xffffffffu - __reduce_max_sync(DG_FULL_MASK, (uint32_t)v);
    }
    const float m = K::value((uint32_t)mx);
    if (m == -INFINITY) {                  // nothing can be drawn
        if (rank == 0 && tid == 0) {
            p.token[row] = -1;
            if (p.logprob) p.logprob[row] = -INFINITY;
        }
        return;
    }
    const Mass mass_of(m, tdiv);
    auto mass = [&](uint32_t key) {
        const float l[1] = {K::value(key)};
        u64 w[1];
        mass_of.of(l, w);
        return w[0];
    };
    // The tokens that the steps look at: the whole table or, once `dense`, those copied together behind it with
    // their masses
    u64* copied_mass = reinterpret_cast<u64*>(vecs + nv);
    uint32_t* copied_key = reinterpret_cast<uint32_t*>(copied_mass + p.room);
    uint32_t* copied_place = copied_key + p.room;
    bool dense = false;
    int count_of = nv * E;
    auto key_at = [&](int i) { return dense ? copied_key[i] : (uint32_t)keys[i]; };
    auto place_at = [&](int i) { return dense ? copied_place[i] : (uint32_t)i; };
    auto vector_keys = [&](const uint4& v, uint32_t* key) {
        const uint32_t x[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int e = 0; e < E; ++e) key[e] = E == 4 ? x[e & 3] : x[e / 2 & 3] >> 16 * (e & 1) & 0xffffu;
    };
    // f(key, mass or 0) for all of them, any order, GROUP of a thread at a time
    auto each = [&](bool with_mass, auto&& f) {
        if (dense) {
#pragma unroll 2
            for (int i = tid; i < count_of; i += ST) f(copied_key[i], with_mass ? copied_mass[i] : 0);
            return;
        }
        constexpr int VECS = GROUP >= E ? GROUP / E : 1, N = VECS * E;
#pragma unroll 1
        for (int i = tid; i < nv; i += VECS * ST) {
            uint32_t key[N];
#pragma unroll
            for (int q = 0; q < VECS; ++q)
                vector_keys(i + q * ST < nv ? vecs[i + q * ST] : make_uint4(0, 0, 0, 0), key + q * E);
            u64 w[N] = {};
            if (with_mass) {
                float l[N];
#pragma unroll
                for (int q = 0; q < N; ++q) l[q] = K::value(key[q]);
                mass_of.of(l, w);
            }
#pragma unroll
            for (int q = 0; q < N; ++q) f(key[q], w[q]);
        }
    };
    // copies the tokens whose keys reach `lo` together, in index order, where there is room for them: four
    // consecutive keys to a lane
    auto copy_together = [&](uint32_t lo) {
        if (MANY || p.room == 0 || dense) return;
        auto four = [&](int i, uint32_t (&key)[4]) {
            if constexpr (sizeof(key_t) == 4) {
                const uint4 v = *reinterpret_cast<const uint4*>(keys + i);
                key[0] = v.x, key[1] = v.y, key[2] = v.z, key[3] = v.w;
            } else {
                const uint2 v = *reinterpret_cast<const uint2*>(keys + i);
                key[0] = v.x & 0xffffu, key[1] = v.x >> 16, key[2] = v.y & 0xffffu, key[3] = v.y >> 16;
            }
        };
        const int piece = ((count_of + WARPS - 1) / WARPS + 3) / 4 * 4, a = min(warp * piece, count_of), b = min(a + piece, count_of);
        uint32_t c = 0;
#pragma unroll 2
        for (int i = a + 4 * lane; i < b; i += 128) {
            uint32_t key[4];
            four(i, key);
#pragma unroll
            for (int e = 0; e < 4; ++e) c += key[e] >= lo;
        }
        c = __reduce_add_sync(DG_FULL_MASK, c);
        u64 n;
        uint32_t at = (uint32_t)block_before(lane == 0 ? c : 0, &n, s);
        if (n > (u64)p.room) return;
        at = __shfl_sync(DG_FULL_MASK, at, 0);
#pragma unroll 2
        for (int base = a; base < b; base += 128) {
            const int i = base + 4 * lane;
            uint32_t key[4] = {0, 0, 0, 0}, to = at;
            if (i < b) four(i, key);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const unsigned is = __ballot_sync(DG_FULL_MASK, key[e] >= lo);
                to += __popc(is & ((1u << lane) - 1));
                at += __popc(is);
            }
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (key[e] >= lo) {
                    copied_key[to] = key[e];
                    copied_place[to++] = (uint32_t)(i + e);
                }
        }
        __syncthreads();
        dense = true;
        count_of = (int)n;
        // their masses, once for all the steps to come
#pragma unroll 1
        for (int i = tid; i < count_of; i += 4 * ST) {
            float l[4];
            u64 w[4];
#pragma unroll
            for (int q = 0; q < 4; ++q) l[q] = K::value(i + q * ST < count_of ? copied_key[i + q * ST] : 1);
            mass_of.of(l, w);
#pragma unroll
            for (int q = 0; q < 4; ++q)
                if (i + q * ST < count_of) copied_mass[i + q * ST] = w[q];
        }
        __syncthreads();
    };

    // ---- collect the tokens that reach `bound`, and draw from them: thread t of the CTA that holds the
    // list.  total_k: what top_p takes its share of, or 0 where that is the mass of the first k of them.
    // Returns whether they were few enough, and enough; uniform over the cluster.
    auto push = [&](int counter, uint32_t key, uint32_t place) {
        const uint32_t at = C > 1 ? remote_add(&s.collected[counter], 0, 1) : atomicAdd(&s.collected[counter], 1u);
        if (at < CAP) {
            const u64 entry = (u64)key << 32 | (0xffffffffu - (uint32_t)(s0 + (int)place - off));
            if (C > 1) remote_store64(&s.list[at], 0, entry);
            else s.list[at] = entry;
        }
    };
    auto collect_and_draw = [&](uint32_t bound, u64 total_k) {
        // the vectors with such a token first, then one thread for each of their elements
#pragma unroll 2
        for (int i = tid; i < nv; i += ST)
            if (K::reaches(vecs[i], bound)) {
                const uint32_t at = atomicAdd(&s.vectors, 1u);
                if (at < CAP) s.queue[at] = (uint32_t)i;
            }
        __syncthreads();
        const uint32_t nq = s.vectors;
        if (nq > CAP) {
            if (tid == 0) {                // more tokens than vectors
                if (C > 1) remote_add(&s.collected[0], 0, nq);
                else s.collected[0] = nq;
            }
        } else {
            for (uint32_t i = tid; i < nq * E; i += ST) {
                const uint32_t place = s.queue[i / E] * E + i % E, key = keys[place];
                if (key >= bound) push(0, key, place);
            }
        }
        join(C);
        const int nc = (int)(C > 1 ? remote_load32(&s.collected[0], 0) : s.collected[0]);
        if (nc > CAP) return false;
        if (rank == 0) {
            auto answer = [&](u64 entry, u64 w, u64 total) {
                p.token[row] = (int64_t)(0xffffffffu - (uint32_t)entry);
                if (p.logprob) p.logprob[row] = logf(__fdiv_rn((float)w, (float)total));
            };
            auto say = [&](bool enough) {  // rank 0's verdict, to all
                if (C == 1) s.flag = enough;
                else if (tid < C) remote_store32(&s.flag, tid, enough);
            };
            const int lim = min(nc, k);
            if (nc <= RANKED) {
                // `part` threads share a token; each compares it with every part-th of the list
                int part = 2;
                while (part < 32 && part * 2 * nc <= ST) part *= 2;
                const int c = tid / part, q = tid % part;
                const u64 mine = c < nc ? s.list[c] : 0;
                const u64 w = c < nc ? mass((uint32_t)(mine >> 32)) : 0;
                if (q == 0 && c < nc) s.masses[c] = w;
                __syncthreads();
                uint32_t rank_ = 0;
                u64 before = 0, sum = 0;
#pragma unroll 4
                for (int i = q; i < nc; i += part) {
                    const u64 e = s.list[i], we = s.masses[i];
                    if (e > mine) ++rank_, before += we;
                }
                for (int o = 1; o < part; o <<= 1) {
                    rank_ += __shfl_xor_sync(DG_FULL_MASK, rank_, o);
                    before += __shfl_xor_sync(DG_FULL_MASK, before, o);
                }
                const bool in_k = c < nc && rank_ < (uint32_t)lim;
                const u64 k_mass = block_sum(in_k && q == 0 ? w : 0, s);     // (masses[] have been read)
                if (total_k == 0) total_k = k_mass;
                const u64 tau = max(fraction_of(P, total_k, true), 1ull);
                const bool enough = k_mass >= tau;
                say(enough);
                const bool keep = in_k && before < tau && w >= least;
                if (q == 0 && c < nc && !keep) s.masses[c] = 0;
                sum = block_sum(keep && q == 0 ? w : 0, s);      // its barriers also order masses[]
                u64 run = 0;               // kept mass of smaller indexes: larger complements
#pragma unroll 4
                for (int i = q; i < nc; i += part)
                    if ((uint32_t)s.list[i] > (uint32_t)mine) run += s.masses[i];
                for (int o = 1; o < part; o <<= 1) run += __shfl_xor_sync(DG_FULL_MASK, run, o);
                const u64 at = fraction_of(U, sum, false);
                if (enough && keep && q == 0 && run <= at && at < run + w) answer(mine, w, sum);
            } else {
                int n2 = 2 * RANKED;
                while (n2 < nc) n2 *= 2;
                if (tid < n2 / 2) {
                    // the first n2 / 2 threads: elements 2t and 2t + 1 of the order
                    const int i0 = 2 * tid;
                    if (i0 >= nc) s.list[i0] = 0;
                    if (i0 + 1 >= nc) s.list[i0 + 1] = 0;
                    part_sync(n2 / 2);
                    sort_list(s.list, n2, true);
                    const u64 e0 = s.list[i0], e1 = s.list[i0 + 1];
                    u64 w0 = i0 < lim ? mass((uint32_t)(e0 >> 32)) : 0, w1 = i0 + 1 < lim ? mass((uint32_t)(e1 >> 32)) : 0;
                    u64 sum;
                    const u64 before = part_before(w0 + w1, &sum, n2 / 2, s);
                    const u64 tau = max(fraction_of(P, total_k ? total_k : sum, true), 1ull);
                    const bool enough = sum >= tau;
                    say(enough);
                    // the kept ones by index, the others behind them
                    if (before + w0 >= tau || w1 < least) w1 = 0;
                    if (before >= tau || w0 < least) w0 = 0;
                    s.list[i0] = w0 ? (u64)(0xffffffffu - (uint32_t)e0) << 32 | e0 >> 32 : ~0ull;
                    s.list[i0 + 1] = w1 ? (u64)(0xffffffffu - (uint32_t)e1) << 32 | e1 >> 32 : ~0ull;
                    part_sync(n2 / 2);
                    sort_list(s.list, n2, false);
                    const u64 d0 = s.list[i0], d1 = s.list[i0 + 1];
                    w0 = ~d0 ? mass((uint32_t)d0) : 0;
                    w1 = ~d1 ? mass((uint32_t)d1) : 0;
                    u64 total;
                    const u64 run = part_before(w0 + w1, &total, n2 / 2, s), at = fraction_of(U, total, false);
                    if (enough && run <= at && at < run + w0 + w1) {
                        const bool second = at >= run + w0;
                        answer(0xffffffffu - ((second ? d1 : d0) >> 32), second ? w1 : w0, total);
                    }
                }
            }
        }
        join(C);                           // rank 0's counter has been read, its verdict is there
        return s.flag != 0;
    };

    uint32_t cut = 0;                      // kept: key > cut, and the first `ties` with key == cut
    u64 ties = 0;
    if (cut_k || cut_p) {
        // ---- the cut by counting.  Tokens 28 T or more below the maximum have no mass: they cannot be drawn,
        // so a cut among them is as good as none, and they are left out.
        const float span = fminf(28.f * tdiv, 3.0e38f), scale = 255.f / span;
        auto far = [&](uint32_t key) {     // bins of the distance below the maximum; monotone in the key
            const float dist = (m - K::value(key)) * scale;
            return dist < 255.f ? (int)dist : dist == dist ? 255 : 0;
        };
        // s.hist, counted by each CTA, becomes s.all_* over the cluster: each CTA gets all counts of its part of
        // the bins, adds them up and sends the sums to all, 16 bytes at a time.  Returns the sum of `extra`.
        auto bin_masses = [&](int b) {
            const u64 w = (u64)s.hist[1][b] + ((u64)s.hist[2][b] << 13) + ((u64)s.hist[3][b] << 26);
            s.hist[1][b] = s.hist[2][b] = s.hist[3][b] = 0;
            return w;
        };
        auto gather = [&](bool by_mass, u64 extra) {
            __syncthreads();
            if (C == 1) {
                if (tid < 256) {
                    s.all_count[tid] = s.hist[0][tid];
                    s.hist[0][tid] = 0;
                    if (by_mass) s.all_mass[tid] = bin_masses(tid);
                }
                __syncthreads();
                return extra;
            }
            const int part = 256 / C;
            const int b4 = 4 * tid, b2 = 2 * (tid - 64);
            const bool counts = tid < 64, masses = by_mass && tid >= 64 && tid < 192;
            if (counts) {
                uint4* at = reinterpret_cast<uint4*>(&s.hist[0][b4]);
                remote_store128(&s.bin_count[rank * part + (b4 & (part - 1))], b4 / part, *at);
                *at = make_uint4(0, 0, 0, 0);
            } else if (masses) {
                const u64 w0 = bin_masses(b2), w1 = bin_masses(b2 + 1);
                remote_store128(&s.bin_mass[rank * part + (b2 & (part - 1))], b2 / part,
                                make_uint4((uint32_t)w0, (uint32_t)(w0 >> 32), (uint32_t)w1, (uint32_t)(w1 >> 32)));
            } else if (tid >= 192 && tid - 192 < C) {
                remote_store64(&s.extra[rank], tid - 192, extra);
            }
            join(C);
            extra = warp_sum(lane < C ? s.extra[lane] : 0);
            if (counts) {
                uint4 v = make_uint4(0, 0, 0, 0);
#pragma unroll 4
                for (int r = 0; r < C; ++r) {
                    const uint4 c = *reinterpret_cast<const uint4*>(&s.bin_count[r * part + (b4 & (part - 1))]);
                    v.x += c.x, v.y += c.y, v.z += c.z, v.w += c.w;
                }
                remote_store128(&s.all_count[rank * part + (b4 & (part - 1))], b4 / part, v);
            } else if (masses) {
                u64 w0 = 0, w1 = 0;
#pragma unroll 4
                for (int r = 0; r < C; ++r) {
                    const ulonglong2 w = *reinterpret_cast<const ulonglong2*>(&s.bin_mass[r * part + (b2 & (part - 1))]);
                    w0 += w.x, w1 += w.y;
                }
                remote_store128(&s.all_mass[rank * part + (b2 & (part - 1))], b2 / part,
                                make_uint4((uint32_t)w0, (uint32_t)(w0 >> 32), (uint32_t)w1, (uint32_t)(w1 >> 32)));
            }
            join(C);
            return extra;
        };
        // the bin in which the running count or mass (from `run0`) reaches the target, and the running value
        // before it; false where it does not.  One warp looks, lane l at bins 8 l to 8 l + 7, then eight lanes at
        // those of the one that holds it.
        auto crossing = [&](bool by_mass, u64 target, u64& run0, int& bin_out) {
            if (warp == 0) {
                u64 v = 0;
#pragma unroll
                for (int i = 0; i < 8; ++i) v += by_mass ? s.all_mass[8 * lane + i] : s.all_count[8 * lane + i];
                u64 run = warp_scan(v, lane) + run0;
                const unsigned hit = __ballot_sync(DG_FULL_MASK, run >= target);
                if (hit) {
                    const int h = __ffs(hit) - 1, b = 8 * h + (lane & 7);
                    run = __shfl_sync(DG_FULL_MASK, run - v, h);
                    v = by_mass ? s.all_mass[b] : s.all_count[b];
                    u64 to = v;
#pragma unroll
                    for (int o = 1; o < 8; o <<= 1) {
                        const u64 x = __shfl_up_sync(DG_FULL_MASK, to, o, 8);
                        if ((lane & 7) >= o) to += x;
                    }
                    const unsigned in = __ballot_sync(DG_FULL_MASK, run + to >= target);
                    if (lane == __ffs(in) - 1) s.cross[0] = (u64)b, s.cross[1] = run + to - v;
                } else if (lane == 0) {
                    s.cross[0] = ~0ull;
                }
            }
            __syncthreads();
            const u64 b = s.cross[0];
            if (b == ~0ull) return false;
            bin_out = (int)b;
            run0 = s.cross[1];
            return true;
        };
        // keys that surely hold bins [blo, bhi], rounding errors of m and the distance included
        auto lowest = [&](int b) {
            const float edge = (float)(b + 1) / scale, fuzz = 1e-6f * (edge + fabsf(m));
            const uint32_t a = K::near(m - edge - fuzz);
            return a <= 2 ? 1u : a - 2;
        };
        auto highest = [&](int b) {
            const float edge = (float)b / scale, fuzz = 1e-6f * (edge + fabsf(m));
            return b == 0 ? (uint32_t)mx : min((uint32_t)mx, K::near(m - edge + fuzz) + 2);
        };

        // The cut: the token at which the count or mass reaches the target, expected in bins [blo, bhi] with
        // `before_bins` tokens before them.  Leaves cut and ties, and returns false where the target is not in
        // those bins.
        int uses = 0;
        auto resolve = [&](bool by_mass, u64 target, int blo, int bhi, u64 before_bins) {
            uint32_t lo = lowest(bhi), hi = highest(blo);
            u64 run0 = before_bins;        // count or mass above the range
            for (int level = 0;; ++level) {
                int shift = 0, bin;
                while (((hi - lo) >> shift) > 255) ++shift;
                u64 above = 0;
                const uint32_t to = by_mass && level == 0 ? 0xffffffffu : hi;      // above the range: exact mass, once
                each(by_mass, [&](uint32_t key, u64 w) {
                    if (key < lo || key > to) return;
                    const int b = key > hi ? -1 : far(key);
                    if (b < blo) above += w;
                    if (b < blo || b > bhi) return;
                    const int at = (int)((hi - key) >> shift);
                    atomicAdd(&s.hist[0][at], 1u);
                    if (by_mass) {
                        atomicAdd(&s.hist[1][at], (uint32_t)w & 0x1fffu);
                        atomicAdd(&s.hist[2][at], (uint32_t)(w >> 13) & 0x1fffu);
                        atomicAdd(&s.hist[3][at], (uint32_t)(w >> 26));
                    }
                });
                if (by_mass && level == 0) above = block_sum(above, s);
                above = gather(by_mass, above);
                if (by_mass && level == 0) {
                    run0 = above;
                    if (run0 >= target) return false;
                }
                if (!crossing(by_mass, target, run0, bin)) return false;
                const uint32_t here = s.all_count[bin];
                const uint32_t top = hi - ((uint32_t)bin << shift), bottom = top - ((1u << shift) - 1);
                lo = bottom > lo && bottom <= top ? bottom : lo;
                hi = top;
                if (shift == 0 || lo == hi) {
                    // one key: as many of its tokens as the target asks for
                    const u64 w = mass(hi);
                    cut = hi;
                    ties = by_mass ? (target - run0 + w - 1) / w : target - run0;
                    if (ties == here) --cut, ties = 0;             // all of them: simply the keys above
                    return true;
                }
                if (here <= RANKED) break;
                __syncthreads();           // s.all_* have been read
            }
            // few tokens: ranked in one CTA
            const int counter = 1 + uses++;
            for (int i = tid; i < count_of; i += ST) {
                const uint32_t key = key_at(i);
                if (key < lo || key > hi) continue;
                const int b = far(key);
                if (b >= blo && b <= bhi) push(counter, key, place_at(i));
            }
            join(C);
            if (rank == 0) {
                const int nc = (int)s.collected[counter];
                const int c = tid >> 1, q = tid & 1;               // two threads to a token
                const u64 mine = c < nc ? s.list[c] : 0;
                const u64 w = c < nc ? mass((uint32_t)(mine >> 32)) : 0;
                if (q == 0 && c < nc) s.masses[c] = w;
                __syncthreads();
                uint32_t rank_ = 0, over = 0, same = 0;
                u64 before = 0;
#pragma unroll 4
                for (int i = q; i < nc; i += 2) {
                    const u64 e = s.list[i], we = s.masses[i];
                    if (e > mine) ++rank_, before += we;
                    over += e >> 32 > mine >> 32;
                    same += e >> 32 == mine >> 32;
                }
                rank_ += __shfl_xor_sync(DG_FULL_MASK, rank_, 1);
                over += __shfl_xor_sync(DG_FULL_MASK, over, 1);
                same += __shfl_xor_sync(DG_FULL_MASK, same, 1);
                before += __shfl_xor_sync(DG_FULL_MASK, before, 1);
                const bool it = by_mass ? run0 + before < target && run0 + before + w >= target
                                        : run0 + rank_ + 1 == target;
                if (c < nc && q == 0 && it) {
                    const uint32_t n = rank_ - over + 1;           // of its key, this many
                    const u64 where = (u64)((uint32_t)(mine >> 32) - (n == same)) << 32 | (n == same ? 0 : n);
                    if (C == 1) s.found[0] = where;
                    else
                        for (int r = 0; r < C; ++r) remote_store64(&s.found[0], r, where);
                }
            }
            join(C);
            const u64 answer = s.found[0];
            cut = (uint32_t)(answer >> 32);
            ties = answer & 0xffffffffu;
            return true;
        };

        // The steps, each of whose pieces stands here once: draw from collected tokens (`from`: the key they
        // reach, or 0), count, cut by top_k, cut by top_p in the bins near a guess, cut by top_p anywhere.
        uint32_t from = collect ? max(bound, 1u) : 0;
        u64 total_k = 0, tau = 0, c0 = 0;
        int blo = 0, bhi = 0;
        enum { COUNT, TOP_K, GUESS, TOP_P, ANYWHERE, DONE };
#pragma unroll 1
        for (int step = COUNT; step != DONE;) {
            if (from) {
                if (collect_and_draw(from, total_k)) return;
                from = 0;
            }
            if (step == COUNT) {
                // counts of all tokens, and the mass where top_k does not limit it
                u64 all = 0;
                each(!cut_k, [&](uint32_t key, u64 w) {
                    const int b = far(key);
                    if (key == 0 || b == 255) return;
                    atomicAdd(&s.hist[0][b], 1u);
                    all += w;
                });
                all = block_sum(all, s);
                total_k = gather(false, all);
                if (tid < 256) s.far_count[tid] = s.all_count[tid];
                step = cut_k ? TOP_K : GUESS;
                if (cut_k) {
                    if (!crossing(false, (u64)k, c0, blo)) step = GUESS;
                    bhi = blo;
                }
            }
            if (step == GUESS) {
                if (!cut_p) break;
                if (cut_k) {               // (the cut has not summed what lies above its bin)
                    u64 w = 0;
                    each(true, [&](uint32_t key, u64 v) { w += key > cut ? v : 0; });
                    w = block_sum(w, s);
                    if (C > 1) w = warp_sum(over_cluster(w, 1, C, rank, s));
                    total_k = w + (ties ? ties * mass(cut) : 0);
                }
                tau = max(fraction_of(P, total_k, true), 1ull);
                if (tau >= total_k) break;
                __syncthreads();
                // nearly where the mass reaches tau: counts times the mass at the middle of each bin
                if (warp == 0) {
                    float v[8], sum = 0.f;
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const int b = 8 * lane + i;
                        v[i] = b < 255 ? (float)s.far_count[b] * __expf(-((float)b + 0.5f) * (28.f / 255.f)) : 0.f;
                        sum += v[i];
                    }
                    float run = sum;
#pragma unroll
                    for (int o = 1; o < 32; o <<= 1) {
                        const float x = __shfl_up_sync(DG_FULL_MASK, run, o);
                        if (lane >= o) run += x;
                    }
                    const float want = (float)tau * (1.f / 1099511627776.f);
                    const unsigned hit = __ballot_sync(DG_FULL_MASK, run >= want);
                    if (lane == (hit ? __ffs(hit) - 1 : 31)) {
                        run -= sum;
                        int b = 8 * lane;
#pragma unroll
                        for (int i = 0; i < 7; ++i)
                            if (b == 8 * lane + i && run + v[i] < want) run += v[i], ++b;
                        s.cross[0] = (u64)min(b, 254);
                    }
                }
                __syncthreads();
                const int guess = (int)s.cross[0];
                blo = max(guess - 1, 0);
                bhi = min(guess + 1, 254);
                uint32_t upto = 0;
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    if (8 * lane + i <= bhi) upto += s.far_count[8 * lane + i];
                upto = __reduce_add_sync(DG_FULL_MASK, upto);
                step = TOP_P;
                if (!cut_k && upto > RANKED && bhi < 254) copy_together(lowest(bhi));
                // few tokens down to there: draw from them (a key below the bin's lowest does no harm)
                if (!cut_k && upto <= RANKED) {
                    from = lowest(bhi);
                    continue;
                }
            }
            const bool by_mass = step != TOP_K;
            const bool found = resolve(by_mass, by_mass ? tau : (u64)k, blo, bhi, c0);
            if (step == TOP_K) {
                step = GUESS;
                copy_together(ties ? cut : cut + 1);
            } else if (step == TOP_P && !found) {
                step = ANYWHERE;
                blo = 0, bhi = 254;
                if (!cut_k) dense = false, count_of = nv * E;
            } else {
                step = DONE;
            }
        }
    }

    // ---- the draw in index order: each warp walks a contiguous piece of the tokens
    const int piece = (count_of + WARPS - 1) / WARPS;
    // tokens with the cut key in [a, b), by one warp
    auto ties_in = [&](int a, int b) {
        uint32_t c = 0;
        for (int i = a + lane; i < b; i += 32) c += key_at(i) == cut;
        return __reduce_add_sync(DG_FULL_MASK, c);
    };
    // f(token, its mass or 0) over [a, b) in index order, a token to a lane, `seen` tokens with the cut key
    // before them
    auto walk = [&](auto group, int a, int b, uint32_t seen, auto&& f) {
        constexpr int N = decltype(group)::value;
#pragma unroll 1
        for (int base = a; base < b; base += 32 * N) {
            uint32_t key[N];
            u64 w[N];
#pragma unroll
            for (int q = 0; q < N; ++q) {
                const int i = base + 32 * q + lane;
                key[q] = i < b ? key_at(i) : 0;
                if (dense) w[q] = i < b ? copied_mass[i] : 0;
            }
            if (!dense) {
                float l[N];
#pragma unroll
                for (int q = 0; q < N; ++q) l[q] = K::value(key[q]);
                mass_of.of(l, w);
            }
#pragma unroll
            for (int q = 0; q < N; ++q) {
                bool in = key[q] > cut;
                if (ties) {
                    const unsigned is = __ballot_sync(DG_FULL_MASK, key[q] == cut);
                    in |= key[q] == cut && seen + __popc(is & ((1u << lane) - 1)) < ties;
                    seen += __popc(is);
                }
                f(base + 32 * q + lane, in && w[q] >= least ? w[q] : 0);
            }
        }
    };
    auto sum_of = [&](auto group, int a, int b, uint32_t seen) {
        u64 v = 0;
        walk(group, a, b, seen, [&](int, u64 w) { v += w; });
        return warp_sum(v);
    };
    int a0 = min(warp * piece, count_of), a1 = min(a0 + piece, count_of);
    uint32_t seen = 0;
    if (ties) {
        const uint32_t c = ties_in(a0, a1);
        u64 all;
        const u64 before = block_before(lane == 0 ? c : 0, &all, s);
        seen = (uint32_t)__shfl_sync(DG_FULL_MASK, before, 0);
        if (C > 1) {
            const u64 v = over_cluster(all, 2, C, rank, s);
            seen += __reduce_add_sync(DG_FULL_MASK, lane < rank ? (uint32_t)v : 0u);
        }
    }
    u64 mine = sum_of(std::integral_constant<int, GROUP>(), a0, a1, seen), total;
    u64 start = block_before(lane == 0 ? mine : 0, &total, s);
    start = __shfl_sync(DG_FULL_MASK, start, 0);
    u64 cta_start = 0;
    const u64 cta_mass = total;
    if (C > 1) {
        const u64 v = over_cluster(total, 3, C, rank, s);
        cta_start = warp_sum(lane < rank ? v : 0);
        total = warp_sum(v);
        start += cta_start;
    }
    const u64 at = fraction_of(U, total, false);
    if (at < cta_start || at >= cta_start + cta_mass) return;
    // the CTA whose keys hold the draw: all its warps share the piece that does
    if (lane == 0 && start <= at && at < start + mine) s.flag = (uint32_t)warp, s.found[0] = start, s.found[1] = seen;
    __syncthreads();
    const int base = min((int)s.flag * piece, count_of), last = min(base + piece, count_of), part = ((last - base + WARPS - 1) / WARPS + 31) / 32 * 32;
    start = s.found[0];
    seen = (uint32_t)s.found[1];
    a0 = min(base + warp * part, last), a1 = min(a0 + part, last);
    if (ties) {
        const uint32_t c = ties_in(a0, a1);
        u64 all;
        const u64 before = block_before(lane == 0 ? c : 0, &all, s);
        seen += (uint32_t)__shfl_sync(DG_FULL_MASK, before, 0);
    }
    const std::integral_constant<int, 1> one_each;             // few tokens to a warp now
    mine = sum_of(one_each, a0, a1, seen);
    u64 all;
    const u64 before = block_before(lane == 0 ? mine : 0, &all, s);
    start += __shfl_sync(DG_FULL_MASK, before, 0);
    if (start <= at && at < start + mine) {
        u64 run = start;
        walk(one_each, a0, a1, seen, [&](int i, u64 w) {
            const u64 inc = warp_scan(w, lane), r = run + inc - w;
            if (r <= at && at < r + w) {
                p.token[row] = (int64_t)s0 + (int)place_at(i) - off;
                if (p.logprob) p.logprob[row] = logf(__fdiv_rn((float)w, (float)total));
            }
            run += __shfl_sync(DG_FULL_MASK, inc, 31);
        });
    }
}

// CTAs per row: as many (up to 16) as give each SM one, with at least 2048 logits each; and as many as a
// slice of at most 84 KB (two CTAs to an SM) asks for.  A CTA's work beyond its logits is the same
// whatever it holds, so more CTAs than SMs cost more than they save.
int cluster_of(int B, int V, size_t elem) {
    int c = 1;
    while (c < 16 && ((int64_t)B * c * 2 <= 148 && V / (2 * c) >= 2048)) c *= 2;
    while (c < 16 && ((size_t)V + c - 1) / c * elem > 84 * 1024) c *= 2;
    return c;
}

template <typename T> int run(SampleParams p, int B, cudaStream_t stream) {
    p.cluster = cluster_of(B, p.V, sizeof(T));
    p.slice = ((p.V + p.cluster - 1) / p.cluster + 7) / 8 * 8;
    if ((int64_t)B * p.cluster > 0x7fffffff) return DG_ERR_UNSUPPORTED;
    // the table and, beside a cluster's slice, room for half of its tokens (16 bytes each) as far as it goes
    size_t smem = (size_t)(p.slice + 16) * sizeof(T) + 16;
    if (p.cluster > 1) {
        const size_t left = (MOST_SMEM - smem) / 16;
        p.room = (int)(left < (size_t)p.slice / 2 ? left : (size_t)p.slice / 2);
        smem += (size_t)p.room * 16;
    }
    auto kern = p.cluster == 1 ? sample_kernel<T, true> : sample_kernel<T, false>;
    return dg_host::launch_lm(kern, dim3((unsigned)(B * p.cluster)), dim3(ST), smem, MOST_SMEM, p.cluster > 1 ? p.cluster : 0, stream,
                              p);
}

}  // namespace

extern "C" int dg_sample(int dtype, int B, int V, const void* logits, int64_t row_stride, const float* u,
                         const float* temperature, float temperature_value, const int32_t* top_k, int32_t top_k_value,
                         const float* top_p, float top_p_value, const float* min_p, float min_p_value, int64_t* token,
                         float* logprob, void* stream) {
    if (dtype == DG_DTYPE_F64) return DG_ERR_UNSUPPORTED;
    if (dtype < DG_DTYPE_F32 || dtype > DG_DTYPE_BF16 || B < 0 || V <= 0) return DG_ERR_INVALID_ARGUMENT;
    if (B == 0) return DG_OK;
    if (!logits || !u || !token) return DG_ERR_INVALID_ARGUMENT;
    if (V > (1 << 18)) return DG_ERR_UNSUPPORTED;              // masses of 2^40 and their sums in 58 bits
    SampleParams p{logits, row_stride, V, 0, 1, 0, u, temperature, top_p, min_p, top_k, temperature_value, top_p_value,
                   min_p_value, top_k_value, token, logprob};
    DG_DISPATCH_LM(dtype, S, { return run<S>(p, B, static_cast<cudaStream_t>(stream)); });
    return DG_OK;
}
