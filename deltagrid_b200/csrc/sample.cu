// sample.cu -- draws one token per row from given uniform numbers, with temperature,
// top-k, top-p and min-p.
//
// Masses are integers: w = floor(2^40 exp((l - max) / T)), summed in 64 bits, so every sum
// is exact and no result depends on the order of a reduction.  The kept set is a prefix of
// the order (logit descending, index ascending).
//
// A row is read once, by one CTA or by a cluster of up to 16 that share its slices, and kept
// in shared memory as integer keys in the order of the values (16 bits for 16-bit logits).
//   1. The j-th largest of 1024 partial maxima is a bound that at least j tokens reach: with
//      j = top_k (or 256 where only top_p cuts) few more than j tokens do.  They are collected
//      in one CTA and sorted; prefix sums of their masses give the cut, a second sort brings
//      the kept ones into index order, and prefix sums again give the token.
//   2. Where more than 1024 tokens reach the bound, or the collected ones do not hold enough
//      mass, the cut key is found by counting: 256 bins over the distance below the maximum,
//      then 256 bins over the keys of the bin that holds the cut, until one key is left.  Then
//      two walks over the keys in index order draw the token.  Without a cut (no top_k, no
//      top_p) only the walks are needed.
// In the first way only collected tokens need an exponential, unless top_p alone cuts.
//
// What bounds it: reading the row once (64 KB of bf16 logits a row, two rows to an SM), then
// the latency of some forty barriers; the row's CTAs idle at neither, as two share an SM.
#include "lm_common.cuh"

namespace {

constexpr int ST = 512;                    // threads per CTA
constexpr int WARPS = ST / 32;
constexpr int CAP = 1024;                  // tokens collected and sorted
typedef unsigned long long u64;

struct SampleParams {
    const void* logits;
    int64_t row_stride;
    int V, slice, cluster;
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
    static constexpr int BITS = 16, PER = 2;
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
    // key `e` of a word, and the larger of its two
    __device__ static __forceinline__ uint32_t at(uint32_t w, int e) { return e ? w >> 16 : w & 0xffffu; }
    __device__ static __forceinline__ uint32_t most(uint32_t w) { return max(w >> 16, w & 0xffffu); }
    __device__ static __forceinline__ uint32_t near(float l) { return one(dg::from_f<T>(l)); }
};
template <> struct Key<float> {
    typedef uint32_t type;
    static constexpr int BITS = 32, PER = 1;
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
    __device__ static __forceinline__ uint32_t at(uint32_t w, int) { return w; }
    __device__ static __forceinline__ uint32_t most(uint32_t w) { return w; }
    __device__ static __forceinline__ uint32_t near(float l) { return one(l); }
};

// The mass of a token; the row's maximum m is above -inf.  Below -28 (2^40 e^-28 < 1) it is 0, as it
// is for -inf and for the undefined quotients of infinite operands.
__device__ __forceinline__ u64 mass_of(float l, float m, float T) {
    if (l == m) return 1ull << 40;
    const float z = __fdiv_rn(l - m, T);
    return z > -28.f ? (u64)__float2ll_rz(expf(z) * 1099511627776.f) : 0ull;
}
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
__device__ __forceinline__ u64 remote_load64(const u64* p, uint32_t rank) {
    u64 v;
    asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(remote(p, rank)) : "memory");
    return v;
}
__device__ __forceinline__ uint32_t remote_load32(const uint32_t* p, uint32_t rank) {
    uint32_t v;
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(remote(p, rank)) : "memory");
    return v;
}
__device__ __forceinline__ void remote_store64(u64* p, uint32_t rank, u64 v) {
    asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(remote(p, rank)), "l"(v) : "memory");
}
__device__ __forceinline__ uint32_t remote_add(uint32_t* p, uint32_t rank, uint32_t v) {
    uint32_t o;
    asm volatile("atom.relaxed.cluster.shared::cluster.add.u32 %0, [%1], %2;" : "=r"(o) : "r"(remote(p, rank)), "r"(v) : "memory");
    return o;
}

struct Shared {
    u64 list[CAP];                         // collected tokens: key << 32 | ~index, or index << 32 | key
    uint32_t hist[4][256];                 // counts, and the masses' 13 + 13 + 14 bits
    u64 bins[2][256];                      // what they amount to; this CTA's, read by the cluster
    u64 warp[WARPS], warp2[WARPS];
    u64 post[8];                           // values that the cluster's other CTAs read
    uint32_t collected;
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
    u64 t = 0;
#pragma unroll
    for (int i = 0; i < WARPS; ++i) t += s.warp[i];
    return t;
}
__device__ __forceinline__ void block_sum2(u64& a, u64& b, Shared& s) {
    a = warp_sum(a);
    b = warp_sum(b);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) s.warp[threadIdx.x >> 5] = a, s.warp2[threadIdx.x >> 5] = b;
    __syncthreads();
    a = b = 0;
#pragma unroll
    for (int i = 0; i < WARPS; ++i) a += s.warp[i], b += s.warp2[i];
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
    u64 before = 0, t = 0;
#pragma unroll
    for (int i = 0; i < WARPS; ++i) {
        if (i == warp) before = t;
        t += s.warp[i];
    }
    *total = t;
    return before + inc - v;
}
// sum, or largest or smallest, of one value per CTA over the cluster; slots of s.post alternate, so that
// a slot is written again only after a barrier that follows its last reading
template <typename F> __device__ __forceinline__ u64 over_cluster(u64 v, int slot, int cluster, Shared& s, F&& f) {
    if (cluster == 1) return v;
    if (threadIdx.x == 0) s.post[slot] = v;
    join(cluster);
    u64 r = remote_load64(&s.post[slot], 0);
    for (int k = 1; k < cluster; ++k) r = f(r, remote_load64(&s.post[slot], k));
    return r;
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

template <typename T>
__global__ void __launch_bounds__(ST, 2) sample_kernel(SampleParams p) {
    typedef Key<T> K;
    typedef typename K::type key_t;
    constexpr int E = 16 / sizeof(T);
    constexpr int W = K::PER;
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ Shared s;
    uint4* vecs = reinterpret_cast<uint4*>(smem);
    const uint32_t* words = reinterpret_cast<const uint32_t*>(smem);
    key_t* keys = reinterpret_cast<key_t*>(smem);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int C = p.cluster, rank = C > 1 ? (int)cluster_rank() : 0, row = blockIdx.x / C;
    const int V = p.V, s0 = min(rank * p.slice, V), n = min(p.slice, V - s0);
    const T* src = static_cast<const T*>(p.logits) + (int64_t)row * p.row_stride + s0;

    // ---- parameters
    const float temp = p.temperature ? p.temperature[row] : p.temperature_v;
    int k = p.top_k ? p.top_k[row] : p.top_k_v;
    const float top_p = p.top_p ? p.top_p[row] : p.top_p_v, min_p = p.min_p ? p.min_p[row] : p.min_p_v, u = p.u[row];

    // ---- the slice as keys: element i at keys[off + i], whole 16-byte vectors of the row on whole
    // vectors of the table, zeros around the slice
    const int head = min((int)((16 - (reinterpret_cast<uintptr_t>(src) & 15)) & 15) / (int)sizeof(T), n);
    const int off = (E - head % E) % E, nv = (off + n + E - 1) / E, body = (n - head) / E, v0 = (off + head) / E;
    const int nw = nv * 4;                 // words
    uint32_t top0 = K::NONE, top1 = K::NONE;       // largest values of this thread's even and odd vectors
    if (tid < 4 * 256) (&s.hist[0][0])[tid] = (&s.hist[0][0])[tid + ST] = 0;
    if (tid == 0) s.collected = 0;
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
    for (int i = tid; i < body; i += 8 * ST) {
        uint4 v[8];
#pragma unroll
        for (int q = 0; q < 8; ++q)
            if (i + q * ST < body) v[q] = dg::ldg16(vsrc + i + q * ST);
#pragma unroll
        for (int q = 0; q < 8; ++q)
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
    const int j_all = cut_k ? k : 256, j = (j_all + C - 1) / C;   // this CTA's share
    bool collect = (cut_k || cut_p) && j <= 512;
    uint32_t bound = 0;
    u64 mx = __reduce_max_sync(DG_FULL_MASK, max(most0, most1));
    if (lane == 0) s.warp[warp] = mx;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < WARPS; ++i) mx = max(mx, s.warp[i]);
    if (collect) {
        // counts of the partial maxima by their keys' distance below the largest (bf16's resolution
        // for 32-bit keys); the bound is the first key of the bin in which the j-th lies
        constexpr int low = K::BITS - 16;
        auto bin_of = [&](uint32_t key) { return min(((uint32_t)mx - key) >> low, 255u); };
        if (most0) atomicAdd(&s.hist[0][bin_of(most0)], 1u);
        if (most1) atomicAdd(&s.hist[0][bin_of(most1)], 1u);
        __syncthreads();
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
        run -= sum;
        uint32_t bin = 8 * lane;
#pragma unroll
        for (int i = 0; i < 7; ++i)
            if (run + v[i] < (uint32_t)j && bin == 8 * lane + i) run += v[i], ++bin;
        bin = __shfl_sync(DG_FULL_MASK, bin, hit ? __ffs(hit) - 1 : 31);
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
        __syncthreads();
        if (tid < 256) s.hist[0][tid] = 0;
    }
    if (C > 1) {
        // j tokens of each CTA reach its bound, so C j reach the smallest
        const u64 both = over_cluster(mx << 32 | (0xffffffffu - bound), 0, C, s, [](u64 a, u64 b) {
            return max(a >> 32, b >> 32) << 32 | max(a & 0xffffffffu, b & 0xffffffffu);
        });
        mx = both >> 32;
        bound = 0xffffffffu - (uint32_t)both;
    }
    const float m = K::value((uint32_t)mx);
    if (m == -INFINITY) {                  // nothing can be drawn
        if (rank == 0 && tid == 0) {
            p.token[row] = -1;
            if (p.logprob) p.logprob[row] = -INFINITY;
        }
        if (C > 1) join(C);                // the others may still read this CTA's slot
        return;
    }
    auto mass = [&](uint32_t key) { return mass_of(K::value(key), m, tdiv); };
    // f(key, place) for the keys of this CTA's words, any order
    auto each = [&](auto&& f) {
#pragma unroll 2
        for (int i = tid; i < nw; i += ST) {
            const uint32_t w = words[i];
#pragma unroll
            for (int e = 0; e < W; ++e) f(K::at(w, e), i * W + e);
        }
    };
    auto add = [](u64 a, u64 b) { return a + b; };

    // ---- the mass of the whole row, where top_k does not fix what top_p is a share of, and of what would
    // be collected: where that is too little, nothing is
    u64 total_k = 0;
    if (!cut_k && cut_p) {
        u64 w = 0, in = 0;
        each([&](uint32_t key, int) {
            const u64 v = key ? mass(key) : 0;
            w += v;
            if (key >= bound) in += v;
        });
        block_sum2(w, in, s);
        total_k = w;
        if (C > 1) {
            if (tid == 0) s.post[1] = w, s.post[2] = in;
            join(C);
            for (int r = 0; r < C; ++r)
                if (r != rank) total_k += remote_load64(&s.post[1], r), in += remote_load64(&s.post[2], r);
        }
        collect = collect && in >= fraction_of(P, total_k, true);
    }

    // ---- collect, sort and draw
    if (collect) {
        for (int i = tid; i < nv; i += ST) {
            const uint4 v = vecs[i];
            if (max(max(K::most(v.x), K::most(v.y)), max(K::most(v.z), K::most(v.w))) < bound) continue;
#pragma unroll 1
            for (int e = 0; e < E; ++e) {
                const uint32_t key = keys[i * E + e];
                if (key >= bound && key) {
                    const uint32_t at = C > 1 ? remote_add(&s.collected, 0, 1) : atomicAdd(&s.collected, 1u);
                    if (at < CAP) {
                        const u64 entry = (u64)key << 32 | (0xffffffffu - (uint32_t)(s0 + i * E + e - off));
                        if (C > 1) remote_store64(&s.list[at], 0, entry);
                        else s.list[at] = entry;
                    }
                }
            }
        }
        join(C);
        if (rank == 0) {
            const int nc = (int)min(s.collected, (uint32_t)CAP + 1);
            int n2 = 64;
            while (n2 < nc) n2 *= 2;
            if (nc <= CAP && tid < n2 / 2) {
                // the first n2 / 2 threads: elements 2t and 2t + 1 of the order
                const int i0 = 2 * tid, lim = min(nc, k);
                if (i0 >= nc) s.list[i0] = 0;
                if (i0 + 1 >= nc) s.list[i0 + 1] = 0;
                part_sync(n2 / 2);
                sort_list(s.list, n2, true);
                const u64 e0 = s.list[i0], e1 = s.list[i0 + 1];
                u64 w0 = i0 < lim ? mass((uint32_t)(e0 >> 32)) : 0, w1 = i0 + 1 < lim ? mass((uint32_t)(e1 >> 32)) : 0;
                u64 sum;
                const u64 before = part_before(w0 + w1, &sum, n2 / 2, s);
                const u64 tau = max(fraction_of(P, cut_k ? sum : total_k, true), 1ull);
                const bool done = cut_k || sum >= tau;
                if (done) {
                    const bool keep0 = i0 < lim && before < tau && w0 >= least;
                    const bool keep1 = i0 + 1 < lim && before + w0 < tau && w1 >= least;
                    u64 kept;              // the first `kept` of the order
                    part_before((u64)keep0 + keep1, &kept, n2 / 2, s);
                    s.list[i0] = keep0 ? (u64)(0xffffffffu - (uint32_t)e0) << 32 | e0 >> 32 : ~0ull;
                    s.list[i0 + 1] = keep1 ? (u64)(0xffffffffu - (uint32_t)e1) << 32 | e1 >> 32 : ~0ull;
                    part_sync(n2 / 2);
                    n2 = 64;
                    while (n2 < (int)kept) n2 *= 2;
                    if (tid < n2 / 2) {
                        sort_list(s.list, n2, false);
                        const u64 d0 = s.list[i0], d1 = s.list[i0 + 1];
                        w0 = i0 < (int)kept ? mass((uint32_t)d0) : 0;
                        w1 = i0 + 1 < (int)kept ? mass((uint32_t)d1) : 0;
                        u64 total;
                        const u64 run = part_before(w0 + w1, &total, n2 / 2, s), at = fraction_of(U, total, false);
                        if (run <= at && at < run + w0 + w1) {
                            const bool second = at >= run + w0;
                            p.token[row] = (int64_t)((second ? d1 : d0) >> 32);
                            if (p.logprob) p.logprob[row] = logf(__fdiv_rn((float)(second ? w1 : w0), (float)total));
                        }
                    }
                }
                if (tid == 0) s.flag = done;
            } else if (nc > CAP && tid == 0) {
                s.flag = 0;
            }
        }
        join(C);
        const bool done = C > 1 ? remote_load32(&s.flag, 0) != 0 : s.flag != 0;
        if (C > 1) join(C);
        if (done) return;
    }

    // ---- the cut by counting
    // the largest key K with measure(key >= K) >= target, and *above = measure(key > K).  The counters are
    // zero before and after a call.
    int buf = 0;
    auto find_cut = [&](bool by_mass, u64 target, u64* above_out) {
        u64 above = 0;
        uint32_t lo = 1, hi = (uint32_t)mx;
        const float scale = 255.f / fminf(28.f * tdiv, 3.0e38f);
        auto far = [&](uint32_t key) {     // bins of the distance below the maximum; monotone in the key
            const float dist = (m - K::value(key)) * scale;
            return dist < 255.f ? (int)dist : dist == dist ? 255 : 0;
        };
        int far_bin = -1, shift = 0;
        while (true) {
            each([&](uint32_t key, int) {
                if (key < lo || key > hi) return;
                int b;
                if (far_bin < 0) b = far(key);
                else if (far(key) != far_bin) return;
                else b = (int)((hi - key) >> shift);
                atomicAdd(&s.hist[0][b], 1u);
                if (by_mass) {
                    const u64 w = mass(key);
                    if (w) {
                        atomicAdd(&s.hist[1][b], (uint32_t)w & 0x1fffu);
                        atomicAdd(&s.hist[2][b], (uint32_t)(w >> 13) & 0x1fffu);
                        atomicAdd(&s.hist[3][b], (uint32_t)(w >> 26));
                    }
                }
            });
            __syncthreads();
            if (tid < 256) {
                s.bins[buf][tid] = by_mass ? (u64)s.hist[1][tid] + ((u64)s.hist[2][tid] << 13) + ((u64)s.hist[3][tid] << 26)
                                           : (u64)s.hist[0][tid];
#pragma unroll
                for (int q = 0; q < 4; ++q) s.hist[q][tid] = 0;
            }
            join(C);
            // every warp finds the bin for itself; lane l: bins 8 l to 8 l + 7
            u64 v[8], sum = 0;
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = C > 1 ? 0 : s.bins[buf][8 * lane + i];
            if (C > 1) {                   // the cluster's sums, a part of the bins to each warp
                const int b = tid >> 1;
                u64 x = 0;
                for (int r = tid & 1; r < C; r += 2) x += remote_load64(&s.bins[buf][b], r);
                x += __shfl_xor_sync(DG_FULL_MASK, x, 1);
                if (!(tid & 1)) s.list[b] = x;
                __syncthreads();
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i] = s.list[8 * lane + i];
            }
            buf ^= 1;
#pragma unroll
            for (int i = 0; i < 8; ++i) sum += v[i];
            const u64 inc = warp_scan(sum, lane) + above;
            const unsigned hit = __ballot_sync(DG_FULL_MASK, inc >= target);
            const int at = hit ? __ffs(hit) - 1 : 31;
            u64 run = inc - sum;
            int bin = 8 * lane;
#pragma unroll
            for (int i = 0; i < 7; ++i)
                if (run + v[i] < target && bin == 8 * lane + i) run += v[i], ++bin;
            bin = __shfl_sync(DG_FULL_MASK, bin, at);
            above = __shfl_sync(DG_FULL_MASK, run, at);
            if (far_bin < 0) {
                // keys that surely hold the bin's, rounding errors of m and the distance included; the
                // digits below only count those in it
                far_bin = bin;
                const float edge = (float)(bin + 1) / scale, fuzz = 1e-6f * (edge + fabsf(m));
                const uint32_t a = K::near(m - edge - fuzz), b = K::near(m - (float)bin / scale + fuzz);
                lo = bin == 255 || a <= 2 ? 1 : a - 2;
                hi = bin == 0 ? (uint32_t)mx : min((uint32_t)mx, b + 2);
            } else {
                const uint32_t top = hi - ((uint32_t)bin << shift), bottom = top - ((1u << shift) - 1);
                lo = bottom > lo && bottom <= top ? bottom : lo;
                hi = top;
            }
            if (lo >= hi) break;
            shift = 0;
            while (((hi - lo) >> shift) > 255) ++shift;
            if (C > 1) __syncthreads();    // list[] has been read
        }
        __syncthreads();
        *above_out = above;
        return hi;
    };
    auto mass_above = [&](uint32_t key, int slot) {
        u64 w = 0;
        each([&](uint32_t kk, int) { if (kk > key) w += mass(kk); });
        return over_cluster(block_sum(w, s), slot, C, s, add);
    };
    uint32_t cut = 0;                      // kept: key > cut, and the first `ties` with key == cut
    u64 ties = 0;
    if (cut_k) {
        u64 above;
        cut = find_cut(false, (u64)k, &above);
        ties = (u64)k - above;
        if (cut_p) total_k = mass_above(cut, 3) + ties * mass(cut);
    }
    if (cut_p) {
        const u64 tau = max(fraction_of(P, total_k, true), 1ull);
        if (tau < total_k) {
            u64 above;
            cut = find_cut(true, tau, &above);
            const u64 w = mass(cut);
            ties = (tau - above + w - 1) / w;
        }
    }

    // ---- the draw in index order: each warp walks a contiguous piece of the words
    const int piece = (nw + WARPS - 1) / WARPS, i0 = min(warp * piece, nw), i1 = min(i0 + piece, nw);
    uint32_t seen0 = 0;                    // tokens with the cut key before this warp's piece
    if (cut) {
        uint32_t c = 0;
        for (int i = i0 + lane; i < i1; i += 32) {
            const uint32_t w = words[i];
#pragma unroll
            for (int e = 0; e < W; ++e) c += K::at(w, e) == cut;
        }
        c = __reduce_add_sync(DG_FULL_MASK, c);
        u64 all;
        const u64 before = block_before(lane == 0 ? c : 0, &all, s);
        seen0 = (uint32_t)__shfl_sync(DG_FULL_MASK, before, 0);
        if (C > 1) {
            if (tid == 0) s.post[4] = all;
            join(C);
            for (int r = 0; r < rank; ++r) seen0 += (uint32_t)remote_load64(&s.post[4], r);
        }
    }
    // f(word index, the masses of this lane's keys in it) in index order; returns when f says so
    auto walk = [&](auto&& f) {
        uint32_t seen = seen0;
        for (int b = i0; b < i1; b += 32) {
            const int i = b + lane;
            const uint32_t word = i < i1 ? words[i] : 0;
            u64 w[W];
            uint32_t t = seen;
            if (cut) {
                unsigned is[W];
#pragma unroll
                for (int e = 0; e < W; ++e) {
                    is[e] = __ballot_sync(DG_FULL_MASK, K::at(word, e) == cut);
                    t += __popc(is[e] & ((1u << lane) - 1));
                    seen += __popc(is[e]);
                }
            }
#pragma unroll
            for (int e = 0; e < W; ++e) {
                const uint32_t key = K::at(word, e);
                w[e] = key > cut || (cut && key == cut && t < ties) ? mass(key) : 0;
                t += key == cut;
                if (w[e] < least) w[e] = 0;
            }
            if (f(i, w)) return;
        }
    };
    u64 mine = 0;
    walk([&](int, const u64 (&w)[W]) {
#pragma unroll
        for (int e = 0; e < W; ++e) mine += w[e];
        return false;
    });
    mine = warp_sum(mine);
    u64 total;
    u64 start = block_before(lane == 0 ? mine : 0, &total, s);
    start = __shfl_sync(DG_FULL_MASK, start, 0);
    if (C > 1) {
        if (tid == 0) s.post[5] = total;
        join(C);
        total = 0;
        for (int r = 0; r < C; ++r) {
            const u64 v = remote_load64(&s.post[5], r);
            if (r < rank) start += v;
            total += v;
        }
        join(C);                           // all slots have been read: any CTA may end
    }
    const u64 at = fraction_of(U, total, false);
    if (start <= at && at < start + mine) {
        u64 run = start;
        walk([&](int i, const u64 (&w)[W]) {
            u64 sum = 0;
#pragma unroll
            for (int e = 0; e < W; ++e) sum += w[e];
            const u64 inc = warp_scan(sum, lane);
            const unsigned hit = __ballot_sync(DG_FULL_MASK, run + inc > at);
            if (hit) {
                if (lane == __ffs(hit) - 1) {
                    const u64 r = run + inc - sum;
                    const int e = W > 1 && at >= r + w[0] ? 1 : 0;
                    const u64 we = w[e ? W - 1 : 0];
                    p.token[row] = (int64_t)s0 + i * W + e - off;
                    if (p.logprob) p.logprob[row] = logf(__fdiv_rn((float)we, (float)total));
                }
                return true;
            }
            run += __shfl_sync(DG_FULL_MASK, inc, 31);
            return false;
        });
    }
}

// CTAs per row: as many (up to 16) as give each SM one, with at least 2048 logits each; and as many as a
// slice of at most 92 KB (two CTAs to an SM) asks for.  A CTA's work beyond its logits is the same
// whatever it holds, so more CTAs than SMs cost more than they save.
int cluster_of(int B, int V, size_t elem) {
    int c = 1;
    while (c < 16 && ((int64_t)B * c * 2 <= 148 && V / (2 * c) >= 2048)) c *= 2;
    while (c < 16 && ((size_t)V + c - 1) / c * elem > 92 * 1024) c *= 2;
    return c;
}

template <typename T> int run(SampleParams p, int B, cudaStream_t stream) {
    p.cluster = cluster_of(B, p.V, sizeof(T));
    p.slice = ((p.V + p.cluster - 1) / p.cluster + 7) / 8 * 8;
    if ((int64_t)B * p.cluster > 0x7fffffff) return DG_ERR_UNSUPPORTED;
    const size_t smem = (size_t)(p.slice + 16) * sizeof(T) + 16;
    auto kern = sample_kernel<T>;
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return dg_host::record_cuda_error(e);
    if (p.cluster == 1) {
        kern<<<(unsigned)B, ST, smem, stream>>>(p);
        return dg_host::check_launch();
    }
    if (p.cluster > 8) {
        e = cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
        if (e != cudaSuccess) return dg_host::record_cuda_error(e);
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(B * p.cluster));
    cfg.blockDim = dim3(ST);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)p.cluster;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    e = cudaLaunchKernelEx(&cfg, kern, p);
    if (e != cudaSuccess) return dg_host::record_cuda_error(e);
    return dg_host::check_launch();
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
    SampleParams p{logits, row_stride, V, 0, 1, u, temperature, top_p, min_p, top_k, temperature_value, top_p_value,
                   min_p_value, top_k_value, token, logprob};
    DG_DISPATCH_LM(dtype, S, { return run<S>(p, B, static_cast<cudaStream_t>(stream)); });
    return DG_OK;
}
