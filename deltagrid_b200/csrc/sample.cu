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
template <typename T> struct Key {         // 16-bit logits, two at a time
    typedef uint16_t type;
    static constexpr int BITS = 16;
    static constexpr bool BF16 = std::is_same<T, __nv_bfloat16>::value;
    __device__ static __forceinline__ uint32_t pair(uint32_t x) {
        const uint32_t inf = BF16 ? 0x7f807f80u : 0x7c007c00u;
        const uint32_t nan = __vcmpgtu2(x & 0x7fff7fffu, inf);
        x = (x & ~nan) | ((inf | 0x80008000u) & nan);
        x &= ~__vcmpeq2(x, 0x80008000u);
        const uint32_t neg = ((x >> 15) & 0x00010001u) * 0xffffu;
        return x ^ (neg | 0x80008000u);
    }
    __device__ static __forceinline__ uint4 vec(uint4 v) { return make_uint4(pair(v.x), pair(v.y), pair(v.z), pair(v.w)); }
    __device__ static __forceinline__ uint32_t one(T l) { return pair(*reinterpret_cast<const uint16_t*>(&l)) & 0xffffu; }
    __device__ static __forceinline__ float value(uint32_t k) {
        const uint32_t b = (k ^ ((k & 0x8000u) ? 0x8000u : 0xffffu)) & 0xffffu;
        if (BF16) return __uint_as_float(b << 16);
        const uint16_t h = (uint16_t)b;
        return __half2float(*reinterpret_cast<const __half*>(&h));
    }
    // the largest key of a vector
    __device__ static __forceinline__ uint32_t most(uint4 v) {
        const uint32_t m = __vmaxu2(__vmaxu2(v.x, v.y), __vmaxu2(v.z, v.w));
        return max(m & 0xffffu, m >> 16);
    }
    __device__ static __forceinline__ uint32_t at(const uint4& v, int e) {
        const uint32_t w = e < 2 ? v.x : e < 4 ? v.y : e < 6 ? v.z : v.w;
        return e & 1 ? w >> 16 : w & 0xffffu;
    }
};
template <> struct Key<float> {
    typedef uint32_t type;
    static constexpr int BITS = 32;
    __device__ static __forceinline__ uint32_t one(float l) {
        if (l != l) l = -INFINITY;
        const uint32_t b = __float_as_uint(l + 0.f);
        return b ^ ((b >> 31) ? 0xffffffffu : 0x80000000u);
    }
    __device__ static __forceinline__ uint4 vec(uint4 v) {
        return make_uint4(one(__uint_as_float(v.x)), one(__uint_as_float(v.y)), one(__uint_as_float(v.z)),
                          one(__uint_as_float(v.w)));
    }
    __device__ static __forceinline__ float value(uint32_t k) {
        return __uint_as_float(k ^ ((k >> 31) ? 0x80000000u : 0xffffffffu));
    }
    __device__ static __forceinline__ uint32_t most(uint4 v) { return max(max(v.x, v.y), max(v.z, v.w)); }
    __device__ static __forceinline__ uint32_t at(const uint4& v, int e) {
        return e == 0 ? v.x : e == 1 ? v.y : e == 2 ? v.z : v.w;
    }
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
    u64 bins[256];
    u64 warp[WARPS];
    u64 post[8];                           // values that the cluster's other CTAs read
    uint32_t collected;
    uint32_t found_bin;
    u64 found_above;
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

// sorts list[0, n2) (n2 a power of two, 64 to 1024), one exchange per thread and stage; exchanges inside
// 64 elements stay within a warp
__device__ __forceinline__ void sort_list(u64* list, int n2, bool descending) {
    const int t = threadIdx.x;
    for (int size = 2; size <= n2; size *= 2)
        for (int j = size / 2; j; j /= 2) {
            if (t < n2 / 2) {
                const int i = 2 * t - (t & (j - 1)), k = i + j;
                const u64 a = list[i], b = list[k];
                const bool down = ((i & size) == 0) == descending;
                if (down ? a < b : a > b) {
                    list[i] = b;
                    list[k] = a;
                }
            }
            if (j > 32 || (j == 1 && size >= 64)) __syncthreads();
            else __syncwarp();
        }
    __syncthreads();
}

template <typename T>
__global__ void __launch_bounds__(ST, 2) sample_kernel(SampleParams p) {
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

    // ---- the slice as keys: element i at keys[off + i], whole 16-byte vectors of the row on whole
    // vectors of the table, zeros around the slice
    const int head = min((int)((16 - (reinterpret_cast<uintptr_t>(src) & 15)) & 15) / (int)sizeof(T), n);
    const int off = (E - head % E) % E, nv = (off + n + E - 1) / E, body = (n - head) / E, v0 = (off + head) / E;
    uint32_t most0 = 0, most1 = 0;         // largest keys of this thread's even and odd vectors
    if (tid < off) keys[tid] = 0;
    if (tid < nv * E - off - n) keys[off + n + tid] = 0;
    if (tid < head) {
        const uint32_t k = K::one(src[tid]);
        keys[off + tid] = (key_t)k;
        most0 = max(most0, k);
    }
    if (tid < n - head - body * E) {
        const uint32_t k = K::one(src[head + body * E + tid]);
        keys[off + head + body * E + tid] = (key_t)k;
        most1 = max(most1, k);
    }
    const uint4* vsrc = reinterpret_cast<const uint4*>(src + head);
    for (int i = tid; i < body; i += 8 * ST) {
        uint4 v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (i + j * ST < body) v[j] = dg::ldg16(vsrc + i + j * ST);
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (i + j * ST < body) {
                v[j] = K::vec(v[j]);
                vecs[v0 + i + j * ST] = v[j];
                const uint32_t k = K::most(v[j]);
                if (j & 1) most1 = max(most1, k);
                else most0 = max(most0, k);
            }
    }
    if (tid == 0) s.collected = 0;

    // ---- parameters
    const float temp = p.temperature ? p.temperature[row] : p.temperature_v;
    const bool greedy = !(temp > 0.f);
    const float tdiv = greedy ? 1.f : temp;
    int k = p.top_k ? p.top_k[row] : p.top_k_v;
    if (k <= 0 || k > V) k = V;
    if (greedy) k = 1;
    const u64 P = (u64)(fminf(fmaxf(p.top_p ? p.top_p[row] : p.top_p_v, 0.f), 1.f) * 16777216.f);
    const u64 least = (u64)(fminf(fmaxf(p.min_p ? p.min_p[row] : p.min_p_v, 0.f), 1.f) * 1099511627776.f);
    const u64 U = (u64)(fminf(fmaxf(p.u[row], 0.f), 1.f - 1.f / 16777216.f) * 16777216.f);
    const bool cut_k = k < V, cut_p = P < (1u << 24);

    // ---- the row's maximum, and the bound
    const int j_all = cut_k ? k : 256, j = (j_all + C - 1) / C;   // this CTA's share
    const bool collect = (cut_k || cut_p) && j <= 512;
    uint32_t bound = 0;
    u64 mx = __reduce_max_sync(DG_FULL_MASK, max(most0, most1));
    if (lane == 0) s.warp[warp] = mx;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < WARPS; ++i) mx = max(mx, s.warp[i]);
    if (collect) {
        // the largest multiple of 2^low that j partial maxima reach; 20 bits of a 32-bit key are enough
        constexpr int low = K::BITS == 32 ? 12 : 0;
        for (int bit = K::BITS - 1; bit >= low; --bit) {
            const uint32_t c = bound | (1u << bit);
            const int reach = __syncthreads_count(most0 >= c) + __syncthreads_count(most1 >= c);
            if (reach >= j) bound = c;
        }
    }
    if (C > 1) {
        // j tokens of each CTA reach its bound, so C j reach the smallest
        const u64 both = over_cluster(mx << 32 | (0xffffffffu - bound), 0, C, s, [](u64 a, u64 b) {
            return max(a >> 32, b >> 32) << 32 | max(a & 0xffffffffu, b & 0xffffffffu);
        });
        mx = both >> 32;
        bound = 0xffffffffu - (uint32_t)both;
    } else {
        __syncthreads();                   // the keys are there
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
    // f(key, place) for the keys of this CTA's vectors, any order
    auto each = [&](auto&& f) {
        for (int i = tid; i < nv; i += ST) {
            const uint4 v = vecs[i];
#pragma unroll
            for (int e = 0; e < E; ++e) f(K::at(v, e), i * E + e);
        }
    };

    // ---- the mass of the whole row, where top_k does not fix what top_p is a share of
    u64 total_k = 0;
    if (!cut_k && cut_p) {
        u64 w = 0;
        each([&](uint32_t key, int) { if (key) w += mass(key); });
        total_k = over_cluster(block_sum(w, s), 1, C, s, [](u64 a, u64 b) { return a + b; });
    }

    // ---- collect, sort and draw
    if (collect) {
        for (int i = tid; i < nv; i += ST) {
            const uint4 v = vecs[i];
            if (K::most(v) < bound) continue;
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const uint32_t key = K::at(v, e);
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
        bool done = false;
        if (rank == 0) {
            const int nc = (int)min(s.collected, (uint32_t)CAP + 1);
            if (nc <= CAP) {
                int n2 = 64;
                while (n2 < nc) n2 *= 2;
                for (int i = nc + tid; i < n2; i += ST) s.list[i] = 0;
                __syncthreads();
                sort_list(s.list, n2, true);
                // thread t: elements 2t and 2t + 1 of the order
                const int i0 = 2 * tid;
                const u64 e0 = i0 < n2 ? s.list[i0] : 0, e1 = i0 < n2 ? s.list[i0 + 1] : 0;
                const int lim = min(nc, k);
                u64 w0 = i0 < lim ? mass((uint32_t)(e0 >> 32)) : 0, w1 = i0 + 1 < lim ? mass((uint32_t)(e1 >> 32)) : 0;
                u64 sum;
                const u64 before = block_before(w0 + w1, &sum, s);
                if (cut_k) total_k = sum;
                const u64 tau = max(fraction_of(P, total_k, true), 1ull);
                done = cut_k || sum >= tau;
                if (done) {
                    const bool keep0 = i0 < lim && before < tau && w0 >= least;
                    const bool keep1 = i0 + 1 < lim && before + w0 < tau && w1 >= least;
                    const int kept = __syncthreads_count(keep0) + __syncthreads_count(keep1);     // the first `kept`
                    n2 = 64;
                    while (n2 < kept) n2 *= 2;
                    if (i0 < n2) {
                        s.list[i0] = keep0 ? (u64)(0xffffffffu - (uint32_t)e0) << 32 | e0 >> 32 : ~0ull;
                        s.list[i0 + 1] = keep1 ? (u64)(0xffffffffu - (uint32_t)e1) << 32 | e1 >> 32 : ~0ull;
                    }
                    __syncthreads();
                    sort_list(s.list, n2, false);
                    const u64 d0 = i0 < kept ? s.list[i0] : 0, d1 = i0 + 1 < kept ? s.list[i0 + 1] : 0;
                    w0 = i0 < kept ? mass((uint32_t)d0) : 0;
                    w1 = i0 + 1 < kept ? mass((uint32_t)d1) : 0;
                    u64 total;
                    const u64 run = block_before(w0 + w1, &total, s), at = fraction_of(U, total, false);
                    if (run <= at && at < run + w0 + w1) {
                        const bool second = at >= run + w0;
                        p.token[row] = (int64_t)((second ? d1 : d0) >> 32);
                        if (p.logprob)
                            p.logprob[row] = logf(__fdiv_rn((float)(second ? w1 : w0), (float)total));
                    }
                }
            }
            if (tid == 0) s.flag = done;
        }
        join(C);
        if (C > 1) {
            done = remote_load32(&s.flag, 0) != 0;
            join(C);
        }
        if (done) return;
    }

    // ---- the cut by counting
    // the largest key K with measure(key >= K) >= target, and *above = measure(key > K)
    auto find_cut = [&](bool by_mass, u64 target, u64* above_out) {
        u64 above = 0;
        uint32_t lo = 1, hi = (uint32_t)mx;
        const float span = fminf(28.f * tdiv, 3.0e38f);
        const float scale = 255.f / span;
        auto far = [&](uint32_t key) {     // bins of the distance below the maximum; monotone in the key
            const float dist = (m - K::value(key)) * scale;
            return dist < 255.f ? (int)dist : dist == dist ? 255 : 0;
        };
        bool first = true;
        int shift = 0;
        while (true) {
            for (int i = tid; i < 4 * 256; i += ST) (&s.hist[0][0])[i] = 0;
            join(C);
            each([&](uint32_t key, int) {
                if (key < lo || key > hi || key == 0) return;
                const int b = first ? far(key) : (int)((hi - key) >> shift);
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
            join(C);
            if (tid < 256) {
                u64 v = 0;
                for (int r = 0; r < C; ++r) {
                    auto get = [&](int q) { return (u64)(C > 1 ? remote_load32(&s.hist[q][tid], r) : s.hist[q][tid]); };
                    v += by_mass ? get(1) + (get(2) << 13) + (get(3) << 26) : get(0);
                }
                s.bins[tid] = v;
            }
            join(C);                       // the counts may be cleared again
            if (warp == 0) {               // lane l: bins 8 l to 8 l + 7
                u64 v[8], sum = 0;
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i] = s.bins[8 * lane + i], sum += v[i];
                const u64 inc = warp_scan(sum, lane) + above;
                const unsigned hit = __ballot_sync(DG_FULL_MASK, inc >= target);
                // (the last bin is taken where rounding could leave none: never, as sums are exact)
                if (lane == (hit ? __ffs(hit) - 1 : 31)) {
                    u64 run = inc - sum;
                    int i = 0;
                    while (i < 7 && run + v[i] < target) run += v[i++];
                    s.found_bin = 8 * lane + i;
                    s.found_above = run;
                }
            }
            __syncthreads();
            const int bin = (int)s.found_bin;
            above = s.found_above;
            if (first) {
                // the keys of the bin
                u64 least_k = 0xffffffffu, most_k = 0;
                each([&](uint32_t key, int) {
                    if (key && far(key) == bin) {
                        least_k = min(least_k, (u64)key);
                        most_k = max(most_k, (u64)key);
                    }
                });
                const uint32_t a = __reduce_min_sync(DG_FULL_MASK, (uint32_t)least_k);
                const uint32_t b = __reduce_max_sync(DG_FULL_MASK, (uint32_t)most_k);
                __syncthreads();
                if (lane == 0) s.warp[warp] = (u64)b << 32 | (0xffffffffu - a);
                __syncthreads();
                u64 ab = 0;
                auto both = [](u64 x, u64 y) { return max(x >> 32, y >> 32) << 32 | max(x & 0xffffffffu, y & 0xffffffffu); };
#pragma unroll
                for (int i = 0; i < WARPS; ++i) ab = both(ab, s.warp[i]);
                ab = over_cluster(ab, 2, C, s, both);
                lo = 0xffffffffu - (uint32_t)ab;
                hi = (uint32_t)(ab >> 32);
                first = false;
            } else {
                const uint32_t top = hi - ((uint32_t)bin << shift);
                const uint32_t bottom = top - ((1u << shift) - 1);
                lo = bottom > lo && bottom <= top ? bottom : lo;
                hi = top;
            }
            if (lo >= hi) break;
            shift = 0;
            while (((hi - lo) >> shift) > 255) ++shift;
        }
        *above_out = above;
        return hi;
    };
    auto mass_above = [&](uint32_t key, int slot) {
        u64 w = 0;
        each([&](uint32_t kk, int) { if (kk > key) w += mass(kk); });
        return over_cluster(block_sum(w, s), slot, C, s, [](u64 a, u64 b) { return a + b; });
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

    // ---- the draw in index order: each warp walks a contiguous piece of the vectors
    const int piece = (nv + WARPS - 1) / WARPS, i0 = min(warp * piece, nv), i1 = min(i0 + piece, nv);
    u64 seen0 = 0;                         // tokens with the cut key before this warp's piece
    if (cut) {
        u64 c = 0;
        for (int i = i0 + lane; i < i1; i += 32) {
            const uint4 v = vecs[i];
#pragma unroll
            for (int e = 0; e < E; ++e) c += K::at(v, e) == cut;
        }
        c = warp_sum(c);
        u64 all;
        seen0 = block_before(lane == 0 ? c : 0, &all, s);
        seen0 = __shfl_sync(DG_FULL_MASK, seen0, 0);
        if (C > 1) {
            if (tid == 0) s.post[4] = all;
            join(C);
            for (int r = 0; r < rank; ++r) seen0 += remote_load64(&s.post[4], r);
        }
    }
    // f(vector index, this lane's masses of it) in index order; returns when f says so
    auto walk = [&](auto&& f) {
        u64 seen = seen0;
        for (int b = i0; b < i1; b += 32) {
            const int i = b + lane;
            uint4 v = make_uint4(0, 0, 0, 0);
            if (i < i1) v = vecs[i];
            u64 t = 0;
            if (cut) {
                u64 c = 0;
#pragma unroll
                for (int e = 0; e < E; ++e) c += K::at(v, e) == cut;
                const u64 inc = warp_scan(c, lane);
                t = seen + inc - c;
                seen += __shfl_sync(DG_FULL_MASK, inc, 31);
            }
            u64 w[E];
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const uint32_t key = K::at(v, e);
                w[e] = key > cut || (cut && key == cut && t < ties) ? mass(key) : 0;
                t += cut && key == cut;
                if (w[e] < least) w[e] = 0;
            }
            if (f(i, w)) return;
        }
    };
    u64 mine = 0;
    walk([&](int, const u64 (&w)[E]) {
#pragma unroll
        for (int e = 0; e < E; ++e) mine += w[e];
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
        walk([&](int i, const u64 (&w)[E]) {
            u64 sum = 0;
#pragma unroll
            for (int e = 0; e < E; ++e) sum += w[e];
            const u64 inc = warp_scan(sum, lane);
            const unsigned hit = __ballot_sync(DG_FULL_MASK, run + inc > at);
            if (hit) {
                if (lane == __ffs(hit) - 1) {
                    u64 r = run + inc - sum;
                    bool open = true;
#pragma unroll
                    for (int e = 0; e < E; ++e) {
                        if (open && at < r + w[e]) {
                            open = false;
                            p.token[row] = (int64_t)s0 + i * E + e - off;
                            if (p.logprob) p.logprob[row] = logf(__fdiv_rn((float)w[e], (float)total));
                        }
                        r += w[e];
                    }
                }
                return true;
            }
            run += __shfl_sync(DG_FULL_MASK, inc, 31);
            return false;
        });
    }
}

// CTAs per row: rows alone where they fill the SMs; else up to 16, with at least 2048 logits each; and
// as many as a slice of at most 96 KB (two CTAs to an SM) asks for.
int cluster_of(int B, int V, size_t elem) {
    int c = 1;
    while (c < 16 && ((int64_t)B * c * 2 <= 296 && V / (2 * c) >= 2048)) c *= 2;
    while (c < 16 && ((size_t)V + c - 1) / c * elem > 96 * 1024) c *= 2;
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
