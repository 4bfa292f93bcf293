// sample.cu -- draws one token per row from given uniform numbers, with temperature,
// top-k, top-p and min-p.
//
// Masses are integers: w = floor(2^40 exp((l - max) / T)), summed in 64 bits, so every sum
// is exact and no result depends on the order of a reduction.  The kept set is a prefix of
// the order (logit descending, index ascending): a cut key and the number of tokens with
// that key that stay.  One CTA per row finds the cut by fixing the key's bits from the top:
// each bit takes one pass that sums the count or mass of the keys above a candidate.
#include "lm_common.cuh"

namespace {

constexpr int ST = 512;                    // threads per row
typedef unsigned long long u64;

struct SampleParams {
    const void* logits;
    int64_t row_stride;
    int V;
    const float* u;
    const float *temperature, *top_p, *min_p;
    const int32_t* top_k;
    float temperature_v, top_p_v, min_p_v;
    int32_t top_k_v;
    int64_t* token;
    float* logprob;
};

// unsigned key in the order of the values; NaN counts as -inf, -0 equals +0
__device__ __forceinline__ uint32_t key_of(float l) {
    if (l != l) l = -INFINITY;
    const uint32_t b = __float_as_uint(l + 0.f);
    return b ^ ((b >> 31) ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t key) {
    return __uint_as_float(key ^ ((key >> 31) ? 0x80000000u : 0xffffffffu));
}
// the mass of a token; the row's maximum m is above -inf.  Below -28 (2^40 e^-28 < 1) it is 0, as it
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

__device__ __forceinline__ u64 block_sum(u64 v, u64* buf) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(DG_FULL_MASK, v, o);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) buf[threadIdx.x >> 5] = v;
    __syncthreads();
    u64 s = 0;
#pragma unroll
    for (int i = 0; i < ST / 32; ++i) s += buf[i];
    return s;
}

template <typename T>
__global__ void __launch_bounds__(ST) sample_kernel(SampleParams p) {
    __shared__ u64 buf[ST / 32];
    __shared__ u64 warp_mass[ST / 32];
    __shared__ int warp_ties[ST / 32];
    const int row = blockIdx.x, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const T* lg = static_cast<const T*>(p.logits) + row * p.row_stride;
    const int V = p.V;
    auto load = [&](int i) {
        const float l = dg::to_f(lg[i]);
        return l != l ? -INFINITY : l;
    };
    u64 mk = 0;
    for (int i = tid; i < V; i += ST) mk = max(mk, (u64)key_of(load(i)));
#pragma unroll
    for (int o = 16; o; o >>= 1) mk = max(mk, __shfl_xor_sync(DG_FULL_MASK, mk, o));
    if (lane == 0) buf[warp] = mk;
    __syncthreads();
    for (int i = 0; i < ST / 32; ++i) mk = max(mk, buf[i]);
    const float m = value_of((uint32_t)mk);
    if (m == -INFINITY) {                                      // nothing can be drawn
        if (tid == 0) {
            p.token[row] = -1;
            if (p.logprob) p.logprob[row] = -INFINITY;
        }
        return;
    }
    const float temp = p.temperature ? p.temperature[row] : p.temperature_v;
    const bool greedy = !(temp > 0.f);
    const float tdiv = greedy ? 1.f : temp;
    int k = p.top_k ? p.top_k[row] : p.top_k_v;
    if (k <= 0 || k > V) k = V;
    if (greedy) k = 1;
    const u64 P = (u64)(fminf(fmaxf(p.top_p ? p.top_p[row] : p.top_p_v, 0.f), 1.f) * 16777216.f);
    const u64 least = (u64)(fminf(fmaxf(p.min_p ? p.min_p[row] : p.min_p_v, 0.f), 1.f) * 1099511627776.f);

    // the largest key K with measure(key >= K) >= target; *above = measure(key > K)
    auto find_cut = [&](bool by_mass, u64 target, u64* above) {
        uint32_t key = 0;
        for (int bit = 31; bit >= 0; --bit) {
            const uint32_t c = key | (1u << bit);
            u64 s = 0;
            for (int i = tid; i < V; i += ST) {
                const float l = load(i);
                if (key_of(l) >= c) s += by_mass ? mass_of(l, m, tdiv) : 1ull;
            }
            if (block_sum(s, buf) >= target) key = c;
        }
        u64 s = 0;
        for (int i = tid; i < V; i += ST) {
            const float l = load(i);
            if (key_of(l) > key) s += by_mass ? mass_of(l, m, tdiv) : 1ull;
        }
        *above = block_sum(s, buf);
        return key;
    };
    auto mass_above = [&](uint32_t key) {
        u64 s = 0;
        for (int i = tid; i < V; i += ST) {
            const float l = load(i);
            if (key_of(l) > key) s += mass_of(l, m, tdiv);
        }
        return block_sum(s, buf);
    };

    uint32_t cut = 0;                        // kept: key > cut, and the first `ties` with key == cut
    u64 ties = (u64)V, total_k;
    if (k < V) {
        u64 above;
        cut = find_cut(false, (u64)k, &above);
        ties = (u64)k - above;
        total_k = mass_above(cut) + ties * mass_of(value_of(cut), m, tdiv);
    } else {
        u64 s = 0;
        for (int i = tid; i < V; i += ST) s += mass_of(load(i), m, tdiv);
        total_k = block_sum(s, buf);
    }
    const u64 tau = max(fraction_of(P, total_k, true), 1ull);
    if (tau < total_k) {
        u64 above;
        cut = find_cut(true, tau, &above);
        const u64 w = mass_of(value_of(cut), m, tdiv);
        ties = (tau - above + w - 1) / w;
    }

    // draw in index order: each warp owns a contiguous piece of the row
    const int piece = (V + ST / 32 - 1) / (ST / 32), i0 = min(warp * piece, V), i1 = min(i0 + piece, V);
    int nt = 0;
    for (int i = i0 + lane; i < i1; i += 32) nt += key_of(load(i)) == cut;
    nt = __reduce_add_sync(DG_FULL_MASK, nt);
    if (lane == 0) warp_ties[warp] = nt;
    __syncthreads();
    u64 before_ties = 0;
    for (int i = 0; i < warp; ++i) before_ties += (u64)warp_ties[i];
    auto walk = [&](auto&& each) {          // each(index, mass, this group's ballot work) in index order
        u64 seen = before_ties;
        for (int j = i0; j < i1; j += 32) {
            const int i = j + lane;
            const float l = i < i1 ? load(i) : -INFINITY;
            const uint32_t key = key_of(l);
            const unsigned tie = __ballot_sync(DG_FULL_MASK, i < i1 && key == cut);
            u64 w = 0;
            if (i < i1 && (key > cut || (key == cut && seen + __popc(tie & ((1u << lane) - 1)) < ties)))
                w = mass_of(l, m, tdiv);
            if (w < least) w = 0;
            seen += __popc(tie);
            if (each(i, w)) return;
        }
    };
    u64 mine = 0;
    walk([&](int, u64 w) { mine += w; return false; });
#pragma unroll
    for (int o = 16; o; o >>= 1) mine += __shfl_xor_sync(DG_FULL_MASK, mine, o);
    if (lane == 0) warp_mass[warp] = mine;
    __syncthreads();
    u64 total = 0, start = 0;
    for (int i = 0; i < ST / 32; ++i) {
        if (i < warp) start += warp_mass[i];
        total += warp_mass[i];
    }
    const float uu = fminf(fmaxf(p.u[row], 0.f), 1.f - 1.f / 16777216.f);
    const u64 at = fraction_of((u64)(uu * 16777216.f), total, false);
    if (start <= at && at < start + warp_mass[warp]) {
        u64 run = start;
        walk([&](int i, u64 w) {
            u64 inc = w;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const u64 v = __shfl_up_sync(DG_FULL_MASK, inc, o);
                if (lane >= o) inc += v;
            }
            const unsigned hit = __ballot_sync(DG_FULL_MASK, run + inc > at);
            if (hit) {
                if (lane == __ffs(hit) - 1) {
                    p.token[row] = i;
                    if (p.logprob) p.logprob[row] = logf(__fdiv_rn((float)w, (float)total));
                }
                return true;
            }
            run += __shfl_sync(DG_FULL_MASK, inc, 31);
            return false;
        });
    }
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
    SampleParams p{logits, row_stride, V, u, temperature, top_p, min_p, top_k, temperature_value, top_p_value,
                   min_p_value, top_k_value, token, logprob};
    DG_DISPATCH_LM(dtype, S, { sample_kernel<S><<<B, ST, 0, static_cast<cudaStream_t>(stream)>>>(p); });
    return dg_host::check_launch();
}
