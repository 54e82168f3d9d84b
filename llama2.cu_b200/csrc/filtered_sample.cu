// filtered_sample.cu -- token ids from logits by temperature, top-k, top-p and
// min-p with one given random number (coin) per row.
//
// A row's entries are ordered by falling logit, ties by rising index.  With
// w_i = exp((l_i - max) / T) every filter keeps a prefix of that order:
//   n0  entries above -infinity that are not NaN
//   n1  = min(n0, top-k, #{w_i >= min-p})
//   n   = the least count whose mass exceeds top-p * (mass of the first n1)
// and the token is the first of the n whose running mass exceeds
// coin * (mass of the n).  So top-p and the draw are the same question, "where
// does the running mass of the order cross a bound", and no sort is needed:
// a radix descent over the 32-bit ordered keys finds the key at the crossing,
// and among equal keys (equal weights) the rank follows by a division.
//
// Ids are decided as in real numbers up to 2^-44 of the largest weight:
// weights are formed in fp64 and summed as 64-bit integers in units of 2^-43,
// so sums do not depend on the order in which they are formed.
#include "device_common.cuh"
#include "fp8_filter_kernels.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace b2s {
namespace {

typedef unsigned long long u64;

constexpr int kFThreads = 512;
constexpr int kFBins = 256;
constexpr double kMassUnit = 8796093022208.0;  // 2^43: 2^20 entries of weight 1 fill 2^63
constexpr float kGreedyBelow = 1e-6f;

template <typename T>
__device__ __forceinline__ float as_f32(T x);
template <>
__device__ __forceinline__ float as_f32<float>(float x) { return x; }
template <>
__device__ __forceinline__ float as_f32<__nv_bfloat16>(__nv_bfloat16 x) { return __bfloat162float(x); }
template <>
__device__ __forceinline__ float as_f32<__half>(__half x) { return __half2float(x); }

// Ordered key: rises with the value, -0 and +0 alike; 0 for what is no
// candidate (NaN, -infinity).
__device__ __forceinline__ uint32_t order_key(float x) {
    const uint32_t b = __float_as_uint(x + 0.0f);
    const uint32_t k = (b & 0x80000000u) ? ~b : (b | 0x80000000u);
    return (x > -__int_as_float(0x7F800000)) ? k : 0u;
}
__device__ __forceinline__ float key_value(uint32_t k) {
    return __uint_as_float((k & 0x80000000u) ? (k & 0x7FFFFFFFu) : ~k);
}

// The settings of one row, with every filter's "off" resolved.
struct RowRule {
    float temperature, topp, minp, coin;
    int topk;
    bool greedy;
};

__device__ __forceinline__ RowRule row_rule(const FilterLaunch& p, int row, bool draw) {
    RowRule r;
    const float t = p.temperature_rows ? p.temperature_rows[row] : p.temperature;
    r.greedy = !(t >= kGreedyBelow);
    r.temperature = fminf(t, 3.402823466e38f);  // so that -infinity / T stays one
    r.topk = p.topk_rows ? p.topk_rows[row] : p.topk;
    r.topp = p.topp_rows ? p.topp_rows[row] : p.topp;
    r.minp = p.minp_rows ? p.minp_rows[row] : p.minp;
    float c = 0.0f;
    if (draw && !r.greedy) {
        if (p.coins) {
            c = p.coins[row];
        } else {
            u64 s = p.rng_state[row];
            c = draw_coin(s);
            p.rng_state[row] = s;
        }
    }
    r.coin = fminf(fmaxf(c, 0.0f), 0x1.fffffep-1f);  // NaN counts as 0
    return r;
}

// exp((x - top) / T); 1 at the top whatever its value is.
__device__ __forceinline__ double weight64(float x, float top, double T) {
    return x == top ? 1.0 : exp(((double)x - (double)top) / T);
}

struct Crossing {
    uint32_t key;   // key of the entry at the crossing
    u64 above;      // entries with a larger key
    u64 mass;       // their mass
    u64 ties;       // entries with this key
    u64 unit;       // mass of one of them
};

struct ExactSmem {
    u64 mass[kFBins];
    unsigned count[kFBins];
    Crossing found;
    u64 red_mass;
    unsigned red_count;
    unsigned red_key;
    float coin;
    int id;
};

// One row, element by element from global memory.
template <typename T>
struct RowView {
    const T* x;
    int vocab;
    float top;
    double temperature;
    __device__ __forceinline__ float value(int i) const { return as_f32<T>(x[i]); }
    __device__ __forceinline__ u64 mass_of(float v) const {
        return (u64)__double2ll_rn(weight64(v, top, temperature) * kMassUnit);
    }
};

// Finds the entry at which the running count (kByMass false) or the running
// mass of the order first exceeds `bound`.  The caller makes sure that the
// whole row's does.  Every thread returns the same.
template <typename T, bool kByMass>
__device__ Crossing find_crossing(const RowView<T>& row, u64 bound, ExactSmem& sm) {
    uint32_t prefix = 0u;
    u64 above = 0, mass = 0;
    for (int shift = 24; shift >= 0; shift -= 8) {
        for (int i = threadIdx.x; i < kFBins; i += kFThreads) {
            sm.mass[i] = 0;
            sm.count[i] = 0;
        }
        __syncthreads();
        for (int i = threadIdx.x; i < row.vocab; i += kFThreads) {
            const float v = row.value(i);
            const uint32_t k = order_key(v);
            if (k != 0u && (shift == 24 || (k >> (shift + 8)) == prefix)) {
                const int bin = (int)((k >> shift) & 255u);
                atomicAdd(&sm.count[bin], 1u);
                atomicAdd(&sm.mass[bin], row.mass_of(v));
            }
        }
        __syncthreads();
        if (threadIdx.x == 0) {
            int bin = kFBins - 1;
            for (; bin > 0; --bin) {
                const u64 next = kByMass ? mass + sm.mass[bin] : above + sm.count[bin];
                if (next > bound) break;
                above += sm.count[bin];
                mass += sm.mass[bin];
            }
            sm.found.key = (prefix << 8) | (uint32_t)bin;
            sm.found.above = above;
            sm.found.mass = mass;
            sm.found.ties = sm.count[bin];
        }
        __syncthreads();
        prefix = sm.found.key;
        above = sm.found.above;
        mass = sm.found.mass;
        __syncthreads();
    }
    Crossing c = sm.found;
    c.unit = row.mass_of(key_value(c.key));
    __syncthreads();
    return c;
}

// Index of the entry with key `key` that has `rank` others of that key before it.
template <typename T>
__device__ int index_of_tie(const RowView<T>& row, uint32_t key, u64 rank, ExactSmem& sm) {
    // the ties are counted in index order, a strip of the row at a time
    __shared__ unsigned warp_count[kFThreads / 32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    u64 before = 0;
    if (threadIdx.x == 0) sm.id = -1;
    for (int i0 = 0; i0 < row.vocab; i0 += kFThreads) {
        const int i = i0 + threadIdx.x;
        const bool hit = i < row.vocab && order_key(row.value(i)) == key;
        const unsigned m = __ballot_sync(kFullMask, hit);
        if (lane == 0) warp_count[warp] = __popc(m);
        __syncthreads();
        u64 b = before;
        for (int w = 0; w < warp; ++w) b += warp_count[w];
        if (hit && b + __popc(m & ((1u << lane) - 1u)) == rank) sm.id = i;
        for (int w = 0; w < kFThreads / 32; ++w) before += warp_count[w];
        __syncthreads();
        if (before > rank) break;
    }
    __syncthreads();
    return sm.id;
}

template <typename T>
__device__ void sample_row_exact(const FilterLaunch& p, int r, ExactSmem& sm) {
    RowView<T> row;
    row.x = static_cast<const T*>(p.logits) + (long long)r * p.ld;
    row.vocab = p.vocab;
    if (threadIdx.x == 0) {
        sm.red_key = 0;
        sm.red_count = 0;
        sm.red_mass = 0;
    }
    __syncthreads();
    RowRule rule = row_rule(p, r, threadIdx.x == 0);
    if (threadIdx.x == 0) sm.coin = rule.coin;  // one thread draws, every thread decides by the same number
    unsigned top_key = 0, candidates = 0;
    bool nan = false;
    for (int i = threadIdx.x; i < p.vocab; i += kFThreads) {
        const float v = row.value(i);
        const unsigned k = order_key(v);
        nan |= v != v;
        top_key = max(top_key, k);
        candidates += k != 0u;
    }
    atomicMax(&sm.red_key, top_key);
    atomicAdd(&sm.red_count, candidates);
    const int any_nan = __syncthreads_or(nan);
    rule.coin = sm.coin;
    top_key = sm.red_key;
    const u64 n0 = sm.red_count;
    __syncthreads();
    int flags = any_nan ? kFlagNan : 0;
    if (n0 == 0) {
        if (threadIdx.x == 0) {
            p.out_ids[r] = 0;
            if (p.logprobs) p.logprobs[r] = __int_as_float(0xFF800000);
            if (p.kept) p.kept[r] = 0;
            if (p.row_flags) p.row_flags[r] = flags | kFlagNoCand;
        }
        __syncthreads();
        return;
    }
    row.top = key_value(top_key);
    row.temperature = rule.greedy ? 1.0 : (double)rule.temperature;
    u64 n = n0, total = 0;
    // mass and count of everything, and of what min-p keeps
    const bool use_minp = rule.minp > 0.0f && !rule.greedy;
    const double minp = fmin((double)rule.minp, 1.0);
    if (threadIdx.x == 0) sm.red_count = 0;
    __syncthreads();
    {
        u64 m = 0;
        unsigned c = 0;
        for (int i = threadIdx.x; i < p.vocab; i += kFThreads) {
            const float v = row.value(i);
            if (order_key(v) != 0u && (!use_minp || weight64(v, row.top, row.temperature) >= minp)) {
                m += row.mass_of(v);
                ++c;
            }
        }
        atomicAdd(&sm.red_mass, m);
        atomicAdd(&sm.red_count, c);
    }
    __syncthreads();
    n = sm.red_count;
    total = sm.red_mass;
    __syncthreads();
    const u64 k = rule.greedy ? 1 : (rule.topk > 0 ? (u64)rule.topk : n);
    if (k < n) {
        const Crossing c = find_crossing<T, false>(row, k - 1, sm);
        n = k;
        total = c.mass + (k - c.above) * c.unit;
    }
    if (!rule.greedy && rule.topp > 0.0f && rule.topp < 1.0f) {
        const u64 bound = (u64)((double)rule.topp * (double)total);
        const Crossing c = find_crossing<T, true>(row, bound, sm);
        const u64 j = c.unit ? (bound - c.mass) / c.unit + 1 : 1;
        if (c.above + j < n) {
            n = c.above + j;
            total = c.mass + j * c.unit;
        }
    }
    const u64 bound = (u64)((double)rule.coin * (double)total);
    const Crossing c = find_crossing<T, true>(row, bound, sm);
    u64 rank = c.unit ? (bound - c.mass) / c.unit : 0;
    if (rank >= c.ties) rank = c.ties - 1;
    const int id = index_of_tie(row, c.key, rank, sm);
    if (threadIdx.x == 0) {
        p.out_ids[r] = id;
        if (p.logprobs) {
            const double d = key_value(c.key) == row.top ? 0.0 : ((double)key_value(c.key) - (double)row.top) / row.temperature;
            p.logprobs[r] = (float)(d - log((double)total / kMassUnit));
        }
        if (p.kept) p.kept[r] = (int)n;
        if (p.row_flags) p.row_flags[r] = flags;
    }
    __syncthreads();
}

template <typename T>
__global__ void __launch_bounds__(kFThreads) filtered_sample_kernel(FilterLaunch p) {
    __shared__ ExactSmem sm;
    for (int r = blockIdx.x; r < p.batch; r += gridDim.x) sample_row_exact<T>(p, r, sm);
}

}  // namespace

int launch_filtered_sample(const FilterLaunch& p, int num_sms, cudaStream_t stream) {
    const int grid = p.batch < 2 * num_sms ? p.batch : 2 * num_sms;
    if (p.dtype == kDtypeF32) filtered_sample_kernel<float><<<grid, kFThreads, 0, stream>>>(p);
    else if (p.dtype == kDtypeBf16) filtered_sample_kernel<__nv_bfloat16><<<grid, kFThreads, 0, stream>>>(p);
    else if (p.dtype == kDtypeF16) filtered_sample_kernel<__half><<<grid, kFThreads, 0, stream>>>(p);
    else return -(int)cudaErrorInvalidValue;
    const cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? 1 : -(int)e;
}

}  // namespace b2s
