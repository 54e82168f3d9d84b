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
// One CTA a row, in passes over it of which only the first reads HBM:
//   1  max, mass S (fp32, with a bound of its error) and the maximum of every
//      chunk of 32 vectors
//   2  a threshold from the chunk maxima below which nothing can be kept or
//      drawn, and the entries above it, from the chunks that hold any: these
//      are sorted and decided in fp64 (sample_from_list)
//   3  where those are too many (a flat row), a histogram of the mass over
//      the logit, which brackets each crossing between two edges, then the
//      sums above the brackets and the entries inside them (sample_by_bins)
// fp32 sums decide only what their error bound allows; else the same sums are
// formed again in fp64.  What fits neither (NaN, infinities, thousands of
// equal logits at a crossing) takes sample_exact: a radix descent over the
// 32-bit ordered keys with masses in fp64 summed as 64-bit integers in units
// of 2^-43, in which equal keys are resolved by division.
// Ids are thus those of real arithmetic up to about 2^-43 of the largest
// weight, whatever the order of the sums was.
#include "device_common.cuh"
#include "fp8_filter_kernels.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace b2s {
namespace {

typedef unsigned long long u64;

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
template <int NT, typename T, bool kByMass>
__device__ Crossing find_crossing(const RowView<T>& row, u64 bound, ExactSmem& sm) {
    uint32_t prefix = 0u;
    u64 above = 0, mass = 0;
    for (int shift = 24; shift >= 0; shift -= 8) {
        for (int i = threadIdx.x; i < kFBins; i += NT) {
            sm.mass[i] = 0;
            sm.count[i] = 0;
        }
        __syncthreads();
        for (int i = threadIdx.x; i < row.vocab; i += NT) {
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
template <int NT, typename T>
__device__ int index_of_tie(const RowView<T>& row, uint32_t key, u64 rank, ExactSmem& sm) {
    // the ties are counted in index order, a strip of the row at a time
    __shared__ unsigned warp_count[NT / 32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    u64 before = 0;
    if (threadIdx.x == 0) sm.id = -1;
    for (int i0 = 0; i0 < row.vocab; i0 += NT) {
        const int i = i0 + threadIdx.x;
        const bool hit = i < row.vocab && order_key(row.value(i)) == key;
        const unsigned m = __ballot_sync(kFullMask, hit);
        if (lane == 0) warp_count[warp] = __popc(m);
        __syncthreads();
        u64 b = before;
        for (int w = 0; w < warp; ++w) b += warp_count[w];
        if (hit && b + __popc(m & ((1u << lane) - 1u)) == rank) sm.id = i;
        for (int w = 0; w < NT / 32; ++w) before += warp_count[w];
        __syncthreads();
        if (before > rank) break;
    }
    __syncthreads();
    return sm.id;
}

// The row by radix descents: right for every row, some hundred times slower than the passes above.
template <int NT, typename T>
__device__ __noinline__ void sample_exact(const FilterLaunch& p, int r, RowRule rule, ExactSmem& sm) {
    RowView<T> row;
    row.x = static_cast<const T*>(p.logits) + (long long)r * p.ld;
    row.vocab = p.vocab;
    if (threadIdx.x == 0) {
        sm.red_key = 0;
        sm.red_count = 0;
        sm.red_mass = 0;
    }
    __syncthreads();
    unsigned top_key = 0, candidates = 0;
    bool nan = false;
    for (int i = threadIdx.x; i < p.vocab; i += NT) {
        const float v = row.value(i);
        const unsigned k = order_key(v);
        nan |= v != v;
        top_key = max(top_key, k);
        candidates += k != 0u;
    }
    atomicMax(&sm.red_key, top_key);
    atomicAdd(&sm.red_count, candidates);
    const int any_nan = __syncthreads_or(nan);
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
        for (int i = threadIdx.x; i < p.vocab; i += NT) {
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
        const Crossing c = find_crossing<NT, T, false>(row, k - 1, sm);
        n = k;
        total = c.mass + (k - c.above) * c.unit;
    }
    if (!rule.greedy && rule.topp > 0.0f && rule.topp < 1.0f) {
        const u64 bound = (u64)((double)rule.topp * (double)total);
        const Crossing c = find_crossing<NT, T, true>(row, bound, sm);
        const u64 j = c.unit ? (bound - c.mass) / c.unit + 1 : 1;
        if (c.above + j < n) {
            n = c.above + j;
            total = c.mass + j * c.unit;
        }
    }
    const u64 bound = (u64)((double)rule.coin * (double)total);
    const Crossing c = find_crossing<NT, T, true>(row, bound, sm);
    u64 rank = c.unit ? (bound - c.mass) / c.unit : 0;
    if (rank >= c.ties) rank = c.ties - 1;
    const int id = index_of_tie<NT>(row, c.key, rank, sm);
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


// ---------------------------------------------------------------------------
// The fast passes
// ---------------------------------------------------------------------------
constexpr int kListCap = 1024;     // entries that can be sorted on chip
constexpr int kBinCap = 2048;      // bins of a histogram
constexpr int kChunkBins = 512;    // bins of the chunk maxima
constexpr int kChunkCap = 2048;    // chunk maxima kept
constexpr int kInFlight = 4;       // vectors a lane loads before it uses them
constexpr float kLog2e = 1.4426950408889634f;

struct Bracket {
    float lo, hi;        // bin coordinates [lo, hi) of the bins that hold the crossing; "above" is below lo
    double mass;         // of the entries above
    int above;           // their number
    int n;               // entries in the bracket's list
};

template <int NT>
struct FastSmem {
    union {
        struct {
            unsigned mass[kBinCap];
            unsigned count[kBinCap];
        } hist;
        struct {
            u64 key[kListCap];   // sorted: falling value, rising index
            double cum[kListCap];
        } list;
        ExactSmem exact;
    };
    float chunk_max[kChunkCap + 4];  // a row that starts between two boundaries has one strip more
    double red_d[NT / 32];
    float red_f[4][NT / 32];
    unsigned red_u[2][NT / 32];
    float coin;
    unsigned n[2];
    int bin[4];
    unsigned cut_count;
    int status;
    int first;
};

// A row as 16-byte vectors from the 16-byte boundary at or before its first
// element: `lead` elements of vector 0 and the end of the last one are not the
// row's and are neither read nor seen (they count as -infinity).
template <typename T>
struct VecRow {
    static constexpr int E = 16 / sizeof(T);
    const T* base;
    int lead, vocab, vecs;
    __device__ __forceinline__ VecRow(const T* x, int v) {
        lead = (int)((reinterpret_cast<uintptr_t>(x) & 15u) / sizeof(T));
        base = x - lead;
        vocab = v;
        vecs = (lead + v + E - 1) / E;
    }
    __device__ __forceinline__ int index(int vec, int e) const { return vec * E + e - lead; }
    __device__ __forceinline__ bool whole(int vec) const { return vec * E >= lead && (vec + 1) * E <= lead + vocab; }
    __device__ __forceinline__ void load(int vec, float (&v)[E]) const {
        if (whole(vec)) {
            const uint4 u = __ldg(reinterpret_cast<const uint4*>(base) + vec);
            unpack(u, v);
        } else {
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const int i = index(vec, e);
                v[e] = (i >= 0 && i < vocab) ? as_f32<T>(base[lead + i]) : -__int_as_float(0x7F800000);
            }
        }
    }
    __device__ __forceinline__ static void unpack(const uint4& u, float (&v)[E]) {
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = __uint_as_float(w[i]);
        } else {
            const T* t = reinterpret_cast<const T*>(&u);
#pragma unroll
            for (int i = 0; i < E; ++i) v[i] = as_f32<T>(t[i]);
        }
    }
};

__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float warp_max_nan(float v) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v = max_nan(v, __shfl_xor_sync(kFullMask, v, o));
    return v;
}

// Sum of `n` values as a tree.
template <int N>
__device__ __forceinline__ float tree_sum(float (&t)[N]) {
#pragma unroll
    for (int h = N / 2; h; h /= 2)
#pragma unroll
        for (int i = 0; i < h; ++i) t[i] += t[i + h];
    return t[0];
}

// Inclusive scan over the CTA's threads.  `part` holds one entry a warp.
template <int NT, typename V>
__device__ __forceinline__ V block_scan(V v, V* part) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const V u = __shfl_up_sync(kFullMask, v, o);
        if (lane >= o) v += u;
    }
    if (lane == 31) part[warp] = v;
    __syncthreads();
    V before = 0;
    for (int w = 0; w < warp; ++w) before += part[w];
    __syncthreads();
    return v + before;
}
template <int NT>
__device__ __forceinline__ double block_sum(double v, double* part) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(kFullMask, v, o);
    if (lane == 0) part[warp] = v;
    __syncthreads();
    double t = 0.0;
#pragma unroll
    for (int w = 0; w < NT / 32; ++w) t += part[w];
    __syncthreads();
    return t;
}

// What pass 1 and the settings say of a row; the same in every thread.
struct RowFacts {
    float top;         // the largest logit
    float low_chunk;   // the smallest finite chunk maximum
    float z;           // log2(e) / T
    double sum;        // mass of the row, off by up to sum_err of it
    double sum_err;
    float low;         // the smallest logit; -infinity when some are masked by it
    float minp_at;     // logits of at least this pass min-p (-infinity when off)
    int chunks;
    int chunk_shift;   // log2 of the 32-vector strips of a chunk
};

// Bound of |sum - true mass| / mass for fp32 weights 2^((x - top) * z), in
// units of 2^-24: the roundings of the difference, of z and of the product make
// 3 ln 2 |log2 w| of a weight, ex2 4; the mean of |log2 w| under the weights is
// H - log2 S <= log2(V / S) bits; the trees have 5 levels, and each change of a
// running maximum costs another ex2 and its argument's error (|d| 2^-d < 0.54
// of the older part).  Sums of trees are fp64.
__device__ __forceinline__ double sum_error(float sum, int vocab, int rescalings) {
    const float bits = fmaxf(__log2f((float)vocab / sum), 0.0f) + 1.0f;
    return 5.97e-8 * (2.1 * (double)bits + 10.0 + 6.0 * (rescalings + 1));
}

enum { kDone = 0, kNeedSum64 = 1, kNeedBins = 2, kNeedExact = 3 };

// Pass 1.  False when the row is for sample_exact (NaN, infinite or no maximum).
template <int NT, typename T>
__device__ bool first_pass(const VecRow<T>& row, FastSmem<NT>& sm, RowFacts& f) {
    constexpr int E = VecRow<T>::E;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const float inf = __int_as_float(0x7F800000);
    const int strips = (row.vecs + 31) >> 5;
    f.chunk_shift = strips > kChunkCap ? 2 : 0;
    f.chunks = (strips + (1 << f.chunk_shift) - 1) >> f.chunk_shift;
    float run_max = -3.402823466e38f, top = -inf, low = inf, low_chunk = inf;
    double run_sum = 0.0;
    int rescalings = 0;
    for (int s0 = warp * kInFlight; s0 < strips; s0 += (NT / 32) * kInFlight) {
        float v[kInFlight][E];
#pragma unroll
        for (int u = 0; u < kInFlight; ++u) row.load((s0 + u) * 32 + lane, v[u]);
        float group = -inf;
#pragma unroll
        for (int u = 0; u < kInFlight; ++u) {
            const int vec = (s0 + u) * 32 + lane;
            float m = v[u][0], l = v[u][0];
#pragma unroll
            for (int e = 1; e < E; ++e) {
                m = max_nan(m, v[u][e]);
                l = fminf(l, v[u][e]);
            }
            if (row.whole(vec)) {
                low = fminf(low, l);
            } else {
#pragma unroll
                for (int e = 0; e < E; ++e)
                    if (row.index(vec, e) >= 0 && row.index(vec, e) < row.vocab) low = fminf(low, v[u][e]);
            }
            m = warp_max_nan(m);
            if (f.chunk_shift == 0) {
                if (lane == 0 && s0 + u < strips) sm.chunk_max[s0 + u] = m;
                if (m > -inf) low_chunk = fminf(low_chunk, m);
            }
            group = max_nan(group, m);
        }
        if (f.chunk_shift != 0) {
            if (lane == 0) sm.chunk_max[s0 >> 2] = group;
            if (group > -inf) low_chunk = fminf(low_chunk, group);
        }
        top = max_nan(top, group);
        if (group > run_max) {  // the whole warp's
            run_sum *= (double)ex2_approx((run_max - group) * f.z);
            run_max = group;
            ++rescalings;
        }
        float t[kInFlight];
#pragma unroll
        for (int u = 0; u < kInFlight; ++u) {
#pragma unroll
            for (int e = 0; e < E; ++e) v[u][e] = ex2_approx((v[u][e] - run_max) * f.z);
            t[u] = tree_sum(v[u]);
        }
        run_sum += (double)tree_sum(t);
    }
    // the maxima are a warp's; the sums and the minimum a lane's
#pragma unroll
    for (int o = 16; o; o >>= 1) low = fminf(low, __shfl_xor_sync(kFullMask, low, o));
    if (lane == 0) {
        sm.red_f[0][warp] = top;
        sm.red_f[1][warp] = low;
        sm.red_f[2][warp] = low_chunk;
        sm.red_u[0][warp] = (unsigned)rescalings;
    }
    __syncthreads();
    top = -inf;
    low = low_chunk = inf;
#pragma unroll
    for (int w = 0; w < NT / 32; ++w) {
        top = max_nan(top, sm.red_f[0][w]);
        low = fminf(low, sm.red_f[1][w]);
        low_chunk = fminf(low_chunk, sm.red_f[2][w]);
        rescalings = max(rescalings, (int)sm.red_u[0][w]);
    }
    f.sum = block_sum<NT>(run_sum * (double)ex2_approx((run_max - top) * f.z), sm.red_d);
    f.sum_err = sum_error((float)f.sum, row.vocab, rescalings + 1);
    f.top = top;
    f.low = low;
    f.low_chunk = low_chunk;
    return top > -inf && top < inf;
}

// The mass in fp64 of the entries whose key is at least `limit`, and their number.
template <int NT, typename T>
__device__ __noinline__ double sum64(const VecRow<T>& row, float top, double temperature, u64 limit, FastSmem<NT>& sm) {
    constexpr int E = VecRow<T>::E;
    double s = 0.0;
    for (int v0 = threadIdx.x; v0 < row.vecs; v0 += NT) {
        float v[E];
        row.load(v0, v);
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const uint32_t k = order_key(v[e]);
            if (k != 0u && (((u64)k << 32) | (0xFFFFFFFFu - (uint32_t)row.index(v0, e))) >= limit)
                s += weight64(v[e], top, temperature);
        }
    }
    return block_sum<NT>(s, sm.red_d);
}

template <int NT, typename T>
__device__ __noinline__ int count_candidates(const VecRow<T>& row, FastSmem<NT>& sm) {
    constexpr int E = VecRow<T>::E;
    int c = 0;
    for (int v0 = threadIdx.x; v0 < row.vecs; v0 += NT) {
        float v[E];
        row.load(v0, v);
#pragma unroll
        for (int e = 0; e < E; ++e) c += v[e] > -__int_as_float(0x7F800000);
    }
    return (int)block_sum<NT>((double)c, sm.red_d);
}

// Appends the entries of one vector that `mask` selects to a list of (key, index).
template <typename T>
__device__ __forceinline__ void push_entries(const VecRow<T>& row, int vec, const float (&v)[VecRow<T>::E],
                                             unsigned mask, u64* list, unsigned cap, unsigned* count) {
    if (mask == 0u) return;
    unsigned at = atomicAdd(count, (unsigned)__popc(mask));
#pragma unroll
    for (int e = 0; e < VecRow<T>::E; ++e)
        if (mask & (1u << e)) {
            if (at < cap) list[at] = ((u64)order_key(v[e]) << 32) | (0xFFFFFFFFu - (uint32_t)row.index(vec, e));
            ++at;
        }
}

// Sorts list[0 .. n) of at most kListCap keys, falling.
template <int NT>
__device__ void sort_list(u64* list, int n) {
    if (n <= 64) {
        if (threadIdx.x < 32) warp_sort_desc<2>(list, n, threadIdx.x & 31);
        __syncthreads();
        return;
    }
    int P = 128;
    while (P < n) P <<= 1;
    for (int i = n + threadIdx.x; i < P; i += NT) list[i] = 0ull;
    __syncthreads();
    block_bitonic_desc(list, P);
}

// cum[i] = base + the mass of the sorted entries 0 .. i.
template <int NT>
__device__ void scan_list(const u64* list, double* cum, int n, double base, float top, double temperature,
                          FastSmem<NT>& sm) {
    constexpr int R = kListCap / NT > 0 ? kListCap / NT : 1;
    double w[R], t = 0.0;
#pragma unroll
    for (int j = 0; j < R; ++j) {
        const int i = (int)threadIdx.x * R + j;
        w[j] = i < n ? weight64(key_value((uint32_t)(list[i] >> 32)), top, temperature) : 0.0;
        t += w[j];
    }
    double c = base + block_scan<NT>(t, sm.red_d) - t;
#pragma unroll
    for (int j = 0; j < R; ++j) {
        const int i = (int)threadIdx.x * R + j;
        c += w[j];
        if (i < n) cum[i] = c;
    }
    __syncthreads();
}

// Number of leading entries with cum <= bound, by one warp.
__device__ __forceinline__ int count_below(const double* cum, int n, double bound) {
    const int lane = threadIdx.x & 31;
    int c = 0;
    for (int i = lane; i - lane < n; i += 32) {
        const unsigned m = __ballot_sync(kFullMask, i < n && cum[i] <= bound);
        c += __popc(m);
        if (m != kFullMask) break;
    }
    return c;
}

__device__ __forceinline__ void write_row(const FilterLaunch& p, int r, int id, float x, float top, double temperature,
                                          double total, int kept) {
    p.out_ids[r] = id;
    if (p.logprobs)
        p.logprobs[r] = (float)((x == top ? 0.0 : ((double)x - (double)top) / temperature) - log(total));
    if (p.kept) p.kept[r] = kept;
    if (p.row_flags) p.row_flags[r] = 0;
}

// Passes 2: the threshold and the list above it.  kNeedBins when the list
// would not hold it, kNeedSum64 when it is there but the bound of f.sum's error
// spans a border (then sum_is64 says that `sum` is exact).
template <int NT>
__device__ int decide_list(const FilterLaunch& p, int r, const RowRule& rule, const RowFacts& f, int n, bool complete,
                           int k, double sum, double err, int candidates, FastSmem<NT>& sm) {
    // one warp
    const int lane = threadIdx.x & 31;
    const double temperature = (double)rule.temperature;
    const u64* key = sm.list.key;
    const double* cum = sm.list.cum;
    const bool limited = k > 0 || rule.minp > 0.0f || complete;
    const bool use_p = rule.topp > 0.0f && rule.topp < 1.0f;
    int kept = n;
    double lo = sum * (1.0 - err), hi = sum * (1.0 + err);
    if (limited) {
        if (rule.minp > 0.0f) {
            int c = 0;
            for (int i = lane; i - lane < n; i += 32)
                c += __popc(__ballot_sync(kFullMask, i < n && key_value((uint32_t)(key[i] >> 32)) >= f.minp_at));
            kept = c;
        }
        if (k > 0 && k < kept) kept = k;
        if (kept < 1) return kNeedExact;
        lo = hi = cum[kept - 1];
    }
    if (use_p) {
        const int at = count_below(cum, kept, (double)rule.topp * lo) + 1;
        if (!limited) {
            if (at > n) return kNeedBins;
            if (count_below(cum, n, (double)rule.topp * hi) + 1 != at) return kNeedSum64;
        }
        kept = min(kept, at);
        lo = hi = cum[kept - 1];
    }
    int at = count_below(cum, limited || use_p ? kept : n, (double)rule.coin * lo);
    if (!limited && !use_p) {
        if (at >= n) return kNeedBins;
        if (count_below(cum, n, (double)rule.coin * hi) != at) return kNeedSum64;
        kept = candidates;
        lo = sum;
    } else if (at > kept - 1) {
        at = kept - 1;
    }
    if (lane == 0)
        write_row(p, r, key_index(key[at]), key_value((uint32_t)(key[at] >> 32)), f.top, temperature, lo, kept);
    return kDone;
}

template <int NT, typename T>
__device__ int sample_from_list(const FilterLaunch& p, int r, const VecRow<T>& row, const RowRule& rule,
                                const RowFacts& f, int k, FastSmem<NT>& sm) {
    constexpr int E = VecRow<T>::E;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const float inf = __int_as_float(0x7F800000);
    const bool use_p = rule.topp > 0.0f && rule.topp < 1.0f;
    const double temperature = (double)rule.temperature;
    float cut = -inf;
    if (row.vocab > kListCap) {
        // chunk maxima over [low_chunk, top]: how many chunks, and how much mass in
        // their maxima alone, lie at or above each bin's lower edge
        const float span = f.top - f.low_chunk;
        const float scale = span > 0.0f ? (float)(kChunkBins - 1) / span : 0.0f;
        for (int i = threadIdx.x; i < kChunkBins; i += NT) sm.hist.mass[i] = sm.hist.count[i] = 0u;
        __syncthreads();
        for (int i = threadIdx.x; i < f.chunks; i += NT) {
            const float m = sm.chunk_max[i];
            if (m > -inf) {
                const int b = min((int)((f.top - m) * scale), kChunkBins - 1);
                atomicAdd(&sm.hist.count[b], 1u);
                atomicAdd(&sm.hist.mass[b], (unsigned)(ex2_approx((m - f.top) * f.z) * 0x1p20f));
            }
        }
        __syncthreads();
        if (warp == 0) {
            constexpr int R = kChunkBins / 32;
            unsigned c = 0, w = 0;
#pragma unroll
            for (int j = 0; j < R; ++j) {
                c += sm.hist.count[lane * R + j];
                w += sm.hist.mass[lane * R + j];
            }
            unsigned ci = c, wi = w;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const unsigned cu = __shfl_up_sync(kFullMask, ci, o), wu = __shfl_up_sync(kFullMask, wi, o);
                if (lane >= o) {
                    ci += cu;
                    wi += wu;
                }
            }
            ci -= c;
            wi -= w;
            // the first bin by which the chunk maxima alone hold k entries, or the mass asked for
            const float part = use_p ? rule.topp : rule.coin;
            const float want = part * (float)f.sum * 1.0001f * 0x1p20f + (float)f.chunks;
            int found = kChunkBins;
#pragma unroll
            for (int j = 0; j < R; ++j) {
                ci += sm.hist.count[lane * R + j];
                wi += sm.hist.mass[lane * R + j];
                const bool there = k > 0 ? ci >= (unsigned)k : (float)wi >= want;
                if (there && found == kChunkBins) found = lane * R + j;
            }
            const unsigned who = __ballot_sync(kFullMask, found < kChunkBins);
            found = __shfl_sync(kFullMask, found, who ? __ffs(who) - 1 : 31);
            float t = found < kChunkBins ? __fsub_rd(f.top, ((float)found + 1.01f) / scale) : -inf;
            if (found < kChunkBins && !(span > 0.0f)) t = f.top;
            if (k == 0 && !(rule.minp > 0.0f)) {
                // what lies below this cannot hold the rest of the mass, however many they are
                const float rest = fmaxf(1.0f - part, 0x1p-24f) * (float)f.sum;
                const float skip = __fsub_rd(f.top, 1.001f * __log2f(1.01f * (float)row.vocab / rest) / f.z);
                if (skip > t) t = skip;
            }
            if (rule.minp > 0.0f) t = k > 0 ? fmaxf(t, f.minp_at) : f.minp_at;
            // chunks that hold entries above the threshold
            unsigned hit = 0;
            for (int i = lane; i < f.chunks; i += 32) hit += sm.chunk_max[i] >= t;
            hit = __reduce_add_sync(kFullMask, hit);
            // entries to expect, were they spread over the chunks at random
            const float g = (float)f.chunks;
            const float expect = (float)hit < g ? -g * __logf(1.0f - (float)hit / g) : 1e9f;
            if (lane == 0) {
                sm.red_f[0][0] = t;
                sm.status = expect <= 0.9f * kListCap ? kDone : kNeedBins;
                sm.n[0] = 0u;
            }
        }
        __syncthreads();
        if (sm.status != kDone) return kNeedBins;
        cut = sm.red_f[0][0];
    } else if (threadIdx.x == 0) {
        sm.n[0] = 0u;
    }
    __syncthreads();
    // the entries at or above the threshold
    const bool complete = !(cut > -inf);
    const int strips = (row.vecs + 31) >> 5;
    for (int c0 = warp * 32; c0 < f.chunks; c0 += NT) {
        unsigned todo = __ballot_sync(kFullMask, c0 + lane < f.chunks && sm.chunk_max[c0 + lane] >= cut);
        while (todo) {
            float v[kInFlight][E];
            int strip[kInFlight];
            if (f.chunk_shift == 0) {
#pragma unroll
                for (int u = 0; u < kInFlight; ++u) {
                    strip[u] = todo ? c0 + __ffs(todo) - 1 : strips;
                    todo &= todo - 1;
                }
            } else {
                const int s0 = (c0 + __ffs(todo) - 1) << 2;
                todo &= todo - 1;
#pragma unroll
                for (int u = 0; u < kInFlight; ++u) strip[u] = s0 + u;
            }
#pragma unroll
            for (int u = 0; u < kInFlight; ++u) row.load(strip[u] * 32 + lane, v[u]);
#pragma unroll
            for (int u = 0; u < kInFlight; ++u) {
                unsigned mask = 0u;
#pragma unroll
                for (int e = 0; e < E; ++e) mask |= (v[u][e] >= cut && v[u][e] > -inf) ? 1u << e : 0u;
                push_entries<T>(row, strip[u] * 32 + lane, v[u], mask, sm.list.key, kListCap, &sm.n[0]);
            }
        }
    }
    __syncthreads();
    const int n = (int)sm.n[0];
    const bool all_of_minp = rule.minp > 0.0f && cut <= f.minp_at;
    if (n > kListCap || (k > 0 && n < k && !complete && !all_of_minp) || n < 1) return kNeedBins;
    sort_list<NT>(sm.list.key, n);
    scan_list<NT>(sm.list.key, sm.list.cum, n, 0.0, f.top, temperature, sm);
    int candidates = row.vocab;
    if (!(f.low > -inf) && k == 0 && !(rule.minp > 0.0f) && !use_p && !complete && p.kept)
        candidates = count_candidates<NT>(row, sm);
    if (warp == 0) {
        const int st = decide_list<NT>(p, r, rule, f, n, complete, k, f.sum, f.sum_err, candidates, sm);
        if (lane == 0) sm.status = st;
    }
    __syncthreads();
    if (sm.status != kNeedSum64) return sm.status;
    const double s64 = sum64<NT>(row, f.top, temperature, 0ull, sm);
    if (warp == 0) {
        const int st = decide_list<NT>(p, r, rule, f, n, complete, k, s64, 0.0, candidates, sm);
        if (lane == 0) sm.status = st;
    }
    __syncthreads();
    return sm.status;
}

// ---- flat rows ----------------------------------------------------------------
// Coordinates of the bins: (top - x) * scale, rising as the logit falls.
struct BinScale {
    float top, scale, z;
    __device__ __forceinline__ float at(float x) const { return (top - x) * scale; }
    __device__ __forceinline__ float weight(float x) const { return ex2_approx((x - top) * z); }
};

// Histogram of count or mass of the entries >= low, and their mass and number.
// mass_unit: units of the mass histogram per weight.
template <int NT, typename T, bool kCount>
__device__ void fill_bins(const VecRow<T>& row, const BinScale& b, float low, float mass_unit, double& mass, int& number,
                          FastSmem<NT>& sm) {
    constexpr int E = VecRow<T>::E;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int strips = (row.vecs + 31) >> 5;
    unsigned* hist = kCount ? sm.hist.count : sm.hist.mass;
    for (int i = threadIdx.x; i < kBinCap; i += NT) hist[i] = 0u;
    __syncthreads();
    double s = 0.0;
    int c = 0;
    for (int s0 = warp * kInFlight; s0 < strips; s0 += (NT / 32) * kInFlight) {
        float v[kInFlight][E];
#pragma unroll
        for (int u = 0; u < kInFlight; ++u) row.load((s0 + u) * 32 + lane, v[u]);
        float t[kInFlight];
#pragma unroll
        for (int u = 0; u < kInFlight; ++u) {
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const float x = v[u][e];
                const bool in = x >= low;
                const int bin = min((int)b.at(x), kBinCap - 1);
                if (kCount) {
                    if (in) atomicAdd(&hist[bin], 1u);
                } else {
                    const float w = in ? b.weight(x) : 0.0f;
                    if (in) atomicAdd(&hist[bin], __float2uint_rn(w * mass_unit));
                    v[u][e] = w;
                }
                c += in;
            }
            t[u] = kCount ? 0.0f : tree_sum(v[u]);
        }
        if (!kCount) s += (double)tree_sum(t);
    }
    mass = kCount ? 0.0 : block_sum<NT>(s, sm.red_d);
    number = (int)block_sum<NT>((double)c, sm.red_d);
}

// First bins whose inclusive running sum exceeds each bound (kBinCap: none).
template <int NT>
__device__ void locate(const unsigned* hist, const float (&bound)[4], int (&bin)[4], FastSmem<NT>& sm) {
    constexpr int R = kBinCap / NT;
    if (threadIdx.x < 4) sm.bin[threadIdx.x] = kBinCap;
    unsigned v[R], t = 0;
#pragma unroll
    for (int j = 0; j < R; ++j) {
        v[j] = hist[threadIdx.x * R + j];
        t += v[j];
    }
    unsigned c = block_scan<NT>(t, sm.red_u[0]) - t;
#pragma unroll
    for (int j = 0; j < R; ++j) {
        const float before = (float)c;
        c += v[j];
#pragma unroll
        for (int q = 0; q < 4; ++q)
            if ((float)c > bound[q] && before <= bound[q]) atomicMin(&sm.bin[q], (int)threadIdx.x * R + j);
    }
    __syncthreads();
#pragma unroll
    for (int q = 0; q < 4; ++q) bin[q] = bound[q] < 0.0f ? 0 : sm.bin[q];
    __syncthreads();
}

// The entries of two brackets (half the list each) and the mass and number above
// them.
template <int NT, typename T, bool kDouble>
__device__ void gather_brackets(const VecRow<T>& row, const BinScale& b, float low, double temperature,
                                Bracket (&br)[2], FastSmem<NT>& sm) {
    constexpr int E = VecRow<T>::E;
    constexpr int U = kInFlight;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int strips = (row.vecs + 31) >> 5;
    if (threadIdx.x < 2) sm.n[threadIdx.x] = 0u;
    __syncthreads();
    double mass[2] = {0.0, 0.0};
    int above[2] = {0, 0};
    for (int s0 = warp * U; s0 < strips; s0 += (NT / 32) * U) {
        float v[U][E], t[2][U];
#pragma unroll
        for (int u = 0; u < U; ++u) row.load((s0 + u) * 32 + lane, v[u]);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            float w[2][E];
            unsigned mask[2] = {0u, 0u};
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const float x = v[u][e], at = b.at(x);
                const bool in = x >= low;
                const float m = kDouble ? 0.0f : b.weight(x);
#pragma unroll
                for (int q = 0; q < 2; ++q) {
                    const bool a = in && at < br[q].lo;
                    above[q] += a;
                    w[q][e] = a ? m : 0.0f;
                    mask[q] |= (in && !a && at < br[q].hi) ? 1u << e : 0u;
                    if (kDouble && a) mass[q] += weight64(x, b.top, temperature);
                }
            }
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                t[q][u] = tree_sum(w[q]);
                push_entries<T>(row, (s0 + u) * 32 + lane, v[u], mask[q], sm.list.key + q * (kListCap / 2),
                                kListCap / 2, &sm.n[q]);
            }
        }
        if (!kDouble) {
            mass[0] += (double)tree_sum(t[0]);
            mass[1] += (double)tree_sum(t[1]);
        }
    }
#pragma unroll
    for (int q = 0; q < 2; ++q) {
        br[q].mass = block_sum<NT>(mass[q], sm.red_d);
        br[q].above = (int)block_sum<NT>((double)above[q], sm.red_d);
        br[q].n = (int)sm.n[q];
    }
}

template <int NT, typename T>
__device__ __noinline__ int sample_by_bins(const FilterLaunch& p, int r, const VecRow<T>& row, const RowRule& rule,
                                           const RowFacts& f, int k, FastSmem<NT>& sm) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const float inf = __int_as_float(0x7F800000);
    const bool use_p = rule.topp > 0.0f && rule.topp < 1.0f;
    const double temperature = (double)rule.temperature;
    float low = rule.minp > 0.0f ? f.minp_at : -3.402823466e38f;  // logits below it are out
    u64 limit = 0;                                                // and so are keys below this
    BinScale b{f.top, 0.0f, f.z};
    const Bracket none{0.0f, 0.0f, 0.0, 0, 0};
    const auto past = [&](int bin) { return bin + 1 < kBinCap ? (float)(bin + 1) : inf; };  // the last bin has no end
    double sum;
    int number;
    if (k > 0) {
        // top-k: the k-th entry in the order
        const float floor_at = fmaxf(fmaxf(low, f.low), f.low_chunk - 2.0f * (f.top - f.low_chunk));
        const float span = f.top - floor_at;
        if (!(span > 0.0f) || !(span < 1e37f)) return kNeedExact;
        b.scale = (float)(kBinCap - 1) / span;
        fill_bins<NT, T, true>(row, b, low, 0.0f, sum, number, sm);
        if (number > k) {
            const float bound[4] = {(float)(k - 1), -1.0f, -1.0f, -1.0f};  // k <= 2^20: exact
            int bin[4];
            locate<NT>(sm.hist.count, bound, bin, sm);
            Bracket br[2] = {{(float)bin[0], past(bin[0]), 0.0, 0, 0}, none};
            gather_brackets<NT, T, false>(row, b, low, temperature, br, sm);
            const int at = k - 1 - br[0].above;
            if (br[0].n > kListCap / 2 || at < 0 || at >= br[0].n) return kNeedExact;
            sort_list<NT>(sm.list.key, br[0].n);
            limit = sm.list.key[at];
            low = key_value((uint32_t)(limit >> 32));
            __syncthreads();
        } else {
            k = 0;
        }
    }
    const bool limited = k > 0 || rule.minp > 0.0f;
    // the mass over the logit, as far down as the rest of it can matter: 48 bits
    // below the top 2^20 entries weigh less than the last coin leaves
    {
        float bits = 48.0f;
        if (!limited) {
            const float rest = fmaxf(1.0f - (use_p ? rule.topp : rule.coin), 0x1p-24f) * (float)f.sum;
            bits = fminf(bits, 1.001f * __log2f(1.01f * (float)row.vocab / rest));
        }
        const float span = f.top - fmaxf(f.top - bits / f.z, fmaxf(low, f.low));
        if (!(span < 1e37f)) return kNeedExact;
        b.scale = span > 0.0f ? (float)(kBinCap - 1) / span : 0.0f;
    }
    const float unit = 0x1p30f / (1.001f * (float)f.sum);
    fill_bins<NT, T, false>(row, b, low, unit, sum, number, sm);
    double err = f.sum_err * f.sum;  // of `sum` and of the masses above the brackets alike
    if (!limited) sum = f.sum;
    if (k > 0) number = k;
    // bins are off by half a unit an entry and by the weights' error
    const float slack = 0.5f * (float)row.vocab + 0x1p30f * 2e-5f;
    const float t = (use_p ? rule.topp : 1.0f) * (float)sum * unit, u = rule.coin * t;
    float bound[4] = {t - slack, t + slack, u - slack, -1.0f};
    int bin[4];
    locate<NT>(sm.hist.mass, bound, bin, sm);
    Bracket br[2] = {none, none};
    if (use_p) {
        if (bin[0] >= kBinCap) return kNeedExact;
        br[0].lo = (float)bin[0];
        br[0].hi = past(bin[1]);
        // what is kept weighs up to one crossing's bins more than top-p asks for
        bound[0] = u + slack + rule.coin * ((float)sm.hist.mass[bin[0]] + (float)sm.hist.mass[min(bin[1], kBinCap - 1)]);
    } else {
        bound[0] = u + slack;
    }
    if (bin[2] >= kBinCap) return kNeedExact;
    br[1].lo = (float)bin[2];
    __syncthreads();
    bound[1] = bound[2] = -1.0f;
    locate<NT>(sm.hist.mass, bound, bin, sm);
    br[1].hi = past(bin[0]);
    for (int precise = k > 0 ? 1 : 0; precise < 2; ++precise) {
        if (precise) {  // entries that equal the k-th and come after it are in the fp32 sum
            sum = sum64<NT>(row, f.top, temperature, k > 0 ? limit : limited ? (u64)order_key(low) << 32 : 0ull, sm);
            err = 0.0;
            gather_brackets<NT, T, true>(row, b, low, temperature, br, sm);
        } else {
            gather_brackets<NT, T, false>(row, b, low, temperature, br, sm);
        }
        if (br[0].n > kListCap / 2 || br[1].n > kListCap / 2) return kNeedExact;
        u64* const list[2] = {sm.list.key, sm.list.key + kListCap / 2};
        double* const cum[2] = {sm.list.cum, sm.list.cum + kListCap / 2};
#pragma unroll
        for (int q = 0; q < 2; ++q) {
            sort_list<NT>(list[q], br[q].n);
            scan_list<NT>(list[q], cum[q], br[q].n, br[q].mass, f.top, temperature, sm);
        }
        if (warp == 0) {
            // place of the crossing of `bnd` in bracket q, where `border` bounds the error of
            // the difference between the bound and a running mass
            const auto place = [&](int q, double bnd, double border, int& st) {
                const int lo = count_below(cum[q], br[q].n, bnd - border), hi = count_below(cum[q], br[q].n, bnd + border);
                if (br[q].mass > bnd + border || lo >= br[q].n) st = kNeedExact;  // not in this bracket
                else if (lo != hi || (br[q].above > 0 && br[q].mass > bnd - border)) st = kNeedSum64;
                return lo;
            };
            int st = kDone, kept = number;
            double total = sum;
            if (use_p) {
                const int at = place(0, (double)rule.topp * sum, 2.0 * err, st);
                if (st == kDone) {
                    kept = min(br[0].above + at + 1, number);  // equals of the k-th behind it are not kept
                    const int last = kept - 1 - br[0].above;
                    if (last < 0) st = kNeedExact;
                    else total = cum[0][last];
                }
            }
            if (st == kDone) {
                const int at = place(1, (double)rule.coin * total, 2.0 * err, st);
                if (st == kDone && lane == 0)
                    write_row(p, r, key_index(list[1][at]), key_value((uint32_t)(list[1][at] >> 32)), f.top,
                              temperature, total, kept);
            }
            if (lane == 0) sm.status = st;
        }
        __syncthreads();
        const int st = sm.status;
        __syncthreads();
        if (st != kNeedSum64) return st;
    }
    return kNeedExact;
}

// The first entry that equals the maximum.
template <int NT, typename T>
__device__ void take_first_max(const FilterLaunch& p, int r, const VecRow<T>& row, const RowFacts& f, FastSmem<NT>& sm) {
    constexpr int E = VecRow<T>::E;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    if (threadIdx.x == 0) sm.first = 0x7FFFFFFF;
    __syncthreads();
    for (int c = warp; c < f.chunks; c += NT / 32) {
        if (sm.chunk_max[c] != f.top) continue;
        for (int s = c << f.chunk_shift; s < (c + 1) << f.chunk_shift; ++s) {
            float v[E];
            row.load(s * 32 + lane, v);
            int at = 0x7FFFFFFF;
#pragma unroll
            for (int e = E - 1; e >= 0; --e)
                if (v[e] == f.top) at = row.index(s * 32 + lane, e);
            if (at != 0x7FFFFFFF) atomicMin(&sm.first, at);
        }
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        p.out_ids[r] = sm.first;
        if (p.logprobs) p.logprobs[r] = 0.0f;
        if (p.kept) p.kept[r] = 1;
        if (p.row_flags) p.row_flags[r] = 0;
    }
}

template <int NT, typename T>
__global__ void __launch_bounds__(NT, 1024 / NT) filtered_sample_kernel(FilterLaunch p) {
    __shared__ FastSmem<NT> sm;
    const int r = blockIdx.x;
    RowRule rule = row_rule(p, r, threadIdx.x == 0);
    if (threadIdx.x == 0) sm.coin = rule.coin;  // one thread draws, every thread decides by the same number
    const T* x = static_cast<const T*>(p.logits) + (long long)r * p.ld;
    const VecRow<T> row(x, p.vocab);
    RowFacts f;
    f.z = rule.greedy ? 1.0f : kLog2e / rule.temperature;
    int st = kNeedExact;
    const bool plain = first_pass<NT>(row, sm, f);
    rule.coin = sm.coin;
    if (plain && rule.greedy) {
        take_first_max<NT>(p, r, row, f, sm);
        return;
    }
    if (plain && f.sum > 0.0) {
        f.minp_at = rule.minp > 0.0f
                        ? __double2float_ru((double)f.top + (double)rule.temperature * log(fmin((double)rule.minp, 1.0)))
                        : -__int_as_float(0x7F800000);
        const int k = rule.topk > 0 && rule.topk < p.vocab ? rule.topk : 0;
        st = sample_from_list<NT>(p, r, row, rule, f, k, sm);
        if (st == kNeedBins) st = sample_by_bins<NT>(p, r, row, rule, f, k, sm);
    }
    __syncthreads();
    if (st != kDone) sample_exact<NT, T>(p, r, rule, sm.exact);
}

template <typename T>
void launch_rows(const FilterLaunch& p, bool wide, cudaStream_t stream) {
    if (wide) filtered_sample_kernel<1024, T><<<p.batch, 1024, 0, stream>>>(p);
    else filtered_sample_kernel<256, T><<<p.batch, 256, 0, stream>>>(p);
}

}  // namespace

int launch_filtered_sample(const FilterLaunch& p, int num_sms, cudaStream_t stream) {
    // Up to two rows an SM: all of an SM's threads on one row, for the row's
    // latency.  More: four rows at a time on an SM, whose passes overlap.
    const bool wide = p.batch <= 2 * num_sms;
    if (p.dtype == kDtypeF32) launch_rows<float>(p, wide, stream);
    else if (p.dtype == kDtypeBf16) launch_rows<__nv_bfloat16>(p, wide, stream);
    else if (p.dtype == kDtypeF16) launch_rows<__half>(p, wide, stream);
    else return -(int)cudaErrorInvalidValue;
    const cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? 1 : -(int)e;
}

}  // namespace b2s
