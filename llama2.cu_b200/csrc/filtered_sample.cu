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
// does the running mass of the order cross a bound", and no sort of the row is
// needed, only the entries around each crossing and the mass above them.
//
// One CTA a row, in passes over it of which only the first reads HBM:
//   1  max, mass S (fp32, with a bound of its error) and the maximum of every
//      chunk, which is what one lane reads of one or a few batches of the row
//   2  a threshold from the chunk maxima below which nothing can be kept or
//      drawn, and the entries above it, from the chunks that hold any: these
//      are put in order and decided in fp64 (sample_from_list)
//   3  where those are too many (a flat row), a histogram of the mass over
//      the logit, which brackets each crossing between two edges, then the
//      fp64 sums above the brackets and the entries inside them (sample_by_bins)
// Pass 1's fp32 sum decides only what its error bound allows; else the row is
// summed again in fp64.  What fits neither (NaN, infinities, more entries in a
// bracket than its list holds, as with equal logits, a top-k larger than the number
// of chunks that hold more than a finite mask) takes sample_exact: a radix descent over the
// 32-bit ordered keys with masses in fp64 summed as 64-bit integers in units
// of 2^-62 to 2^-61 of the row's mass, in which equal keys are resolved by division.
// Ids are thus those of real arithmetic up to about 2^-43 of the row's mass,
// whatever the order of the sums was.
#include "device_common.cuh"
#include "fp8_filter_kernels.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

namespace b2s {
namespace {

typedef unsigned long long u64;

constexpr int kFBins = 256;
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
    r.temperature = t;
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

// The temperature in fp64.  Infinity counts as a number that no difference of two
// logits comes near: finite logits weigh the same, and -infinity nothing.
__device__ __forceinline__ double temperature64(float t) { return t > 3.402823466e38f ? 1e300 : (double)t; }

// The smallest logit that passes min-p, in every path the same: of real weights, where a
// weight rounded to 64 bits could be 1 below the top.
__device__ __forceinline__ float minp_threshold(float top, float t, float minp) {
    const float inf = __int_as_float(0x7F800000);
    if (top == inf) return top;
    if (t == inf) return -3.402823466e38f;
    return __double2float_ru((double)top + (double)t * log(fmin((double)minp, 1.0)));
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

// Whether the 8-bit product left this logit out (its own NaN, of the two types it writes).
__device__ __forceinline__ bool unfinished(float x) { return __float_as_uint(x) == kUnfinishedF32; }
__device__ __forceinline__ bool unfinished(__nv_bfloat16 x) { return __bfloat16_as_ushort(x) == kUnfinishedBf16; }
__device__ __forceinline__ bool unfinished(__half) { return false; }

// One row, element by element from global memory.
template <typename T>
struct RowView {
    const T* x;
    int vocab;
    float top;
    double temperature;
    double units;  // of mass in a weight of 1: a power of two, the row's mass is 2^61 to 2^62 of them
    __device__ __forceinline__ float value(int i) const { return as_f32<T>(x[i]); }
    __device__ __forceinline__ u64 mass_of(float v) const {
        return (u64)__double2ll_rn(weight64(v, top, temperature) * units);
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
        // The lanes of one bin add together first: a row's leading digits are few, and
        // those of a row of equal logits one.  A mass is at most 2^62: three words of 21
        // bits, whose sums over a warp fit 32.
        for (int base = 0; base < row.vocab; base += NT) {
            const int i = base + (int)threadIdx.x;
            const float v = i < row.vocab ? row.value(i) : -__int_as_float(0x7F800000);
            const uint32_t k = order_key(v);
            const bool in = k != 0u && (shift == 24 || (k >> (shift + 8)) == prefix);
            if (!__any_sync(kFullMask, in)) continue;
            const int bin = in ? (int)((k >> shift) & 255u) : kFBins;
            const unsigned group = __match_any_sync(kFullMask, bin);
            if (!in) continue;
            const u64 m = row.mass_of(v);
            const unsigned lo = __reduce_add_sync(group, (unsigned)m & 0x1FFFFFu);
            const unsigned mid = __reduce_add_sync(group, (unsigned)(m >> 21) & 0x1FFFFFu);
            const unsigned hi = __reduce_add_sync(group, (unsigned)(m >> 42));
            if ((int)(threadIdx.x & 31) == __ffs(group) - 1) {
                atomicAdd(&sm.count[bin], (unsigned)__popc(group));
                atomicAdd(&sm.mass[bin], ((u64)hi << 42) + ((u64)mid << 21) + lo);
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

// The row by radix descents: right for every row, and slow (a row of 32000 fp32 by itself:
// 0.48 ms with all logits equal, 0.37 with a NaN, 0.26 with an infinity; 14 us by the
// list, 50 by the bins).  Masses are rounded to units of the row's mass: in units of 2^-43
// of the largest weight, which needs two words and not three (0.32 with a NaN), 50000
// roundings moved borders among the lightest entries.
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
    bool nan = false, lost = false;
    for (int i = threadIdx.x; i < p.vocab; i += NT) {
        const float v = row.value(i);
        const unsigned k = order_key(v);
        nan |= v != v;
        lost |= unfinished(row.x[i]);
        top_key = max(top_key, k);
        candidates += k != 0u;
    }
    atomicMax(&sm.red_key, top_key);
    atomicAdd(&sm.red_count, candidates);
    const int any_nan = __syncthreads_or(nan);
    top_key = sm.red_key;
    const u64 n0 = sm.red_count;
    const bool timeout = p.from_product && __syncthreads_or(lost);
    __syncthreads();
    int flags = any_nan ? kFlagNan : 0;
    if (n0 == 0 || timeout) {  // of a row whose logits are not all there, nothing is used
        if (threadIdx.x == 0) {
            p.out_ids[r] = 0;
            if (p.logprobs) p.logprobs[r] = __int_as_float(0xFF800000);
            if (p.kept) p.kept[r] = 0;
            if (p.row_flags) p.row_flags[r] = timeout ? kFlagTimeout : flags | kFlagNoCand;
        }
        __syncthreads();
        return;
    }
    row.top = key_value(top_key);
    row.temperature = rule.greedy ? 1.0 : temperature64(rule.temperature);
    u64 n = n0, total = 0;
    // mass and count of everything, and of what min-p keeps
    const bool use_minp = rule.minp > 0.0f && !rule.greedy;
    const float minp_at = use_minp ? minp_threshold(row.top, rule.temperature, rule.minp) : 0.0f;
    {
        // the mass in fp32, off by far less than 1%, which the units leave room for; the same in every call
        // (a fixed order of sums)
        __shared__ float part[NT / 32];
        const float z = (float)(1.4426950408889634074 / row.temperature);
        float s = 0.0f;
        for (int i = threadIdx.x; i < p.vocab; i += NT) {
            const float v = row.value(i);
            if (order_key(v) != 0u) s += v == row.top ? 1.0f : ex2_approx(fmaxf(v - row.top, -3.402823466e38f) * z);
        }
#pragma unroll
        for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(kFullMask, s, o);
        if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = s;
        if (threadIdx.x == 0) sm.red_count = 0;
        __syncthreads();
        s = 0.0f;
        for (int w = 0; w < NT / 32; ++w) s += part[w];
        row.units = scalbn(1.0, 61 - ilogbf(1.01f * s));  // 1 <= s <= 2^20
    }
    {
        u64 m = 0;
        unsigned c = 0;
        for (int i = threadIdx.x; i < p.vocab; i += NT) {
            const float v = row.value(i);
            if (order_key(v) != 0u && (!use_minp || v >= minp_at)) {
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
            p.logprobs[r] = (float)(d - log((double)total / row.units));
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
constexpr int kChunkCap = 2048;    // chunk maxima kept: 64 groups of batches, one a lane
constexpr int kU = 4;              // vectors of a lane in a batch
constexpr int kFewChunks = 192;    // chunks of the second try of pass 2
constexpr int kCoarse = 16;        // bins that are too few for a threshold with many chunks above it
constexpr int kShortList = 128;    // a list of up to this many is put in order by counting
constexpr float kLowest = -3.402823466e38f;

template <int NT>
struct FastSmem {
    union {
        struct {
            unsigned bin[kBinCap];
        } hist;
        unsigned chunk_bin[kChunkBins];  // zero when pass 2 starts, over before the list does
        struct {
            u64 key[kListCap];   // sorted: falling value, rising index
            union {
                double cum[kListCap];
                int hit[kChunkCap];  // chunks that hold entries above the threshold
            };
        } list;
        ExactSmem exact;
    };
    float chunk_max[kChunkCap];
    double red_d[NT / 32];
    float red_f[4][NT / 32];  // by warp: maximum, minimum, smallest chunk maximum, reference of the sum
    unsigned red_u[NT / 32];
    float coin;
    unsigned n[2];
    unsigned hits;
    int bin[4];
    int status;
    int first;
};

// A row as 16-byte vectors from the 16-byte boundary at or before its first
// element: `lead` elements of vector 0 and the end of the last one are not the
// row's and are neither read nor seen (they count as -infinity).  A warp loads
// batches of 32 * kU vectors, of which lane l has vectors l, l + 32, ..
template <typename T>
struct VecRow {
    static constexpr int E = 16 / sizeof(T);
    const T* base;
    int lead, vocab, vecs, batches;
    int whole_from;
    unsigned whole_count;
    __device__ __forceinline__ VecRow(const T* x, int v) {
        lead = (int)((reinterpret_cast<uintptr_t>(x) & 15u) / sizeof(T));
        base = x - lead;
        vocab = v;
        vecs = (lead + v + E - 1) / E;
        batches = (vecs + 32 * kU - 1) / (32 * kU);
        whole_from = lead ? 1 : 0;
        whole_count = (unsigned)max((lead + v) / E - whole_from, 0);
    }
    __device__ __forceinline__ int index(int vec, int e) const { return vec * E + e - lead; }
    __device__ __forceinline__ bool whole(int vec) const { return (unsigned)(vec - whole_from) < whole_count; }
    __device__ __forceinline__ uint4 load(int vec) const {
        if (whole(vec)) return __ldg(reinterpret_cast<const uint4*>(base) + vec);
        constexpr uint32_t none = sizeof(T) == 4 ? 0xFF800000u : std::is_same<T, __half>::value ? 0xFC00FC00u : 0xFF80FF80u;
        uint4 u = make_uint4(none, none, none, none);
        if (vec < vecs) {
            uint32_t w[4] = {none, none, none, none};
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const int i = index(vec, e);
                if (i >= 0 && i < vocab) {
                    if (sizeof(T) == 4) {
                        w[e & 3] = reinterpret_cast<const uint32_t*>(base)[lead + i];
                    } else {
                        const uint32_t h = reinterpret_cast<const unsigned short*>(base)[lead + i];
                        const int s = 16 * (e & 1);
                        w[(e >> 1) & 3] = (w[(e >> 1) & 3] & ~(0xFFFFu << s)) | (h << s);
                    }
                }
            }
            u = make_uint4(w[0], w[1], w[2], w[3]);
        }
        return u;
    }
    __device__ __forceinline__ void load_batch(int batch, int lane, uint4 (&raw)[kU]) const {
        const int first = batch * 32 * kU;
        if (first >= whole_from && first + 32 * kU <= whole_from + (int)whole_count) {
            const uint4* q = reinterpret_cast<const uint4*>(base) + first + lane;
#pragma unroll
            for (int u = 0; u < kU; ++u) raw[u] = __ldg(q + 32 * u);
        } else {
#pragma unroll 1
            for (int u = 0; u < kU; ++u) {
                const uint4 w = load(first + 32 * u + lane);
                if (u == 0) raw[0] = w;
                if (u == 1) raw[1] = w;
                if (u == 2) raw[2] = w;
                if (u == 3) raw[3] = w;
            }
        }
    }
    __device__ __forceinline__ static void widen(const uint4& u, float (&v)[E]) {
        const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (sizeof(T) == 4) {
                v[i] = __uint_as_float(w[i]);
            } else if constexpr (std::is_same<T, __half>::value) {
                const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
                v[2 * i] = f.x;
                v[2 * i + 1] = f.y;
            } else {
                v[2 * i] = __uint_as_float(w[i] << 16);
                v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
            }
        }
    }
};

__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float max_nan(float a, float b, float c) {
    float r;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
__device__ __forceinline__ float warp_max(float v) {
    float r;
    asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
    return r;
}
__device__ __forceinline__ float warp_max_nan(float v) {
    float r;
    asm volatile("redux.sync.max.NaN.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
    return r;
}
__device__ __forceinline__ float warp_min(float v) {
    float r;
    asm volatile("redux.sync.min.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
    return r;
}

// Two fp32 numbers in one register pair, and the instructions on them.
__device__ __forceinline__ u64 pack2(float a, float b) {
    u64 r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ void unpack2(u64 v, float& a, float& b) {
    asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v));
}
__device__ __forceinline__ u64 fma2(u64 a, u64 b, u64 c) {
    u64 r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ u64 add2(u64 a, u64 b) {
    u64 r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}

// 2^t for t up to 1 (0 below -1000), 2^-44 relative: n = rint(t), and
// 1 + f * P(f) for 2^f, f = t - n, P of degree 8 interpolating (2^f - 1) / f at
// the Chebyshev nodes of [-1/2, 1/2].
__device__ __forceinline__ double exp2_64(double t) {
    const double big = 6755399441055744.0;  // 1.5 * 2^52: its sum with t holds rint(t) in the low word
    const double s = t + big;
    const double f = t - (s - big);
    double p = 0x1.b63880a30e9ffp-24;
    p = fma(p, f, 0x1.63d136366db24p-20);
    p = fma(p, f, 0x1.ffcb9515a8016p-17);
    p = fma(p, f, 0x1.4308ac85aa947p-13);
    p = fma(p, f, 0x1.5d87fe86fe88ep-10);
    p = fma(p, f, 0x1.3b2ab7181b755p-7);
    p = fma(p, f, 0x1.c6b08d7047e52p-5);
    p = fma(p, f, 0x1.ebfbdff823cedp-3);
    p = fma(p, f, 0x1.62e42fefa39efp-1);
    p = fma(p, f, 1.0);
    const double r = __hiloint2double(__double2hiint(p) + (__double2loint(s) << 20), __double2loint(p));
    return t >= -1000.0 ? r : 0.0;
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
#pragma unroll
    for (int w = 0; w < NT / 32; ++w) before += w < warp ? part[w] : V(0);
    __syncthreads();
    return v + before;
}
template <int NT, typename V>
__device__ __forceinline__ V block_sum(V v, V* part) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(kFullMask, v, o);
    if (lane == 0) part[warp] = v;
    __syncthreads();
    V t = 0;
#pragma unroll
    for (int w = 0; w < NT / 32; ++w) t += part[w];
    __syncthreads();
    return t;
}

// What pass 1 and the settings say of a row; the same in every thread.
struct RowFacts {
    float top;         // the largest logit
    float low_chunk;   // the smallest finite chunk maximum
    float z;           // log2(e) / T, as one fp32 number
    double z64;
    float sum;         // mass of the row (the top's is 1), off by up to sum_err of it
    float sum_err;
    float low;         // the smallest logit where pass 1 was asked for it, else -infinity
    float minp_at;     // logits of at least this pass min-p (-infinity when off)
    int chunks;
    int chunk_shift;   // log2 of the batches of a chunk
    // the difference first, which fp64 holds: x * z - top * z would round the second product,
    // by 2^-38 of the weight at top / T = 30000
    __device__ __forceinline__ double weight(float x) const { return exp2_64(((double)x - (double)top) * z64); }
};

enum { kDone = 0, kNeedSum64 = 1, kNeedBins = 2, kNeedExact = 3 };

// Pass 1: maximum, chunk maxima and mass; with kLow the minimum too (an open
// row with -infinity among its entries has to count its candidates).  A chunk is
// what one lane reads of 2^chunk_shift batches.  Weights are 2^t, t = x * z - R with
// an integer R and z in two words: two FMAs, each off by 2^-24 |t| at most.  R is a
// warp's own, the rounded exponent of the largest logit when it was set, and is set
// again (which rescales the sum by a power of two, exactly) as soon as t would pass
// kRefBits.  So |t| is at most |log2 w| + kRefBits + 1 for a weight w against the row's top,
// or against the warp's when that is lower, and the mean of |log2 w| under the weights is
// H - log2 S <= log2(V / S).  Where x * z is large, z's first word puts R and the limit
// off by 2^-22 |x * z| each.  The sum of the weights is thus off by
//   2^-24 * (2 ln 2 * (log2(V / S) + kRefBits + 1 + 2^-20 |top * z|) + 4 + 5 + 1)
// relative at most: the arguments, ex2 (2^-22), the trees (5 levels) and the result.
// Sums of trees are fp64.  An R that lags by more than a few bits is what the bound
// cannot have: at 40 octaves, each argument's rounding is 2^-19 of its weight.
constexpr float kRefBits = 4.0f;

template <int NT, typename T, bool kLow>
__device__ __forceinline__ void first_pass(const VecRow<T>& row, int shift, uint4 (&raw)[kU], FastSmem<NT>& sm,
                                           RowFacts& f) {
    constexpr int E = VecRow<T>::E;
    constexpr int NW = NT / 32;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const float inf = __int_as_float(0x7F800000);
    const float z_hi = __double2float_rd(f.z64);
    // above 0, for -infinity to stay itself: the smallest number there is, as z itself is that small
    // where T is that large
    const float z_lo = fmaxf(__double2float_rd(f.z64 - (double)z_hi), 0x1p-149f);
    const int group = (1 << shift) - 1;
    const u64 zz_hi = pack2(z_hi, z_hi), zz_lo = pack2(z_lo, z_lo);
    // R starts as the smallest there is: entries that x * z takes below it (a mask of the type's lowest
    // value at a T below 1.4) weigh nothing, and must not make R infinite and the weights NaN
    float ref = -3e38f, limit = -inf, top = -inf, chunk = -inf, low = inf, low_chunk = inf;
    double run_sum = 0.0;
    int b = warp << shift;
    while (b < row.batches) {
        const int now = b;
        b = ((b + 1) & group) ? b + 1 : b + 1 + ((NW - 1) << shift);
        float m = -inf;
#pragma unroll
        for (int u = 0; u < kU; ++u) {
            float v[E];
            VecRow<T>::widen(raw[u], v);
#pragma unroll
            for (int e = 0; e < E; e += 2) m = max_nan(m, v[e], v[e + 1]);
            if (kLow) {
                const int vec = (now * kU + u) * 32 + lane;
#pragma unroll
                for (int e = 0; e < E; ++e)
                    if (row.whole(vec) || (row.index(vec, e) >= 0 && row.index(vec, e) < row.vocab)) low = fminf(low, v[e]);
            }
        }
        chunk = max_nan(chunk, m);
        if (b >= row.batches || (b >> shift) != (now >> shift)) {
            sm.chunk_max[((now >> shift) << 5) | lane] = chunk;
            low_chunk = fminf(low_chunk, chunk > -inf ? chunk : inf);
            top = max_nan(top, chunk);
            chunk = -inf;
        }
        if (__any_sync(kFullMask, m > limit)) {
            const float r = fmaxf(rintf(warp_max(m) * z_hi), ref), d = ref - r;
            run_sum *= d > -126.0f ? (double)__int_as_float((127 + (int)d) << 23) : 0.0;
            ref = r;
            limit = (r + kRefBits) / z_hi;
        }
        const u64 rr = pack2(-ref, -ref);
        u64 t[kU];
#pragma unroll
        for (int u = 0; u < kU; ++u) {
            float v[E];
            VecRow<T>::widen(raw[u], v);
            u64 w[E / 2];
#pragma unroll
            for (int i = 0; i < E / 2; ++i) {
                const u64 x = pack2(v[2 * i], v[2 * i + 1]);
                float a, c;
                unpack2(fma2(x, zz_lo, fma2(x, zz_hi, rr)), a, c);
                w[i] = pack2(ex2_approx(a), ex2_approx(c));
            }
#pragma unroll
            for (int h = E / 4; h; h /= 2)
#pragma unroll
                for (int i = 0; i < h; ++i) w[i] = add2(w[i], w[i + h]);
            t[u] = w[0];
        }
        float a, c;
        unpack2(add2(add2(t[0], t[1]), add2(t[2], t[3])), a, c);
        run_sum += (double)(a + c);
        if (b < row.batches) row.load_batch(b, lane, raw);
    }
    // all of these are a lane's; then a warp's; then the row's, in every warp
    top = warp_max_nan(top);
    low_chunk = warp_min(low_chunk);
    if (kLow) low = warp_min(low);
#pragma unroll
    for (int o = 16; o; o >>= 1) run_sum += __shfl_xor_sync(kFullMask, run_sum, o);
    if (lane == 0) {
        sm.red_f[0][warp] = top;
        sm.red_f[1][warp] = low;
        sm.red_f[2][warp] = low_chunk;
        sm.red_f[3][warp] = ref;
        sm.red_d[warp] = run_sum;
    }
    __syncthreads();
    const int w = lane < NW ? lane : 0;
    top = warp_max_nan(sm.red_f[0][w]);
    if (kLow) low = warp_min(sm.red_f[1][w]);
    low_chunk = warp_min(sm.red_f[2][w]);
    const float all = rintf(top * z_hi);
    double s = lane < NW ? sm.red_d[w] * exp2_64(fmin((double)(sm.red_f[3][w] - all), 0.0)) : 0.0;
#pragma unroll
    for (int o = NW / 2; o; o >>= 1) s += __shfl_xor_sync(kFullMask, s, o);
    s = __shfl_sync(kFullMask, s, 0);
    f.sum = (float)(s * exp2_64((double)all - (double)top * f.z64));
    const float bits = fmaxf(__log2f((float)row.vocab / f.sum), 0.0f) + kRefBits + 1.0f + 1e-6f * fabsf(all);
    f.sum_err = 6e-8f * (1.39f * bits + 10.5f);  // 2^-24 and 2 ln 2, with room for second orders
    // where z's second word is a subnormal number it is off by up to 2^-149, times logits 2^129 apart
    f.sum_err += f.z < 0x1p-100f ? 7e-7f : 0.0f;
    f.top = top;
    f.low = kLow ? low : -inf;
    f.low_chunk = low_chunk;
    f.chunk_shift = shift;
    f.chunks = ((row.batches + group) >> shift) << 5;
}

// The mass in fp64 of the whole row, of weights as the lists have them.
template <int NT, typename T>
__device__ __noinline__ double sum64(const VecRow<T>& row, const RowFacts& f, FastSmem<NT>& sm) {
    constexpr int E = VecRow<T>::E;
    double s = 0.0;
    for (int vec = threadIdx.x; vec < row.vecs; vec += NT) {
        float v[E];
        VecRow<T>::widen(row.load(vec), v);
#pragma unroll
        for (int e = 0; e < E; ++e) s += f.weight(v[e]);
    }
    return block_sum<NT>(s, sm.red_d);
}

template <int NT, typename T>
__device__ __noinline__ int count_candidates(const VecRow<T>& row, FastSmem<NT>& sm) {
    constexpr int E = VecRow<T>::E;
    unsigned c = 0;
    for (int vec = threadIdx.x; vec < row.vecs; vec += NT) {
        float v[E];
        VecRow<T>::widen(row.load(vec), v);
#pragma unroll
        for (int e = 0; e < E; ++e) c += v[e] > -__int_as_float(0x7F800000);
    }
    return (int)block_sum<NT>(c, sm.red_u);
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

// One compare-exchange step of a bitonic network over 128 keys of a warp
// (key r * 32 + lane), `first` the index of key 0 in the whole array.
__device__ __forceinline__ void warp_step(u64 (&k)[4], int first, int size, int stride, int lane) {
    u64 o[4];
#pragma unroll
    for (int r = 0; r < 4; ++r)
        o[r] = stride == 64 ? k[r ^ 2] : stride == 32 ? k[r ^ 1] : __shfl_xor_sync(kFullMask, k[r], stride);
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        const int i = first + r * 32 + lane;
        const bool take_max = ((i & stride) == 0) == ((i & size) == 0);
        k[r] = take_max ? (k[r] > o[r] ? k[r] : o[r]) : (k[r] < o[r] ? k[r] : o[r]);
    }
}

// Sorts list[0 .. n) of at most kListCap keys, falling: bitonic, in which the
// steps inside 128 keys are a warp's own and only those across pass through
// shared memory and a barrier (9 for 1024 keys, not 55).
template <int NT>
__device__ void sort_list(u64* list, int n) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int P = 128;
    while (P < n) P <<= 1;
    for (int first = warp * 128; first < P; first += NT / 32 * 128) {
        u64 k[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) k[r] = first + r * 32 + lane < n ? list[first + r * 32 + lane] : 0ull;
#pragma unroll
        for (int size = 2; size <= 128; size <<= 1)
#pragma unroll
            for (int stride = size >> 1; stride > 0; stride >>= 1) warp_step(k, first, size, stride, lane);
#pragma unroll
        for (int r = 0; r < 4; ++r) list[first + r * 32 + lane] = k[r];
    }
    __syncthreads();
    for (int size = 256; size <= P; size <<= 1) {
        for (int stride = size >> 1; stride >= 128; stride >>= 1) {
            for (int q = threadIdx.x; q < (P >> 1); q += NT) {
                const int i = 2 * stride * (q / stride) + (q % stride), l = i + stride;
                const u64 x = list[i], y = list[l];
                if (((i & size) == 0) ? (x < y) : (x > y)) {
                    list[i] = y;
                    list[l] = x;
                }
            }
            __syncthreads();
        }
        for (int first = warp * 128; first < P; first += NT / 32 * 128) {
            u64 k[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) k[r] = list[first + r * 32 + lane];
#pragma unroll
            for (int stride = 64; stride > 0; stride >>= 1) warp_step(k, first, size, stride, lane);
#pragma unroll
            for (int r = 0; r < 4; ++r) list[first + r * 32 + lane] = k[r];
        }
        __syncthreads();
    }
}

// cum[i] = base + the mass of the sorted entries 0 .. i.
template <int NT>
__device__ void scan_list(const u64* list, double* cum, int n, double base, const RowFacts& f, FastSmem<NT>& sm) {
    constexpr int R = (kListCap + NT - 1) / NT;
    double w[R], t = 0.0;
#pragma unroll
    for (int j = 0; j < R; ++j) {
        const int i = (int)threadIdx.x * R + j;
        w[j] = i < n ? f.weight(key_value((uint32_t)(list[i] >> 32))) : 0.0;
        t += w[j];
    }
    double c = base + (block_scan<NT>(t, sm.red_d) - t);
#pragma unroll
    for (int j = 0; j < R; ++j) {
        const int i = (int)threadIdx.x * R + j;
        c += w[j];
        if (i < n) cum[i] = c;
    }
    __syncthreads();
}

// A list of up to kShortList keys in order, each at the number of keys above it
// (counted by NT / kShortList or twice as many threads a key), behind the list;
// its weights in the same order.
template <int NT>
__device__ __forceinline__ const u64* order_short_list(u64* list, double* weight, int n, const RowFacts& f) {
    const int parts = n <= kShortList / 2 ? NT / (kShortList / 2) : NT / kShortList;
    const int i = (int)threadIdx.x / parts, part = (int)threadIdx.x % parts;
    u64* sorted = list + kListCap / 2;
    const u64 key = i < n ? list[i] : 0ull;
    int above = 0;
    if (i < n)
        for (int j = part; j < n; j += parts) above += list[j] > key;
    for (int o = parts >> 1; o; o >>= 1) above += __shfl_xor_sync(kFullMask, above, o);
    if (i < n && part == 0) {
        sorted[above] = key;
        weight[above] = f.weight(key_value((uint32_t)(key >> 32)));
    }
    __syncthreads();
    return sorted;
}

// Weights into their running sums, by one warp.
__device__ __forceinline__ void scan_warp(double* cum, int n, int lane) {
    double before = 0.0;
    for (int i = lane; i - lane < n; i += 32) {
        double c = i < n ? cum[i] : 0.0;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const double u = __shfl_up_sync(kFullMask, c, o);
            if (lane >= o) c += u;
        }
        if (i < n) cum[i] = before + c;
        before += __shfl_sync(kFullMask, c, 31);
    }
    __syncwarp();
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

__device__ __forceinline__ void write_row(const FilterLaunch& p, int r, u64 key, const RowFacts& f, double total,
                                          int kept) {
    p.out_ids[r] = key_index(key);
    if (p.logprobs) {
        const double d = ((double)key_value((uint32_t)(key >> 32)) - (double)f.top) * f.z64;
        const float t = (float)total;  // ln in fp32 plus what the rounding of its argument left
        p.logprobs[r] = (float)(d * 0.69314718055994530942 - ((double)logf(t) + (total - (double)t) / (double)t));
    }
    if (p.kept) p.kept[r] = kept;
    if (p.row_flags) p.row_flags[r] = 0;
}

// Decides a row by its sorted list, by one warp.  kNeedBins when the list does
// not reach far enough, kNeedSum64 when `sum`, off by up to err, leaves a border
// open.  `complete`: every candidate is listed.
template <int NT>
__device__ int decide_list(const FilterLaunch& p, int r, const RowRule& rule, const RowFacts& f, const u64* key, int n,
                           bool complete, int k, double sum, double err, int candidates, FastSmem<NT>& sm) {
    const int lane = threadIdx.x & 31;
    const double* cum = sm.list.cum;
    const bool use_p = rule.topp > 0.0f && rule.topp < 1.0f;
    const bool listed = k > 0 || rule.minp > 0.0f || complete;  // the mass that top-p and the draw refer to
    int kept = n;
    double lo = sum - err, hi = sum + err;
    if (listed) {
        if (rule.minp > 0.0f) {
            kept = 0;
            for (int i = lane; i - lane < n; i += 32)
                kept += __popc(__ballot_sync(kFullMask, i < n && key_value((uint32_t)(key[i] >> 32)) >= f.minp_at));
        }
        if (k > 0 && k < kept) kept = k;
        if (kept < 1) return kNeedExact;
        lo = hi = cum[kept - 1];
    }
    if (use_p) {
        const int at = count_below(cum, kept, (double)rule.topp * lo) + 1;
        if (!listed) {
            if (at > n) return kNeedBins;
            if (count_below(cum, n, (double)rule.topp * hi) + 1 != at) return kNeedSum64;
        }
        kept = min(kept, at);
        lo = hi = cum[kept - 1];
    }
    int at = count_below(cum, kept, (double)rule.coin * lo);
    if (!listed && !use_p) {
        if (at >= n) return kNeedBins;
        if (count_below(cum, n, (double)rule.coin * hi) != at) return kNeedSum64;
        if (p.logprobs && err > 0x1p-18 * sum) return kNeedSum64;  // logits far from 0 against T
        kept = candidates;
        lo = sum;
    }
    at = min(at, kept - 1);
    if (lane == 0) write_row(p, r, key[at], f, lo, kept);
    return kDone;
}

// A threshold by number where the one by mass asks for too long a list: heavy entries
// that share a chunk are missing from the mass of the maxima, which then reaches for
// entries far below them.  The kFewChunks largest maxima, if these nearly hold `mass`:
// their chunks are listed and the threshold is returned, else NaN.  About 1 peaked
// row in 1300 is such a one.  For the kernel of few rows, where one of them is the call's
// time (64 x 128000 bf16, top-p: 102 us by the bins, 27 so); with many rows they hide
// behind the others, and the tries of the rest cost more (4096 x 32000 206 -> 215 us).
template <int NT>
__device__ __noinline__ float cut_by_number(int chunks, float top, float low_chunk, float z, float mass,
                                            FastSmem<NT>& sm) {
    const int lane = threadIdx.x & 31;
    const float inf = __int_as_float(0x7F800000);
    const float scale = (float)(kChunkBins - 1) / (top - low_chunk);
    __syncthreads();
    for (int i = threadIdx.x; i < kChunkBins; i += NT) sm.chunk_bin[i] = 0u;
    if (threadIdx.x == 0) sm.hits = 0u;
    __syncthreads();
    for (int i = threadIdx.x; i < chunks; i += NT) {
        const float m = sm.chunk_max[i];
        if (m > -inf) atomicAdd(&sm.chunk_bin[min((int)((top - m) * scale), kChunkBins - 1)], 1u);
    }
    __syncthreads();
    constexpr int R = kChunkBins / 32;  // every warp forms the same threshold
    unsigned c = 0;
    for (int j = 0; j < R; ++j) c += sm.chunk_bin[lane * R + j];
    unsigned ci = c;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const unsigned cu = __shfl_up_sync(kFullMask, ci, o);
        if (lane >= o) ci += cu;
    }
    ci -= c;
    int found = kChunkBins;
    for (int j = 0; j < R; ++j) {
        ci += sm.chunk_bin[lane * R + j];
        if (ci >= kFewChunks && found == kChunkBins) found = lane * R + j;
    }
    found = __reduce_min_sync(kFullMask, found);
    const float cut = __fsub_rd(top, ((float)found + 1.01f) / scale);
    float held = 0.0f;
    for (int i = threadIdx.x; i < chunks; i += NT) {
        const float m = sm.chunk_max[i];
        if (m >= cut) {
            held += ex2_approx((m - top) * z);
            sm.list.hit[atomicAdd(&sm.hits, 1u)] = i;
        }
    }
    const double all = block_sum<NT>((double)held, sm.red_d);
    return all >= 0.75 * (double)mass && sm.hits <= 2 * kFewChunks ? cut : __int_as_float(0x7FC00000);
}

// The threshold of pass 2 once more, with bins over the chunk maxima from `coarse` on
// only, and the chunks above it listed again: for rows whose range is stretched far below what
// matters, as by logits masked with a large negative number, so that one bin holds all the
// others (32000 fp32, top-k 50, half of them at the lowest value: 263 us by the radix path that a
// list too long ends in, 21 so).  Leaves the smallest of these maxima in sm.red_f[2][0].
template <int NT>
__device__ __noinline__ float finer_cut(int chunks, float top, float z, float coarse, bool by_count, float want,
                                        FastSmem<NT>& sm) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const float inf = __int_as_float(0x7F800000);
    float low = inf;
    for (int i = threadIdx.x; i < chunks; i += NT)
        if (sm.chunk_max[i] >= coarse) low = fminf(low, sm.chunk_max[i]);
    low = warp_min(low);
    __syncthreads();
    if (lane == 0) sm.red_f[2][warp] = low;
    for (int i = threadIdx.x; i < kChunkBins; i += NT) sm.chunk_bin[i] = 0u;
    if (threadIdx.x == 0) sm.hits = 0u;
    __syncthreads();
    low = warp_min(sm.red_f[2][lane < NT / 32 ? lane : 0]);
    const float scale = top > low ? (float)(kChunkBins - 1) / (top - low) : 0.0f;
    for (int i = threadIdx.x; i < chunks; i += NT) {
        const float m = sm.chunk_max[i];
        if (m >= low)
            atomicAdd(&sm.chunk_bin[min((int)((top - m) * scale), kChunkBins - 1)],
                      by_count ? 1u : (unsigned)(ex2_approx((m - top) * z) * 0x1p20f));
    }
    __syncthreads();
    constexpr int R = kChunkBins / 32;  // every warp forms the same threshold
    unsigned c = 0;
    for (int j = 0; j < R; ++j) c += sm.chunk_bin[lane * R + j];
    unsigned ci = c;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const unsigned cu = __shfl_up_sync(kFullMask, ci, o);
        if (lane >= o) ci += cu;
    }
    ci -= c;
    int found = kChunkBins;
    for (int j = 0; j < R; ++j) {
        ci += sm.chunk_bin[lane * R + j];
        if ((float)ci >= want && found == kChunkBins) found = lane * R + j;
    }
    found = __reduce_min_sync(kFullMask, found);
    float cut = coarse;  // min-p's, or the rest's, where that leaves too few
    if (found < kChunkBins) cut = top > low ? fmaxf(__fsub_rd(top, ((float)found + 1.01f) / scale), coarse) : low;
    for (int i = threadIdx.x; i < chunks; i += NT)
        if (sm.chunk_max[i] >= cut) sm.list.hit[atomicAdd(&sm.hits, 1u)] = i;
    if (threadIdx.x == 0) sm.red_f[2][0] = low;
    __syncthreads();
    return cut;
}

// Pass 2: a threshold below which nothing can be kept or drawn, and the row
// decided by the list of the entries above it.
template <int NT, typename T>
__device__ __forceinline__ int sample_from_list(const FilterLaunch& p, int r, const VecRow<T>& row, const RowRule& rule,
                                                RowFacts& f, int k, FastSmem<NT>& sm) {
    constexpr int E = VecRow<T>::E;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const float inf = __int_as_float(0x7F800000);
    const bool use_p = rule.topp > 0.0f && rule.topp < 1.0f;
    // neither top-k nor min-p: the mass is the row's
    const bool open = k == 0 && !(rule.minp > 0.0f);
    // chunk maxima over [low_chunk, top]: how many, and how much mass in them alone,
    // lie at or above each bin's lower edge.  Bin b is at 32 * (b % 16) + b / 16, so
    // that the lanes of the scan, 16 bins each, read 32 banks.
    float span = f.top - f.low_chunk;
    const float scale = span > 0.0f ? (float)(kChunkBins - 1) / span : 0.0f;
    if (open || k > 0) {
        for (int i = threadIdx.x; i < f.chunks; i += NT) {
            const float m = sm.chunk_max[i];
            if (m > -inf) {
                const int b = min((int)((f.top - m) * scale), kChunkBins - 1);
                const int at = ((b & 15) << 5) | (b >> 4);
                atomicAdd(&sm.chunk_bin[at], k > 0 ? 1u : (unsigned)(ex2_approx((m - f.top) * f.z) * 0x1p20f));
            }
        }
        __syncthreads();
    }
    // every warp forms the same threshold
    float cut = -inf, want = 0.0f;
    int found = kChunkBins;
    if (open || k > 0) {
        constexpr int R = kChunkBins / 32;
        unsigned v[R], c = 0;
#pragma unroll
        for (int j = 0; j < R; ++j) c += v[j] = sm.chunk_bin[j * 32 + lane];
        unsigned ci = c;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const unsigned cu = __shfl_up_sync(kFullMask, ci, o);
            if (lane >= o) ci += cu;
        }
        ci -= c;
        // the first bin by which the chunk maxima alone hold k entries, or the mass asked for
        // (each is rounded down to 2^-20 of the largest; decide_list sees to the rest)
        const float part = use_p ? rule.topp : rule.coin;
        want = k > 0 ? (float)k : part * f.sum * 1.00001f * 0x1p20f;
#pragma unroll
        for (int j = 0; j < R; ++j) {
            ci += v[j];
            if ((float)ci >= want && found == kChunkBins) found = lane * R + j;
        }
        found = __reduce_min_sync(kFullMask, found);
        if (found < kChunkBins) cut = span > 0.0f ? __fsub_rd(f.top, ((float)found + 1.01f) / scale) : f.top;
        if (open) {
            // what lies below this cannot hold the rest of the mass, however many they are
            const float rest = fmaxf(1.0f - part, 0x1p-24f) * f.sum;
            cut = fmaxf(cut, __fsub_rd(f.top, 1.001f * __log2f(1.01f * (float)row.vocab / rest) / f.z));
        }
    }
    if (rule.minp > 0.0f) cut = fmaxf(cut, f.minp_at);
    // chunks that hold entries above the threshold
    for (int c = threadIdx.x; c < f.chunks; c += NT) {
        const bool hit = sm.chunk_max[c] >= cut;
        const unsigned who = __ballot_sync(kFullMask, hit);
        if (who == 0u) continue;
        unsigned at = 0;
        if (lane == 0) at = atomicAdd(&sm.hits, (unsigned)__popc(who));
        at = __shfl_sync(kFullMask, at, 0) + __popc(who & ((1u << lane) - 1u));
        if (hit) sm.list.hit[at] = c;
    }
    __syncthreads();
    int hits = (int)sm.hits;
    if (found < kCoarse && hits > kFewChunks) {
        cut = finer_cut<NT>(f.chunks, f.top, f.z, fmaxf(cut, kLowest), k > 0, want, sm);
        hits = (int)sm.hits;
        f.low_chunk = sm.red_f[2][0];
        span = f.top - f.low_chunk;
    }
    // entries to expect, were they spread over the chunks at random
    const float g = (float)f.chunks;
    const float expect = hits < f.chunks ? -g * __logf(1.0f - (float)hits / g) : 1e9f;
    if (row.vocab <= kShortList) {  // the whole row is a short list
        cut = -inf;
        hits = f.chunks;
        __syncthreads();
        for (int c = threadIdx.x; c < f.chunks; c += NT) sm.list.hit[c] = c;
        __syncthreads();
    } else if (expect > fminf(0.9f * kListCap, 64.0f + 0.125f * (float)row.vocab)) {
        // too many for the list, or more to sort than the row is to read again
        if (NT != 1024 || !open || f.chunks < 2 * kFewChunks || !(span > 0.0f) || !(span < 1e37f)) return kNeedBins;
        const float part = use_p ? rule.topp : rule.coin;
        cut = cut_by_number<NT>(f.chunks, f.top, f.low_chunk, f.z, part * f.sum, sm);
        if (!(cut >= f.low_chunk)) return kNeedBins;
        hits = (int)sm.hits;
    }
    const bool complete = !(cut > -inf);
    const int per = 2 + f.chunk_shift, items = hits << per;  // kU << chunk_shift vectors a chunk, one a thread
    for (int i = threadIdx.x; i < items; i += 2 * NT) {
        uint4 raw[2];
        int vec[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int it = i + u * NT, c = it < items ? sm.list.hit[it >> per] : 0;
            vec[u] = it < items ? ((((c >> 5) << per) + (it & ((1 << per) - 1))) << 5) | (c & 31) : row.vecs;
            raw[u] = row.load(vec[u]);
        }
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            float v[E];
            VecRow<T>::widen(raw[u], v);
            unsigned mask = 0u;
#pragma unroll
            for (int e = 0; e < E; ++e) mask |= (v[e] >= cut && v[e] > -inf) ? 1u << e : 0u;
            push_entries<T>(row, vec[u], v, mask, sm.list.key, kListCap, &sm.n[0]);
        }
    }
    __syncthreads();
    const int n = (int)sm.n[0];
    const bool all_of_minp = rule.minp > 0.0f && cut <= f.minp_at;
    if (n > kListCap || n < 1 || (k > 0 && n < k && !complete && !all_of_minp)) return kNeedBins;
    int candidates = row.vocab;
    if (open && !use_p && !complete && !(f.low > -inf) && p.kept) candidates = count_candidates<NT>(row, sm);
    const u64* key = sm.list.key;
    if (n > kShortList) {
        sort_list<NT>(sm.list.key, n);
        scan_list<NT>(sm.list.key, sm.list.cum, n, 0.0, f, sm);
    } else {
        key = order_short_list<NT>(sm.list.key, sm.list.cum, n, f);
    }
    if (warp == 0) {
        if (n <= kShortList) scan_warp(sm.list.cum, n, lane);
        const int st = decide_list<NT>(p, r, rule, f, key, n, complete, k, (double)f.sum, (double)f.sum * f.sum_err,
                                       candidates, sm);
        if (lane == 0) sm.status = st;
    }
    __syncthreads();
    if (sm.status != kNeedSum64) return sm.status;
    const double s64 = sum64<NT>(row, f, sm);
    if (warp == 0) {
        const int st = decide_list<NT>(p, r, rule, f, key, n, complete, k, s64, 0.0, candidates, sm);
        if (lane == 0) sm.status = st;
    }
    __syncthreads();
    return sm.status;
}

// ---- flat rows ----------------------------------------------------------------
struct Bracket {
    float lo, hi;   // bin coordinates [lo, hi) of the bins that hold the crossing; "above" is below lo
    double mass;    // of the entries above
    int above;      // their number
    int n;          // entries in the bracket's list
};

// Coordinates of the bins: (top - x) * scale, rising as the logit falls.
struct BinScale {
    float top, scale;
    __device__ __forceinline__ float at(float x) const { return (top - x) * scale; }
};

// Histogram of the count (kCount) or of the fp32 mass, in `unit`s, of the
// entries >= low that have a bin, and the number of all entries >= low.
template <int NT, typename T, bool kCount>
__device__ __forceinline__ int fill_bins(const VecRow<T>& row, const BinScale& b, float z, float low, float unit,
                                         FastSmem<NT>& sm) {
    constexpr int E = VecRow<T>::E;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    unsigned* hist = sm.hist.bin;
    for (int i = threadIdx.x; i < kBinCap; i += NT) hist[i] = 0u;
    __syncthreads();
    unsigned c = 0;
    for (int i = warp; i < row.batches; i += NT / 32) {
        uint4 raw[kU];
        row.load_batch(i, lane, raw);
#pragma unroll
        for (int u = 0; u < kU; ++u) {
            float v[E];
            VecRow<T>::widen(raw[u], v);
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const bool in = v[e] >= low;
                const float at = b.at(v[e]);
                c += in;
                if (in && at < (float)kBinCap)
                    atomicAdd(&hist[(int)at], kCount ? 1u : __float2uint_rn(ex2_approx((v[e] - b.top) * z) * unit));
            }
        }
    }
    return (int)block_sum<NT>(c, sm.red_u);
}

// First bins whose inclusive running sum exceeds each bound (kBinCap: none; 0 for a bound below 0).
template <int NT>
__device__ __forceinline__ void locate(const float (&bound)[4], int (&bin)[4], FastSmem<NT>& sm) {
    constexpr int R = kBinCap / NT;
    const unsigned* hist = sm.hist.bin;
    if (threadIdx.x < 4) sm.bin[threadIdx.x] = kBinCap;
    unsigned t = 0;
    for (int j = 0; j < R; ++j) t += hist[threadIdx.x * R + j];
    unsigned c = block_scan<NT>(t, sm.red_u) - t;
    for (int j = 0; j < R; ++j) {
        const float before = (float)c;
        c += hist[threadIdx.x * R + j];
#pragma unroll
        for (int q = 0; q < 4; ++q)
            if ((float)c > bound[q] && before <= bound[q]) atomicMin(&sm.bin[q], (int)threadIdx.x * R + j);
    }
    __syncthreads();
#pragma unroll
    for (int q = 0; q < 4; ++q) bin[q] = bound[q] < 0.0f ? 0 : sm.bin[q];
    __syncthreads();
}

// The entries of two brackets (list 1 from `split` on) and, with kMass, the
// masses in fp64: above each bracket and in all.  Entries below `low`, and
// those that equal it with an index above `last`, are not seen.  Returns the
// mass of all.
template <int NT, typename T, bool kMass>
__device__ __forceinline__ double gather_brackets(const VecRow<T>& row, const RowFacts& f, const BinScale& b, float low,
                                                  int last, int split, Bracket (&br)[2], FastSmem<NT>& sm) {
    constexpr int E = VecRow<T>::E;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    if (threadIdx.x < 2) sm.n[threadIdx.x] = 0u;
    __syncthreads();
    double all = 0.0, mass[2] = {0.0, 0.0};
    unsigned above = 0;
    for (int i = warp; i < row.batches; i += NT / 32) {
        uint4 raw[kU];
        row.load_batch(i, lane, raw);
#pragma unroll 1
        for (int u = 0; u < kU; ++u) {
            const int vec = (i * kU + u) * 32 + lane;
            float v[E];
            uint4 w = raw[0];
            if (u == 1) w = raw[1];
            if (u == 2) w = raw[2];
            if (u == 3) w = raw[3];
            VecRow<T>::widen(w, v);
            unsigned mask0 = 0u, mask1 = 0u;
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const float at = b.at(v[e]);
                bool in = v[e] >= low;
                if (v[e] == low && row.index(vec, e) > last) in = false;
                const bool a0 = in && at < br[0].lo, a1 = in && at < br[1].lo;
                above += a0;
                mask0 |= (in && !a0 && at < br[0].hi) ? 1u << e : 0u;
                mask1 |= (in && !a1 && at < br[1].hi) ? 1u << e : 0u;
                if (kMass) {
                    const double m = in ? f.weight(v[e]) : 0.0;
                    all += m;
                    mass[0] += a0 ? m : 0.0;
                    mass[1] += a1 ? m : 0.0;
                }
            }
            push_entries<T>(row, vec, v, mask0, sm.list.key, split, &sm.n[0]);
            push_entries<T>(row, vec, v, mask1, sm.list.key + split, kListCap - split, &sm.n[1]);
        }
    }
    br[0].above = (int)block_sum<NT>(above, sm.red_u);
    if (kMass) {
        all = block_sum<NT>(all, sm.red_d);
        br[0].mass = block_sum<NT>(mass[0], sm.red_d);
        br[1].mass = block_sum<NT>(mass[1], sm.red_d);
    }
    br[0].n = (int)sm.n[0];
    br[1].n = (int)sm.n[1];
    return all;
}

// Pass 3: the crossings by histogram.  Brackets are first as narrow as the
// histogram's typical error makes them, then as wide as its largest.
template <int NT, typename T>
__device__ __noinline__ int sample_by_bins(const FilterLaunch& p, int r, const VecRow<T>& row, const RowRule& rule,
                                           const RowFacts& f, int k, FastSmem<NT>& sm) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const float inf = __int_as_float(0x7F800000);
    const bool use_p = rule.topp > 0.0f && rule.topp < 1.0f;
    float low = rule.minp > 0.0f ? f.minp_at : kLowest;  // logits below it are out,
    int last = 0x7FFFFFFF;                               // and so are equal ones with a larger index
    BinScale b{f.top, 0.0f};
    const Bracket none{0.0f, 0.0f, 0.0, 0, 0};
    int number = 0;
    if (k > 0) {
        // top-k: the k-th entry in the order
        const float span = f.top - fmaxf(fmaxf(low, f.low), f.low_chunk - 2.0f * (f.top - f.low_chunk));
        if (!(span > 0.0f) || !(span < 1e37f)) return kNeedExact;
        b.scale = (float)(kBinCap - 1) / span;
        number = fill_bins<NT, T, true>(row, b, f.z, low, 0.0f, sm);
        if (number > k) {
            const float bound[4] = {(float)(k - 1), -1.0f, -1.0f, -1.0f};  // k <= 2^20: exact
            int bin[4];
            locate<NT>(bound, bin, sm);
            if (bin[0] >= kBinCap) return kNeedExact;
            Bracket br[2] = {{(float)bin[0], (float)(bin[0] + 1), 0.0, 0, 0}, none};
            gather_brackets<NT, T, false>(row, f, b, low, last, kListCap, br, sm);
            const int at = k - 1 - br[0].above;
            if (br[0].n > kListCap || at < 0 || at >= br[0].n) return kNeedExact;
            sort_list<NT>(sm.list.key, br[0].n);
            low = key_value((uint32_t)(sm.list.key[at] >> 32));
            last = key_index(sm.list.key[at]);
            number = k;
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
            const float rest = fmaxf(1.0f - (use_p ? rule.topp : rule.coin), 0x1p-24f) * f.sum;
            bits = fminf(bits, 1.001f * __log2f(1.01f * (float)row.vocab / rest));
        }
        const float span = f.top - fmaxf(f.top - bits / f.z, fmaxf(low, f.low));
        if (!(span < 1e37f)) return kNeedExact;
        b.scale = span > 0.0f ? (float)(kBinCap - 1) / span : 0.0f;
    }
    const int split = use_p ? kListCap / 2 : 0;
    const float unit = 0x1p30f / (1.001f * f.sum);
    double limited_sum = -1.0;
    for (int wide = 0; wide < 2; ++wide) {
        const int counted = fill_bins<NT, T, false>(row, b, f.z, low, unit, sm);
        if (k == 0) number = counted;
        // an entry is off by up to half a unit, at random by a third; the weights by
        // 2e-5 at most
        const float slack = wide ? 0.5f * (float)row.vocab + 0x1p30f * 2e-5f
                                 : 3.0f * sqrtf((float)row.vocab) + 0x1p30f * 1e-6f;
        float total_units = f.sum * unit;
        if (limited && limited_sum < 0.0) {
            unsigned t = 0;
            for (int i = threadIdx.x; i < kBinCap; i += NT) t += sm.hist.bin[i];
            total_units = (float)block_sum<NT>(t, sm.red_u);
        } else if (limited) {
            total_units = (float)limited_sum * unit;
        }
        const float t = (use_p ? rule.topp : 1.0f) * total_units, u = rule.coin * t;
        float bound[4] = {t - slack, t + slack, u - slack, -1.0f};
        int bin[4];
        locate<NT>(bound, bin, sm);
        Bracket br[2] = {none, none};
        const auto past = [&](int q) { return q < kBinCap ? (float)(q + 1) : inf; };
        if (bin[2] >= kBinCap || (use_p && bin[0] >= kBinCap)) return kNeedExact;
        bound[0] = u + slack;
        if (use_p) {
            br[0].lo = (float)bin[0];
            br[0].hi = past(bin[1]);
            // what is kept weighs up to one crossing's bins more than top-p asks for
            bound[0] += rule.coin * ((float)sm.hist.bin[bin[0]] + (float)sm.hist.bin[min(bin[1], kBinCap - 1)]);
        }
        br[1].lo = (float)bin[2];
        bound[1] = bound[2] = -1.0f;
        __syncthreads();
        locate<NT>(bound, bin, sm);
        br[1].hi = past(bin[0]);
        const double sum = gather_brackets<NT, T, true>(row, f, b, low, last, split, br, sm);
        if (br[0].n > split || br[1].n > kListCap - split) return kNeedExact;
        u64* const list[2] = {sm.list.key, sm.list.key + split};
        double* const cum[2] = {sm.list.cum, sm.list.cum + split};
#pragma unroll 1
        for (int q = use_p ? 0 : 1; q < 2; ++q) {
            sort_list<NT>(list[q], br[q].n);
            scan_list<NT>(list[q], cum[q], br[q].n, br[q].mass, f, sm);
        }
        if (warp == 0) {
            int st = kDone, kept = number;
            double total = sum;
            if (use_p) {
                const double bnd = (double)rule.topp * sum;
                const int at = count_below(cum[0], br[0].n, bnd);
                if (br[0].mass > bnd || at >= br[0].n) {
                    st = kNeedSum64;  // not in this bracket
                } else {
                    kept = br[0].above + at + 1;
                    total = cum[0][at];
                }
            }
            const double bnd = (double)rule.coin * total;
            const int at = count_below(cum[1], br[1].n, bnd);
            if (br[1].mass > bnd || at >= br[1].n) st = kNeedSum64;
            if (st == kDone && lane == 0) write_row(p, r, list[1][at], f, total, kept);
            if (lane == 0) sm.status = st;
        }
        __syncthreads();
        const int st = sm.status;
        if (st == kDone) return kDone;
        limited_sum = sum;
        __syncthreads();
    }
    return kNeedExact;
}

// The first entry that equals the maximum.
template <int NT, typename T>
__device__ __forceinline__ void take_first_max(const FilterLaunch& p, int r, const VecRow<T>& row, const RowFacts& f,
                                               FastSmem<NT>& sm) {
    constexpr int E = VecRow<T>::E;
    if (threadIdx.x == 0) sm.first = 0x7FFFFFFF;
    __syncthreads();
    for (int c = threadIdx.x; c < f.chunks; c += NT) {
        if (sm.chunk_max[c] != f.top) continue;
        int at = 0x7FFFFFFF;
        for (int j = 0; j < kU << f.chunk_shift; ++j) {
            const int vec = ((((c >> 5) << f.chunk_shift) * kU + j) << 5) | (c & 31);
            float v[E];
            VecRow<T>::widen(row.load(vec), v);
#pragma unroll
            for (int e = 0; e < E; ++e)
                if (v[e] == f.top) at = min(at, row.index(vec, e));
        }
        atomicMin(&sm.first, at);
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        p.out_ids[r] = sm.first;
        if (p.logprobs) p.logprobs[r] = 0.0f;
        if (p.kept) p.kept[r] = 1;
        if (p.row_flags) p.row_flags[r] = 0;
    }
}

// p stays where the launch put it: by value, its address for the functions out of line
// would be of a copy that every thread makes (4096 x 32000 top-p 227 -> 205 us without).
template <int NT, typename T>
__global__ void __launch_bounds__(NT, 1024 / NT) filtered_sample_kernel(const __grid_constant__ FilterLaunch p) {
    __shared__ FastSmem<NT> sm;
    const int r = blockIdx.x;
    const VecRow<T> row(static_cast<const T*>(p.logits) + (long long)r * p.ld, p.vocab);
    int shift = 0;
    while (((row.batches - 1) >> shift) >= kChunkCap / 32) ++shift;
    uint4 raw[kU];  // the first batch is on its way while the settings are read
    if ((threadIdx.x >> 5) << shift < row.batches) row.load_batch((threadIdx.x >> 5) << shift, threadIdx.x & 31, raw);
    RowRule rule = row_rule(p, r, threadIdx.x == 0);
    for (int i = threadIdx.x; i < kChunkBins; i += NT) sm.chunk_bin[i] = 0u;
    if (threadIdx.x == 0) {
        sm.coin = rule.coin;  // one thread draws, every thread decides by the same number
        sm.hits = 0u;
        sm.n[0] = 0u;
    }
    RowFacts f;
    f.z64 = rule.greedy ? 1.0 : 1.4426950408889634074 / temperature64(rule.temperature);
    f.z = (float)f.z64;
    const int k = rule.topk > 0 && rule.topk < p.vocab ? rule.topk : 0;
    const bool open = !rule.greedy && k == 0 && !(rule.minp > 0.0f) && !(rule.topp > 0.0f && rule.topp < 1.0f);
    if (open) first_pass<NT, T, true>(row, shift, raw, sm, f);
    else first_pass<NT, T, false>(row, shift, raw, sm, f);
    rule.coin = sm.coin;
    const bool plain = f.top > -__int_as_float(0x7F800000) && f.top < __int_as_float(0x7F800000);  // and no NaN
    int st = kNeedExact;
    if (plain && rule.greedy) {
        take_first_max<NT>(p, r, row, f, sm);
        return;
    }
    if (plain && f.sum > 0.0f && f.sum < 1e30f) {
        f.minp_at = rule.minp > 0.0f ? minp_threshold(f.top, rule.temperature, rule.minp) : -__int_as_float(0x7F800000);
        st = sample_from_list<NT>(p, r, row, rule, f, k, sm);
        if (st == kNeedBins) st = sample_by_bins<NT>(p, r, row, rule, f, k, sm);
    }
    __syncthreads();
    if (st != kDone) sample_exact<NT, T>(p, r, rule, sm.exact);
}

template <typename T>
void launch_rows(const FilterLaunch& p, int num_sms, cudaStream_t stream) {
    // Measured (1 B200): 4096 x 32000 fp32, top-p of Zipf rows: 206 us, of which pass 1,
    // all of the HBM traffic, 101; 1 x 32000 13 us; 64 x 128000 bf16 19 us (39 where a row's
    // border is left open by pass 1 and its mass summed again).
    // Threads of a row.  Up to two rows an SM: enough of them that a warp has a batch
    // or two, for the row's latency.  More rows: several on an SM at a time, whose
    // passes overlap; a row of at most 16 batches leaves 8 warps too little between
    // their barriers (4096 x 6000 bf16: 73 us with 8 warps, 52 with 4).
    const long long batches = ((long long)p.vocab * sizeof(T) + 2047) / 2048;
    const bool few = p.batch <= 2 * num_sms;
    if (few && batches > 16) filtered_sample_kernel<1024, T><<<p.batch, 1024, 0, stream>>>(p);
    else if (few || batches > 16) filtered_sample_kernel<256, T><<<p.batch, 256, 0, stream>>>(p);
    else filtered_sample_kernel<128, T><<<p.batch, 128, 0, stream>>>(p);
}

}  // namespace

int launch_filtered_sample(const FilterLaunch& p, int num_sms, cudaStream_t stream) {
    if (p.dtype == kDtypeF32) launch_rows<float>(p, num_sms, stream);
    else if (p.dtype == kDtypeBf16) launch_rows<__nv_bfloat16>(p, num_sms, stream);
    else if (p.dtype == kDtypeF16) launch_rows<__half>(p, num_sms, stream);
    else return -(int)cudaErrorInvalidValue;
    const cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? 1 : -(int)e;
}

}  // namespace b2s
