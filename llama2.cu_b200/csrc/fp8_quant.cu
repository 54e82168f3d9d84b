// fp8_quant.cu -- operands of the 8-bit classifier: float8 e4m3 values with
// one fp32 scale per block of 128 consecutive columns (activations: a block
// is 1 x 128; weights: 128 x 128), and the final RMSNorm that writes such
// rows in the same pass.
//
// Per block: amax = max |x|, s = max(RN(amax / 448), 2^-126), and
// q = RN_e4m3(RN(x / s)) (448 is the largest e4m3 value; ties to even).  The
// scale is rounded to fp32 before the division, so q * s is the nearest the
// format has to x under the scale that is stored (a quotient within 2^-24 of a
// tie counts as the tie).  The clamp gives a block of zeros a scale that can be
// divided by.  A block that holds a NaN or an infinity gets scale NaN and NaN
// values: whatever is computed from it shows.
//
// All three are bound by memory: an element is read once (4 or 2 bytes) and
// written once (1 byte).  What stands in the way is the number of instructions
// an element costs, so a lane has eight elements of one or two blocks (the scale,
// its reciprocal and the addresses are worked out once for them), the division is
// a product and two FMAs, and the kernels come in two forms.  kWhole, where rows
// start on 16 bytes and have a multiple of eight columns: the eight are
// consecutive, 16 lanes have a block's row.  Else they are four columns 32 apart of
// one block's row, which the whole warp has, and four of another's, so that the
// scalar loads and stores of a warp are of consecutive elements
// (weights 20001 x 1601 fp16: 36 us, 64 with consecutive ones).
// Measured (1 B200): weights 32000 x 4096 bf16 62 us on the device (60 of bytes),
// RMSNorm 8192 x 4096 fp32 35 us (26 of bytes).
#include "device_common.cuh"
#include "fp8_filter_kernels.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace b2s {
namespace {

constexpr int kQBlock = 128;
constexpr int kQThreads = 256;
constexpr int kN = 8;                // consecutive elements of a lane
constexpr int kG = kQBlock / kN;     // lanes of a block's row: two rows a warp
constexpr float kFp8Max = 448.0f;

__device__ __forceinline__ float widen(float x) { return x; }
__device__ __forceinline__ float widen(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float widen(__half x) { return __half2float(x); }

// Eight elements as they are in memory.
template <typename T>
struct Raw {
    uint32_t w[kN * sizeof(T) / 4];
};

// Eight elements: consecutive from p, there when n > 0 (kWhole); else four from p
// and four from p + second, 32 apart, of which those exist whose distance is below
// n and n2.
template <typename T, bool kWhole>
__device__ __forceinline__ Raw<T> load_raw(const T* p, int n, long long second, int n2) {
    constexpr int W = kN * sizeof(T) / 4;
    Raw<T> r;
#pragma unroll
    for (int i = 0; i < W; ++i) r.w[i] = 0u;
    if (kWhole) {
        if (n > 0) {
#pragma unroll
            for (int i = 0; i < W / 4; ++i) {
                const uint4 u = __ldcs(reinterpret_cast<const uint4*>(p) + i);
                r.w[4 * i] = u.x;
                r.w[4 * i + 1] = u.y;
                r.w[4 * i + 2] = u.z;
                r.w[4 * i + 3] = u.w;
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < kN; ++i) {
            const T* q = p + (i < 4 ? 0 : second) + (i & 3) * 32;
            if ((i & 3) * 32 < (i < 4 ? n : n2)) {
                if (sizeof(T) == 4) r.w[i % W] = __ldcs(reinterpret_cast<const uint32_t*>(q));
                else r.w[i / 2] |= (uint32_t)__ldcs(reinterpret_cast<const unsigned short*>(q)) << (16 * (i & 1));
            }
        }
    }
    return r;
}

template <typename T>
__device__ __forceinline__ void widen_raw(const Raw<T>& r, float (&v)[kN]) {
    const T* t = reinterpret_cast<const T*>(r.w);
#pragma unroll
    for (int i = 0; i < kN; ++i) v[i] = widen(t[i]);
}

// Two e4m3 values, a in the low byte: nearest, ties to even, up to 448, NaN kept.
__device__ __forceinline__ uint32_t e4m3_pair(float a, float b) {
    unsigned short r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(b), "f"(a));
    return r;
}

template <bool kWhole>
__device__ __forceinline__ void store_fp8(uint8_t* p, int n, long long second, int n2, const float (&v)[kN]) {
    const uint32_t lo = e4m3_pair(v[0], v[1]) | (e4m3_pair(v[2], v[3]) << 16);
    const uint32_t hi = e4m3_pair(v[4], v[5]) | (e4m3_pair(v[6], v[7]) << 16);
    if (kWhole) {
        if (n > 0) __stcs(reinterpret_cast<uint2*>(p), make_uint2(lo, hi));
    } else {
#pragma unroll
        for (int i = 0; i < kN; ++i)
            if ((i & 3) * 32 < (i < 4 ? n : n2))
                p[(i < 4 ? 0 : second) + (i & 3) * 32] = (uint8_t)((i < 4 ? lo : hi) >> (8 * (i & 3)));
    }
}

// Largest magnitude as bits (NaN > infinity > every finite value): of eight fp32
// numbers, and of eight elements as they are in memory, where two 16-bit ones
// are compared at once, accumulated into m and turned into fp32 bits at the end.
__device__ __forceinline__ uint32_t abs_max_bits(const float (&v)[kN], int first, int n) {
    uint32_t m = 0u;
#pragma unroll
    for (int i = 0; i < kN; ++i)
        if (i >= first && i < first + n) m = max(m, __float_as_uint(v[i]) & 0x7FFFFFFFu);
    return m;
}
template <typename T>
__device__ __forceinline__ uint32_t raw_abs_max(uint32_t m, const Raw<T>& r, int first, int n) {
    constexpr int W = kN * (int)sizeof(T) / 4;
#pragma unroll
    for (int i = 0; i < W; ++i) {
        if (i < first * W / kN || i >= (first + n) * W / kN) continue;
        if (sizeof(T) == 4) m = max(m, r.w[i] & 0x7FFFFFFFu);
        else m = __vmaxu2(m, r.w[i] & 0x7FFF7FFFu);
    }
    return m;
}
template <typename T>
__device__ __forceinline__ uint32_t magnitude_bits(uint32_t m) {
    if constexpr (sizeof(T) == 4) {
        return m;
    } else {
        const unsigned short h = (unsigned short)max(m & 0xFFFFu, m >> 16);
        return __float_as_uint(widen(*reinterpret_cast<const T*>(&h)));
    }
}
// Largest of `m` in each half of the warp, the lanes of a block.
__device__ __forceinline__ uint32_t half_warp_max(uint32_t m) {
    const bool low = (threadIdx.x & 16) == 0;
    const uint32_t a = __reduce_max_sync(kFullMask, low ? m : 0u), b = __reduce_max_sync(kFullMask, low ? 0u : m);
    return low ? a : b;
}

// RN(amax / 448) by the reciprocal and one FMA correction, which is the correctly
// rounded quotient while nothing leaves the normal range (P. Markstein,
// "Computation of elementary functions on the IBM RISC System/6000 processor",
// IBM J. Res. Dev. 34(1), 1990).
__device__ __forceinline__ float block_scale(uint32_t amax_bits) {
    if (amax_bits >= 0x7F800000u) return __uint_as_float(0x7FFFFFFFu);
    const float a = __uint_as_float(amax_bits);
    if (a < 0x1p-60f) return fmaxf(__fdiv_rn(a, kFp8Max), 0x1p-126f);
    const float q = __fmul_rn(a, 1.0f / kFp8Max);
    return __fmaf_rn(__fmaf_rn(-q, kFp8Max, a), 1.0f / kFp8Max, q);
}

// v[i] = RN(v[i] / s) in the same way.  With s in [2^-60, 2^60] no intermediate of
// a v above 2^-12 s leaves the normal range, and a smaller v gives 0 either way
// (half the smallest e4m3 value is 2^-10).
__device__ __forceinline__ void divide_by_scale(float (&v)[kN], float s, int first, int n) {
    if (s < 0x1p-60f || s > 0x1p60f) {  // both by the same power of two, into the range
        const float f = s < 1.0f ? 0x1p80f : 0x1p-80f;
        s *= f;
#pragma unroll
        for (int i = 0; i < kN; ++i)
            if (i >= first && i < first + n) v[i] *= f;
    }
    const float r = __frcp_rn(s);
#pragma unroll
    for (int i = 0; i < kN; ++i)
        if (i >= first && i < first + n) {
            const float q = __fmul_rn(v[i], r);
            v[i] = __fmaf_rn(__fmaf_rn(-q, s, v[i]), r, q);
        }
}

// One row's 1 x 128 blocks: divides a lane's eight values by their blocks' scales,
// of which the largest magnitudes (m of the first four or of all eight, m2 of the
// last four) are this lane's, and writes the scales; `block` is the first block
// that the lane has a part of, `there` and `there2` say whether it and the next exist.
template <bool kWhole>
__device__ __forceinline__ void scale_blocks(float (&v)[kN], uint32_t m, uint32_t m2, float* scale, bool there,
                                             bool there2) {
    const int lane = threadIdx.x & 31;
    if (kWhole) {
        const float s = block_scale(half_warp_max(m));
        divide_by_scale(v, s, 0, kN);
        if (lane % kG == 0 && there) *scale = s;
    } else {
        const float s = block_scale(__reduce_max_sync(kFullMask, m)), s2 = block_scale(__reduce_max_sync(kFullMask, m2));
        divide_by_scale(v, s, 0, 4);
        divide_by_scale(v, s2, 4, 4);
        if (lane == 0 && there) scale[0] = s;
        if (lane == 0 && there2) scale[1] = s2;
    }
}
// Column of a lane's first element in the 256 columns of a warp.
template <bool kWhole>
__device__ __forceinline__ int lane_column() {
    return (int)(threadIdx.x & 31) * (kWhole ? kN : 1);
}

// ---- activations: 1 x 128 blocks -------------------------------------------------
// A warp takes kUnits * 256 consecutive columns of a row at a time.
template <typename T, bool kWhole>
__global__ void __launch_bounds__(kQThreads)
    quantize_rows_kernel(const T* x, long long ld, unsigned items, unsigned segs, int dim, uint8_t* q, float* scales) {
    constexpr int kUnits = sizeof(T) == 4 ? 2 : 4;
    const int nb = (dim + kQBlock - 1) / kQBlock;
    for (unsigned it = blockIdx.x * (kQThreads / 32) + (threadIdx.x >> 5); it < items; it += gridDim.x * (kQThreads / 32)) {
        const unsigned row = it / segs;
        const int col = (int)(it - row * segs) * (kUnits * 32 * kN) + lane_column<kWhole>();
        const T* xp = x + (long long)row * ld + col;
        uint8_t* qp = q + (long long)row * dim + col;
        Raw<T> raw[kUnits];
#pragma unroll
        for (int k = 0; k < kUnits; ++k) {
            const int n = dim - col - k * 32 * kN;
            raw[k] = load_raw<T, kWhole>(xp + k * 32 * kN, n, kQBlock, n - kQBlock);
        }
#pragma unroll
        for (int k = 0; k < kUnits; ++k) {
            const int c = col + k * 32 * kN, n = dim - c;
            float v[kN];
            widen_raw(raw[k], v);
            const uint32_t m = magnitude_bits<T>(raw_abs_max(0u, raw[k], 0, kWhole ? kN : 4));
            const uint32_t m2 = kWhole ? 0u : magnitude_bits<T>(raw_abs_max(0u, raw[k], 4, 4));
            scale_blocks<kWhole>(v, m, m2, scales + (long long)row * nb + c / kQBlock, n > 0, n > kQBlock);
            store_fp8<kWhole>(qp + k * 32 * kN, n, kQBlock, n - kQBlock, v);
        }
    }
}

// ---- weights: 128 x 128 blocks ----------------------------------------------------
// One CTA a block, which it holds in registers as it was loaded between the
// maximum and the division.
template <typename T, bool kWhole>
__global__ void __launch_bounds__(kQThreads, sizeof(T) == 4 ? 2 : 4)
    quantize_blocks_kernel(const T* x, long long ld, int rows, int dim, uint8_t* q, float* scales) {
    // rows of one step: 16 lanes a row, or a warp for a row and the one 8 below
    constexpr int kRowsPer = kQThreads / kG;
    constexpr int kSteps = kQBlock / kRowsPer;
    __shared__ uint32_t red[kQThreads / 32];
    const int nb = (dim + kQBlock - 1) / kQBlock;
    const int br = blockIdx.x / nb, bc = blockIdx.x - br * nb;
    const int col = bc * kQBlock + (kWhole ? (int)(threadIdx.x % kG) * kN : (int)(threadIdx.x & 31));
    const int row0 = br * kQBlock + (int)threadIdx.x / (kWhole ? kG : 32);
    const T* xp = x + (long long)row0 * ld + col;
    uint8_t* qp = q + (long long)row0 * dim + col;
    const int cols = min(dim, (bc + 1) * kQBlock) - col;  // of this block from `col` on
    Raw<T> raw[kSteps];
    uint32_t m = 0u;
#pragma unroll
    for (int k = 0; k < kSteps; ++k) {
        const int row = row0 + k * kRowsPer;
        raw[k] = load_raw<T, kWhole>(xp + (long long)k * kRowsPer * ld, row < rows ? cols : 0, 8 * ld,
                                     row + 8 < rows ? cols : 0);
    }
#pragma unroll
    for (int k = 0; k < kSteps; ++k) m = raw_abs_max(m, raw[k], 0, kN);
    m = __reduce_max_sync(kFullMask, magnitude_bits<T>(m));
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = m;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kQThreads / 32; ++i) m = max(m, red[i]);
    const float s = block_scale(m);
    if (threadIdx.x == 0) scales[(long long)br * nb + bc] = s;
#pragma unroll
    for (int k = 0; k < kSteps; ++k) {
        const int row = row0 + k * kRowsPer;
        float v[kN];
        widen_raw(raw[k], v);
        divide_by_scale(v, s, 0, kN);
        store_fp8<kWhole>(qp + (long long)k * kRowsPer * dim, row < rows ? cols : 0, 8LL * dim, row + 8 < rows ? cols : 0, v);
    }
}

// ---- RMSNorm and quantisation -----------------------------------------------------
// v = weight * (x * r), r = 1 / sqrt(mean(x^2) + 1e-5), in fp32 as
// rmsnorm_bf16_kernel forms it, then the 1 x 128 blocks of v.  One CTA a row;
// the first kHeld groups of eight of a thread stay in registers between the sum
// and the division (kHeld by the width, all of a row up to 8192 wide), the rest
// is read again.
template <typename T, int kHeld, bool kWhole>
__global__ void __launch_bounds__(kQThreads, kHeld <= 2 ? 5 : 3)
    rmsnorm_fp8_kernel(const T* x, long long ld, const float* weight, int dim, uint8_t* q, float* scales) {
    constexpr int kSpan = kQThreads * kN;  // elements of one step of the CTA
    __shared__ float red[kQThreads / 32];
    const int warp_j0 = (int)(threadIdx.x >> 5) * 32 * kN, j0 = warp_j0 + lane_column<kWhole>();
    const int nb = (dim + kQBlock - 1) / kQBlock;
    const T* xr = x + (long long)blockIdx.x * ld + j0;
    uint8_t* qr = q + (long long)blockIdx.x * dim + j0;
    float* sr = scales + (long long)blockIdx.x * nb;
    Raw<T> raw[kHeld];
    float ss = 0.0f;
    const auto add_squares = [&](const Raw<T>& r) {
        float t[kN];
        widen_raw(r, t);
#pragma unroll
        for (int i = 0; i < kN; ++i) ss = __fmaf_rn(t[i], t[i], ss);
    };
#pragma unroll
    for (int k = 0; k < kHeld; ++k) {
        const int n = dim - j0 - k * kSpan;
        raw[k] = load_raw<T, kWhole>(xr + k * kSpan, n, kQBlock, n - kQBlock);
    }
#pragma unroll
    for (int k = 0; k < kHeld; ++k) add_squares(raw[k]);
    for (int j = kHeld * kSpan; j0 + j < dim; j += kSpan)
        add_squares(load_raw<T, kWhole>(xr + j, dim - j0 - j, kQBlock, dim - j0 - j - kQBlock));
#pragma unroll
    for (int o = 16; o; o >>= 1) ss += __shfl_xor_sync(kFullMask, ss, o);
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = ss;
    __syncthreads();
    float tot = 0.0f;
#pragma unroll
    for (int i = 0; i < kQThreads / 32; ++i) tot += red[i];
    const float r = __fdiv_rn(1.0f, __fsqrt_rn(__fadd_rn(__fdiv_rn(tot, (float)dim), 1e-5f)));
    const auto finish = [&](const Raw<T>& raw8, int j) {
        const int n = dim - j0 - j;  // columns from the lane's first one on
        float t[kN], w[kN];
        widen_raw(raw8, t);
        const float* wp = weight + j0 + j;
        if (kWhole) {
            float4 a = make_float4(0.0f, 0.0f, 0.0f, 0.0f), b = a;
            if (n > 0) {
                a = __ldg(reinterpret_cast<const float4*>(wp));
                b = __ldg(reinterpret_cast<const float4*>(wp) + 1);
            }
            w[0] = a.x, w[1] = a.y, w[2] = a.z, w[3] = a.w;
            w[4] = b.x, w[5] = b.y, w[6] = b.z, w[7] = b.w;
#pragma unroll
            for (int i = 0; i < kN; ++i) t[i] = __fmul_rn(w[i], __fmul_rn(r, t[i]));
            if (n <= 0) {  // a column past the row is 0 whatever r is
#pragma unroll
                for (int i = 0; i < kN; ++i) t[i] = 0.0f;
            }
        } else {
#pragma unroll
            for (int i = 0; i < kN; ++i) {
                const int at = (i & 3) * 32 + (i < 4 ? 0 : kQBlock);
                t[i] = at < n ? __fmul_rn(__ldg(wp + at), __fmul_rn(r, t[i])) : 0.0f;
            }
        }
        scale_blocks<kWhole>(t, abs_max_bits(t, 0, kWhole ? kN : 4), kWhole ? 0u : abs_max_bits(t, 4, 4),
                             sr + (j0 + j) / kQBlock, n > 0, n > kQBlock);
        store_fp8<kWhole>(qr + j, n, kQBlock, n - kQBlock, t);
    };
#pragma unroll
    for (int k = 0; k < kHeld; ++k)
        if (warp_j0 + k * kSpan < dim) finish(raw[k], k * kSpan);  // whole warps: the maximum needs every lane
    for (int j = kHeld * kSpan; warp_j0 + j < dim; j += kSpan) finish(load_raw<T, kWhole>(xr + j, dim - j0 - j, kQBlock, dim - j0 - j - kQBlock), j);
}

bool aligned(const void* p, unsigned n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

template <typename T, bool kWhole>
cudaError_t launch_quantize_t(const QuantLaunch& p, int num_sms, cudaStream_t stream) {
    const T* x = static_cast<const T*>(p.x);
    uint8_t* q = static_cast<uint8_t*>(p.q);
    if (p.norm_weight) {
        const auto launch = [&](auto kernel) {
            kernel<<<p.rows, kQThreads, 0, stream>>>(x, p.ld, p.norm_weight, p.dim, q, p.scales);
        };
        constexpr int kSpan = kQThreads * kN;
        if (p.dim <= kSpan) launch(rmsnorm_fp8_kernel<T, 1, kWhole>);
        else if (p.dim <= 2 * kSpan) launch(rmsnorm_fp8_kernel<T, 2, kWhole>);
        else launch(rmsnorm_fp8_kernel<T, 4, kWhole>);
    } else if (p.block_rows == 1) {
        constexpr int kCols = (sizeof(T) == 4 ? 2 : 4) * 32 * kN;
        const unsigned segs = (unsigned)(p.dim + kCols - 1) / kCols;
        const unsigned items = (unsigned)p.rows * segs;
        unsigned grid = (items + kQThreads / 32 - 1) / (kQThreads / 32);
        if (grid > 16u * num_sms) grid = 16u * num_sms;
        quantize_rows_kernel<T, kWhole><<<grid, kQThreads, 0, stream>>>(x, p.ld, items, segs, p.dim, q, p.scales);
    } else {
        const int grid = ((p.rows + kQBlock - 1) / kQBlock) * ((p.dim + kQBlock - 1) / kQBlock);
        quantize_blocks_kernel<T, kWhole><<<grid, kQThreads, 0, stream>>>(x, p.ld, p.rows, p.dim, q, p.scales);
    }
    return cudaGetLastError();
}

template <typename T>
cudaError_t launch_quantize_t(const QuantLaunch& p, int num_sms, cudaStream_t stream) {
    const bool whole = p.dim % kN == 0 && p.ld % (16 / (int)sizeof(T)) == 0 && aligned(p.x, 16) && aligned(p.q, 8) &&
                       aligned(p.norm_weight, 16);
    return whole ? launch_quantize_t<T, true>(p, num_sms, stream) : launch_quantize_t<T, false>(p, num_sms, stream);
}

}  // namespace

int launch_quantize_fp8(const QuantLaunch& p, int num_sms, cudaStream_t stream) {
    cudaError_t e = cudaErrorInvalidValue;
    if (p.dtype == kDtypeF32) e = launch_quantize_t<float>(p, num_sms, stream);
    else if (p.dtype == kDtypeBf16) e = launch_quantize_t<__nv_bfloat16>(p, num_sms, stream);
    else if (p.dtype == kDtypeF16) e = launch_quantize_t<__half>(p, num_sms, stream);
    return e == cudaSuccess ? 1 : -(int)e;
}

}  // namespace b2s
