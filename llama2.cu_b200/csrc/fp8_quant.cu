// fp8_quant.cu -- operands of the 8-bit classifier: float8 e4m3 values with
// one fp32 scale per block of 128 consecutive columns (activations: a block
// is 1 x 128; weights: 128 x 128), and the final RMSNorm that writes such
// rows in the same pass.
//
// Per block: amax = max |x|, s = max(RN(amax / 448), 2^-126), and
// q = RN_e4m3(RN(x / s)) (448 is the largest e4m3 value; ties to even).  The
// scale is rounded to fp32 before the division, so q * s is the nearest the
// format has to x under the scale that is stored.  The clamp gives a block of
// zeros a scale that can be divided by.  A block that holds a NaN or an
// infinity gets scale NaN and NaN values: whatever is computed from it shows.
//
// Both are bound by memory: an element is read once (4 or 2 bytes) and
// written once (1 byte); the division is a product with the rounded
// reciprocal and one FMA correction.
#include "device_common.cuh"
#include "fp8_filter_kernels.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

namespace b2s {
namespace {

constexpr int kQBlock = 128;
constexpr int kQThreads = 256;
constexpr float kFp8Max = 448.0f;

__device__ __forceinline__ float widen(float x) { return x; }
__device__ __forceinline__ float widen(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float widen(__half x) { return __half2float(x); }

// N consecutive elements from p (n of them exist, the rest read as 0).
template <typename T, int N>
__device__ __forceinline__ void load_elems(const T* p, int n, bool vec, float (&v)[N]) {
    if (vec && n >= N) {
        static_assert(sizeof(T) * N == 16, "16-byte loads");
        const uint4 u = *reinterpret_cast<const uint4*>(p);
        const T* t = reinterpret_cast<const T*>(&u);
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = widen(t[i]);
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = i < n ? widen(p[i]) : 0.0f;
    }
}

template <int N>
__device__ __forceinline__ void store_fp8(uint8_t* p, int n, bool vec, const float (&v)[N]) {
    uint32_t w[N / 4];
#pragma unroll
    for (int i = 0; i < N / 4; ++i) {
        const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(v[4 * i], v[4 * i + 1]), __NV_SATFINITE, __NV_E4M3);
        const uint32_t hi =
            __nv_cvt_float2_to_fp8x2(make_float2(v[4 * i + 2], v[4 * i + 3]), __NV_SATFINITE, __NV_E4M3);
        w[i] = lo | (hi << 16);
    }
    if (vec && n >= N) {
        if (N == 4) *reinterpret_cast<uint32_t*>(p) = w[0];
        else *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[N / 4 - 1]);
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (i < n) p[i] = (uint8_t)(w[i / 4] >> (8 * (i & 3)));
    }
}

// Largest magnitude as bits: NaN > infinity > every finite value.
template <int N>
__device__ __forceinline__ uint32_t abs_max_bits(const float (&v)[N]) {
    uint32_t m = 0u;
#pragma unroll
    for (int i = 0; i < N; ++i) m = max(m, __float_as_uint(v[i]) & 0x7FFFFFFFu);
    return m;
}

__device__ __forceinline__ float block_scale(uint32_t amax_bits) {
    if (amax_bits >= 0x7F800000u) return __uint_as_float(0x7FFFFFFFu);
    return fmaxf(__fdiv_rn(__uint_as_float(amax_bits), kFp8Max), 0x1p-126f);
}

// v[i] / s, correctly rounded where the result matters to e4m3: the product
// with r = RN(1/s) and one FMA correction (P. Markstein, "Computation of
// elementary functions on the IBM RISC System/6000 processor", IBM J. Res.
// Dev. 34(1), 1990).  With 2^-60 <= s <= 2^60 no intermediate of an x above
// 2^-12 s leaves the normal range, and a smaller x gives 0 either way (half
// the smallest e4m3 value is 2^-10).
template <int N>
__device__ __forceinline__ void divide_by_scale(float (&v)[N], float s) {
    if (s >= 0x1p-60f && s <= 0x1p60f) {
        const float r = __frcp_rn(s);
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const float q = __fmul_rn(v[i], r);
            v[i] = __fmaf_rn(__fmaf_rn(-q, s, v[i]), r, q);
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = __fdiv_rn(v[i], s);
    }
}

// ---- activations: 1 x 128 blocks -------------------------------------------------
// A block is one group of 128 / N lanes with 16 bytes of input each, so a warp
// holds one fp32 block or two 16-bit ones; kUnits blocks a group are in flight.
template <typename T>
__global__ void __launch_bounds__(kQThreads)
    quantize_rows_kernel(const T* x, long long ld, int rows, int dim, uint8_t* q, float* scales, int vec_in,
                         int vec_out) {
    constexpr int N = 16 / sizeof(T);
    constexpr int G = kQBlock / N;  // lanes of a block
    constexpr int kUnits = 4;
    const int nb = (dim + kQBlock - 1) / kQBlock;
    const long long units = (long long)rows * nb;
    const int gl = threadIdx.x % G;
    const long long groups = (long long)gridDim.x * (kQThreads / G);
    const long long first = (long long)blockIdx.x * (kQThreads / G) + threadIdx.x / G;
    for (long long u0 = first; u0 - first % (32 / G) < units; u0 += groups * kUnits) {  // whole warps stay together
        float v[kUnits][N];
        int n[kUnits], row[kUnits], blk[kUnits];
#pragma unroll
        for (int k = 0; k < kUnits; ++k) {
            const long long u = u0 + k * groups;
            row[k] = (int)(u / nb);
            blk[k] = (int)(u - (long long)row[k] * nb);
            n[k] = u < units ? min(N, dim - blk[k] * kQBlock - gl * N) : -1;
            load_elems<T, N>(x + (n[k] > 0 ? (long long)row[k] * ld + blk[k] * kQBlock + gl * N : 0), n[k], vec_in != 0,
                             v[k]);
        }
#pragma unroll
        for (int k = 0; k < kUnits; ++k) {
            uint32_t m = abs_max_bits(v[k]);
#pragma unroll
            for (int o = G / 2; o; o >>= 1) m = max(m, __shfl_xor_sync(kFullMask, m, o));
            const float s = block_scale(m);
            divide_by_scale(v[k], s);
            if (u0 + k * groups < units && gl == 0) scales[(long long)row[k] * nb + blk[k]] = s;
            if (n[k] > 0)
                store_fp8<N>(q + (long long)row[k] * dim + blk[k] * kQBlock + gl * N, n[k], vec_out != 0, v[k]);
        }
    }
}

// ---- weights: 128 x 128 blocks ----------------------------------------------------
// One CTA a block, which it holds in registers (64 elements a thread) between
// the maximum and the division.
template <typename T>
__global__ void __launch_bounds__(kQThreads)
    quantize_blocks_kernel(const T* x, long long ld, int rows, int dim, uint8_t* q, float* scales, int vec_in,
                           int vec_out) {
    constexpr int N = 16 / sizeof(T);
    constexpr int G = kQBlock / N;              // threads of a row
    constexpr int kRowsPer = kQThreads / G;     // rows of one step
    constexpr int kSteps = kQBlock / kRowsPer;
    __shared__ uint32_t red[kQThreads / 32];
    const int nb = (dim + kQBlock - 1) / kQBlock;
    const int br = blockIdx.x / nb, bc = blockIdx.x % nb;
    const int col = bc * kQBlock + (threadIdx.x % G) * N;
    const int row0 = br * kQBlock + threadIdx.x / G;
    float v[kSteps][N];
    uint32_t m = 0u;
#pragma unroll
    for (int k = 0; k < kSteps; ++k) {
        const int row = row0 + k * kRowsPer;
        const int n = row < rows ? min(N, dim - col) : -1;
        load_elems<T, N>(x + (n > 0 ? (long long)row * ld + col : 0), n, vec_in != 0, v[k]);
    }
#pragma unroll
    for (int k = 0; k < kSteps; ++k) m = max(m, abs_max_bits(v[k]));
#pragma unroll
    for (int o = 16; o; o >>= 1) m = max(m, __shfl_xor_sync(kFullMask, m, o));
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = m;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kQThreads / 32; ++i) m = max(m, red[i]);
    const float s = block_scale(m);
    if (threadIdx.x == 0) scales[(long long)br * nb + bc] = s;
#pragma unroll
    for (int k = 0; k < kSteps; ++k) {
        const int row = row0 + k * kRowsPer;
        const int n = row < rows ? min(N, dim - col) : -1;
        divide_by_scale(v[k], s);
        if (n > 0) store_fp8<N>(q + (long long)row * dim + col, n, vec_out != 0, v[k]);
    }
}

// ---- RMSNorm and quantisation -----------------------------------------------------
// v = weight * (x * r), r = 1 / sqrt(mean(x^2) + 1e-5), in fp32 as
// rmsnorm_bf16_kernel forms it, then the 1 x 128 blocks of v.  One CTA a row;
// the first kHeld groups of elements a thread meets stay in registers between
// the sum and the division (every row up to 8192 wide in fp32, 16384 in 16
// bits), the rest is read again.
template <typename T>
__global__ void __launch_bounds__(kQThreads)
    rmsnorm_fp8_kernel(const T* x, long long ld, const float* weight, int dim, uint8_t* q, float* scales, int vec_in,
                       int vec_out, int vec_w) {
    constexpr int N = 16 / sizeof(T);
    constexpr int G = kQBlock / N;
    constexpr int kHeld = 8;
    constexpr int kSpan = kQThreads * N;  // elements of one step of the CTA
    __shared__ float red[kQThreads / 32];
    const T* xr = x + (long long)blockIdx.x * ld;
    const int nb = (dim + kQBlock - 1) / kQBlock;
    float v[kHeld][N];
    float ss = 0.0f;
#pragma unroll
    for (int k = 0; k < kHeld; ++k) {
        const int j = k * kSpan + (int)threadIdx.x * N;
        load_elems<T, N>(xr + (j < dim ? j : 0), dim - j, vec_in != 0, v[k]);
    }
#pragma unroll
    for (int k = 0; k < kHeld; ++k)
#pragma unroll
        for (int i = 0; i < N; ++i) ss = __fmaf_rn(v[k][i], v[k][i], ss);
    for (int j = kHeld * kSpan + (int)threadIdx.x * N; j < dim; j += kSpan) {
        float t[N];
        load_elems<T, N>(xr + j, dim - j, vec_in != 0, t);
#pragma unroll
        for (int i = 0; i < N; ++i) ss = __fmaf_rn(t[i], t[i], ss);
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) ss += __shfl_xor_sync(kFullMask, ss, o);
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = ss;
    __syncthreads();
    float tot = 0.0f;
#pragma unroll
    for (int i = 0; i < kQThreads / 32; ++i) tot += red[i];
    const float r = __fdiv_rn(1.0f, __fsqrt_rn(__fadd_rn(__fdiv_rn(tot, (float)dim), 1e-5f)));
    uint8_t* qr = q + (long long)blockIdx.x * dim;
    float* sr = scales + (long long)blockIdx.x * nb;
    auto finish = [&](float (&t)[N], int j) {
        float w[N];
        if (vec_w && dim - j >= N) {
#pragma unroll
            for (int i = 0; i < N / 4; ++i) {
                const float4 f = __ldg(reinterpret_cast<const float4*>(weight + j) + i);
                w[4 * i] = f.x;
                w[4 * i + 1] = f.y;
                w[4 * i + 2] = f.z;
                w[4 * i + 3] = f.w;
            }
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i) w[i] = j + i < dim ? __ldg(weight + j + i) : 0.0f;
        }
#pragma unroll
        for (int i = 0; i < N; ++i) t[i] = __fmul_rn(w[i], __fmul_rn(r, t[i]));
        if (j + N > dim) {  // a column past the row is 0 whatever r is
#pragma unroll
            for (int i = 0; i < N; ++i)
                if (j + i >= dim) t[i] = 0.0f;
        }
        uint32_t m = abs_max_bits(t);
#pragma unroll
        for (int o = G / 2; o; o >>= 1) m = max(m, __shfl_xor_sync(kFullMask, m, o));
        const float s = block_scale(m);
        divide_by_scale(t, s);
        if (j < dim) {
            if (threadIdx.x % G == 0) sr[j / kQBlock] = s;
            store_fp8<N>(qr + j, dim - j, vec_out != 0, t);
        }
    };
#pragma unroll
    for (int k = 0; k < kHeld; ++k) {
        const int j = k * kSpan + (int)threadIdx.x * N;
        if (j - (int)(threadIdx.x & 31) * N < dim) finish(v[k], j);  // whole warps: the shuffles need every lane
    }
    for (int j = kHeld * kSpan + (int)threadIdx.x * N; j - (int)(threadIdx.x & 31) * N < dim; j += kSpan) {
        float t[N];
        load_elems<T, N>(xr + (j < dim ? j : 0), dim - j, vec_in != 0, t);
        finish(t, j);
    }
}

bool aligned(const void* p, unsigned n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

template <typename T>
cudaError_t launch_quantize_t(const QuantLaunch& p, int num_sms, cudaStream_t stream) {
    constexpr int N = 16 / sizeof(T);
    const T* x = static_cast<const T*>(p.x);
    uint8_t* q = static_cast<uint8_t*>(p.q);
    const int vec_in = aligned(x, 16) && p.ld % N == 0;
    const int vec_out = aligned(q, N) && p.dim % N == 0;
    const int nb = (p.dim + kQBlock - 1) / kQBlock;
    if (p.norm_weight) {
        rmsnorm_fp8_kernel<T><<<p.rows, kQThreads, 0, stream>>>(x, p.ld, p.norm_weight, p.dim, q, p.scales, vec_in,
                                                                vec_out, aligned(p.norm_weight, 16));
    } else if (p.block_rows == 1) {
        const long long units = (long long)p.rows * nb;
        const long long per_cta = kQThreads / (kQBlock / N);
        long long grid = (units + per_cta - 1) / per_cta;
        if (grid > 8LL * num_sms) grid = 8LL * num_sms;
        quantize_rows_kernel<T><<<(int)grid, kQThreads, 0, stream>>>(x, p.ld, p.rows, p.dim, q, p.scales, vec_in,
                                                                     vec_out);
    } else {
        const int grid = ((p.rows + kQBlock - 1) / kQBlock) * nb;
        quantize_blocks_kernel<T><<<grid, kQThreads, 0, stream>>>(x, p.ld, p.rows, p.dim, q, p.scales, vec_in, vec_out);
    }
    return cudaGetLastError();
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
