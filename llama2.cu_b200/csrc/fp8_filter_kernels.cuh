// fp8_filter_kernels.cuh -- launch interface of the filtered sampler and of the
// 8-bit classifier's kernels.  The launch functions return the number of
// kernels launched (>= 1) or a negative cudaError_t.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

namespace b2s {

// Element types of the 16- and 32-bit inputs (mirrors of the public SAMPLER_DTYPE_* values).
constexpr int kDtypeF32 = 0, kDtypeBf16 = 1, kDtypeF16 = 2;

// What the product writes for a logit that it did not finish because a device wait ran
// out: a NaN of a payload that no arithmetic has (instructions give 0x7FFFFFFF and 0x7FFF).
constexpr uint32_t kUnfinishedF32 = 0xFFC0BAD0u;
constexpr uint16_t kUnfinishedBf16 = 0xFFDAu;

// float8 e4m3 values and fp32 scales of blocks of 128 columns (fp8_quant.cu).
struct QuantLaunch {
    const void* x;             // [rows, ld], dtype
    int dtype;
    long long ld;
    int rows;
    int dim;
    int block_rows;            // 1 or 128
    const float* norm_weight;  // [dim]: RMSNorm first (block_rows 1), or nullptr
    void* q;                   // e4m3 [rows, dim]
    float* scales;             // [ceil(rows / block_rows), ceil(dim / 128)]
};

// logits[B, V] = H[B, D] . W[V, D]^T from e4m3 operands with a scale per 1 x 128
// block of H and per 128 x 128 block of W (fp8_gemm.cu).
struct Fp8GemmLaunch {
    const void* h;          // e4m3 [batch, dim]
    const float* h_scales;  // [batch, ceil(dim / 128)]
    const void* w;          // e4m3 [vocab, dim]
    const float* w_scales;  // [ceil(vocab / 128), ceil(dim / 128)]
    int batch;
    int dim;                // multiple of 16
    int vocab;
    void* logits;           // fp32 or bf16 [batch, ld]
    int out_bf16;
    long long ld;
    int* error_word;
    unsigned wait_test;     // self-test: no products are issued, waits run out after so many polls; else 0
    int box_rows;           // set by the launch: rows of H that a tile loads
    int vec_out;            // set by the launch: rows of logits start on 16-byte boundaries
};

// Sampling by temperature, top-k, top-p and min-p (filtered_sample.cu).
struct FilterLaunch {
    const void* logits;  // [batch, ld], dtype
    int dtype;
    int from_product;    // the logits are the 8-bit product's, which marks what it did not finish
    long long ld;
    int batch;
    int vocab;
    float temperature, topp, minp;  // when the per-row array is nullptr
    int topk;
    const float* temperature_rows;
    const int* topk_rows;
    const float* topp_rows;
    const float* minp_rows;
    const float* coins;              // given coins, or nullptr: drawn from rng_state
    unsigned long long* rng_state;
    int* out_ids;
    float* logprobs;                 // optional [batch]
    int* kept;                       // optional [batch]
    int* row_flags;                  // optional [batch]
};

int launch_quantize_fp8(const QuantLaunch& p, int num_sms, cudaStream_t stream);
int launch_fp8_gemm(const Fp8GemmLaunch& p, int num_sms, cudaStream_t stream);
int launch_filtered_sample(const FilterLaunch& p, int num_sms, cudaStream_t stream);

}  // namespace b2s
