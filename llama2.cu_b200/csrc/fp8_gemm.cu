// fp8_gemm.cu -- the classifier projection from 8-bit operands:
//   logits[b, v] = sum over blocks g of 128 columns
//                  hs[b, g] * ws[v / 128, g] * sum_{k in g} hq[b, k] * wq[v, k]
// hq, wq float8 e4m3, the scales fp32, on the 5th-generation tensor cores
// (tcgen05.mma kind::f8f6f4, fp32 accumulator in TMEM).
//
// The scales differ from block to block, so the tensor core sums one block of
// 128 at a time (four K = 32 instructions into a TMEM buffer of its own), and
// the fold warps add that buffer into fp32 registers with one FMA per element
// (two per instruction, fma.f32x2) while the tensor core works on the next block
// in the other buffer.  One persistent CTA per SM:
//   warp 0      TMA producer: operand boxes of 128 bytes by the tile's rows,
//               128-byte swizzle, into a ring of stages
//   warp 1      MMA issuer (one thread)
//   warp 2      TMEM allocation / release
//   warps 4..   fold: one TMEM lane a thread, 128 columns at most; at the end
//               of a tile they write the logits
// Large batches have H on the 128 TMEM lanes (its scale is the thread's own, W's
// one number per block: one FMA an element) and 256 columns of W, which two
// warpgroups fold; a thread then holds 128 sums, so the fold warps take registers
// over from the others (setmaxnreg).  They write through shared memory, 32 x 32
// logits a warp at a time, so that whole 128-byte lines go out.
// Small batches (kWLanes) have W on the lanes: NT is the padded batch, H's scales
// come from shared memory, and reading W is all that counts.  The rows of W are
// cut into tiles of equal height, at most 128, such that every SM gets the same
// number (32000 rows: 294 tiles of 109, two an SM, not 250 of 128).
// Every mbarrier wait is bounded; a timeout sets the error word and drains
// the pipeline.
#include "device_common.cuh"
#include "fp8_filter_kernels.cuh"
#include "tcgen05_common.cuh"

#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <atomic>

namespace b2s {
namespace {

constexpr int kFM = 128;      // TMEM lanes of a tile
constexpr int kFK = 128;      // K of a block, a stage and one accumulation
constexpr int kFABytes = kFM * kFK;
constexpr int kFGroupM = 16;  // row tiles swept together (L2 reuse of W)

template <int NT, bool kWLanes>
struct Fp8Cfg {
    static constexpr int kGroups = NT > 128 ? NT / 128 : 1;  // warpgroups of the fold
    static constexpr int kCols = NT / kGroups;               // columns a thread folds
    static constexpr int kThreads = 128 + 128 * kGroups;
    static constexpr int kBBytes = NT * kFK;
    static constexpr int kStages = (NT == 256) ? 4 : (NT >= 64 ? 6 : 8);
    static constexpr bool kStaged = !kWLanes;                // logits leave through shared memory
    static constexpr int kStageOut = kStaged ? 4 * kGroups * 32 * 32 : 1;
    static constexpr int kTmemCols = 2 * NT < 32 ? 32 : 2 * NT;
    // Instruction descriptor, kind::f8f6f4: fp32 accumulator (bits 4-5 = 1), A and B e4m3 (bits 7-9,
    // 10-12 = 0), both K-major (bits 15, 16 = 0), N >> 3 in bits 17-22, M >> 4 in bits 24-28.
    static constexpr uint32_t kIdesc = (1u << 4) | ((uint32_t)(NT >> 3) << 17) | ((uint32_t)(kFM >> 4) << 24);
};

template <int kStages>
struct Fp8Bars {
    unsigned long long full[kStages];
    unsigned long long empty[kStages];
    unsigned long long tmem_full[2];
    unsigned long long tmem_empty[2];
    unsigned long long drain;
    uint32_t tmem_base;
    int abort;
};

template <int NT, bool kWLanes>
struct Fp8Smem {
    using C = Fp8Cfg<NT, kWLanes>;
    uint8_t a[C::kStages][kFABytes];  // 1024-byte aligned (the swizzle atom)
    uint8_t b[C::kStages][C::kBBytes];
    float out[C::kStageOut];
    Fp8Bars<C::kStages> bar;
};

// D[tmem] (+)= A[smem] . B[smem]^T, kind::f8f6f4 (e4m3 inputs, fp32 accumulator)
__device__ __forceinline__ void tc_mma_fp8(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc,
                                           uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
        "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
        : "memory");
}

// 32 (16) consecutive fp32 columns of this thread's TMEM lane; the values are
// there after tmem_wait on them.
__device__ __forceinline__ void tmem_load(uint32_t taddr, uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, "
        "%14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
          "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
          "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr));
}
__device__ __forceinline__ void tmem_load(uint32_t taddr, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, "
        "%14, %15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr));
}
// Waits for this thread's TMEM loads; the values pass through, so that no use of
// them can be moved before it.
__device__ __forceinline__ void tmem_wait(uint32_t (&r)[16]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                   "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])
                 :
                 : "memory");
}
__device__ __forceinline__ void tmem_wait(uint32_t (&r)[32]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                   "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]),
                   "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]),
                   "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]),
                   "+r"(r[30]), "+r"(r[31])
                 :
                 : "memory");
}

// acc[0], acc[1] += t0 * f0, t1 * f1
__device__ __forceinline__ void fold2(unsigned long long& acc, uint32_t t0, uint32_t t1, unsigned long long f) {
    asm("{\n\t.reg .b64 t;\n\tmov.b64 t, {%1, %2};\n\tfma.rn.f32x2 %0, t, %3, %0;\n\t}"
        : "+l"(acc)
        : "r"(t0), "r"(t1), "l"(f));
}
__device__ __forceinline__ unsigned long long pair_of(float a, float b) {
    unsigned long long r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float2 halves_of(unsigned long long v) {
    float2 f;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(f.x), "=f"(f.y) : "l"(v));
    return f;
}

template <class Bars>
__device__ __forceinline__ bool fp8_aborted(const Bars& b) {
    return *(const volatile int*)&b.abort != 0;
}
template <class Bars>
__device__ __forceinline__ bool fp8_wait(unsigned long long* bar, unsigned parity, Bars& b, int* error_word) {
    if (mbar_wait_bounded(bar, parity)) return true;
    b.abort = 1;
    atomicOr(error_word, 2);
    return false;
}

__device__ __forceinline__ void store_logit(const Fp8GemmLaunch& p, long long at, float v) {
    if (p.out_bf16) static_cast<__nv_bfloat16*>(p.logits)[at] = __float2bfloat16_rn(v);
    else static_cast<float*>(p.logits)[at] = v;
}

// 32 x 32 logits from the warp's shared memory: rows row0 .., columns col0 ...
// Whole 16-byte pieces where the rows allow it, else 32 columns of a row at a time.
__device__ __forceinline__ void write_block(const Fp8GemmLaunch& p, const float* out, int row0, int col0, int lane) {
    const float4* out4 = reinterpret_cast<const float4*>(out);
    if (p.vec_out && col0 + 32 <= p.vocab) {
        if (p.out_bf16) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int r = i * 8 + lane / 4, j = 2 * (lane & 3);
                const float4 a = out4[r * 8 + (j ^ (r & 7))], b = out4[r * 8 + ((j + 1) ^ (r & 7))];
                const __nv_bfloat162 w[4] = {__floats2bfloat162_rn(a.x, a.y), __floats2bfloat162_rn(a.z, a.w),
                                             __floats2bfloat162_rn(b.x, b.y), __floats2bfloat162_rn(b.z, b.w)};
                if (row0 + r < p.batch)
                    *reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(p.logits) + (long long)(row0 + r) * p.ld + col0 +
                                              8 * (lane & 3)) = *reinterpret_cast<const uint4*>(w);
            }
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int r = i * 4 + lane / 8, j = lane & 7;
                const float4 a = out4[r * 8 + (j ^ (r & 7))];
                if (row0 + r < p.batch)
                    *reinterpret_cast<float4*>(static_cast<float*>(p.logits) + (long long)(row0 + r) * p.ld + col0 + 4 * j) = a;
            }
        }
    } else if (col0 + lane < p.vocab) {
#pragma unroll 4
        for (int r = 0; r < 32; ++r)
            if (row0 + r < p.batch)
                store_logit(p, (long long)(row0 + r) * p.ld + col0 + lane, out[r * 32 + (((lane / 4) ^ (r & 7)) << 2) + (lane & 3)]);
    }
}

template <int NT, bool kWLanes>
__global__ void __launch_bounds__(Fp8Cfg<NT, kWLanes>::kThreads, 1)
    fp8_gemm_kernel(const __grid_constant__ CUtensorMap tmap_a, const __grid_constant__ CUtensorMap tmap_b,
                    Fp8GemmLaunch p) {
    using C = Fp8Cfg<NT, kWLanes>;
    extern __shared__ __align__(16) unsigned char fsm_raw[];
    Fp8Smem<NT, kWLanes>& sm =
        *reinterpret_cast<Fp8Smem<NT, kWLanes>*>((reinterpret_cast<uintptr_t>(fsm_raw) + 1023) & ~(uintptr_t)1023);
    auto& bar = sm.bar;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int rows_a = kWLanes ? p.vocab : p.batch, rows_b = kWLanes ? p.batch : p.vocab;
    const int mt = (rows_a + p.tile_rows - 1) / p.tile_rows;  // tile_rows: 128, or fewer rows of W
    const int nt = (rows_b + NT - 1) / NT;
    const int ntiles = mt * nt;
    const int nk = (p.dim + kFK - 1) / kFK;

    if (tid == 0) {
        for (int s = 0; s < C::kStages; ++s) {
            mbar_init(&bar.full[s], 1);
            mbar_init(&bar.empty[s], 1);
        }
        for (int a = 0; a < 2; ++a) {
            mbar_init(&bar.tmem_full[a], 1);
            mbar_init(&bar.tmem_empty[a], 4 * C::kGroups);  // one arrival per fold warp
        }
        mbar_init(&bar.drain, 1);
        bar.abort = 0;
        fence_mbar_init();
    }
    if (warp == 2) {
        tmem_alloc(smem_addr(&bar.tmem_base), C::kTmemCols);
        tmem_relinquish();
    }
    // small batches: H's scales, transposed to [block][row], behind the ring
    float* hs_sm = reinterpret_cast<float*>(&sm + 1);
    if (kWLanes) {
        for (int i = tid; i < nk * NT; i += C::kThreads) {
            const int b = i % NT, g = i / NT;
            hs_sm[i] = b < p.batch ? p.h_scales[(long long)b * nk + g] : 0.0f;
        }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = bar.tmem_base;

    auto coords = [&](int tile, int& mb, int& nb) {
        const int per_group = kFGroupM * nt;
        const int g = tile / per_group;
        const int r = tile - g * per_group;
        const int gm = min(kFGroupM, mt - g * kFGroupM);
        nb = r / gm;
        mb = g * kFGroupM + (r - nb * gm);
    };

    // 384 threads at 168 registers: the two fold warpgroups take 208, the other 88
    if (warp < 4) {
    if (C::kGroups == 2) asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
    if (warp == 0 && lane == 0) {
        // ---- TMA producer
        int stage = 0;
        unsigned phase = 0;
        for (int tile = blockIdx.x; tile < ntiles && !fp8_aborted(bar); tile += gridDim.x) {
            int mb, nb;
            coords(tile, mb, nb);
            for (int k = 0; k < nk; ++k) {
                if (!fp8_wait(&bar.empty[stage], phase ^ 1u, bar, p.error_word)) break;
                mbar_arrive_expect_tx(&bar.full[stage], p.tile_rows * kFK + C::kBBytes);
                tma_load_2d(sm.a[stage], &tmap_a, k * kFK, mb * p.tile_rows, &bar.full[stage]);
                tma_load_2d(sm.b[stage], &tmap_b, k * kFK, nb * NT, &bar.full[stage]);
                if (++stage == C::kStages) {
                    stage = 0;
                    phase ^= 1u;
                }
            }
        }
        // drain: every stage this thread filled completes before the CTA exits
        for (int s = 0; s < C::kStages; ++s) {
            if (!mbar_wait_bounded(&bar.empty[stage], phase ^ 1u)) break;
            if (++stage == C::kStages) {
                stage = 0;
                phase ^= 1u;
            }
        }
    } else if (warp == 1 && lane == 0) {
        // ---- MMA issuer: one accumulation of its own for every block of 128
        int stage = 0;
        unsigned phase = 0;
        unsigned it = 0;
        bool ok = true;
        for (int tile = blockIdx.x; tile < ntiles && ok && !fp8_aborted(bar); tile += gridDim.x) {
            for (int k = 0; k < nk; ++k, ++it) {
                const unsigned buf = it & 1u;
                if (!fp8_wait(&bar.tmem_empty[buf], ((it >> 1) & 1u) ^ 1u, bar, p.error_word) ||
                    !fp8_wait(&bar.full[stage], phase, bar, p.error_word)) {
                    ok = false;
                    break;
                }
                tc_fence_after();
                const uint32_t a0 = smem_addr(sm.a[stage]), b0 = smem_addr(sm.b[stage]);
#pragma unroll
                for (int kk = 0; kk < kFK / 32; ++kk)  // 32 e4m3 = 32 bytes inside the swizzled 128-byte row
                    tc_mma_fp8(tmem + buf * NT, smem_desc_sw128(a0 + kk * 32), smem_desc_sw128(b0 + kk * 32),
                               C::kIdesc, kk != 0 ? 1u : 0u);
                tc_commit(&bar.empty[stage]);
                tc_commit(&bar.tmem_full[buf]);
                if (++stage == C::kStages) {
                    stage = 0;
                    phase ^= 1u;
                }
            }
        }
        // every MMA this thread issued is complete before TMEM is released
        tc_commit(&bar.drain);
        mbar_wait_bounded(&bar.drain, 0);
    }
    } else {
        if (C::kGroups == 2) asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
        // ---- fold: warp w reads TMEM lanes 32 * (w % 4) .. +31
        const int q = warp & 3;
        const int col0 = ((warp - 4) >> 2) * C::kCols;
        constexpr int kPart = C::kCols >= 64 ? 32 : 16;             // columns of one TMEM load
        constexpr int kTwo = C::kCols >= 2 * kPart ? 2 : 1;         // loads in flight
        float* const out = sm.out + (C::kStaged ? (warp - 4) * 1024 : 0);
        unsigned it = 0;
        bool ok = true;
        for (int tile = blockIdx.x; tile < ntiles && ok; tile += gridDim.x) {
            int mb, nb;
            coords(tile, mb, nb);
            const int in_tile = q * 32 + lane;
            const int row = mb * p.tile_rows + in_tile;  // row of the operand on the lanes
            const bool row_ok = in_tile < p.tile_rows && row < rows_a;
            unsigned long long acc[C::kCols / 2];
#pragma unroll
            for (int j = 0; j < C::kCols / 2; ++j) acc[j] = 0ull;
            const int wcol = nb * NT + col0;  // first of this thread's columns (of W, when W is not on the lanes)
            const float* own_scale = kWLanes ? p.w_scales + (long long)(row / kFK) * nk : p.h_scales + (long long)row * nk;
            const float* tile_scale = p.w_scales + (long long)(wcol / kFK) * nk;
            const bool col_ok = kWLanes || wcol < p.vocab;
            const auto scale_of = [&](int k) {
                float s = row_ok && col_ok ? __ldg(own_scale + k) : 0.0f;
                if (!kWLanes && row_ok && col_ok) s *= __ldg(tile_scale + k);
                return s;
            };
            float s = scale_of(0);
            for (int k = 0; k < nk; ++k, ++it) {
                const unsigned buf = it & 1u;
                const float s_next = k + 1 < nk ? scale_of(k + 1) : 0.0f;
                const bool got = fp8_wait(&bar.tmem_full[buf], (it >> 1) & 1u, bar, p.error_word);
                if (!__all_sync(kFullMask, got ? 1 : 0) || fp8_aborted(bar)) {
                    ok = false;
                    break;
                }
                tc_fence_after();
                const uint32_t src = tmem + ((uint32_t)(q * 32) << 16) + buf * NT + (uint32_t)col0;
                const unsigned long long ss = pair_of(s, s);
#pragma unroll
                for (int c = 0; c < C::kCols; c += kTwo * kPart) {
                    uint32_t t[kTwo][kPart];
#pragma unroll
                    for (int h = 0; h < kTwo; ++h) tmem_load(src + (uint32_t)(c + h * kPart), t[h]);
#pragma unroll
                    for (int h = 0; h < kTwo; ++h) tmem_wait(t[h]);
                    if (c + kTwo * kPart >= C::kCols) {  // the buffer has been read
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(&bar.tmem_empty[buf]);
                    }
#pragma unroll
                    for (int h = 0; h < kTwo; ++h)
#pragma unroll
                        for (int j = 0; j < kPart; j += 2) {
                            const int at = c + h * kPart + j;
                            unsigned long long f = ss;
                            if (kWLanes) {
                                const float2 hs = *reinterpret_cast<const float2*>(hs_sm + k * NT + at);
                                f = pair_of(s * hs.x, s * hs.y);
                            }
                            fold2(acc[at / 2], t[h][j], t[h][j + 1], f);
                        }
                }
                s = s_next;
            }
            ok = __all_sync(kFullMask, ok ? 1 : 0);
            if (!ok) break;
            if (kWLanes) {  // a lane per vocabulary entry: 32 consecutive logits of a row per store
#pragma unroll
                for (int j = 0; j < C::kCols; ++j) {
                    const int b = nb * NT + j;
                    const float2 v = halves_of(acc[j / 2]);
                    if (row_ok && b < p.batch) store_logit(p, (long long)b * p.ld + row, (j & 1) ? v.y : v.x);
                }
            } else {
                // 32 columns at a time through the warp's 32 x 32 floats; the 16-byte piece j of
                // row r is at piece j ^ (r % 8), so neither side meets bank conflicts
                float4* const out4 = reinterpret_cast<float4*>(out);
                const int row0 = row - lane;
#pragma unroll
                for (int c = 0; c < C::kCols; c += 32) {
                    __syncwarp();
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        const float2 a = halves_of(acc[c / 2 + 2 * j]), b = halves_of(acc[c / 2 + 2 * j + 1]);
                        out4[lane * 8 + (j ^ (lane & 7))] = make_float4(a.x, a.y, b.x, b.y);
                    }
                    __syncwarp();
                    write_block(p, out, row0, wcol + c, lane);
                }
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 2) {
        tc_fence_after();
        tmem_dealloc(tmem, C::kTmemCols);
    }
}

// 2-D e4m3 K-major tensor [rows, dim], box [box_rows, 128].
bool make_tmap_fp8(CUtensorMap* m, const void* base, int rows, int dim, int box_rows) {
    EncodeTiledFn enc = get_encode_fn();
    if (!enc) return false;
    const cuuint64_t dims[2] = {(cuuint64_t)dim, (cuuint64_t)rows};
    const cuuint64_t strides[1] = {(cuuint64_t)dim};
    const cuuint32_t box[2] = {(cuuint32_t)kFK, (cuuint32_t)box_rows};
    const cuuint32_t estr[2] = {1, 1};
    return enc(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, estr,
               CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
               CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int NT, bool kWLanes>
cudaError_t launch_fp8(Fp8GemmLaunch p, int num_sms, cudaStream_t stream) {
    using C = Fp8Cfg<NT, kWLanes>;
    const void* a = kWLanes ? p.w : p.h;
    const void* b = kWLanes ? p.h : p.w;
    const int rows_a = kWLanes ? p.vocab : p.batch, rows_b = kWLanes ? p.batch : p.vocab;
    p.tile_rows = kFM;
    if (kWLanes) {  // as many tiles an SM as 128 rows each would take, of equal height
        const int rounds = (rows_a + kFM * num_sms - 1) / (kFM * num_sms);
        p.tile_rows = (rows_a + rounds * num_sms - 1) / (rounds * num_sms);
    }
    p.vec_out = (reinterpret_cast<uintptr_t>(p.logits) & 15u) == 0 && p.ld % (p.out_bf16 ? 8 : 4) == 0;
    CUtensorMap ta, tb;
    if (!make_tmap_fp8(&ta, a, rows_a, p.dim, p.tile_rows) || !make_tmap_fp8(&tb, b, rows_b, p.dim, NT))
        return cudaErrorInvalidValue;
    const int nk = (p.dim + kFK - 1) / kFK;
    const size_t smem = sizeof(Fp8Smem<NT, kWLanes>) + 1024 + (kWLanes ? (size_t)nk * NT * sizeof(float) : 0);
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    static std::atomic<unsigned long long> attr_done{0};
    const unsigned long long bit = 1ull << (dev & 63);
    if (!(attr_done.load() & bit)) {
        e = cudaFuncSetAttribute(fp8_gemm_kernel<NT, kWLanes>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                 kFp8MaxSmem);
        if (e != cudaSuccess) return e;
        attr_done.fetch_or(bit);
    }
    const long long tiles = (long long)((rows_a + p.tile_rows - 1) / p.tile_rows) * ((rows_b + NT - 1) / NT);
    const int grid = tiles < num_sms ? (int)tiles : num_sms;
    fp8_gemm_kernel<NT, kWLanes><<<grid, C::kThreads, smem, stream>>>(ta, tb, p);
    return cudaGetLastError();
}

}  // namespace

int launch_fp8_gemm(const Fp8GemmLaunch& p, int num_sms, cudaStream_t stream) {
    const int nk = (p.dim + kFK - 1) / kFK;
    cudaError_t e;
    // W on the lanes while the padded batch is one column tile and H's scales fit behind the ring.
    if (p.batch <= 16 && nk <= 512) e = launch_fp8<16, true>(p, num_sms, stream);
    else if (p.batch <= 32 && nk <= 256) e = launch_fp8<32, true>(p, num_sms, stream);
    else if (p.batch <= 64 && nk <= 128) e = launch_fp8<64, true>(p, num_sms, stream);
    else e = launch_fp8<256, false>(p, num_sms, stream);
    return e == cudaSuccess ? 1 : -(int)e;
}

}  // namespace b2s
