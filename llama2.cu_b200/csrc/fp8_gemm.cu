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
//               128-byte swizzle, into a ring of four stages
//   warp 1      MMA issuer (one thread)
//   warp 2      TMEM allocation / release
//   warps 4-11  fold: one row of H a thread, 128 columns (rows of W) a warpgroup;
//               at the end of a tile they write the logits
// H is on the 128 TMEM lanes whatever the batch is: an instruction costs its 128
// lanes' time anyway (about 97 ns with 16 columns, 130 with 256), so W on the
// lanes, which looks better for a single row, was slower there too (35 us for
// 1 x 4096 x 32000).  A tile has up to 256 columns, in 32s, chosen by the host so that
// the tiles fill the SMs evenly.  A fold thread holds 128 sums, so the fold warps
// take registers over from the others (setmaxnreg).  They write through shared
// memory, 32 x 32 logits a warp at a time, so that whole 128-byte lines go out.
//
// What bounds it: for large batches the way of a TMEM buffer from its last product
// to its next first one (commit, loads, release, issue: some 650 ns, of which the
// other buffer's product covers 520), for small ones two chains of about the same
// length: the stream of W, and its blocks one after the other in each SM (32 of 520 to
// 650 ns at 4096 wide), which the batch makes no longer.
// Measured (1 B200): 8192 x 4096 x 32000 1.45 ms under the power cap, 1.23 in runs too
// short to reach it (0.92 with one accumulation over all of K, which the scales do not
// allow); 1 x 4096 x 32000 28 us, 31 with new inputs each time, of which 20 are the bytes.
// Every mbarrier wait is bounded; a timeout sets the error word, fills the rest of the
// CTA's tiles with a NaN of its own and drains the pipeline.
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

constexpr int kFM = 128;      // rows of H in a tile (TMEM lanes)
constexpr int kFN = 256;      // columns of a tile, at most; the stride of the TMEM buffers
constexpr int kFK = 128;      // K of a block, a stage and one accumulation
constexpr int kFStages = 4;
constexpr int kFCols = kFN / 2;                 // columns a warpgroup folds
constexpr int kFThreads = 128 + 2 * 128;
constexpr int kFABytes = kFM * kFK;
constexpr int kFBBytes = kFN * kFK;
constexpr int kFTmemCols = 2 * kFN;
constexpr int kFGroupM = 16;  // row tiles swept together (L2 reuse of W)

struct Fp8Smem {
    uint8_t a[kFStages][kFABytes];  // 1024-byte aligned (the swizzle atom)
    uint8_t b[kFStages][kFBBytes];
    float out[8][32 * 32];          // by fold warp
    unsigned long long full[kFStages];
    unsigned long long empty[kFStages];
    unsigned long long tmem_full[2];
    unsigned long long tmem_empty[2];
    unsigned long long drain;
    uint32_t tmem_base;
    int abort;
};
constexpr size_t kFp8SmemBytes = sizeof(Fp8Smem) + 1024;  // + alignment slack
static_assert(kFp8SmemBytes <= 227 * 1024, "one CTA's shared memory");

// D[tmem] (+)= A[smem] . B[smem]^T, kind::f8f6f4 (e4m3 inputs, fp32 accumulator)
__device__ __forceinline__ void tc_mma_fp8(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc,
                                           bool accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
        "l"(adesc), "l"(bdesc), "r"(idesc), "r"((uint32_t)accumulate)
        : "memory");
}

// 32 consecutive fp32 columns of this thread's TMEM lane; the values are there
// after tmem_wait on them.
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
// Waits for this thread's TMEM loads; the values pass through, so that no use of
// them can be moved before it.
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

__device__ __forceinline__ bool fp8_aborted(const Fp8Smem& sm) { return *(const volatile int*)&sm.abort != 0; }
// Bounded wait, inline: one thread issues all products and one all copies, and
// every instruction of their loops is on a block's way.
__device__ __forceinline__ bool fp8_wait(unsigned long long* bar, unsigned parity, Fp8Smem& sm, int* error_word,
                                         unsigned limit) {
    for (unsigned i = 0; i < limit; ++i)
        if (mbar_try_wait(bar, parity)) return true;
    sm.abort = 1;
    atomicOr(error_word, 2);
    return false;
}

// A warp's 32 rows of `out`, 128 bytes each (32 fp32 or 64 bf16 logits, the 16-byte
// piece j of row r at piece j ^ (r % 8)), to rows row0 .. and the n columns from
// col0 on.  Whole 16-byte pieces where the rows allow it; else a row at a time, bf16
// in pairs that start on 4 bytes.
template <typename T>
__device__ __forceinline__ void write_block(const Fp8GemmLaunch& p, const T* out, int row0, int col0, int n, int lane) {
    constexpr int kPer = 16 / sizeof(T);  // elements of a piece
    const uint4* out4 = reinterpret_cast<const uint4*>(out);
    T* const to = static_cast<T*>(p.logits) + (long long)row0 * p.ld + col0;
    const int rows = min(32, p.batch - row0);
    const auto at = [&](int r, int c) { return out[r * 8 * kPer + (((c / kPer) ^ (r & 7)) * kPer) + c % kPer]; };
    if (p.vec_out && n % kPer == 0) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int r = i * 4 + lane / 8, j = lane & 7;
            if (r < rows && j * kPer < n) *reinterpret_cast<uint4*>(to + r * p.ld + j * kPer) = out4[r * 8 + (j ^ (r & 7))];
        }
    } else if (sizeof(T) == 4) {
#pragma unroll 4
        for (int r = 0; r < 32; ++r)
            if (r < rows && lane < n) to[r * p.ld + lane] = at(r, lane);
    } else {
        // rows of one parity start alike: their pairs from column `odd` on, then the single
        // columns that are left at either end, a lane a row
#pragma unroll
        for (int par = 0; par < 2; ++par) {
            T* q = to + par * p.ld;
            const int odd = (int)(reinterpret_cast<uintptr_t>(q) >> 1 & 1u), c = 2 * lane + odd;
            const bool there = c + 1 < n;
            const long long step = 2 * p.ld;
            q += c;
#pragma unroll 8
            for (int r = par; r < 32; r += 2, q += step)
                if (r < rows && there) {
                    T pair[2] = {at(r, c), at(r, c + 1)};
                    *reinterpret_cast<uint32_t*>(q) = *reinterpret_cast<const uint32_t*>(pair);
                }
        }
        if (lane < rows) {
            T* const q = to + lane * p.ld;
            const int odd = (int)(reinterpret_cast<uintptr_t>(q) >> 1 & 1u);
            if (odd) q[0] = at(lane, 0);
            if ((n - odd) & 1) q[n - 1] = at(lane, n - 1);
        }
    }
}

__device__ __forceinline__ void fp8_tile_coords(int tile, int mt, int nt, int& m_blk, int& n_blk) {
    const int per_group = kFGroupM * nt;
    const int g = tile / per_group;
    const int r = tile - g * per_group;
    const int gm = min(kFGroupM, mt - g * kFGroupM);
    n_blk = r / gm;
    m_blk = g * kFGroupM + (r - n_blk * gm);
}

// The fold warps' part: 128 columns of every tile of NC.  Both warpgroups run the
// same instructions, also where NC leaves the second fewer columns (it folds what
// its TMEM columns hold and writes NC - 128): a loop of its own for it cost a
// quarter of the rate, in instruction fetches.
template <int NC>
__device__ __forceinline__ void fold_tiles(const Fp8GemmLaunch& p, Fp8Smem& sm, uint32_t tmem, int mt, int nt, int nk,
                                           unsigned limit) {
    constexpr bool kAligned = NC % kFK == 0;  // the columns lie in one block of 128 rows of W
    constexpr int kCols = kFCols;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, q = warp & 3;
    const int col0 = warp < 8 ? 0 : kFCols;
    const int ntiles = mt * nt;
    const int wblocks = (p.vocab + kFK - 1) / kFK;
    unsigned it = 0;
    bool ok = true;
    int tile = blockIdx.x;
    for (; tile < ntiles && ok; tile += gridDim.x) {
        int mb, nb;
        fp8_tile_coords(tile, mt, nt, mb, nb);
        const int row0 = mb * kFM + q * 32, row = row0 + lane;
        const int wcol = nb * NC + col0;
        if (NC < kFN && row0 >= p.batch) {  // no rows of H here: the buffers are given back unread
            for (int k = 0; k < nk; ++k, ++it) {
                ok = ok && fp8_wait(&sm.tmem_full[it & 1u], it >> 1 & 1u, sm, p.error_word, limit);
                __syncwarp();
                if (lane == 0) mbar_arrive(&sm.tmem_empty[it & 1u]);
            }
            ok = __all_sync(kFullMask, ok ? 1 : 0);
            continue;
        }
        unsigned long long acc[kCols / 2];
#pragma unroll
        for (int j = 0; j < kCols / 2; ++j) acc[j] = 0ull;
        // `bound` of the columns belong to the first of the two blocks of W that they can lie in
        const int wb = wcol / kFK, bound = (wb + 1) * kFK - wcol;
        const float* own_scale = p.h_scales + (long long)row * nk;
        const float* lo_scale = p.w_scales + (long long)wb * nk;
        // The scales are on their way for two blocks before they are multiplied: L1, beside
        // 227 KB of shared memory, does not hold the rows' lines from block to block.
        const bool use = row < p.batch && wb < wblocks, use_hi = !kAligned && use && bound < kCols && wb + 1 < wblocks;
        float own0 = use ? __ldg(own_scale) : 0.0f, own1 = use && nk > 1 ? __ldg(own_scale + 1) : 0.0f;
        float lo0 = use ? __ldg(lo_scale) : 0.0f, lo1 = use && nk > 1 ? __ldg(lo_scale + 1) : 0.0f;
        float hi0 = use_hi ? __ldg(lo_scale + nk) : 0.0f, hi1 = use_hi && nk > 1 ? __ldg(lo_scale + nk + 1) : 0.0f;
        for (int k = 0; k < nk; ++k, ++it) {
            const unsigned buf = it & 1u;
            const bool more = k + 2 < nk;
            const float own2 = use && more ? __ldg(own_scale + k + 2) : 0.0f;
            const float lo2 = use && more ? __ldg(lo_scale + k + 2) : 0.0f;
            const float hi2 = use_hi && more ? __ldg(lo_scale + nk + k + 2) : 0.0f;
            // After a wait that ran out the rest of the tile is folded without waiting (and not
            // written): nothing but the wait stands between a buffer's arrival and its loads (a
            // look at the abort word here cost a quarter of the rate).
            ok = ok && fp8_wait(&sm.tmem_full[buf], it >> 1 & 1u, sm, p.error_word, limit);
            __syncwarp();
            tc_fence_after();
            const uint32_t src = tmem + ((uint32_t)(q * 32) << 16) + buf * kFN + (uint32_t)col0;
            const unsigned long long s_lo = pair_of(own0 * lo0, own0 * lo0);
            const unsigned long long s_hi = kAligned ? s_lo : pair_of(own0 * hi0, own0 * hi0);
#pragma unroll
            for (int c = 0; c < kCols; c += 64) {
                uint32_t t0[32], t1[32];
                tmem_load(src + (uint32_t)c, t0);
                tmem_load(src + (uint32_t)(c + 32), t1);
                tmem_wait(t0);
                tmem_wait(t1);
                if (c + 64 >= kCols) {  // the buffer has been read
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&sm.tmem_empty[buf]);
                }
                const unsigned long long f0 = kAligned || c < bound ? s_lo : s_hi;
                const unsigned long long f1 = kAligned || c + 32 < bound ? s_lo : s_hi;
#pragma unroll
                for (int j = 0; j < 32; j += 2) fold2(acc[(c + j) / 2], t0[j], t0[j + 1], f0);
#pragma unroll
                for (int j = 0; j < 32; j += 2) fold2(acc[(c + 32 + j) / 2], t1[j], t1[j + 1], f1);
            }
            own0 = own1, own1 = own2;
            lo0 = lo1, lo1 = lo2;
            hi0 = hi1, hi1 = hi2;
        }
        ok = __all_sync(kFullMask, ok ? 1 : 0);
        if (!ok) break;
        // 128 bytes of each row at a time through the warp's shared memory, so that whole lines go
        // out; piece j of row r is at piece j ^ (r % 8), so neither side meets bank conflicts
        const int left = min(NC - col0, p.vocab - wcol);  // columns to write
        uint4* const out4 = reinterpret_cast<uint4*>(sm.out[warp - 4]);
        if (p.out_bf16) {
#pragma unroll
            for (int c = 0; c < kCols; c += 64) {
                if (c >= left) break;
                __syncwarp();
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    uint32_t w[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float2 a = halves_of(acc[c / 2 + 4 * j + i]);
                        const __nv_bfloat162 h = __floats2bfloat162_rn(a.x, a.y);
                        w[i] = *reinterpret_cast<const uint32_t*>(&h);
                    }
                    out4[lane * 8 + (j ^ (lane & 7))] = make_uint4(w[0], w[1], w[2], w[3]);
                }
                __syncwarp();
                write_block(p, reinterpret_cast<const __nv_bfloat16*>(out4), row0, wcol + c, min(64, left - c), lane);
            }
        } else {
#pragma unroll
            for (int c = 0; c < kCols; c += 32) {
                if (c >= left) break;
                __syncwarp();
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const float2 a = halves_of(acc[c / 2 + 2 * j]), b = halves_of(acc[c / 2 + 2 * j + 1]);
                    out4[lane * 8 + (j ^ (lane & 7))] = make_uint4(__float_as_uint(a.x), __float_as_uint(a.y),
                                                                   __float_as_uint(b.x), __float_as_uint(b.y));
                }
                __syncwarp();
                write_block(p, reinterpret_cast<const float*>(out4), row0, wcol + c, min(32, left - c), lane);
            }
        }
    }
    if (!ok)  // this tile and those behind it
        for (; tile < ntiles; tile += gridDim.x) {
            int mb, nb;
            fp8_tile_coords(tile, mt, nt, mb, nb);
            const int row = mb * kFM + q * 32 + lane, wcol = nb * NC + col0;
            if (row >= p.batch) continue;
            const long long at = (long long)row * p.ld + wcol;
            for (int c = min(NC - col0, p.vocab - wcol) - 1; c >= 0; --c) {
                if (p.out_bf16) static_cast<uint16_t*>(p.logits)[at + c] = kUnfinishedBf16;
                else static_cast<uint32_t*>(p.logits)[at + c] = kUnfinishedF32;
            }
        }
}

// kTest: the self-test's form, which issues no products, so that the fold warps' first
// wait runs out on a barrier nothing arrives at.
template <int NC, bool kTest>
__global__ void __launch_bounds__(kFThreads, 1)
    fp8_gemm_kernel(const __grid_constant__ CUtensorMap tmap_h, const __grid_constant__ CUtensorMap tmap_w,
                    Fp8GemmLaunch p) {
    extern __shared__ __align__(16) unsigned char fsm_raw[];
    Fp8Smem& sm = *reinterpret_cast<Fp8Smem*>((reinterpret_cast<uintptr_t>(fsm_raw) + 1023) & ~(uintptr_t)1023);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int mt = (p.batch + kFM - 1) / kFM;
    const int nt = (p.vocab + NC - 1) / NC;
    const int ntiles = mt * nt;
    const int nk = (p.dim + kFK - 1) / kFK;
    const unsigned limit = kTest ? p.wait_test : kSpinLimit;

    const auto load_stage = [&](unsigned stage, int k, int mb, int nb) {
        mbar_arrive_expect_tx(&sm.full[stage], (unsigned)(p.box_rows + NC) * kFK);
        tma_load_2d(sm.a[stage], &tmap_h, k * kFK, mb * kFM, &sm.full[stage]);
        tma_load_2d(sm.b[stage], &tmap_w, k * kFK, nb * NC, &sm.full[stage]);
    };
    if (tid == 0) {
        for (int s = 0; s < kFStages; ++s) {
            mbar_init(&sm.full[s], 1);
            mbar_init(&sm.empty[s], 1);
        }
        for (int a = 0; a < 2; ++a) {
            mbar_init(&sm.tmem_full[a], 1);
            mbar_init(&sm.tmem_empty[a], NC > kFCols ? 8 : 4);  // one arrival per fold warp
        }
        mbar_init(&sm.drain, 1);
        sm.abort = 0;
        fence_mbar_init();
        // the first stages are on their way while TMEM is allocated
        int mb, nb;
        fp8_tile_coords(blockIdx.x, mt, nt, mb, nb);
        for (int k = 0; k < min(nk, kFStages); ++k) load_stage(k, k, mb, nb);
    }
    if (warp == 2) {
        tmem_alloc(smem_addr(&sm.tmem_base), kFTmemCols);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = sm.tmem_base;

    // 384 threads at 168 registers: the two fold warpgroups take 216, the other 72
    if (warp < 4) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
        if (warp == 0 && lane == 0) {
            // ---- TMA producer
            const int ahead = min(nk, kFStages);  // issued above
            unsigned stage = ahead == kFStages ? 0 : ahead, phase = ahead == kFStages ? 1 : 0;
            int k = ahead;
            for (int tile = blockIdx.x; tile < ntiles && !fp8_aborted(sm); tile += gridDim.x, k = 0) {
                int mb, nb;
                fp8_tile_coords(tile, mt, nt, mb, nb);
                for (; k < nk; ++k) {
                    if (!fp8_wait(&sm.empty[stage], phase ^ 1u, sm, p.error_word, limit)) break;
                    load_stage(stage, k, mb, nb);
                    if (++stage == kFStages) {
                        stage = 0;
                        phase ^= 1u;
                    }
                }
            }
            // drain: every copy this thread issued has landed before the CTA exits, whether or not
            // products still took it (from `stage` on, a stage's last fill is of the pass before) ..
            for (unsigned s = 0; s < kFStages; ++s) mbar_wait_bounded(&sm.full[s], s < stage ? phase : phase ^ 1u);
            // .. and every stage it filled has been given back, if products went on
            for (int s = 0; s < kFStages; ++s) {
                if (!mbar_wait_bounded(&sm.empty[stage], phase ^ 1u, limit)) break;
                if (++stage == kFStages) {
                    stage = 0;
                    phase ^= 1u;
                }
            }
        } else if (warp == 1 && lane == 0) {
            // ---- MMA issuer: one accumulation of its own for every block of 128.
            // Instruction descriptor, kind::f8f6f4: fp32 accumulator (bits 4-5 = 1), A and B e4m3
            // (bits 7-9, 10-12 = 0), both K-major (bits 15, 16 = 0), N >> 3 in bits 17-22, M >> 4 in
            // bits 24-28.
            constexpr uint32_t idesc = (1u << 4) | ((uint32_t)(NC >> 3) << 17) | ((uint32_t)(kFM >> 4) << 24);
            const uint64_t da0 = smem_desc_sw128(smem_addr(sm.a[0])), db0 = smem_desc_sw128(smem_addr(sm.b[0]));
            unsigned stage = 0, phase = 0, it = 0;
            bool ok = !kTest;
            for (int tile = blockIdx.x; tile < ntiles && ok && !fp8_aborted(sm); tile += gridDim.x) {
                for (int k = 0; k < nk; ++k, ++it) {
                    const unsigned buf = it & 1u, turn = it >> 1 & 1u;
                    if (!fp8_wait(&sm.tmem_empty[buf], turn ^ 1u, sm, p.error_word, limit) ||
                        !fp8_wait(&sm.full[stage], phase, sm, p.error_word, limit)) {
                        ok = false;
                        break;
                    }
                    tc_fence_after();
                    const uint64_t da = da0 + stage * (kFABytes >> 4), db = db0 + stage * (kFBBytes >> 4);
#pragma unroll
                    for (int kk = 0; kk < kFK / 32; ++kk)  // 32 bytes (2 in the descriptor) on inside the swizzled 128-byte row
                        tc_mma_fp8(tmem + buf * kFN, da + 2 * kk, db + 2 * kk, idesc, kk != 0);
                    tc_commit(&sm.tmem_full[buf]);
                    tc_commit(&sm.empty[stage]);
                    if (++stage == kFStages) {
                        stage = 0;
                        phase ^= 1u;
                    }
                }
            }
            // every MMA this thread issued is complete before TMEM is released
            tc_commit(&sm.drain);
            mbar_wait_bounded(&sm.drain, 0);
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
        // ---- fold: warp w reads TMEM lanes 32 * (w % 4) .. +31
        if (NC > kFCols || warp < 8) fold_tiles<NC>(p, sm, tmem, mt, nt, nk, limit);
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 2) {
        tc_fence_after();
        tmem_dealloc(tmem, kFTmemCols);
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

template <int NC, bool kTest = false>
cudaError_t launch_fp8(const Fp8GemmLaunch& p, int num_sms, cudaStream_t stream) {
    CUtensorMap th, tw;
    if (!make_tmap_fp8(&th, p.h, p.batch, p.dim, p.box_rows) || !make_tmap_fp8(&tw, p.w, p.vocab, p.dim, NC))
        return cudaErrorInvalidValue;
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    static std::atomic<unsigned long long> attr_done{0};
    const unsigned long long bit = 1ull << (dev & 63);
    if (!(attr_done.load() & bit)) {
        e = cudaFuncSetAttribute(fp8_gemm_kernel<NC, kTest>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                 (int)kFp8SmemBytes);
        if (e != cudaSuccess) return e;
        attr_done.fetch_or(bit);
    }
    const long long tiles = (long long)((p.batch + kFM - 1) / kFM) * ((p.vocab + NC - 1) / NC);
    const int grid = tiles < num_sms ? (int)tiles : num_sms;
    fp8_gemm_kernel<NC, kTest><<<grid, kFThreads, kFp8SmemBytes, stream>>>(th, tw, p);
    return cudaGetLastError();
}

}  // namespace

int launch_fp8_gemm(const Fp8GemmLaunch& args, int num_sms, cudaStream_t stream) {
    Fp8GemmLaunch p = args;
    p.box_rows = p.batch < kFM ? (p.batch + 7) / 8 * 8 : kFM;
    p.vec_out = (reinterpret_cast<uintptr_t>(p.logits) & 15u) == 0 && p.ld % (p.out_bf16 ? 8 : 4) == 0;
    // Columns of a tile: such that the rounds of tiles that an SM goes through, each as long as its
    // columns (and some 64 more: a block's way through the buffers), are shortest.
    const long long mt = (p.batch + kFM - 1) / kFM;
    long long best = 0;
    int cols = kFN;
    for (int c = kFN; c >= kFCols; c -= 32) {
        const long long tiles = mt * ((p.vocab + c - 1) / c);
        const long long cost = (tiles + num_sms - 1) / num_sms * (c + 64);
        if (best == 0 || cost < best) {
            best = cost;
            cols = c;
        }
    }
    cudaError_t e;
    if (p.wait_test) e = launch_fp8<kFCols, true>(p, num_sms, stream);
    else if (cols == 256) e = launch_fp8<256>(p, num_sms, stream);
    else if (cols == 224) e = launch_fp8<224>(p, num_sms, stream);
    else if (cols == 192) e = launch_fp8<192>(p, num_sms, stream);
    else if (cols == 160) e = launch_fp8<160>(p, num_sms, stream);
    else e = launch_fp8<128>(p, num_sms, stream);
    return e == cudaSuccess ? 1 : -(int)e;
}

}  // namespace b2s
