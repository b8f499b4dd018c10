// Orthogonalised updates by Newton-Schulz products, and Muon's step.
//
// X = U / (|U|_F + eps); then `steps` times, on the narrow side s x s,
//   A = X X^T (or X^T X),  M = a I + b A + c A^2,  X <- M X (or X M).
// Each is a GEMM on the tensor cores (csrc/tc05.cuh).  The polynomial needs
// no pass of its own: with Z = A + (b / 2c) I, M = c Z^2 + (a - b^2 / 4c) I,
// so each epilogue scales and shifts a diagonal.
//
// Precision.  Every operand v is held as S v = hi + lo, two fp16 values (22
// bits), S a power of two that keeps the iteration's values below fp16's
// largest, and a product is hi hi + hi lo + lo hi in fp32: three MMAs for
// one.  Its error is that of 32-bit arithmetic (measured in the tests); one
// MMA per product loses a rank-deficient update's small directions, which
// five steps amplify 3.44^5 times (2e-2 of the result on a low-rank update
// against 5e-6).
//
// A and A^2 are symmetric: their tiles on and below the diagonal are
// computed and mirrored.  Rows and columns past a matrix's own are zeros
// that TMA fills in, so any size works and nothing is padded in memory but
// the row pitch (to 16 bytes).

#include <cooperative_groups.h>
#include <cuda.h>
#include <cudaTypedefs.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include <atomic>
#include <mutex>

#include "../../include/scacchi_b200.h"
#include "tc05.cuh"

namespace {

using namespace tc05;
namespace cg = cooperative_groups;

constexpr int kBM = 128;           // rows of a CTA's output tile
constexpr int kBK = 64;            // K of a stage: 128 bytes of fp16
constexpr int kEpiWarps = 8;       // two per TMEM lane quadrant, half the tile's columns each
constexpr int kThreads = 64 + 32 * kEpiWarps;  // producer, MMA issuer, epilogue
constexpr int kMaxSplit = 8;       // CTAs of a cluster that share a tile's K
constexpr int kNormBlocks = 128;   // most partial sums of squares per matrix
constexpr int kPatch = 2 * 32 * 64;  // an epilogue warp's 32 x 32 block as two fp16 parts

__device__ uint32_t g_muon_error;
std::atomic<uint64_t> g_muon_launches{0};

enum Mode : int { kGram = 0, kSquare = 1, kUpdate = 2, kLast = 3 };

struct Product {
  int mode, sym;
  int rows, cols, k;            // of the output, and the summed length
  int tiles_n, per_batch, tiles;
  float scale, diag;            // the output is scale acc + diag on the diagonal
  // last: the result, or the weight's step w <- decay w - step x
  void *out;
  int dtype;                    // 0 float32, 1 bfloat16, 2 float16
  float *weight;
  float decay, step;
};

// A tile's place: matrix, tile row (of BM rows), tile column.  Symmetric
// outputs list, row by row, the tiles that touch the lower triangle.
template <int BM, int BN>
__device__ __forceinline__ void locate(const Product &q, int t, int &batch, int &i, int &j) {
  batch = t / q.per_batch;
  int u = t - batch * q.per_batch;
  if (!q.sym) {
    i = u / q.tiles_n;
    j = u - i * q.tiles_n;
    return;
  }
  i = 0;
  for (;;) {
    int n = (i * BM + BM - 1) / BN + 1;
    n = n < q.tiles_n ? n : q.tiles_n;
    if (u < n) break;
    u -= n;
    ++i;
  }
  j = u;
}

__device__ __forceinline__ void split_half(float v, __half &hi, __half &lo) {
  hi = __float2half_rn(v);
  lo = __float2half_rn(v - __half2float(hi));
}

// A warp's 32 x 32 block in the fragment layout (tmem_ld16x256_x4):
// element (row 16 h + 8 u + t/4, column 8 j + 2 (t%4) + e) of thread t is
// v[16 h + 4 j + 2 u + e].
//
// The last product's block goes to the user's matrix: four lanes write (or
// update) 8 neighbouring columns of a row.
__device__ __forceinline__ void emit_last(const Product &q, int batch, int r0, int c0, const float *v) {
  const int lane = threadIdx.x & 31, row = r0 + (lane >> 2), col = c0 + 2 * (lane & 3);
  const int64_t base = ((int64_t)batch * q.rows + row) * q.cols + col;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    float w[16];
    if (q.weight) {
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int dr = 16 * h + 8 * (i >> 1 & 1), dc = 8 * (i >> 2) + (i & 1);
        if (row + dr < q.rows && col + dc < q.cols) w[i] = q.weight[base + (int64_t)dr * q.cols + dc];
      }
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int dr = 16 * h + 8 * (i >> 1 & 1), dc = 8 * (i >> 2) + (i & 1);
      if (row + dr < q.rows && col + dc < q.cols) {
        const int64_t at = base + (int64_t)dr * q.cols + dc;
        const float y = v[16 * h + i] * q.scale;
        if (q.weight)
          q.weight[at] = fmaf(-q.step, y, q.decay * w[i]);
        else if (q.dtype == 0)
          static_cast<float *>(q.out)[at] = y;
        else if (q.dtype == 1)
          static_cast<__nv_bfloat16 *>(q.out)[at] = __float2bfloat16_rn(y);
        else
          static_cast<__half *>(q.out)[at] = __float2half_rn(y);
      }
    }
  }
}

// The block of an operand of the next product: split into hi and lo, laid
// out by stmatrix (rows of 64 bytes, 64B-swizzled) and stored by TMA, which
// leaves out what lies past the matrix; for a symmetric output whose mirror
// tile is not computed, once more transposed.  hi and lo have a patch each,
// so one is filled while the other is read.
__device__ __forceinline__ void emit_block(const Product &q, const CUtensorMap *map_d, int batch, int r0, int c0,
                                           bool mirror, const float *v, uint8_t *patch) {
  const int lane = threadIdx.x & 31;
  uint32_t hi[16], lo[16];  // [row group 2 h + u][column group j]
  const bool on_diagonal = r0 == c0;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const int h = i >> 3, u = i >> 2 & 1, j = i & 3;
    float x = v[16 * h + 4 * j + 2 * u] * q.scale, y = v[16 * h + 4 * j + 2 * u + 1] * q.scale;
    if (on_diagonal) {
      const int d = 16 * h + 8 * u + (lane >> 2) - (8 * j + 2 * (lane & 3));
      if (d == 0) x += q.diag;
      if (d == 1) y += q.diag;
    }
    const __half2 a = __floats2half2_rn(x, y);
    const float2 f = __half22float2(a);
    const __half2 b = __floats2half2_rn(x - f.x, y - f.y);
    hi[i] = *reinterpret_cast<const uint32_t *>(&a);
    lo[i] = *reinterpret_cast<const uint32_t *>(&b);
  }
  const uint32_t base = smem_u32(patch);
  const int sub = lane & 7, mat = lane >> 3;
#pragma unroll
  for (int turned = 0; turned < 2; ++turned) {
    if (turned && !mirror) break;
    const int x = turned ? r0 : c0, y = turned ? c0 : r0;
#pragma unroll
    for (int part = 0; part < 2; ++part) {
      const uint32_t(&p)[16] = part ? lo : hi;
      if (lane == 0) tma_store_wait_read<1>();  // this part's patch is free
      __syncwarp();
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int row = 8 * g + sub;
        const uint32_t at = base + part * 2048 + row * 64 + ((mat ^ (row >> 1 & 3)) << 4);
        if (turned)
          stmatrix_x4_trans(at, p[g], p[4 + g], p[8 + g], p[12 + g]);
        else
          stmatrix_x4(at, p[4 * g], p[4 * g + 1], p[4 * g + 2], p[4 * g + 3]);
      }
      fence_proxy_async();
      __syncwarp();
      if (lane == 0) {
        tma_store_3d(map_d, patch + part * 2048, x, y, 2 * batch + part);
        tma_store_commit();
      }
    }
  }
}

// Whether the tile that holds (c, r) is absent from the symmetric list.
template <int BM, int BN>
__device__ __forceinline__ bool mirrored(const Product &q, int r, int c) {
  return q.sym && r / BN * BN > c / BM * BM + BM - 1;
}

// The tensor core truncates each time it adds to a TMEM accumulator: about
// 1.5e-7 of the result per MMA once five steps have amplified it, 5.7e-5
// at K = 2048.  So an accumulator takes one stage (K = 64), its eight small
// cross products before the four large ones, and the epilogue warps add the
// stages in fp32 registers, rounding to nearest, while the next stage runs
// on the other accumulator (1.3e-6 at 2048 x 2048, where 32-bit arithmetic
// gives 3.3e-6).
template <int COLS>
__device__ __forceinline__ void add_stage(float (&sum)[COLS], uint32_t acc) {
#pragma unroll
  for (int g = 0; g < COLS / 16; ++g) {
    uint32_t v[16];
    tmem_ld16x256_x4(acc + ((uint32_t)(16 * (g & 1)) << 16) + (g >> 1) * 32, v);
    tmem_wait_ld();
#pragma unroll
    for (int e = 0; e < 16; ++e) sum[g * 16 + e] += __uint_as_float(v[e]);
  }
}

// Descriptors of a stage's operands: the first stage's, advanced by whole
// 16-byte units (an address stays within the field's 14 bits).  The MMA
// warp keeps its control flow uniform and elects a lane for the issue
// alone: with the loop inside `lane == 0` each MMA took 100 clocks to issue.
template <bool kAMn, bool kBMn>
struct StageDesc {
  uint64_t a_hi, b_hi;
  uint32_t a_part, b_part;
  __device__ __forceinline__ StageDesc(uint32_t stage0, uint32_t a_bytes, uint32_t b_bytes) {
    a_hi = desc_sw128(stage0, kAMn ? 64 * kBK * 2 : 16);
    b_hi = desc_sw128(stage0 + 2 * a_bytes, kBMn ? 64 * kBK * 2 : 16);
    a_part = a_bytes >> 4;
    b_part = b_bytes >> 4;
  }
  __device__ __forceinline__ uint64_t a(bool lo, int k, uint32_t at) const {
    return a_hi + (lo ? a_part : 0u) + at + (uint32_t)k * (kAMn ? 2048u >> 4 : 32u >> 4);
  }
  __device__ __forceinline__ uint64_t b(bool lo, int k, uint32_t at) const {
    return b_hi + (lo ? b_part : 0u) + at + (uint32_t)k * (kBMn ? 2048u >> 4 : 32u >> 4);
  }
};

// one operand part of a stage: `rows` rows of the tile (from `at`) by 64 of K
template <bool kMn, typename Load>
__device__ __forceinline__ void load_operand(uint8_t *dst, int rows, int at, int kb, Load load) {
  if (kMn) {
    for (int m = 0; m < rows; m += 64) load(dst + m * kBK * 2, at + m, kb * kBK);
  } else {
    load(dst, kb * kBK, at);
  }
}

// ---------------------------------------------------------------------------
// pairs of CTAs: 256 x BN tiles
// ---------------------------------------------------------------------------

template <int BN>
struct PairLayout {
  static constexpr int kA = kBM * kBK * 2, kB = BN / 2 * kBK * 2;  // one part of a stage's operands in one CTA
  static constexpr int kStage = 2 * (kA + kB);
  static constexpr int kStages = BN == 256 ? 3 : 4;
  static constexpr int kPatches = kStages * kStage;
  static constexpr int kBars = kPatches + kEpiWarps * kPatch;
  static constexpr int kBytes = kBars + 8 * (2 * kStages + 4) + 16 + 1024;  // + alignment slack
  static_assert(kBytes <= 227 * 1024, "shared memory budget");
};

// D[i, j] = A[i, k] B[j, k]; A and B are K-major (their rows run along k) or
// MN-major (k counts rows).  Persistent over the tiles.
//
// A single CTA's 128 x 256 tile needs 96 KB of operands per stage, and 148
// of them drew 13 TB/s from L2, its limit here: 1.08 us a stage, against
// 0.82 us of MMA.  A pair shares B, 64 KB a CTA.
template <int BN, bool kAMn, bool kBMn>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
    ns_pair_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
                   const __grid_constant__ CUtensorMap map_d, const __grid_constant__ Product q) {
  using L = PairLayout<BN>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  uint64_t *full = reinterpret_cast<uint64_t *>(smem + L::kBars);  // the even CTA's counts both CTAs' loads
  uint64_t *empty = full + L::kStages;
  uint64_t *acc_full = empty + L::kStages;
  uint64_t *acc_empty = acc_full + 2;                              // the even CTA's counts both epilogues
  uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(acc_empty + 2);
  volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_slot + 1);
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int kblocks = (q.k + kBK - 1) / kBK;
  const int rank = (int)cg::this_cluster().block_rank();
  const int first = blockIdx.x / 2, step = gridDim.x / 2;

  if (threadIdx.x == 0) {
    prefetch_map(&map_a);
    prefetch_map(&map_b);
    for (int s = 0; s < L::kStages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(&acc_full[s], 1);
      mbar_init(&acc_empty[s], 2 * kEpiWarps);
    }
    *abort_flag = 0;
    fence_barrier_init();
  }
  __syncwarp();
  if (warp == 1) {
    tmem_alloc_pair(tmem_slot, 2 * BN);
    tmem_relinquish_pair();
  }
  tc_fence_before();
  cg::this_cluster().sync();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  cudaTriggerProgrammaticLaunchCompletion();
  cudaGridDependencySynchronize();

  if (warp == 0) {
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0, issued = 0, parity = 0;
      bool stop = false;
      for (int t = first; t < q.tiles && !stop; t += step) {
        int batch, i, j;
        locate<2 * kBM, BN>(q, t, batch, i, j);
        for (int kb = 0; kb < kblocks; ++kb) {
          if (*abort_flag || !mbar_wait(&empty[stage], phase ^ 1u, abort_flag, &g_muon_error)) {
            stop = true;
            break;
          }
          uint8_t *at = smem + stage * L::kStage;
          const uint32_t bar = cluster_addr(smem_u32(&full[stage]), 0);
          if (rank == 0) mbar_expect_tx(&full[stage], 2 * L::kStage);
#pragma unroll
          for (int part = 0; part < 2; ++part) {
            load_operand<kAMn>(at + part * L::kA, kBM, (2 * i + rank) * kBM, kb, [&](uint8_t *dst, int x, int y) {
              tma_load_3d_pair(dst, &map_a, bar, x, y, 2 * batch + part);
            });
            load_operand<kBMn>(at + 2 * L::kA + part * L::kB, BN / 2, j * BN + rank * (BN / 2), kb,
                               [&](uint8_t *dst, int x, int y) {
                                 tma_load_3d_pair(dst, &map_b, bar, x, y, 2 * batch + part);
                               });
          }
          issued |= 1u << stage;
          parity = (parity & ~(1u << stage)) | (phase << stage);
          if (++stage == L::kStages) {
            stage = 0;
            phase ^= 1u;
          }
        }
      }
      // every load of the pair lands before either CTA may exit (the
      // cluster barrier below)
      if (rank == 0)
        for (int s = 0; s < L::kStages; ++s)
          if (issued >> s & 1u) mbar_drain(&full[s], parity >> s & 1u);
    }
  } else if (warp == 1) {
    if (rank == 0) {
      int stage = 0, slot = 0;
      uint32_t phase = 0, acc_phase = 0;
      bool ok = true;
      const StageDesc<kAMn, kBMn> desc(smem_u32(smem), L::kA, L::kB);
      for (int t = first; t < q.tiles && ok; t += step) {
        for (int kb = 0; kb < kblocks; ++kb) {
          ok = mbar_wait_warp(&acc_empty[slot], acc_phase ^ 1u, abort_flag, &g_muon_error) &&
               mbar_wait_warp(&full[stage], phase, abort_flag, &g_muon_error);
          if (!ok) break;
          tc_fence_after();
          if (elect_one()) {
            constexpr uint32_t idesc = idesc_f16(2 * kBM, BN, kAMn, kBMn);
            const uint32_t d = tmem + (uint32_t)(slot * BN), at = (uint32_t)(stage * L::kStage) >> 4;
#pragma unroll
            for (int term = 0; term < 3; ++term)
#pragma unroll
              for (int k = 0; k < kBK / 16; ++k)
                umma_f16_pair(d, desc.a(term == 1, k, at), desc.b(term == 0, k, at), idesc, (term | k) != 0);
            umma_commit_pair(&empty[stage]);
            umma_commit_pair(&acc_full[slot]);
          }
          __syncwarp();
          if (++stage == L::kStages) {
            stage = 0;
            phase ^= 1u;
          }
          if (++slot == 2) {
            slot = 0;
            acc_phase ^= 1u;
          }
        }
      }
    }
  } else {
    constexpr int kCols = BN / 2;              // columns of a warp
    const int quad = warp & 3;                 // the TMEM lanes this warp may read
    const int half = (warp - 2) >> 2;
    uint8_t *patch = smem + L::kPatches + (warp - 2) * kPatch;
    int slot = 0;
    uint32_t acc_phase = 0;
    bool ok = true;
    for (int t = first; t < q.tiles && ok; t += step) {
      float sum[kCols];
#pragma unroll
      for (int e = 0; e < kCols; ++e) sum[e] = 0.0f;
      for (int kb = 0; kb < kblocks; ++kb) {
        int go = 0;
        if (lane == 0) go = !*abort_flag && mbar_wait(&acc_full[slot], acc_phase, abort_flag, &g_muon_error);
        ok = __shfl_sync(0xffffffffu, go, 0) != 0;
        if (!ok) break;
        tc_fence_after();
        add_stage<kCols>(sum, tmem + (uint32_t)(slot * BN + half * kCols) + ((uint32_t)(quad * 32) << 16));
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster(cluster_addr(smem_u32(&acc_empty[slot]), 0));
        if (++slot == 2) {
          slot = 0;
          acc_phase ^= 1u;
        }
      }
      if (!ok) break;
      int batch, i, j;
      locate<2 * kBM, BN>(q, t, batch, i, j);
      const int r0 = (2 * i + rank) * kBM + quad * 32;
#pragma unroll
      for (int g = 0; g < kCols / 32; ++g) {
        const int c0 = j * BN + half * kCols + g * 32;
        if (r0 < q.rows && c0 < q.cols) {
          if (q.mode == kLast)
            emit_last(q, batch, r0, c0, sum + g * 32);
          else
            emit_block(q, &map_d, batch, r0, c0, mirrored<2 * kBM, BN>(q, r0, c0), sum + g * 32, patch);
        }
      }
    }
    if (lane == 0) tma_store_wait_all();
  }
  __syncwarp();
  tc_fence_before();
  cg::this_cluster().sync();
  if (warp == 1) tmem_dealloc_pair(tmem, 2 * BN);
}

// ---------------------------------------------------------------------------
// one 128 x 128 tile per CTA, or per cluster
// ---------------------------------------------------------------------------

struct TileLayout {
  static constexpr int kBN = 128;
  static constexpr int kA = kBM * kBK * 2, kB = kBN * kBK * 2;
  static constexpr int kStage = 2 * (kA + kB);
  static constexpr int kStages = 3;
  static constexpr int kPatches = kStages * kStage;
  static constexpr int kBars = kPatches + kEpiWarps * kPatch;
  static constexpr int kBytes = kBars + 8 * (2 * kStages + 4) + 16 + 1024;  // + alignment slack
  static_assert(kBytes <= 227 * 1024, "shared memory budget");
  static_assert(kBN * kBM * 4 <= kPatches, "the partial sums take the stages' place");
};

// The same product for outputs of few tiles: the CTAs of a cluster share one
// tile's K, each reducing its share of the columns from all of them through
// distributed shared memory, so that a small output with a long sum does
// not leave most SMs idle.
template <bool kAMn, bool kBMn>
__global__ void __launch_bounds__(kThreads, 1)
    ns_tile_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
                   const __grid_constant__ CUtensorMap map_d, const __grid_constant__ Product q) {
  using L = TileLayout;
  constexpr int BN = L::kBN;
  extern __shared__ uint8_t smem_raw[];
  uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  uint64_t *full = reinterpret_cast<uint64_t *>(smem + L::kBars);
  uint64_t *empty = full + L::kStages;
  uint64_t *acc_full = empty + L::kStages;
  uint64_t *acc_empty = acc_full + 2;
  uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(acc_empty + 2);
  volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_slot + 1);
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int kblocks = (q.k + kBK - 1) / kBK;
  const int ctas = (int)cg::this_cluster().num_blocks(), rank = (int)cg::this_cluster().block_rank();
  const int kb0 = rank * kblocks / ctas, kb1 = (rank + 1) * kblocks / ctas;
  int batch, i, j;
  locate<kBM, BN>(q, blockIdx.x / ctas, batch, i, j);

  if (threadIdx.x == 0) {
    prefetch_map(&map_a);
    prefetch_map(&map_b);
    for (int s = 0; s < L::kStages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(&acc_full[s], 1);
      mbar_init(&acc_empty[s], kEpiWarps);
    }
    *abort_flag = 0;
    fence_barrier_init();
  }
  __syncwarp();
  if (warp == 1) {
    tmem_alloc(tmem_slot, 2 * BN);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  cudaTriggerProgrammaticLaunchCompletion();
  cudaGridDependencySynchronize();

  if (warp == 0) {
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0, issued = 0, parity = 0;
      for (int kb = kb0; kb < kb1; ++kb) {
        if (*abort_flag || !mbar_wait(&empty[stage], phase ^ 1u, abort_flag, &g_muon_error)) break;
        uint8_t *at = smem + stage * L::kStage;
        mbar_expect_tx(&full[stage], L::kStage);
#pragma unroll
        for (int part = 0; part < 2; ++part) {
          load_operand<kAMn>(at + part * L::kA, kBM, i * kBM, kb, [&](uint8_t *dst, int x, int y) {
            tma_load_3d(dst, &map_a, &full[stage], x, y, 2 * batch + part);
          });
          load_operand<kBMn>(at + 2 * L::kA + part * L::kB, BN, j * BN, kb, [&](uint8_t *dst, int x, int y) {
            tma_load_3d(dst, &map_b, &full[stage], x, y, 2 * batch + part);
          });
        }
        issued |= 1u << stage;
        parity = (parity & ~(1u << stage)) | (phase << stage);
        if (++stage == L::kStages) {
          stage = 0;
          phase ^= 1u;
        }
      }
      // every load into shared memory lands before the CTA may exit
      for (int s = 0; s < L::kStages; ++s)
        if (issued >> s & 1u) mbar_drain(&full[s], parity >> s & 1u);
    }
  } else if (warp == 1) {
    int stage = 0, slot = 0;
    uint32_t phase = 0, acc_phase = 0;
    const StageDesc<kAMn, kBMn> desc(smem_u32(smem), L::kA, L::kB);
    for (int kb = kb0; kb < kb1; ++kb) {
      if (!mbar_wait_warp(&acc_empty[slot], acc_phase ^ 1u, abort_flag, &g_muon_error) ||
          !mbar_wait_warp(&full[stage], phase, abort_flag, &g_muon_error))
        break;
      tc_fence_after();
      if (elect_one()) {
        constexpr uint32_t idesc = idesc_f16(kBM, BN, kAMn, kBMn);
        const uint32_t d = tmem + (uint32_t)(slot * BN), at = (uint32_t)(stage * L::kStage) >> 4;
#pragma unroll
        for (int term = 0; term < 3; ++term)
#pragma unroll
          for (int k = 0; k < kBK / 16; ++k)
            umma_f16(d, desc.a(term == 1, k, at), desc.b(term == 0, k, at), idesc, (term | k) != 0);
        umma_commit(&empty[stage]);
        umma_commit(&acc_full[slot]);
      }
      __syncwarp();
      if (++stage == L::kStages) {
        stage = 0;
        phase ^= 1u;
      }
      if (++slot == 2) {
        slot = 0;
        acc_phase ^= 1u;
      }
    }
  } else {
    constexpr int kCols = BN / 2;              // columns of a warp
    const int quad = warp & 3;                 // the TMEM lanes this warp may read
    const int half = (warp - 2) >> 2;
    const int r0 = i * kBM + quad * 32;
    uint8_t *patch = smem + L::kPatches + (warp - 2) * kPatch;
    int slot = 0;
    uint32_t acc_phase = 0;
    bool ok = true;
    float sum[kCols];
#pragma unroll
    for (int e = 0; e < kCols; ++e) sum[e] = 0.0f;
    for (int kb = kb0; kb < kb1; ++kb) {
      int go = 0;
      if (lane == 0) go = !*abort_flag && mbar_wait(&acc_full[slot], acc_phase, abort_flag, &g_muon_error);
      ok = __shfl_sync(0xffffffffu, go, 0) != 0;
      if (!ok) break;
      tc_fence_after();
      add_stage<kCols>(sum, tmem + (uint32_t)(slot * BN + half * kCols) + ((uint32_t)(quad * 32) << 16));
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&acc_empty[slot]);
      if (++slot == 2) {
        slot = 0;
        acc_phase ^= 1u;
      }
    }
    auto emit = [&](int c0, const float *v) {
      if (r0 >= q.rows || c0 >= q.cols) return;
      if (q.mode == kLast)
        emit_last(q, batch, r0, c0, v);
      else
        emit_block(q, &map_d, batch, r0, c0, mirrored<kBM, BN>(q, r0, c0), v, patch);
    };
    if (ctas == 1) {
      if (ok) {
#pragma unroll
        for (int g = 0; g < kCols / 32; ++g) emit(j * BN + half * kCols + g * 32, sum + g * 32);
      }
    } else {
      // Each CTA finishes BN / ctas columns, as blocks of 32 x 32: its
      // owner's warps take them in turn.  Partial sums arrive as [source]
      // [block][element][lane], four elements at a time.
      __syncwarp();
      cg::this_cluster().sync();  // every CTA is done with its stages
      const int blocks = 16 / ctas;  // of this CTA: 4 quads x BN / 32 columns, shared out
#pragma unroll
      for (int g = 0; g < kCols / 32; ++g) {
        const int id = quad + 4 * (half * (kCols / 32) + g);  // block of the tile
        float4 *buf = cg::this_cluster().map_shared_rank(reinterpret_cast<float4 *>(smem), id / blocks);
        float4 *at = buf + (rank * blocks + id % blocks) * 256 + lane;
#pragma unroll
        for (int e = 0; e < 8; ++e)
          at[e * 32] = make_float4(sum[g * 32 + 4 * e], sum[g * 32 + 4 * e + 1], sum[g * 32 + 4 * e + 2],
                                   sum[g * 32 + 4 * e + 3]);
      }
      cg::this_cluster().sync();
      if (warp - 2 < blocks && ok) {
        const float4 *at = reinterpret_cast<const float4 *>(smem) + (warp - 2) * 256 + lane;
        float v[32];
#pragma unroll
        for (int e = 0; e < 32; ++e) v[e] = 0.0f;
        for (int from = 0; from < ctas; ++from)
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float4 f = at[from * blocks * 256 + e * 32];
            v[4 * e] += f.x;
            v[4 * e + 1] += f.y;
            v[4 * e + 2] += f.z;
            v[4 * e + 3] += f.w;
          }
        const int id = rank * blocks + warp - 2, row = i * kBM + (id & 3) * 32, c0 = j * BN + (id >> 2) * 32;
        if (row < q.rows && c0 < q.cols) {
          if (q.mode == kLast)
            emit_last(q, batch, row, c0, v);
          else
            emit_block(q, &map_d, batch, row, c0, mirrored<kBM, BN>(q, row, c0), v, patch);
        }
      }
    }
    if (lane == 0) tma_store_wait_all();
  }
  if (ctas > 1 && warp < 2) {  // the epilogue's two cluster barriers are everyone's
    __syncwarp();
    cg::this_cluster().sync();
    cg::this_cluster().sync();
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) tmem_dealloc(tmem, 2 * BN);
}

// ---------------------------------------------------------------------------
// the update's norm, and its split
// ---------------------------------------------------------------------------

struct Source {
  const void *in;      // the matrix, or the gradient
  int dtype;
  float *momentum;     // Muon: updated in place by the norm kernel
  float beta, rest;    // beta and 1 - beta
  int nesterov;
};

__device__ __forceinline__ float load_any(const void *p, int dtype, int64_t i) {
  if (dtype == 0) return static_cast<const float *>(p)[i];
  if (dtype == 1) return __bfloat162float(static_cast<const __nv_bfloat16 *>(p)[i]);
  return __half2float(static_cast<const __half *>(p)[i]);
}

__device__ __forceinline__ float muon_direction(const Source &s, float g, float m) {
  return s.nesterov ? fmaf(s.beta, m, s.rest * g) : m;
}

// sum of squares of each matrix in 64 bits (an update may be small enough
// that its squares leave fp32), one partial per block
__global__ void __launch_bounds__(256) ns_norm_kernel(Source s, int64_t elems, double *partial) {
  __shared__ double part[8];
  const int64_t base = (int64_t)blockIdx.y * elems;
  double sum = 0.0;
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < elems; i += (int64_t)gridDim.x * blockDim.x) {
    float u = load_any(s.in, s.dtype, base + i);
    if (s.momentum) {
      const float m = fmaf(s.beta, s.momentum[base + i], s.rest * u);
      s.momentum[base + i] = m;
      u = muon_direction(s, u, m);
    }
    sum = fma((double)u, (double)u, sum);
  }
  for (int off = 16; off; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = sum;
  __syncthreads();
  if (threadIdx.x == 0) {
    double total = 0.0;
    for (int i = 0; i < 8; ++i) total += part[i];
    partial[blockIdx.y * kNormBlocks + blockIdx.x] = total;
  }
}

// S u / (|u| + eps) as hi + lo, eight columns per thread
__global__ void __launch_bounds__(256) ns_split_kernel(Source s, const double *partial, int blocks, int rows, int cols,
                                                       int64_t pitch, int64_t part, double scale, double eps,
                                                       __half *dst) {
  __shared__ double s_factor;
  cudaTriggerProgrammaticLaunchCompletion();
  cudaGridDependencySynchronize();
  if (threadIdx.x < 32) {
    double sum = 0.0;
    for (int i = threadIdx.x; i < blocks; i += 32) sum += partial[blockIdx.y * kNormBlocks + i];
    for (int off = 16; off; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
    if (threadIdx.x == 0) s_factor = scale / (sqrt(sum) + eps);
  }
  __syncthreads();
  const double f64 = s_factor;
  const float f = (float)f64;
  const bool in_32 = f64 > 1e-30 && f64 < 1e30;  // a factor beyond is applied in 64 bits
  const int64_t base = (int64_t)blockIdx.y * rows * cols;
  const int chunks = (int)(pitch / 8);
  const int64_t total = (int64_t)rows * chunks;
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < total; i += (int64_t)gridDim.x * blockDim.x) {
    const int64_t r = i / chunks;
    const int c = (int)(i - r * chunks) * 8;
    __half hi[8], lo[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      float u = 0.0f;
      if (c + e < cols) {
        const int64_t at = base + r * cols + c + e;
        u = load_any(s.in, s.dtype, at);
        if (s.momentum) u = muon_direction(s, u, s.momentum[at]);
      }
      split_half(in_32 ? u * f : (float)((double)u * f64), hi[e], lo[e]);
    }
    __half *at = dst + (int64_t)blockIdx.y * 2 * part + r * pitch + c;
    *reinterpret_cast<uint4 *>(at) = *reinterpret_cast<const uint4 *>(hi);
    *reinterpret_cast<uint4 *>(at + part) = *reinterpret_cast<const uint4 *>(lo);
  }
}

// ---------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------

PFN_cuTensorMapEncodeTiled_v12000 encode_fn() {
  static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void *p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
  });
  return fn;
}

template <typename... P, typename... A>
cudaError_t launch(void (*kernel)(P...), dim3 grid, int threads, size_t smem, cudaStream_t st, bool dependent,
                   int cluster, A... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3((unsigned)threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  int n = 0;
  if (dependent) {
    attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[n++].val.programmaticStreamSerializationAllowed = 1;
  }
  if (cluster > 1) {
    attr[n].id = cudaLaunchAttributeClusterDimension;
    attr[n].val.clusterDim.x = (unsigned)cluster;
    attr[n].val.clusterDim.y = attr[n].val.clusterDim.z = 1;
    ++n;
  }
  cfg.attrs = attr;
  cfg.numAttrs = n;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, args...);
  if (e == cudaSuccess) g_muon_launches.fetch_add(1, std::memory_order_relaxed);
  return e;
}

// [batch][2][rows][pitch]
struct Stack {
  __half *p;
  int64_t batch;
  int rows, cols;
  int64_t pitch, part;
};

int64_t pitch_of(int64_t cols) { return (cols + 7) / 8 * 8; }

int64_t stack_bytes(int64_t batch, int64_t rows, int64_t cols) {
  return (batch * 2 * rows * pitch_of(cols) * 2 + 255) / 256 * 256;
}

// Tensor maps of a call's stacks: [parts][rows][cols] of fp16, each encoded
// once: boxes of 64 columns x box_rows rows to load, or (box_rows = 0) the
// 32 x 32 blocks of an epilogue warp to store.
struct Maps {
  static constexpr int kMost = 20;
  CUtensorMap map[kMost];
  const __half *base[kMost];
  int box[kMost], n = 0;

  const CUtensorMap *get(const Stack &k, int box_rows) {
    for (int i = 0; i < n; ++i)
      if (base[i] == k.p && box[i] == box_rows) return &map[i];
    auto fn = encode_fn();
    if (!fn || n == kMost) return nullptr;
    cuuint64_t dims[3] = {(cuuint64_t)k.cols, (cuuint64_t)k.rows, (cuuint64_t)k.batch * 2};
    cuuint64_t strides[2] = {(cuuint64_t)k.pitch * 2, (cuuint64_t)k.part * 2};
    const bool store = box_rows == 0;
    cuuint32_t shape[3] = {store ? 32u : 64u, store ? 32u : (cuuint32_t)box_rows, 1};
    cuuint32_t estr[3] = {1, 1, 1};
    if (fn(&map[n], CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, k.p, dims, strides, shape, estr,
           CU_TENSOR_MAP_INTERLEAVE_NONE, store ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B,
           CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
      return nullptr;
    base[n] = k.p;
    box[n] = box_rows;
    return &map[n++];
  }
};

// the device: its SMs, and how many clusters of 2, 4 and 8 CTAs of the tile
// kernel it runs at once
struct Device {
  int sms, clusters[4];
};

constexpr int kMaxDevices = 64;

template <bool kAMn, bool kBMn>
cudaError_t set_up() {
  cudaError_t e = cudaFuncSetAttribute(ns_tile_kernel<kAMn, kBMn>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                       TileLayout::kBytes);
  if (e == cudaSuccess)
    e = cudaFuncSetAttribute(ns_pair_kernel<256, kAMn, kBMn>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             PairLayout<256>::kBytes);
  if (e == cudaSuccess)
    e = cudaFuncSetAttribute(ns_pair_kernel<128, kAMn, kBMn>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             PairLayout<128>::kBytes);
  return e;
}

// the current device's properties, read once (and its kernels' shared
// memory allowed); null where that fails
const Device *device() {
  static Device known[kMaxDevices];
  static std::atomic<int> ready[kMaxDevices];
  static std::mutex lock;
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices) return nullptr;
  if (ready[dev].load(std::memory_order_acquire)) return &known[dev];
  std::lock_guard<std::mutex> hold(lock);
  if (ready[dev].load(std::memory_order_relaxed)) return &known[dev];
  Device d = {};
  if (cudaDeviceGetAttribute(&d.sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return nullptr;
  if (set_up<false, false>() != cudaSuccess || set_up<true, true>() != cudaSuccess ||
      set_up<false, true>() != cudaSuccess)
    return nullptr;
  for (int z = 1; z < 4; ++z) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(1u << z);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = TileLayout::kBytes;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = 1u << z;
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    if (cudaOccupancyMaxActiveClusters(&d.clusters[z], ns_tile_kernel<false, false>, &cfg) != cudaSuccess) return nullptr;
  }
  known[dev] = d;
  ready[dev].store(1, std::memory_order_release);
  return &known[dev];
}

int64_t tile_count(const Product &q, int64_t batch, int bm, int bn) {
  const int64_t tm = (q.rows + bm - 1) / bm, tn = (q.cols + bn - 1) / bn;
  if (!q.sym) return tm * tn * batch;
  int64_t n = 0;
  for (int64_t i = 0; i < tm; ++i) {
    const int64_t w = (i * bm + bm - 1) / bn + 1;
    n += w < tn ? w : tn;
  }
  return n * batch;
}

template <int BN, bool kAMn, bool kBMn>
cudaError_t run_pair(Product q, const Stack &a, const Stack &b, const Stack &to, Maps &maps, const Device &d, int64_t tiles,
                     cudaStream_t st) {
  const CUtensorMap *ma = maps.get(a, kAMn ? kBK : kBM), *mb = maps.get(b, kBMn ? kBK : BN / 2);
  const CUtensorMap *md = maps.get(to, 0);
  if (!ma || !mb || !md || tiles > INT32_MAX / 2) return cudaErrorInvalidValue;
  q.tiles_n = (q.cols + BN - 1) / BN;
  q.tiles = (int)tiles;
  q.per_batch = (int)(tiles / a.batch);
  const int pairs = q.tiles < d.sms / 2 ? q.tiles : d.sms / 2;
  return launch(ns_pair_kernel<BN, kAMn, kBMn>, dim3((unsigned)(2 * pairs)), kThreads,
                (size_t)PairLayout<BN>::kBytes, st, true, 1, *ma, *mb, *md, q);
}

// The kernel and the CTAs that share a tile's K.  In units of one stage of a
// 256 x 256 pair tile (0.82 us): a 256 x 128 pair tile's takes 0.6, a
// 128 x 128 tile's 0.8 (it draws the most from L2 per product); splitting
// K costs about 2 more.  What leaves SMs idle is a tile count below a wave,
// or just above one.
template <bool kAMn, bool kBMn>
cudaError_t product(const Product &q, const Stack &a, const Stack &b, const Stack &to, Maps &maps, const Device &d,
                    cudaStream_t st) {
  const int64_t kblocks = (q.k + kBK - 1) / kBK, pairs = d.sms / 2;
  const int64_t p256 = tile_count(q, a.batch, 256, 256), p128 = tile_count(q, a.batch, 256, 128);
  const int64_t t128 = tile_count(q, a.batch, 128, 128);
  const double cost256 = (double)((p256 + pairs - 1) / pairs * kblocks);
  const double cost128 = 0.6 * (double)((p128 + pairs - 1) / pairs * kblocks);
  double best = 0.8 * (double)((t128 + d.sms - 1) / d.sms * kblocks);
  int split = 1;
  for (int z = 1; z < 4 && (1 << z) <= kblocks; ++z) {
    if (t128 > d.clusters[z]) break;
    const double cost = 0.8 * (double)((kblocks + (1 << z) - 1) >> z) + 2.0;
    if (cost < best) {
      best = cost;
      split = 1 << z;
    }
  }
  if (cost256 <= cost128 && cost256 <= best) return run_pair<256, kAMn, kBMn>(q, a, b, to, maps, d, p256, st);
  if (cost128 <= best) return run_pair<128, kAMn, kBMn>(q, a, b, to, maps, d, p128, st);
  const CUtensorMap *ma = maps.get(a, kAMn ? kBK : kBM), *mb = maps.get(b, kBMn ? kBK : TileLayout::kBN);
  const CUtensorMap *md = maps.get(to, 0);
  if (!ma || !mb || !md || t128 * kMaxSplit > INT32_MAX) return cudaErrorInvalidValue;
  Product t = q;
  t.tiles_n = (q.cols + TileLayout::kBN - 1) / TileLayout::kBN;
  t.tiles = (int)t128;
  t.per_batch = (int)(t128 / a.batch);
  return launch(ns_tile_kernel<kAMn, kBMn>, dim3((unsigned)(t.tiles * split)), kThreads, (size_t)TileLayout::kBytes, st,
                true, split, *ma, *mb, *md, t);
}

int newton_schulz(const scacchi_newton_schulz &n, const Source &src, Product last, void *workspace, cudaStream_t st) {
  const Device *dev = device();
  if (!dev) return SCACCHI_ECUDA;
  const int sms = dev->sms;
  Maps maps;
  const int s = n.rows < n.cols ? n.rows : n.cols;
  const bool tall = n.rows > n.cols;
  uint8_t *at = static_cast<uint8_t *>(workspace);
  double *partial = reinterpret_cast<double *>(at);
  at += (size_t)n.batch * kNormBlocks * sizeof(double);
  auto stack = [&](int rows, int cols) {
    Stack k = {reinterpret_cast<__half *>(at), n.batch, rows, cols, pitch_of(cols), rows * pitch_of(cols)};
    at += stack_bytes(n.batch, rows, cols);
    return k;
  };
  Stack x = stack(n.rows, n.cols), y = stack(n.rows, n.cols);
  const Stack gram = stack(s, s), poly = stack(s, s);
  const double scale = ldexp(1.0, n.scale_exponent);
  const int64_t elems = (int64_t)n.rows * n.cols;

  int64_t blocks = (elems + 4095) / 4096;
  const int64_t share = (4 * (int64_t)sms + n.batch - 1) / n.batch;
  blocks = blocks < share ? blocks : share;
  blocks = blocks < kNormBlocks ? blocks : kNormBlocks;
  if (launch(ns_norm_kernel, dim3((unsigned)blocks, (unsigned)n.batch), 256, 0, st, false, 1, src, elems, partial) !=
      cudaSuccess)
    return SCACCHI_ECUDA;
  const int64_t chunks = (int64_t)n.rows * (x.pitch / 8);
  int64_t split_blocks = (chunks + 255) / 256;
  const int64_t split_share = (8 * (int64_t)sms + n.batch - 1) / n.batch;
  split_blocks = split_blocks < split_share ? split_blocks : split_share;
  if (launch(ns_split_kernel, dim3((unsigned)split_blocks, (unsigned)n.batch), 256, 0, st, true, 1, src,
             (const double *)partial, (int)blocks, n.rows, n.cols, x.pitch, x.part, scale, n.eps, x.p) != cudaSuccess)
    return SCACCHI_ECUDA;

  // M = c Z^2 + (a - b^2 / 4c) I with Z = A + (b / 2c) I: the square alone,
  // with shifted diagonals; without c, M = b A + a I takes no product
  const bool quintic = n.c != 0.0;
  for (int k = 0; k < n.steps; ++k) {
    Product q = {};
    q.sym = 1;
    q.rows = q.cols = s;
    q.mode = kGram;
    q.k = tall ? n.rows : n.cols;
    q.scale = (float)((quintic ? 1.0 : n.b) / scale);
    q.diag = (float)((quintic ? n.b / (2.0 * n.c) : n.a) * scale);
    const Stack &first = quintic ? gram : poly;
    cudaError_t e = tall ? product<true, true>(q, x, x, first, maps, *dev, st)
                         : product<false, false>(q, x, x, first, maps, *dev, st);
    if (e != cudaSuccess) return SCACCHI_ECUDA;
    if (quintic) {
      q.mode = kSquare;
      q.k = s;
      q.scale = (float)(n.c / scale);
      q.diag = (float)((n.a - n.b * n.b / (4.0 * n.c)) * scale);
      if (product<false, false>(q, gram, gram, poly, maps, *dev, st) != cudaSuccess) return SCACCHI_ECUDA;
    }
    const bool final = k + 1 == n.steps;
    Product u = final ? last : Product{};
    u.mode = final ? kLast : kUpdate;
    u.scale = (float)(final ? 1.0 / (scale * scale) : 1.0 / scale);
    u.rows = n.rows;
    u.cols = n.cols;
    u.k = s;
    e = tall ? product<false, false>(u, x, poly, y, maps, *dev, st)
             : product<false, true>(u, poly, x, y, maps, *dev, st);
    if (e != cudaSuccess) return SCACCHI_ECUDA;
    const Stack t = x;
    x = y;
    y = t;
  }
  return SCACCHI_OK;
}

bool bad_shape(const scacchi_newton_schulz *n) {
  return !n || n->batch < 0 || n->batch > 65535 || n->rows < 1 || n->cols < 1 || n->rows > SCACCHI_MUON_MAX_SIDE ||
         n->cols > SCACCHI_MUON_MAX_SIDE || n->dtype < 0 || n->dtype > 2 || n->steps < 1 || n->steps > 64 ||
         !isfinite(n->a) || !isfinite(n->b) || !isfinite(n->c) || !(n->eps >= 0.0) || !isfinite(n->eps) ||
         n->scale_exponent < 0 || n->scale_exponent > 15;
}

size_t elem_size(int dtype) { return dtype == 0 ? 4 : 2; }

bool misaligned(const void *p, size_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) != 0; }

}  // namespace

extern "C" {

int32_t scacchi_muon_scale_exponent(double a, double b, double c, int32_t steps) {
  if (!isfinite(a) || !isfinite(b) || !isfinite(c) || steps < 1 || steps > 64) return -1;
  // the shift b / 2c has to stay of the order of A for Z^2 to keep its digits
  const double shift = c == 0.0 ? 0.0 : b / (2.0 * c);
  if (!(fabs(shift) <= 8.0)) return -1;
  // the singular values start in [0, 1]: follow a grid of them through the
  // steps; the operands' entries are at most the largest of sigma,
  // |sigma^2 + shift| and |a + b sigma^2 + c sigma^4|
  double most = 1.0;
  for (int i = 0; i <= 4096; ++i) {
    double v = i / 4096.0;
    for (int k = 0; k < steps; ++k) {
      const double v2 = v * v, p = a + v2 * (b + c * v2);
      most = fmax(most, fmax(fabs(p), fmax(fabs(v), fmax(v2, fabs(v2 + shift)))));
      if (!(most < 1e6)) return -1;
      v *= p;
    }
    most = fmax(most, fabs(v));
    if (!(most < 1e6)) return -1;
  }
  int e = 15;
  while (e >= 0 && ldexp(1.1 * most, e) > 65504.0) --e;
  // fewer than 2^6 steps between 1 and the largest value left: diverging
  return e >= 6 ? e : -1;
}

size_t scacchi_muon_workspace_bytes(int32_t batch, int32_t rows, int32_t cols) {
  if (batch < 1 || rows < 1 || cols < 1) return 0;
  const int64_t s = rows < cols ? rows : cols;
  return (size_t)batch * kNormBlocks * sizeof(double) + 2 * (size_t)stack_bytes(batch, rows, cols) +
         2 * (size_t)stack_bytes(batch, s, s);
}

int scacchi_orthogonalize(const scacchi_newton_schulz *params, const void *matrix, void *out, void *workspace,
                          void *stream) {
  if (bad_shape(params)) return SCACCHI_EINVAL;
  if (params->batch == 0) return SCACCHI_OK;
  const size_t size = elem_size(params->dtype);
  if (!matrix || !out || !workspace || misaligned(matrix, size) || misaligned(out, size) || misaligned(workspace, 256))
    return SCACCHI_EINVAL;
  Source src = {};
  src.in = matrix;
  src.dtype = params->dtype;
  Product last = {};
  last.out = out;
  last.dtype = params->dtype;
  return newton_schulz(*params, src, last, workspace, static_cast<cudaStream_t>(stream));
}

int scacchi_muon_update(const scacchi_newton_schulz *params, const void *gradient, float *momentum, float *weight,
                        double beta, int32_t nesterov, float decay, float step, void *workspace, void *stream) {
  if (bad_shape(params) || !(beta >= 0.0 && beta < 1.0) || !isfinite(decay) || !isfinite(step))
    return SCACCHI_EINVAL;
  if (params->batch == 0) return SCACCHI_OK;
  if (!gradient || !momentum || !weight || !workspace || misaligned(gradient, elem_size(params->dtype)) ||
      misaligned(momentum, 4) || misaligned(weight, 4) || misaligned(workspace, 256))
    return SCACCHI_EINVAL;
  Source src = {};
  src.in = gradient;
  src.dtype = params->dtype;
  src.momentum = momentum;
  src.beta = (float)beta;
  src.rest = (float)(1.0 - beta);
  src.nesterov = nesterov != 0;
  Product last = {};
  last.weight = weight;
  last.decay = decay;
  last.step = step;
  return newton_schulz(*params, src, last, workspace, static_cast<cudaStream_t>(stream));
}

int scacchi_muon_error(uint32_t *flags) {
  if (!flags) return SCACCHI_EINVAL;
  uint32_t zero = 0;
  if (cudaMemcpyFromSymbol(flags, g_muon_error, sizeof(uint32_t)) != cudaSuccess) return SCACCHI_ECUDA;
  if (*flags && cudaMemcpyToSymbol(g_muon_error, &zero, sizeof(uint32_t)) != cudaSuccess) return SCACCHI_ECUDA;
  return SCACCHI_OK;
}

uint64_t scacchi_muon_launch_count(void) { return g_muon_launches.load(std::memory_order_relaxed); }

}  // extern "C"
