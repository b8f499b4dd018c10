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
// Layout.  An operand is stored in panels of 64 columns, each row of a panel
// 128 bytes with its 16-byte chunks already in the 128B-swizzled order of
// shared memory (chunk c of row r at c ^ (r & 7)).  Any rows of a panel are
// one contiguous piece, which serves as a K-major tile (the panel along K)
// or an MN-major one (its rows along K) alike, and an epilogue warp's 32
// rows leave as one 4 KB copy.  Rows are padded to 64 and columns to whole
// panels with zeros, which every product keeps zero, so any size works.
//
// A and A^2 are symmetric: only blocks on and below the diagonal of 256 x 256
// blocks are computed and stored; one above it is read as its mirror image,
// MN-major for K-major.
//
// What bounds it (device times, by graph replays): at 2048 x 2048 and above
// the tensor cores, three products for one, at 1.1 PFLOP/s (2048 x 2048 fp32
// 452 us for 515 GFLOP issued; the pair kernel keeps the tensor pipe busy for
// 73 % of a CTA's time); below, latency: seventeen dependent launches of 7 us
// or more (300 x 300 117 us), or for narrow matrices one launch's phases
// (162 x 82 49 us).
//
// Every wait is bounded (2 s).  One that runs out raises g_muon_error and, in
// the kernels of one product, the call's flag in its workspace; a narrow
// matrix, or any whose flag stands before the last product, is not written.

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
constexpr int kBK = 64;            // K of a stage: a panel
constexpr int kSym = 256;          // blocks of a symmetric matrix that are stored whole
constexpr int kBox = 64 * kBK * 2; // 64 rows of a panel
constexpr int kEpiWarps = 8;       // two per TMEM lane quadrant, half the tile's columns each
constexpr int kThreads = 128 + 32 * kEpiWarps;  // producer, MMA issuer, two idle warps; epilogue
// The pair kernel's registers per thread: kLaunchRegisters at launch (the
// host checks that the build has them), shared out again for the sums:
// 128 x 48 + 256 x 224 = 63488 of 384 x 168 = 64512.
constexpr int kLaunchRegisters = 168, kFewRegisters = 48, kManyRegisters = 224;
static_assert(128 * kFewRegisters + 32 * kEpiWarps * kManyRegisters <= kThreads * kLaunchRegisters,
              "setmaxnreg would wait forever");
constexpr int kMaxSplit = 8;       // CTAs of a cluster that share a tile's K
constexpr int kNormBlocks = 1024;  // most partial sums of squares per matrix
constexpr int kPatch = 32 * 32 * 4;  // an epilogue warp's 32 x 32 block in fp32

__device__ uint32_t g_muon_error;
std::atomic<uint64_t> g_muon_launches{0};

enum Major : int { kAlongK = 0, kAlongMN = 1, kSymmetric = 2 };  // of an operand: K-, MN-major, or by the block

struct Product {
  int last, sym;                // the last update, and a symmetric output
  int a_major, b_major;
  int a_rows, b_rows;           // padded rows of the operands' panels
  int rows, cols, k;            // of the output, and the summed length
  int tiles_n, per_batch, tiles;
  float scale, diag;            // the output is scale acc + diag on the diagonal
  __half *dst;                  // an operand of the next product: [batch][2][panel][dst_rows][64]
  int dst_rows, dst_panels;
  // last: the result, or the weight's step w <- decay w - step x
  void *out;
  int dtype;                    // 0 float32, 1 bfloat16, 2 float16
  float *weight;
  float decay, step;
  uint32_t *failed;             // of this call: a wait of one of its products ran out
};

// Whether a product's output is written: the user's matrix is not once an
// earlier product of the call was left unfinished.
__device__ __forceinline__ bool may_write(const Product &q) { return !q.last || __ldcg(q.failed) == 0u; }

// Tiles of tile row i of a symmetric output: those of the stored blocks, of
// which 128 x 128 tiles leave out the one that its neighbour writes turned.
template <int BM, int BN>
__host__ __device__ __forceinline__ int row_tiles(int i, int tiles_n) {
  const int n = BM == BN && BM < kSym ? i + 1 : ((i * BM) / kSym + 1) * (kSym / BN);
  return n < tiles_n ? n : tiles_n;
}

// A tile's place: matrix, tile row (of BM rows), tile column.
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
  for (int n; u >= (n = row_tiles<BM, BN>(i, q.tiles_n)); ++i) u -= n;
  j = u;
}

// Whether the 64 K of stage kb are read MN-major for rows `at`.. of an operand
__device__ __forceinline__ bool along_mn(int major, int at, int kb) {
  return major == kAlongMN || (major == kSymmetric && kb / (kSym / kBK) > at / kSym);
}

// one part of a stage's operand: `rows` of the output's rows or columns
// (from `at`) by 64 of K, in boxes of 64 rows of a panel
template <typename Load>
__device__ __forceinline__ void load_operand(uint8_t *dst, int rows, int at, int kb, bool mn, int panel_rows,
                                             Load load) {
  for (int m = 0; m < rows; m += 64, dst += kBox)
    load(dst, mn ? ((at + m) / 64) * panel_rows + kb * kBK : kb * panel_rows + at + m);
}

// Descriptors of a stage's operands: the first stage's, advanced by whole
// 16-byte units (an address stays within the field's 14 bits).  The MMA
// warp keeps its control flow uniform and elects a lane for the issue alone.
struct StageDesc {
  uint64_t a, b;
  uint32_t a_part, b_part, a_step, b_step;
  __device__ __forceinline__ StageDesc(uint32_t stage, uint32_t a_bytes, uint32_t b_bytes, bool a_mn, bool b_mn) {
    a = desc_sw128(stage, a_mn);
    b = desc_sw128(stage + 2 * a_bytes, b_mn);
    a_part = a_bytes >> 4;
    b_part = b_bytes >> 4;
    a_step = a_mn ? 2048u >> 4 : 32u >> 4;
    b_step = b_mn ? 2048u >> 4 : 32u >> 4;
  }
  // hi lo, lo hi, hi hi: the small products first
  __device__ __forceinline__ uint64_t a_of(int term, int k) const { return a + (term == 1 ? a_part : 0u) + k * a_step; }
  __device__ __forceinline__ uint64_t b_of(int term, int k) const { return b + (term == 0 ? b_part : 0u) + k * b_step; }
};

// eight values as hi and lo halves
__device__ __forceinline__ void split8(const float *v, uint4 &hi, uint4 &lo) {
  uint32_t h[4], l[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const __half2 a = __floats2half2_rn(v[2 * e], v[2 * e + 1]);
    const float2 f = __half22float2(a);
    const __half2 b = __floats2half2_rn(v[2 * e] - f.x, v[2 * e + 1] - f.y);
    h[e] = *reinterpret_cast<const uint32_t *>(&a);
    l[e] = *reinterpret_cast<const uint32_t *>(&b);
  }
  hi = make_uint4(h[0], h[1], h[2], h[3]);
  lo = make_uint4(l[0], l[1], l[2], l[3]);
}

// Place of row `row`, 4-float chunk `chunk` in an epilogue patch: rows of
// 32 floats, chunks swizzled so that a row per lane, eight columns of a row
// per lane and a column per lane all spread over the banks.
__device__ __forceinline__ int patch_at(int row, int chunk) {
  return row * 32 + ((chunk ^ ((row ^ (row >> 3)) & 7)) << 2);
}

// What becomes of a warp's 32 rows (a row per lane) by COLS columns, 32
// columns at a time: turned through the warp's patch of shared memory, then
// written in whole pieces of rows, as hi + lo in the panels of the next
// product's operand, or to the user's matrix.
//
// `mirror`: written turned as well, in the place of a tile that is not
// computed.
//
// This code runs once per tile, so what it costs is mostly fetching it:
// unrolled over the blocks (some 40 KB of instructions) it took 4 us for a
// warp's 32 columns, rolled 1 us.
template <int COLS>
__device__ __forceinline__ void emit(const Product &q, int batch, int r0, int c_first, bool mirror,
                                     const float (&sum)[COLS], float *patch) {
  const int lane = threadIdx.x & 31;
#pragma unroll 1
  for (int g = 0; g < COLS / 32; ++g) {
    const int c0 = c_first + 32 * g;
    if (q.last ? r0 >= q.rows || c0 >= q.cols : r0 >= q.dst_rows || c0 >= q.dst_panels * 64) break;
#pragma unroll
    for (int i = 0; i < COLS / 32; ++i)
      if (i == g) {
#pragma unroll
        for (int k = 0; k < 8; ++k)
          *reinterpret_cast<float4 *>(patch + patch_at(lane, k)) = make_float4(
              sum[32 * i + 4 * k], sum[32 * i + 4 * k + 1], sum[32 * i + 4 * k + 2], sum[32 * i + 4 * k + 3]);
      }
    __syncwarp();
    if (q.last) {
      // a column per lane
      const int64_t base = ((int64_t)batch * q.rows + r0) * q.cols + c0 + lane;
      const int n = q.rows - r0 < 32 ? q.rows - r0 : 32;
      if (c0 + lane < q.cols) {
        if (q.weight) {
          // half of the block's weights are requested before the first is used
#pragma unroll 1
          for (int half = 0; half < n; half += 16) {
            float w[16];
#pragma unroll
            for (int e = 0; e < 16; ++e)
              if (half + e < n) w[e] = q.weight[base + (int64_t)(half + e) * q.cols];
#pragma unroll
            for (int e = 0; e < 16; ++e)
              if (half + e < n)
                q.weight[base + (int64_t)(half + e) * q.cols] =
                    fmaf(-q.step, patch[patch_at(half + e, lane >> 2) + (lane & 3)] * q.scale, q.decay * w[e]);
          }
        } else {
#pragma unroll 8
          for (int row = 0; row < n; ++row) {
            const float y = patch[patch_at(row, lane >> 2) + (lane & 3)] * q.scale;
            const int64_t at = base + (int64_t)row * q.cols;
            if (q.dtype == 0)
              static_cast<float *>(q.out)[at] = y;
            else if (q.dtype == 1)
              static_cast<__nv_bfloat16 *>(q.out)[at] = __float2bfloat16_rn(y);
            else
              static_cast<__half *>(q.out)[at] = __float2half_rn(y);
          }
        }
      }
    } else {
      // eight columns of a row per lane: 64 bytes of eight rows at a time;
      // turned, eight rows of a column
      const int64_t part = (int64_t)q.dst_panels * q.dst_rows * 64;
      const int oct = lane & 3;
#pragma unroll 1
      for (int turned = 0; turned <= (int)mirror; ++turned) {
        const int rows_at = turned ? c0 : r0, cols_at = turned ? r0 : c0, chunk = (cols_at & 32) / 8 + oct;
        if (rows_at >= q.dst_rows || cols_at >= q.dst_panels * 64) break;
        __half *to = q.dst + (int64_t)batch * 2 * part + ((int64_t)(cols_at / 64) * q.dst_rows + rows_at) * 64;
        // row - column offset of the diagonal
        const int diagonal = q.diag != 0.0f ? cols_at + 8 * oct - rows_at : 1 << 30;
#pragma unroll 2
        for (int row = lane >> 2; row < 32; row += 8) {
          float y[8];
          if (turned) {
#pragma unroll
            for (int e = 0; e < 8; ++e) y[e] = patch[patch_at(8 * oct + e, row >> 2) + (row & 3)];
          } else {
            *reinterpret_cast<float4 *>(y) = *reinterpret_cast<const float4 *>(patch + patch_at(row, 2 * oct));
            *reinterpret_cast<float4 *>(y + 4) = *reinterpret_cast<const float4 *>(patch + patch_at(row, 2 * oct + 1));
          }
#pragma unroll
          for (int e = 0; e < 8; ++e)
            y[e] = y[e] * q.scale + (row - diagonal == e && rows_at + row < q.rows ? q.diag : 0.0f);
          uint4 hi, lo;
          split8(y, hi, lo);
          __half *at = to + row * 64 + ((chunk ^ (row & 7)) << 3);
          *reinterpret_cast<uint4 *>(at) = hi;
          *reinterpret_cast<uint4 *>(at + part) = lo;
        }
      }
    }
    __syncwarp();
  }
}

// The tensor core truncates each time it adds to a TMEM accumulator: about
// 1.5e-7 of the result per MMA once five steps have amplified it, 5.7e-5
// at K = 2048.  So an accumulator takes one stage (K = 64), its eight small
// cross products before the four large ones, and the epilogue warps add the
// stages in fp32 registers, rounding to nearest, while the next stage runs
// on the other accumulator (2.3e-6 at 2048 x 2048, where 32-bit arithmetic
// gives 3.4e-6).
template <int COLS>
__device__ __forceinline__ void add_stage(float (&sum)[COLS], uint32_t acc) {
#pragma unroll
  for (int g = 0; g < COLS / 16; ++g) {
    uint32_t v[16];
    tmem_ld16(acc + g * 16, v);
    tmem_wait_ld();
#pragma unroll
    for (int e = 0; e < 16; ++e) sum[g * 16 + e] += __uint_as_float(v[e]);
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
  static constexpr int kSlots = 512 / BN;                          // accumulators in TMEM
  static constexpr int kPatches = kStages * kStage;
  static constexpr int kBars = kPatches + kEpiWarps * kPatch;
  static constexpr int kBytes = kBars + 8 * (2 * kStages + 2 * kSlots) + 16 + 1024;  // + alignment slack
  static_assert(kBytes <= 227 * 1024, "shared memory budget");
};

// D[i, j] = A[i, k] B[j, k], persistent over the tiles.
//
// A single CTA's 128 x 256 tile needs 96 KB of operands per stage, which
// its shared memory cannot take in while the MMAs read theirs (240 KB of
// 128 bytes a clock: 1.08 us a stage, against 0.82 us of MMA).  A pair
// shares B: 64 KB a CTA.
template <int BN>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
    ns_pair_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
                   const __grid_constant__ Product q) {
  using L = PairLayout<BN>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  uint64_t *full = reinterpret_cast<uint64_t *>(smem + L::kBars);  // the even CTA's counts both CTAs' loads
  uint64_t *empty = full + L::kStages;
  uint64_t *acc_full = empty + L::kStages;
  uint64_t *acc_empty = acc_full + L::kSlots;                      // the even CTA's counts both epilogues
  uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(acc_empty + L::kSlots);
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
    for (int s = 0; s < L::kSlots; ++s) {
      mbar_init(&acc_full[s], 1);
      mbar_init(&acc_empty[s], 2 * kEpiWarps);
    }
    *abort_flag = 0;
    fence_barrier_init();
  }
  __syncwarp();
  if (warp == 1) {
    tmem_alloc_pair(tmem_slot, 512);
    tmem_relinquish_pair();
  }
  tc_fence_before();
  cg::this_cluster().sync();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  cudaTriggerProgrammaticLaunchCompletion();
  cudaGridDependencySynchronize();

  if (warp < 4) {
    registers_dec<kFewRegisters>();
    if (warp == 0 && lane == 0) {
      int stage = 0;
      uint32_t phase = 0, issued = 0, parity = 0;
      bool stop = false;
      for (int t = first; t < q.tiles && !stop; t += step) {
        int batch, i, j;
        locate<2 * kBM, BN>(q, t, batch, i, j);
        const int a_at = (2 * i + rank) * kBM, b_at = j * BN + rank * (BN / 2);
        for (int kb = 0; kb < kblocks; ++kb) {
          if (*abort_flag || !mbar_wait(&empty[stage], phase ^ 1u, abort_flag, &g_muon_error, q.failed)) {
            stop = true;
            break;
          }
          uint8_t *at = smem + stage * L::kStage;
          const uint32_t bar = cluster_addr(smem_u32(&full[stage]), 0);
          if (rank == 0) mbar_expect_tx(&full[stage], 2 * L::kStage);
          const bool a_mn = along_mn(q.a_major, a_at, kb), b_mn = along_mn(q.b_major, b_at, kb);
#pragma unroll
          for (int part = 0; part < 2; ++part) {
            load_operand(at + part * L::kA, kBM, a_at, kb, a_mn, q.a_rows,
                         [&](uint8_t *dst, int y) { tma_load_3d_pair(dst, &map_a, bar, 0, y, 2 * batch + part); });
            load_operand(at + 2 * L::kA + part * L::kB, BN / 2, b_at, kb, b_mn, q.b_rows,
                         [&](uint8_t *dst, int y) { tma_load_3d_pair(dst, &map_b, bar, 0, y, 2 * batch + part); });
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
    } else if (warp == 1 && rank == 0) {
      int stage = 0, slot = 0;
      uint32_t phase = 0, acc_phase = 0;
      bool ok = true;
      for (int t = first; t < q.tiles && ok; t += step) {
        int batch, i, j;
        locate<2 * kBM, BN>(q, t, batch, i, j);
        for (int kb = 0; kb < kblocks; ++kb) {
          // one mode for the pair: its rows lie within one stored block
          const bool a_mn = along_mn(q.a_major, 2 * i * kBM, kb), b_mn = along_mn(q.b_major, j * BN, kb);
          const StageDesc desc(smem_u32(smem + stage * L::kStage), L::kA, L::kB, a_mn, b_mn);
          const uint32_t idesc = idesc_f16(2 * kBM, BN, a_mn, b_mn), d = tmem + (uint32_t)(slot * BN);
          ok = mbar_wait_warp(&acc_empty[slot], acc_phase ^ 1u, abort_flag, &g_muon_error, q.failed) &&
               mbar_wait_warp(&full[stage], phase, abort_flag, &g_muon_error, q.failed);
          if (!ok) break;
          tc_fence_after();
          if (elect_one()) {
#pragma unroll
            for (int term = 0; term < 3; ++term)
#pragma unroll
              for (int k = 0; k < kBK / 16; ++k)
                umma_f16_pair(d, desc.a_of(term, k), desc.b_of(term, k), idesc, (term | k) != 0);
            umma_commit_pair(&empty[stage]);
            umma_commit_pair(&acc_full[slot]);
          }
          __syncwarp();
          if (++stage == L::kStages) {
            stage = 0;
            phase ^= 1u;
          }
          if (++slot == L::kSlots) {
            slot = 0;
            acc_phase ^= 1u;
          }
        }
      }
    }
  } else {
    registers_inc<kManyRegisters>();
    constexpr int kCols = BN / 2;              // columns of a warp
    const int quad = warp & 3;                 // the TMEM lanes this warp may read
    const int half = (warp - 4) >> 2;
    float *patch = reinterpret_cast<float *>(smem + L::kPatches + (warp - 4) * kPatch);
    int slot = 0;
    uint32_t acc_phase = 0;
    bool ok = true;
    for (int t = first; t < q.tiles && ok; t += step) {
      float sum[kCols];
#pragma unroll
      for (int e = 0; e < kCols; ++e) sum[e] = 0.0f;
      for (int kb = 0; kb < kblocks; ++kb) {
        int go = 0;
        if (lane == 0) go = !*abort_flag && mbar_wait(&acc_full[slot], acc_phase, abort_flag, &g_muon_error, q.failed);
        ok = __shfl_sync(0xffffffffu, go, 0) != 0;
        if (!ok) break;
        tc_fence_after();
        add_stage<kCols>(sum, tmem + (uint32_t)(slot * BN + half * kCols) + ((uint32_t)(quad * 32) << 16));
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_cluster(cluster_addr(smem_u32(&acc_empty[slot]), 0));
        if (++slot == L::kSlots) {
          slot = 0;
          acc_phase ^= 1u;
        }
      }
      if (!ok) break;
      int batch, i, j;
      locate<2 * kBM, BN>(q, t, batch, i, j);
      if (may_write(q))
        emit<kCols>(q, batch, (2 * i + rank) * kBM + quad * 32, j * BN + half * kCols, false, sum, patch);
    }
  }
  __syncwarp();
  tc_fence_before();
  cg::this_cluster().sync();
  if (warp == 1) tmem_dealloc_pair(tmem, 512);
}

// ---------------------------------------------------------------------------
// one 128 x 128 tile per CTA, or per cluster
// ---------------------------------------------------------------------------

struct TileLayout {
  static constexpr int kBN = 128;
  static constexpr int kA = kBM * kBK * 2, kB = kBN * kBK * 2;
  static constexpr int kStage = 2 * (kA + kB);
  static constexpr int kStages = 3;
  static constexpr int kSlots = 4;
  static constexpr int kPatches = kStages * kStage;
  static constexpr int kBars = kPatches + kEpiWarps * kPatch;
  static constexpr int kBytes = kBars + 8 * (2 * kStages + 2 * kSlots) + 16 + 1024;  // + alignment slack
  static_assert(kBytes <= 227 * 1024, "shared memory budget");
  static_assert((16 + kMaxSplit) * 32 * 32 * 4 <= kPatches, "the partial sums take the stages' place");
};

// The same product for outputs of few tiles: the CTAs of a cluster share one
// tile's K, each finishing its share of the columns from all of them through
// distributed shared memory, so that a small output with a long sum does
// not leave most SMs idle.
__global__ void __launch_bounds__(kThreads, 1)
    ns_tile_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
                   const __grid_constant__ Product q) {
  using L = TileLayout;
  constexpr int BN = L::kBN;
  extern __shared__ uint8_t smem_raw[];
  uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  uint64_t *full = reinterpret_cast<uint64_t *>(smem + L::kBars);
  uint64_t *empty = full + L::kStages;
  uint64_t *acc_full = empty + L::kStages;
  uint64_t *acc_empty = acc_full + L::kSlots;
  uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(acc_empty + L::kSlots);
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
    for (int s = 0; s < L::kSlots; ++s) {
      mbar_init(&acc_full[s], 1);
      mbar_init(&acc_empty[s], kEpiWarps);
    }
    *abort_flag = 0;
    fence_barrier_init();
  }
  __syncwarp();
  if (warp == 1) {
    tmem_alloc(tmem_slot, 512);
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
        if (*abort_flag || !mbar_wait(&empty[stage], phase ^ 1u, abort_flag, &g_muon_error, q.failed)) break;
        uint8_t *at = smem + stage * L::kStage;
        mbar_expect_tx(&full[stage], L::kStage);
        const bool a_mn = along_mn(q.a_major, i * kBM, kb), b_mn = along_mn(q.b_major, j * BN, kb);
#pragma unroll
        for (int part = 0; part < 2; ++part) {
          load_operand(at + part * L::kA, kBM, i * kBM, kb, a_mn, q.a_rows,
                       [&](uint8_t *dst, int y) { tma_load_3d(dst, &map_a, &full[stage], 0, y, 2 * batch + part); });
          load_operand(at + 2 * L::kA + part * L::kB, BN, j * BN, kb, b_mn, q.b_rows,
                       [&](uint8_t *dst, int y) { tma_load_3d(dst, &map_b, &full[stage], 0, y, 2 * batch + part); });
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
    for (int kb = kb0; kb < kb1; ++kb) {
      const bool a_mn = along_mn(q.a_major, i * kBM, kb), b_mn = along_mn(q.b_major, j * BN, kb);
      const StageDesc desc(smem_u32(smem + stage * L::kStage), L::kA, L::kB, a_mn, b_mn);
      const uint32_t idesc = idesc_f16(kBM, BN, a_mn, b_mn), d = tmem + (uint32_t)(slot * BN);
      if (!mbar_wait_warp(&acc_empty[slot], acc_phase ^ 1u, abort_flag, &g_muon_error, q.failed) ||
          !mbar_wait_warp(&full[stage], phase, abort_flag, &g_muon_error, q.failed))
        break;
      tc_fence_after();
      if (elect_one()) {
#pragma unroll
        for (int term = 0; term < 3; ++term)
#pragma unroll
          for (int k = 0; k < kBK / 16; ++k)
            umma_f16(d, desc.a_of(term, k), desc.b_of(term, k), idesc, (term | k) != 0);
        umma_commit(&empty[stage]);
        umma_commit(&acc_full[slot]);
      }
      __syncwarp();
      if (++stage == L::kStages) {
        stage = 0;
        phase ^= 1u;
      }
      if (++slot == L::kSlots) {
        slot = 0;
        acc_phase ^= 1u;
      }
    }
  } else if (warp >= 4) {
    constexpr int kCols = BN / 2;              // columns of a warp: a panel
    const int quad = warp & 3;                 // the TMEM lanes this warp may read
    const int half = (warp - 4) >> 2;
    float *patch = reinterpret_cast<float *>(smem + L::kPatches + (warp - 4) * kPatch);
    int slot = 0;
    uint32_t acc_phase = 0;
    bool ok = true;
    float sum[kCols];
#pragma unroll
    for (int e = 0; e < kCols; ++e) sum[e] = 0.0f;
    for (int kb = kb0; kb < kb1; ++kb) {
      int go = 0;
      if (lane == 0) go = !*abort_flag && mbar_wait(&acc_full[slot], acc_phase, abort_flag, &g_muon_error, q.failed);
      ok = __shfl_sync(0xffffffffu, go, 0) != 0;
      if (!ok) break;
      tc_fence_after();
      add_stage<kCols>(sum, tmem + (uint32_t)(slot * BN + half * kCols) + ((uint32_t)(quad * 32) << 16));
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&acc_empty[slot]);
      if (++slot == L::kSlots) {
        slot = 0;
        acc_phase ^= 1u;
      }
    }
    // the tile right of it in the diagonal's 256 x 256 block is its mirror image
    const bool mirror = q.sym && (i & 1) && j == i - 1;
    if (ctas == 1) {
      if (ok && may_write(q)) emit<kCols>(q, batch, i * kBM + quad * 32, j * BN + half * kCols, mirror, sum, patch);
    } else {
      // The CTAs finish the tile's sixteen 32 x 32 blocks in turn, a warp
      // each; the others' partial sums arrive as [source][block][four
      // elements][lane].
      const int most = (16 + ctas - 1) / ctas;
      __syncwarp();
      cg::this_cluster().sync();  // every CTA is done with its stages
#pragma unroll
      for (int g = 0; g < kCols / 32; ++g) {
        const int id = (half * (kCols / 32) + g) * 4 + quad;
        float4 *to = cg::this_cluster().map_shared_rank(reinterpret_cast<float4 *>(smem), id % ctas);
        to += (rank * most + id / ctas) * 256 + lane;
#pragma unroll
        for (int e = 0; e < 8; ++e)
          to[e * 32] = make_float4(sum[32 * g + 4 * e], sum[32 * g + 4 * e + 1], sum[32 * g + 4 * e + 2],
                                   sum[32 * g + 4 * e + 3]);
      }
      cg::this_cluster().sync();
      const int id = (warp - 4) * ctas + rank;
      if (warp - 4 < most && id < 16 && ok && may_write(q)) {
        const float4 *at = reinterpret_cast<const float4 *>(smem) + (warp - 4) * 256 + lane;
        float v[32];
#pragma unroll
        for (int e = 0; e < 32; ++e) v[e] = 0.0f;
        for (int from = 0; from < ctas; ++from)
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float4 f = at[from * most * 256 + e * 32];
            v[4 * e] += f.x;
            v[4 * e + 1] += f.y;
            v[4 * e + 2] += f.z;
            v[4 * e + 3] += f.w;
          }
        emit<32>(q, batch, i * kBM + (id & 3) * 32, j * BN + (id >> 2) * 32, mirror, v, patch);
      }
    }
  }
  if (ctas > 1 && warp < 4) {  // the epilogue's two cluster barriers are everyone's
    __syncwarp();
    cg::this_cluster().sync();
    cg::this_cluster().sync();
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) tmem_dealloc(tmem, 512);
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

__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }

__device__ __forceinline__ float muon_direction(const Source &s, float g, float m) {
  return s.nesterov ? fmaf(s.beta, m, s.rest * g) : m;
}

// sum of eight squares, in 64 bits where 32 would lose them (a conversion
// per element takes the time of the load)
__device__ __forceinline__ double sum_of_squares(const float (&u)[8]) {
  float s = 0.0f, most = 0.0f;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    s = fmaf(u[e], u[e], s);
    most = fmaxf(most, fabsf(u[e]));
  }
  if (most == 0.0f || (most > 1e-15f && most < 1e18f)) return (double)s;  // NaN stays in s
  double d = 0.0;
  for (int e = 0; e < 8; ++e) d = fma((double)u[e], (double)u[e], d);
  return d;
}

// eight neighbouring elements as floats; `vec`: they start on 16 bytes
template <typename T>
__device__ __forceinline__ void load8(const T *p, bool vec, int left, float (&f)[8]) {
  if (vec) {
    constexpr int kWords = 8 * (int)sizeof(T) / 16;
    uint4 raw[kWords];
#pragma unroll
    for (int i = 0; i < kWords; ++i) raw[i] = reinterpret_cast<const uint4 *>(p)[i];
    const T *v = reinterpret_cast<const T *>(raw);
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = to_f(v[e]);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = e < left ? to_f(p[e]) : 0.0f;
  }
}

template <typename T>
__device__ __forceinline__ double norm_part(const Source &s, int64_t base, int64_t elems, bool vec) {
  const T *in = static_cast<const T *>(s.in) + base;
  float *momentum = s.momentum ? s.momentum + base : nullptr;
  const int64_t stride = (int64_t)gridDim.x * blockDim.x * 8;
  double sum = 0.0;
#pragma unroll 2
  for (int64_t i = ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) * 8; i < elems; i += stride) {
    const int left = elems - i < 8 ? (int)(elems - i) : 8;
    float u[8], m[8];
    load8(in + i, vec, left, u);
    if (momentum) {
      load8(momentum + i, vec, left, m);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        m[e] = fmaf(s.beta, m[e], s.rest * u[e]);
        u[e] = muon_direction(s, u[e], m[e]);
      }
      if (vec) {
        *reinterpret_cast<float4 *>(momentum + i) = make_float4(m[0], m[1], m[2], m[3]);
        *reinterpret_cast<float4 *>(momentum + i + 4) = make_float4(m[4], m[5], m[6], m[7]);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (e < left) momentum[i + e] = m[e];
      }
    }
    sum += sum_of_squares(u);
  }
  return sum;
}

// sum of squares of each matrix (in 64 bits: an update may be small enough
// that its squares leave fp32), one partial per block, and Muon's momentum.
// Bound by memory: 8192 x 2048 bf16 14 us (2.4 TB/s; 70 with 128 blocks of
// single elements)
__global__ void __launch_bounds__(256) ns_norm_kernel(Source s, int64_t elems, int vec, double *partial,
                                                      uint32_t *failed) {
  __shared__ double part[8];
  if (blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x == 0) *failed = 0;
  const int64_t base = (int64_t)blockIdx.y * elems;
  double sum = s.dtype == 0   ? norm_part<float>(s, base, elems, vec)
               : s.dtype == 1 ? norm_part<__nv_bfloat16>(s, base, elems, vec)
                              : norm_part<__half>(s, base, elems, vec);
  for (int off = 16; off; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = sum;
  __syncthreads();
  if (threadIdx.x == 0) {
    double total = 0.0;
    for (int i = 0; i < 8; ++i) total += part[i];
    partial[(int64_t)blockIdx.y * gridDim.x + blockIdx.x] = total;
  }
}

// S u / (|u| + eps) as hi + lo in panels, a 16-byte chunk of each per thread:
// 8192 x 2048 bf16 21 us (4.8 TB/s)
__global__ void __launch_bounds__(256) ns_split_kernel(Source s, const double *partial, int blocks, int rows, int cols,
                                                       int panel_rows, int panels, int vec, double scale, double eps,
                                                       __half *dst) {
  __shared__ double s_factor;
  cudaTriggerProgrammaticLaunchCompletion();
  cudaGridDependencySynchronize();
  if (threadIdx.x < 32) {
    double sum = 0.0;
    for (int i = threadIdx.x; i < blocks; i += 32) sum += partial[(int64_t)blockIdx.y * blocks + i];
    for (int off = 16; off; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
    if (threadIdx.x == 0) s_factor = scale / (sqrt(sum) + eps);
  }
  __syncthreads();
  const double f64 = s_factor;
  const float f = (float)f64;
  const bool in_32 = f64 > 1e-30 && f64 < 1e30;  // a factor beyond is applied in 64 bits
  const int64_t base = (int64_t)blockIdx.y * rows * cols;
  const int chunks = panels * 8;
  const int64_t total = (int64_t)panel_rows * chunks, part = (int64_t)panels * panel_rows * 64;
  __half *out = dst + (int64_t)blockIdx.y * 2 * part;
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < total; i += (int64_t)gridDim.x * blockDim.x) {
    const int64_t r = i / chunks;
    const int c8 = (int)(i - r * chunks), c = c8 * 8;
    float u[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) u[e] = 0.0f;
    const int left = r < rows ? (cols - c < 8 ? cols - c : 8) : 0;
    if (left > 0) {
      const int64_t at = base + r * cols + c;
      if (s.dtype == 0)
        load8(static_cast<const float *>(s.in) + at, vec, left, u);
      else if (s.dtype == 1)
        load8(static_cast<const __nv_bfloat16 *>(s.in) + at, vec, left, u);
      else
        load8(static_cast<const __half *>(s.in) + at, vec, left, u);
      if (s.momentum) {
        float m[8];
        load8(s.momentum + at, vec, left, m);
#pragma unroll
        for (int e = 0; e < 8; ++e) u[e] = muon_direction(s, u[e], m[e]);
      }
      if (in_32) {
#pragma unroll
        for (int e = 0; e < 8; ++e) u[e] *= f;
      } else {
        for (int e = 0; e < 8; ++e) u[e] = (float)((double)u[e] * f64);
      }
    }
    uint4 hi, lo;
    split8(u, hi, lo);
    __half *at = out + ((int64_t)(c8 >> 3) * panel_rows + r) * 64 + (((c8 & 7) ^ (int)(r & 7)) << 3);
    *reinterpret_cast<uint4 *>(at) = hi;
    *reinterpret_cast<uint4 *>(at + part) = lo;
  }
}

// ---------------------------------------------------------------------------
// narrow sides up to 128: all steps in one launch, a cluster per matrix
// ---------------------------------------------------------------------------

struct Narrow {
  Source src;
  int rows, cols;          // the user's matrix
  int side, length, tall;  // its narrow and long side, and which is which
  int panels, steps;       // 64 along the long side each
  int quintic;
  double scale, eps;
  float inv;               // 2^-e
  float diag1, scale1;     // after X X^T
  float diag2, scale2;     // after Z^2
  void *out;
  int dtype;
  float *weight;
  float decay, step;
};

struct NarrowLayout {
  static constexpr int kMostPanels = 3;                          // of X in one CTA
  static constexpr int kX = kMostPanels * kBM * 128;             // one part
  static constexpr int kZ = 2 * kBM * 128;
  static constexpr int kZAt = 2 * kX, kRAt = kZAt + 2 * kZ;      // Z (then M), and the partial sums
  static constexpr int kBars = kRAt + kBM * kBM * 4;
  static constexpr int kBytes = kBars + 64 + 8 * 8 + 1024;       // + alignment slack
  static_assert(kBytes <= 227 * 1024, "shared memory budget");
};
constexpr int kNarrowThreads = 512;  // a warp takes 32 rows by 32 columns of each result
static_assert(NarrowLayout::kMostPanels * 64 * kBM * 4 <= NarrowLayout::kBars - NarrowLayout::kZAt, "scratch");

// byte of 8-column chunk `chunk` (of the slice) of row `row` in swizzled panels of 128 rows
__device__ __forceinline__ int narrow_at(int row, int chunk) {
  return (chunk >> 3) * (kBM * 128) + row * 128 + (((chunk ^ row) & 7) << 4);
}

// 32 columns of the summed accumulators of a row (TMEM lane) per thread.
// The last one's may reach 16 columns past the accumulators where their width
// is an odd multiple of 16, but not past TMEM's 512: such accumulators fill
// 512 columns only at a width of 16, and at most 12 of those are in use.
__device__ __forceinline__ void read_sum(float (&sum)[32], uint32_t acc, int count, uint32_t stride) {
#pragma unroll
  for (int e = 0; e < 32; ++e) sum[e] = 0.0f;
#pragma unroll 1
  for (int a = 0; a < count; ++a, acc += stride) add_stage<32>(sum, acc);
}

// The last product's 32 rows (of the narrow side) by 32 of the long side, a
// row per lane, to the user's matrix: turned through the warp's patch, so
// that lanes write along the axis that is contiguous there.
__device__ __forceinline__ void narrow_out(const Narrow &q, int64_t base, int r0, int c0, const float (&v)[32],
                                           float *patch) {
  const int lane = threadIdx.x & 31;
  const float inv2 = q.inv * q.inv;
#pragma unroll
  for (int k = 0; k < 8; ++k)
    *reinterpret_cast<float4 *>(patch + patch_at(lane, k)) =
        make_float4(v[4 * k], v[4 * k + 1], v[4 * k + 2], v[4 * k + 3]);
  __syncwarp();
  const int fixed = q.tall ? r0 + lane : c0 + lane;
  const int n = q.tall ? q.length - c0 : q.side - r0;  // of the other axis, one per iteration
  const int64_t stride = q.tall ? q.side : q.length, at = base + (int64_t)(q.tall ? c0 : r0) * stride + fixed;
  if (fixed < (q.tall ? q.side : q.length)) {
#pragma unroll 1
    for (int k = 0; k < 32 && k < n; k += 8) {
      float y[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int row = q.tall ? lane : k + e, col = q.tall ? k + e : lane;
        y[e] = patch[patch_at(row, col >> 2) + (col & 3)] * inv2;
        if (q.weight && k + e < n) y[e] = fmaf(-q.step, y[e], q.decay * q.weight[at + (k + e) * stride]);
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        if (k + e >= n) break;
        if (q.weight)
          q.weight[at + (k + e) * stride] = y[e];
        else if (q.dtype == 0)
          static_cast<float *>(q.out)[at + (k + e) * stride] = y[e];
        else if (q.dtype == 1)
          static_cast<__nv_bfloat16 *>(q.out)[at + (k + e) * stride] = __float2bfloat16_rn(y[e]);
        else
          static_cast<__half *>(q.out)[at + (k + e) * stride] = __float2half_rn(y[e]);
      }
    }
  }
  __syncwarp();
}

// Chunk `id` of a slice: its row (narrow side) and place along the slice.
// Lanes run along the axis that is contiguous in memory.
__device__ __forceinline__ void narrow_chunk(const Narrow &q, int id, int chunks, int &row, int &chunk) {
  if (q.tall) {
    row = id & (kBM - 1);
    chunk = id / kBM;
  } else {
    row = id / chunks;
    chunk = id - row * chunks;
  }
}

// The slice's update (and the momentum it leaves), eight neighbours along
// the long side per chunk, into fp32 scratch; returns the sum of squares.
template <typename T>
__device__ __forceinline__ double narrow_load(const Narrow &q, int64_t base, int col0, int chunks, float *scratch) {
  const T *in = static_cast<const T *>(q.src.in);
  double sum = 0.0;
  const int total = kBM * chunks;
  const int64_t stride = q.tall ? q.side : 1;
#pragma unroll 1
  for (int id0 = threadIdx.x; id0 < total; id0 += 2 * kNarrowThreads) {
    float u[2][8], m[2][8];
    int64_t at[2];
    int left[2];  // elements of the chunk that the matrix has
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int id = id0 + i * kNarrowThreads;
      int row, chunk;
      narrow_chunk(q, id, chunks, row, chunk);
      const int col = col0 + chunk * 8;
      left[i] = id < total && row < q.side ? q.length - col : 0;
      at[i] = base + (q.tall ? (int64_t)col * q.side + row : (int64_t)row * q.length + col);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        u[i][e] = e < left[i] ? to_f(in[at[i] + e * stride]) : 0.0f;
        if (q.src.momentum) m[i][e] = e < left[i] ? q.src.momentum[at[i] + e * stride] : 0.0f;
      }
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int id = id0 + i * kNarrowThreads;
      if (id >= total) break;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        if (q.src.momentum) {
          m[i][e] = fmaf(q.src.beta, m[i][e], q.src.rest * u[i][e]);
          if (e < left[i]) q.src.momentum[at[i] + e * stride] = m[i][e];
          u[i][e] = muon_direction(q.src, u[i][e], m[i][e]);
        }
      }
      sum += sum_of_squares(u[i]);
      float4 *to = reinterpret_cast<float4 *>(scratch + id * 8);
      to[0] = make_float4(u[i][0], u[i][1], u[i][2], u[i][3]);
      to[1] = make_float4(u[i][4], u[i][5], u[i][6], u[i][7]);
    }
  }
  return sum;
}

// 32 columns of row `row` of Z or M, a row per lane: scale v + diag on the
// diagonal, and zeros past the narrow side
__device__ __forceinline__ void narrow_square(uint8_t *z, int part, int row, int col, int side, float scale, float diag,
                                              const float (&v)[32]) {
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    float y[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int at = col + 8 * c + e;
      y[e] = at < side ? v[8 * c + e] * scale + (row == at ? diag : 0.0f) : 0.0f;
    }
    uint4 hi, lo;
    split8(y, hi, lo);
    *reinterpret_cast<uint4 *>(z + narrow_at(row, col / 8 + c)) = hi;
    *reinterpret_cast<uint4 *>(z + part + narrow_at(row, col / 8 + c)) = lo;
  }
}

// A matrix whose narrow side is at most 128 lives in the shared memory of a
// cluster for all its steps: X [side <= 128][length], a slice of whole
// panels per CTA (transposed on the way in and out if it is tall).  A step:
// every CTA's product X X^T over its slice; the partial sums reduced, a
// share of the rows per CTA, and Z = A + shift I handed to all through
// distributed shared memory; M = c Z^2 + d I and X <- M X in every CTA for
// its own slice.  Nothing but the matrix itself crosses global memory, and
// seventeen launches of 7 us become one (162 x 82 49 us, 12 matrices of
// 1152 x 128 82 us, 86 as Muon's step; one launch per product took 94 and 125).
//
// What bounds it is latency: about ten dependent phases a step, each far
// below the tensor cores' or shared memory's rate.
__global__ void __launch_bounds__(kNarrowThreads, 1) ns_narrow_kernel(const __grid_constant__ Narrow q) {
  using L = NarrowLayout;
  extern __shared__ uint8_t smem_raw[];
  uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  uint64_t *done = reinterpret_cast<uint64_t *>(smem + L::kBars);
  uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(done + 1);
  volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_slot + 1);
  double *norms = reinterpret_cast<double *>(smem + L::kBars + 64);  // one per CTA of the cluster
  __shared__ double s_part[kNarrowThreads / 32];
  const auto cluster = cg::this_cluster();
  const int ctas = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
  const int quad = warp & 3;
  const int64_t base = (int64_t)(blockIdx.x / ctas) * q.rows * q.cols;
  const int panel0 = rank * q.panels / ctas, mine = (rank + 1) * q.panels / ctas - panel0;

  if (tid == 0) {
    mbar_init(done, 1);
    *abort_flag = 0;
    fence_barrier_init();
  }
  __syncwarp();
  if (warp == 0) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }

  float *scratch = reinterpret_cast<float *>(smem + L::kZAt);  // 96 KB of what Z and the sums take later
  const int chunks = mine * 8;
  double sum = q.src.dtype == 0   ? narrow_load<float>(q, base, panel0 * 64, chunks, scratch)
               : q.src.dtype == 1 ? narrow_load<__nv_bfloat16>(q, base, panel0 * 64, chunks, scratch)
                                  : narrow_load<__half>(q, base, panel0 * 64, chunks, scratch);
  for (int off = 16; off; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
  if (lane == 0) s_part[warp] = sum;
  __syncthreads();
  cluster.sync();  // the other CTAs run: their shared memory may be written
  if (tid < ctas) {
    double total = 0.0;
    for (int i = 0; i < kNarrowThreads / 32; ++i) total += s_part[i];
    cluster.map_shared_rank(norms, tid)[rank] = total;
  }
  tc_fence_before();
  cluster.sync();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  {
    double total = 0.0;
    for (int i = 0; i < ctas; ++i) total += norms[i];
    const double f64 = q.scale / (sqrt(total) + q.eps);
    const float f = (float)f64;
    auto split = [&](auto scaled) {
#pragma unroll 2
      for (int id = tid; id < kBM * chunks; id += kNarrowThreads) {
        int row, chunk;
        narrow_chunk(q, id, chunks, row, chunk);
        float u[8];
        *reinterpret_cast<float4 *>(u) = *reinterpret_cast<const float4 *>(scratch + id * 8);
        *reinterpret_cast<float4 *>(u + 4) = *reinterpret_cast<const float4 *>(scratch + id * 8 + 4);
#pragma unroll
        for (int e = 0; e < 8; ++e) u[e] = scaled(u[e]);
        uint4 hi, lo;
        split8(u, hi, lo);
        *reinterpret_cast<uint4 *>(smem + narrow_at(row, chunk)) = hi;
        *reinterpret_cast<uint4 *>(smem + L::kX + narrow_at(row, chunk)) = lo;
      }
    };
    if (f64 > 1e-30 && f64 < 1e30)
      split([=](float u) { return u * f; });
    else
      split([=](float u) { return (float)((double)u * f64); });  // a factor beyond is applied in 64 bits
  }

  if (ctas > 1) cluster.sync();  // the scratch is read: partial sums may arrive in its place

  // A warp whose wait ran out takes no further part: it issues and reads no
  // product, tells the cluster, and goes on to the barriers alone.
  bool alive = true;
  uint32_t parity = 0, issued = 0;
  const uint32_t x_at = smem_u32(smem), z_at = smem_u32(smem + L::kZAt);
  // One product: `ksteps` of 16, `sub` of them per accumulator of n columns
  // (of the 512 that there are).  b_mn: B's panels lie along N and K counts
  // their rows.
  auto product = [&](uint32_t a, uint32_t a_part, uint32_t b, uint32_t b_part, int ksteps, int sub, int n,
                     bool b_mn) {
    fence_proxy_async();
    tc_fence_before();
    __syncthreads();
    if (warp == 0 && alive) {
      tc_fence_after();
      if (elect_one()) {
        const uint32_t idesc = idesc_f16(kBM, n, false, b_mn);
        // N along B's panels of 128 rows: the next 64 columns are a panel on
        const uint64_t da = desc_sw128(a, false), db = desc_sw128(b, b_mn, kBM * 128);
        for (int k0 = 0, acc = 0; k0 < ksteps; k0 += sub, acc += n)
          for (int term = 0; term < 3; ++term)
            for (int k = k0; k < k0 + sub && k < ksteps; ++k) {
              const uint32_t along = (uint32_t)(k >> 2) * (kBM * 128) + (uint32_t)(k & 3) * 32;  // K-major
              const uint32_t ao = (term == 1 ? a_part : 0u) + along;
              const uint32_t bo = (term == 0 ? b_part : 0u) + (b_mn ? (uint32_t)k * 2048u : along);
              umma_f16(tmem + (uint32_t)acc, da + (ao >> 4), db + (bo >> 4), idesc, term != 0 || k != k0);
            }
        umma_commit(done);
      }
      issued = parity;
      __syncwarp();
    }
    if (alive && !mbar_wait_warp(done, parity, abort_flag, &g_muon_error)) {
      alive = false;
      if (lane < ctas) *cluster.map_shared_rank(const_cast<int *>(abort_flag), lane) = 1;
    }
    parity ^= 1u;
    __syncwarp();
    tc_fence_after();
  };

  const int mine_steps = ((mine * 64 < q.length - panel0 * 64 ? mine * 64 : q.length - panel0 * 64) + 15) / 16;
  const int side_steps = (q.side + 15) / 16, side_n = side_steps * 16;
  // K steps per accumulator: as few as TMEM's columns allow
  auto sub_of = [](int ksteps, int n) {
    const int accs = 512 / n;
    return (ksteps + accs - 1) / accs;
  };
  const int n_update = mine * 64;
  const int gram_sub = sub_of(mine_steps, side_n), square_sub = sub_of(side_steps, side_n);
  const int update_sub = sub_of(side_steps, n_update);
  const int gram_accs = (mine_steps + gram_sub - 1) / gram_sub, square_accs = (side_steps + square_sub - 1) / square_sub;
  const int update_accs = (side_steps + update_sub - 1) / update_sub;
  const uint32_t lanes = (uint32_t)(quad * 32) << 16;
  const int row = quad * 32 + lane, col = (warp >> 2) * 32;  // of this thread's 32 entries of Z and M
  float v[32];
  for (int step = 0; step < q.steps; ++step) {
    // X X^T over this slice
    product(x_at, L::kX, x_at, L::kX, mine_steps, gram_sub, side_n, false);
    read_sum(v, tmem + lanes + (uint32_t)col, alive && col < side_n ? gram_accs : 0, (uint32_t)side_n);
    if (ctas == 1) {
      narrow_square(smem + L::kZAt, L::kZ, row, col, q.side, q.scale1, q.diag1, v);
    } else {
      // partial sums to the CTA that owns the row, as [source][4 columns]
      // [row], rows permuted so that the columns of a row spread over the
      // banks; its rows of Z to all
      const int own = kBM / ctas;
      float4 *to = cluster.map_shared_rank(reinterpret_cast<float4 *>(smem + L::kRAt), row / own);
      to += (rank * 32 + col / 4) * own;
#pragma unroll
      for (int e = 0; e < 8; ++e)
        to[e * own + ((row % own) ^ ((col / 8 + e / 2) & 7))] =
            make_float4(v[4 * e], v[4 * e + 1], v[4 * e + 2], v[4 * e + 3]);
      cluster.sync();
      const float4 *from = reinterpret_cast<const float4 *>(smem + L::kRAt);
      for (int id = tid; id < own * 16; id += kNarrowThreads) {
        const int r = id >> 4, c8 = id & 15, pos = r ^ (c8 & 7);
        float y[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] = 0.0f;
        for (int c = 0; c < ctas; ++c) {
          const float4 f0 = from[(c * 32 + 2 * c8) * own + pos], f1 = from[(c * 32 + 2 * c8 + 1) * own + pos];
          y[0] += f0.x;
          y[1] += f0.y;
          y[2] += f0.z;
          y[3] += f0.w;
          y[4] += f1.x;
          y[5] += f1.y;
          y[6] += f1.z;
          y[7] += f1.w;
        }
        const int at = rank * own + r;
#pragma unroll
        for (int e = 0; e < 8; ++e)
          y[e] = 8 * c8 + e < q.side ? y[e] * q.scale1 + (at == 8 * c8 + e ? q.diag1 : 0.0f) : 0.0f;
        uint4 hi, lo;
        split8(y, hi, lo);
        for (int c = 0; c < ctas; ++c) {
          uint8_t *z = cluster.map_shared_rank(smem + L::kZAt, c);
          *reinterpret_cast<uint4 *>(z + narrow_at(at, c8)) = hi;
          *reinterpret_cast<uint4 *>(z + L::kZ + narrow_at(at, c8)) = lo;
        }
      }
      cluster.sync();
    }
    if (q.quintic) {
      product(z_at, L::kZ, z_at, L::kZ, side_steps, square_sub, side_n, false);
      read_sum(v, tmem + lanes + (uint32_t)col, alive && col < side_n ? square_accs : 0, (uint32_t)side_n);
      narrow_square(smem + L::kZAt, L::kZ, row, col, q.side, q.scale2, q.diag2, v);
    }
    // X <- M X
    product(z_at, L::kZ, x_at, L::kX, side_steps, update_sub, n_update, true);
    const bool last = step + 1 == q.steps;
    if (last) {
      // a matrix is written whole or, where a wait of any CTA ran out, not at all
      cluster.sync();
      if (*abort_flag) break;
    }
#pragma unroll 1
    for (int c = col; c < n_update; c += 128) {
      read_sum(v, tmem + lanes + (uint32_t)c, alive ? update_accs : 0, (uint32_t)n_update);
      if (!last) {
#pragma unroll
        for (int e = 0; e < 32; ++e) v[e] *= q.inv;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          uint4 hi, lo;
          split8(v + 8 * k, hi, lo);
          *reinterpret_cast<uint4 *>(smem + narrow_at(row, c / 8 + k)) = hi;
          *reinterpret_cast<uint4 *>(smem + L::kX + narrow_at(row, c / 8 + k)) = lo;
        }
      } else {
        narrow_out(q, base, quad * 32, panel0 * 64 + c, v, reinterpret_cast<float *>(smem + L::kRAt) + warp * 1024);
      }
    }
  }
  // (the last access to another CTA's memory lies before the last step's barrier)
  if (warp == 0 && !alive) mbar_drain(done, issued);
  tc_fence_before();
  __syncthreads();
  if (warp == 0) tmem_dealloc(tmem, 512);
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

// [batch][2][panels][panel_rows][64] of fp16, and the map that loads boxes
// of 64 rows of it
struct Stack {
  __half *p;
  int64_t batch;
  int panel_rows, panels;
  CUtensorMap map;

  bool place(uint8_t *at, int64_t matrices, int rows, int cols) {
    p = reinterpret_cast<__half *>(at);
    batch = matrices;
    panel_rows = (rows + 63) / 64 * 64;
    panels = (cols + 63) / 64;
    const auto fn = encode_fn();
    cuuint64_t dims[3] = {64, (cuuint64_t)panel_rows * panels, (cuuint64_t)batch * 2};
    cuuint64_t strides[2] = {128, (cuuint64_t)panel_rows * panels * 128};
    cuuint32_t box[3] = {64, 64, 1};
    cuuint32_t estr[3] = {1, 1, 1};
    return fn && fn(&map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, p, dims, strides, box, estr,
                    CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                    CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
  }
};

// partial sums of squares of a matrix, at most
int64_t norm_blocks(int64_t rows, int64_t cols) {
  const int64_t blocks = (rows * cols + 2047) / 2048;
  return blocks < kNormBlocks ? blocks : kNormBlocks;
}

constexpr int64_t kFlagBytes = 256;  // a call's flag, at the start of its workspace

int64_t norm_bytes(int64_t batch, int64_t rows, int64_t cols) {
  return (batch * norm_blocks(rows, cols) * (int64_t)sizeof(double) + 255) / 256 * 256;
}

int64_t stack_bytes(int64_t batch, int64_t rows, int64_t cols) {
  return batch * 2 * ((rows + 63) / 64 * 64) * ((cols + 63) / 64) * 128;
}

// the device: its SMs, and how many clusters of 2 to 8 CTAs of the tile
// kernel it runs at once
struct Device {
  int sms, clusters[kMaxSplit + 1];
};

constexpr int kMaxDevices = 64;

template <int BN>
cudaError_t set_up_pair() {
  cudaFuncAttributes a;
  const cudaError_t e = cudaFuncGetAttributes(&a, ns_pair_kernel<BN>);
  if (e != cudaSuccess) return e;
  if (a.numRegs < kLaunchRegisters) return cudaErrorInvalidConfiguration;
  return cudaFuncSetAttribute(ns_pair_kernel<BN>, cudaFuncAttributeMaxDynamicSharedMemorySize, PairLayout<BN>::kBytes);
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
  if (cudaFuncSetAttribute(ns_tile_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, TileLayout::kBytes) !=
          cudaSuccess ||
      cudaFuncSetAttribute(ns_narrow_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, NarrowLayout::kBytes) !=
          cudaSuccess ||
      set_up_pair<256>() != cudaSuccess || set_up_pair<128>() != cudaSuccess)
    return nullptr;
  d.clusters[1] = d.sms;
  for (int z = 2; z <= kMaxSplit; ++z) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)z);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = TileLayout::kBytes;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = (unsigned)z;
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    if (cudaOccupancyMaxActiveClusters(&d.clusters[z], ns_tile_kernel, &cfg) != cudaSuccess) return nullptr;
  }
  known[dev] = d;
  ready[dev].store(1, std::memory_order_release);
  return &known[dev];
}

template <int BM, int BN>
int64_t tile_count(const Product &q, int64_t batch) {
  const int tm = (q.rows + BM - 1) / BM, tn = (q.cols + BN - 1) / BN;
  if (!q.sym) return (int64_t)tm * tn * batch;
  int64_t n = 0;
  for (int i = 0; i < tm; ++i) n += row_tiles<BM, BN>(i, tn);
  return n * batch;
}

template <int BN>
cudaError_t run_pair(Product q, const Stack &a, const Stack &b, const Device &d, int64_t tiles, cudaStream_t st) {
  if (tiles > INT32_MAX / 2) return cudaErrorInvalidValue;
  q.tiles_n = (q.cols + BN - 1) / BN;
  q.tiles = (int)tiles;
  q.per_batch = (int)(tiles / a.batch);
  const int pairs = q.tiles < d.sms / 2 ? q.tiles : d.sms / 2;
  return launch(ns_pair_kernel<BN>, dim3((unsigned)(2 * pairs)), kThreads, (size_t)PairLayout<BN>::kBytes, st, true, 1,
                a.map, b.map, q);
}

// The kernel and the CTAs that share a tile's K, by their measured times in
// us beyond what every launch takes: a stage of a 256 x 256 pair tile 0.9 and
// its epilogue, which hides less behind the next tile than a 256 x 128
// one's, 3; a 256 x 128 pair tile 0.53 and 0.5, the last one's 2; a 128 x
// 128 tile, which draws the most operands per product, 0.65 and 1.5 (3.5
// where a symmetric one is written twice), or with its K split 4.2 (two
// cluster barriers and the exchange).  What leaves SMs idle is a tile count
// below a wave, or just above one.
cudaError_t product(Product q, const Stack &a, const Stack &b, const Stack &to, uint32_t *failed, const Device &d,
                    cudaStream_t st) {
  q.failed = failed;
  q.a_rows = a.panel_rows;
  q.b_rows = b.panel_rows;
  q.dst = to.p;
  q.dst_rows = to.panel_rows;
  q.dst_panels = to.panels;
  const int64_t kblocks = (q.k + kBK - 1) / kBK, pairs = d.sms / 2;
  const int64_t p256 = tile_count<256, 256>(q, a.batch), p128 = tile_count<256, 128>(q, a.batch);
  const int64_t t128 = tile_count<128, 128>(q, a.batch);
  const double cost256 = (double)((p256 + pairs - 1) / pairs) * (0.9 * (double)kblocks + 3.0) + 2.2;
  const double cost128 = (double)((p128 + pairs - 1) / pairs) * (0.53 * (double)kblocks + 0.5) + 2.0;
  double best = (double)((t128 + d.sms - 1) / d.sms) * (0.65 * (double)kblocks + (q.sym ? 3.5 : 1.5));
  int split = 1;
  for (int z = 2; z <= kMaxSplit && z <= kblocks; ++z) {
    if (t128 > d.clusters[z]) continue;
    const double cost = 0.65 * (double)((kblocks + z - 1) / z) + 4.2;
    if (cost < best) {
      best = cost;
      split = z;
    }
  }
  if (cost256 < cost128 && cost256 <= best) return run_pair<256>(q, a, b, d, p256, st);
  if (cost128 <= best) return run_pair<128>(q, a, b, d, p128, st);
  if (t128 * kMaxSplit > INT32_MAX) return cudaErrorInvalidValue;
  q.tiles_n = (q.cols + TileLayout::kBN - 1) / TileLayout::kBN;
  q.tiles = (int)t128;
  q.per_batch = (int)(t128 / a.batch);
  return launch(ns_tile_kernel, dim3((unsigned)(q.tiles * split)), kThreads, (size_t)TileLayout::kBytes, st, true,
                split, a.map, b.map, q);
}

// Narrow matrices: the CTAs of a matrix's cluster, 0 where it does not fit.
// A single CTA takes about 30 us, a cluster's exchanges 25 more, and each
// panel of the longest slice 4 (the phases that grow with it), in as many
// waves as the device's clusters of that size make of the stack.
int narrow_ctas(const scacchi_newton_schulz &n, const Device &d) {
  const int side = n.rows < n.cols ? n.rows : n.cols, panels = ((n.rows < n.cols ? n.cols : n.rows) + 63) / 64;
  if (side > kBM) return 0;
  int best = 0;
  int64_t best_cost = 0;
  for (int z = 0; z < 4; ++z) {
    const int ctas = 1 << z, slice = (panels + ctas - 1) / ctas, at_once = d.clusters[ctas];
    if (slice > NarrowLayout::kMostPanels || ctas > panels || at_once < 1) continue;
    const int64_t cost = ((int64_t)n.batch + at_once - 1) / at_once * ((z ? 55 : 30) + 4 * slice);
    if (!best || cost < best_cost) {
      best = ctas;
      best_cost = cost;
    }
  }
  return best;
}

int newton_schulz_narrow(const scacchi_newton_schulz &n, const Source &src, const Product &last, int ctas,
                         cudaStream_t st) {
  Narrow q = {};
  q.src = src;
  q.rows = n.rows;
  q.cols = n.cols;
  q.tall = n.rows > n.cols;
  q.side = q.tall ? n.cols : n.rows;
  q.length = q.tall ? n.rows : n.cols;
  q.panels = (q.length + 63) / 64;
  q.steps = n.steps;
  q.quintic = n.c != 0.0;
  q.scale = ldexp(1.0, n.scale_exponent);
  q.eps = n.eps;
  q.inv = (float)(1.0 / q.scale);
  q.scale1 = (float)((q.quintic ? 1.0 : n.b) / q.scale);
  q.diag1 = (float)((q.quintic ? n.b / (2.0 * n.c) : n.a) * q.scale);
  if (q.quintic) {
    q.scale2 = (float)(n.c / q.scale);
    q.diag2 = (float)((n.a - n.b * n.b / (4.0 * n.c)) * q.scale);
  }
  q.out = last.out;
  q.dtype = last.dtype;
  q.weight = last.weight;
  q.decay = last.decay;
  q.step = last.step;
  return launch(ns_narrow_kernel, dim3((unsigned)(n.batch * ctas)), kNarrowThreads, (size_t)NarrowLayout::kBytes, st,
                false, ctas, q) == cudaSuccess
             ? SCACCHI_OK
             : SCACCHI_ECUDA;
}

int newton_schulz(const scacchi_newton_schulz &n, const Source &src, Product last, void *workspace, cudaStream_t st) {
  const Device *dev = device();
  if (!dev) return SCACCHI_ECUDA;
  if (const int ctas = narrow_ctas(n, *dev)) return newton_schulz_narrow(n, src, last, ctas, st);
  const int sms = dev->sms;
  const int s = n.rows < n.cols ? n.rows : n.cols;
  const bool tall = n.rows > n.cols;
  uint8_t *at = static_cast<uint8_t *>(workspace);
  uint32_t *failed = reinterpret_cast<uint32_t *>(at);
  double *partial = reinterpret_cast<double *>(at + kFlagBytes);
  at += kFlagBytes + norm_bytes(n.batch, n.rows, n.cols);
  Stack x, y, gram, poly;
  const int64_t wide = stack_bytes(n.batch, n.rows, n.cols), narrow = stack_bytes(n.batch, s, s);
  if (!x.place(at, n.batch, n.rows, n.cols) || !y.place(at + wide, n.batch, n.rows, n.cols) ||
      !gram.place(at + 2 * wide, n.batch, s, s) || !poly.place(at + 2 * wide + narrow, n.batch, s, s))
    return SCACCHI_ECUDA;
  const double scale = ldexp(1.0, n.scale_exponent);
  const int64_t elems = (int64_t)n.rows * n.cols;

  // 16-byte vectors where every matrix starts on one
  auto on_16 = [](const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; };
  const int vec = elems % 8 == 0 && on_16(src.in) && (!src.momentum || on_16(src.momentum));
  int64_t blocks = norm_blocks(n.rows, n.cols);
  const int64_t share = (8 * (int64_t)sms + n.batch - 1) / n.batch;
  blocks = blocks < share ? blocks : share;
  if (launch(ns_norm_kernel, dim3((unsigned)blocks, (unsigned)n.batch), 256, 0, st, false, 1, src, elems, vec,
             partial, failed) != cudaSuccess)
    return SCACCHI_ECUDA;
  const int64_t chunks = (int64_t)x.panel_rows * x.panels * 8;
  const int split_vec = vec && n.cols % 8 == 0;  // rows too
  int64_t split_blocks = (chunks + 255) / 256;
  const int64_t split_share = (8 * (int64_t)sms + n.batch - 1) / n.batch;
  split_blocks = split_blocks < split_share ? split_blocks : split_share;
  if (launch(ns_split_kernel, dim3((unsigned)split_blocks, (unsigned)n.batch), 256, 0, st, true, 1, src,
             (const double *)partial, (int)blocks, n.rows, n.cols, x.panel_rows, x.panels, split_vec, scale, n.eps,
             x.p) != cudaSuccess)
    return SCACCHI_ECUDA;

  // M = c Z^2 + (a - b^2 / 4c) I with Z = A + (b / 2c) I: the square alone,
  // with shifted diagonals; without c, M = b A + a I takes no product
  const bool quintic = n.c != 0.0;
  Stack *now = &x, *next = &y;
  for (int k = 0; k < n.steps; ++k) {
    Product q = {};
    q.sym = 1;
    q.rows = q.cols = s;
    q.a_major = q.b_major = tall ? kAlongMN : kAlongK;
    q.k = tall ? n.rows : n.cols;
    q.scale = (float)((quintic ? 1.0 : n.b) / scale);
    q.diag = (float)((quintic ? n.b / (2.0 * n.c) : n.a) * scale);
    if (product(q, *now, *now, quintic ? gram : poly, failed, *dev, st) != cudaSuccess) return SCACCHI_ECUDA;
    if (quintic) {
      q.a_major = q.b_major = kSymmetric;
      q.k = s;
      q.scale = (float)(n.c / scale);
      q.diag = (float)((n.a - n.b * n.b / (4.0 * n.c)) * scale);
      if (product(q, gram, gram, poly, failed, *dev, st) != cudaSuccess) return SCACCHI_ECUDA;
    }
    const bool final = k + 1 == n.steps;
    Product u = final ? last : Product{};
    u.last = final;
    u.scale = (float)(final ? 1.0 / (scale * scale) : 1.0 / scale);
    u.rows = n.rows;
    u.cols = n.cols;
    u.k = s;
    u.a_major = tall ? kAlongK : kSymmetric;
    u.b_major = tall ? kSymmetric : kAlongMN;
    if (product(u, tall ? *now : poly, tall ? poly : *now, *next, failed, *dev, st) != cudaSuccess)
      return SCACCHI_ECUDA;
    Stack *t = now;
    now = next;
    next = t;
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
  return (size_t)(kFlagBytes + norm_bytes(batch, rows, cols) + 2 * stack_bytes(batch, rows, cols) +
                  2 * stack_bytes(batch, s, s));
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
