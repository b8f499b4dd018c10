// Orthogonalised updates by Newton-Schulz products, and Muon's step.
//
// X = U / (|U|_F + eps); then `steps` times, on the narrow side s x s,
//   A = X X^T (or X^T X),  M = a I + b A + c A^2,  X <- M X (or X M).
// Each is a GEMM on the tensor cores (csrc/tc05.cuh): a tcgen05 kernel with
// TMA-fed operands and the polynomial in its epilogue.
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

constexpr int kBM = 128;           // rows of an output tile
constexpr int kBK = 64;            // K of a stage: 128 bytes of fp16
constexpr int kThreads = 192;      // producer, MMA issuer, four epilogue warps
constexpr int kEpiThreads = 128;
constexpr int kNormBlocks = 128;   // most partial sums of squares per matrix

__device__ uint32_t g_muon_error;
std::atomic<uint64_t> g_muon_launches{0};

enum Mode : int { kGram = 0, kSquare = 1, kUpdate = 2, kLast = 3 };

struct Product {
  int mode, sym;
  int rows, cols, k;            // of the output, and the summed length
  int tiles_n, per_batch, tiles;
  float inv;                    // 2^-e: an accumulator of S^2 v becomes S v
  float a, b, c;                // square: a S, b, c
  __half *dst;                  // [batch][2][rows][pitch]
  const __half *gram;           // square: A, like dst
  int64_t part, pitch;          // elements between hi and lo, and between rows
  // last: the result, or the weight's step w <- decay w - step x
  void *out;
  int dtype;                    // 0 float32, 1 bfloat16, 2 float16
  float *weight;
  float decay, step;
};

template <int BN>
struct Layout {
  static constexpr int kA = kBM * kBK * 2, kB = BN * kBK * 2;   // one part of a stage's operands
  static constexpr int kStage = 2 * (kA + kB);
  static constexpr int kStages = BN == 256 ? 2 : 3;
  static constexpr int kBars = kStages * kStage;
  static constexpr int kBytes = kBars + 8 * (2 * kStages + 4) + 16 + 1024;  // + alignment slack
  static_assert(kBytes <= 227 * 1024, "shared memory budget");
};

// A tile's place: matrix, tile row, tile column.  Symmetric outputs list,
// row by row, the tiles that touch the lower triangle.
template <int BN>
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
    int n = (i * kBM + kBM - 1) / BN + 1;
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

// D[i, j] += A[i, k] B[j, k]; A and B are K-major (their rows run along k)
// or MN-major (k counts rows).  Three MMAs per K step (see above).
template <int BN, bool kAMn, bool kBMn>
__global__ void __launch_bounds__(kThreads, 1) ns_product_kernel(const __grid_constant__ CUtensorMap map_a,
                                                                 const __grid_constant__ CUtensorMap map_b,
                                                                 const __grid_constant__ Product q) {
  using L = Layout<BN>;
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

  if (threadIdx.x == 0) {
    prefetch_map(&map_a);
    prefetch_map(&map_b);
    for (int s = 0; s < L::kStages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(&acc_full[s], 1);
      mbar_init(&acc_empty[s], kEpiThreads);
    }
    *abort_flag = 0;
    fence_barrier_init();
  }
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
      bool stop = false;
      for (int t = blockIdx.x; t < q.tiles && !stop; t += gridDim.x) {
        int batch, i, j;
        locate<BN>(q, t, batch, i, j);
        for (int kb = 0; kb < kblocks; ++kb) {
          if (*abort_flag || !mbar_wait(&empty[stage], phase ^ 1u, abort_flag, &g_muon_error)) {
            stop = true;
            break;
          }
          uint8_t *at = smem + stage * L::kStage;
          mbar_expect_tx(&full[stage], L::kStage);
#pragma unroll
          for (int part = 0; part < 2; ++part) {
            uint8_t *pa = at + part * L::kA, *pb = at + 2 * L::kA + part * L::kB;
            if (kAMn) {
              for (int m = 0; m < kBM / 64; ++m)
                tma_load_3d(pa + m * 64 * kBK * 2, &map_a, &full[stage], i * kBM + m * 64, kb * kBK, 2 * batch + part);
            } else {
              tma_load_3d(pa, &map_a, &full[stage], kb * kBK, i * kBM, 2 * batch + part);
            }
            if (kBMn) {
              for (int n = 0; n < BN / 64; ++n)
                tma_load_3d(pb + n * 64 * kBK * 2, &map_b, &full[stage], j * BN + n * 64, kb * kBK, 2 * batch + part);
            } else {
              tma_load_3d(pb, &map_b, &full[stage], kb * kBK, j * BN, 2 * batch + part);
            }
          }
          issued |= 1u << stage;
          parity = (parity & ~(1u << stage)) | (phase << stage);
          if (++stage == L::kStages) {
            stage = 0;
            phase ^= 1u;
          }
        }
      }
      // every load into shared memory lands before the CTA may exit
      for (int s = 0; s < L::kStages; ++s)
        if (issued >> s & 1u) mbar_drain(&full[s], parity >> s & 1u);
    }
  } else if (warp == 1) {
    if (lane == 0) {
      constexpr uint32_t idesc = idesc_f16(kBM, BN, kAMn, kBMn);
      constexpr uint32_t a_step = kAMn ? 2048 : 32, b_step = kBMn ? 2048 : 32;
      constexpr uint32_t a_lead = kAMn ? 64 * kBK * 2 : 16, b_lead = kBMn ? 64 * kBK * 2 : 16;
      int stage = 0, slot = 0;
      uint32_t phase = 0, acc_phase = 0;
      bool ok = true;
      for (int t = blockIdx.x; t < q.tiles && ok; t += gridDim.x) {
        if (*abort_flag || !mbar_wait(&acc_empty[slot], acc_phase ^ 1u, abort_flag, &g_muon_error)) break;
        tc_fence_after();
        const uint32_t d = tmem + (uint32_t)(slot * BN);
        for (int kb = 0; kb < kblocks; ++kb) {
          if (!mbar_wait(&full[stage], phase, abort_flag, &g_muon_error)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t ah = smem_u32(smem + stage * L::kStage), al = ah + L::kA;
          const uint32_t bh = ah + 2 * L::kA, bl = bh + L::kB;
#pragma unroll
          for (int k = 0; k < kBK / 16; ++k) {
            const uint64_t dah = desc_sw128(ah + k * a_step, a_lead), dal = desc_sw128(al + k * a_step, a_lead);
            const uint64_t dbh = desc_sw128(bh + k * b_step, b_lead), dbl = desc_sw128(bl + k * b_step, b_lead);
            umma_f16(d, dah, dbh, idesc, (kb | k) != 0);
            umma_f16(d, dah, dbl, idesc, 1u);
            umma_f16(d, dal, dbh, idesc, 1u);
          }
          umma_commit(&empty[stage]);
          if (++stage == L::kStages) {
            stage = 0;
            phase ^= 1u;
          }
        }
        if (!ok) break;
        umma_commit(&acc_full[slot]);
        if (++slot == 2) {
          slot = 0;
          acc_phase ^= 1u;
        }
      }
    }
  } else {
    const int quad = warp & 3;  // the TMEM lanes this warp may read
    int slot = 0;
    uint32_t acc_phase = 0;
    for (int t = blockIdx.x; t < q.tiles; t += gridDim.x) {
      int batch, i, j;
      locate<BN>(q, t, batch, i, j);
      bool ok = false;
      if (lane == 0) ok = !*abort_flag && mbar_wait(&acc_full[slot], acc_phase, abort_flag, &g_muon_error);
      if (!__shfl_sync(0xffffffffu, (int)ok, 0)) break;
      tc_fence_after();
      const int r = i * kBM + quad * 32 + lane;
      const bool in_row = r < q.rows;
      const uint32_t acc = tmem + (uint32_t)(slot * BN) + ((uint32_t)(quad * 32) << 16);
      for (int cc = 0; cc < BN / 32; ++cc) {
        const int c0 = j * BN + cc * 32;
        if (c0 >= q.cols) break;
        uint32_t v[32];
        tmem_ld32(acc + cc * 32, v);
        tmem_wait_ld();
        if (q.mode == kLast) {
          if (!in_row) continue;
          const int64_t at = ((int64_t)batch * q.rows + r) * q.cols + c0;
          const int n = q.cols - c0 < 32 ? q.cols - c0 : 32;
          const float inv2 = q.inv * q.inv;
          if (q.weight) {
            float *w = q.weight + at;
#pragma unroll
            for (int e = 0; e < 32; ++e)
              if (e < n) w[e] = fmaf(-q.step, __uint_as_float(v[e]) * inv2, q.decay * w[e]);
          } else if (q.dtype == 0) {
#pragma unroll
            for (int e = 0; e < 32; ++e)
              if (e < n) static_cast<float *>(q.out)[at + e] = __uint_as_float(v[e]) * inv2;
          } else if (q.dtype == 1) {
#pragma unroll
            for (int e = 0; e < 32; ++e)
              if (e < n) static_cast<__nv_bfloat16 *>(q.out)[at + e] = __float2bfloat16_rn(__uint_as_float(v[e]) * inv2);
          } else {
#pragma unroll
            for (int e = 0; e < 32; ++e)
              if (e < n) static_cast<__half *>(q.out)[at + e] = __float2half_rn(__uint_as_float(v[e]) * inv2);
          }
          continue;
        }
        const int64_t base = (int64_t)batch * 2 * q.part;
        // the tile that holds this block's mirror image is not computed:
        // write it from here
        const bool mirror = q.sym && (i * kBM) / BN > (c0 / kBM * kBM + kBM - 1) / BN;
#pragma unroll
        for (int e8 = 0; e8 < 4; ++e8) {
          const int c = c0 + e8 * 8;
          __half hi[8], lo[8];
          float add[8];
          const int64_t at = base + (int64_t)r * q.pitch + c;
#pragma unroll
          for (int e = 0; e < 8; ++e) add[e] = 0.0f;
          if (q.mode == kSquare && in_row && c < q.pitch) {
            const uint4 gh = *reinterpret_cast<const uint4 *>(q.gram + at);
            const uint4 gl = *reinterpret_cast<const uint4 *>(q.gram + at + q.part);
            const __half *h = reinterpret_cast<const __half *>(&gh), *l = reinterpret_cast<const __half *>(&gl);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              add[e] = q.b * (__half2float(h[e]) + __half2float(l[e]));
              if (r == c + e) add[e] += q.a;
            }
          }
          const float scale = q.mode == kSquare ? q.c * q.inv : q.inv;
#pragma unroll
          for (int e = 0; e < 8; ++e) split_half(fmaf(scale, __uint_as_float(v[e8 * 8 + e]), add[e]), hi[e], lo[e]);
          if (in_row && c < q.pitch) {  // the pitch is a multiple of 8: whole vectors
            *reinterpret_cast<uint4 *>(q.dst + at) = *reinterpret_cast<const uint4 *>(hi);
            *reinterpret_cast<uint4 *>(q.dst + at + q.part) = *reinterpret_cast<const uint4 *>(lo);
          }
          if (mirror && in_row) {
#pragma unroll
            for (int e = 0; e < 8; ++e)
              if (c + e < q.cols) {
                const int64_t back = base + (int64_t)(c + e) * q.pitch + r;
                q.dst[back] = hi[e];
                q.dst[back + q.part] = lo[e];
              }
          }
        }
      }
      tc_fence_before();
      mbar_arrive(&acc_empty[slot]);
      if (++slot == 2) {
        slot = 0;
        acc_phase ^= 1u;
      }
    }
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

// [parts][rows][cols] of fp16, boxes of 64 columns x box_rows rows
bool make_map(CUtensorMap *map, const __half *base, int64_t parts, int rows, int cols, int64_t pitch, int64_t part,
              int box_rows) {
  auto fn = encode_fn();
  if (!fn) return false;
  cuuint64_t dims[3] = {(cuuint64_t)cols, (cuuint64_t)rows, (cuuint64_t)parts};
  cuuint64_t strides[2] = {(cuuint64_t)pitch * 2, (cuuint64_t)part * 2};
  cuuint32_t box[3] = {64, (cuuint32_t)box_rows, 1};
  cuuint32_t estr[3] = {1, 1, 1};
  return fn(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, const_cast<__half *>(base), dims, strides, box, estr,
            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

int sm_count() {
  int dev = 0, n = 0;
  if (cudaGetDevice(&dev) != cudaSuccess ||
      cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n <= 0)
    return 148;
  return n;
}

template <typename... P, typename... A>
cudaError_t launch(void (*kernel)(P...), dim3 grid, int threads, size_t smem, cudaStream_t st, bool dependent,
                   A... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3((unsigned)threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = dependent ? 1 : 0;
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

template <int BN, bool kAMn, bool kBMn>
cudaError_t run_product(Product q, const Stack &a, const Stack &b, int sms, cudaStream_t st) {
  CUtensorMap ma, mb;
  if (!make_map(&ma, a.p, a.batch * 2, a.rows, a.cols, a.pitch, a.part, kAMn ? kBK : kBM) ||
      !make_map(&mb, b.p, b.batch * 2, b.rows, b.cols, b.pitch, b.part, kBMn ? kBK : BN))
    return cudaErrorInvalidValue;
  const int tiles_m = (q.rows + kBM - 1) / kBM;
  q.tiles_n = (q.cols + BN - 1) / BN;
  q.per_batch = 0;
  for (int i = 0; i < tiles_m; ++i) {
    const int n = (i * kBM + kBM - 1) / BN + 1;
    q.per_batch += q.sym && n < q.tiles_n ? n : q.tiles_n;
  }
  if ((int64_t)q.per_batch * a.batch > INT32_MAX) return cudaErrorInvalidValue;
  q.tiles = (int)(q.per_batch * a.batch);
  cudaError_t e = cudaFuncSetAttribute(ns_product_kernel<BN, kAMn, kBMn>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                       Layout<BN>::kBytes);
  if (e != cudaSuccess) return e;
  return launch(ns_product_kernel<BN, kAMn, kBMn>, dim3((unsigned)(q.tiles < sms ? q.tiles : sms)), kThreads,
                (size_t)Layout<BN>::kBytes, st, true, ma, mb, q);
}

// The tile's width: 256 columns feed the tensor cores best, 128 spread a
// small output over more SMs.  A 128-wide tile takes about 0.6 of a 256-wide
// one's time, so the narrower is taken where it saves more waves than that.
int64_t tile_count(const Product &q, int64_t batch, int bn) {
  const int64_t tm = (q.rows + kBM - 1) / kBM, tn = (q.cols + bn - 1) / bn;
  int64_t n = 0;
  for (int64_t i = 0; i < tm; ++i) {
    const int64_t w = (i * kBM + kBM - 1) / bn + 1;
    n += q.sym && w < tn ? w : tn;
  }
  return n * batch;
}

template <bool kAMn, bool kBMn>
cudaError_t product(const Product &q, const Stack &a, const Stack &b, int sms, cudaStream_t st) {
  const int64_t wide = (tile_count(q, a.batch, 256) + sms - 1) / sms;
  const int64_t narrow = (tile_count(q, a.batch, 128) + sms - 1) / sms;
  return 0.6 * (double)narrow < (double)wide ? run_product<128, kAMn, kBMn>(q, a, b, sms, st)
                                             : run_product<256, kAMn, kBMn>(q, a, b, sms, st);
}

int newton_schulz(const scacchi_newton_schulz &n, const Source &src, Product last, void *workspace, cudaStream_t st) {
  const int sms = sm_count();
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
  if (launch(ns_norm_kernel, dim3((unsigned)blocks, (unsigned)n.batch), 256, 0, st, false, src, elems, partial) !=
      cudaSuccess)
    return SCACCHI_ECUDA;
  const int64_t chunks = (int64_t)n.rows * (x.pitch / 8);
  int64_t split_blocks = (chunks + 255) / 256;
  const int64_t split_share = (8 * (int64_t)sms + n.batch - 1) / n.batch;
  split_blocks = split_blocks < split_share ? split_blocks : split_share;
  if (launch(ns_split_kernel, dim3((unsigned)split_blocks, (unsigned)n.batch), 256, 0, st, true, src,
             (const double *)partial, (int)blocks, n.rows, n.cols, x.pitch, x.part, scale, n.eps, x.p) != cudaSuccess)
    return SCACCHI_ECUDA;

  for (int k = 0; k < n.steps; ++k) {
    Product q = {};
    q.inv = (float)(1.0 / scale);
    q.sym = 1;
    q.rows = q.cols = s;
    q.dst = gram.p;
    q.part = gram.part;
    q.pitch = gram.pitch;
    q.mode = kGram;
    q.k = tall ? n.rows : n.cols;
    cudaError_t e = tall ? product<true, true>(q, x, x, sms, st) : product<false, false>(q, x, x, sms, st);
    if (e != cudaSuccess) return SCACCHI_ECUDA;
    q.mode = kSquare;
    q.k = s;
    q.dst = poly.p;
    q.gram = gram.p;
    q.a = (float)(n.a * scale);
    q.b = (float)n.b;
    q.c = (float)n.c;
    if (product<false, false>(q, gram, gram, sms, st) != cudaSuccess) return SCACCHI_ECUDA;
    const bool final = k + 1 == n.steps;
    Product u = final ? last : Product{};
    u.inv = q.inv;
    u.mode = final ? kLast : kUpdate;
    u.rows = n.rows;
    u.cols = n.cols;
    u.k = s;
    u.dst = y.p;
    u.part = y.part;
    u.pitch = y.pitch;
    e = tall ? product<false, false>(u, x, poly, sms, st) : product<false, true>(u, poly, x, sms, st);
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
  // the singular values start in [0, 1]: follow a grid of them through the
  // steps; the operands' entries are at most the largest of sigma, sigma^2
  // and |a + b sigma^2 + c sigma^4|
  double most = 1.0;
  for (int i = 0; i <= 4096; ++i) {
    double v = i / 4096.0;
    for (int k = 0; k < steps; ++k) {
      const double v2 = v * v, p = a + v2 * (b + c * v2);
      most = fmax(most, fmax(fabs(p), fmax(fabs(v), v2)));
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
