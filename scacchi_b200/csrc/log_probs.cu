// Log-probabilities of one action per row of logits, with the row's entropy
// and its best actions, and the gradient of both in the logits.
//
// Over the kept actions (legal, logit above -inf), with M = max x,
// u = (x - M) / T, s = sum e^u and t = sum u e^u:
//
//   log_sum  = log s            log_prob = u_a - log s
//   entropy  = log s - t / s    top k by x, the lower index first among equals
//   dx_i     = (g ([i = a] - p_i) - h p_i (log p_i + entropy)) / T,
//              p_i = e^(u_i - log s), for gradients g of log_prob, h of entropy
//
// Logits are read once.  Warps stage batches of short rows in shared memory
// and give each row some lanes, one where 32 rows fit.  Longer rows go through
// a CTA, or a cluster of them where rows are few: every thread keeps the
// maximum of what it has seen and s and t relative to it, and they are joined
// at the row's end.
//
// The best k of a long row come from the same maxima.  Split its threads into
// at least 64 groups: of the groups' maxima the k-th largest, L, has k elements
// at or above it, so the best k are among the elements >= L, and only the parts
// of threads whose maximum reaches L are looked at again: for 64 groups of
// independent logits 64 ln(64 / (64 - k)) elements, 24 for k = 20.  They are
// ranked by counting.  Where more than kCandidates elements reach L (many equal
// ones) the CTA takes the maximum below the last one k times.
//
// Device times, by graph replays: 4096 rows of 32000 bf16 59 us (4.5 TB/s), with
// the 20 best 70, with a mask 96 and 112; of fp16 64 and 73; of fp32 86 us (6.1
// TB/s) and 101.  262144 rows of 82 fp32 20 us (4.3 TB/s), with the 4 best 34, with
// a mask 29 and 47.  8 rows of 131071 fp32 with the 20 best 8 us.  Gradients: 4096 x
// 32000 bf16 79 us (6.6 TB/s), with a mask 95; 262144 x 82 fp32 with a mask 46 us
// (4.3 TB/s).
//
// Long rows of fp32 and long gradients are bound by memory.  Long bf16 rows
// issue 9 instructions an element on 68 % of the cycles (the exponentials alone
// are not the bound: without them 56 us for 61), their ends 1700 a row.  Short
// rows issue 15 to 50 instructions for 32 elements (masks and best actions) on
// 54 to 71 % of the cycles: shared memory leaves 14 to 23 warps an SM.

#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include <algorithm>
#include <atomic>
#include <type_traits>

#include "../../include/scacchi_b200.h"
#include "row_log.cuh"

namespace cg = cooperative_groups;

namespace {

std::atomic<uint64_t> g_log_probs_launches{0};

constexpr unsigned kFull = 0xffffffffu;
constexpr int kThreads = 256;
// Threads of a long row's CTA: 4096 x 32000 bf16 58 us with 128, 67 with 256,
// whose row ends hold up more warps, and 65 with 64.
constexpr int kLong = 128;
constexpr int kWarps = kLong / 32;
constexpr int kMaxShort = 512;      // actions of a short row
// and, where there are eight rows an SM at least, of a row that still goes that way.  bf16 this way, and as
// long rows, without best actions, with 4 and with 20: 20000 x 1000 17, 27 and 57 us (80, 124 and 135), x 2048
// 32, 46 and 98 (80, 124 and 134), x 2500 37, 57 and 122 (81, 126 and 136), x 4000 63, 98 and 214 (82, 127 and
// 136); 1184 x 1000 4, 7 and 16 (8, 11 and 12), x 2048 5, 8 and 17 (8, 11 and 12).  fp32 20000 x 2048 39, 66 and
// 158 (69, 114 and 122).  Gradients: 20000 x 1000 bf16 24 (41), fp32 33 (41), 1184 x 1000 bf16 4.2 (3.8).
constexpr int kMaxMany = 2048, kMaxManyGradient = 1024;
constexpr int kMaxActions = SCACCHI_MAX_ACTIONS;
constexpr int kMaxTop = SCACCHI_MAX_TOP;
constexpr int kMaxCluster = 16;
constexpr int kMaxGroups = 64;  // of a row's threads: four warps of sixteen CTAs, or 64 of fewer
constexpr int kCandidates = 512;
constexpr int kParts = 8;           // of a thread's chunks, each with its maximum
constexpr float kLog2E = 1.44269504088896341f;
constexpr float kLn2 = 0.693147180559945309f;
constexpr float kNothing = -1.0e4f;  // 2^kNothing is 0, and 0 times it is 0

struct Params {
  const void *logits;
  const uint8_t *legal;
  const int32_t *action;
  float *log_prob, *entropy, *max_logit, *log_sum, *top_log_prob;
  int32_t *top_action;
  // of the gradient: max_logit, log_sum and entropy are inputs
  const float *grad_log_prob, *grad_entropy;
  void *grad;
  int64_t rows, stride;
  int actions, top;
  int group;     // lanes of a short row
  float scale;   // log2(e) / T
  float inverse; // 1 / T
  double inverse64;
};

template <typename T>
__device__ __forceinline__ float to_f(T v) {
  if constexpr (std::is_same_v<T, float>) return v;
  if constexpr (std::is_same_v<T, __nv_bfloat16>) return __bfloat162float(v);
  if constexpr (std::is_same_v<T, __half>) return __half2float(v);
}
template <typename T>
__device__ __forceinline__ T from_f(float v) {
  if constexpr (std::is_same_v<T, float>) return v;
  if constexpr (std::is_same_v<T, __nv_bfloat16>) return __float2bfloat16_rn(v);
  if constexpr (std::is_same_v<T, __half>) return __float2half_rn(v);
}

// a pair of bfloat16 or float16 as floats
template <typename T>
__device__ __forceinline__ float2 floats(uint32_t u) {
  if constexpr (std::is_same_v<T, __nv_bfloat16>)
    return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u));
  return __half22float2(*reinterpret_cast<const __half2 *>(&u));
}

template <typename T, int W>
struct alignas(sizeof(T) * W) Vec {
  T v[W];
};

__device__ __forceinline__ float exp2_fast(float t) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(t));
  return y;
}
// the larger one, NaN where either is
__device__ __forceinline__ float max_nan(float a, float b) {
  float y;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}

// u log2 e of a logit relative to the row's maximum (0 where the row has
// none): the difference first, so that a row's offset costs no digits
__device__ __forceinline__ float exponent_of(float x, float top, float scale) {
  return max_nan((x - top) * scale, kNothing);
}

// Logits in their order, as whole numbers: -0 and 0 are equal
__device__ __forceinline__ uint32_t order_of(float x) {
  const uint32_t b = __float_as_uint(x + 0.0f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float logit_of(uint32_t order) {
  return __uint_as_float(order & 0x80000000u ? order & 0x7fffffffu : ~order);
}
// by value, then by the lower index; 0 is below every element
__device__ __forceinline__ uint64_t key_of(float x, int a) {
  return (uint64_t)order_of(x) << 32 | (uint32_t)~a;
}

// The logarithm and what it is subtracted from are held in 64 bits, and each
// result is rounded once: the action's log-probability is the policy loss's
// old_log_prob, whose ratio takes its own from 64 bits too.
struct Row {
  float top, entropy;
  double log_sum;
};

__device__ __forceinline__ Row finish_row(float top, float s, float t) {
  Row r;
  r.top = s != s ? s : top;  // (maxima pass over what is no number, and +inf leaves a sum that is none)
  r.log_sum = log_row_sum(s);
  r.entropy = s == 0.0f ? 0.0f : (float)(r.log_sum - (double)(kLn2 * t / s));
  return r;
}
__device__ __forceinline__ float log_prob_of(const Params &p, float x, float top, double log_sum) {
  return (float)(((double)x - (double)top) * p.inverse64 - log_sum);
}

// A row's action, where it has one, and its logit, -inf where it is not kept
struct Played {
  bool inside;
  float x;
};
template <typename T>
__device__ __forceinline__ Played played(const Params &p, int64_t row) {
  const int a = p.action[row];
  Played q = {a >= 0 && a < p.actions, -INFINITY};
  if (q.inside && (!p.legal || p.legal[row * p.actions + a]))
    q.x = to_f(static_cast<const T *>(p.logits)[row * p.stride + a]);
  return q;
}

__device__ __forceinline__ void write_row(const Params &p, int64_t row, const Row &r, const Played &q) {
  p.log_prob[row] = !q.inside ? 0.0f : q.x == -INFINITY ? -INFINITY : log_prob_of(p, q.x, r.top, r.log_sum);
  p.entropy[row] = r.entropy;
  p.max_logit[row] = r.top;
  p.log_sum[row] = (float)r.log_sum;
}

__device__ __forceinline__ void write_top(const Params &p, int64_t row, const Row &r, int rank, float x, int a) {
  p.top_action[row * p.top + rank] = a;
  p.top_log_prob[row * p.top + rank] = a < 0 ? -INFINITY : log_prob_of(p, x, r.top, r.log_sum);
}

template <int Bytes>
__device__ __forceinline__ void copy_async(void *to, const void *from) {
  const uint32_t at = (uint32_t)__cvta_generic_to_shared(to);
  if constexpr (Bytes == 16)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(at), "l"(from) : "memory");
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(at), "l"(from) : "memory");
}

// ---------------------------------------------------------------------------
// short rows: p.group lanes each
// ---------------------------------------------------------------------------

// A warp takes a batch of rows, 32 / group of them, into shared memory and each
// row's lanes read vectors of W elements of it: 82 actions have a lane to
// themselves, so the row's ends (logarithms, divisions, results) cost a warp
// once in 32 rows.  Neighbouring rows lie A elements apart; W is chosen with
// A / W odd where A allows it, and reads meet no bank twice.
//
// A lane's elements form parts of about eight, whose maxima lie beside them:
// the best k take k rounds over the parts and one part's elements.
constexpr int kShortThreads = 128;
constexpr int kShortWarps = kShortThreads / 32;
constexpr int kPartElements = 8;

struct Batch {  // of a warp, in bytes from its own shared memory's begin
  int pitch, legal_pitch;  // of a row and of its mask
  int legal, maxima, results, bytes;
  int vectors, parts;  // of a lane
};

// Rows of `row` bytes, `pitch` apart in shared memory; they are one piece
// there unless both are multiples of 16 bytes, and so is `from`
template <int Size>
__device__ __forceinline__ void stage(uint8_t *to, const uint8_t *from, int rows, int row, int pitch) {
  const int lane = threadIdx.x & 31, bytes = rows * row;
  if (pitch != row) {
    const int each = row / 16;
    for (int i = lane; i < rows * each; i += 32) copy_async<16>(to + 16 * i + i / each * (pitch - row), from + 16 * i);
    return;
  }
  const int phase = (int)(reinterpret_cast<uintptr_t>(from) & 15);
  to += phase;
  const int head = min(bytes, (16 - phase) & 15), body = (bytes - head) / 16, tail = head + 16 * body;
  for (int i = lane; i < body; i += 32) copy_async<16>(to + head + 16 * i, from + head + 16 * i);
  using Word = std::conditional_t<Size == 4, uint32_t, std::conditional_t<Size == 2, uint16_t, uint8_t>>;
  if (lane * Size < head) *reinterpret_cast<Word *>(to + lane * Size) = *reinterpret_cast<const Word *>(from + lane * Size);
  if (tail + lane * Size < bytes)
    *reinterpret_cast<Word *>(to + tail + lane * Size) = *reinterpret_cast<const Word *>(from + tail + lane * Size);
}

template <typename T, int W>
__global__ void __launch_bounds__(kShortThreads) short_kernel(const __grid_constant__ Params p,
                                                              const __grid_constant__ Batch b) {
  extern __shared__ __align__(16) uint8_t shared_bytes[];
  const int lane = threadIdx.x & 31, group = p.group, sub = lane & (group - 1), mine = lane / group;
  uint8_t *own = shared_bytes + (threadIdx.x / 32) * b.bytes;
  float *maxima = reinterpret_cast<float *>(own + b.maxima) + lane;  // of the lane's parts, 32 apart
  const int rows = 32 / group, all = p.actions / W;                  // vectors of a row
  const int64_t batches = (p.rows + rows - 1) / rows;
  for (int64_t batch = (int64_t)blockIdx.x * kShortWarps + threadIdx.x / 32; batch < batches;
       batch += (int64_t)gridDim.x * kShortWarps) {
    const int64_t first = batch * rows;
    const int count = (int)min((int64_t)rows, p.rows - first);
    const T *from = static_cast<const T *>(p.logits) + first * p.stride;
    const uint8_t *mask = p.legal ? p.legal + first * p.actions : nullptr;
    int phase = 0;
    // (a single row of others may begin anywhere, but pieces of 16 bytes may not)
    if (p.stride == p.actions || (count == 1 && b.pitch == p.actions * (int)sizeof(T))) {
      phase = (int)(reinterpret_cast<uintptr_t>(from) & 15);
      stage<sizeof(T)>(own, reinterpret_cast<const uint8_t *>(from), count, p.actions * (int)sizeof(T), b.pitch);
    } else {
      for (int r = 0; r < count; ++r)
        for (int i = lane; i < p.actions; i += 32) reinterpret_cast<T *>(own + r * b.pitch)[i] = from[r * p.stride + i];
    }
    if (mask) stage<1>(own + b.legal, mask, count, p.actions, b.legal_pitch);
    asm volatile("cp.async.wait_all;" ::: "memory");
    const bool live = mine < count;
    const int64_t row = first + mine;
    const int action = live ? p.action[row] : -1;
    __syncwarp();

    Vec<T, W> *x = reinterpret_cast<Vec<T, W> *>(own + phase + mine * b.pitch);
    const Vec<uint8_t, W> *legal = reinterpret_cast<const Vec<uint8_t, W> *>(
        own + b.legal + (reinterpret_cast<uintptr_t>(mask) & 15) + mine * b.legal_pitch);
    constexpr int kEach = kPartElements / W;  // vectors of a part
    float top = -INFINITY;
    if (live) {
      for (int part = 0, v = sub; part < b.parts; ++part) {
        float most = -INFINITY;
#pragma unroll
        for (int k = 0; k < kEach; ++k, v += group) {
          if (v >= all) break;
          Vec<T, W> q = x[v];
          if (mask) {
            const Vec<uint8_t, W> keep = legal[v];
#pragma unroll
            for (int w = 0; w < W; ++w)
              if (!keep.v[w]) q.v[w] = from_f<T>(-INFINITY);
            x[v] = q;
          }
#pragma unroll
          for (int w = 0; w < W; ++w) most = fmaxf(most, to_f(q.v[w]));
        }
        if (p.top) maxima[32 * part] = most;
        top = fmaxf(top, most);
      }
    }
    for (int off = group >> 1; off; off >>= 1) top = fmaxf(top, __shfl_xor_sync(kFull, top, off));
    const float base = top == -INFINITY ? 0.0f : top;
    float s = 0.0f, t = 0.0f;
    if (live) {
#pragma unroll 4
      for (int v = sub; v < all; v += group) {
        const Vec<T, W> q = x[v];
#pragma unroll
        for (int w = 0; w < W; ++w) {
          const float u = exponent_of(to_f(q.v[w]), base, p.scale), e = exp2_fast(u);
          s += e;
          t = fmaf(e, u, t);
        }
      }
    }
    for (int off = group >> 1; off; off >>= 1) {
      s += __shfl_xor_sync(kFull, s, off);
      t += __shfl_xor_sync(kFull, t, off);
    }
    const Row r = finish_row(top, s, t);
    __syncwarp();
    if (live && sub == 0) {
      float lp = 0.0f;
      if (action >= 0 && action < p.actions) {
        const float xa = to_f(reinterpret_cast<const T *>(x)[action]);
        lp = xa == -INFINITY ? -INFINITY : log_prob_of(p, xa, top, r.log_sum);
      }
      p.log_prob[row] = lp;
      p.entropy[row] = r.entropy;
      p.max_logit[row] = r.top;
      p.log_sum[row] = (float)r.log_sum;
    }
    if (p.top) {
      float *values = reinterpret_cast<float *>(own + b.results);
      int *places = reinterpret_cast<int *>(values + rows * p.top);
      // (halves, whose difference stays in range; the logarithm in two parts costs a round less than 64 bits:
      // 262144 x 82 fp32 with 4 best 34.4 us for 35.1)
      const float twice = 2.0f * p.inverse, high = (float)r.log_sum, low = (float)(r.log_sum - (double)high);
      for (int rank = 0; rank < p.top; ++rank) {
        // the first part with the lane's largest, since indices ascend
        float best = -INFINITY;
        int part = 0;
        if (live) {
          for (int i = 0; i < b.parts; ++i) {
            const float most = maxima[32 * i];
            if (most > best) {
              best = most;
              part = i;
            }
          }
        }
        int at = 0x7fffffff;
        if (best > -INFINITY) {
#pragma unroll
          for (int k = kEach - 1; k >= 0; --k) {
            const int v = sub + (part * kEach + k) * group;
            if (v >= all) continue;
            const Vec<T, W> q = x[v];
#pragma unroll
            for (int w = W - 1; w >= 0; --w)
              if (to_f(q.v[w]) == best) at = v * W + w;
          }
        }
        const int candidate = at;
        for (int off = group >> 1; off; off >>= 1) {
          const float other = __shfl_xor_sync(kFull, best, off);
          const int place = __shfl_xor_sync(kFull, at, off);
          if (other > best || (other == best && place < at)) {
            best = other;
            at = place;
          }
        }
        if (live && at != 0x7fffffff && at == candidate) {  // taken out, and its part's maximum is the next one
          reinterpret_cast<T *>(x)[at] = from_f<T>(-INFINITY);
          float most = -INFINITY;
#pragma unroll
          for (int k = 0; k < kEach; ++k) {
            const int v = sub + (part * kEach + k) * group;
            if (v >= all) break;
            const Vec<T, W> q = x[v];
#pragma unroll
            for (int w = 0; w < W; ++w) most = fmaxf(most, to_f(q.v[w]));
          }
          maxima[32 * part] = most;
        }
        if (live && sub == 0) {
          values[mine * p.top + rank] =
              at == 0x7fffffff ? -INFINITY : fmaf(fmaf(0.5f, best, -0.5f * top), twice, -high) - low;
          places[mine * p.top + rank] = at == 0x7fffffff ? -1 : at;
        }
      }
      __syncwarp();
      for (int i = lane; i < count * p.top; i += 32) {
        p.top_log_prob[first * p.top + i] = values[i];
        p.top_action[first * p.top + i] = places[i];
      }
    }
    __syncwarp();
  }
}

// What a row's gradient needs: with v = (x - base) scale - log_sum, p = 2^v,
// d = p (offset + slope v), and g more at the action.  (offset and slope are
// negative: p goes with them.)
struct RowGradient {
  float base, log_sum, offset, slope;
  float g;
  int action;  // -1 where it is not kept
};
// in two steps, whose loads depend on one another
template <typename T>
struct RowLoads {
  float top, log_sum, entropy, g, h, x;
  int action;
  bool kept;
  __device__ __forceinline__ void first(const Params &p, int64_t row) {
    top = p.max_logit[row];
    log_sum = p.log_sum[row];
    action = p.action[row];
    g = p.grad_log_prob ? p.grad_log_prob[row] : 0.0f;
    h = p.grad_entropy ? p.grad_entropy[row] : 0.0f;
    entropy = p.grad_entropy ? p.entropy[row] : 0.0f;
  }
  __device__ __forceinline__ void second(const Params &p, int64_t row) {
    kept = action >= 0 && action < p.actions;
    x = kept ? to_f(static_cast<const T *>(p.logits)[row * p.stride + action]) : 0.0f;
    if (kept && p.legal) kept = p.legal[row * p.actions + action];
  }
  __device__ __forceinline__ RowGradient finish(const Params &p) const {
    const bool keep = kept && x != -INFINITY;
    RowGradient r = {top, log_sum * kLog2E, 0.0f, -h * p.inverse * kLn2, keep ? g * p.inverse : 0.0f, keep ? action : -1};
    if (top == -INFINITY) r.base = r.log_sum = 0.0f;
    r.offset = -(r.g + (h == 0.0f ? 0.0f : h * p.inverse * entropy));
    return r;
  }
};

__device__ __forceinline__ float2 gradient_of(const RowGradient &r, float2 x, float scale) {
  float2 v = __ffma2_rn(__fadd2_rn(x, make_float2(-r.base, -r.base)), make_float2(scale, scale),
                        make_float2(-r.log_sum, -r.log_sum));
  v = make_float2(max_nan(v.x, kNothing), max_nan(v.y, kNothing));
  return __fmul2_rn(make_float2(exp2_fast(v.x), exp2_fast(v.y)),
                    __ffma2_rn(make_float2(r.slope, r.slope), v, make_float2(r.offset, r.offset)));
}
__device__ __forceinline__ float gradient_of(const RowGradient &r, float x, float scale) {
  const float v = max_nan(fmaf(x - r.base, scale, -r.log_sum), kNothing);
  return exp2_fast(v) * fmaf(r.slope, v, r.offset);
}

// The gradient of short rows.  CTAs take groups of rows in turn, whole 16-byte
// pieces of them in order where rows are dense (C cells of W elements each, a
// cell within a row); a group's first threads gather what the next one's rows
// need while this one is computed.
constexpr int kMaxRows = 256;  // of a group
constexpr int kGradientCtas = 8;  // of an SM: 262144 x 82 fp32 39 us, 42 with six and more registers each
constexpr int kGroupElements = 6144;
template <typename T, int W, int C>
__global__ void __launch_bounds__(kThreads, kGradientCtas) short_gradient_kernel(const __grid_constant__ Params p, int rows,
                                                                  uint32_t reciprocal) {
  constexpr int N = W * C;
  __shared__ RowGradient tables[2][kMaxRows];
  const int all = p.actions / W;  // cells of a row
  const int64_t groups = (p.rows + rows - 1) / rows;
  const bool gathers = (int)threadIdx.x < rows;
  RowLoads<T> loads;
  {
    const int64_t row = (int64_t)blockIdx.x * rows + threadIdx.x;
    if (gathers && row < p.rows) {
      loads.first(p, row);
      loads.second(p, row);
      tables[0][threadIdx.x] = loads.finish(p);
    }
  }
  __syncthreads();
  int turn = 0;
  for (int64_t group = blockIdx.x; group < groups; group += gridDim.x, turn ^= 1) {
    const int64_t first = group * rows, next = (group + gridDim.x) * rows + threadIdx.x;
    const int count = (int)min((int64_t)rows, p.rows - first), cells = count * all;
    const RowGradient *table = tables[turn];
    const T *logits = static_cast<const T *>(p.logits) + first * p.stride;
    const uint8_t *legal = p.legal ? p.legal + first * p.actions : nullptr;
    T *grad = static_cast<T *>(p.grad) + first * p.actions;
    const bool gather = gathers && next < p.rows;
    if (gather) loads.first(p, next);
    for (int begin = 0; begin < cells; begin += kThreads * C) {
      const int cell = begin + (int)threadIdx.x * C;
      int row = all == 1 ? cell : (int)__umulhi((uint32_t)cell, reciprocal), at = cell - row * all;
      Vec<T, N> q;
      Vec<uint8_t, N> keep;
      const bool whole = cell + C <= cells;
      if (whole) {
        q = *reinterpret_cast<const Vec<T, N> *>(C > 1 ? logits + cell * W : logits + row * p.stride + at * W);
        if (legal) keep = *reinterpret_cast<const Vec<uint8_t, N> *>(legal + cell * W);
      } else if (cell < cells) {
#pragma unroll
        for (int n = 0; n < N; ++n)
          if (cell * W + n < cells * W) {
            q.v[n] = C > 1 ? logits[cell * W + n] : logits[row * p.stride + at * W + n];
            keep.v[n] = !legal || legal[cell * W + n];
          }
      }
      if (begin == 0 && gather) loads.second(p, next);
      if (cell >= cells) continue;
      Vec<T, N> out;
#pragma unroll
      for (int c = 0; c < C; ++c) {
        const RowGradient r = table[row < count ? row : 0];
        float d[W];
        if constexpr (W % 2 == 0) {
#pragma unroll
          for (int w = 0; w < W; w += 2) {
            const float2 two = gradient_of(r, make_float2(to_f(q.v[c * W + w]), to_f(q.v[c * W + w + 1])), p.scale);
            d[w] = two.x;
            d[w + 1] = two.y;
          }
        } else {
          d[0] = gradient_of(r, to_f(q.v[c]), p.scale);
        }
        const int action = r.action - at * W;  // of the cell
#pragma unroll
        for (int w = 0; w < W; ++w) {
          if (w == action) d[w] += r.g;
          out.v[c * W + w] = from_f<T>(legal && !keep.v[c * W + w] ? 0.0f : d[w]);
        }
        if (++at == all) {
          at = 0;
          ++row;
        }
      }
      if (whole) {
        *reinterpret_cast<Vec<T, N> *>(grad + cell * W) = out;
      } else {
#pragma unroll
        for (int n = 0; n < N; ++n)
          if (cell * W + n < cells * W) grad[cell * W + n] = out.v[n];
      }
    }
    if (gather) tables[turn ^ 1][threadIdx.x] = loads.finish(p);
    __syncthreads();
  }
}

// ---------------------------------------------------------------------------
// long rows: a cluster each
// ---------------------------------------------------------------------------

// A chunk of kVectors vectors a thread: their loads are in flight together,
// and one comparison decides whether its sums change their base.
constexpr int kVectors = 4;
// What is below kFloor counts as -inf in a row whose maximum is above kLow: 2^((kFloor -
// kLow) scale) is 0 at every temperature.  A row whose maximum is above kHigh is not summed
// this way either: exponents might end at -inf, and 0 times that is no number.
constexpr float kFloor = -0x1p100f, kLow = -0x1p99f, kHigh = 0x1p99f;

// 32 bits of -inf
template <typename T>
constexpr uint32_t kMinusInfinity = std::is_same_v<T, float> ? 0xff800000u
                                    : std::is_same_v<T, __half> ? 0xfc00fc00u : 0xff80ff80u;

// Chunks on their way from memory: every thread copies its own vectors (and
// the words that hold their masks' bytes) and reads them alone, so nothing
// but its own copies is waited for.  Two stages: three measured the same.
template <typename T, bool Masked>
struct Ring {
  static constexpr int kStages = 2, kWords = Masked ? 4 / sizeof(T) + 1 : 0;
  uint4 q[kStages][kVectors][kLong];
  uint32_t m[kStages][kVectors][Masked ? kWords : 1][Masked ? kLong : 1];
};

// -inf where the mask's byte is 0
template <typename T>
__device__ __forceinline__ void apply(const uint32_t (&m)[4 / sizeof(T)], uint4 &q) {
  uint32_t *word = reinterpret_cast<uint32_t *>(&q);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t keep = sizeof(T) == 4 ? __byte_perm(__vcmpne4(m[0], 0u), 0u, 0x1111 * i)
                                         : __byte_perm(__vcmpne4(m[sizeof(T) == 4 ? 0 : i / 2], 0u), 0u,
                                                       i & 1 ? 0x3322 : 0x1100);
    word[i] = (word[i] & keep) | (kMinusInfinity<T> & ~keep);
  }
}

// A row's elements as the threads of its cluster take them: vectors from the
// first 16-byte boundary on, thread after thread, and the head's and the
// tail's elements one by one by the last threads, which may have a vector less.
template <typename T, bool Masked>
struct Slice {
  static constexpr int W = 16 / sizeof(T);
  const T *x;
  const uint8_t *legal;
  int actions, head, vectors;

  __device__ Slice(const Params &p, int64_t row) {
    x = static_cast<const T *>(p.logits) + row * p.stride;
    legal = Masked ? p.legal + row * p.actions : nullptr;
    actions = p.actions;
    head = min(actions, (int)((16 - (reinterpret_cast<uintptr_t>(x) & 15)) & 15) / (int)sizeof(T));
    vectors = (actions - head) / W;
  }
  // the thread's odd element, or -1
  __device__ int odd(int index, int threads) const {
    const int back = threads - 1 - index, tail = head + vectors * W;
    return back < head ? back : back - head < actions - tail ? tail + back - head : -1;
  }
  __device__ int first(int v) const { return head + v * W; }
  // the mask's bytes of the W elements from `a` on
  __device__ void mask(const Params &p, int a, uint32_t (&m)[W / 4]) const {
    const uint8_t *bytes = legal + a;
    const int off = (int)(reinterpret_cast<uintptr_t>(bytes) & 3);
    const uint32_t *word = reinterpret_cast<const uint32_t *>(bytes - off);
    if (off == 0) {
#pragma unroll
      for (int w = 0; w < W / 4; ++w) m[w] = word[w];
    } else if (bytes - off >= p.legal && bytes + W + 4 <= p.legal + p.rows * p.actions) {
#pragma unroll
      for (int w = 0; w < W / 4; ++w) m[w] = __funnelshift_r(word[w], word[w + 1], 8 * off);
    } else {
#pragma unroll
      for (int w = 0; w < W; ++w) m[w / 4] = (w & 3 ? m[w / 4] : 0u) | (uint32_t)bytes[w] << (8 * (w & 3));
    }
  }
  // how far a vector's mask begins behind a word's
  __device__ int shift(int v) const { return (int)(reinterpret_cast<uintptr_t>(legal + first(v)) & 3); }
  // requests the vectors v, v + threads, ...; -inf where there is none
  __device__ void request(const Params &p, int v, int threads, Ring<T, Masked> &ring, int stage) const {
    const uint4 *at = reinterpret_cast<const uint4 *>(x + head) + v;
    const uint32_t none = kMinusInfinity<T>;
#pragma unroll
    for (int k = 0; k < kVectors; ++k) {
      uint4 *to = &ring.q[stage][k][threadIdx.x];
      if (v + k * threads >= vectors) {
        *to = make_uint4(none, none, none, none);
        continue;
      }
      copy_async<16>(to, at + k * threads);
      if constexpr (Masked) {
        const uint8_t *bytes = legal + first(v + k * threads), *word = bytes - shift(v + k * threads);
        if (word >= p.legal && word + 4 * ring.kWords <= p.legal + p.rows * p.actions) {
#pragma unroll
          for (int w = 0; w < ring.kWords; ++w) copy_async<4>(&ring.m[stage][k][w][threadIdx.x], word + 4 * w);
        } else {  // some of these words reach beyond the mask
#pragma unroll
          for (int w = 0; w < ring.kWords; ++w) {
            uint32_t u = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i)
              if (word + 4 * w + i >= bytes && word + 4 * w + i < bytes + W) u |= (uint32_t)word[4 * w + i] << (8 * i);
            ring.m[stage][k][w][threadIdx.x] = u;
          }
        }
      }
    }
  }
  // what was requested, with -inf where the mask's byte is 0
  __device__ void take(int v, int threads, const Ring<T, Masked> &ring, int stage, uint4 (&q)[kVectors]) const {
#pragma unroll
    for (int k = 0; k < kVectors; ++k) {
      q[k] = ring.q[stage][k][threadIdx.x];
      if constexpr (Masked) {
        const int bits = 8 * shift(v + k * threads);
        uint32_t m[W / 4];
#pragma unroll
        for (int w = 0; w < W / 4; ++w)
          m[w] = __funnelshift_r(ring.m[stage][k][w][threadIdx.x], ring.m[stage][k][w + 1][threadIdx.x], bits);
        apply<T>(m, q[k]);
      }
    }
  }
  // -inf where the element is not kept
  __device__ float element(int a) const { return !Masked || legal[a] ? to_f(x[a]) : -INFINITY; }
};

// the largest of three, without those that are NaN
__device__ __forceinline__ float max3(float a, float b, float c) {
  float y;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
  return y;
}

// A chunk as pairs of floats, what is below kFloor raised to it, NaN kept.
// bfloat16 stays packed until a pair is needed, so that raising it and the
// chunk's maximum take half an instruction an element.
template <typename T>
struct Chunk {
  static constexpr int W = 16 / sizeof(T), N = W * kVectors;
  float y[N];
  __device__ explicit Chunk(const uint4 (&q)[kVectors]) {
    const uint32_t *word = reinterpret_cast<const uint32_t *>(q);
    if constexpr (std::is_same_v<T, float>) {
#pragma unroll
      for (int i = 0; i < N; ++i) y[i] = max_nan(__uint_as_float(word[i]), kFloor);
    } else {
#pragma unroll
      for (int i = 0; i < N / 2; ++i) {
        const float2 two = floats<T>(word[i]);
        y[2 * i] = max_nan(two.x, kFloor);
        y[2 * i + 1] = max_nan(two.y, kFloor);
      }
    }
  }
  __device__ float2 pair(int i) const { return make_float2(y[2 * i], y[2 * i + 1]); }
  __device__ float largest() const {
    float m[4];
#pragma unroll
    for (int c = 0; c < 4; ++c) m[c] = fmaxf(y[c], y[c + 4]);
#pragma unroll
    for (int i = 8; i < N; i += 8)
#pragma unroll
      for (int c = 0; c < 4; ++c) m[c] = max3(m[c], y[i + c], y[i + c + 4]);
    return max3(m[0], m[1], fmaxf(m[2], m[3]));
  }
};
template <>
struct Chunk<__nv_bfloat16> {
  static constexpr int W = 8, N = W * kVectors;
  __nv_bfloat162 y[N / 2];
  __device__ explicit Chunk(const uint4 (&q)[kVectors]) {
    const __nv_bfloat162 floor = __float2bfloat162_rn(kFloor), *two = reinterpret_cast<const __nv_bfloat162 *>(q);
#pragma unroll
    for (int i = 0; i < N / 2; ++i) y[i] = __hmax2_nan(two[i], floor);
  }
  __device__ float2 pair(int i) const { return floats<__nv_bfloat16>(*reinterpret_cast<const uint32_t *>(&y[i])); }
  __device__ float largest() const {
    __nv_bfloat162 m[4];
#pragma unroll
    for (int c = 0; c < 4; ++c) m[c] = __hmax2(y[c], y[c + 4]);
#pragma unroll
    for (int i = 8; i < N / 2; ++i) m[i & 3] = __hmax2(m[i & 3], y[i]);
    const __nv_bfloat162 one = __hmax2(__hmax2(m[0], m[1]), __hmax2(m[2], m[3]));
    return fmaxf(__low2float(one), __high2float(one));
  }
};

// Sums of a thread or of more: s = sum 2^v, t = sum v 2^v, v = (x - top) scale
struct Sums {
  float top, s, t;
};
__device__ __forceinline__ void rebase(Sums &a, float top, float scale) {
  if (a.s != 0.0f) {
    const float d = (a.top - top) * scale, f = exp2_fast(d);
    a.t = f == 0.0f ? 0.0f : f * fmaf(d, a.s, a.t);
    a.s *= f;
  }
  a.top = top;
}

// returns the chunk's maximum
template <typename T>
__device__ __forceinline__ float add_chunk(const Chunk<T> &y, float scale, Sums &a) {
  const float most = y.largest();
  if (most > a.top) rebase(a, most, scale);
  const float2 scale2 = make_float2(scale, scale), top2 = make_float2(-a.top, -a.top);
  float2 s[2] = {}, t[2] = {};
#pragma unroll
  for (int i = 0; i < Chunk<T>::N / 2; ++i) {
    const float2 v = __fmul2_rn(__fadd2_rn(y.pair(i), top2), scale2);
    const float2 e = make_float2(exp2_fast(v.x), exp2_fast(v.y));
    s[i & 1] = __fadd2_rn(s[i & 1], e);
    t[i & 1] = __ffma2_rn(e, v, t[i & 1]);
  }
  s[0] = __fadd2_rn(s[0], s[1]);
  t[0] = __fadd2_rn(t[0], t[1]);
  a.s += s[0].x + s[0].y;
  a.t += t[0].x + t[0].y;
  return most;
}

struct Shared {
  float4 maxima[kMaxGroups / 4];
  float2 sums[kMaxCluster * kWarps];
  uint64_t keys[kCandidates];
  float parts[kParts][kLong];  // maxima of the threads' parts
  uint16_t reach[kParts * kLong];
  int count[2], reaching[2];  // of rows in turn
  float limit;
  uint64_t best[kWarps];
};

// The groups' maxima to every CTA of the cluster; returns the row's
__device__ __forceinline__ float exchange(Shared &sh, float top, int ctas, int rank, int groups) {
  cg::cluster_group cluster = cg::this_cluster();
  const int per_cta = groups / ctas, width = kLong / per_cta;  // threads of a group
  for (int off = width >> 1; off; off >>= 1) top = fmaxf(top, __shfl_xor_sync(kFull, top, off));
  if ((threadIdx.x & (width - 1)) == 0) {
    const int g = rank * per_cta + threadIdx.x / width;
    if (ctas == 1)
      reinterpret_cast<float *>(sh.maxima)[g] = top;
    else
      for (int c = 0; c < ctas; ++c) reinterpret_cast<float *>(cluster.map_shared_rank(&sh, c)->maxima)[g] = top;
  }
  if (ctas == 1)
    __syncthreads();
  else
    cluster.sync();
  float largest = -INFINITY;
  for (int g = threadIdx.x & 31; g < groups / 4; g += 32) {
    const float4 m = sh.maxima[g];
    largest = fmaxf(largest, fmaxf(fmaxf(m.x, m.y), fmaxf(m.z, m.w)));
  }
#pragma unroll
  for (int off = 16; off; off >>= 1) largest = fmaxf(largest, __shfl_xor_sync(kFull, largest, off));
  return largest;
}

// The top-th largest of the groups' maxima, equal ones by their place
__device__ __forceinline__ void find_limit(Shared &sh, int groups, int top) {
  if ((int)threadIdx.x < groups) {
    const float mine = reinterpret_cast<const float *>(sh.maxima)[threadIdx.x];
    int above = 0;
    for (int g = 0; g < groups / 4; ++g) {
      const float4 m = sh.maxima[g];
      const int i = 4 * g - (int)threadIdx.x;
      above += m.x > mine || (m.x == mine && i < 0);
      above += m.y > mine || (m.y == mine && i + 1 < 0);
      above += m.z > mine || (m.z == mine && i + 2 < 0);
      above += m.w > mine || (m.w == mine && i + 3 < 0);
    }
    if (above == top - 1) sh.limit = mine;
  }
}

__device__ __forceinline__ void candidate(Shared *home, int turn, float v, float limit, int a) {
  if (v >= limit && v > -INFINITY) {
    const int at = atomicAdd(&home->count[turn], 1);
    if (at < kCandidates) home->keys[at] = key_of(v, a);
  }
}

// A row with more than kCandidates elements at the limit is read `top` times by
// its cluster's first CTA: 4096 x 32000 bf16 of equal logits with 1, 5 and 20 best
// 0.71, 0.99 and 2.6 ms (other logits with 20: 70 us), 8 x 131071 fp32 0.24, 0.40
// and 1.0.
//
// The row's numbers and its best actions, by the first CTA.  What it reads of
// `sh` is written again after the next row's exchange, where all its threads meet.
template <typename T, bool Masked>
__device__ __forceinline__ void finish_long(const Params &p, Shared &sh, const Slice<T, Masked> &slice, int64_t row,
                                            float largest, int turn, int ctas) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int count = p.top ? sh.count[turn] : 0;
  // a warp without candidates has nothing to write
  if (warp && 32 * warp >= count && 32 * warp >= p.top && count <= kCandidates) return;
  Played q = {false, 0.0f};
  if (threadIdx.x == 0) q = played<T>(p, row);  // (on its way while the sums are added)
  float s = 0.0f, t = 0.0f;
  for (int i = lane; i < ctas * kWarps; i += 32) {
    s += sh.sums[i].x;
    t += sh.sums[i].y;
  }
#pragma unroll
  for (int off = 16; off; off >>= 1) {
    s += __shfl_xor_sync(kFull, s, off);
    t += __shfl_xor_sync(kFull, t, off);
  }
  const Row r = finish_row(largest, s, t);
  if (threadIdx.x == 0) write_row(p, row, r, q);
  if (!p.top) return;
  if (count <= kCandidates) {
    for (int i = threadIdx.x; i < count; i += kLong) {
      const uint64_t mine = sh.keys[i];
      int above = 0;
      for (int j = 0; j < count; ++j) above += sh.keys[j] > mine;
      if (above < p.top) write_top(p, row, r, above, logit_of((uint32_t)(mine >> 32)), (int)~(uint32_t)mine);
    }
    for (int i = count + threadIdx.x; i < p.top; i += kLong) write_top(p, row, r, i, 0.0f, -1);
    return;
  }
  uint64_t last = ~0ull;
  for (int i = 0; i < p.top; ++i) {
    uint64_t best = 0;
    for (int k = threadIdx.x; k < p.actions; k += kLong) {
      const float v = slice.element(k);
      if (!(v > -INFINITY)) continue;
      const uint64_t key = key_of(v, k);
      if (key < last && key > best) best = key;
    }
#pragma unroll
    for (int off = 16; off; off >>= 1) best = max(best, __shfl_xor_sync(kFull, best, off));
    if (lane == 0) sh.best[warp] = best;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kWarps; ++w) best = max(best, sh.best[w]);
    __syncthreads();
    last = best;
    if (threadIdx.x == 0) write_top(p, row, r, i, logit_of((uint32_t)(best >> 32)), (int)~(uint32_t)best);
  }
}

template <bool Masked>
constexpr int kLongCtas = Masked ? 5 : 6;  // of an SM: registers and, with masks, shared memory

// Clusters take row after row.  A thread's next chunks, the next row's among
// them, are on their way while this one is added up and the row is finished.
template <typename T, bool Masked>
__global__ void __launch_bounds__(kLong, kLongCtas<Masked>) long_kernel(const __grid_constant__ Params p) {
  constexpr int W = 16 / sizeof(T), kStages = Ring<T, Masked>::kStages;
  extern __shared__ __align__(16) uint8_t ring_bytes[];
  __shared__ Shared sh;
  Ring<T, Masked> &ring = *reinterpret_cast<Ring<T, Masked> *>(ring_bytes);
  cg::cluster_group cluster = cg::this_cluster();
  const int ctas = cluster.num_blocks(), rank = cluster.block_rank();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int index = rank * kLong + threadIdx.x, threads = ctas * kLong, step = kVectors * threads;
  const int groups = max(64, kWarps * ctas);
  if (threadIdx.x < 2) sh.count[threadIdx.x] = sh.reaching[threadIdx.x] = 0;
  // the cluster's CTAs have begun, and counts are set, before the first write into another's memory
  if (ctas > 1) cluster.barrier_arrive();
  Shared *home = ctas == 1 ? &sh : cluster.map_shared_rank(&sh, 0);

  const int64_t rows_apart = gridDim.x / ctas;
  // of every row: one that begins off a boundary may leave its last chunk empty
  const int chunks = max(1, (p.actions / W + step - 1) / step), per_part = (chunks + kParts - 1) / kParts;
  // what is requested next
  int64_t ahead_row = blockIdx.x / ctas;
  int ahead_chunk = 0, ahead_stage = 0, stage = 0;
  Slice<T, Masked> ahead(p, ahead_row);
  auto request = [&]() {
    if (ahead_row < p.rows) {
      ahead.request(p, index + ahead_chunk * step, threads, ring, ahead_stage);
      if (++ahead_chunk == chunks) {
        ahead_chunk = 0;
        ahead_row += rows_apart;
        if (ahead_row < p.rows) ahead = Slice<T, Masked>(p, ahead_row);
      }
    }
    ahead_stage = ahead_stage + 1 == kStages ? 0 : ahead_stage + 1;
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
#pragma unroll 1
  for (int i = 0; i + 1 < kStages; ++i) request();

  bool begun = ctas == 1;
  int turn = 0;
  for (int64_t row = blockIdx.x / ctas; row < p.rows; row += rows_apart, turn ^= 1) {
    const Slice<T, Masked> slice(p, row);
    const int odd = slice.odd(index, threads);
    Sums a = {-INFINITY, 0.0f, 0.0f};
    if (odd >= 0) {
      const float y = max_nan(slice.element(odd), kFloor);
      a = Sums{y, 1.0f, 0.0f};
      if (y != y) a = Sums{-INFINITY, y, y};
    }
    float part = -INFINITY;
#pragma unroll 1
    for (int chunk = 0, left = per_part, to = 0; chunk < chunks; ++chunk) {
      request();
      asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 1) : "memory");
      uint4 q[kVectors];
      slice.take(index + chunk * step, threads, ring, stage, q);
      stage = stage + 1 == kStages ? 0 : stage + 1;
      part = fmaxf(part, add_chunk(Chunk<T>(q), p.scale, a));
      if (--left == 0 || chunk + 1 == chunks) {
        if (p.top) sh.parts[to][threadIdx.x] = part;
        ++to;
        part = -INFINITY;
        left = per_part;
      }
    }

    if (!begun) cluster.barrier_wait();
    begun = true;
    float largest = exchange(sh, a.top, ctas, rank, groups);
    // a row masked throughout by low values, or with an infinity or near it: element by element, as they are
    // (4096 x 32000 bf16 with a mask, of which one row in 64 has nothing left, 119 us for 96)
    const bool plain = largest >= kLow && largest <= kHigh;
    if (!plain) {
      a.top = odd >= 0 ? slice.element(odd) : -INFINITY;
      for (int i = 0; i * per_part < chunks; ++i) {
        part = -INFINITY;
        for (int v = index + i * per_part * step; v < min(slice.vectors, (i + 1) * per_part * step); v += threads)
          for (int w = 0; w < W; ++w) part = fmaxf(part, slice.element(slice.first(v) + w));
        if (p.top) sh.parts[i][threadIdx.x] = part;
        a.top = fmaxf(a.top, part);
      }
      if (ctas > 1)
        cluster.sync();  // before the maxima are written again
      else
        __syncthreads();
      largest = exchange(sh, a.top, ctas, rank, groups);
      const float base = largest == -INFINITY ? 0.0f : largest;
      a.s = a.t = 0.0f;
      auto one = [&](float x) {
        const float u = exponent_of(x, base, p.scale), e = exp2_fast(u);
        a.s += e;
        a.t = fmaf(e, u, a.t);
      };
      if (odd >= 0) one(slice.element(odd));
      for (int v = index; v < slice.vectors; v += threads)
        for (int w = 0; w < W; ++w) one(slice.element(slice.first(v) + w));
    }
    const float own = a.top;  // the largest of the thread's own elements
    if (plain) rebase(a, largest, p.scale);
    if (threadIdx.x == 0) sh.count[turn ^ 1] = sh.reaching[turn ^ 1] = 0;

    if (p.top) {
      find_limit(sh, groups, p.top);
      __syncthreads();
      const float limit = plain && sh.limit <= kFloor ? -INFINITY : sh.limit;
      // the parts that reach the limit, and their vectors over all threads of the CTA
      if (own >= limit && own > -INFINITY) {
        for (int i = 0; i * per_part < chunks; ++i)
          if (sh.parts[i][threadIdx.x] >= limit)
            sh.reach[atomicAdd(&sh.reaching[turn], 1)] = (uint16_t)(i * kLong + threadIdx.x);
        if (odd >= 0) candidate(home, turn, slice.element(odd), limit, odd);
      }
      __syncthreads();
      const int each = kVectors * per_part, items = sh.reaching[turn] * each;
      for (int i = threadIdx.x; i < items; i += kLong) {
        const int n = i / each, which = sh.reach[n];
        const int v = rank * kLong + which % kLong + (which / kLong * each + i - n * each) * threads;
        if (v >= slice.vectors) continue;
        const int first = slice.first(v);
        const Vec<T, W> q = *reinterpret_cast<const Vec<T, W> *>(slice.x + first);
        uint32_t high = 0;
#pragma unroll
        for (int w = 0; w < W; ++w) high |= (to_f(q.v[w]) >= limit ? 1u : 0u) << w;
        for (; high; high &= high - 1) {
          const int k = first + __ffs(high) - 1;
          candidate(home, turn, slice.element(k), limit, k);
        }
      }
    }
#pragma unroll
    for (int off = 16; off; off >>= 1) {
      a.s += __shfl_xor_sync(kFull, a.s, off);
      a.t += __shfl_xor_sync(kFull, a.t, off);
    }
    if (lane == 0) home->sums[rank * kWarps + warp] = make_float2(a.s, a.t);
    if (ctas == 1)
      __syncthreads();
    else
      cluster.sync();
    if (rank == 0) finish_long<T, Masked>(p, sh, slice, row, largest, turn, ctas);
  }
}

// A long row's gradient: elements alone, so a CTA takes a piece of a row.
// Vectors where a row and its gradient lie alike.
constexpr int kAhead = 4;  // vectors of a thread, whose loads are in flight together
template <typename T, bool Vector>
constexpr int kPiece = kThreads * kAhead * (Vector ? 16 / (int)sizeof(T) : 4);
template <typename T, bool Vector, bool Masked>
__global__ void __launch_bounds__(kThreads) long_gradient_kernel(const __grid_constant__ Params p, int pieces) {
  constexpr int W = 16 / sizeof(T);
  const int64_t row = blockIdx.x / pieces;
  const int piece = blockIdx.x - (int)(row * pieces);
  const Slice<T, Masked> slice(p, row);
  const T *x = slice.x;
  T *grad = static_cast<T *>(p.grad) + row * p.actions;
  const int head = Vector ? slice.head : 0, begin = head + piece * kPiece<T, Vector>;
  const int whole = Vector ? slice.first(slice.vectors) : p.actions;
  RowLoads<T> loads;
  loads.first(p, row);
  if constexpr (Vector) {
    uint4 q[kAhead];
    uint32_t m[Masked ? kAhead : 1][W / 4];
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const int i = begin + (k * kThreads + (int)threadIdx.x) * W;
      if (i >= whole) continue;
      q[k] = *reinterpret_cast<const uint4 *>(x + i);
      if constexpr (Masked) slice.mask(p, i, m[k]);
    }
    loads.second(p, row);
    const RowGradient r = loads.finish(p);
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const int i = begin + (k * kThreads + (int)threadIdx.x) * W;
      if (i >= whole) continue;
      if constexpr (Masked) apply<T>(m[k], q[k]);
      uint32_t *word = reinterpret_cast<uint32_t *>(&q[k]);
#pragma unroll
      for (int w = 0; w < 4; w += sizeof(T) == 4 ? 2 : 1) {
        if constexpr (sizeof(T) == 4) {
          const float2 d = gradient_of(r, make_float2(__uint_as_float(word[w]), __uint_as_float(word[w + 1])), p.scale);
          word[w] = __float_as_uint(d.x);
          word[w + 1] = __float_as_uint(d.y);
        } else {
          const float2 d = gradient_of(r, floats<T>(word[w]), p.scale);
          if constexpr (std::is_same_v<T, __half>)
            *reinterpret_cast<__half2 *>(&word[w]) = __floats2half2_rn(d.x, d.y);
          else
            *reinterpret_cast<__nv_bfloat162 *>(&word[w]) = __floats2bfloat162_rn(d.x, d.y);
        }
      }
      *reinterpret_cast<uint4 *>(grad + i) = q[k];
    }
  } else {
    loads.second(p, row);
    const RowGradient r = loads.finish(p);
#pragma unroll 4
    for (int k = 0; k < kPiece<T, Vector> / kThreads; ++k) {
      const int i = begin + k * kThreads + (int)threadIdx.x;
      if (i < whole) grad[i] = from_f<T>(gradient_of(r, slice.element(i), p.scale));
    }
  }
  const RowGradient r = loads.finish(p);
  // the elements before the first vector and behind the last
  if (Vector && piece == 0) {
    const int i = (int)threadIdx.x < head ? (int)threadIdx.x : whole + (int)threadIdx.x - head;
    if (i < head || (i >= whole && i < p.actions)) grad[i] = from_f<T>(gradient_of(r, slice.element(i), p.scale));
  }
  // the action's element once more, by one thread behind a barrier: testing every vector costs the others 10 %
  const bool here = r.action >= 0 && (r.action < head || r.action >= whole
                                          ? piece == 0
                                          : (r.action - head) / kPiece<T, Vector> == piece);
  if (!here) return;
  __syncthreads();
  if (threadIdx.x == 0) grad[r.action] = from_f<T>(gradient_of(r, loads.x, p.scale) + r.g);
}

// ---------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------

bool misaligned(const void *q, size_t a) { return (reinterpret_cast<uintptr_t>(q) & (a - 1)) != 0; }

cudaError_t launched() {
  g_log_probs_launches.fetch_add(1, std::memory_order_relaxed);
  return cudaGetLastError();
}

// Rows and lanes of a batch: the fewest lanes a row with which reads of
// neighbouring rows share no bank, a warp's rows stay within kBatchBytes, and
// (when rows are few) every SM has eight warps' work.
constexpr int kBatchBytes = 11 * 1024, kSharedBytes = 220 * 1024;
template <typename T, int W>
cudaError_t short_rows(Params &p, bool gradient, int sms, cudaStream_t st) {
  const int all = p.actions / W;
  if (gradient) {
    // (whole eights of rows: a group then begins on a 16-byte boundary where the first does)
    const int rows = std::max(8, std::min(kMaxRows, kGroupElements / p.actions / 8 * 8));
    // cell / all for cells below 2^13 (8 rows of kMaxManyGradient, or kGroupElements): the quotient's error cell / 2^32 stays below 1 / all
    const uint32_t reciprocal = (uint32_t)((1ull << 32) / all + 1);
    const unsigned ctas = (unsigned)std::min<int64_t>((p.rows + rows - 1) / rows, (int64_t)sms * kGradientCtas);
    constexpr int C = 16 / (W * (int)sizeof(T));
    const uintptr_t at = reinterpret_cast<uintptr_t>(p.logits) | reinterpret_cast<uintptr_t>(p.grad);
    if (C > 1 && at % 16 == 0 && reinterpret_cast<uintptr_t>(p.legal) % (W * C) == 0 && p.stride == p.actions)
      short_gradient_kernel<T, W, C><<<ctas, kThreads, 0, st>>>(p, rows, reciprocal);
    else
      short_gradient_kernel<T, W, 1><<<ctas, kThreads, 0, st>>>(p, rows, reciprocal);
    return launched();
  }
  const int row_bytes = p.actions * ((int)sizeof(T) + (p.legal ? 1 : 0));
  // rows of whole 16-byte pieces lie 16 bytes further apart where that is odd, others share banks
  auto apart = [](const void *q, int64_t bytes) {
    return bytes % 32 == 0 && reinterpret_cast<uintptr_t>(q) % 16 == 0 ? (int)bytes + 16 : (int)bytes;
  };
  Batch b;
  b.pitch = apart(p.logits, (int64_t)p.actions * sizeof(T));
  b.legal_pitch = apart(p.legal, p.actions);
  p.group = b.pitch != p.actions * (int)sizeof(T) ? 1 : std::min(8, all & -all);
  while (p.group < 32 && (32 / p.group * row_bytes > kBatchBytes || p.rows * p.group < (int64_t)8 * 32 * sms)) p.group *= 2;
  const int rows = 32 / p.group;
  auto up = [](int n) { return (n + 15) / 16 * 16; };
  b.vectors = (all + p.group - 1) / p.group;
  b.parts = (b.vectors * W + kPartElements - 1) / kPartElements;
  b.legal = up(rows * b.pitch + 16);
  b.maxima = b.legal + (p.legal ? up(rows * b.legal_pitch + 16) : 0);
  b.results = b.maxima + (p.top ? 128 * b.parts : 0);
  b.bytes = b.results + up(8 * rows * p.top);
  const int bytes = kShortWarps * b.bytes;
  static std::atomic<uint64_t> allowed{0};
  int dev = 0;
  if (cudaError_t e = cudaGetDevice(&dev)) return e;
  const uint64_t bit = 1ull << (dev & 63);
  if (!(allowed.load(std::memory_order_acquire) & bit)) {
    const cudaError_t e =
        cudaFuncSetAttribute(short_kernel<T, W>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSharedBytes);
    if (e != cudaSuccess) return e;
    allowed.fetch_or(bit, std::memory_order_release);
  }
  const int64_t batches = (p.rows + rows - 1) / rows, wanted = (batches + kShortWarps - 1) / kShortWarps;
  const int64_t ctas = std::min<int64_t>(wanted, (int64_t)sms * std::min(12, kSharedBytes / (bytes + 1024)));
  short_kernel<T, W><<<(unsigned)ctas, kShortThreads, bytes, st>>>(p, b);
  return launched();
}

template <typename T, bool Vector, bool Masked>
cudaError_t launch_gradient(const Params &p, cudaStream_t st) {
  const int pieces = (p.actions + kPiece<T, Vector> - 1) / kPiece<T, Vector>;
  if (p.rows * pieces > 0x7fffffff) return cudaErrorInvalidValue;
  long_gradient_kernel<T, Vector, Masked><<<(unsigned)(p.rows * pieces), kThreads, 0, st>>>(p, pieces);
  return launched();
}

template <typename T, bool Masked>
cudaError_t launch_long(const Params &p, int sms, cudaStream_t st) {
  // a cluster of CTAs while rows leave SMs without work and pieces keep four vectors a thread
  int ctas = 1;
  while (ctas < kMaxCluster && p.rows * ctas * 2 <= 2 * sms && p.actions / (ctas * 2) >= 4096) ctas *= 2;
  constexpr int kRing = (int)sizeof(Ring<T, Masked>);
  static std::atomic<uint64_t> allowed{0};
  int dev = 0;
  if (cudaError_t e = cudaGetDevice(&dev)) return e;
  const uint64_t bit = 1ull << (dev & 63);
  if (!(allowed.load(std::memory_order_acquire) & bit)) {
    cudaError_t e = cudaFuncSetAttribute(long_kernel<T, Masked>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e == cudaSuccess)
      e = cudaFuncSetAttribute(long_kernel<T, Masked>, cudaFuncAttributeMaxDynamicSharedMemorySize, kRing);
    if (e != cudaSuccess) return e;
    allowed.fetch_or(bit, std::memory_order_release);
  }
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = ctas;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(std::min<int64_t>(p.rows, std::max(1, kLongCtas<Masked> * sms / ctas)) * ctas));
  cfg.blockDim = dim3(kLong);
  cfg.dynamicSmemBytes = kRing;
  cfg.stream = st;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, long_kernel<T, Masked>, p);
  if (e != cudaSuccess) return e;
  return launched();
}

template <typename T>
cudaError_t run(Params &p, bool gradient, int sms, cudaStream_t st) {
  if (p.actions <= kMaxShort || (p.actions <= (gradient ? kMaxManyGradient : kMaxMany) && p.rows >= (int64_t)8 * sms)) {
    // the widest loads that rows' places allow
    auto fits = [&](int w) {
      const uintptr_t all = reinterpret_cast<uintptr_t>(p.logits) | (uintptr_t)p.stride * sizeof(T) |
                            reinterpret_cast<uintptr_t>(p.grad) | (uintptr_t)p.actions * sizeof(T);
      return all % (w * sizeof(T)) == 0 && reinterpret_cast<uintptr_t>(p.legal) % w == 0;
    };
    if (fits(4)) return short_rows<T, 4>(p, gradient, sms, st);
    if (fits(2)) return short_rows<T, 2>(p, gradient, sms, st);
    return short_rows<T, 1>(p, gradient, sms, st);
  }
  if (gradient) {
    const bool vector = !(((reinterpret_cast<uintptr_t>(p.logits) ^ reinterpret_cast<uintptr_t>(p.grad)) & 15) ||
                          (p.rows > 1 && ((p.stride - p.actions) * sizeof(T) & 15)));
    if (p.legal) return vector ? launch_gradient<T, true, true>(p, st) : launch_gradient<T, false, true>(p, st);
    return vector ? launch_gradient<T, true, false>(p, st) : launch_gradient<T, false, false>(p, st);
  }
  return p.legal ? launch_long<T, true>(p, sms, st) : launch_long<T, false>(p, sms, st);
}

int sm_count() {
  int dev = 0, n = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return 148;
  if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n <= 0) return 148;
  return n;
}

int dispatch(Params &p, int32_t dtype, bool gradient, void *stream) {
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int sms = sm_count();
  const cudaError_t e = dtype == 0   ? run<float>(p, gradient, sms, st)
                        : dtype == 1 ? run<__nv_bfloat16>(p, gradient, sms, st)
                                     : run<__half>(p, gradient, sms, st);
  return e == cudaSuccess ? SCACCHI_OK : e == cudaErrorInvalidValue ? SCACCHI_EINVAL : SCACCHI_ECUDA;
}

bool rows_ok(const scacchi_log_prob_rows *r, int64_t num_rows, int32_t num_actions, int32_t dtype, double temperature) {
  if (!r || num_rows < 0 || num_actions < 1 || num_actions > kMaxActions || dtype < 0 || dtype > 2 ||
      !(temperature >= 1e-3 && temperature <= 1e3))
    return false;
  if (num_rows == 0) return true;
  return num_rows <= (int64_t)1 << 31 && r->logits && r->action && r->stride >= num_actions &&
         !misaligned(r->logits, dtype == 0 ? 4 : 2) && !misaligned(r->action, 4);
}

}  // namespace

extern "C" {

int scacchi_log_probs(const scacchi_log_prob_rows *rows, const scacchi_log_prob_out *out, int64_t num_rows,
                      int32_t num_actions, int32_t dtype, double temperature, int32_t top, void *stream) {
  if (!rows_ok(rows, num_rows, num_actions, dtype, temperature) || !out || top < 0 || top > kMaxTop)
    return SCACCHI_EINVAL;
  if (num_rows == 0) return SCACCHI_OK;
  for (const void *q : {(const void *)out->log_prob, (const void *)out->entropy, (const void *)out->max_logit,
                        (const void *)out->log_sum})
    if (!q || misaligned(q, 4)) return SCACCHI_EINVAL;
  if (top && (!out->top_log_prob || !out->top_action || misaligned(out->top_log_prob, 4) ||
              misaligned(out->top_action, 4)))
    return SCACCHI_EINVAL;
  Params p = {};
  p.logits = rows->logits;
  p.legal = rows->legal;
  p.action = rows->action;
  p.log_prob = out->log_prob;
  p.entropy = out->entropy;
  p.max_logit = out->max_logit;
  p.log_sum = out->log_sum;
  p.top_log_prob = out->top_log_prob;
  p.top_action = out->top_action;
  p.rows = num_rows;
  p.stride = rows->stride;
  p.actions = num_actions;
  p.top = top;
  p.scale = (float)(1.44269504088896340736 / temperature);
  p.inverse64 = 1.0 / temperature;
  p.inverse = (float)p.inverse64;
  return dispatch(p, dtype, false, stream);
}

int scacchi_log_probs_gradient(const scacchi_log_prob_rows *rows, const float *max_logit, const float *log_sum,
                               const float *entropy, const float *grad_log_prob, const float *grad_entropy,
                               int64_t num_rows, int32_t num_actions, int32_t dtype, double temperature,
                               void *grad_logits, void *stream) {
  if (!rows_ok(rows, num_rows, num_actions, dtype, temperature)) return SCACCHI_EINVAL;
  if (num_rows == 0) return SCACCHI_OK;
  if (!max_logit || !log_sum || !grad_logits || (grad_entropy && !entropy) || misaligned(max_logit, 4) ||
      misaligned(log_sum, 4) || misaligned(entropy, 4) || misaligned(grad_log_prob, 4) ||
      misaligned(grad_entropy, 4) || misaligned(grad_logits, dtype == 0 ? 4 : 2))
    return SCACCHI_EINVAL;
  Params p = {};
  p.logits = rows->logits;
  p.legal = rows->legal;
  p.action = rows->action;
  p.max_logit = const_cast<float *>(max_logit);
  p.log_sum = const_cast<float *>(log_sum);
  p.entropy = const_cast<float *>(entropy);
  p.grad_log_prob = grad_log_prob;
  p.grad_entropy = grad_entropy;
  p.grad = grad_logits;
  p.rows = num_rows;
  p.stride = rows->stride;
  p.actions = num_actions;
  p.scale = (float)(1.44269504088896340736 / temperature);
  p.inverse = (float)(1.0 / temperature);
  return dispatch(p, dtype, true, stream);
}

uint64_t scacchi_log_probs_launch_count(void) { return g_log_probs_launches.load(std::memory_order_relaxed); }

}  // extern "C"
