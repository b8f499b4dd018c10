// An AdamW step over many tensors in one launch, with moments in 32 bits or
// in 8, and the norm of many gradients.
//
//   g <- c g,   c = max_norm / max(norm, max_norm)
//   m <- b1 m + (1 - b1) g
//   v <- b2 v + (1 - b2) g^2,   r = sqrt v
//   w <- (1 - lr wd) w - (lr / (1 - b1^t)) m / (r / sqrt(1 - b2^t) + eps)
//
// 8-bit moments hold m and r, 256 elements in a block that shares a power of
// two, 2^e the binade of its largest: x = 2^e y with y an unsigned float of
// 8 (r) or 7 (m, and a sign) bits: 4 bits of exponent, the rest fraction,
// the exponent 14 standing for [1, 2), 0 for the subnormals below 2^-13.  A
// code is the upper part of the float 2^-113 y, whose exponent field begins
// at the same zero, so encoding is an addition and a shift of its bits, for
// subnormals alike, and decoding is a shift.  A root instead of v halves the
// exponents that a block spans: 2^-17 of the largest is still told apart.
//
// Rounding is stochastic: with b2 = 0.999 v moves by 1e-3 of itself a step
// at most when gradients fade, a sixtieth of the code's half step, and would
// never move when rounded to nearest.  Sixteen random bits an element come
// from Threefry-2x32 under fold_in(key, t): four consecutive elements share
// the 64 bits of one counter, so results depend neither on the launch's shape
// nor on the tensors' alignment.  The root and a bfloat16 weight take the
// same sixteen bits times an odd number (a bijection of 16 bits): their
// rounding does not follow the first moment's.  A root above zero never
// rounds to zero, which would leave m / eps.
//
// What is rounded to a code is computed without contraction (this file
// compiles with -fmad=false), so that the definition in plain operations
// gives the same codes.

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include <algorithm>
#include <atomic>
#include <type_traits>
#include <utility>
#include <vector>

#include "../../include/scacchi_b200.h"
#include "threefry.h"

namespace {

std::atomic<uint64_t> g_adamw_launches{0};

constexpr unsigned kFull = 0xffffffffu;
constexpr int kThreads = 256;
constexpr int kBlock = 256;   // elements that share an exponent; tensors begin at whole blocks
constexpr int kChunk = 4096;  // elements of a tensor that a CTA takes
constexpr int kNormChunk = 8192;
constexpr int kMaxPartials = 148 * 6;  // CTAs of a norm's launch
constexpr int kMaxDtype = 2;

// What a step's launches share, in device memory.
struct State {
  int64_t step;
  uint32_t key0, key1;  // of this step
  float clip, size, inv_root;
  int32_t skip;
  double learning_rate;
  uint64_t unused[2];
};
static_assert(sizeof(State) == 56 && sizeof(State) <= SCACCHI_ADAMW_STATE_BYTES, "state");

// A tensor of a launch's table, which travels in the kernel's parameters: no
// copy to the device, and a captured launch keeps it.
struct Entry {
  void *weight;
  const void *gradient;
  int64_t count, offset;
  double weight_decay;
  int32_t kind;   // weight's type + 4 x gradient's, + 16 x (both on 16-byte boundaries)
  int32_t first;  // its first CTA
};

template <int N>
struct Table {
  Entry entry[N];
  int32_t tensors;
};

struct Moments {
  void *first, *second;
  uint8_t *first_exponent, *second_exponent;
  const State *state;
  float b1, b1c, b2, b2c, eps;
  bool stochastic;
};

// The entry whose CTAs hold `cta`: entries without CTAs are left out of the
// table, so firsts ascend.
template <int N>
__device__ __forceinline__ int find(const Table<N> &t, int cta) {
  int lo = 0, hi = t.tensors;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (t.entry[mid].first <= cta)
      lo = mid;
    else
      hi = mid;
  }
  return lo;
}

template <typename T>
__device__ __forceinline__ float to_f(T v) {
  if constexpr (std::is_same_v<T, float>) return v;
  if constexpr (std::is_same_v<T, __nv_bfloat16>) return __bfloat162float(v);
  if constexpr (std::is_same_v<T, __half>) return __half2float(v);
}

template <typename T, int W>
struct alignas(sizeof(T) * W > 16 ? 16 : sizeof(T) * W) Vec {
  T v[W];
};

// W elements at x[i], zero past `count`
template <typename T, int W>
__device__ __forceinline__ void load(const T *x, int64_t i, int64_t count, bool whole, float (&f)[W]) {
  if (whole) {
    const Vec<T, W> p = *reinterpret_cast<const Vec<T, W> *>(x + i);
#pragma unroll
    for (int w = 0; w < W; ++w) f[w] = to_f(p.v[w]);
  } else {
#pragma unroll
    for (int w = 0; w < W; ++w) f[w] = i + w < count ? to_f(x[i + w]) : 0.0f;
  }
}

// A weight's type: float32 as it is, bfloat16 to nearest or by random bits
template <typename T>
__device__ __forceinline__ T to_weight(float w, bool stochastic, uint32_t random) {
  if constexpr (std::is_same_v<T, float>) {
    return w;
  } else {
    if (!stochastic || w != w) return __float2bfloat16_rn(w);
    return __ushort_as_bfloat16((unsigned short)((__float_as_uint(w) + (random * 0x85ebu & 0xffffu)) >> 16));
  }
}

template <typename T, int W>
__device__ __forceinline__ void store(T *x, int64_t i, int64_t count, bool whole, const Vec<T, W> &p) {
  if (whole) {
    *reinterpret_cast<Vec<T, W> *>(x + i) = p;
  } else {
#pragma unroll
    for (int w = 0; w < W; ++w)
      if (i + w < count) x[i + w] = p.v[w];
  }
}

__device__ __forceinline__ float power_of_two(int field) { return __int_as_float(field << 23); }

// Sixteen random bits of each of four elements, of which the first has index
// 4 q among the moments
__device__ __forceinline__ void random4(const State &s, int64_t q, uint32_t (&r)[4]) {
  const sk_key k = sk_threefry(sk_key{s.key0, s.key1}, (uint32_t)(q >> 32), (uint32_t)q);
  r[0] = k.k0 & 0xffffu;
  r[1] = k.k0 >> 16;
  r[2] = k.k1 & 0xffffu;
  r[3] = k.k1 >> 16;
}

struct Element {
  float m, v, root;
};

__device__ __forceinline__ Element moments_of(const Moments &p, float clip, float g, float m, float v) {
  Element e;
  g = g * clip;
  e.m = m * p.b1 + g * p.b1c;
  e.v = v * p.b2 + g * g * p.b2c;
  e.root = sqrtf(e.v);
  return e;
}

__device__ __forceinline__ float weight_of(const Moments &p, const State &s, float decay, float w, const Element &e) {
  return w * decay - __fdividef(s.size * e.m, e.root * s.inv_root + p.eps);
}

// Moments of 32 bits: four elements of each array a thread and pass.
template <typename PT, typename GT>
__device__ __forceinline__ void step32(const Moments &p, const Entry &e, const State &s, int chunk) {
  constexpr int W = 4, kPasses = kChunk / (kThreads * W);
  float *first = static_cast<float *>(p.first) + e.offset, *second = static_cast<float *>(p.second) + e.offset;
  PT *weight = static_cast<PT *>(e.weight);
  const GT *gradient = static_cast<const GT *>(e.gradient);
  const bool aligned = e.kind & 16;
  const float decay = (float)(1.0 - s.learning_rate * e.weight_decay);
  if (s.skip) return;
#pragma unroll 2
  for (int pass = 0; pass < kPasses; ++pass) {
    const int64_t i = (int64_t)chunk * kChunk + (pass * kThreads + (int)threadIdx.x) * W;
    if (i >= e.count) continue;
    const bool whole = aligned && i + W <= e.count;
    float g[W], w[W];
    load<GT, W>(gradient, i, e.count, whole, g);
    load<PT, W>(weight, i, e.count, whole, w);
    Vec<float, W> m = *reinterpret_cast<const Vec<float, W> *>(first + i);
    Vec<float, W> v = *reinterpret_cast<const Vec<float, W> *>(second + i);
    uint32_t random[W] = {};
    if constexpr (!std::is_same_v<PT, float>)
      if (p.stochastic) random4(s, (e.offset + i) >> 2, random);
    Vec<PT, W> out;
#pragma unroll
    for (int j = 0; j < W; ++j) {
      const Element x = moments_of(p, s.clip, g[j], m.v[j], v.v[j]);
      m.v[j] = x.m;
      v.v[j] = x.v;
      out.v[j] = to_weight<PT>(weight_of(p, s, decay, w[j], x), p.stochastic, random[j]);
    }
    *reinterpret_cast<Vec<float, W> *>(first + i) = m;
    *reinterpret_cast<Vec<float, W> *>(second + i) = v;
    store<PT, W>(weight, i, e.count, whole, out);
  }
}

// 2^(field - 127), NaN where a block holds what is not finite
__device__ __forceinline__ float block_scale(uint32_t field) {
  return __uint_as_float(field == 255u ? 0x7fc00000u : field << 23);
}
__device__ __forceinline__ float decode_first(uint32_t code, float scale) {
  return __uint_as_float(((code & 0x7fu) << 20) | ((code & 0x80u) << 24)) * 0x1p113f * scale;
}
__device__ __forceinline__ float decode_root(uint32_t code, float scale) {
  return __uint_as_float(code << 19) * 0x1p113f * scale;
}

// The exponent field of a block from the bits of its largest element, of
// which every lane of the warp has its own largest: what is below 2^-100
// rounds on the grid of 2^-100 (it stays exact in bfloat16), above 2^126
// the largest codes hold it
__device__ __forceinline__ uint32_t block_field(uint32_t bits) {
  bits = __reduce_max_sync(kFull, bits);
  return bits >= 0x7f800000u ? 255u : min(max(bits >> 23, 27u), 253u);
}

// Moments of 8 bits: a warp takes a block of 256, eight elements a lane.
template <typename PT, typename GT>
__device__ __forceinline__ void step8(const Moments &p, const Entry &e, const State &s, int chunk) {
  constexpr int W = 8, kWarps = kThreads / 32, kPasses = kChunk / (kWarps * kBlock);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  PT *weight = static_cast<PT *>(e.weight);
  const GT *gradient = static_cast<const GT *>(e.gradient);
  const bool aligned = e.kind & 16;
  const float decay = (float)(1.0 - s.learning_rate * e.weight_decay);
  if (s.skip) return;
#pragma unroll 1
  for (int pass = 0; pass < kPasses; ++pass) {
    const int64_t start = (int64_t)chunk * kChunk + (pass * kWarps + warp) * kBlock;
    if (start >= e.count) break;
    const int64_t i = start + lane * W, block = (e.offset + start) / kBlock;
    const bool whole = aligned && i + W <= e.count;
    float g[W], w[W];
    load<GT, W>(gradient, i, e.count, whole, g);
    load<PT, W>(weight, i, e.count, whole, w);
    uint2 *first = reinterpret_cast<uint2 *>(static_cast<uint8_t *>(p.first) + e.offset + i);
    uint2 *second = reinterpret_cast<uint2 *>(static_cast<uint8_t *>(p.second) + e.offset + i);
    const uint2 mc = *first, rc = *second;
    const float m_scale = block_scale(p.first_exponent[block]), r_scale = block_scale(p.second_exponent[block]);
    uint32_t random[W];
    random4(s, (e.offset + i) >> 2, *reinterpret_cast<uint32_t(*)[4]>(random));
    random4(s, ((e.offset + i) >> 2) + 1, *reinterpret_cast<uint32_t(*)[4]>(random + 4));
    float m[W], r[W];
    uint32_t m_most = 0, r_most = 0;
    Vec<PT, W> out;
#pragma unroll
    for (int j = 0; j < W; ++j) {
      const uint32_t mb = (j < 4 ? mc.x : mc.y) >> (8 * (j & 3)) & 0xffu;
      const uint32_t rb = (j < 4 ? rc.x : rc.y) >> (8 * (j & 3)) & 0xffu;
      const float root = decode_root(rb, r_scale);
      const Element x = moments_of(p, s.clip, g[j], decode_first(mb, m_scale), root * root);
      m[j] = x.m;
      r[j] = x.root;
      m_most = max(m_most, __float_as_uint(x.m) & 0x7fffffffu);
      r_most = max(r_most, __float_as_uint(x.root) & 0x7fffffffu);
      out.v[j] = to_weight<PT>(weight_of(p, s, decay, w[j], x), p.stochastic, random[j]);
    }
    store<PT, W>(weight, i, e.count, whole, out);
    const uint32_t m_field = block_field(m_most), r_field = block_field(r_most);
    // 2^-e, then 2^-113: one factor would leave the range of floats
    const float m_down = power_of_two(254 - (int)min(m_field, 253u)), r_down = power_of_two(254 - (int)min(r_field, 253u));
    uint2 mo = {0, 0}, ro = {0, 0};
#pragma unroll
    for (int j = 0; j < W; ++j) {
      const float y = fabsf(m[j]) * m_down * 0x1p-113f, z = r[j] * r_down * 0x1p-113f;
      uint32_t mb = (__float_as_uint(y) + (random[j] << 4) + 8u) >> 20;
      uint32_t rb = (__float_as_uint(z) + ((random[j] * 0x9e37u & 0xffffu) << 3) + 4u) >> 19;
      mb = min(mb, 0x7eu) | (__float_as_uint(m[j]) >> 24 & 0x80u);
      rb = min(max(rb, r[j] > 0.0f ? 1u : 0u), 0xffu);
      (j < 4 ? mo.x : mo.y) |= mb << (8 * (j & 3));
      (j < 4 ? ro.x : ro.y) |= rb << (8 * (j & 3));
    }
    *first = mo;
    *second = ro;
    if (lane == 0) {
      p.first_exponent[block] = (uint8_t)m_field;
      p.second_exponent[block] = (uint8_t)r_field;
    }
  }
}

template <int Bits, typename PT, typename GT>
__device__ __forceinline__ void step_chunk(const Moments &p, const Entry &e, const State &s, int chunk) {
  if constexpr (Bits == 32)
    step32<PT, GT>(p, e, s, chunk);
  else
    step8<PT, GT>(p, e, s, chunk);
}

template <int Bits, int N>
__global__ void __launch_bounds__(kThreads) adamw_kernel(const __grid_constant__ Table<N> table,
                                                         const __grid_constant__ Moments p) {
  const Entry &e = table.entry[find(table, blockIdx.x)];
  const int chunk = blockIdx.x - e.first;
  const State s = *p.state;
  switch (e.kind & 15) {
    case 0: return step_chunk<Bits, float, float>(p, e, s, chunk);
    case 4: return step_chunk<Bits, float, __nv_bfloat16>(p, e, s, chunk);
    case 8: return step_chunk<Bits, float, __half>(p, e, s, chunk);
    case 1: return step_chunk<Bits, __nv_bfloat16, float>(p, e, s, chunk);
    case 5: return step_chunk<Bits, __nv_bfloat16, __nv_bfloat16>(p, e, s, chunk);
    case 9: return step_chunk<Bits, __nv_bfloat16, __half>(p, e, s, chunk);
  }
}

// A step's scalars.  A norm that is not finite skips the step: nothing is
// written and the count stays.
struct Begin {
  State *state;
  const float *norm, *learning_rate;
  double rate, log_b1, log_b2, max_norm;
  uint32_t key0, key1;
};
__global__ void adamw_begin_kernel(const Begin p) {
  State s = *p.state;
  s.clip = 1.0f;
  s.skip = 0;
  if (p.norm) {
    const float norm = *p.norm;
    s.skip = !isfinite(norm);
    s.clip = (float)(p.max_norm / fmax((double)norm, p.max_norm));
  }
  s.learning_rate = p.learning_rate ? (double)*p.learning_rate : p.rate;
  if (!s.skip) s.step += 1;
  const double t = (double)s.step;
  s.size = (float)(s.learning_rate / -expm1(t * p.log_b1));
  s.inv_root = (float)(1.0 / sqrt(-expm1(t * p.log_b2)));
  const sk_key k = sk_fold_in(sk_key{p.key0, p.key1}, (uint32_t)s.step);
  s.key0 = k.k0;
  s.key1 = k.k1;
  *p.state = s;
}

// The values of 8-bit moments, exact in bfloat16: eight a thread
__global__ void __launch_bounds__(kThreads) adamw_moments_kernel(const uint8_t *first, const uint8_t *second,
                                                                 const uint8_t *first_exponent,
                                                                 const uint8_t *second_exponent, int64_t count,
                                                                 __nv_bfloat16 *first_out, __nv_bfloat16 *root_out) {
  const int64_t i = ((int64_t)blockIdx.x * kThreads + threadIdx.x) * 8;
  if (i >= count) return;
  const uint2 mc = *reinterpret_cast<const uint2 *>(first + i), rc = *reinterpret_cast<const uint2 *>(second + i);
  const float m_scale = block_scale(first_exponent[i / kBlock]), r_scale = block_scale(second_exponent[i / kBlock]);
  Vec<__nv_bfloat16, 8> m, r;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const uint32_t mb = (j < 4 ? mc.x : mc.y) >> (8 * (j & 3)) & 0xffu;
    const uint32_t rb = (j < 4 ? rc.x : rc.y) >> (8 * (j & 3)) & 0xffu;
    m.v[j] = __float2bfloat16_rn(decode_first(mb, m_scale));
    r.v[j] = __float2bfloat16_rn(decode_root(rb, r_scale));
  }
  *reinterpret_cast<Vec<__nv_bfloat16, 8> *>(first_out + i) = m;
  *reinterpret_cast<Vec<__nv_bfloat16, 8> *>(root_out + i) = r;
}

// ---------------------------------------------------------------------------
// the norm
// ---------------------------------------------------------------------------

// every thread ends with the CTA's sum, added in a fixed order
__device__ __forceinline__ double cta_sum(double v) {
  __shared__ double warps[kThreads / 32];
#pragma unroll
  for (int off = 16; off; off >>= 1) v += __shfl_xor_sync(kFull, v, off);
  if ((threadIdx.x & 31) == 0) warps[threadIdx.x >> 5] = v;
  __syncthreads();
  double sum = 0.0;
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w) sum += warps[w];
  return sum;
}

// Squares are exact in 64 bits and so is nearly their sum: neither a
// gradient of 1e20 nor one of 1e-25 is lost, and the factor that clips does
// not depend on the launch's shape.
template <typename T>
__device__ __forceinline__ double squares(const Entry &e, int64_t begin) {
  constexpr int W = 16 / sizeof(T), kAhead = 4;  // vectors of a thread in flight together
  const T *x = static_cast<const T *>(e.gradient);
  const int64_t end = min(e.count, begin + kNormChunk);
  double sum = 0.0;
  if (e.kind & 16) {
    for (int64_t i = begin + (int)threadIdx.x * W; i < end; i += kAhead * kThreads * W) {
      float f[kAhead][W];
#pragma unroll
      for (int k = 0; k < kAhead; ++k) {
        const int64_t at = i + k * kThreads * W;
        if (at < end)
          load<T, W>(x, at, e.count, at + W <= e.count, f[k]);
        else
#pragma unroll
          for (int w = 0; w < W; ++w) f[k][w] = 0.0f;
      }
#pragma unroll
      for (int k = 0; k < kAhead; ++k)
#pragma unroll
        for (int w = 0; w < W; ++w) sum = fma((double)f[k][w], (double)f[k][w], sum);
    }
  } else {
#pragma unroll 4
    for (int64_t i = begin + threadIdx.x; i < end; i += kThreads) {
      const double f = (double)to_f(x[i]);
      sum = fma(f, f, sum);
    }
  }
  return sum;
}

constexpr int kNormCtas = 6;  // of an SM
template <int N>
__global__ void __launch_bounds__(kThreads, kNormCtas) norm_kernel(const __grid_constant__ Table<N> table, int chunks,
                                                                   double *partial) {
  double sum = 0.0;
  for (int chunk = blockIdx.x; chunk < chunks; chunk += gridDim.x) {
    const Entry &e = table.entry[find(table, chunk)];
    const int64_t begin = (int64_t)(chunk - e.first) * kNormChunk;
    switch (e.kind >> 2 & 3) {
      case 0: sum += squares<float>(e, begin); break;
      case 1: sum += squares<__nv_bfloat16>(e, begin); break;
      default: sum += squares<__half>(e, begin); break;
    }
  }
  sum = cta_sum(sum);
  if (threadIdx.x == 0) partial[blockIdx.x] = sum;
}

__global__ void __launch_bounds__(kThreads) norm_finish_kernel(const double *partial, int count, float *norm) {
  double sum = 0.0;
  for (int i = threadIdx.x; i < count; i += kThreads) sum += partial[i];
  sum = cta_sum(sum);
  if (threadIdx.x == 0) *norm = (float)sqrt(sum);
}

// ---------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------

bool misaligned(const void *q, size_t a) { return (reinterpret_cast<uintptr_t>(q) & (a - 1)) != 0; }
size_t size_of(int dtype) { return dtype == 0 ? 4 : 2; }

struct Span {
  uintptr_t begin, end;
};
Span span(const void *q, uint64_t bytes) {
  return Span{reinterpret_cast<uintptr_t>(q), reinterpret_cast<uintptr_t>(q) + bytes};
}

// Whether two of `own` meet, or one of `read` meets one of `own`
bool overlap(std::vector<Span> &own, const std::vector<Span> &read) {
  std::sort(own.begin(), own.end(), [](const Span &a, const Span &b) { return a.begin < b.begin; });
  for (size_t i = 1; i < own.size(); ++i)
    if (own[i].begin < own[i - 1].end) return true;
  for (const Span &r : read) {
    auto it = std::lower_bound(own.begin(), own.end(), r.end, [](const Span &a, uintptr_t v) { return a.begin < v; });
    if (it != own.begin() && (it - 1)->end > r.begin) return true;
  }
  return false;
}

// The tensors that hold anything, each with its first chunk of `size`
// elements
struct Chunked {
  std::vector<Entry> entries;
  std::vector<int64_t> chunks;
};
bool chunked(const scacchi_adamw_tensor *tensors, int32_t n, int64_t size, Chunked &out) {
  for (int32_t i = 0; i < n; ++i) {
    const scacchi_adamw_tensor &t = tensors[i];
    if (t.count == 0 || !t.gradient) continue;
    const bool aligned = !misaligned(t.weight, 16) && !misaligned(t.gradient, 16);
    const int64_t chunks = (t.count + size - 1) / size;
    if (chunks > (int64_t)1 << 30) return false;
    out.entries.push_back(Entry{t.weight, t.gradient, t.count, t.offset, t.weight_decay,
                                t.weight_dtype + 4 * t.gradient_dtype + (aligned ? 16 : 0), 0});
    out.chunks.push_back(chunks);
  }
  return true;
}

// As many entries as a launch's table and grid take, from `at` on; their
// chunks, or 0 at the end
template <int N>
int fill(Table<N> &table, const Chunked &all, size_t &at) {
  int64_t total = 0;
  table.tensors = 0;
  while (at < all.entries.size() && table.tensors < N && total + all.chunks[at] <= ((int64_t)1 << 30)) {
    Entry &e = table.entry[table.tensors++];
    e = all.entries[at];
    e.first = (int32_t)total;
    total += all.chunks[at++];
  }
  return (int)total;
}

cudaError_t launched() {
  g_adamw_launches.fetch_add(1, std::memory_order_relaxed);
  return cudaGetLastError();
}

template <int Bits, int N>
cudaError_t launch_step(const Chunked &all, const Moments &p, cudaStream_t st) {
  static thread_local Table<N> table;
  size_t at = 0;
  while (const int chunks = fill(table, all, at)) {
    adamw_kernel<Bits, N><<<chunks, kThreads, 0, st>>>(table, p);
    if (cudaError_t e = launched()) return e;
  }
  return cudaSuccess;
}

template <int N>
cudaError_t launch_norm(const Chunked &all, double *partial, int *partials, cudaStream_t st) {
  static thread_local Table<N> table;
  size_t at = 0;
  while (const int chunks = fill(table, all, at)) {
    const int ctas = std::min(chunks, kMaxPartials);
    norm_kernel<N><<<ctas, kThreads, 0, st>>>(table, chunks, partial + *partials);
    if (cudaError_t e = launched()) return e;
    *partials += ctas;
  }
  return cudaSuccess;
}

// Tables of a size near what is needed: a launch copies its parameters
constexpr int kTables[] = {16, 80, 512};

}  // namespace

extern "C" {

size_t scacchi_gradient_norm_workspace_bytes(int32_t tensors) {
  if (tensors < 0) return 0;
  return ((size_t)tensors / kTables[2] + 1) * kMaxPartials * sizeof(double);
}

int scacchi_gradient_norm(const scacchi_adamw_tensor *tensors, int32_t num_tensors, float *norm, void *workspace,
                          void *stream) {
  if (num_tensors < 0 || (num_tensors && !tensors) || !norm || misaligned(norm, 4) || !workspace ||
      misaligned(workspace, 8))
    return SCACCHI_EINVAL;
  for (int32_t i = 0; i < num_tensors; ++i) {
    const scacchi_adamw_tensor &t = tensors[i];
    if (t.count < 0 || t.gradient_dtype < 0 || t.gradient_dtype > kMaxDtype || (t.count && !t.gradient) ||
        misaligned(t.gradient, size_of(t.gradient_dtype)))
      return SCACCHI_EINVAL;
  }
  try {
    Chunked all;
    if (!chunked(tensors, num_tensors, kNormChunk, all)) return SCACCHI_EINVAL;
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    double *partial = static_cast<double *>(workspace);
    int partials = 0;
    const size_t n = all.entries.size();
    cudaError_t e = n <= kTables[0]   ? launch_norm<kTables[0]>(all, partial, &partials, st)
                    : n <= kTables[1] ? launch_norm<kTables[1]>(all, partial, &partials, st)
                                      : launch_norm<kTables[2]>(all, partial, &partials, st);
    if (e != cudaSuccess) return SCACCHI_ECUDA;
    norm_finish_kernel<<<1, kThreads, 0, st>>>(partial, partials, norm);
    return launched() == cudaSuccess ? SCACCHI_OK : SCACCHI_ECUDA;
  } catch (...) {
    return SCACCHI_ECUDA;
  }
}

int scacchi_adamw_step(const scacchi_adamw *params, const scacchi_adamw_tensor *tensors, int32_t num_tensors,
                       void *stream) {
  if (!params || num_tensors < 0 || (num_tensors && !tensors)) return SCACCHI_EINVAL;
  const scacchi_adamw &a = *params;
  const bool eight = a.state_bits == 8;
  if ((a.state_bits != 32 && !eight) || !(a.beta1 >= 0.0 && a.beta1 < 1.0) || !(a.beta2 >= 0.0 && a.beta2 < 1.0) ||
      !(a.eps >= 0.0f && a.eps <= 1e30f) || !isfinite(a.learning_rate) || a.moments < 0 || a.moments % kBlock ||
      !a.state || misaligned(a.state, 8) || misaligned(a.norm, 4) || misaligned(a.learning_rate_at, 4) ||
      (a.norm && !(a.max_norm > 0.0 && isfinite(a.max_norm))) || (eight && !a.stochastic))
    return SCACCHI_EINVAL;
  if (a.moments && (!a.first || !a.second || misaligned(a.first, 16) || misaligned(a.second, 16) ||
                    (eight && (!a.first_exponent || !a.second_exponent))))
    return SCACCHI_EINVAL;
  try {
    std::vector<Span> own, read;
    int64_t next = 0;
    for (int32_t i = 0; i < num_tensors; ++i) {
      const scacchi_adamw_tensor &t = tensors[i];
      if (t.weight_dtype < 0 || t.weight_dtype > 1 || t.gradient_dtype < 0 || t.gradient_dtype > kMaxDtype ||
          t.count < 0 || t.offset % kBlock || t.offset < next || t.count > a.moments || t.offset > a.moments - t.count ||
          !isfinite(t.weight_decay) || (t.count && !t.weight) || misaligned(t.weight, size_of(t.weight_dtype)) ||
          misaligned(t.gradient, size_of(t.gradient_dtype)))
        return SCACCHI_EINVAL;
      next = t.offset + t.count;
      if (!t.count) continue;
      own.push_back(span(t.weight, t.count * size_of(t.weight_dtype)));
      if (t.gradient) read.push_back(span(t.gradient, t.count * size_of(t.gradient_dtype)));
    }
    if (a.moments) {
      const uint64_t size = eight ? 1 : 4;
      own.push_back(span(a.first, a.moments * size));
      own.push_back(span(a.second, a.moments * size));
      if (eight) {
        own.push_back(span(a.first_exponent, a.moments / kBlock));
        own.push_back(span(a.second_exponent, a.moments / kBlock));
      }
    }
    own.push_back(span(a.state, SCACCHI_ADAMW_STATE_BYTES));
    if (a.norm) read.push_back(span(a.norm, 4));
    if (a.learning_rate_at) read.push_back(span(a.learning_rate_at, 4));
    Chunked all;
    if (overlap(own, read) || !chunked(tensors, num_tensors, kChunk, all)) return SCACCHI_EINVAL;
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    State *state = static_cast<State *>(a.state);
    adamw_begin_kernel<<<1, 1, 0, st>>>(Begin{state, a.norm, a.learning_rate_at, a.learning_rate, log(a.beta1),
                                              log(a.beta2), a.max_norm, a.key0, a.key1});
    if (launched() != cudaSuccess) return SCACCHI_ECUDA;
    const Moments p = {a.first, a.second, a.first_exponent, a.second_exponent, state, (float)a.beta1,
                       (float)(1.0 - a.beta1), (float)a.beta2, (float)(1.0 - a.beta2), a.eps, a.stochastic != 0};
    const size_t n = all.entries.size();
    cudaError_t e;
    if (eight)
      e = n <= kTables[0]   ? launch_step<8, kTables[0]>(all, p, st)
          : n <= kTables[1] ? launch_step<8, kTables[1]>(all, p, st)
                            : launch_step<8, kTables[2]>(all, p, st);
    else
      e = n <= kTables[0]   ? launch_step<32, kTables[0]>(all, p, st)
          : n <= kTables[1] ? launch_step<32, kTables[1]>(all, p, st)
                            : launch_step<32, kTables[2]>(all, p, st);
    return e == cudaSuccess ? SCACCHI_OK : SCACCHI_ECUDA;
  } catch (...) {
    return SCACCHI_ECUDA;
  }
}

int scacchi_adamw_moments(const uint8_t *first, const uint8_t *second, const uint8_t *first_exponent,
                          const uint8_t *second_exponent, int64_t moments, void *first_out, void *root_out,
                          void *stream) {
  if (moments < 0 || moments % kBlock) return SCACCHI_EINVAL;
  if (moments == 0) return SCACCHI_OK;
  if (!first || !second || !first_exponent || !second_exponent || !first_out || !root_out || misaligned(first, 16) ||
      misaligned(second, 16) || misaligned(first_out, 16) || misaligned(root_out, 16))
    return SCACCHI_EINVAL;
  const int64_t ctas = (moments + kThreads * 8 - 1) / (kThreads * 8);
  if (ctas > 0x7fffffff) return SCACCHI_EINVAL;
  adamw_moments_kernel<<<(unsigned)ctas, kThreads, 0, static_cast<cudaStream_t>(stream)>>>(
      first, second, first_exponent, second_exponent, moments, static_cast<__nv_bfloat16 *>(first_out),
      static_cast<__nv_bfloat16 *>(root_out));
  return launched() == cudaSuccess ? SCACCHI_OK : SCACCHI_ECUDA;
}

uint64_t scacchi_adamw_launch_count(void) { return g_adamw_launches.load(std::memory_order_relaxed); }

}  // extern "C"
