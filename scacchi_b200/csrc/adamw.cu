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
//
// Device times, by graph replays: 50.4 M float32 weights and gradients with
// 32-bit moments 212 us (6.7 TB/s, the copy's rate); 67.1 M bfloat16 weights and
// gradients with moments of 8 bits 228 us (2.9 TB/s; 104 us at a copy's rate),
// with float32 weights 206 us (4.6 TB/s); reading 8-bit moments out 62 us
// (6.5 TB/s).  The norm of 67.1 M bfloat16 gradients 28 us (4.7 TB/s), of 50.4 M
// float32 33 us (6.1 TB/s), off their 16-byte boundaries 39 us and (67.1 M) 45;
// 66 small tensors 6 us.
//
// 32-bit moments are bound by memory.  Those of 8 bits are bound by the
// instructions of this implementation, 101 an element (94 with float32 weights)
// on 80 % of the cycles, the pipe of logic and additions 69 % busy: 19 are the
// random bits', which the definition asks for, the rest decoding, roots, quotients
// and encoding, of which nothing says that it takes so many.

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
// Elements of a tensor that a CTA takes.  Longer chunks put the CTAs of a
// moment further apart in memory, and powers of two meet the same channels: a
// step of 67.1 M bfloat16 weights with 8-bit moments 215 us with 4096, 237 with
// 2048, 299 with 8192, 267 with 16384.
constexpr int kChunk = 4096;
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

// Four elements as they lie in memory.  A tensor's whole vectors are loaded and
// stored at once; what stands off a 16-byte boundary or at the tensor's end
// goes element by element.  Nothing is converted on either way, so that a
// thread's loads are all on their way before it waits for the first.
template <typename T>
using Four = std::conditional_t<sizeof(T) == 4, uint4, uint2>;

template <typename T>
using Bits = std::conditional_t<sizeof(T) == 4, uint32_t, uint16_t>;
template <typename T>
__device__ __forceinline__ Four<T> load_slowly(const T *x, int64_t i, int64_t count) {
  const Bits<T> *from = reinterpret_cast<const Bits<T> *>(x) + i;
  const uint32_t a = i < count ? from[0] : 0, b = i + 1 < count ? from[1] : 0, c = i + 2 < count ? from[2] : 0,
                 d = i + 3 < count ? from[3] : 0;
  if constexpr (sizeof(T) == 4)
    return make_uint4(a, b, c, d);
  else
    return make_uint2(a | b << 16, c | d << 16);
}
template <typename T>
__device__ __forceinline__ void store_slowly(T *x, int64_t i, int64_t count, const Four<T> &q) {
  Bits<T> *to = reinterpret_cast<Bits<T> *>(x) + i;
  if constexpr (sizeof(T) == 4) {
    if (i < count) to[0] = q.x;
    if (i + 1 < count) to[1] = q.y;
    if (i + 2 < count) to[2] = q.z;
    if (i + 3 < count) to[3] = q.w;
  } else {
    if (i < count) to[0] = (uint16_t)q.x;
    if (i + 1 < count) to[1] = (uint16_t)(q.x >> 16);
    if (i + 2 < count) to[2] = (uint16_t)q.y;
    if (i + 3 < count) to[3] = (uint16_t)(q.y >> 16);
  }
}
template <typename T>
__device__ __forceinline__ float2 pair_of(Four<T> q, int pair) {
  if constexpr (sizeof(T) == 4) {
    return pair ? make_float2(__uint_as_float(q.z), __uint_as_float(q.w))
                : make_float2(__uint_as_float(q.x), __uint_as_float(q.y));
  } else {
    const uint32_t u = pair ? q.y : q.x;
    if constexpr (std::is_same_v<T, __half>) return __half22float2(*reinterpret_cast<const __half2 *>(&u));
    return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u));
  }
}

// one of the two sixteen bits of a word
__device__ __forceinline__ uint32_t half_of(uint32_t word, int i) { return i & 1 ? word >> 16 : word & 0xffffu; }

// A pair of weights as bfloat16: to nearest, or up where the random bits reach
// (the upper halves of sums; a NaN would run over)
__device__ __forceinline__ uint32_t to_pair(float a, float b, bool stochastic, uint32_t ra, uint32_t rb) {
  if (!stochastic || a != a || b != b) {
    const __nv_bfloat162 two = __floats2bfloat162_rn(a, b);
    if (!stochastic) return *reinterpret_cast<const uint32_t *>(&two);
    const uint32_t x = a != a ? 0x7fff0000u : __float_as_uint(a) + (ra * 0x85eb0000u >> 16);
    const uint32_t y = b != b ? 0x7fff0000u : __float_as_uint(b) + (rb * 0x85eb0000u >> 16);
    return __byte_perm(x, y, 0x7632);
  }
  return __byte_perm(__float_as_uint(a) + (ra * 0x85eb0000u >> 16), __float_as_uint(b) + (rb * 0x85eb0000u >> 16), 0x7632);
}
template <typename T>
__device__ __forceinline__ Four<T> to_weights(float2 a, float2 b, bool stochastic, uint2 random) {
  if constexpr (sizeof(T) == 4)
    return make_uint4(__float_as_uint(a.x), __float_as_uint(a.y), __float_as_uint(b.x), __float_as_uint(b.y));
  else
    return make_uint2(to_pair(a.x, a.y, stochastic, half_of(random.x, 0), half_of(random.x, 1)),
                      to_pair(b.x, b.y, stochastic, half_of(random.y, 0), half_of(random.y, 1)));
}

__device__ __forceinline__ float power_of_two(int field) { return __int_as_float(field << 23); }

// Sixteen random bits of each of four elements, two in a word, of which the
// first has index 4 q among the moments
__device__ __forceinline__ uint2 random4(const State &s, int64_t q) {
  const sk_key k = sk_threefry(sk_key{s.key0, s.key1}, (uint32_t)((uint64_t)q >> 32), (uint32_t)q);
  return make_uint2(k.k0, k.k1);
}

__device__ __forceinline__ float reciprocal(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float2 both(float x) { return make_float2(x, x); }
__device__ __forceinline__ float2 operator*(float2 a, float2 b) { return __fmul2_rn(a, b); }
// (one by one: the compiler fuses a pair's sum with the product before it, and codes would differ from the
// definition's here and there)
__device__ __forceinline__ float2 operator+(float2 a, float2 b) {
  return make_float2(__fadd_rn(a.x, b.x), __fadd_rn(a.y, b.y));
}

// m and v become the new moments, of which the root is returned
__device__ __forceinline__ float2 moments_of(const Moments &p, float clip, float2 g, float2 &m, float2 &v) {
  g = g * both(clip);
  m = m * both(p.b1) + g * both(p.b1c);
  v = v * both(p.b2) + g * g * both(p.b2c);
  return make_float2(sqrtf(v.x), sqrtf(v.y));
}
// The quotient takes one step of Newton's method from the approximate
// reciprocal, as exact as a division: bfloat16 weights round by random bits, and
// what 32 bits lose shows there as whole steps.  An infinite root (of a square
// beyond float32) has the reciprocal 0 and moves nothing; 1e37 in its place
// keeps the residual a number.  A root that is NaN makes the reciprocal NaN.
__device__ __forceinline__ float2 weights_of(const Moments &p, const State &s, float decay, float2 w, float2 m, float2 root) {
  float2 den = __ffma2_rn(root, both(s.inv_root), both(p.eps));
  const float2 r = make_float2(reciprocal(den.x), reciprocal(den.y));
  den = make_float2(fminf(den.x, 1e37f), fminf(den.y, 1e37f));
  const float2 update = m * both(-s.size);
  float2 q = update * r;
  q = __ffma2_rn(__ffma2_rn(make_float2(-den.x, -den.y), q, update), r, q);
  return __ffma2_rn(w, both(decay), q);
}

// Moments of 32 bits: four elements of each array a thread and pass.
template <typename PT, typename GT>
__device__ __forceinline__ void step32(const Moments &p, const Entry &e, const State &s, int chunk) {
  constexpr int W = 4;
  constexpr int kPasses = kChunk / (kThreads * W);
  PT *weight = static_cast<PT *>(e.weight);
  const GT *gradient = static_cast<const GT *>(e.gradient);
  float4 *first = reinterpret_cast<float4 *>(static_cast<float *>(p.first) + e.offset);
  float4 *second = reinterpret_cast<float4 *>(static_cast<float *>(p.second) + e.offset);
  const float decay = (float)(1.0 - s.learning_rate * e.weight_decay);
  if (s.skip) return;
#pragma unroll 2
  for (int pass = 0; pass < kPasses; ++pass) {
    const int64_t i = (int64_t)chunk * kChunk + (pass * kThreads + (int)threadIdx.x) * W;
    if (i >= e.count) continue;
    const bool whole = (e.kind & 16) && i + W <= e.count;
    Four<GT> g;
    Four<PT> w;
    if (whole) {
      g = *reinterpret_cast<const Four<GT> *>(gradient + i);
      w = *reinterpret_cast<const Four<PT> *>(weight + i);
    } else {
      g = load_slowly(gradient, i, e.count);
      w = load_slowly(weight, i, e.count);
    }
    const float4 mq = first[i / W], vq = second[i / W];
    uint2 random = {0, 0};
    if constexpr (!std::is_same_v<PT, float>)
      if (p.stochastic) random = random4(s, (e.offset + i) >> 2);
    float2 m[2] = {{mq.x, mq.y}, {mq.z, mq.w}}, v[2] = {{vq.x, vq.y}, {vq.z, vq.w}}, next[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const float2 root = moments_of(p, s.clip, pair_of<GT>(g, j), m[j], v[j]);
      next[j] = weights_of(p, s, decay, pair_of<PT>(w, j), m[j], root);
    }
    first[i / W] = make_float4(m[0].x, m[0].y, m[1].x, m[1].y);
    second[i / W] = make_float4(v[0].x, v[0].y, v[1].x, v[1].y);
    w = to_weights<PT>(next[0], next[1], p.stochastic, random);
    if (whole)
      *reinterpret_cast<Four<PT> *>(weight + i) = w;
    else
      store_slowly(weight, i, e.count, w);
  }
}

// 2^(field - 126), NaN where a block holds what is not finite
__device__ __forceinline__ float block_scale(uint32_t field) {
  return __uint_as_float(field == 255u ? 0x7fc00000u : (field + 1) << 23);
}
// Two of a word's four codes.  A code's fields are those of a float16 from its
// exponent's lowest bit on, and that float16 is half the code's value below
// the block's exponent.
__device__ __forceinline__ float2 decode_first(uint32_t codes, int pair) {
  const uint32_t up = __byte_perm(codes, 0u, pair ? 0x3424 : 0x1404);
  const uint32_t h = (up >> 1 & 0x3f803f80u) | (up & 0x80008000u);
  return __half22float2(*reinterpret_cast<const __half2 *>(&h));
}
__device__ __forceinline__ float2 decode_root(uint32_t codes, int pair) {
  const uint32_t h = __byte_perm(codes, 0u, pair ? 0x4342 : 0x4140) << 6;
  return __half22float2(*reinterpret_cast<const __half2 *>(&h));
}

// The exponent field of a block from its largest element, of which every lane
// of the warp has its own largest: what is below 2^-100 rounds on the grid of
// 2^-100 (it stays exact in bfloat16), above 2^126 the largest codes hold it
__device__ __forceinline__ uint32_t block_field(float most) {
  const uint32_t bits = __reduce_max_sync(kFull, __float_as_uint(most));
  return bits >= 0x7f800000u ? 255u : min(max(bits >> 23, 27u), 253u);
}
// the larger of a and |b|, |c|, NaN where any is
__device__ __forceinline__ float max_of(float a, float b, float c) {
  float y;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(fabsf(b)), "f"(fabsf(c)));
  return y;
}
// byte 3 of each
__device__ __forceinline__ uint32_t upper_bytes(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  return __byte_perm(__byte_perm(a, b, 0x0073), __byte_perm(c, d, 0x0073), 0x5410);
}
template <int Bytes>
__device__ __forceinline__ void copy_async(void *to, const void *from) {
  const uint32_t at = (uint32_t)__cvta_generic_to_shared(to);
  asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(at), "l"(from), "n"(Bytes) : "memory");
}

// A warp's block on its way from memory: a lane copies and reads its own places
// alone, four elements of either half
struct Staged {
  uint4 gradient[2][32], weight[2][32];
  uint32_t first[2][32], second[2][32];
};

// Moments of 8 bits: a warp takes block after block, the next one's data on
// their way while this one is computed.  Pairs of floats throughout.
template <typename PT, typename GT>
__device__ __forceinline__ void step8(const Moments &p, const Entry &e, const State &s, int chunk,
                                      Staged (*shared)[kThreads / 32]) {
  constexpr int W = 4, kWarps = kThreads / 32;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  PT *weight = static_cast<PT *>(e.weight);
  const GT *gradient = static_cast<const GT *>(e.gradient);
  const float decay = (float)(1.0 - s.learning_rate * e.weight_decay);
  if (s.skip) return;
  const int64_t begin = (int64_t)chunk * kChunk, end = min(e.count, begin + kChunk);
  uint32_t fields[2] = {0, 0};  // of the block ahead
  auto request = [&](int64_t start, int stage) {
    if (start < end) {
      Staged &to = shared[stage][warp];
      const uint32_t *first = reinterpret_cast<const uint32_t *>(static_cast<const uint8_t *>(p.first) + e.offset + start) + lane;
      const uint32_t *second = reinterpret_cast<const uint32_t *>(static_cast<const uint8_t *>(p.second) + e.offset + start) + lane;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int64_t i = start + h * (kBlock / 2) + lane * W;
        Four<GT> *g = reinterpret_cast<Four<GT> *>(&to.gradient[h][lane]);
        Four<PT> *w = reinterpret_cast<Four<PT> *>(&to.weight[h][lane]);
        if ((e.kind & 16) && start + kBlock <= e.count) {
          copy_async<sizeof(Four<GT>)>(g, gradient + i);
          copy_async<sizeof(Four<PT>)>(w, weight + i);
        } else {
          *g = load_slowly(gradient, i, e.count);
          *w = load_slowly(weight, i, e.count);
        }
        copy_async<4>(&to.first[h][lane], first + h * (kBlock / 8));
        copy_async<4>(&to.second[h][lane], second + h * (kBlock / 8));
      }
      fields[0] = p.first_exponent[(uint64_t)(e.offset + start) / kBlock];
      fields[1] = p.second_exponent[(uint64_t)(e.offset + start) / kBlock];
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  request(begin + warp * kBlock, 0);
  int stage = 0;
#pragma unroll 1
  for (int64_t start = begin + warp * kBlock; start < end; start += kWarps * kBlock, stage ^= 1) {
    const int64_t block = (uint64_t)(e.offset + start) / kBlock;
    const uint32_t m_old = fields[0], r_old = fields[1];
    request(start + kWarps * kBlock, stage ^ 1);
    uint32_t *first = reinterpret_cast<uint32_t *>(static_cast<uint8_t *>(p.first) + e.offset + start) + lane;
    uint32_t *second = reinterpret_cast<uint32_t *>(static_cast<uint8_t *>(p.second) + e.offset + start) + lane;
    const bool whole = (e.kind & 16) && start + kBlock <= e.count;
    const int64_t i = start + lane * W, other = i + kBlock / 2;
    // (while the loads are on their way)
    const uint2 random[2] = {random4(s, (e.offset + i) >> 2), random4(s, (e.offset + other) >> 2)};
    asm volatile("cp.async.wait_group 1;" ::: "memory");
    const Staged &now = shared[stage][warp];
    Four<PT> w[2];
    const float2 m_scale = both(block_scale(m_old)), r_scale = both(block_scale(r_old));
    float2 m[2][2], r[2][2];
    float m_most = 0.0f, r_most = 0.0f;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const Four<GT> g = *reinterpret_cast<const Four<GT> *>(&now.gradient[h][lane]);
      w[h] = *reinterpret_cast<const Four<PT> *>(&now.weight[h][lane]);
      const uint32_t mc = now.first[h][lane], rc = now.second[h][lane];
      float2 next[2];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const float2 r0 = decode_root(rc, j) * r_scale;
        float2 v = r0 * r0;
        m[h][j] = decode_first(mc, j) * m_scale;
        r[h][j] = moments_of(p, s.clip, pair_of<GT>(g, j), m[h][j], v);
        m_most = max_of(m_most, m[h][j].x, m[h][j].y);
        r_most = max_of(r_most, r[h][j].x, r[h][j].y);
        next[j] = weights_of(p, s, decay, pair_of<PT>(w[h], j), m[h][j], r[h][j]);
      }
      w[h] = to_weights<PT>(next[0], next[1], p.stochastic, random[h]);
    }
    if (whole) {
      *reinterpret_cast<Four<PT> *>(weight + i) = w[0];
      *reinterpret_cast<Four<PT> *>(weight + other) = w[1];
    } else {
      store_slowly(weight, i, e.count, w[0]);
      store_slowly(weight, other, e.count, w[1]);
    }
    const uint32_t m_field = block_field(m_most), r_field = block_field(r_most);
    if (m_field == 253u) {  // what is beyond the largest code takes it: a sum's carry would reach the sign
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        float2 &two = m[k / 2][k % 2];
        two = make_float2(fminf(fmaxf(two.x, -0x1.cp127f), 0x1.cp127f), fminf(fmaxf(two.y, -0x1.cp127f), 0x1.cp127f));
      }
    }
    // 2^-e, then 2^-113: one factor would leave the range of floats
    const float2 m_down = both(power_of_two(254 - (int)min(m_field, 253u)));
    const float2 r_down = both(power_of_two(254 - (int)min(r_field, 253u)));
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      // sums whose upper byte is the code, the random bits below it: 16 (bits + 16 u + 8), 32 (bits + 8 u' + 4)
      uint32_t mb[W], rb[W];
#pragma unroll
      for (int j = 0; j < W; ++j) {
        const float2 y = m[h][j / 2] * m_down * both(0x1p-113f), z = r[h][j / 2] * r_down * both(0x1p-113f);
        const uint32_t u = half_of(j < 2 ? random[h].x : random[h].y, j);
        const uint32_t yb = __float_as_uint(j & 1 ? y.y : y.x), zb = __float_as_uint(j & 1 ? z.y : z.x);
        mb[j] = (yb * 16u + (u * 256u + 128u)) | (yb & 0x80000000u);
        rb[j] = zb * 32u + ((u * 0x9e370000u + 0x8000u) >> 8);
      }
      const uint32_t mo = upper_bytes(mb[0], mb[1], mb[2], mb[3]);
      uint32_t ro = upper_bytes(rb[0], rb[1], rb[2], rb[3]);
      if ((ro - 0x01010101u) & ~ro & 0x80808080u) {  // a byte of zero: the borrow reaches its upper bit
#pragma unroll
        for (int j = 0; j < W; ++j)
          if ((j & 1 ? r[h][j / 2].y : r[h][j / 2].x) > 0.0f && !(ro >> (8 * j) & 0xffu)) ro |= 1u << (8 * j);
      }
      first[h * (kBlock / 8)] = mo;
      second[h * (kBlock / 8)] = ro;
    }
    if (lane == 0) {
      p.first_exponent[block] = (uint8_t)m_field;
      p.second_exponent[block] = (uint8_t)r_field;
    }
  }
}

template <int Bits, typename PT, typename GT>
__device__ __forceinline__ void step_chunk(const Moments &p, const Entry &e, const State &s, int chunk,
                                           Staged (*shared)[kThreads / 32]) {
  if constexpr (Bits == 32)
    step32<PT, GT>(p, e, s, chunk);
  else
    step8<PT, GT>(p, e, s, chunk, shared);
}

template <int Bits, int N>
__global__ void __launch_bounds__(kThreads, Bits == 8 ? 4 : 5) adamw_kernel(const __grid_constant__ Table<N> table,
                                                                           const __grid_constant__ Moments p) {
  __shared__ Staged shared[Bits == 8 ? 2 : 1][Bits == 8 ? kThreads / 32 : 1];
  Staged(*staged)[kThreads / 32] = reinterpret_cast<Staged(*)[kThreads / 32]>(&shared[0][0]);
  const Entry &e = table.entry[find(table, blockIdx.x)];
  const int chunk = blockIdx.x - e.first;
  const State s = *p.state;
  switch (e.kind & 15) {
    case 0: return step_chunk<Bits, float, float>(p, e, s, chunk, staged);
    case 4: return step_chunk<Bits, float, __nv_bfloat16>(p, e, s, chunk, staged);
    case 8: return step_chunk<Bits, float, __half>(p, e, s, chunk, staged);
    case 1: return step_chunk<Bits, __nv_bfloat16, float>(p, e, s, chunk, staged);
    case 5: return step_chunk<Bits, __nv_bfloat16, __nv_bfloat16>(p, e, s, chunk, staged);
    case 9: return step_chunk<Bits, __nv_bfloat16, __half>(p, e, s, chunk, staged);
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
  uint4 m, r;
  uint32_t *mw = reinterpret_cast<uint32_t *>(&m), *rw = reinterpret_cast<uint32_t *>(&r);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float2 a = decode_first(j < 2 ? mc.x : mc.y, j & 1) * both(m_scale);
    const float2 b = decode_root(j < 2 ? rc.x : rc.y, j & 1) * both(r_scale);
    // (exact: the lower halves are zero)
    mw[j] = __byte_perm(__float_as_uint(a.x), __float_as_uint(a.y), 0x7632);
    rw[j] = __byte_perm(__float_as_uint(b.x), __float_as_uint(b.y), 0x7632);
  }
  *reinterpret_cast<uint4 *>(first_out + i) = m;
  *reinterpret_cast<uint4 *>(root_out + i) = r;
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
__device__ __forceinline__ double square_of(uint32_t word, double sum) {
  if constexpr (std::is_same_v<T, float>) {
    const double f = (double)__uint_as_float(word);
    return fma(f, f, sum);
  } else {
    float2 two;
    if constexpr (std::is_same_v<T, __half>)
      two = __half22float2(*reinterpret_cast<const __half2 *>(&word));
    else
      two = make_float2(__uint_as_float(word << 16), __uint_as_float(word & 0xffff0000u));
    return fma((double)two.y, (double)two.y, fma((double)two.x, (double)two.x, sum));
  }
}
// 16 bytes of elements, one by one where they begin off a boundary
template <typename T>
__device__ __forceinline__ uint4 vector_of(const T *x, bool aligned) {
  if (aligned) return *reinterpret_cast<const uint4 *>(x);
  constexpr int64_t N = 16 / sizeof(T);
  if constexpr (sizeof(T) == 4) {
    return load_slowly(x, 0, N);
  } else {
    const uint2 low = load_slowly(x, 0, N), high = load_slowly(x + 4, 0, N);
    return make_uint4(low.x, low.y, high.x, high.y);
  }
}
// (each element goes to the same thread whatever the tensor's alignment: the
// order of the sum, and with it the norm's last bit, depends on sizes alone)
template <typename T, bool Aligned>
__device__ __forceinline__ double squares(const Entry &e, int64_t begin) {
  constexpr int W = 16 / sizeof(T), kAhead = 4;  // vectors of a thread in flight together
  const T *x = static_cast<const T *>(e.gradient) + begin;
  const int count = (int)min((int64_t)kNormChunk, e.count - begin), vectors = count / W;
  double sum = 0.0;
  for (int i = threadIdx.x; i < vectors; i += kAhead * kThreads) {
    uint4 q[kAhead];
#pragma unroll
    for (int k = 0; k < kAhead; ++k)
      q[k] = i + k * kThreads < vectors ? vector_of(x + (i + k * kThreads) * W, Aligned) : make_uint4(0, 0, 0, 0);
#pragma unroll
    for (int k = 0; k < kAhead; ++k)
      sum = square_of<T>(q[k].w, square_of<T>(q[k].z, square_of<T>(q[k].y, square_of<T>(q[k].x, sum))));
  }
#pragma unroll 1
  for (int i = vectors * W + (int)threadIdx.x; i < count; i += kThreads)
    sum = fma((double)to_f(x[i]), (double)to_f(x[i]), sum);
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
    if (e.kind & 16) {
      switch (e.kind >> 2 & 3) {
        case 0: sum += squares<float, true>(e, begin); break;
        case 1: sum += squares<__nv_bfloat16, true>(e, begin); break;
        default: sum += squares<__half, true>(e, begin); break;
      }
    } else {
      switch (e.kind >> 2 & 3) {
        case 0: sum += squares<float, false>(e, begin); break;
        case 1: sum += squares<__nv_bfloat16, false>(e, begin); break;
        default: sum += squares<__half, false>(e, begin); break;
      }
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

constexpr int64_t kMaxChunks = (int64_t)1 << 30;  // of a launch

// The tensors that hold anything, each with its number of chunks
struct Chunked {
  std::vector<Entry> entries;
  std::vector<int64_t> chunks;
};
// (`norm`: of gradients alone, weights are not looked at)
bool chunked(const scacchi_adamw_tensor *tensors, int32_t n, bool norm, Chunked &out) {
  const int64_t size = norm ? kNormChunk : kChunk;
  for (int32_t i = 0; i < n; ++i) {
    const scacchi_adamw_tensor &t = tensors[i];
    if (t.count == 0 || !t.gradient) continue;
    const bool aligned = (norm || !misaligned(t.weight, 16)) && !misaligned(t.gradient, 16);
    const int64_t chunks = (t.count - 1) / size + 1;
    if (chunks > kMaxChunks) return false;
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
  while (at < all.entries.size() && table.tensors < N && total + all.chunks[at] <= kMaxChunks) {
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
    if (!chunked(tensors, num_tensors, true, all)) return SCACCHI_EINVAL;
    // the workspace holds the partials of launches with full tables: gradients that are listed
    // again and again may fill a grid before its table
    int64_t total = 0;
    for (const int64_t chunks : all.chunks) total += chunks;
    if (total > kMaxChunks) return SCACCHI_EINVAL;
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
      !(a.eps == 0.0f || (a.eps >= 1e-30f && a.eps <= 1e30f)) || !isfinite(a.learning_rate) || a.moments < 0 || a.moments % kBlock ||
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
    if (overlap(own, read) || !chunked(tensors, num_tensors, false, all)) return SCACCHI_EINVAL;
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
