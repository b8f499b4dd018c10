// Clipped policy loss with a KL term, its per-row statistics and its
// gradient in the logits, for rows of `actions` logits.
//
// With keep = legal and x > -inf, m = max x, s = sum e^{x-m}, p = e^{x-m}/s
// over the kept actions, k the row's action, g its advantage and w its
// share of the loss:
//
//   log_prob  = x_k - m - log s,   ratio = e^{log_prob - old}
//   surrogate = -min(ratio g, clip(ratio, 1 - lo, 1 + hi) g)
//   sampled KL (reference log-prob q of the action):
//     e^y - 1 - y with y = q - log_prob;  d/dlog_prob = 1 - e^y
//   full KL (reference logits r): with d = x - r, mu = sum p d,
//     KL(p || softmax r) = log sum p e^{-(d-mu)} = log1p(sum p phi(mu-d)),
//     phi(y) = e^y - 1 - y >= 0;   dKL/dx_a = p_a (d_a - mu)
//   loss      = sum w (surrogate + beta KL)
//   dx_a      = w (c (delta_ak - p_a) + beta p_a (d_a - mu))
//   c         = (clipped ? 0 : -g ratio) + beta (1 - e^y)
//
// phi's form keeps the KL's leading digits when the two policies are near
// each other, where sum p (log p - log q) in 32 bits loses them.
//
// One pass over memory: short rows live in the registers of a few lanes,
// long ones in the shared memory of a CTA or of a cluster, so every input is
// read once and every output written once.  Row sums are held in 32 bits,
// the log-probability is finished in 64 from them and the loss is summed in
// 64.  A row whose ratio lies within kBorderTol (kShortBorderTol) of a clip
// border is evaluated again in 64 bits, so the side it falls on does not
// depend on 32-bit rounding.
//
// Device times, by graph replays: 262144 rows of 82 fp32 actions with the
// full KL 105 us (2.7 TB/s, 43 % of a copy's rate), with a sampled KL 62 us
// (3.2 TB/s); 4096 rows of 32000 bf16 137 us (3.8 TB/s), with the full KL 445
// us; 8 rows of 131071 fp32 24 us.
//
// What bounds it is not memory (30 to 41 % of DRAM's rate).  Short rows with
// the full KL issue 96 instructions an action on 58 % of the cycles: 128
// registers leave 16 warps an SM, which wait on their own results and on
// instruction fetch.  Long rows issue 23 an action without it on 67 %, with
// the exponentials' pipe at 52 % and shared memory at 47 %.  A few rows are
// latency: one row's phases across a cluster.
//
// Exponentials are ex2.approx of (x - m) log2 e: the difference first, in
// every pass, so that only |x - m|, which p weights, is rounded and scaled
// (a fused x log2 e - m log2 e loses digits as m grows); their errors
// (2^-22, and |x - m| 2^-23) average out over a row's sum.  The accurate
// expf() takes three times the instructions and made the kernel issue-bound.

#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include <atomic>
#include <type_traits>

#include "../../include/scacchi_b200.h"

namespace cg = cooperative_groups;

namespace {

std::atomic<uint64_t> g_policy_launches{0};

constexpr unsigned kFull = 0xffffffffu;
constexpr int kShortThreads = 256;
constexpr int kLongThreads = 256;
constexpr int kMaxWarps = 8;  // of a long row's CTA
static_assert(kLongThreads == 32 * kMaxWarps, "warps");
constexpr int kMaxCluster = 16;
constexpr int kMaxShort = 512;     // actions of a short row
constexpr int kMaxActions = 262144;
constexpr int kLongShared = 224 * 1024;  // of an SM, for the slices of its CTAs
constexpr int kMaxPartials = 148 * 16;
// What the 32-bit log-probability may be off by: terms within 2^-22 + 2.3 x
// 2^-24 |x - m| each (the difference, the product and log2 e), weighted by p
// (sum p |x - m| <= log of the actions, 11 for a slice of kLongShared / 2
// bytes: 1.8e-6); a thread's adds, at most 4 for eight elements and 28 of such
// sums (that slice over 256 threads), and the tree's (2.5e-6); and up to 28
// changes of a thread's maximum, 2^-22 of the sum each at worst (6.7e-6, in
// rows that ascend; 1e-6 was measured, and 3e-6 in all is what other rows
// stay below)
constexpr double kBorderTol = 1.1e-5;
// and of a short row: sum p |x - m| <= 6.3, 24 adds and the tree's, no changes
// of the maximum (2.9e-6).  (A row next to a border holds its warp up: 262144
// x 82 fp32 with a sampled KL 62 us at 8e-6, 64 at 1.1e-5)
constexpr double kShortBorderTol = 4e-6;
// Up to this many logits every row's log-probability is evaluated in 64 bits:
// the terms of a few rows may cancel to a loss that shows the 1e-7 of each.
// The host needs 25 us for a call, and the kernels stay below that: 64 x 82
// fp32 14 us (6 without), 8 x 131071 fp32 25 us (19 without).
constexpr int64_t kFineLogits = 1 << 20;
constexpr float kFarKl = 1.0e4f;   // sum p phi above this (KL > 9): the direct difference is exact enough
constexpr float kLowest = -1.0e30f;  // what is below is a mask's value where the row has any above
constexpr float kLog2E = 1.44269504088896341f;

struct Params {
  const void *logits, *reference;
  const uint8_t *legal;
  const int32_t *action;
  const float *old_log_prob, *advantage, *weight, *reference_log_prob;
  float *loss, *log_prob, *kl;
  uint8_t *clipped;
  void *grad;
  double *partial;
  int64_t rows, stride, reference_stride;
  int actions;
  int group;        // lanes of a short row
  int slice_bytes;  // of shared memory for a warp's batch, or a CTA's slice, of the logits
  int mask_bytes, x_pitch, r_pitch;  // of a warp's batch: Batch
  double clip_low, clip_high, log_low, log_high;  // borders of the ratio and their logarithms
  float beta, even_weight;
  bool fine;  // every row's log-probability in 64 bits
};

template <typename T>
__device__ __forceinline__ float to_f(T v);
template <>
__device__ __forceinline__ float to_f(float v) { return v; }
template <>
__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
template <>
__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
template <typename T>
__device__ __forceinline__ T from_f(float v);
template <>
__device__ __forceinline__ float from_f(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half from_f(float v) { return __float2half_rn(v); }

template <typename T, int W>
struct alignas(sizeof(T) * W) Vec {
  T v[W];
};

// a vector's elements as floats, and back; 16-bit ones two at a time
template <typename T, int W>
__device__ __forceinline__ void unpack(const Vec<T, W> &p, float (&f)[W]) {
#pragma unroll
  for (int w = 0; w < W; ++w) f[w] = to_f(p.v[w]);
}
template <int W>
__device__ __forceinline__ void unpack(const Vec<__nv_bfloat16, W> &p, float (&f)[W]) {
  if constexpr (W % 2 == 0) {
    const uint32_t *u = reinterpret_cast<const uint32_t *>(&p);
#pragma unroll
    for (int w = 0; w < W; w += 2) {
      f[w] = __uint_as_float(u[w / 2] << 16);
      f[w + 1] = __uint_as_float(u[w / 2] & 0xffff0000u);
    }
  } else {
#pragma unroll
    for (int w = 0; w < W; ++w) f[w] = to_f(p.v[w]);
  }
}
template <typename T, int W>
__device__ __forceinline__ Vec<T, W> pack(const float (&f)[W]) {
  Vec<T, W> p;
  if constexpr (sizeof(T) == 2 && W % 2 == 0) {
#pragma unroll
    for (int w = 0; w < W; w += 2) {
      if constexpr (std::is_same_v<T, __nv_bfloat16>)
        *reinterpret_cast<__nv_bfloat162 *>(p.v + w) = __floats2bfloat162_rn(f[w], f[w + 1]);
      else
        *reinterpret_cast<__half2 *>(p.v + w) = __floats2half2_rn(f[w], f[w + 1]);
    }
  } else {
#pragma unroll
    for (int w = 0; w < W; ++w) p.v[w] = from_f<T>(f[w]);
  }
  return p;
}

// e^y - 1 - y for |y| < 1 to 1.2e-7 of itself: y^2 times the Chebyshev
// interpolant of degree 6 of (e^y - 1 - y) / y^2 on [-1, 1]
__device__ __forceinline__ float phi_small(float y) {
  float c = 2.535864489e-05f;
  c = fmaf(c, y, 2.032920127e-04f);
  c = fmaf(c, y, 1.388539492e-03f);
  c = fmaf(c, y, 8.330884178e-03f);
  c = fmaf(c, y, 4.166673667e-02f);
  c = fmaf(c, y, 1.666669734e-01f);
  c = fmaf(c, y, 0.4999999978f);
  return c * (y * y);
}

__device__ __forceinline__ float exp2_fast(float t) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(t));
  return y;
}

// e^u for u <= 0 or small (see above)
__device__ __forceinline__ float exp_fast(float u) { return exp2_fast(u * kLog2E); }

// e^{x - top} of a vector's elements, the same bits: differences and
// products two at a time (4096 x 32000 bf16 137 us, 143 one at a time)
template <int W>
__device__ __forceinline__ void exps(const float (&x)[W], float top, float (&e)[W]) {
  if constexpr (W % 2 == 0) {
#pragma unroll
    for (int w = 0; w < W; w += 2) {
      const float2 u = __fmul2_rn(__fadd2_rn(make_float2(x[w], x[w + 1]), make_float2(-top, -top)),
                                  make_float2(kLog2E, kLog2E));
      e[w] = exp2_fast(u.x);
      e[w + 1] = exp2_fast(u.y);
    }
  } else {
#pragma unroll
    for (int w = 0; w < W; ++w) e[w] = exp_fast(x[w] - top);
  }
}

// log of a positive finite float to 1e-9: s = 2^k f with f in [1/sqrt 2,
// sqrt 2), log f = 2 atanh(q), q = (f - 1) / (f + 1), |q| < 0.172: the odd
// series to q^11 in 64 bits (next term 2e-11).  Zero, infinity and NaN go
// to log().
__device__ __forceinline__ double log_row_sum(float s) {
  if (!(s >= 1.17549435e-38f && s <= 3.4e38f)) return log((double)s);
  const int bits = __float_as_int(s);
  int k = (bits >> 23) - 127;
  float f = __int_as_float((bits & 0x007fffff) | 0x3f800000);
  if (f > 1.41421356f) {
    f *= 0.5f;
    k += 1;
  }
  const double den = (double)f + 1.0;
  double r = (double)__frcp_rn((float)den);
  r = r * (2.0 - den * r);
  const double q = ((double)f - 1.0) * r, q2 = q * q;
  double c = 1.0 / 11.0;
  c = fma(c, q2, 1.0 / 9.0);
  c = fma(c, q2, 1.0 / 7.0);
  c = fma(c, q2, 1.0 / 5.0);
  c = fma(c, q2, 1.0 / 3.0);
  c = fma(c, q2, 1.0);
  return fma(2.0 * q, c, (double)k * 0.693147180559945309417);
}

// e^u for u <= 0 to 1e-11 of itself, without a branch: u = k ln 2 + r, |r| <=
// ln 2 / 2, the exponential series to r^9 (next term 7e-12), and 2^k.  Below
// e^-700, and for minus infinity, 1e-304; NaN stays.
__device__ __forceinline__ double exp_64(double u) {
  u = u < -700.0 ? -700.0 : u;
  const double k = rint(u * 1.44269504088896340736), r = fma(k, -0.693147180559945309417, u), r2 = r * r;
  const double a = fma(r, 1.0 / 362880, 1.0 / 40320), b = fma(r, 1.0 / 5040, 1.0 / 720);
  const double c = fma(r, 1.0 / 120, 1.0 / 24), d = fma(r, 1.0 / 6, 0.5);
  const double p = fma(fma(fma(fma(a, r2, b), r2, c), r2, d), r2, 1.0 + r);
  return p * __hiloint2double((1023 + (int)k) << 20, 0);
}

// ---------------------------------------------------------------------------
// the threads of one row: some lanes of a warp, or the CTAs of a cluster
// ---------------------------------------------------------------------------

struct SumOp {
  template <typename U>
  __device__ static U apply(U a, U b) { return a + b; }
  template <typename U>
  __device__ static U none(U) { return U(0); }
};
struct MaxOp {
  template <typename U>
  __device__ static U apply(U a, U b) { return a > b ? a : b; }
  template <typename U>
  __device__ static U none(U) { return U(-INFINITY); }
};

// max, sum of e^{x - max} and of d e^{x - max}
struct alignas(16) Stats {
  float top, sum, mean;
};

__device__ __forceinline__ void rescale(Stats &v, float top) {
  const float f = v.top == -INFINITY ? 0.0f : exp_fast(v.top - top);
  v.sum *= f;
  v.mean *= f;
  v.top = top;
}

// every lane ends with the same bits: the butterfly adds the same pairs
struct Lanes {
  int lanes;
  unsigned mask;
  __device__ int index() const { return threadIdx.x & (lanes - 1); }
  __device__ int size() const { return lanes; }
  template <typename Op, typename U>
  __device__ U reduce(U v) const {
    for (int off = lanes >> 1; off; off >>= 1) v = Op::apply(v, __shfl_xor_sync(mask, v, off));
    return v;
  }
};

// Three levels of butterflies: a warp's lanes, the CTA's warps, the
// cluster's CTAs (each sends its own result to all).  Every thread ends with
// the same bits.
struct Ctas {
  Stats *slots;  // shared: two banks of kMaxWarps of the warps', two of kMaxCluster of the CTAs'
  int ctas, rank;
  mutable int bank;
  __device__ int index() const { return rank * blockDim.x + threadIdx.x; }
  __device__ int size() const { return ctas * blockDim.x; }

  template <typename U, typename Join>
  __device__ static U butterfly(U v, int width, Join join) {
    for (int off = width >> 1; off; off >>= 1) v = join(v, shuffle(v, off));
    return v;
  }
  __device__ static float shuffle(float v, int off) { return __shfl_xor_sync(kFull, v, off); }
  __device__ static double shuffle(double v, int off) { return __shfl_xor_sync(kFull, v, off); }
  __device__ static Stats shuffle(Stats v, int off) {
    return Stats{shuffle(v.top, off), shuffle(v.sum, off), shuffle(v.mean, off)};
  }
  // A bank is written again two reductions later, and every thread has
  // passed a barrier of the one between them, so its readers are done.
  template <typename U, typename Join>
  __device__ U all(U v, U none, Join join) const {
    static_assert(sizeof(U) <= sizeof(Stats), "slot");
    const int lane = threadIdx.x & 31, warps = blockDim.x >> 5;
    Stats *mine = slots + bank * kMaxWarps, *theirs = slots + 2 * kMaxWarps + bank * kMaxCluster;
    bank ^= 1;
    v = butterfly(v, 32, join);
    if (warps > 1) {
      if (lane == 0) *reinterpret_cast<U *>(mine + (threadIdx.x >> 5)) = v;
      __syncthreads();
      v = butterfly(lane < warps ? *reinterpret_cast<const U *>(mine + lane) : none, kMaxWarps, join);
      v = broadcast(v);
    }
    if (ctas > 1) {
      if ((int)threadIdx.x < ctas)
        *reinterpret_cast<U *>(cg::this_cluster().map_shared_rank(theirs, threadIdx.x) + rank) = v;
      cg::this_cluster().sync();
      v = butterfly(lane < ctas ? *reinterpret_cast<const U *>(theirs + lane) : none, kMaxCluster, join);
      v = broadcast(v);
    }
    return v;
  }
  // lanes beyond the butterfly's width hold another result
  __device__ static float broadcast(float v) { return __shfl_sync(kFull, v, 0); }
  __device__ static double broadcast(double v) { return __shfl_sync(kFull, v, 0); }
  __device__ static Stats broadcast(Stats v) {
    return Stats{broadcast(v.top), broadcast(v.sum), broadcast(v.mean)};
  }
  template <typename Op, typename U>
  __device__ U reduce(U v) const {
    return all(v, Op::none(U()), [](U a, U b) { return Op::apply(a, b); });
  }
  __device__ Stats stats(Stats v) const {
    return all(v, Stats{-INFINITY, 0.0f, 0.0f}, [](Stats a, Stats b) {
      const float top = fmaxf(a.top, b.top);
      rescale(a, top);
      rescale(b, top);
      return Stats{top, a.sum + b.sum, a.mean + b.mean};
    });
  }
};

// A row in 64 bits, read again: log sum e^{x - top} over the kept actions,
// and with `want_kl` the KL as the difference mean(x - r) - lse(x) + lse(r),
// of x - top throughout: beside 1e38 the rest is lost.  Taken by rows far
// from the reference, and by short rows next to a clip border or of a small
// call (kFineLogits).
template <typename T, typename Grp>
__device__ __noinline__ double2 row_in_64(const Params &p, const Grp &grp, int64_t row, float top, bool want_kl) {
  const int A = p.actions;
  const T *x = static_cast<const T *>(p.logits) + row * p.stride;
  const T *r = static_cast<const T *>(p.reference) + row * p.reference_stride;
  const uint8_t *legal = p.legal ? p.legal + row * A : nullptr;
  double s = 0.0, sd = 0.0, rtop = -INFINITY;
  for (int a = grp.index(); a < A; a += grp.size()) {
    const float xa = to_f(x[a]);
    if ((legal && !legal[a]) || xa == -INFINITY) continue;
    const double e = exp((double)xa - (double)top);
    s += e;
    if (want_kl) {
      const double ra = to_f(r[a]);
      sd += e * (((double)xa - (double)top) - ra);
      rtop = ra > rtop ? ra : rtop;
    }
  }
  s = grp.template reduce<SumOp>(s);
  const double log_sum = log(s);
  double kl = 0.0;
  if (want_kl) {
    sd = grp.template reduce<SumOp>(sd);
    rtop = grp.template reduce<MaxOp>(rtop);
    double sr = 0.0;
    for (int a = grp.index(); a < A; a += grp.size()) {
      if ((legal && !legal[a]) || to_f(x[a]) == -INFINITY) continue;
      sr += exp((double)to_f(r[a]) - rtop);
    }
    sr = grp.template reduce<SumOp>(sr);
    kl = (sd / s + rtop) + (log(sr) - log_sum);
  }
  return make_double2(log_sum, kl);
}

// ---------------------------------------------------------------------------
// one row
// ---------------------------------------------------------------------------

// A row's scalars, all requested with its logits: each met late would stall
// the row for a memory latency of its own.
struct RowIn {
  float xk, old, adv, ref;
  bool counts;
};

template <typename T>
__device__ __forceinline__ RowIn row_in(const Params &p, int64_t row, const T *x, const uint8_t *legal, int k,
                                        bool counts) {
  RowIn in = {0.0f, 0.0f, 0.0f, 0.0f, counts};
  if (counts) {
    in.xk = to_f(x[k]);
    const bool allowed = !legal || legal[k];
    in.old = p.old_log_prob[row];
    in.adv = p.advantage[row];
    if (p.reference_log_prob) in.ref = p.reference_log_prob[row];
    in.counts = allowed && in.xk != -INFINITY;
  }
  return in;
}

// What a row's gradient is made of: g_a = p_a ((d_a - mean) wb - wc), plus wc
// at the action.
struct RowOut {
  double share;
  float wc, wb;
};

// a log-ratio that 32-bit sums may have put on the wrong side of the clip
__device__ __forceinline__ bool near_border(const Params &p, double delta, double tol) {
  return fabs(delta - p.log_high) < tol || fabs(delta - p.log_low) < tol;
}

// The row's statistics from its sums, by every thread alike; thread 0 of the
// group writes them.  `settled`: log_sum is in 64 bits where it has to be.
template <typename T, bool Kl, typename Grp>
__device__ __forceinline__ RowOut finish_row(const Params &p, const Grp &grp, int64_t row, float weight,
                                             const RowIn &in, float top, double log_sum, bool settled, float kl_sum) {
  double lp = ((double)in.xk - (double)top) - log_sum, delta = lp - (double)in.old;
  const bool far = Kl && !(kl_sum < kFarKl);
  float kl = Kl ? log1pf(kl_sum) : 0.0f;
  if (far || (!settled && (p.fine || near_border(p, delta, kShortBorderTol)))) {
    const double2 fine = row_in_64<T>(p, grp, row, top, far);
    lp = ((double)in.xk - (double)top) - fine.x;
    delta = lp - (double)in.old;
    if (far) kl = (float)fine.y;
  }
  const bool clipped = in.adv >= 0.0f ? delta > p.log_high : delta < p.log_low;
  // (in 64 bits: the rows' terms cancel in the loss.)  An advantage of 0 adds
  // nothing, whatever the ratio overflows to, unless that is NaN
  // (weighted first: a ratio may leave 32 bits where the row's share does not)
  const double gain = (double)weight * (double)in.adv;
  double term = clipped || (in.adv == 0.0f && delta == delta) ? 0.0 : -gain * exp(delta);
  float wc = (float)term;
  if (clipped) term = -gain * (in.adv >= 0.0f ? p.clip_high : p.clip_low);
  if (!Kl && p.reference_log_prob) {
    const float y = (float)((double)in.ref - lp), em = expm1f(y);
    kl = fabsf(y) < 1.0f ? phi_small(y) : em - y;
    if (p.beta != 0.0f) wc = fmaf(-weight * p.beta, em, wc);
  }
  // (without a coefficient the KL is a statistic alone, and may be infinite)
  if (p.beta != 0.0f) term += (double)weight * ((double)p.beta * (double)kl);
  if (grp.index() == 0) {
    p.log_prob[row] = (float)lp;
    p.clipped[row] = clipped;
    if (p.kl) p.kl[row] = kl;
  }
  return RowOut{term, wc, weight * p.beta};
}

__device__ __forceinline__ void empty_row(const Params &p, int64_t row) {
  p.log_prob[row] = 0.0f;
  p.clipped[row] = 0;
  if (p.kl) p.kl[row] = 0.0f;
}

// p phi(y) of one action whose y = mean - d is not within (-1, 1).  An e^y
// that overflows, or meets a p that underflowed, makes the row a far one.  Out
// of line: few actions are that far, and e^y for all of them is a third of the
// row's work.
__device__ __noinline__ float kl_part_far(float pa, float y) {
  return pa > 0.0f ? fmaf(pa, expf(y), -pa * (1.0f + y)) : (y > 60.0f ? INFINITY : pa * 0.0f);
}

// ---------------------------------------------------------------------------
// rows on their way to shared memory
// ---------------------------------------------------------------------------

// the place of `from` within 16 bytes, in elements
template <typename E>
__device__ __forceinline__ int phase_of(const E *from) {
  return (int)((reinterpret_cast<uintptr_t>(from) & 15) / sizeof(E));
}

template <int Bytes>
__device__ __forceinline__ void copy_async(void *to, const void *from) {
  const uint32_t dst = (uint32_t)__cvta_generic_to_shared(to);
  if (Bytes == 16)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(from) : "memory");
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(from) : "memory");
}

// Copies `count` elements, by `threads` threads, to the same place within 16
// bytes as they have in global memory, so that whole vectors move at any
// alignment: asynchronous copies of 16 bytes, of 4 at the ends, and where
// even those do not fit, plain ones.
template <typename E>
__device__ __forceinline__ void stage(E *to, const E *from, int count, int t, int threads) {
  constexpr int kVec = 16 / (int)sizeof(E), kWord = 4 / (int)sizeof(E);
  const int phase = phase_of(from), head = (kVec - phase) % kVec;
  const int first = head < count ? head : count, vecs = (count - first) / kVec, last = first + vecs * kVec;
  for (int i = t; i < vecs; i += threads) copy_async<16>(to + first + i * kVec, from + first + i * kVec);
  const int ends = first + count - last;
  if (phase % kWord == 0 && first % kWord == 0 && count % kWord == 0) {
    for (int i = t * kWord; i < ends; i += threads * kWord) {
      const int at = i < first ? i : last + i - first;
      copy_async<4>(to + at, from + at);
    }
  } else {
    for (int i = t; i < ends; i += threads) {
      const int at = i < first ? i : last + i - first;
      to[at] = from[at];
    }
  }
}

// ---------------------------------------------------------------------------
// short rows: `group` lanes of a warp each, their elements in registers
// ---------------------------------------------------------------------------

// CTAs an SM, as the registers of a thread's elements allow
template <int Elems, bool Kl>
constexpr int kShortCtas = Kl && Elems > 12 ? 2 : 3;

// One array's rows of a warp's batch in shared memory.
template <typename E>
struct Batch {
  E *at;      // of the warp's buffer
  int pitch;  // elements between rows that are staged one by one, 0 if the rows are one piece

  __device__ __forceinline__ void load(const E *first, int64_t stride, int rows, int A, int lane) const {
    if (!pitch) {
      stage(at + phase_of(first), first, rows * A, lane, 32);
    } else {
      for (int i = 0; i < rows; ++i)
        stage(at + i * pitch + phase_of(first + i * stride), first + i * stride, A, lane, 32);
    }
  }
  __device__ __forceinline__ const E *row(const E *first, int64_t stride, int i, int A) const {
    return pitch ? at + i * pitch + phase_of(first + i * stride) : at + phase_of(first) + i * A;
  }
};

// The copies of a batch whose rows are one piece of global memory: 16 bytes
// each in the middle, 4 at the ends.
struct Piece {
  const uint8_t *from;  // of the first batch
  int64_t step;         // bytes from batch to batch
  int phase, first, vecs, words;
  bool ok;              // the ends are whole words, and every batch is alike

  __device__ __forceinline__ void copy(uint32_t to, int64_t turn, int lane) const {
    // (read once: nothing in shared memory is kept across an asm)
    const int head = first, n = vecs, ends = words;
    const uint8_t *src = from + turn * step;
    to += (uint32_t)phase;
    for (int i = lane; i < n; i += 32)
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to + head + 16 * i), "l"(src + head + 16 * i)
                   : "memory");
    if (lane < ends) {
      const int at = 4 * lane < head ? 4 * lane : 4 * lane + 16 * n;
      asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(to + at), "l"(src + at) : "memory");
    }
  }
};

__device__ __forceinline__ Piece piece_of(const void *from, int bytes, int64_t step) {
  Piece p;
  p.from = static_cast<const uint8_t *>(from);
  p.step = step;
  p.phase = (int)(reinterpret_cast<uintptr_t>(from) & 15);
  const int head = (16 - p.phase) & 15;
  p.first = head < bytes ? head : bytes;
  p.vecs = (bytes - p.first) / 16;
  p.words = (bytes - 16 * p.vecs) / 4;  // at most 3 at each end
  p.ok = p.phase % 4 == 0 && bytes % 4 == 0 && step % 16 == 0;
  return p;
}

// A batch is the rows that a warp takes at once, one per lane group; while
// it is computed the next one is on its way, its scalars in registers.
struct Scalars {
  float weight, old, adv, ref;
  int action;
};

__device__ __forceinline__ Scalars scalars_of(const Params &p, int64_t row) {
  Scalars s = {0.0f, 0.0f, 0.0f, 0.0f, -1};
  if (row < p.rows) {
    s.weight = p.weight ? p.weight[row] : p.even_weight;
    s.action = p.action[row];
    s.old = p.old_log_prob[row];
    s.adv = p.advantage[row];
    if (p.reference_log_prob) s.ref = p.reference_log_prob[row];
  }
  return s;
}

// V vectors of W elements per thread; thread t of the group holds vectors
// t, t + G, ... of the row.  Returns the row's share of the loss.
template <typename T, int W, int V, bool Kl>
__device__ __forceinline__ double short_row(const Params &p, const Lanes &grp, int64_t row, const Scalars &s,
                                            const T *sx, const T *sr, const uint8_t *sl) {
  const int A = p.actions, t = grp.index(), G = grp.size(), k = s.action;
  T *grad = p.grad ? static_cast<T *>(p.grad) + row * A : nullptr;
  using Pack = Vec<T, W>;
  RowIn in = {0.0f, s.old, s.adv, s.ref, s.weight != 0.0f && k >= 0 && k < A};
  if (in.counts) {
    in.xk = to_f(sx[k]);
    in.counts = (!sl || sl[k]) && in.xk != -INFINITY;
  }
  if (!in.counts) {
    if (t == 0) empty_row(p, row);
    if (grad) {
      Pack z;
#pragma unroll
      for (int w = 0; w < W; ++w) z.v[w] = from_f<T>(0.0f);
#pragma unroll
      for (int v = 0; v < V; ++v) {
        const int a = (v * G + t) * W;
        if (a < A) *reinterpret_cast<Pack *>(grad + a) = z;
      }
    }
    return 0.0;
  }
  // an action that is illegal, or has a logit of -inf, keeps x = -inf and
  // d = 0, as places past the row do (the buffer goes on there)
  float e[V * W], d[Kl ? V * W : 1], top = -INFINITY;
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const int a = (v * G + t) * W;
    const bool inside = a < A;
    const Pack xv = *reinterpret_cast<const Pack *>(sx + a);
    Pack rv;
    Vec<uint8_t, W> lv;
    if (Kl) rv = *reinterpret_cast<const Pack *>(sr + a);
    if (sl) lv = *reinterpret_cast<const Vec<uint8_t, W> *>(sl + a);
#pragma unroll
    for (int w = 0; w < W; ++w) {
      const int i = v * W + w;
      const float xa = to_f(xv.v[w]);
      const bool keep = xa != -INFINITY && inside && (!sl || lv.v[w] != 0);
      e[i] = keep ? xa : -INFINITY;
      top = fmaxf(top, e[i]);
      if (Kl) d[Kl ? i : 0] = keep ? xa - to_f(rv.v[w]) : 0.0f;
    }
  }
  top = grp.reduce<MaxOp>(top);
  float sum = 0.0f, mean = 0.0f, kl = 0.0f;
#pragma unroll
  for (int i = 0; i < V * W; ++i) {
    e[i] = exp_fast(e[i] - top);
    sum += e[i];
    if (Kl) mean = fmaf(e[i], d[Kl ? i : 0], mean);
  }
  sum = grp.reduce<SumOp>(sum);
  const float inv = 1.0f / sum;
  if (Kl) {
    mean = grp.reduce<SumOp>(mean) * inv;
    bool some = false;
#pragma unroll
    for (int i = 0; i < V * W; ++i) {
      const float y = mean - d[Kl ? i : 0];
      const bool near = fabsf(y) < 1.0f;
      some |= !near;
      kl = fmaf(near ? e[i] : 0.0f, phi_small(near ? y : 0.0f), kl);
    }
    kl *= inv;
    if (some) {
#pragma unroll
      for (int i = 0; i < V * W; ++i)
        if (const float y = mean - d[Kl ? i : 0]; !(fabsf(y) < 1.0f)) {
          if (e[i] != 0.0f) {
            kl += kl_part_far(e[i] * inv, y);
          } else {
            // (a place that is not kept has d = 0.)  The gradient is 0, where
            // a logit of the type's lowest value leaves a d that overflows
            if (y > 60.0f && d[Kl ? i : 0] != 0.0f) kl = INFINITY;
            d[Kl ? i : 0] = mean;
          }
        }
    }
    // actions with p = 0 whose logits are equal (d = 0) count above 60, and
    // are looked up there alone (telling them from places that are not kept
    // element by element took 121 us for 262144 x 82 fp32, not 105)
    if (mean > 60.0f) {
#pragma unroll 1
      for (int a = t; a < A; a += G) {
        const float xa = to_f(sx[a]);
        if (xa != to_f(sr[a]) || xa == -INFINITY || (sl && !sl[a])) continue;
        if (exp_fast(xa - top) == 0.0f) kl = INFINITY;
      }
    }
    kl = grp.reduce<SumOp>(kl);
  }
  const RowOut out = finish_row<T, Kl>(p, grp, row, s.weight, in, top, log_row_sum(sum), false, kl);
  if (grad) {
    const float wc = -out.wc * inv, wb = out.wb * inv;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const int a = (v * G + t) * W;
      Pack o;
#pragma unroll
      for (int w = 0; w < W; ++w) {
        const int i = v * W + w;
        float g = (Kl ? fmaf(wb, d[Kl ? i : 0] - mean, wc) : wc) * e[i];
        if (a + w == k) g += out.wc;
        o.v[w] = from_f<T>(g);
      }
      if (a < A) *reinterpret_cast<Pack *>(grad + a) = o;
    }
  }
  return out.share;
}

template <typename T, int W, int V, bool Kl>
__global__ void __launch_bounds__(kShortThreads, kShortCtas<V * W, Kl>)
    policy_loss_short_kernel(const __grid_constant__ Params p) {
  extern __shared__ __align__(16) uint8_t s_rows[];
  __shared__ double s_part[kShortThreads / 32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, G = p.group, A = p.actions;
  Lanes grp;
  grp.lanes = G;
  grp.mask = G == 32 ? kFull : ((1u << G) - 1u) << (lane & ~(G - 1));
  const int per_warp = 32 / G;
  const int64_t step = (int64_t)gridDim.x * (kShortThreads / 32) * per_warp;
  int64_t first = ((int64_t)blockIdx.x * (kShortThreads / 32) + warp) * per_warp;
  const T *x = static_cast<const T *>(p.logits), *r = static_cast<const T *>(p.reference);
  const int buffer = (Kl ? 2 : 1) * p.slice_bytes + (p.legal ? p.mask_bytes : 0);
  uint8_t *const base = s_rows + warp * 2 * buffer;
  // A full batch of rows in one piece starts at the same place within 16
  // bytes every time (the step is a multiple of 16 rows): its copies are
  // worked out once, and kept in shared memory, not in the registers that
  // the elements need (262144 x 82 fp32 with a sampled KL 60 us for 69).
  __shared__ Piece s_pieces[kShortThreads / 32][3];
  const Piece &px = s_pieces[warp][0], &pr = s_pieces[warp][1], &pl = s_pieces[warp][2];
  if (lane == 0) {
    s_pieces[warp][0] = piece_of(x + first * p.stride, per_warp * A * (int)sizeof(T), step * p.stride * (int)sizeof(T));
    s_pieces[warp][1] = piece_of(r + first * p.reference_stride, per_warp * A * (int)sizeof(T),
                                 step * p.reference_stride * (int)sizeof(T));
    s_pieces[warp][2] = piece_of(p.legal + first * A, per_warp * A, step * A);
  }
  __syncwarp();
  const bool pieces = !p.x_pitch && px.ok && (!Kl || (!p.r_pitch && pr.ok)) && (!p.legal || pl.ok);
  const uint32_t base_at = (uint32_t)__cvta_generic_to_shared(base);
  int64_t turn = 0;
  auto request = [&](int64_t at, int bank) {
    if (pieces && at + per_warp <= p.rows) {
      const uint32_t to = base_at + (uint32_t)(bank * buffer);
      px.copy(to, turn, lane);
      if (Kl) pr.copy(to + p.slice_bytes, turn, lane);
      if (p.legal) pl.copy(to + (Kl ? 2 : 1) * p.slice_bytes, turn, lane);
    } else if (at < p.rows) {
      const int rows = p.rows - at < per_warp ? (int)(p.rows - at) : per_warp;
      uint8_t *buf = base + bank * buffer;
      Batch<T>{reinterpret_cast<T *>(buf), p.x_pitch}.load(x + at * p.stride, p.stride, rows, A, lane);
      if (Kl)
        Batch<T>{reinterpret_cast<T *>(buf + p.slice_bytes), p.r_pitch}.load(r + at * p.reference_stride,
                                                                            p.reference_stride, rows, A, lane);
      if (p.legal) Batch<uint8_t>{buf + (Kl ? 2 : 1) * p.slice_bytes, 0}.load(p.legal + at * A, A, rows, A, lane);
    }
    ++turn;
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  double sum = 0.0;
  int bank = 0;
  request(first, 0);
  Scalars next = scalars_of(p, first + lane / G);
  for (; first < p.rows; first += step, bank ^= 1) {
    const Scalars now = next;
    request(first + step, bank ^ 1);
    next = scalars_of(p, first + step + lane / G);
    asm volatile("cp.async.wait_group 1;" ::: "memory");
    __syncwarp();
    const int64_t row = first + lane / G;
    if (row < p.rows) {
      uint8_t *buf = base + bank * buffer;
      const T *sx, *sr = nullptr;
      const uint8_t *sl = nullptr;
      if (pieces) {
        sx = reinterpret_cast<const T *>(buf + px.phase) + lane / G * A;
        if (Kl) sr = reinterpret_cast<const T *>(buf + p.slice_bytes + pr.phase) + lane / G * A;
        if (p.legal) sl = buf + (Kl ? 2 : 1) * p.slice_bytes + pl.phase + lane / G * A;
      } else {
        sx = Batch<T>{reinterpret_cast<T *>(buf), p.x_pitch}.row(x + first * p.stride, p.stride, lane / G, A);
        if (Kl)
          sr = Batch<T>{reinterpret_cast<T *>(buf + p.slice_bytes), p.r_pitch}.row(r + first * p.reference_stride,
                                                                                   p.reference_stride, lane / G, A);
        if (p.legal)
          sl = Batch<uint8_t>{buf + (Kl ? 2 : 1) * p.slice_bytes, 0}.row(p.legal + first * A, A, lane / G, A);
      }
      const double share = short_row<T, W, V, Kl>(p, grp, row, now, sx, sr, sl);
      if (grp.index() == 0) sum += share;
    }
    __syncwarp();  // the buffer is read: the batch after the next may take it
  }
  for (int off = 16; off; off >>= 1) sum += __shfl_xor_sync(kFull, sum, off);
  if (lane == 0) s_part[warp] = sum;
  __syncthreads();
  if (threadIdx.x == 0) {
    double total = 0.0;
    for (int i = 0; i < kShortThreads / 32; ++i) total += s_part[i];
    if (gridDim.x == 1)
      p.loss[0] = (float)total;
    else
      p.partial[blockIdx.x] = total;
  }
}

// ---------------------------------------------------------------------------
// long rows: a CTA each, or a cluster's slices, in shared memory
// ---------------------------------------------------------------------------

// Passes over the slice's elements, W at a time where the row's arrays start
// at the same place within a vector (vector v then holds elements v W -
// lead.. of each), else by themselves (W = 1).
//
// Three passes read shared memory: the online maximum and sums, the KL's
// sum, the gradient; each computes e^x again, which is cheaper than the
// registers or the memory to keep it (and lets two to sixteen CTAs share an
// SM, so that one loads while others compute).
template <typename T, int W, bool Kl>
__global__ void __launch_bounds__(kLongThreads, 4) policy_loss_long_kernel(const __grid_constant__ Params p) {
  extern __shared__ __align__(16) uint8_t s_rows[];
  __shared__ __align__(16) Stats s_slots[2 * kMaxWarps + 2 * kMaxCluster];
  using Pack = Vec<T, W>;
  using Mask = Vec<uint8_t, W>;
  Ctas grp;
  grp.slots = s_slots;
  grp.ctas = (int)cg::this_cluster().num_blocks();
  grp.rank = (int)cg::this_cluster().block_rank();
  grp.bank = 0;
  const int A = p.actions, t = threadIdx.x, threads = blockDim.x;
  const int lo = (int)((int64_t)A * grp.rank / grp.ctas) / 16 * 16;
  const int hi = grp.rank + 1 == grp.ctas ? A : (int)((int64_t)A * (grp.rank + 1) / grp.ctas) / 16 * 16;
  const int n = hi - lo;
  T *const sx_at = reinterpret_cast<T *>(s_rows);
  T *const sr_at = reinterpret_cast<T *>(s_rows + p.slice_bytes);
  uint8_t *const sl_at = s_rows + (Kl ? 2 : 1) * p.slice_bytes;
  const int64_t first = blockIdx.x / grp.ctas, step = gridDim.x / grp.ctas;
  double share = 0.0;
  // A CTA's shared memory may be written by the others only once it runs:
  // each arrives here, and waits after its first row is requested (every
  // cluster has one), so that the row's latency hides the barrier's.
  if (grp.ctas > 1) cg::this_cluster().barrier_arrive();
  for (int64_t row = first; row < p.rows; row += step) {
    const float weight = p.weight ? p.weight[row] : p.even_weight;
    const int k = p.action[row];
    const T *x = static_cast<const T *>(p.logits) + row * p.stride;
    const T *r = Kl ? static_cast<const T *>(p.reference) + row * p.reference_stride : nullptr;
    const uint8_t *legal = p.legal ? p.legal + row * A : nullptr;
    T *grad = p.grad ? static_cast<T *>(p.grad) + row * A + lo : nullptr;
    const bool wanted = weight != 0.0f && k >= 0 && k < A;
    T *sx = sx_at + phase_of(x + lo), *sr = sr_at;
    uint8_t *sl = sl_at;
    if (wanted) {
      stage(sx, x + lo, n, t, threads);
      if (Kl) {
        sr += phase_of(r + lo);
        stage(sr, r + lo, n, t, threads);
      }
      if (legal) {
        sl += phase_of(legal + lo);
        stage(sl, legal + lo, n, t, threads);
      }
    }
    const RowIn in = row_in<T>(p, row, x, legal, k, wanted);
    if (grp.ctas > 1 && row == first) cg::this_cluster().barrier_wait();
    asm volatile("cp.async.wait_all;" ::: "memory");
    __syncthreads();
    if (!in.counts) {
      if (grp.index() == 0) empty_row(p, row);
      if (grad)
        for (int i = t; i < n; i += threads) grad[i] = from_f<T>(0.0f);
      __syncthreads();
      continue;
    }
    // vector v covers elements v W - lead .. + W - 1
    const int lead = phase_of(x + lo) % W, vecs = (n + lead + W - 1) / W;
    // logits, and the difference to the reference, of one vector; -inf and 0
    // where there is no kept action
    auto load = [&](int v, float(&xa)[W], float(&da)[W]) {
      const int a = v * W - lead;
      unpack(*reinterpret_cast<const Pack *>(sx + a), xa);
      if (a < 0 || a + W > n) {
#pragma unroll
        for (int w = 0; w < W; ++w)
          if (a + w < 0 || a + w >= n) xa[w] = -INFINITY;
      }
      if (legal) {
        const Mask lv = *reinterpret_cast<const Mask *>(sl + a);
#pragma unroll
        for (int w = 0; w < W; ++w) xa[w] = lv.v[w] ? xa[w] : -INFINITY;
      }
      if (Kl) {
        float ra[W];
        unpack(*reinterpret_cast<const Pack *>(sr + a), ra);
#pragma unroll
        for (int w = 0; w < W; ++w) da[w] = xa[w] == -INFINITY ? 0.0f : xa[w] - ra[w];
      }
    };
    // single elements are taken eight at a time, so that no chain of adds is
    // longer than a row of vectors has (kBorderTol)
    constexpr int kTake = W == 1 ? 8 : 1, kElems = kTake * W;
    // The maximum starts at kLowest, so that logits of the type's lowest value
    // have no part before a larger one is met: their differences to the
    // reference would overflow the mean.  A row without one starts from -inf.
    Stats st;
    for (float least = Kl ? kLowest : -INFINITY;; least = -INFINITY) {
      st = {least, 0.0f, 0.0f};
      // st.top, or 0 without an action yet, when only a NaN has a part in the sum
      float from = least == -INFINITY ? 0.0f : least;
      for (int first_v = t; first_v < vecs; first_v += kTake * threads) {
        float xa[kElems], da[kElems];
#pragma unroll
        for (int i = 0; i < kTake; ++i) {
          const int v = first_v + i * threads;
          float xv[W], dv[W];
          const bool inside = kTake == 1 || v < vecs;
          load(inside ? v : vecs - 1, xv, dv);
#pragma unroll
          for (int w = 0; w < W; ++w) {
            xa[i * W + w] = inside ? xv[w] : -INFINITY;
            if (Kl) da[i * W + w] = inside ? dv[w] : 0.0f;
          }
        }
        float top = xa[0];
#pragma unroll
        for (int w = 1; w < kElems; ++w) top = fmaxf(top, xa[w]);
        if (top > st.top) {
          rescale(st, top);
          from = top;
        }
        float e[kElems], sum[2] = {0.0f, 0.0f}, mean[2] = {0.0f, 0.0f};
        exps(xa, from, e);
#pragma unroll
        for (int w = 0; w < kElems; ++w) {
          sum[w & 1] += e[w];
          if (Kl) mean[w & 1] = fmaf(e[w], da[w], mean[w & 1]);
        }
        st.sum += sum[0] + sum[1];
        if (Kl) st.mean += mean[0] + mean[1];
      }
      st = grp.stats(st);
      if (st.sum != 0.0f || least == -INFINITY) break;
    }
    const float inv = 1.0f / st.sum, mean = st.mean * inv;
    float kl = 0.0f;
    if (Kl) {
      for (int v = t; v < vecs; v += threads) {
        float xa[W], da[W], e[W], part = 0.0f;
        bool some = false;
        load(v, xa, da);
        exps(xa, st.top, e);
#pragma unroll
        for (int w = 0; w < W; ++w) {
          const float y = mean - da[w];
          const bool near = fabsf(y) < 1.0f;
          some |= !near;
          part = fmaf(near ? e[w] : 0.0f, phi_small(near ? y : 0.0f), part);
        }
        kl = fmaf(part, inv, kl);
        if (some) {
#pragma unroll 1
          for (int w = 0; w < W; ++w) {
            // from shared memory again: registers are not indexed
            const int a = v * W - lead + w;
            if (a < 0 || a >= n || (legal && !sl[a])) continue;
            const float xw = to_f(sx[a]), dw = xw - to_f(sr[a]);
            if (xw == -INFINITY || fabsf(mean - dw) < 1.0f) continue;
            kl += kl_part_far(exp_fast(xw - st.top) * inv, mean - dw);
          }
        }
      }
      kl = grp.reduce<SumOp>(kl);
    }
    double log_sum = log_row_sum(st.sum);
    const bool fine =
        p.fine || near_border(p, ((double)in.xk - (double)st.top) - log_sum - (double)in.old, kBorderTol);
    if (fine) {  // as row_in_64, from shared memory (out of line it was slower)
      double s = 0.0;
      for (int v = t; v < vecs; v += threads) {
        float xa[W], da[W];
        load(v, xa, da);
#pragma unroll
        for (int w = 0; w < W; ++w) s += exp_64((double)xa[w] - (double)st.top);
      }
      log_sum = log(grp.reduce<SumOp>(s));
    }
    const RowOut out = finish_row<T, Kl>(p, grp, row, weight, in, st.top, log_sum, true, kl);
    share += out.share;
    if (grad) {
      const float wc = -out.wc * inv, wb = out.wb * inv;
      const int at_k = k - lo + lead;  // the action, counted from vector 0
      if (Kl && !(fabsf(wb) <= 1.0f)) {
        // p = 0 has no gradient, where a logit of the type's lowest value
        // leaves a d that overflows once multiplied by wb.  (Each thread
        // writes the elements that it reads.)
        for (int v = t; v < vecs; v += threads)
#pragma unroll 1
          for (int a = max(v * W - lead, 0); a < min(v * W - lead + W, n); ++a)
            if (exp_fast(to_f(sx[a]) - st.top) == 0.0f) sr[a] = sx[a];
      }
      for (int v = t; v < vecs; v += threads) {
        float xa[W], da[W], e[W];
        load(v, xa, da);
        exps(xa, st.top, e);
        const int a = v * W - lead;
#pragma unroll
        for (int w = 0; w < W; ++w) xa[w] = (Kl ? fmaf(wb, da[w] - mean, wc) : wc) * e[w];
        if (at_k / W == v && at_k >= 0) {
#pragma unroll
          for (int w = 0; w < W; ++w)
            if (v * W + w == at_k) xa[w] += out.wc;
        }
        const Pack o = pack<T, W>(xa);
        if (a >= 0 && a + W <= n) {
          *reinterpret_cast<Pack *>(grad + a) = o;
        } else {
#pragma unroll
          for (int w = 0; w < W; ++w)
            if (a + w >= 0 && a + w < n) grad[a + w] = o.v[w];
        }
      }
    }
    __syncthreads();  // the slice is read: the next row may take its place
  }
  if (grp.index() == 0) {
    if (step == 1)
      p.loss[0] = (float)share;
    else
      p.partial[first] = share;
  }
  if (grp.ctas > 1) cg::this_cluster().sync();  // a CTA's slots outlive their readers
}

// the CTAs' sums in a fixed order
__global__ void policy_loss_sum_kernel(const double *partial, int n, float *loss) {
  __shared__ double s_part[32];
  cudaGridDependencySynchronize();
  double sum = 0.0;
  for (int i = threadIdx.x; i < n; i += blockDim.x) sum += partial[i];
  for (int off = 16; off; off >>= 1) sum += __shfl_xor_sync(kFull, sum, off);
  if ((threadIdx.x & 31) == 0) s_part[threadIdx.x >> 5] = sum;
  __syncthreads();
  if (threadIdx.x == 0) {
    double total = 0.0;
    for (int i = 0; i < (int)(blockDim.x >> 5); ++i) total += s_part[i];
    loss[0] = (float)total;
  }
}

// ---------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------

constexpr int kMaxDevices = 64;

int current_device() {
  int dev = 0;
  return cudaGetDevice(&dev) == cudaSuccess && dev >= 0 && dev < kMaxDevices ? dev : 0;
}

int sm_count() {
  static std::atomic<int> known[kMaxDevices];
  const int dev = current_device();
  int n = known[dev].load(std::memory_order_relaxed);
  if (n) return n;
  if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n <= 0) return 148;
  known[dev].store(n, std::memory_order_relaxed);
  return n;
}

// the kernel may use kLongShared bytes, and clusters above 8 CTAs if
// `large`; asked once per kernel and device
template <typename K>
cudaError_t allow(K *kernel, std::atomic<uint64_t> &done, bool large) {
  const uint64_t bit = 1ull << current_device();
  if (done.load(std::memory_order_acquire) & bit) return cudaSuccess;
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kLongShared);
  if (e == cudaSuccess && large) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
  if (e == cudaSuccess) done.fetch_or(bit, std::memory_order_release);
  return e;
}

template <typename T, int W, int V, bool Kl>
cudaError_t launch_short(Params &p, int *ctas, cudaStream_t st) {
  const int per_warp = 32 / p.group, warps = kShortThreads / 32;
  // rows that follow one another are staged as one piece
  const int pitch = (p.actions * (int)sizeof(T) + 31) / 16 * 16 / (int)sizeof(T);
  p.x_pitch = p.stride == p.actions ? 0 : pitch;
  p.r_pitch = !Kl || p.reference_stride == p.actions ? 0 : pitch;
  // a lane's vectors past the last row are read too, and ignored
  const int past = p.group * V * W;
  const int row = p.x_pitch || p.r_pitch ? pitch : p.actions;
  p.slice_bytes = ((per_warp * row + past) * (int)sizeof(T) + 31) / 16 * 16;
  p.mask_bytes = (per_warp * p.actions + past + 47) / 16 * 16;
  const int smem = warps * 2 * ((Kl ? 2 : 1) * p.slice_bytes + (p.legal ? p.mask_bytes : 0));
  static std::atomic<uint64_t> allowed{0};
  const cudaError_t e = allow(policy_loss_short_kernel<T, W, V, Kl>, allowed, false);
  if (e != cudaSuccess) return e;
  const int64_t need = (p.rows + per_warp * warps - 1) / (per_warp * warps);
  const int most = sm_count() * kShortCtas<V * W, Kl>;
  *ctas = (int)(need < most ? need : most);
  policy_loss_short_kernel<T, W, V, Kl><<<*ctas, kShortThreads, smem, st>>>(p);
  return cudaPeekAtLastError();
}

// Lanes of a short row: 4 to 32, with 4 to 24 elements each: the split with
// the fewest idle places, and among those the fewest lanes: a batch costs
// some 550 instructions besides its elements' (its copies, its rows' ends),
// which more rows share.
template <typename T, int W, bool Kl>
cudaError_t by_lanes(Params &p, int *ctas, cudaStream_t st) {
  constexpr int kElems[] = {4, 6, 8, 12, 16, 24};
  int best = 0, elems = 0;
  for (int e : kElems)
    for (int g = 4; g <= 32; g *= 2)
      if (g * e >= p.actions && (!best || g * e < best * elems || (g * e == best * elems && g < best))) {
        best = g;
        elems = e;
      }
  p.group = best;
  if (elems == 4) return launch_short<T, W, 4 / W, Kl>(p, ctas, st);
  if (elems == 6) return launch_short<T, W, 6 / W, Kl>(p, ctas, st);
  if (elems == 8) return launch_short<T, W, 8 / W, Kl>(p, ctas, st);
  if (elems == 12) return launch_short<T, W, 12 / W, Kl>(p, ctas, st);
  if (elems == 16) return launch_short<T, W, 16 / W, Kl>(p, ctas, st);
  return launch_short<T, W, 24 / W, Kl>(p, ctas, st);
}

// Long rows: a cluster where half an SM's shared memory does not hold the
// row, or where the rows leave SMs idle (down to 4096 actions a CTA);
// threads for four vectors or more each (256 at most: 512 took 166 us for
// 4096 x 32000 bf16 where 256 take 145); and as many CTAs an SM as its shared
// memory holds.
template <typename T, int W, bool Kl>
cudaError_t by_cta(Params &p, int *ctas, cudaStream_t st) {
  const int64_t sms = sm_count();
  // a slice may begin 16 elements early, lie 15 bytes into its place, and be
  // read to the end of its last vector
  auto bytes = [&](int cluster) {
    const int64_t slice = (p.actions + cluster - 1) / cluster + 16;
    p.slice_bytes = (int)((slice * (int64_t)sizeof(T) + 47) / 16 * 16);
    return (int64_t)(Kl ? 2 : 1) * p.slice_bytes + (p.legal ? (slice + 47) / 16 * 16 : 0);
  };
  int cluster = 1;
  while (cluster < kMaxCluster && bytes(cluster) > kLongShared / 2) cluster *= 2;
  while (cluster < kMaxCluster && p.rows * cluster * 2 <= sms && p.actions / cluster > 4096) cluster *= 2;
  const int64_t smem = bytes(cluster);
  if (smem > kLongShared) return cudaErrorInvalidValue;
  const int vecs = (p.actions / cluster + W - 1) / W;
  int threads = 64;
  while (threads < kLongThreads && threads * 4 < vecs) threads *= 2;
  static std::atomic<uint64_t> allowed{0};
  const cudaError_t e = allow(policy_loss_long_kernel<T, W, Kl>, allowed, true);
  if (e != cudaSuccess) return e;
  int64_t resident = kLongShared / (smem + 2048);
  if (resident > 1024 / threads) resident = 1024 / threads;  // the registers' limit
  if (resident < 1) resident = 1;
  int64_t most = sms * resident / cluster;
  if (most > kMaxPartials) most = kMaxPartials;
  if (most < 1) most = 1;
  *ctas = (int)(p.rows < most ? p.rows : most);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(*ctas * cluster));
  cfg.blockDim = dim3((unsigned)threads);
  cfg.dynamicSmemBytes = (size_t)smem;
  cfg.stream = st;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = (unsigned)cluster;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, policy_loss_long_kernel<T, W, Kl>, p);
}

// vectors of W elements need every row of every array to start on one
bool rows_aligned(const Params &p, int w, size_t size) {
  auto ok = [](const void *q, size_t bytes) { return (reinterpret_cast<uintptr_t>(q) & (bytes - 1)) == 0; };
  return p.actions % w == 0 && p.stride % w == 0 && ok(p.logits, w * size) &&
         (!p.reference || (p.reference_stride % w == 0 && ok(p.reference, w * size))) &&
         (!p.legal || ok(p.legal, (size_t)w)) && (!p.grad || ok(p.grad, w * size));
}

// or, for the shared memory of long rows, all arrays' rows to start at the
// same place within one
bool same_phase(const Params &p, int w, size_t size) {
  auto at = [&](const void *q, size_t s) { return (int)(reinterpret_cast<uintptr_t>(q) / s % (size_t)w); };
  const int x = at(p.logits, size);
  return (p.stride - p.actions) % w == 0 &&
         (!p.reference || ((p.reference_stride - p.stride) % w == 0 && at(p.reference, size) == x)) &&
         (!p.legal || at(p.legal, 1) == x) && (!p.grad || at(p.grad, size) == x);
}

template <typename T, bool Kl>
cudaError_t by_type(Params &p, int *ctas, cudaStream_t st) {
  if (p.actions <= kMaxShort)
    return rows_aligned(p, 2, sizeof(T)) ? by_lanes<T, 2, Kl>(p, ctas, st) : by_lanes<T, 1, Kl>(p, ctas, st);
  constexpr int kWide = 16 / (int)sizeof(T);
  return same_phase(p, kWide, sizeof(T)) ? by_cta<T, kWide, Kl>(p, ctas, st) : by_cta<T, 1, Kl>(p, ctas, st);
}

}  // namespace

extern "C" {

size_t scacchi_policy_loss_workspace_bytes(void) { return kMaxPartials * sizeof(double); }

int scacchi_policy_loss(const scacchi_policy_rows *rows, const scacchi_policy_out *out, int64_t num_rows,
                        int32_t num_actions, int32_t dtype, double clip_low, double clip_high, float kl_coefficient,
                        void *workspace, void *stream) {
  if (!rows || !out || num_rows < 0 || num_actions < 1 || num_actions > kMaxActions || dtype < 0 || dtype > 2 ||
      !(clip_low >= 0.0 && clip_low < 1.0) || !(clip_high >= 0.0) || !isfinite(clip_high) ||
      !isfinite(kl_coefficient) || !out->loss)
    return SCACCHI_EINVAL;
  const bool full = rows->reference_logits != nullptr, sampled = rows->reference_log_prob != nullptr;
  if (full && sampled) return SCACCHI_EINVAL;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (num_rows == 0)
    return cudaMemsetAsync(out->loss, 0, sizeof(float), st) == cudaSuccess ? SCACCHI_OK : SCACCHI_ECUDA;
  const size_t size = dtype == 0 ? 4 : 2;
  auto bad = [](const void *q, size_t a) { return (reinterpret_cast<uintptr_t>(q) & (a - 1)) != 0; };
  if (!rows->logits || !rows->action || !rows->old_log_prob || !rows->advantage || !out->log_prob || !out->clipped ||
      !workspace || rows->logits_stride < num_actions || (full && rows->reference_stride < num_actions))
    return SCACCHI_EINVAL;
  if (((full || sampled) && !out->kl) || bad(rows->logits, size) || bad(rows->reference_logits, size) ||
      bad(out->grad_logits, size) || bad(rows->action, 4) || bad(rows->old_log_prob, 4) || bad(rows->advantage, 4) ||
      bad(rows->weight, 4) || bad(rows->reference_log_prob, 4) || bad(out->loss, 4) || bad(out->log_prob, 4) ||
      bad(out->kl, 4) || bad(workspace, 8))
    return SCACCHI_EINVAL;
  Params p = {};
  p.logits = rows->logits;
  p.reference = rows->reference_logits;
  p.legal = rows->legal;
  p.action = rows->action;
  p.old_log_prob = rows->old_log_prob;
  p.advantage = rows->advantage;
  p.weight = rows->weight;
  p.reference_log_prob = rows->reference_log_prob;
  p.loss = out->loss;
  p.log_prob = out->log_prob;
  p.kl = out->kl;
  p.clipped = out->clipped;
  p.grad = out->grad_logits;
  p.partial = static_cast<double *>(workspace);
  p.rows = num_rows;
  p.stride = rows->logits_stride;
  p.reference_stride = rows->reference_stride;
  p.actions = num_actions;
  p.clip_low = 1.0 - clip_low;
  p.clip_high = 1.0 + clip_high;
  p.log_low = log1p(-clip_low);
  p.log_high = log1p(clip_high);
  p.beta = kl_coefficient;
  p.even_weight = (float)(1.0 / (double)num_rows);
  p.fine = num_rows <= kFineLogits / num_actions;
  int ctas = 0;
  cudaError_t err;
  if (dtype == 0)
    err = full ? by_type<float, true>(p, &ctas, st) : by_type<float, false>(p, &ctas, st);
  else if (dtype == 1)
    err = full ? by_type<__nv_bfloat16, true>(p, &ctas, st) : by_type<__nv_bfloat16, false>(p, &ctas, st);
  else
    err = full ? by_type<__half, true>(p, &ctas, st) : by_type<__half, false>(p, &ctas, st);
  if (err != cudaSuccess) return SCACCHI_ECUDA;
  g_policy_launches.fetch_add(1, std::memory_order_relaxed);
  if (ctas > 1) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(1);
    cfg.blockDim = dim3(256);
    cfg.stream = st;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    if (cudaLaunchKernelEx(&cfg, policy_loss_sum_kernel, (const double *)p.partial, ctas, p.loss) != cudaSuccess)
      return SCACCHI_ECUDA;
    g_policy_launches.fetch_add(1, std::memory_order_relaxed);
  }
  return SCACCHI_OK;
}

uint64_t scacchi_policy_loss_launch_count(void) { return g_policy_launches.load(std::memory_order_relaxed); }

}  // extern "C"
