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
// One pass: a row's logits (and reference logits) are loaded once into the
// registers of its group of threads, reduced there, and its gradient is
// written from them, so the traffic is one read per input and one write
// per output, and the kernel is bound by HBM on large batches.  Row sums
// are held in 32 bits, the log-probability is finished in 64 from them and
// the loss is summed in 64.  A row whose ratio lies within kBorderTol of a
// clip border is evaluated again in 64 bits, so the side it falls on does
// not depend on 32-bit rounding.

#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include <atomic>

#include "../../include/scacchi_b200.h"

namespace cg = cooperative_groups;

namespace {

std::atomic<uint64_t> g_policy_launches{0};

constexpr unsigned kFull = 0xffffffffu;
constexpr int kSubThreads = 256;   // CTA of the several-rows-per-warp kernel
constexpr int kMaxWarps = 16;      // CTA of the row-per-CTA kernel: 512 threads
constexpr int kMaxCluster = 16;
constexpr int kMaxSubActions = 512;
constexpr int kMaxActions = kMaxCluster * 512 * 32;
constexpr int kMaxPartials = 148 * 16;
// the 32-bit log-probability is within 3e-6 of the exact one: terms within
// 2^-24 |x - m| + 2 ulp each weighted by p (sum p |x - m| <= 13 at 2^18
// actions: 1e-6) and up to 32 rounded adds per thread plus the tree (2e-6)
constexpr double kBorderTol = 8e-6;
constexpr float kFarKl = 1.0e4f;   // sum p phi above this (KL > 9): the direct difference is exact enough

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
  int actions, group;
  double clip_low, clip_high, log_low, log_high;  // borders of the ratio and their logarithms
  float beta, even_weight;
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

// e^y - 1 - y: its Taylor series for |y| < 1 (terms to y^11, 2 / 12! of the
// leading one), the definition beyond, where it no longer cancels
__device__ __forceinline__ float phi_small(float y) {
  float c = 1.0f / 39916800.0f;
  c = fmaf(c, y, 1.0f / 3628800.0f);
  c = fmaf(c, y, 1.0f / 362880.0f);
  c = fmaf(c, y, 1.0f / 40320.0f);
  c = fmaf(c, y, 1.0f / 5040.0f);
  c = fmaf(c, y, 1.0f / 720.0f);
  c = fmaf(c, y, 1.0f / 120.0f);
  c = fmaf(c, y, 1.0f / 24.0f);
  c = fmaf(c, y, 1.0f / 6.0f);
  c = fmaf(c, y, 0.5f);
  return c * y * y;
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

// ---------------------------------------------------------------------------
// the threads of one row: G lanes of a warp, or the CTAs of a cluster
// ---------------------------------------------------------------------------

struct SumOp {
  template <typename U>
  __device__ static U apply(U a, U b) { return a + b; }
};
struct MaxOp {
  template <typename U>
  __device__ static U apply(U a, U b) { return a > b ? a : b; }
};

template <bool Cta>
struct Group;

// every lane ends with the same bits: the butterfly adds the same pairs
template <>
struct Group<false> {
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

// warp butterflies, then the warps' results of every CTA of the cluster in
// rank and warp order, which is the same for every thread
template <>
struct Group<true> {
  double *slots;  // shared: two banks of kMaxWarps partials, alternating
  int ctas, rank;
  mutable int bank;
  __device__ int index() const { return rank * blockDim.x + threadIdx.x; }
  __device__ int size() const { return ctas * blockDim.x; }
  __device__ void sync() const {
    if (ctas > 1)
      cg::this_cluster().sync();
    else
      __syncthreads();
  }
  template <typename Op, typename U>
  __device__ U reduce(U v) const {
    for (int off = 16; off; off >>= 1) v = Op::apply(v, __shfl_xor_sync(kFull, v, off));
    // a bank is written again two reductions later, and every thread has
    // passed the barrier between them, so its readers are done
    double *mine = slots + bank * kMaxWarps;
    bank ^= 1;
    if ((threadIdx.x & 31) == 0) *reinterpret_cast<U *>(mine + (threadIdx.x >> 5)) = v;
    sync();
    const int warps = blockDim.x >> 5;
    U r{};
    for (int c = 0; c < ctas; ++c) {
      const double *from = ctas > 1 ? cg::this_cluster().map_shared_rank(mine, c) : mine;
      for (int i = 0; i < warps; ++i) {
        const U u = *reinterpret_cast<const U *>(from + i);
        r = (c | i) ? Op::apply(r, u) : u;
      }
    }
    return r;
  }
};

// A row in 64 bits, read again: log sum e^x over the kept actions, and
// with `want_kl` the KL as the difference mean(x - r) - lse(x) + lse(r).
// Taken by the few rows next to a clip border or far from the reference.
template <typename T, bool Cta>
__device__ __noinline__ double2 row_in_64(const Group<Cta> &grp, const T *x, const T *r, const uint8_t *legal, int A,
                                          float top, bool want_kl) {
  double s = 0.0, sd = 0.0, rtop = -INFINITY;
  for (int a = grp.index(); a < A; a += grp.size()) {
    const float xa = to_f(x[a]);
    if ((legal && !legal[a]) || xa == -INFINITY) continue;
    const double e = exp((double)xa - (double)top);
    s += e;
    if (want_kl) {
      const double ra = to_f(r[a]);
      sd += e * ((double)xa - ra);
      rtop = ra > rtop ? ra : rtop;
    }
  }
  s = grp.template reduce<SumOp>(s);
  const double lse = (double)top + log(s);
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
    kl = sd / s - lse + rtop + log(sr);
  }
  return make_double2(lse, kl);
}

// ---------------------------------------------------------------------------
// one row
// ---------------------------------------------------------------------------

// V vectors of W elements per thread; thread t of the group holds vectors
// t, t + G, ... of the row.  Returns the row's share of the loss.
template <typename T, int W, int V, bool Kl, bool Cta>
__device__ __forceinline__ double one_row(const Params &p, const Group<Cta> &grp, int64_t row, float weight, int k) {
  const int A = p.actions, t = grp.index(), G = grp.size();
  const T *x = static_cast<const T *>(p.logits) + row * p.stride;
  const T *r = Kl ? static_cast<const T *>(p.reference) + row * p.reference_stride : nullptr;
  const uint8_t *legal = p.legal ? p.legal + row * A : nullptr;
  T *grad = p.grad ? static_cast<T *>(p.grad) + row * A : nullptr;
  bool counts = weight != 0.0f && k >= 0 && k < A;
  float xk = 0.0f;
  using Pack = Vec<T, W>;
  Pack xv[V], rv[Kl ? V : 1];
  Vec<uint8_t, W> lv[V];
  if (counts) {
    // every load of the row is issued before the first is used
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const int a = (v * G + t) * W;
      if (a < A) {
        xv[v] = *reinterpret_cast<const Pack *>(x + a);
        if (Kl) rv[Kl ? v : 0] = *reinterpret_cast<const Pack *>(r + a);
        if (legal) lv[v] = *reinterpret_cast<const Vec<uint8_t, W> *>(legal + a);
      }
    }
    xk = to_f(x[k]);
    counts = !(legal && !legal[k]) && xk != -INFINITY;
  }
  if (!counts) {
    if (t == 0) {
      p.log_prob[row] = 0.0f;
      p.clipped[row] = 0;
      if (p.kl) p.kl[row] = 0.0f;
    }
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
  // illegal actions become -inf, as places past the row are
  float top = -INFINITY;
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const bool in = (v * G + t) * W < A;
#pragma unroll
    for (int w = 0; w < W; ++w) {
      if (!in || (legal && !lv[v].v[w])) xv[v].v[w] = from_f<T>(-INFINITY);
      top = fmaxf(top, to_f(xv[v].v[w]));
    }
  }
  top = grp.template reduce<MaxOp>(top);
  float s = 0.0f, sd = 0.0f;
#pragma unroll
  for (int v = 0; v < V; ++v)
#pragma unroll
    for (int w = 0; w < W; ++w) {
      const float xa = to_f(xv[v].v[w]);
      const float e = expf(xa - top);
      s += e;
      if (Kl && xa != -INFINITY) sd = fmaf(e, xa - to_f(rv[Kl ? v : 0].v[w]), sd);
    }
  s = grp.template reduce<SumOp>(s);
  const float inv = 1.0f / s;
  double lp = ((double)xk - (double)top) - log_row_sum(s);
  float kl = 0.0f, mean = 0.0f;
  bool far = false;
  if (Kl) {
    mean = grp.template reduce<SumOp>(sd) * inv;
    float q = 0.0f;
#pragma unroll
    for (int v = 0; v < V; ++v)
#pragma unroll
      for (int w = 0; w < W; ++w) {
        const float xa = to_f(xv[v].v[w]);
        if (xa != -INFINITY) {
          const float ra = to_f(rv[Kl ? v : 0].v[w]);
          const float y = mean - (xa - ra), pa = expf(xa - top) * inv;
          // p e^y = e^{r + mu - m} / s, which cannot overflow before the KL does
          q += fabsf(y) < 1.0f ? pa * phi_small(y) : expf((ra + mean) - top) * inv - pa * (1.0f + y);
        }
      }
    q = grp.template reduce<SumOp>(q);
    far = !(q < kFarKl);
    kl = log1pf(q);
  }
  double delta = lp - (double)p.old_log_prob[row];
  if (far || fabs(delta - p.log_high) < kBorderTol || fabs(delta - p.log_low) < kBorderTol) {
    const double2 fine = row_in_64<T, Cta>(grp, x, r, legal, A, top, far);
    lp = (double)xk - fine.x;
    delta = lp - (double)p.old_log_prob[row];
    if (far) kl = (float)fine.y;
  }
  const float adv = p.advantage[row];
  const bool clipped = adv >= 0.0f ? delta > p.log_high : delta < p.log_low;
  const float ratio = expf((float)delta);
  // an advantage of 0 adds nothing, whatever the ratio overflows to
  float c = clipped || adv == 0.0f ? 0.0f : -adv * ratio;
  double term = clipped ? -(double)adv * (adv >= 0.0f ? p.clip_high : p.clip_low) : (double)c;
  if (!Kl && p.reference_log_prob) {
    const float y = (float)((double)p.reference_log_prob[row] - lp);
    const float em = expm1f(y);
    kl = fabsf(y) < 1.0f ? phi_small(y) : em - y;
    c = fmaf(-p.beta, em, c);
  }
  term += (double)p.beta * (double)kl;
  if (t == 0) {
    p.log_prob[row] = (float)lp;
    p.clipped[row] = clipped;
    if (p.kl) p.kl[row] = kl;
  }
  if (grad) {
    const float wc = weight * c, wb = weight * p.beta;
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const int a = (v * G + t) * W;
      Pack o;
#pragma unroll
      for (int w = 0; w < W; ++w) {
        const float xa = to_f(xv[v].v[w]);
        float g = -wc;
        if (Kl && xa != -INFINITY) g = fmaf(wb, (xa - to_f(rv[Kl ? v : 0].v[w])) - mean, g);
        g *= expf(xa - top) * inv;
        if (a + w == k) g += wc;
        o.v[w] = from_f<T>(xa == -INFINITY ? 0.0f : g);
      }
      if (a < A) *reinterpret_cast<Pack *>(grad + a) = o;
    }
  }
  return (double)weight * term;
}

// Several rows per warp: `group` lanes each.
template <typename T, int W, int V, bool Kl>
__global__ void __launch_bounds__(kSubThreads) policy_loss_rows_kernel(Params p) {
  __shared__ double s_part[kSubThreads / 32];
  const int lane = threadIdx.x & 31, G = p.group;
  Group<false> grp;
  grp.lanes = G;
  grp.mask = G == 32 ? kFull : ((1u << G) - 1u) << (lane & ~(G - 1));
  const int per_cta = kSubThreads / G;
  double sum = 0.0;
  int64_t row = (int64_t)blockIdx.x * per_cta + threadIdx.x / G;
  const int64_t step = (int64_t)gridDim.x * per_cta;
  // the next row's weight and action are requested a row ahead
  float w_next = 0.0f;
  int k_next = 0;
  if (row < p.rows) {
    w_next = p.weight ? p.weight[row] : p.even_weight;
    k_next = p.action[row];
  }
  for (; row < p.rows; row += step) {
    const float w = w_next;
    const int k = k_next;
    if (row + step < p.rows) {
      w_next = p.weight ? p.weight[row + step] : p.even_weight;
      k_next = p.action[row + step];
    }
    const double share = one_row<T, W, V, Kl, false>(p, grp, row, w, k);
    if (grp.index() == 0) sum += share;
  }
  __syncwarp();
  for (int off = 16; off; off >>= 1) sum += __shfl_xor_sync(kFull, sum, off);
  if (lane == 0) s_part[threadIdx.x >> 5] = sum;
  __syncthreads();
  if (threadIdx.x == 0) {
    double total = 0.0;
    for (int i = 0; i < kSubThreads / 32; ++i) total += s_part[i];
    if (gridDim.x == 1)
      p.loss[0] = (float)total;
    else
      p.partial[blockIdx.x] = total;
  }
}

// One row per CTA, or per cluster of CTAs.
template <typename T, int W, int V, bool Kl>
__global__ void __launch_bounds__(512) policy_loss_cta_kernel(Params p) {
  __shared__ double s_slots[2 * kMaxWarps];
  Group<true> grp;
  grp.slots = s_slots;
  grp.ctas = (int)cg::this_cluster().num_blocks();
  grp.rank = (int)cg::this_cluster().block_rank();
  grp.bank = 0;
  const int64_t first = blockIdx.x / grp.ctas, step = gridDim.x / grp.ctas;
  double sum = 0.0;
  for (int64_t row = first; row < p.rows; row += step) {
    const float w = p.weight ? p.weight[row] : p.even_weight;
    sum += one_row<T, W, V, Kl, true>(p, grp, row, w, p.action[row]);
  }
  if (grp.index() == 0) {
    if (step == 1)
      p.loss[0] = (float)sum;
    else
      p.partial[first] = sum;
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

int sm_count() {
  int dev = 0, n = 0;
  if (cudaGetDevice(&dev) != cudaSuccess ||
      cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n <= 0)
    return 148;
  return n;
}

template <typename T, int W, int V, bool Kl>
cudaError_t launch_rows(const Params &p, int *ctas, cudaStream_t st) {
  const int per_cta = kSubThreads / p.group;
  const int64_t need = (p.rows + per_cta - 1) / per_cta;
  const int most = sm_count() * 8 < kMaxPartials ? sm_count() * 8 : kMaxPartials;
  *ctas = (int)(need < most ? need : most);
  policy_loss_rows_kernel<T, W, V, Kl><<<*ctas, kSubThreads, 0, st>>>(p);
  return cudaPeekAtLastError();
}

template <typename T, int W, int V, bool Kl>
cudaError_t launch_cta(const Params &p, int threads, int cluster, int *ctas, cudaStream_t st) {
  const int most = sm_count() * 4 / cluster;
  const int clusters = (int)(p.rows < most ? p.rows : most);
  *ctas = clusters;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(clusters * cluster));
  cfg.blockDim = dim3((unsigned)threads);
  cfg.stream = st;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = (unsigned)cluster;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  if (cluster > 8) {
    const cudaError_t e = cudaFuncSetAttribute(policy_loss_cta_kernel<T, W, V, Kl>,
                                               cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e != cudaSuccess) return e;
  }
  return cudaLaunchKernelEx(&cfg, policy_loss_cta_kernel<T, W, V, Kl>, p);
}

// Threads per row.  Up to 512 actions a row is shared by 4 to 32 lanes of
// a warp, 4 to 16 elements each: the split with the fewest idle places,
// and among those the fewest lanes (shorter butterflies, more rows a warp).
template <typename T, int W, bool Kl>
cudaError_t by_rows(Params &p, int *ctas, cudaStream_t st) {
  int best = 0, best_elems = 4;
  for (int elems = 4; elems <= 16; elems += 4)
    for (int g = 32; g >= 4; g >>= 1) {
      const int places = g * elems;
      if (places < p.actions) continue;
      if (!best || places < best * best_elems || (places == best * best_elems && g < best)) {
        best = g;
        best_elems = elems;
      }
    }
  p.group = best;
  if (best_elems == 4) return launch_rows<T, W, 4 / W, Kl>(p, ctas, st);
  if (best_elems == 8) return launch_rows<T, W, 8 / W, Kl>(p, ctas, st);
  if (best_elems == 12) return launch_rows<T, W, 12 / W, Kl>(p, ctas, st);
  return launch_rows<T, W, 16 / W, Kl>(p, ctas, st);
}

// Longer rows: 512 threads with up to 32 elements each, and as many CTAs
// as the row needs; where the rows leave SMs idle the cluster grows to
// share them.
template <typename T, int W, bool Kl>
cudaError_t by_cta(const Params &p, int *ctas, cudaStream_t st) {
  const int64_t sms = sm_count();
  int cluster = 1;
  while (cluster < kMaxCluster && (int64_t)cluster * 512 * 32 < p.actions) cluster *= 2;
  while (cluster < kMaxCluster && p.rows * cluster * 2 <= sms && (int64_t)cluster * 512 * 4 < p.actions) cluster *= 2;
  int threads = 512;
  const int per_cta = (p.actions + cluster - 1) / cluster;
  while (threads > 128 && threads / 2 * 8 >= per_cta) threads /= 2;
  const int elems = (per_cta + threads - 1) / threads;
  if (elems <= 8) return launch_cta<T, W, 8 / W, Kl>(p, threads, cluster, ctas, st);
  if (elems <= 16) return launch_cta<T, W, 16 / W, Kl>(p, threads, cluster, ctas, st);
  return launch_cta<T, W, 32 / W, Kl>(p, threads, cluster, ctas, st);
}

// vectors of W elements need every row of every array to start on one
bool rows_aligned(const Params &p, int w, size_t size) {
  auto ok = [](const void *q, size_t bytes) { return (reinterpret_cast<uintptr_t>(q) & (bytes - 1)) == 0; };
  return p.actions % w == 0 && p.stride % w == 0 && ok(p.logits, w * size) &&
         (!p.reference || (p.reference_stride % w == 0 && ok(p.reference, w * size))) &&
         (!p.legal || ok(p.legal, (size_t)w)) && (!p.grad || ok(p.grad, w * size));
}

template <typename T, bool Kl>
cudaError_t by_type(Params &p, int *ctas, cudaStream_t st) {
  if (p.actions <= kMaxSubActions)
    return rows_aligned(p, 2, sizeof(T)) ? by_rows<T, 2, Kl>(p, ctas, st) : by_rows<T, 1, Kl>(p, ctas, st);
  constexpr int kWide = 16 / (int)sizeof(T);
  return rows_aligned(p, kWide, sizeof(T)) ? by_cta<T, kWide, Kl>(p, ctas, st) : by_cta<T, 1, Kl>(p, ctas, st);
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
