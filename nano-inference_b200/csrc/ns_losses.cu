// Operators on the logits of sampled tokens (sm_100a): token log-probabilities
// and entropies with their gradient, the clipped policy loss and the preference
// loss (include/ns_losses.h).
//
// Mathematics.  With s = log2(e) / T, m the row's largest logit and
//   t_j = (x_j - m) s,   S = sum_j 2^t_j,   U = sum_j 2^t_j t_j
// (t_j <= 0, so nothing overflows, and x_j - m is taken before the scale, so a
// row whose logits are all the type's lowest value still gets its uniform
// distribution), ln p_j = ln2 (t_j - log2 S) and the entropy is
// ln2 (log2 S - U / S).  One pass over the row keeps a running (m, S, U) per
// thread and rescales it when m rises; partial rows join by the same rule.  The
// gradient of a * logprob + h * entropy is
//   dx_j = (a 1{j = target} - p_j (a + h (ln p_j + H))) / T.
//
// Bound: HBM.  A forward reads the logits once, a gradient reads them and
// writes as many bytes.
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstring>
#include <mutex>

#include "ns_common.cuh"
#include "ns_losses.h"

namespace cg = cooperative_groups;

namespace ns {
namespace {

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxCluster = 8;
constexpr float kLog2e = 1.4426950408889634f;
constexpr double kLn2 = 0.6931471805599453;

enum Op { kLogprob = 0, kPolicy = 1, kPreference = 2 };

template <int DT>
struct Elem;
template <>
struct Elem<NS_DTYPE_F32> {
  using T = float;
  static constexpr int E = 4;                          // elements of a 16-byte vector
  static constexpr uint32_t kNegInf2 = 0xFF800000u;    // -inf in every element of a 32-bit word
  static __device__ __forceinline__ float load(const T* p) { return *p; }
  static __device__ __forceinline__ void store(T* p, float v) { *p = v; }
  static __device__ __forceinline__ void unpack(const uint4& q, float (&v)[4]) {
    v[0] = __uint_as_float(q.x), v[1] = __uint_as_float(q.y);
    v[2] = __uint_as_float(q.z), v[3] = __uint_as_float(q.w);
  }
  static __device__ __forceinline__ uint4 pack(const float (&v)[4]) {
    return make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
  }
};
template <>
struct Elem<NS_DTYPE_BF16> {
  using T = __nv_bfloat16;
  static constexpr int E = 8;
  static constexpr uint32_t kNegInf2 = 0xFF80FF80u;
  static __device__ __forceinline__ float load(const T* p) { return __bfloat162float(*p); }
  static __device__ __forceinline__ void store(T* p, float v) { *p = __float2bfloat16_rn(v); }
  static __device__ __forceinline__ void unpack(const uint4& q, float (&v)[8]) {
    const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = __uint_as_float(w[i] << 16);
      v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
    }
  }
  static __device__ __forceinline__ uint4 pack(const float (&v)[8]) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __nv_bfloat162 b = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
      memcpy(&w[i], &b, 4);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
};
template <>
struct Elem<NS_DTYPE_F16> {
  using T = __half;
  static constexpr int E = 8;
  static constexpr uint32_t kNegInf2 = 0xFC00FC00u;
  static __device__ __forceinline__ float load(const T* p) { return __half2float(*p); }
  static __device__ __forceinline__ void store(T* p, float v) { *p = __float2half_rn(v); }
  static __device__ __forceinline__ void unpack(const uint4& q, float (&v)[8]) {
    const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      __half2 h;
      memcpy(&h, &w[i], 4);
      const float2 f = __half22float2(h);
      v[2 * i] = f.x;
      v[2 * i + 1] = f.y;
    }
  }
  static __device__ __forceinline__ uint4 pack(const float (&v)[8]) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __half2 h = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
      memcpy(&w[i], &h, 4);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
};

struct LossArgs {
  const void* logits;
  int64_t rows, vocab, row_stride;
  const int64_t* targets;
  const float* temperature;
  float temperature_all;
  // forward results
  float *logprobs, *entropy, *stats;
  // policy
  const float *old_logprobs, *ref_logprobs, *advantages, *weights;
  float clip_low, clip_high, kl_coef, entropy_coef;
  float *row_loss, *kl, *row_grad;
  // preference
  const int64_t* seq_offsets;
  int64_t pairs;
  // gradient
  const float *grad_logprobs, *grad_entropy;
  void* grad_logits;
  int64_t grad_stride;
};

// The row's scale log2(e) / T and 1 / T; NaN for a temperature that gives no
// distribution.  0 stands for 1.  A denormal T would make the scale infinite
// and 0 * inf of the largest logit NaN, so it stops at the largest float.
__device__ __forceinline__ void row_scale(const LossArgs& a, int64_t row, float& s, double& inv_t) {
  float t = a.temperature ? a.temperature[row] : a.temperature_all;
  if (t == 0.0f) t = 1.0f;
  const bool ok = t > 0.0f && t < INFINITY;
  s = ok ? fminf(kLog2e / t, 3.402823466e38f) : NAN;
  inv_t = ok ? 1.0 / double(t) : double(NAN);
}

// Running (m, S, U) of a part of a row.  m = -inf: nothing but -inf so far.
struct Part {
  float m, s, u;
};

// The part rescaled to a largest logit of m >= p.m.
template <bool ENT>
__device__ __forceinline__ void rescale(Part& p, float m, float scale) {
  if (p.m == m) return;
  // 2^d is 0 from -200 on; d itself may be -inf (nothing summed yet, or a
  // distance that overflows), and 0 * -inf is not 0
  const float d = fmaxf((p.m - m) * scale, -200.0f);
  const float f = ex2_approx(d);
  if (ENT) p.u = f * fmaf(d, p.s, p.u);
  p.s *= f;
  p.m = m;
}

// Adds N values to the part: one comparison of their maximum, one exponential each.
template <bool ENT, int N>
__device__ __forceinline__ void add(Part& p, const float (&x)[N], float scale) {
  float top = x[0];
#pragma unroll
  for (int i = 1; i < N; ++i) top = fmaxf(top, x[i]);
  if (top > p.m) rescale<ENT>(p, top, scale);
  const float m = p.m == -INFINITY ? 0.0f : p.m;   // -inf - -inf would be NaN
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const float t = (x[i] - m) * scale;
    const float e = ex2_approx(t);
    p.s += e;
    // t is held above -200, where e is 0, so that 0 * -inf does not arise; a
    // NaN t has made e and S NaN
    if (ENT) p.u = fmaf(e, fmaxf(t, -200.0f), p.u);
  }
}

template <bool ENT>
__device__ __forceinline__ Part warp_join(Part p, float scale) {
  float m = p.m;
#pragma unroll
  for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(~0u, m, o));
  rescale<ENT>(p, m, scale);
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    p.s += __shfl_xor_sync(~0u, p.s, o);
    if (ENT) p.u += __shfl_xor_sync(~0u, p.u, o);
  }
  return p;
}

// The vectors of a row: `head` elements before the first 16-byte boundary, nv
// whole vectors, then the rest.
struct Span {
  int64_t head, nv;
};
template <int E>
__device__ __forceinline__ Span row_span(const void* row, int64_t vocab) {
  const int64_t head = min(vocab, int64_t((16 - (reinterpret_cast<uintptr_t>(row) & 15)) & 15) / (16 / E));
  return {head, (vocab - head) / E};
}

// Block `rank` of `blocks` adds its share of the row; every thread returns the block's part.
template <int DT, bool ENT>
__device__ __forceinline__ Part block_part(const void* base, int64_t vocab, float scale, int rank, int blocks,
                                           Part* shared) {
  using D = Elem<DT>;
  using T = typename D::T;
  constexpr int E = D::E, U = 4;
  const T* row = static_cast<const T*>(base);
  const Span sp = row_span<E>(row, vocab);
  const int64_t v0 = sp.nv * rank / blocks, v1 = sp.nv * (rank + 1) / blocks;
  const uint4* vec = reinterpret_cast<const uint4*>(row + sp.head);
  Part p = {-INFINITY, 0.0f, 0.0f};
  for (int64_t v = v0 + threadIdx.x; v < v1; v += U * kThreads) {
    uint4 q[U];
#pragma unroll
    for (int k = 0; k < U; ++k) {
      const int64_t at = v + k * kThreads;
      q[k] = at < v1 ? vec[at] : make_uint4(D::kNegInf2, D::kNegInf2, D::kNegInf2, D::kNegInf2);
    }
#pragma unroll
    for (int k = 0; k < U; ++k) {
      float x[E];
      D::unpack(q[k], x);
      add<ENT>(p, x, scale);
    }
  }
  if (rank == 0 && threadIdx.x < sp.head) {
    const float x[1] = {D::load(row + threadIdx.x)};
    add<ENT>(p, x, scale);
  }
  const int64_t tail = sp.head + sp.nv * E + threadIdx.x;
  if (rank == blocks - 1 && tail < vocab) {
    const float x[1] = {D::load(row + tail)};
    add<ENT>(p, x, scale);
  }
  p = warp_join<ENT>(p, scale);
  if ((threadIdx.x & 31) == 0) shared[threadIdx.x >> 5] = p;
  __syncthreads();
  const int lane = threadIdx.x & 31;
  p = lane < kWarps ? shared[lane] : Part{-INFINITY, 0.0f, 0.0f};
  return warp_join<ENT>(p, scale);
}

// What a row's (m, S, U) and target give.  Sums are taken in 64 bits, so that
// differences from a reference's log-probability keep their digits; the
// logarithm is split as exponent * ln2 + ln(mantissa), whose second part lies
// in [0, ln2) and is exact to 2^-25.
struct RowResult {
  double logprob;
  float entropy, log2s;
};
template <bool ENT>
__device__ __forceinline__ RowResult finish(const Part& p, float x_target, double inv_t) {
  int ex;
  const float mant = 2.0f * frexpf(p.s, &ex);       // S >= 1 for a row with a distribution
  const double ln_s = p.s < INFINITY && p.s > 0.0f ? double(ex - 1) * kLn2 + double(logf(mant)) : double(NAN);
  RowResult r;
  r.logprob = (double(x_target) - double(p.m)) * inv_t - ln_s;
  r.log2s = float(ln_s / kLn2);
  r.entropy = ENT ? float(ln_s - kLn2 * double(p.u) / double(p.s)) : 0.0f;
  if (!isfinite(inv_t)) r.logprob = NAN;
  return r;
}

struct PolicyRow {
  float loss, kl, a, h;
};
__device__ __forceinline__ PolicyRow policy_row(const LossArgs& a, int64_t row, double logprob, float entropy, float w) {
  const float adv = a.advantages[row];
  const float ratio = expf(float(logprob - double(a.old_logprobs[row])));
  const float inside = ratio * adv;
  const float clipped = fminf(fmaxf(ratio, 1.0f - a.clip_low), 1.0f + a.clip_high) * adv;
  PolicyRow r = {0.0f, 0.0f, 0.0f, 0.0f};
  // fmin drops a NaN, so the comparison keeps it; without an advantage there is no term (0 * inf is NaN)
  if (adv != 0.0f || isnan(ratio)) {
    r.loss = -(clipped < inside ? clipped : inside);
    r.a = clipped < inside ? 0.0f : -inside;
  }
  if (a.ref_logprobs) {
    const float d = float(double(a.ref_logprobs[row]) - logprob);
    const float g = expm1f(d);
    r.kl = g - d;
    if (a.kl_coef != 0.0f) {
      r.loss = fmaf(a.kl_coef, r.kl, r.loss);
      r.a = fmaf(-a.kl_coef, g, r.a);
    }
  }
  if (a.entropy_coef != 0.0f) {
    r.loss = fmaf(-a.entropy_coef, entropy, r.loss);
    r.h = -a.entropy_coef * w;
  }
  r.a *= w;
  return r;
}

// Whether the row holds a token, by operator.
template <int OP>
__device__ __forceinline__ bool row_alive(const LossArgs& a, int64_t row, float& w) {
  w = 1.0f;
  if (a.targets[row] < 0) return false;
  if (OP == kPolicy) {
    w = a.weights ? a.weights[row] : 1.0f / float(a.rows);
    return w != 0.0f;
  }
  if (OP == kPreference) return row >= a.seq_offsets[0] && row < a.seq_offsets[2 * a.pairs];
  return true;
}

// One cluster of blocks per row.
template <int DT, bool ENT, int OP>
__global__ void __launch_bounds__(kThreads) forward_kernel(const LossArgs a) {
  using D = Elem<DT>;
  using T = typename D::T;
  __shared__ Part warp_parts[kWarps];
  __shared__ Part block_parts[kMaxCluster];
  cg::cluster_group cluster = cg::this_cluster();
  const int blocks = int(cluster.num_blocks()), rank = int(cluster.block_rank());
  const int64_t row = blockIdx.x / blocks;
  float w;
  const bool alive = row_alive<OP>(a, row, w);
  if (!alive) {            // the same for every block of the cluster
    if (rank == 0 && threadIdx.x == 0) {
      a.logprobs[row] = 0.0f;
      if (a.entropy) a.entropy[row] = 0.0f;
      if (a.stats) a.stats[2 * row] = a.stats[2 * row + 1] = 0.0f;
      if (OP == kPolicy) {
        a.row_loss[row] = 0.0f;
        if (a.kl) a.kl[row] = 0.0f;
        a.row_grad[row] = a.row_grad[a.rows + row] = 0.0f;
      }
      if (OP == kPreference) a.row_grad[row] = 0.0f;
    }
    return;
  }
  float scale;
  double inv_t;
  row_scale(a, row, scale, inv_t);
  const T* x = static_cast<const T*>(a.logits) + row * a.row_stride;
  const int64_t target = a.targets[row];
  const float x_target = target < a.vocab ? D::load(x + target) : NAN;
  Part p = block_part<DT, ENT>(x, a.vocab, scale, rank, blocks, warp_parts);
  if (blocks > 1) {
    if (threadIdx.x == 0) *cluster.map_shared_rank(&block_parts[rank], 0) = p;
    cluster.sync();
    if (rank == 0) {
      const int lane = threadIdx.x & 31;
      p = lane < blocks ? block_parts[lane] : Part{-INFINITY, 0.0f, 0.0f};
      p = warp_join<ENT>(p, scale);
    }
  }
  if (rank != 0 || threadIdx.x != 0) return;
  const RowResult r = finish<ENT>(p, x_target, inv_t);
  a.logprobs[row] = float(r.logprob);
  if (ENT) a.entropy[row] = isnan(r.logprob) ? NAN : r.entropy;
  if (a.stats) {
    a.stats[2 * row] = p.m;
    a.stats[2 * row + 1] = isnan(r.logprob) ? NAN : r.log2s;
  }
  if (OP == kPolicy) {
    const PolicyRow l = policy_row(a, row, r.logprob, r.entropy, w);
    a.row_loss[row] = l.loss;
    if (a.kl) a.kl[row] = l.kl;
    a.row_grad[row] = l.a;
    a.row_grad[a.rows + row] = l.h;
  }
  if (OP == kPreference)   // the row's gain; the pair kernel turns it into the coefficient
    a.row_grad[row] = float(r.logprob - (a.ref_logprobs ? double(a.ref_logprobs[row]) : 0.0));
}

__device__ __forceinline__ double block_sum(double v, double* shared) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
  if ((threadIdx.x & 31) == 0) shared[threadIdx.x >> 5] = v;
  __syncthreads();
  const int lane = threadIdx.x & 31;
  v = lane < int(blockDim.x / 32) ? shared[lane] : 0.0;
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
  return v;
}

// The policy loss: the rows' losses by their weights, in 64 bits and in one order.
__global__ void __launch_bounds__(1024) policy_sum_kernel(const LossArgs a, float* loss) {
  __shared__ double shared[32];
  double v = 0.0;
  for (int64_t i = threadIdx.x; i < a.rows; i += 1024) {
    const double w = a.weights ? double(a.weights[i]) : 1.0 / double(a.rows);
    if (a.targets[i] >= 0 && w != 0.0) v += w * double(a.row_loss[i]);
  }
  v = block_sum(v, shared);
  if (threadIdx.x == 0) *loss = float(v);
}

// The pairs: one warp sums a sequence's gains, then the pair's loss, and the
// rows' coefficients over the gains.
__global__ void __launch_bounds__(1024) pair_kernel(const LossArgs a, float beta, float smoothing, int average,
                                                    float* loss, float* pair_loss, float* rewards) {
  __shared__ double shared[32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  double total = 0.0;
  for (int64_t p = warp; p < a.pairs; p += 32) {
    int64_t lo[2], hi[2];
    double reward[2], share[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      lo[k] = max(a.seq_offsets[2 * p + k], int64_t(0));
      hi[k] = min(a.seq_offsets[2 * p + k + 1], a.rows);
      double sum = 0.0;
      int64_t count = 0;
      for (int64_t i = lo[k] + lane; i < hi[k]; i += 32) {
        sum += double(a.row_grad[i]);
        count += a.targets[i] >= 0;
      }
#pragma unroll
      for (int o = 16; o; o >>= 1) {
        sum += __shfl_xor_sync(~0u, sum, o);
        count += __shfl_xor_sync(~0u, count, o);
      }
      share[k] = average ? 1.0 / double(max(count, int64_t(1))) : 1.0;
      reward[k] = double(beta) * sum * share[k];
    }
    const double h = reward[0] - reward[1];
    // ln sigmoid(h) = min(h, 0) - ln(1 + exp(-|h|)), and the same with -h
    const float tail = log1pf(expf(-fabsf(float(h))));
    const double win = fmin(h, 0.0) - double(tail), lose = fmin(-h, 0.0) - double(tail);
    const double e = double(smoothing);
    const double l = isnan(h) ? h : -(1.0 - e) * win - e * lose;
    const double up = 1.0 / (1.0 + double(expf(float(-h)))), down = 1.0 / (1.0 + double(expf(float(h))));
    const double slope = (e * up - (1.0 - e) * down) * double(beta) / double(a.pairs);
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const float c = float((k ? -slope : slope) * share[k]);
      for (int64_t i = lo[k] + lane; i < hi[k]; i += 32) a.row_grad[i] = a.targets[i] >= 0 ? c : 0.0f;
    }
    if (lane == 0) {
      pair_loss[p] = float(l);
      rewards[2 * p] = float(reward[0]);
      rewards[2 * p + 1] = float(reward[1]);
      total += l;
    }
  }
  total = block_sum(total, shared);
  if (threadIdx.x == 0) *loss = a.pairs ? float(total / double(a.pairs)) : 0.0f;
}

// Gradient of one value: g = -p (A + B t') with t' = log2 p.
struct GradRow {
  float m, log2s, scale, ca, cb, at;   // at: added at the target
  int64_t target;
};
template <bool ENT>
__device__ __forceinline__ float grad_value(const GradRow& g, float x) {
  const float t = fmaf(x - g.m, g.scale, -g.log2s);
  const float p = ex2_approx(t);
  return ENT ? -p * fmaf(g.cb, fmaxf(t, -200.0f), g.ca) : -p * g.ca;
}

constexpr int kGradVecs = 8;    // vectors of a thread

// One block per (row, chunk of 512 x 8 vectors).
template <int DT, bool ENT>
__global__ void __launch_bounds__(kThreads) grad_kernel(const LossArgs a, int chunks) {
  using D = Elem<DT>;
  using T = typename D::T;
  constexpr int E = D::E;
  const int64_t row = blockIdx.x / chunks;
  const int chunk = int(blockIdx.x % chunks);
  const T* x = static_cast<const T*>(a.logits) + row * a.row_stride;
  T* out = static_cast<T*>(a.grad_logits) + row * a.grad_stride;
  const float ga = a.grad_logprobs ? a.grad_logprobs[row] : 0.0f;
  const float gh = ENT ? a.grad_entropy[row] : 0.0f;
  const bool zero = a.targets[row] < 0 || (ga == 0.0f && gh == 0.0f);
  GradRow g = {};
  if (!zero) {
    double inv_t;
    row_scale(a, row, g.scale, inv_t);
    g.m = a.stats[2 * row];
    if (g.m == -INFINITY) g.m = 0.0f;        // no distribution: log2 S is NaN
    g.log2s = a.stats[2 * row + 1];
    g.target = a.targets[row];
    g.at = float(double(ga) * inv_t);
    g.ca = float((double(ga) + (ENT ? double(gh) * double(a.entropy[row]) : 0.0)) * inv_t);
    g.cb = ENT ? float(double(gh) * kLn2 * inv_t) : 0.0f;
  }
  const Span sp = row_span<E>(out, a.vocab);
  if (((reinterpret_cast<uintptr_t>(x) ^ reinterpret_cast<uintptr_t>(out)) & 15) != 0) {
    // the rows start on different 16-byte phases: element by element
    const int64_t per = int64_t(kThreads) * kGradVecs * E;
    const int64_t end = min(a.vocab, (chunk + 1) * per);
    for (int64_t j = chunk * per + threadIdx.x; j < end; j += kThreads) {
      float v = 0.0f;
      if (!zero) {
        v = grad_value<ENT>(g, D::load(x + j));
        if (j == g.target) v += g.at;
      }
      D::store(out + j, v);
    }
    return;
  }
  const uint4* src = reinterpret_cast<const uint4*>(x + sp.head);
  uint4* dst = reinterpret_cast<uint4*>(out + sp.head);
  const int64_t base = int64_t(chunk) * kThreads * kGradVecs + threadIdx.x;
  if (zero) {
#pragma unroll
    for (int k = 0; k < kGradVecs; ++k)
      if (base + k * kThreads < sp.nv) dst[base + k * kThreads] = make_uint4(0, 0, 0, 0);
  } else {
    uint4 q[kGradVecs];
#pragma unroll
    for (int k = 0; k < kGradVecs; ++k)
      if (base + k * kThreads < sp.nv) q[k] = src[base + k * kThreads];
#pragma unroll
    for (int k = 0; k < kGradVecs; ++k) {
      const int64_t v = base + k * kThreads;
      if (v >= sp.nv) continue;
      float f[E];
      D::unpack(q[k], f);
#pragma unroll
      for (int i = 0; i < E; ++i) f[i] = grad_value<ENT>(g, f[i]);
      const int64_t j = g.target - (sp.head + v * E);
      if (uint64_t(j) < uint64_t(E)) {
#pragma unroll
        for (int i = 0; i < E; ++i)
          if (i == int(j)) f[i] += g.at;
      }
      dst[v] = D::pack(f);
    }
  }
  if (chunk == 0) {     // the elements before the first whole vector and after the last
    const int64_t rest = sp.head + sp.nv * E, edge = sp.head + (a.vocab - rest);
    if (threadIdx.x < edge) {
      const int64_t j = threadIdx.x < sp.head ? threadIdx.x : rest + (threadIdx.x - sp.head);
      float v = 0.0f;
      if (!zero) {
        v = grad_value<ENT>(g, D::load(x + j));
        if (j == g.target) v += g.at;
      }
      D::store(out + j, v);
    }
  }
}

// ---------------------------------------------------------------------------
// launches
// ---------------------------------------------------------------------------
int sm_count(int* out) {
  static std::mutex mu;
  static int sms[64];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return NS_ERR_CUDA;
  std::lock_guard<std::mutex> lk(mu);
  if (sms[dev] == 0 && cudaDeviceGetAttribute(&sms[dev], cudaDevAttrMultiProcessorCount, dev) != cudaSuccess)
    return NS_ERR_CUDA;
  *out = sms[dev];
  return NS_OK;
}

template <int DT, bool ENT, int OP>
int launch_forward(const LossArgs& a, cudaStream_t stream) {
  int sms = 0;
  if (const int rc = sm_count(&sms)) return rc;
  // blocks per row: enough to give every SM two, each thread at least one vector
  int blocks = 1;
  while (blocks < kMaxCluster && a.rows * blocks < 2 * sms && a.vocab >= int64_t(2) * blocks * kThreads * Elem<DT>::E)
    blocks *= 2;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(unsigned(a.rows * blocks));
  cfg.blockDim = dim3(kThreads);
  cfg.stream = stream;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = unsigned(blocks);
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, forward_kernel<DT, ENT, OP>, a) == cudaSuccess ? NS_OK : NS_ERR_CUDA;
}

template <int OP>
int forward(const LossArgs& a, int dtype, cudaStream_t stream) {
  const bool ent = a.entropy != nullptr;
  switch (dtype) {
    case NS_DTYPE_F32:
      return ent ? launch_forward<NS_DTYPE_F32, true, OP>(a, stream) : launch_forward<NS_DTYPE_F32, false, OP>(a, stream);
    case NS_DTYPE_BF16:
      return ent ? launch_forward<NS_DTYPE_BF16, true, OP>(a, stream) : launch_forward<NS_DTYPE_BF16, false, OP>(a, stream);
    default:
      return ent ? launch_forward<NS_DTYPE_F16, true, OP>(a, stream) : launch_forward<NS_DTYPE_F16, false, OP>(a, stream);
  }
}

template <int DT>
int launch_grad(const LossArgs& a, cudaStream_t stream) {
  const int64_t per = int64_t(kThreads) * kGradVecs * Elem<DT>::E;
  const int chunks = int((a.vocab + per - 1) / per);
  const int64_t blocks = a.rows * chunks;
  if (blocks > 0x7FFFFFFF) return NS_ERR_INVALID_ARGUMENT;
  if (a.grad_entropy)
    grad_kernel<DT, true><<<unsigned(blocks), kThreads, 0, stream>>>(a, chunks);
  else
    grad_kernel<DT, false><<<unsigned(blocks), kThreads, 0, stream>>>(a, chunks);
  return cudaGetLastError() == cudaSuccess ? NS_OK : NS_ERR_CUDA;
}

int gradient(const LossArgs& a, int dtype, cudaStream_t stream) {
  switch (dtype) {
    case NS_DTYPE_F32: return launch_grad<NS_DTYPE_F32>(a, stream);
    case NS_DTYPE_BF16: return launch_grad<NS_DTYPE_BF16>(a, stream);
    default: return launch_grad<NS_DTYPE_F16>(a, stream);
  }
}

bool temperature_ok(const float* temperature, float all) { return temperature || (all >= 0.0f && all < INFINITY); }

int check_rows(int dtype, int64_t rows, int64_t vocab, int64_t row_stride, const float* temperature, float all) {
  if (dtype != NS_DTYPE_F32 && dtype != NS_DTYPE_BF16 && dtype != NS_DTYPE_F16) return NS_ERR_UNSUPPORTED_DTYPE;
  if (rows < 0 || vocab <= 0 || row_stride < vocab) return NS_ERR_INVALID_ARGUMENT;
  if (vocab > (int64_t(1) << 24) || rows > (int64_t(1) << 24)) return NS_ERR_INVALID_ARGUMENT;
  return temperature_ok(temperature, all) ? NS_OK : NS_ERR_INVALID_ARGUMENT;
}

LossArgs row_args(const void* logits, int64_t rows, int64_t vocab, int64_t row_stride, const int64_t* targets,
                  const float* temperature, float temperature_all) {
  LossArgs a = {};
  a.logits = logits;
  a.rows = rows;
  a.vocab = vocab;
  a.row_stride = row_stride;
  a.targets = targets;
  a.temperature = temperature;
  a.temperature_all = temperature_all;
  return a;
}

// A gradient that takes the logits' place has their stride.
bool grad_ok(const void* logits, int64_t row_stride, const void* grad, int64_t grad_stride, int64_t vocab) {
  return grad_stride >= vocab && (grad != logits || grad_stride == row_stride);
}

}  // namespace
}  // namespace ns

extern "C" {

int ns_token_logprobs(const void* logits, int dtype, int64_t rows, int64_t vocab, int64_t row_stride,
                      const int64_t* targets, const float* temperature, float temperature_all, float* logprobs,
                      float* entropy, float* stats, ns_stream_t stream) {
  if (const int rc = ns::check_rows(dtype, rows, vocab, row_stride, temperature, temperature_all)) return rc;
  if (rows == 0) return NS_OK;
  if (!logits || !targets || !logprobs) return NS_ERR_INVALID_ARGUMENT;
  ns::LossArgs a = ns::row_args(logits, rows, vocab, row_stride, targets, temperature, temperature_all);
  a.logprobs = logprobs;
  a.entropy = entropy;
  a.stats = stats;
  return ns::forward<ns::kLogprob>(a, dtype, reinterpret_cast<cudaStream_t>(stream));
}

int ns_token_logprobs_grad(const void* logits, int dtype, int64_t rows, int64_t vocab, int64_t row_stride,
                           const int64_t* targets, const float* temperature, float temperature_all,
                           const float* stats, const float* entropy, const float* grad_logprobs,
                           const float* grad_entropy, void* grad_logits, int64_t grad_stride, ns_stream_t stream) {
  if (const int rc = ns::check_rows(dtype, rows, vocab, row_stride, temperature, temperature_all)) return rc;
  if (grad_stride < vocab) return NS_ERR_INVALID_ARGUMENT;
  if (rows == 0) return NS_OK;
  if (!logits || !targets || !stats || !grad_logits || (grad_entropy && !entropy)) return NS_ERR_INVALID_ARGUMENT;
  if (!ns::grad_ok(logits, row_stride, grad_logits, grad_stride, vocab)) return NS_ERR_INVALID_ARGUMENT;
  ns::LossArgs a = ns::row_args(logits, rows, vocab, row_stride, targets, temperature, temperature_all);
  a.stats = const_cast<float*>(stats);
  a.entropy = const_cast<float*>(entropy);
  a.grad_logprobs = grad_logprobs;
  a.grad_entropy = grad_entropy;
  a.grad_logits = grad_logits;
  a.grad_stride = grad_stride;
  return ns::gradient(a, dtype, reinterpret_cast<cudaStream_t>(stream));
}

int ns_policy_loss(const void* logits, int dtype, int64_t rows, int64_t vocab, int64_t row_stride,
                   const int64_t* targets, const float* temperature, float temperature_all,
                   const float* old_logprobs, const float* ref_logprobs, const float* advantages,
                   const float* weights, float clip_low, float clip_high, float kl_coef, float entropy_coef,
                   float* loss, float* row_loss, float* logprobs, float* entropy, float* kl, float* stats,
                   float* row_grad, void* grad_logits, int64_t grad_stride, ns_stream_t stream) {
  if (const int rc = ns::check_rows(dtype, rows, vocab, row_stride, temperature, temperature_all)) return rc;
  if (!(clip_low >= 0.0f && clip_low <= 1.0f) || !(clip_high >= 0.0f && clip_high < INFINITY) ||
      !std::isfinite(kl_coef) || !std::isfinite(entropy_coef))
    return NS_ERR_INVALID_ARGUMENT;
  if (!loss || (grad_logits && grad_stride < vocab)) return NS_ERR_INVALID_ARGUMENT;
  const cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (rows == 0) return cudaMemsetAsync(loss, 0, sizeof(float), s) == cudaSuccess ? NS_OK : NS_ERR_CUDA;
  if (!logits || !targets || !old_logprobs || !advantages || !row_loss || !logprobs || !stats || !row_grad)
    return NS_ERR_INVALID_ARGUMENT;
  if ((kl_coef != 0.0f || kl) && !ref_logprobs) return NS_ERR_INVALID_ARGUMENT;
  if (entropy_coef != 0.0f && !entropy) return NS_ERR_INVALID_ARGUMENT;
  if (grad_logits && !ns::grad_ok(logits, row_stride, grad_logits, grad_stride, vocab)) return NS_ERR_INVALID_ARGUMENT;
  ns::LossArgs a = ns::row_args(logits, rows, vocab, row_stride, targets, temperature, temperature_all);
  a.logprobs = logprobs;
  a.entropy = entropy;
  a.stats = stats;
  a.old_logprobs = old_logprobs;
  a.ref_logprobs = ref_logprobs;
  a.advantages = advantages;
  a.weights = weights;
  a.clip_low = clip_low;
  a.clip_high = clip_high;
  a.kl_coef = kl_coef;
  a.entropy_coef = entropy_coef;
  a.row_loss = row_loss;
  a.kl = kl;
  a.row_grad = row_grad;
  if (const int rc = ns::forward<ns::kPolicy>(a, dtype, s)) return rc;
  ns::policy_sum_kernel<<<1, 1024, 0, s>>>(a, loss);
  if (cudaGetLastError() != cudaSuccess) return NS_ERR_CUDA;
  if (!grad_logits) return NS_OK;
  a.grad_logprobs = row_grad;
  a.grad_entropy = entropy_coef != 0.0f ? row_grad + rows : nullptr;
  a.grad_logits = grad_logits;
  a.grad_stride = grad_stride;
  return ns::gradient(a, dtype, s);
}

int ns_preference_loss(const void* logits, int dtype, int64_t rows, int64_t vocab, int64_t row_stride,
                       const int64_t* targets, const float* temperature, float temperature_all,
                       const int64_t* seq_offsets, int64_t pairs, const float* ref_logprobs, float beta,
                       float label_smoothing, int average, float* loss, float* pair_loss, float* rewards,
                       float* logprobs, float* stats, float* row_grad, void* grad_logits, int64_t grad_stride,
                       ns_stream_t stream) {
  if (const int rc = ns::check_rows(dtype, rows, vocab, row_stride, temperature, temperature_all)) return rc;
  if (!std::isfinite(beta) || !(label_smoothing >= 0.0f && label_smoothing < 1.0f) || pairs < 0 ||
      pairs > (int64_t(1) << 24))
    return NS_ERR_INVALID_ARGUMENT;
  if (!loss || !seq_offsets || (pairs > 0 && (!pair_loss || !rewards)) || (grad_logits && grad_stride < vocab))
    return NS_ERR_INVALID_ARGUMENT;
  const cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (rows > 0) {
    if (!logits || !targets || !logprobs || !stats || !row_grad) return NS_ERR_INVALID_ARGUMENT;
    if (grad_logits && !ns::grad_ok(logits, row_stride, grad_logits, grad_stride, vocab)) return NS_ERR_INVALID_ARGUMENT;
  }
  ns::LossArgs a = ns::row_args(logits, rows, vocab, row_stride, targets, temperature, temperature_all);
  a.logprobs = logprobs;
  a.stats = stats;
  a.ref_logprobs = ref_logprobs;
  a.row_grad = row_grad;
  a.seq_offsets = seq_offsets;
  a.pairs = pairs;
  if (rows > 0)
    if (const int rc = ns::forward<ns::kPreference>(a, dtype, s)) return rc;
  ns::pair_kernel<<<1, 1024, 0, s>>>(a, beta, label_smoothing, average, loss, pair_loss, rewards);
  if (cudaGetLastError() != cudaSuccess) return NS_ERR_CUDA;
  if (!grad_logits || rows == 0) return NS_OK;
  a.grad_logprobs = row_grad;
  a.grad_logits = grad_logits;
  a.grad_stride = grad_stride;
  return ns::gradient(a, dtype, s);
}

}  // extern "C"
