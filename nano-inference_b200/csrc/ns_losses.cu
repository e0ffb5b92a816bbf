// Operators on the logits of sampled tokens (sm_100a): token log-probabilities
// and entropies with their gradient, the clipped policy loss and the preference
// loss (include/ns_losses.h).
//
// Mathematics.  With s = log2(e) / T, c the target's logit and
//   t_j = (x_j - c) s,   S = sum_j 2^t_j,   U = sum_j 2^t_j t_j,
// ln p_j = ln2 (t_j - log2 S), so the target's log-probability is -ln S, and
// the entropy is ln2 (log2 S - U / S).  Any offset near the row's largest logit
// would do in fp32; the target's is known before the row is read and is the
// same for every thread and block of the row, so no maximum is kept and no sum
// is ever rescaled: the exponential's error enters once.  A row whose S leaves
// [2^-60, 2^100] (a target less likely than 2^-100, or barred), or whose entropy
// is less than a 256th of |ln S|, is added up again with a running maximum;
// there, and for fp32 always, the difference is taken before the scale, so a row
// whose logits are all the type's lowest value still gets its uniform
// distribution.  The gradient of a * logprob + h * entropy is
//   dx_j = (a 1{j = target} - p_j (a + h (ln p_j + H))) / T.
//
// Bound: HBM.  A forward reads the logits once, a gradient reads them and
// writes as many bytes; the policy loss keeps a row on chip between its sums
// and its gradient, and reads it once.  Measured, us and share of the 6554 GB/s
// that a copy reaches (calls in one graph):
//   forward   2048 x 151936 bf16 95 (1.00)    600 x 151936 fp32 56 (1.00)    2048 x 32000 bf16 28 (0.72)
//   gradient  2048 x 151936 bf16 191 (0.99)   600 x 151936 fp32 110 (1.01)   2048 x 32000 bf16 43 (0.92)
//   policy    2048 x 151936 bf16 212 (0.90)   600 x 151936 fp32 124 (0.90)   2048 x 32000 bf16 55 (0.73)
// and with entropies 97, 57, 29 (forward), 194, 111, 44 (gradient), 229, 130, 58 (policy).
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

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxCluster = 8;
constexpr int kBatch = 2;          // 16-byte loads that a thread of a forward issues ahead of its sums; 4 and 8 were no faster
constexpr float kLog2e = 1.4426950408889634f;
constexpr double kLn2 = 0.6931471805599453;
// Mean relative error of ex2.approx.ftz.f32, measured over 4 M arguments an interval: -5.0e-8 from -30 to -1, -2.2e-8
// from -1 to 0, 0.6e-8 from 0 to 1, 3.3e-8 from 1 to 32.  The target of a draw has half of the row's mass above it on
// average, so S is low by half the sum of the outer two; a row whose mass is all on one side is 4.2e-8 away from that.
// Log-probabilities of drawn targets are then off by 0.2e-8 on average (600 rows of 151936), where the error of the
// negative arguments alone gave -3.3e-8.
constexpr double kEx2Mean = 0.85e-8;

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

// Two fp32 values in a 64-bit register: one instruction for both.
using F2 = unsigned long long;
__device__ __forceinline__ F2 f2(float lo, float hi) {
  F2 d;
  asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(lo), "f"(hi));
  return d;
}
__device__ __forceinline__ void split(F2 v, float& lo, float& hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v)); }
__device__ __forceinline__ F2 add2(F2 a, F2 b) {
  F2 d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ F2 mul2(F2 a, F2 b) {
  F2 d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
  F2 d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}

// t = (x - c) s for pairs of logits.  fp32: difference, then product.  16-bit
// logits: one multiply-add x s - fl(c s); the rounding of c s moves every t of
// the row alike and is taken into account exactly, as is that of the gradient's
// offset c s + log2 S.  Rows whose |c s| is not below kNearOffset, where that is
// at most 2^-14, are added up around 0, most of them in vain, and go the way of
// `sums_far`: they are cold (|logit| / T past 710).
constexpr float kNearOffset = 1024.0f;
template <int DT>
struct ScaledPairs {
  F2 a, b;
  static __device__ __forceinline__ ScaledPairs of(float c, float scale) {
    if constexpr (DT == NS_DTYPE_F32) return {f2(-c, -c), f2(scale, scale)};
    const float off = -__fmul_rn(c, scale);
    return {f2(scale, scale), f2(off, off)};
  }
  __device__ __forceinline__ F2 operator()(F2 x) const {
    if constexpr (DT == NS_DTYPE_F32) return mul2(add2(x, a), b);
    return fma2(x, a, b);
  }
};
// The same for one value.
template <int DT>
__device__ __forceinline__ float scaled_one(float x, float c, float scale) {
  return DT == NS_DTYPE_F32 ? (x - c) * scale : fmaf(x, scale, -__fmul_rn(c, scale));
}
// The offset c of a row's sums: the target's logit, 0 where that will not do.
template <int DT>
__device__ __forceinline__ float row_offset(float x_target, float scale) {
  const bool ok = DT == NS_DTYPE_F32 ? isfinite(x_target) : fabsf(x_target * scale) < kNearOffset;
  return ok ? x_target : 0.0f;
}

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
  int64_t give_up;          // the row at which a wait counts as run out (tests); kGiveUpNever
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
__device__ __forceinline__ void row_scale(float t, float& s, double& inv_t) {
  if (t == 0.0f) t = 1.0f;
  const bool ok = t > 0.0f && t < INFINITY;
  s = ok ? fminf(kLog2e / t, 3.402823466e38f) : NAN;
  inv_t = ok ? 1.0 / double(t) : double(NAN);
}
__device__ __forceinline__ void row_scale(const LossArgs& a, int64_t row, float& s, double& inv_t) {
  row_scale(a.temperature ? a.temperature[row] : a.temperature_all, s, inv_t);
}

constexpr int64_t kGiveUpNever = -2;     // -1 ends a block's rows

// Running (m, S, U) of a part of a row.  m = -inf: nothing but -inf so far.
// Sums around the target's logit have it, or 0, as m.
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

// One thread's running sums.  S in two parts: beside a row's one likely column,
// whose 2^t is 1, the others are too small for fp32, and an entropy is made of
// them.  (The same in 64 bits took a fifth longer.)  That column adds 0 to U.
struct Running {
  float m, s, low, u;
};

// Adds N values to the sums: one comparison of their maximum, one exponential each.
template <bool ENT, int N>
__device__ __forceinline__ void add(Running& p, const float (&x)[N], float scale) {
  float top = x[0];
#pragma unroll
  for (int i = 1; i < N; ++i) top = fmaxf(top, x[i]);
  if (top > p.m) {
    const float d = fmaxf((p.m - top) * scale, -200.0f);    // as in rescale
    const float f = ex2_approx(d);
    if (ENT) p.u = f * fmaf(d, p.s, p.u);
    p.s *= f;
    p.low *= f;
    p.m = top;
  }
  const float m = p.m == -INFINITY ? 0.0f : p.m;   // -inf - -inf would be NaN
  float s = 0.0f, u = 0.0f;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const float t = (x[i] - m) * scale;
    const float e = ex2_approx(t);
    s += e;
    // t is held above -200, where e is 0, so that 0 * -inf does not arise; a
    // NaN t has made e and S NaN
    if (ENT) u = fmaf(e, fmaxf(t, -200.0f), u);
  }
  const float sum = p.s + s, added = sum - p.s;    // and what the addition lost, exactly
  p.low += (p.s - (sum - added)) + (s - added);
  p.s = sum;
  if (ENT) p.u += u;
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

// One thread's part of share `rank` of `blocks` of a row with a running
// maximum: the part of a thread whose columns rise is rescaled.
template <int DT, bool ENT, int THREADS>
__device__ __forceinline__ Part thread_running(const void* base, int64_t vocab, float scale, int rank, int blocks, int tid) {
  using D = Elem<DT>;
  using T = typename D::T;
  constexpr int E = D::E;
  const T* row = static_cast<const T*>(base);
  const Span sp = row_span<E>(row, vocab);
  const int64_t v0 = sp.nv * rank / blocks, v1 = sp.nv * (rank + 1) / blocks;
  const uint4* vec = reinterpret_cast<const uint4*>(row + sp.head);
  Running p = {-INFINITY, 0.0f, 0.0f, 0.0f};
  const uint4 none = make_uint4(D::kNegInf2, D::kNegInf2, D::kNegInf2, D::kNegInf2);
  // loads ahead: with 4 in a warp's rows the compiler gives the whole kernel a slower form
  constexpr int kAgain = THREADS == 32 ? 2 : 4;
  for (int64_t v = v0 + tid; v < v1; v += kAgain * THREADS) {
    uint4 q[kAgain];
#pragma unroll
    for (int k = 0; k < kAgain; ++k) q[k] = v + k * THREADS < v1 ? vec[v + k * THREADS] : none;
#pragma unroll
    for (int k = 0; k < kAgain; ++k) {
      float x[E];
      D::unpack(q[k], x);
      add<ENT>(p, x, scale);
    }
  }
  const int64_t tail = sp.head + sp.nv * E + tid;
  const float x[2] = {rank == 0 && tid < sp.head ? D::load(row + tid) : -INFINITY,
                      rank == blocks - 1 && tail < vocab ? D::load(row + tail) : -INFINITY};
  add<ENT>(p, x, scale);
  return {p.m, p.s + p.low, p.u};
}
// The same joined over each of the warps that hold the THREADS threads.
template <int DT, bool ENT, int THREADS>
__device__ __noinline__ Part warp_running(const void* base, int64_t vocab, float scale, int rank, int blocks, int tid) {
  return warp_join<ENT>(thread_running<DT, ENT, THREADS>(base, vocab, scale, rank, blocks, tid), scale);
}
template <int DT, bool ENT>
__device__ __noinline__ Part block_running(const void* base, int64_t vocab, float scale, int rank, int blocks,
                                           Part* shared) {
  Part p = warp_running<DT, ENT, kThreads>(base, vocab, scale, rank, blocks, threadIdx.x);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) shared[threadIdx.x >> 5] = p;
  __syncthreads();
  const int lane = threadIdx.x & 31;
  p = lane < kWarps ? shared[lane] : Part{-INFINITY, 0.0f, 0.0f};
  return warp_join<ENT>(p, scale);
}

// Adds a vector's 2^t, and 2^t t, to the sums; of the 2^t the vector's own sum
// first, so that small values are not lost one by one beside a large sum (they
// made log-probabilities 8e-8 high on average at V = 151936).  t is held
// above -200, where 2^t is 0, so that 0 * -inf does not arise; a NaN t has made
// 2^t NaN.
template <int DT, bool ENT>
__device__ __forceinline__ void add_vector(const uint4& q, const ScaledPairs<DT>& scaled, F2& s, F2& u) {
  using D = Elem<DT>;
  constexpr int P = D::E / 2;
  float x[D::E];
  F2 e[P];
  D::unpack(q, x);
#pragma unroll
  for (int i = 0; i < P; ++i) {
    float a, b;
    split(scaled(f2(x[2 * i], x[2 * i + 1])), a, b);
    e[i] = f2(ex2_approx(a), ex2_approx(b));
    if (ENT) u = fma2(e[i], f2(fmaxf(a, -200.0f), fmaxf(b, -200.0f)), u);
  }
  if constexpr (ENT && DT == NS_DTYPE_F32) {      // the products leave no registers for it
    s = add2(add2(s, e[0]), e[1]);
  } else if constexpr (ENT) {                     // and here for two at a time
#pragma unroll
    for (int i = 0; i < P; i += 2) s = add2(s, add2(e[i], e[i + 1]));
  } else {
#pragma unroll
    for (int n = P / 2; n; n /= 2)
#pragma unroll
      for (int i = 0; i < n; ++i) e[i] = add2(e[i], e[i + n]);
    s = add2(s, e[0]);
  }
}

// A call's kernels follow one another closely: each lets the next one start (its
// blocks take places as they fall free), and that one waits until every block
// before it has ended and what they wrote is there; 1 to 2 us a call.  A third
// kernel waits for the second, which has itself waited for the first.
__device__ __forceinline__ void let_next_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void wait_for_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

struct RowShared {
  Part warp[kWarps];
  Part block[kMaxCluster];
};

// Whether the row has to be added up around its largest logit: S says that c
// lies too far from it, or the entropy, ln S - ln2 U / S, is so much smaller
// than the two that their roundings show (2e-7 of |ln S| as a root mean square,
// 4e-7 beside many small terms).  A target of more than 2^-8 is never that far,
// and of drawn targets one in 256 at most is 256 entropies unlikely.  With 2^-6
// and 64, rows of most calls were.  NaN: the row holds one, and no offset helps.
template <bool ENT>
__device__ __forceinline__ bool sums_far(const Part& p) {
  if (p.s < 0x1p-60f || p.s > 0x1p100f) return true;
  if (!ENT) return false;
  const float l = __log2f(p.s);
  return fabsf(l) > 8.0f && 256.0f * fmaf(l, p.s, -p.u) < fabsf(l) * p.s;
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
  return v;
}

// One thread's sums around c over part `rank` of `parts` of a row that THREADS threads add up.
template <int DT, bool ENT, int THREADS>
__device__ __forceinline__ Part thread_sums(const void* base, int64_t vocab, float c, float scale, int rank, int parts,
                                            int tid) {
  using D = Elem<DT>;
  using T = typename D::T;
  constexpr int E = D::E;
  const T* row = static_cast<const T*>(base);
  const Span sp = row_span<E>(row, vocab);
  const int v0 = int(sp.nv * rank / parts), n = int(sp.nv * (rank + 1) / parts) - v0;
  const uint4* vec = reinterpret_cast<const uint4*>(row + sp.head) + v0;
  const uint4 none = make_uint4(D::kNegInf2, D::kNegInf2, D::kNegInf2, D::kNegInf2);
  uint4 q[kBatch];
#pragma unroll
  for (int k = 0; k < kBatch; ++k) {
    const int v = tid + k * THREADS;
    q[k] = v < n ? vec[v] : none;
  }
  // the elements before the first 16-byte boundary and after the last whole vector
  const int64_t tail = sp.head + sp.nv * E + tid;
  const float edge[2] = {rank == 0 && tid < sp.head ? D::load(row + tid) : -INFINITY,
                         rank == parts - 1 && tail < vocab ? D::load(row + tail) : -INFINITY};
  const auto scaled = ScaledPairs<DT>::of(c, scale);
  F2 s[2] = {0, 0}, u[2] = {0, 0};
  for (int v = tid; v < n; v += kBatch * THREADS) {
    uint4 next[kBatch];
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      const int at = v + (kBatch + k) * THREADS;
      next[k] = at < n ? vec[at] : none;
    }
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      add_vector<DT, ENT>(q[k], scaled, s[k & 1], u[k & 1]);
      q[k] = next[k];
    }
  }
  Part p;
  p.m = c;
  float lo, hi;
  split(add2(s[0], s[1]), lo, hi);
  p.s = lo + hi;
  split(add2(u[0], u[1]), lo, hi);
  p.u = lo + hi;
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const float t = scaled_one<DT>(edge[k], c, scale), e = ex2_approx(t);
    p.s += e;
    if (ENT) p.u = fmaf(e, fmaxf(t, -200.0f), p.u);
  }
  return p;
}

// The sums around c over part `rank` of `parts` of a row, in every thread.
template <int DT, bool ENT>
__device__ __forceinline__ Part part_sums(const void* base, int64_t vocab, float c, float scale, int rank, int parts,
                                          Part* shared) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  Part p = thread_sums<DT, ENT, kThreads>(base, vocab, c, scale, rank, parts, threadIdx.x);
  p.s = warp_sum(p.s);
  if (ENT) p.u = warp_sum(p.u);
  if (lane == 0) shared[warp] = p;
  __syncthreads();
  p.s = warp_sum(lane < kWarps ? shared[lane].s : 0.0f);
  if (ENT) p.u = warp_sum(lane < kWarps ? shared[lane].u : 0.0f);
  return p;
}

__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }

// The row's sums around c over the whole cluster, the same in every thread of it.
template <int DT, bool ENT>
__device__ __forceinline__ Part row_sums(const void* base, int64_t vocab, float c, float scale, RowShared& sh,
                                         cg::cluster_group& cluster, bool& near) {
  const int blocks = int(cluster.num_blocks()), rank = int(cluster.block_rank()), lane = threadIdx.x & 31;
  if (blocks > 1) cluster_arrive();
  Part p = part_sums<DT, ENT>(base, vocab, c, scale, rank, blocks, sh.warp);
  if (blocks > 1) {
    cluster_wait();                    // every block has started: its shared memory may be written
    if (int(threadIdx.x) < blocks) *cluster.map_shared_rank(&sh.block[rank], threadIdx.x) = p;
    cluster.sync();
    p.s = warp_sum(lane < blocks ? sh.block[lane].s : 0.0f);
    if (ENT) p.u = warp_sum(lane < blocks ? sh.block[lane].u : 0.0f);
  }
  near = !sums_far<ENT>(p);          // the same for the whole cluster
  if (near) return p;
  p = block_running<DT, ENT>(base, vocab, scale, rank, blocks, sh.warp);
  if (blocks > 1) {
    cluster.sync();                    // every block has read the first sums
    if (int(threadIdx.x) < blocks) *cluster.map_shared_rank(&sh.block[rank], threadIdx.x) = p;
    cluster.sync();
    p = lane < blocks ? sh.block[lane] : Part{-INFINITY, 0.0f, 0.0f};
    p = warp_join<ENT>(p, scale);
  }
  return p;
}

// What a row's sums and target give, in 64 bits, so that differences from a
// reference's log-probability keep their digits.  The target's t uses the same
// rounded scale, and `near` the same rounded offset, as the sums.  The
// logarithm is split as exponent * ln2 + ln(mantissa), whose second part lies
// in [0, ln2) and is off by 2^-24 at most.
struct RowResult {
  double logprob;
  float entropy, log2s;      // log2 S around m s, not rounded
};
template <int DT, bool ENT>
__device__ __forceinline__ RowResult finish(const Part& p, float x_target, float scale, bool near) {
  int ex;
  const float mant = 2.0f * frexpf(p.s, &ex);
  const double ln_s = p.s < INFINITY && p.s > 0.0f ? double(ex - 1) * kLn2 + double(logf(mant)) : double(NAN);
  // how far the sums' offset lies from m s
  const double moved = DT != NS_DTYPE_F32 && near ? double(__fmul_rn(p.m, scale)) - double(p.m) * double(scale) : 0.0;
  // the exponentials are kEx2Mean low on average, all but for the target's own, 2^0 = 1, which is 1 / S of S as long
  // as the sums' offset is the target's logit; around 0 the target has no such part, and S may be as small as 2^-60.
  // A sequence's reward adds such errors up, a gradient's p divides them out
  const double ln_all = ln_s + (near && p.m == x_target ? kEx2Mean * (1.0 - double(1.0f / p.s)) : 0.0);
  RowResult r;
  r.logprob = ((double(x_target) - double(p.m)) * double(scale) - moved) * kLn2 - ln_all;
  if (r.logprob > 0.0) r.logprob = 0.0;          // a rounding of S
  r.log2s = float(ln_s * (1.0 / kLn2) + moved);
  // a difference of two numbers of the size of ln S, the quotient with its remainder; roundings must not make it negative
  const float mean = p.u / p.s, rest = __fdividef(fmaf(-mean, p.s, p.u), p.s);
  const float entropy = ENT ? fmaf(-float(kLn2), rest, float(fma(-kLn2, double(mean), ln_all))) : 0.0f;
  r.entropy = entropy < 0.0f ? 0.0f : entropy;
  if (isnan(r.logprob)) r.log2s = r.entropy = NAN;
  return r;
}

struct PolicyIn {
  float old, adv, ref, w;
};
struct PolicyRow {
  float loss, kl, a, h;
};
__device__ __forceinline__ PolicyIn policy_in(const LossArgs& a, int64_t row, float w) {
  return {a.old_logprobs[row], a.advantages[row], a.ref_logprobs ? a.ref_logprobs[row] : 0.0f, w};
}
__device__ __forceinline__ PolicyRow policy_row(const LossArgs& a, const PolicyIn& in, double logprob, float entropy) {
  const float ratio = expf(float(logprob - double(in.old)));
  const float inside = ratio * in.adv;
  const float clipped = fminf(fmaxf(ratio, 1.0f - a.clip_low), 1.0f + a.clip_high) * in.adv;
  PolicyRow r = {0.0f, 0.0f, 0.0f, 0.0f};
  // fmin drops a NaN, so the comparison keeps it; without an advantage there is no term (0 * inf is NaN)
  if (in.adv != 0.0f || isnan(ratio)) {
    r.loss = -(clipped < inside ? clipped : inside);
    r.a = clipped < inside ? 0.0f : -inside;
  }
  if (a.ref_logprobs) {
    const float d = float(double(in.ref) - logprob);
    const float g = expm1f(d);
    // e^d - 1 - d: near 0 by its series, d^2 / 2 (1 + d / 3 (1 + d / 4 (...))), whose next term is 2^-28 at 1/2
    float series = 1.0f;
#pragma unroll
    for (int i = 9; i > 2; --i) series = fmaf(d * (1.0f / float(i)), series, 1.0f);
    r.kl = fabsf(d) < 0.5f ? 0.5f * d * d * series : g - d;
    if (a.kl_coef != 0.0f) {
      r.loss = fmaf(a.kl_coef, r.kl, r.loss);
      r.a = fmaf(-a.kl_coef, g, r.a);
    }
  }
  if (a.entropy_coef != 0.0f) {
    r.loss = fmaf(-a.entropy_coef, entropy, r.loss);
    r.h = -a.entropy_coef * in.w;
  }
  r.a *= in.w;
  return r;
}
__device__ __forceinline__ void write_policy_row(const LossArgs& a, int64_t row, const PolicyRow& l) {
  a.row_loss[row] = l.loss;
  if (a.kl) a.kl[row] = l.kl;
  a.row_grad[row] = l.a;
  a.row_grad[a.rows + row] = l.h;
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

// Gradient of one value: g = p (A + B log2 p), log2 p = (x - c) s - log2 S.
struct alignas(16) GradRow {
  float c, log2s, scale, ca, cb;
  float at;                  // the value at the target
  bool zero, wide, later;    // wide: |c s| is too large for one multiply-add; later: there is no gradient yet
  int target;                // past the vocabulary: none
};
template <int DT, bool ENT>
__device__ __forceinline__ float grad_value(const GradRow& g, float x) {
  const float t = fmaf(x - g.c, g.scale, -g.log2s);
  return ex2_approx(t) * (ENT ? fmaf(g.cb, fmaxf(t, -200.0f), g.ca) : g.ca);
}
// A coefficient over T, held at `most` where a small T would take it past fp32:
// 0 times infinity must not arise in a column without probability (A + B log2 p is
// A - 200 B there).
__device__ __forceinline__ float held(double v, double inv_t, float most) {
  const float f = float(v * inv_t);
  return fabsf(f) > most && !isinf(v) ? copysignf(most, f) : f;
}
// a and h: dloss/dlogprob and dloss/dentropy of the row
template <int DT, bool ENT>
__device__ __forceinline__ GradRow grad_row(float c, float log2s, float scale, double inv_t, float a, float h,
                                            float entropy, int64_t target, float x_target) {
  GradRow g;
  g.c = c == -INFINITY ? 0.0f : c;      // no distribution: log2 S is NaN
  g.log2s = log2s;
  g.scale = scale;
  g.wide = DT != NS_DTYPE_F32 && !(fabsf(g.c * scale) < kNearOffset);
  // at the target a (1 - p) - h p (ln p + H): where p is near 1, 1 - p must come from ln p, and that from the difference
  // (a - a: an infinite coefficient has no gradient here, as it has none where p is 0)
  const float t = fmaf(x_target - g.c, scale, -log2s);
  const float ln_p = t > 0.0f ? 0.0f : t * float(kLn2);      // above 0 by a rounding of S
  const float at = -a * expm1f(ln_p) + (a - a) - (ENT ? h * ex2_approx(t) * (fmaxf(ln_p, -200.0f) + entropy) : 0.0f);
  g.at = float(double(at) * inv_t);
  g.ca = -held(double(a) + (ENT ? double(h) * double(entropy) : 0.0), inv_t, 0x1p127f);
  g.cb = ENT ? -held(double(h) * kLn2, inv_t, 0x1p119f) : 0.0f;
  if (DT != NS_DTYPE_F32 && !g.wide) {
    // One multiply-add to t' = x s - fl(c s + log2 S).  What the product and the sum leave out, d, is a factor of the
    // row's p: 2^(t' - d) (A + B (t' - d)).  It is below 2^-13, so that 2^-d is 1 - d ln2 to 2^-27.
    const float off = __fmul_rn(g.c, scale), whole = __fadd_rn(off, log2s), added = __fsub_rn(whole, off);
    const float d = fmaf(g.c, scale, -off) + __fadd_rn(__fsub_rn(off, __fsub_rn(whole, added)), __fsub_rn(log2s, added));
    const float f = fmaf(-d, float(kLn2), 1.0f);
    g.c = 0.0f;
    g.log2s = whole;
    g.ca = f * (ENT ? fmaf(-g.cb, d, g.ca) : g.ca);
    g.cb *= f;
  }
  g.zero = a == 0.0f && h == 0.0f;
  g.later = false;
  g.target = int(target < (int64_t(1) << 24) ? target : int64_t(1) << 24);
  return g;
}
// The same for a vector; the constants of the row are in pairs.  c is 0 in
// 16-bit rows that are not wide: one multiply-add to log2 p.
template <int DT>
struct GradPairs {
  F2 a, b, l, ca, cb;
  __device__ __forceinline__ explicit GradPairs(const GradRow& g) : ca(f2(g.ca, g.ca)), cb(f2(g.cb, g.cb)) {
    if constexpr (DT == NS_DTYPE_F32) {
      a = f2(-g.c, -g.c), b = f2(g.scale, g.scale), l = f2(-g.log2s, -g.log2s);
    } else {
      a = f2(g.scale, g.scale), b = f2(-g.log2s, -g.log2s), l = 0;
    }
  }
  __device__ __forceinline__ F2 operator()(F2 x) const {
    if constexpr (DT == NS_DTYPE_F32) return fma2(add2(x, a), b, l);
    return fma2(x, a, b);
  }
};
template <int DT, bool ENT>
__device__ __forceinline__ uint4 grad_vector(const GradPairs<DT>& g, const uint4& q) {
  using D = Elem<DT>;
  float x[D::E];
  D::unpack(q, x);
#pragma unroll
  for (int i = 0; i < D::E; i += 2) {
    float a, b;
    split(g(f2(x[i], x[i + 1])), a, b);
    const F2 p = f2(ex2_approx(a), ex2_approx(b));
    const F2 w = ENT ? fma2(g.cb, f2(fmaxf(a, -200.0f), fmaxf(b, -200.0f)), g.ca) : g.ca;
    split(mul2(p, w), x[i], x[i + 1]);
  }
  return D::pack(x);
}
template <int DT, bool ENT>
__device__ __forceinline__ void grad_element(const GradRow& g, float x, typename Elem<DT>::T* out, int64_t j) {
  Elem<DT>::store(out + j, j == g.target ? g.at : grad_value<DT, ENT>(g, x));
}

// Block `rank`'s share of a row's gradient element by element: the rows start on
// different 16-byte phases, or the row is wide.
template <int DT, bool ENT, int THREADS>
__device__ __forceinline__ void write_elements(const GradRow& g, const void* base, void* grad, int64_t vocab, int rank,
                                               int blocks) {
  using T = typename Elem<DT>::T;
  const T* row = static_cast<const T*>(base);
  const int64_t end = vocab * (rank + 1) / blocks;
  for (int64_t j = vocab * rank / blocks + threadIdx.x; j < end; j += THREADS)
    grad_element<DT, ENT>(g, Elem<DT>::load(row + j), static_cast<T*>(grad), j);
}

// Zeros in block `rank`'s share of a row.
template <int DT, int THREADS>
__device__ __forceinline__ void write_zeros(void* grad, int64_t vocab, int rank, int blocks) {
  using T = typename Elem<DT>::T;
  constexpr int E = Elem<DT>::E;
  T* out = static_cast<T*>(grad);
  const Span sp = row_span<E>(out, vocab);
  uint4* dst = reinterpret_cast<uint4*>(out + sp.head);
  const int v1 = int(sp.nv * (rank + 1) / blocks);
  for (int v = int(sp.nv * rank / blocks) + threadIdx.x; v < v1; v += THREADS) dst[v] = make_uint4(0, 0, 0, 0);
  const int64_t tail = sp.head + sp.nv * E + threadIdx.x;
  if (rank == 0 && threadIdx.x < sp.head) Elem<DT>::store(out + threadIdx.x, 0.0f);
  if (rank == blocks - 1 && tail < vocab) Elem<DT>::store(out + tail, 0.0f);
}

// The numbers of a row that holds no token.
template <int OP>
__device__ __forceinline__ void write_dead_row(const LossArgs& a, int64_t row) {
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

// What a forward call leaves of a row (one thread).
template <int DT, bool ENT, int OP>
__device__ __forceinline__ void write_row(const LossArgs& a, int64_t row, const Part& p, float x_target, float scale,
                                          float w, bool near) {
  const RowResult r = finish<DT, ENT>(p, x_target, scale, near);
  a.logprobs[row] = float(r.logprob);
  if (ENT) a.entropy[row] = r.entropy;
  if (a.stats) {
    a.stats[2 * row] = p.m;
    a.stats[2 * row + 1] = r.log2s;
  }
  if (OP == kPolicy) write_policy_row(a, row, policy_row(a, policy_in(a, row, w), r.logprob, r.entropy));
  if (OP == kPreference)   // the row's gain; the pair kernel turns it into the coefficient
    a.row_grad[row] = float(r.logprob - (a.ref_logprobs ? double(a.ref_logprobs[row]) : 0.0));
}

// One cluster of blocks per row.
template <int DT, bool ENT, int OP>
__global__ void __launch_bounds__(kThreads, 5) forward_kernel(const LossArgs a) {
  if (OP != kLogprob) let_next_start();
  using D = Elem<DT>;
  using T = typename D::T;
  __shared__ RowShared sh;
  cg::cluster_group cluster = cg::this_cluster();
  const int blocks = int(cluster.num_blocks()), rank = int(cluster.block_rank());
  const int64_t row = blockIdx.x / blocks;
  float w;
  if (!row_alive<OP>(a, row, w)) {            // the same for every block of the cluster
    if (rank == 0 && threadIdx.x == 0) write_dead_row<OP>(a, row);
    return;
  }
  float scale;
  double inv_t;
  row_scale(a, row, scale, inv_t);
  const T* x = static_cast<const T*>(a.logits) + row * a.row_stride;
  const int64_t target = a.targets[row];
  const float x_target = target < a.vocab ? D::load(x + target) : NAN;
  bool near;
  const Part p = row_sums<DT, ENT>(x, a.vocab, row_offset<DT>(x_target, scale), scale, sh, cluster, near);
  if (threadIdx.x == 0 && rank == 0) write_row<DT, ENT, OP>(a, row, p, x_target, scale, w, near);
}

// One warp per row, for rows so short that a block's barriers would be most of
// the work.  8192 x 2000 bf16: 33 us by blocks.
template <int DT, bool ENT, int OP>
__global__ void __launch_bounds__(kThreads) forward_rows_kernel(const LossArgs a) {
  if (OP != kLogprob) let_next_start();
  using D = Elem<DT>;
  using T = typename D::T;
  const int64_t row = int64_t(blockIdx.x) * kWarps + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (row >= a.rows) return;
  float w;
  if (!row_alive<OP>(a, row, w)) {
    if (lane == 0) write_dead_row<OP>(a, row);
    return;
  }
  float scale;
  double inv_t;
  row_scale(a, row, scale, inv_t);
  const T* x = static_cast<const T*>(a.logits) + row * a.row_stride;
  const int64_t target = a.targets[row];
  const float x_target = target < a.vocab ? D::load(x + target) : NAN;
  const float c = row_offset<DT>(x_target, scale);
  Part p = thread_sums<DT, ENT, 32>(x, a.vocab, c, scale, 0, 1, lane);
  p.s = warp_sum(p.s);
  if (ENT) p.u = warp_sum(p.u);
  const bool near = !sums_far<ENT>(p);
  if (!near) p = warp_running<DT, ENT, 32>(x, a.vocab, scale, 0, 1, lane);
  if (lane == 0) write_row<DT, ENT, OP>(a, row, p, x_target, scale, w, near);
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
  wait_for_previous();
  double v = 0.0;
  for (int64_t i = threadIdx.x; i < a.rows; i += 1024) {
    const double w = a.weights ? double(a.weights[i]) : 1.0 / double(a.rows);
    if (a.targets[i] >= 0 && w != 0.0) v += w * double(a.row_loss[i]);
  }
  v = block_sum(v, shared);
  if (threadIdx.x == 0) *loss = float(v);
}

// The pairs: warps sum the sequences' gains (several a sequence while they are
// few), one thread a pair turns two sums into the pair's loss, and the warps
// write the rows' coefficients over the gains.
__global__ void __launch_bounds__(1024) pair_kernel(const LossArgs a, float beta, float smoothing, int average,
                                                    float* loss, float* pair_loss, float* rewards) {
  __shared__ double sums[32], shared[32];
  __shared__ int counts[32];
  __shared__ float coef[32];
  let_next_start();
  wait_for_previous();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int each = 1;                           // warps of a sequence
  while (each < 16 && 2 * a.pairs * each * 2 <= 32) each *= 2;
  const int at_once = 32 / each, step = 32 * each;
  double total = 0.0;
  for (int64_t first = 0; first < 2 * a.pairs; first += at_once) {
    const int64_t seq = first + warp / each;
    int64_t lo = 0, hi = 0;
    if (seq < 2 * a.pairs) {
      lo = max(a.seq_offsets[seq], int64_t(0)) + warp % each * 32 + lane;
      hi = min(a.seq_offsets[seq + 1], a.rows);
    }
    double sum = 0.0;
    int count = 0;
#pragma unroll 4
    for (int64_t i = lo; i < hi; i += step) {
      sum += double(a.row_grad[i]);
      count += a.targets[i] >= 0;
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) {
      sum += __shfl_xor_sync(~0u, sum, o);
      count += __shfl_xor_sync(~0u, count, o);
    }
    if (lane == 0) sums[warp] = sum, counts[warp] = count;
    __syncthreads();
    const int64_t p = first / 2 + threadIdx.x;
    if (threadIdx.x < at_once / 2 && p < a.pairs) {
      double reward[2], share[2];
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const int w = (2 * int(threadIdx.x) + k) * each;
        double s = 0.0;
        int n = 0;
        for (int i = 0; i < each; ++i) s += sums[w + i], n += counts[w + i];
        share[k] = average ? 1.0 / double(max(n, 1)) : 1.0;
        reward[k] = double(beta) * s * share[k];
      }
      const double h = reward[0] - reward[1];
      // ln sigmoid(h) = min(h, 0) - ln(1 + exp(-|h|)), and the same with -h
      const float tail = log1pf(expf(-fabsf(float(h))));
      const double win = fmin(h, 0.0) - double(tail), lose = fmin(-h, 0.0) - double(tail);
      const double e = double(smoothing);
      // without smoothing an infinite margin must not meet 0 * inf
      const double l = isnan(h) ? h : -(1.0 - e) * win - (e != 0.0 ? e * lose : 0.0);
      const double up = 1.0 / (1.0 + double(expf(float(-h)))), down = 1.0 / (1.0 + double(expf(float(h))));
      const double slope = (e * up - (1.0 - e) * down) * double(beta) / double(a.pairs);
      coef[2 * threadIdx.x] = float(slope * share[0]);
      coef[2 * threadIdx.x + 1] = float(-slope * share[1]);
      pair_loss[p] = float(l);
      rewards[2 * p] = float(reward[0]);
      rewards[2 * p + 1] = float(reward[1]);
      total += l;
    }
    __syncthreads();
    const float c = coef[warp / each];
    for (int64_t i = lo; i < hi; i += step) a.row_grad[i] = a.targets[i] >= 0 ? c : 0.0f;
  }
  total = block_sum(total, shared);
  if (threadIdx.x == 0) *loss = a.pairs ? float(total / double(a.pairs)) : 0.0f;
}

constexpr int kGradThreads = 128;
constexpr int kGradVecs = 8;    // vectors of a thread

// Chunk `chunk` of `chunks` of a row's gradient.
template <int DT, bool ENT>
__device__ __forceinline__ void write_chunk(const GradRow& g, const void* base, void* grad, int64_t vocab, int chunk,
                                            int chunks) {
  using D = Elem<DT>;
  using T = typename D::T;
  constexpr int E = D::E;
  const T* x = static_cast<const T*>(base);
  T* out = static_cast<T*>(grad);
  if (g.zero) {
    write_zeros<DT, kGradThreads>(out, vocab, chunk, chunks);
    return;
  }
  const bool same = ((reinterpret_cast<uintptr_t>(x) ^ reinterpret_cast<uintptr_t>(out)) & 15) == 0;
  if (!same || (DT != NS_DTYPE_F32 && g.wide)) {
    write_elements<DT, ENT, kGradThreads>(g, x, out, vocab, chunk, chunks);
    return;
  }
  const Span sp = row_span<E>(x, vocab);
  const int v0 = int(sp.nv * chunk / chunks), n = int(sp.nv * (chunk + 1) / chunks) - v0;
  const int j0 = int(sp.head) + v0 * E;
  const uint4* src = reinterpret_cast<const uint4*>(x + j0) + threadIdx.x;
  uint4* dst = reinterpret_cast<uint4*>(out + j0) + threadIdx.x;
  const GradPairs<DT> pairs(g);
  uint4 q[kGradVecs];
#pragma unroll
  for (int k = 0; k < kGradVecs; ++k)
    if (int(threadIdx.x) + k * kGradThreads < n) q[k] = src[k * kGradThreads];
#pragma unroll
  for (int k = 0; k < kGradVecs; ++k)
    if (int(threadIdx.x) + k * kGradThreads < n) dst[k * kGradThreads] = grad_vector<DT, ENT>(pairs, q[k]);
  // the target's value over its vector, by the thread that wrote it
  const unsigned at = unsigned(g.target - j0);
  if (at < unsigned(n) * E && int(at / E) % kGradThreads == int(threadIdx.x)) D::store(out + g.target, g.at);
  const int64_t tail = sp.head + sp.nv * E + threadIdx.x;
  if (chunk == 0 && threadIdx.x < sp.head)
    grad_element<DT, ENT>(g, D::load(x + threadIdx.x), out, threadIdx.x);
  if (chunk == chunks - 1 && tail < vocab) grad_element<DT, ENT>(g, D::load(x + tail), out, tail);
}

// The gradient alone: one block per (row, chunk of kGradThreads x kGradVecs vectors),
// from the last row on, whose logits L2 still holds from the sums.
template <int DT, bool ENT>
__global__ void __launch_bounds__(kGradThreads) grad_kernel(const LossArgs a, int chunks) {
  let_next_start();
  wait_for_previous();
  using D = Elem<DT>;
  using T = typename D::T;
  const int64_t row = a.rows - 1 - blockIdx.x / chunks;
  const int chunk = int(blockIdx.x % chunks);
  const T* x = static_cast<const T*>(a.logits) + row * a.row_stride;
  T* out = static_cast<T*>(a.grad_logits) + row * a.grad_stride;
  const float ga = a.grad_logprobs ? a.grad_logprobs[row] : 0.0f;
  const float gh = ENT ? a.grad_entropy[row] : 0.0f;
  const int64_t target = a.targets[row];
  GradRow g = {};
  g.zero = target < 0 || (ga == 0.0f && gh == 0.0f);
  if (!g.zero) {
    float scale;
    double inv_t;
    row_scale(a, row, scale, inv_t);
    // every thread reads the target's logit before it writes; in place, the one that uses it is its writer
    g = grad_row<DT, ENT>(a.stats[2 * row], a.stats[2 * row + 1], scale, inv_t, ga, gh, ENT ? a.entropy[row] : 0.0f,
                          target, target < a.vocab ? D::load(x + target) : NAN);
  }
  write_chunk<DT, ENT>(g, x, out, a.vocab, chunk, chunks);
}

// ---------------------------------------------------------------------------
// Policy loss and gradient from one reading of the logits
// ---------------------------------------------------------------------------
// A row's gradient needs the row's sums first, so a block keeps the row (or a
// cluster's block its share of it) on chip between the two.  Persistent
// clusters, to which the rows are dealt out.  A producer warp copies rows in
// chunks into a ring in shared memory.  The row warps add a row up as its
// chunks land: the first chunks they keep in registers and hand back at
// once, the others stay in the ring.  They join their sums (over the cluster
// through the peers' shared memory) and write the gradient, the ring's chunks
// first, handing each back as it is done, so the reads of the next row run
// under the writes of this one.  The logits cross L2 and DRAM once.
//
// What bounds it: 2 exponentials a logit are 70 % of the time that bf16's 4
// bytes a logit need, and a row's sums cannot end before its last chunk lands.
// Loading the registers straight from memory instead was slower (10 us a row of
// 123 KB): beside 215 KB of shared memory L1 has room for few loads.
// The shapes of a block: 15 row warps with registers, alone on an SM; 15 with
// a smaller ring, two to an SM; 7, three to an SM.
enum Shape { kLarge = 0, kMedium = 1, kSmall = 2 };
template <int SHAPE>
struct HeldShape {
  static constexpr int kRowWarps = SHAPE == kSmall ? 7 : 15;
  static constexpr int kRowThreads = kRowWarps * 32;
  static constexpr int kThreads = kRowThreads + 32;          // and the producer warp
  static constexpr int kLaneVecs = SHAPE == kLarge ? 4 : 2;  // of a chunk
  static constexpr int kChunkVecs = kRowThreads * kLaneVecs;
  static constexpr int kChunkBytes = kChunkVecs * 16;
  static constexpr int kHold = SHAPE == kLarge ? 4 : 0;      // chunks in registers
  static constexpr int kSlots = SHAPE == kSmall ? 10 : 7;
  static constexpr int kBlocks = SHAPE == kLarge ? 1 : SHAPE == kMedium ? 2 : 3;
  static constexpr int kMostVecs = (kHold + kSlots - 1) * kChunkVecs;
  static constexpr uint32_t kSmem = uint32_t(kSlots) * kChunkBytes;
};

// What the producer says of a row, with its first chunk.
struct RowInfo {
  int64_t row;            // -1 ends the rows
  int alive;              // 0: it holds no token, and there is no more to say
  int64_t target;
  double inv_t;
  float x_target, scale;
  PolicyIn in;
};
constexpr int kPutOffList = 32;
struct HeldShared {
  uint64_t full[16], empty[16];    // of the ring's chunks
  uint64_t bar[2];                 // sums of the cluster's blocks, by turn
  float2 part[2][kMaxCluster];     // (S, U) of each block
  float2 warp_part[16];
  Part again_part[16];             // of the warps, for a row that was put off
  int put_off, put_off_row[kPutOffList];    // how many rows were, and the first of them
  RowInfo info[16];                // of the row whose first chunk lies in the slot
  GradRow coef;
};

__device__ __forceinline__ uint32_t peer_addr(const void* p, int rank) {
  uint32_t d;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(d) : "r"(smem_addr(p)), "r"(rank));
  return d;
}
// Stores 8 bytes in a peer block's shared memory and counts them on its barrier.
__device__ __forceinline__ void send(uint32_t dst, float a, float b, uint32_t bar) {
  asm volatile("st.async.shared::cluster.mbarrier::complete_tx::bytes.v2.f32 [%0], {%1, %2}, [%3];" ::"r"(dst), "f"(a),
               "f"(b), "r"(bar)
               : "memory");
}
// mbar_wait_bounded, whose limit is wall time, in the time that the kernel runs:
// a poll counts for a millisecond at most, so that a context that was suspended
// for long does not find its waits run out.
__device__ __forceinline__ bool mbar_wait_running(uint64_t* bar, uint32_t parity) {
  if (mbar_try_wait(bar, parity)) return true;
  uint64_t last = global_timer_ns(), waited = 0;
  while (!mbar_try_wait(bar, parity)) {
    const uint64_t now = global_timer_ns();
    waited += min(now - last, uint64_t(1000000));
    last = now;
    if (waited > kWaitTimeoutNs) return false;
  }
  return true;
}
__device__ __forceinline__ void mbar_arrive(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_addr(bar)) : "memory");
}
// The barriers of the row warps; the second tells all of them whether one says so.
template <int THREADS>
__device__ __forceinline__ void row_barrier() {
  asm volatile("bar.sync 1, %0;" ::"n"(THREADS) : "memory");
}
template <int THREADS>
__device__ __forceinline__ bool row_barrier_any(bool says) {
  uint32_t any;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.u32 q, %1, 0;\n\t"
      "bar.red.or.pred p, 1, %2, q;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(any)
      : "r"(uint32_t(says)), "n"(THREADS)
      : "memory");
  return any != 0;
}

// A cluster's rows in order.  The rows that hold a token are dealt out in turn,
// and so are those that do not, so every cluster has its share of both however
// the padding lies.  One warp looks through the rows, 32 at a time; the numbers
// that say which are which come 128 rows at a time and as many ahead.
struct RowWalk {
  static constexpr int kAhead = 4;
  int64_t base = 0;                 // of the 32 rows looked at next
  unsigned alive = 0, dead = 0;     // those before them, modulo the clusters
  uint32_t mine = 0, mine_alive = 0;
  uint32_t held = 0;                // bit i: this lane's row of the block's i-th 32 holds a token
  bool next_held[kAhead];
  __device__ __forceinline__ void look(const LossArgs& a, int64_t block) {
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int64_t row = block + 32 * i + (threadIdx.x & 31), at = min(row, a.rows - 1);
      const float w = a.weights ? a.weights[at] : 1.0f;
      next_held[i] = (a.targets[at] >= 0) & (w != 0.0f) & (row < a.rows);
    }
  }
  // The masks of the next 32 rows that are this cluster's.
  __device__ __forceinline__ void step(const LossArgs& a, unsigned cluster, unsigned clusters) {
    const int i = int(base >> 5) & (kAhead - 1);
    if (i == 0) {
      if (base == 0) look(a, 0);
      held = 0;
#pragma unroll
      for (int j = 0; j < kAhead; ++j) held |= uint32_t(next_held[j]) << j;
      look(a, base + 32 * kAhead);
    }
    const bool here = base + (threadIdx.x & 31) < a.rows, hold = (held >> i) & 1;
    const uint32_t lower = lanemask_lt(), holds = __ballot_sync(~0u, hold), rest = __ballot_sync(~0u, here && !hold);
    const unsigned turn = hold ? alive + __popc(holds & lower) : dead + __popc(rest & lower);
    alive += __popc(holds), dead += __popc(rest);
    bool is_mine;
    if (clusters >= 32) {           // one round at most goes by in 32 rows
      is_mine = turn == cluster || turn == cluster + clusters;
      if (alive >= clusters) alive -= clusters;
      if (dead >= clusters) dead -= clusters;
    } else {
      is_mine = turn % clusters == cluster;
      alive %= clusters, dead %= clusters;
    }
    mine = __ballot_sync(~0u, here && is_mine);
    mine_alive = holds;
    base += 32;
  }
};

// A block's vectors [v0, v0 + n) of a row that starts at `base`; `shift` is log2 of the cluster's blocks.
struct Share {
  int head, v0, n;
};
template <int E>
__device__ __forceinline__ Share row_share(const void* base, int vocab, int rank, int shift) {
  Share s;
  s.head = min(vocab, int(((16 - (uint32_t(reinterpret_cast<uintptr_t>(base)) & 15)) & 15) / (16 / E)));
  const int nv = (vocab - s.head) / E;          // at most 2^22, and rank + 1 at most 2^3
  s.v0 = nv * rank >> shift;
  s.n = (nv * (rank + 1) >> shift) - s.v0;
  return s;
}

// A row's sums turned into its results and its gradient's constants (one thread).
template <int DT, bool ENT>
__device__ __forceinline__ void finish_policy_row(const LossArgs& a, int64_t row, const Part& p, const RowInfo& info,
                                                  bool near, bool write, GradRow& coef) {
  const RowResult r = finish<DT, ENT>(p, info.x_target, info.scale, near);
  const PolicyRow l = policy_row(a, info.in, r.logprob, r.entropy);
  coef = grad_row<DT, ENT>(p.m, r.log2s, info.scale, info.inv_t, l.a, l.h, r.entropy, info.target, info.x_target);
  if (write) {
    a.logprobs[row] = float(r.logprob);
    if (ENT) a.entropy[row] = r.entropy;
    a.stats[2 * row] = p.m;
    a.stats[2 * row + 1] = r.log2s;
    write_policy_row(a, row, l);
  }
}

// A row whose sums have to be taken around its largest logit, read again by the
// row warps of its cluster's first block.
template <int DT, bool ENT, int SHAPE>
__device__ __noinline__ void put_off_row(const LossArgs& a, HeldShared& sh, int64_t row) {
  using D = Elem<DT>;
  using T = typename D::T;
  constexpr int E = D::E, kRowWarps = HeldShape<SHAPE>::kRowWarps, kRowThreads = HeldShape<SHAPE>::kRowThreads;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const T* x = static_cast<const T*>(a.logits) + row * a.row_stride;
  T* out = static_cast<T*>(a.grad_logits) + row * a.grad_stride;
  RowInfo info;
  row_scale(a, row, info.scale, info.inv_t);
  Part p = warp_running<DT, ENT, kRowThreads>(x, a.vocab, info.scale, 0, 1, tid);
  if (lane == 0) sh.again_part[warp] = p;
  row_barrier<kRowThreads>();
  if (warp == 0) {
    p = warp_join<ENT>(lane < kRowWarps ? sh.again_part[lane] : Part{-INFINITY, 0.0f, 0.0f}, info.scale);
    if (lane == 0) {
      info.target = a.targets[row];
      info.x_target = info.target < a.vocab ? D::load(x + info.target) : NAN;
      info.in = policy_in(a, row, a.weights ? a.weights[row] : 1.0f / float(a.rows));
      finish_policy_row<DT, ENT>(a, row, p, info, false, true, sh.coef);
    }
  }
  row_barrier<kRowThreads>();
  const GradRow g = sh.coef;
  if (g.zero) {
    write_zeros<DT, kRowThreads>(out, a.vocab, 0, 1);
    return;
  }
  if (((reinterpret_cast<uintptr_t>(x) ^ reinterpret_cast<uintptr_t>(out)) & 15) != 0) {
    write_elements<DT, ENT, kRowThreads>(g, x, out, a.vocab, 0, 1);
    return;
  }
  const Span sp = row_span<E>(x, a.vocab);
  const uint4* src = reinterpret_cast<const uint4*>(x + sp.head);
  uint4* dst = reinterpret_cast<uint4*>(out + sp.head);
  const int nv = int(sp.nv), at = int(g.target - sp.head);
  constexpr int kEach = 4;                // vectors ahead: in place, no load may be moved before a store
#pragma unroll 1
  for (int v = tid; v < nv; v += kEach * kRowThreads) {
    uint4 q[kEach];
#pragma unroll
    for (int i = 0; i < kEach; ++i) q[i] = src[min(v + i * kRowThreads, nv - 1)];
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      if (v + i * kRowThreads >= nv) break;
      float f[E];
      D::unpack(q[i], f);
#pragma unroll
      for (int j = 0; j < E; ++j) f[j] = (v + i * kRowThreads) * E + j == at ? g.at : grad_value<DT, ENT>(g, f[j]);
      dst[v + i * kRowThreads] = D::pack(f);
    }
  }
  const int64_t tail = sp.head + sp.nv * E + tid;
  if (tid < sp.head) grad_element<DT, ENT>(g, D::load(x + tid), out, tid);
  if (tail < a.vocab) grad_element<DT, ENT>(g, D::load(x + tail), out, tail);
}

// Those rows, when the others are done: a target that is all but impossible, one
// that is unlikely in a row of little entropy, or 16-bit logits past kNearOffset,
// which a low temperature makes of all rows.  The first of them are listed, and
// all are marked by a log2 S that no row has.  Calls of their own, so that the
// registers of the row loop are not shared with them.
constexpr float kPutOff = -INFINITY;
template <int DT, bool ENT, int SHAPE>
__device__ __noinline__ void put_off_rows(const LossArgs& a, HeldShared& sh, unsigned cluster, unsigned clusters) {
  const int count = sh.put_off;
  if (count <= kPutOffList) {
    for (int i = 0; i < count; ++i) put_off_row<DT, ENT, SHAPE>(a, sh, sh.put_off_row[i]);
    return;
  }
  RowWalk walk;
  while (walk.base < a.rows) {
    walk.step(a, cluster, clusters);
    for (uint32_t mine = walk.mine & walk.mine_alive; mine; mine &= mine - 1) {
      const int64_t row = walk.base - 32 + __ffs(mine) - 1;
      // every thread reads the mark before the first of the row's barriers, behind which it goes
      if (a.stats[2 * row + 1] == kPutOff) put_off_row<DT, ENT, SHAPE>(a, sh, row);
    }
  }
}

// A wait of the block's ran out: rows of its cluster are left over, and may be
// half written.  All of them that hold a token become NaN, and so does the loss.
template <int DT, int SHAPE>
__device__ __noinline__ void void_rows(const LossArgs& a, unsigned cluster, unsigned clusters) {
  using T = typename Elem<DT>::T;
  constexpr int kRowThreads = HeldShape<SHAPE>::kRowThreads;
  RowWalk walk;
  while (walk.base < a.rows) {
    walk.step(a, cluster, clusters);
    for (uint32_t mine = walk.mine; mine; mine &= mine - 1) {
      const int i = __ffs(mine) - 1;
      const int64_t row = walk.base - 32 + i;
      T* out = static_cast<T*>(a.grad_logits) + row * a.grad_stride;
      if (!((walk.mine_alive >> i) & 1)) {
        if (threadIdx.x == 0) write_dead_row<kPolicy>(a, row);
        write_zeros<DT, kRowThreads>(out, a.vocab, 0, 1);
        continue;
      }
      if (threadIdx.x == 0) {
        a.logprobs[row] = a.row_loss[row] = a.row_grad[row] = a.row_grad[a.rows + row] = NAN;
        a.stats[2 * row] = a.stats[2 * row + 1] = NAN;
        if (a.entropy) a.entropy[row] = NAN;
        if (a.kl) a.kl[row] = NAN;
      }
      for (int64_t j = threadIdx.x; j < a.vocab; j += kRowThreads) Elem<DT>::store(out + j, NAN);
    }
  }
}

template <int DT, bool ENT, int SHAPE>
__global__ void __launch_bounds__(HeldShape<SHAPE>::kThreads, HeldShape<SHAPE>::kBlocks)
    policy_kernel(const __grid_constant__ LossArgs a) {
  let_next_start();
  using D = Elem<DT>;
  using T = typename D::T;
  using H = HeldShape<SHAPE>;
  constexpr int kRowWarps = H::kRowWarps, kRowThreads = H::kRowThreads;
  constexpr int E = D::E, kHold = H::kHold, kSlots = H::kSlots, kLaneVecs = H::kLaneVecs, kChunkVecs = H::kChunkVecs;
  __shared__ HeldShared sh;
  extern __shared__ __align__(128) uint4 ring[];
  cg::cluster_group cluster = cg::this_cluster();
  const int blocks = int(cluster.num_blocks()), rank = int(cluster.block_rank());
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, tid = threadIdx.x;
  const int shift = 31 - __clz(blocks);           // blocks is a power of two
  if (tid < kSlots) {
    mbar_init(&sh.full[tid], 1);
    mbar_init(&sh.empty[tid], kRowWarps);
  }
  if (tid == 0) {
    mbar_init(&sh.bar[0], 1);
    mbar_init(&sh.bar[1], 1);
    sh.put_off = 0;
  }
  fence_mbar_init();
  __syncthreads();
  if (blocks > 1) cluster.sync();       // the peers' barriers exist
  const auto logits_row = [&](int64_t row) { return static_cast<const T*>(a.logits) + row * a.row_stride; };

  bool bad = false;               // a wait ran out: the same in every row warp once they have left their loop
  if (warp == kRowWarps) {
    // ------------------------------------------------------------ producer warp
    const uint64_t policy = l2_policy_evict_first();
    RowWalk walk;
    int slot = 0;
    uint32_t phase = 1;                 // the first round finds the slots empty
    RowInfo mine = {};                  // lane i: of the i-th of 32 rows
    for (bool end = false; !end && !bad;) {
      while (walk.mine == 0 && walk.base < a.rows) {
        walk.step(a, blockIdx.x >> shift, gridDim.x >> shift);
        if ((walk.mine >> lane) & 1) {
          mine.row = walk.base - 32 + lane;
          mine.alive = (walk.mine_alive >> lane) & 1;
          if (mine.alive) {
            mine.target = a.targets[mine.row];
            row_scale(a, mine.row, mine.scale, mine.inv_t);
            mine.in = policy_in(a, mine.row, a.weights ? a.weights[mine.row] : 1.0f / float(a.rows));
            mine.x_target = mine.target < a.vocab ? D::load(logits_row(mine.row) + mine.target) : NAN;
          }
        }
      }
      end = walk.mine == 0;
      const int of = end ? 0 : __ffs(walk.mine) - 1;
      walk.mine &= walk.mine - 1;
      const int64_t row = __shfl_sync(~0u, mine.row, of);
      Share s = {};
      const uint4* src = nullptr;
      if (!end && __shfl_sync(~0u, mine.alive, of)) {
        const T* x = logits_row(row);
        s = row_share<E>(x, int(a.vocab), rank, shift);
        src = reinterpret_cast<const uint4*>(x + s.head) + s.v0;
      }
      int at = 0;
      do {                              // a row has one chunk at least: it carries the row's numbers
        bad = __any_sync(~0u, !mbar_wait_running(&sh.empty[slot], phase));
        if (bad) break;
        if (at == 0 && lane == of) {
          sh.info[slot] = mine;
          if (end) sh.info[slot].row = -1;
        }
        __syncwarp();
        if (lane == 0) {
          const uint32_t bytes = uint32_t(min(kChunkVecs, s.n - at)) * 16;
          mbar_arrive_expect_tx(&sh.full[slot], bytes);
          if (bytes) bulk_g2s(ring + slot * kChunkVecs, src + at, bytes, &sh.full[slot], policy);
        }
        at += kChunkVecs;
        if (++slot == kSlots) {
          slot = 0;
          phase ^= 1;
        }
      } while (at < s.n);
    }
    // the copies end before the block does: those of this round, and of the last in the slots from `slot` on
    for (int i = 0; i < kSlots; ++i) mbar_wait_running(&sh.full[i], i < slot ? phase ^ 1 : phase);
  } else {
    // --------------------------------------------------------------- row warps
    uint32_t joined = 0, phase = 0;
    int slot = 0;
    uint4 held[kHold ? kHold : 1][kLaneVecs];
    // Rows whose stride is whole vectors all start at the same phase: the share is looked up anew only for another.
    Share s = {};
    int edge_at = -1;
    uint32_t start = ~0u;
    while (true) {
      // ---- the row's sums, chunk after chunk as they land
      const int first_slot = slot;
      F2 sum[2] = {0, 0}, u[2] = {0, 0};
      if (!bad) bad = !mbar_wait_running(&sh.full[slot], phase);
      bad = __any_sync(~0u, bad);
      const int64_t row = bad ? -1 : sh.info[first_slot].row;
      if (row == a.give_up && warp == kRowWarps - 1 && rank == blocks - 1) bad = true;
      if (row < 0 || bad) {       // the rows are done, or a wait ran out: all warps leave at the same barrier
        bad = row_barrier_any<kRowThreads>(bad);
        break;
      }
      const T* x = logits_row(row);
      T* out = static_cast<T*>(a.grad_logits) + row * a.grad_stride;
      if (!sh.info[first_slot].alive) {
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh.empty[slot]);
        if (++slot == kSlots) {
          slot = 0;
          phase ^= 1;
        }
        if (rank == 0 && tid == 0) write_dead_row<kPolicy>(a, row);
        write_zeros<DT, kRowThreads>(out, a.vocab, rank, blocks);
        continue;
      }
      if ((uint32_t(reinterpret_cast<uintptr_t>(x)) & 15) != start) {
        start = uint32_t(reinterpret_cast<uintptr_t>(x)) & 15;
        s = row_share<E>(x, int(a.vocab), rank, shift);
        // the element of this thread outside the row's vectors: the first block's threads 0.. hold those before,
        // the last one's threads 16.. those after
        const int nv = (int(a.vocab) - s.head) / E, tail = s.head + nv * E + tid - 16;
        edge_at = rank == 0 && tid < s.head ? tid : rank == blocks - 1 && tid >= 16 && tail < int(a.vocab) ? tail : -1;
      }
      const float edge = edge_at >= 0 ? D::load(x + edge_at) : -INFINITY;
      const float scale = sh.info[first_slot].scale, c = row_offset<DT>(sh.info[first_slot].x_target, scale);
      const auto scaled = ScaledPairs<DT>::of(c, scale);
      RowInfo info;
      if (warp == 0) info = sh.info[first_slot];
      const auto take = [&](int at, uint4 (&q)[kLaneVecs]) {      // the chunk at vector `at` of the share
        if (at > 0 && !bad) bad = !mbar_wait_running(&sh.full[slot], phase);
        const uint4* src = ring + slot * kChunkVecs + tid;
        if (at + kChunkVecs <= s.n) {
#pragma unroll
          for (int i = 0; i < kLaneVecs; ++i) q[i] = src[i * kRowThreads];
#pragma unroll
          for (int i = 0; i < kLaneVecs; ++i) add_vector<DT, ENT>(q[i], scaled, sum[i & 1], u[i & 1]);
        } else {
#pragma unroll
          for (int i = 0; i < kLaneVecs; ++i)
            if (at + i * kRowThreads + tid < s.n) {
              q[i] = src[i * kRowThreads];
              add_vector<DT, ENT>(q[i], scaled, sum[i & 1], u[i & 1]);
            }
        }
      };
      const auto advance = [&]() {
        if (++slot == kSlots) {
          slot = 0;
          phase ^= 1;
        }
      };
      const auto hand_back = [&](int chunk) {
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh.empty[chunk]);
      };
#pragma unroll
      for (int j = 0; j < kHold; ++j)
        if (j == 0 || j * kChunkVecs < s.n) {
          take(j * kChunkVecs, held[j]);
          hand_back(slot);
          advance();
        }
      const int ring_slot = slot;
      for (int at = kHold * kChunkVecs; at < s.n || at == 0; at += kChunkVecs) {
        uint4 q[kLaneVecs];
        take(at, q);
        advance();
      }
      {
        const float t = scaled_one<DT>(edge, c, scale), e = ex2_approx(t);
        float lo, hi;
        split(add2(sum[0], sum[1]), lo, hi);
        const float total = warp_sum(lo + hi + e);
        split(add2(u[0], u[1]), lo, hi);
        const float mean = ENT ? warp_sum(lo + hi + e * fmaxf(t, -200.0f)) : 0.0f;
        bad = __any_sync(~0u, bad);
        if (lane == 0) sh.warp_part[warp] = make_float2(total, mean);
      }
      if (row_barrier_any<kRowThreads>(bad)) {
        bad = true;               // some warp's wait ran out
        break;
      }
      // ---- joined, and turned into the row's numbers, by the first warp
      if (warp == 0) {
        float2 v = lane < kRowWarps ? sh.warp_part[lane] : make_float2(0.0f, 0.0f);
        Part p = {c, warp_sum(v.x), ENT ? warp_sum(v.y) : 0.0f};
        if (blocks > 1) {
          // a peer may be one join ahead of this block, never two: two barriers take turns
          const int turn = int(joined & 1);
          if (lane == 0) mbar_arrive_expect_tx(&sh.bar[turn], uint32_t(blocks) * 8);
          __syncwarp();
          if (lane < blocks) send(peer_addr(&sh.part[turn][rank], lane), p.s, p.u, peer_addr(&sh.bar[turn], lane));
          if (!bad) bad = __any_sync(~0u, !mbar_wait_running(&sh.bar[turn], (joined >> 1) & 1));
          ++joined;
          v = lane < blocks ? sh.part[turn][lane] : make_float2(0.0f, 0.0f);
          p.s = warp_sum(v.x);
          if (ENT) p.u = warp_sum(v.y);
        }
        if (bad) p.s = NAN;             // a wait ran out: the row has no result
        if (lane == 0) {
          if (sums_far<ENT>(p)) {       // the same for the whole cluster
            sh.coef.later = true;
            if (rank == 0) a.stats[2 * row + 1] = kPutOff;
            if (sh.put_off < kPutOffList) sh.put_off_row[sh.put_off] = int(row);
            ++sh.put_off;
          } else {
            finish_policy_row<DT, ENT>(a, row, p, info, true, rank == 0, sh.coef);
          }
        }
      }
      row_barrier<kRowThreads>();
      // ---- its gradient; every chunk goes to the next row as it is done
      const GradRow g = sh.coef;
      if (edge_at >= 0 && !g.later) {
        if (g.zero)
          D::store(out + edge_at, 0.0f);
        else
          grad_element<DT, ENT>(g, edge, out, edge_at);
      }
      T* mine = out + s.head + int64_t(s.v0) * E;
      const auto write = [&](const auto& put) {
        int chunk = ring_slot;
        for (int at = kHold * kChunkVecs; at < s.n || at == 0; at += kChunkVecs) {
          const uint4* q = ring + chunk * kChunkVecs + tid;
#pragma unroll
          for (int i = 0; i < kLaneVecs; ++i)
            if (at + i * kRowThreads + tid < s.n) put(q[i * kRowThreads], at + i * kRowThreads + tid);
          hand_back(chunk);
          if (++chunk == kSlots) chunk = 0;
        }
#pragma unroll
        for (int j = 0; j < kHold; ++j)
#pragma unroll
          for (int i = 0; i < kLaneVecs; ++i)
            if (const int v = j * kChunkVecs + i * kRowThreads + tid; v < s.n) put(held[j][i], v);
      };
      uint4* dst = reinterpret_cast<uint4*>(mine);
      const GradPairs<DT> pairs(g);
      const bool same = ((reinterpret_cast<uintptr_t>(x) ^ reinterpret_cast<uintptr_t>(out)) & 15) == 0;
      if (g.later) {
        write([](const uint4&, int) {});
      } else if (!same || (DT != NS_DTYPE_F32 && g.wide)) {
        // the rows start on different 16-byte phases, or the row is wide: element by element
        write([&](const uint4& q, int v) {
          float f[E];
          D::unpack(q, f);
#pragma unroll
          for (int i = 0; i < E; ++i) D::store(mine + v * E + i, g.zero ? 0.0f : grad_value<DT, ENT>(g, f[i]));
        });
      } else if (g.zero) {
        write([&](const uint4&, int v) { dst[v] = make_uint4(0, 0, 0, 0); });
      } else {
        write([&](const uint4& q, int v) { dst[v] = grad_vector<DT, ENT>(pairs, q); });
      }
      // the target's value over its vector, by the thread that wrote it
      const unsigned target = unsigned(g.target - s.head) - unsigned(s.v0) * E;
      if (!g.zero && !g.later && target < unsigned(s.n) * E && int(target / E) % kRowThreads == tid) D::store(mine + target, g.at);
    }
    if (!bad && rank == 0 && sh.put_off) put_off_rows<DT, ENT, SHAPE>(a, sh, blockIdx.x >> shift, gridDim.x >> shift);
  }
  if (blocks > 1) cluster.sync();        // no block leaves while a peer may still write to it
  if (bad && warp < kRowWarps) void_rows<DT, SHAPE>(a, blockIdx.x >> shift, gridDim.x >> shift);
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

// `blocks`: of a cluster; one of 1 is not the same as none (policy_kernel took 3 us
// longer at 2048 x 32000 without).  `follows`: the kernel waits for the one before it by
// wait_for_previous, and may be started before that one has ended.
template <typename... Args>
int launch(void (*kernel)(Args...), int64_t grid, int threads, int blocks, size_t smem, bool follows, cudaStream_t stream,
           Args... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(unsigned(grid));
  cfg.blockDim = dim3(unsigned(threads));
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute at[1];
  cfg.attrs = at;
  if (follows) {
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.numAttrs = 1;
  } else {
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = unsigned(blocks);
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    cfg.numAttrs = 1;
  }
  return cudaLaunchKernelEx(&cfg, kernel, args...) == cudaSuccess ? NS_OK : NS_ERR_CUDA;
}

template <int DT, bool ENT, int OP>
int launch_forward(const LossArgs& a, cudaStream_t stream) {
  int sms = 0;
  if (const int rc = sm_count(&sms)) return rc;
  const int64_t vectors = a.vocab / Elem<DT>::E;
  // a warp per row while rows are short and many: 4096 x 8000 bf16 15 us against 21, 1024 x 4000 6 against 8,
  // 4096 x 16000 27 against 32, 2048 x 9000 9 against 12; even at 300 rows of 1000 vectors, at 1000 x 9000 and
  // at 2048 x 16000 (there, with entropy, 17 against 15), and worse at 2048 x 32000, 33 against 28
  if (vectors <= 1024 ? a.rows >= 2 * sms : vectors <= 2560 && 2 * a.rows >= 3 * vectors) {
    return launch(forward_rows_kernel<DT, ENT, OP>, (a.rows + kWarps - 1) / kWarps, kThreads, 1, 0, false, stream, a);
  }
  // blocks per row: enough to give every SM two, each thread at least one vector
  int blocks = 1;
  while (blocks < kMaxCluster && a.rows * blocks < 2 * sms && vectors >= int64_t(2) * blocks * kThreads) blocks *= 2;
  return launch(forward_kernel<DT, ENT, OP>, a.rows * blocks, kThreads, blocks, 0, false, stream, a);
}

template <int OP, int DT>
int forward_typed(const LossArgs& a, cudaStream_t stream) {
  if constexpr (OP == kPreference)
    return launch_forward<DT, false, OP>(a, stream);
  else
    return a.entropy ? launch_forward<DT, true, OP>(a, stream) : launch_forward<DT, false, OP>(a, stream);
}

template <int OP>
int forward(const LossArgs& a, int dtype, cudaStream_t stream) {
  switch (dtype) {
    case NS_DTYPE_F32: return forward_typed<OP, NS_DTYPE_F32>(a, stream);
    case NS_DTYPE_BF16: return forward_typed<OP, NS_DTYPE_BF16>(a, stream);
    default: return forward_typed<OP, NS_DTYPE_F16>(a, stream);
  }
}

// Blocks per row of policy_kernel: the fewest that hold a row on chip; 0 when kMaxCluster do not.
template <int SHAPE>
int held_blocks(int64_t vectors) {
  for (int blocks = 1; blocks <= kMaxCluster; blocks *= 2)
    if ((vectors + blocks - 1) / blocks <= HeldShape<SHAPE>::kMostVecs) return blocks;
  return 0;
}

template <int DT, bool ENT, int SHAPE>
int launch_policy(const LossArgs& a, int blocks, cudaStream_t stream) {
  using H = HeldShape<SHAPE>;
  static std::mutex mu;
  static int known[64][kMaxCluster + 1];         // clusters that a device holds at once
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return NS_ERR_CUDA;
  int clusters = 0;
  {
    std::lock_guard<std::mutex> lk(mu);
    if (known[dev][blocks] == 0) {
      if (cudaFuncSetAttribute(policy_kernel<DT, ENT, SHAPE>, cudaFuncAttributeMaxDynamicSharedMemorySize, H::kSmem) !=
          cudaSuccess)
        return NS_ERR_CUDA;
      cudaLaunchConfig_t cfg = {};
      cfg.gridDim = dim3(unsigned(blocks) * 64);
      cfg.blockDim = dim3(H::kThreads);
      cfg.dynamicSmemBytes = H::kSmem;
      cudaLaunchAttribute at[1];
      at[0].id = cudaLaunchAttributeClusterDimension;
      at[0].val.clusterDim.x = unsigned(blocks);
      at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
      cfg.attrs = at;
      cfg.numAttrs = 1;
      int n = 0;
      if (cudaOccupancyMaxActiveClusters(&n, policy_kernel<DT, ENT, SHAPE>, &cfg) != cudaSuccess || n < 1) return NS_ERR_CUDA;
      known[dev][blocks] = n;
    }
    clusters = known[dev][blocks];
  }
  const int64_t grid = std::min<int64_t>(a.rows, clusters) * blocks;
  return launch(policy_kernel<DT, ENT, SHAPE>, grid, H::kThreads, blocks, H::kSmem, false, stream, a);
}

template <int DT, int SHAPE>
int launch_shape(const LossArgs& a, int blocks, cudaStream_t stream) {
  return a.entropy ? launch_policy<DT, true, SHAPE>(a, blocks, stream) : launch_policy<DT, false, SHAPE>(a, blocks, stream);
}

// The gradient with the loss in one launch; `held` is false where a launch for
// the sums and one for the gradient do better (rows too short) or must (rows
// past the chip).  Measured on a B200, us by shape (large / medium / small /
// two launches):
//   2048 x 16000 bf16    53 / 46 / 36 / 39      4096 x 8000 bf16   81 / 72 / 54 / 37
//   2048 x 32000 bf16    69 / 62 / 53 / 69       777 x 64007 fp16  52 / 48 / 45 / 54
//   1000 x 100000 bf16   79 / 98 / -  / -       2048 x 151936 bf16 214 / 264 / 290 / 285
//    333 x 151936 bf16   55 / 49 / -  / 62       600 x 151936 fp32 134 / 123 / - / 170
// Short rows spend their time in joins, which more blocks of an SM hide.
// 16-bit rows are bound by their exponentials and want whole SMs without a
// cluster's join; fp32 rows and few rows want their columns spread.  A handful
// of rows is even: 16 x 32000 bf16 takes 11.0 against 9.4 in a graph, 12.3
// against 14.4 launch by launch.
template <int DT>
int policy_held(const LossArgs& a, cudaStream_t stream, bool* held) {
  int sms = 0;
  if (const int rc = sm_count(&sms)) return rc;
  const int64_t vectors = a.vocab / Elem<DT>::E;
  const int small = held_blocks<kSmall>(vectors), medium = held_blocks<kMedium>(vectors), large = held_blocks<kLarge>(vectors);
  *held = true;
  if (vectors >= 1800) {
    if (small == 1 || (small == 2 && DT != NS_DTYPE_F32)) return launch_shape<DT, kSmall>(a, small, stream);
    if (medium && (DT == NS_DTYPE_F32 || 2 * a.rows < 5 * sms)) return launch_shape<DT, kMedium>(a, medium, stream);
    if (large) return launch_shape<DT, kLarge>(a, large, stream);
  }
  *held = false;
  return NS_OK;
}

int policy_held(const LossArgs& a, int dtype, cudaStream_t stream, bool* held) {
  switch (dtype) {
    case NS_DTYPE_F32: return policy_held<NS_DTYPE_F32>(a, stream, held);
    case NS_DTYPE_BF16: return policy_held<NS_DTYPE_BF16>(a, stream, held);
    default: return policy_held<NS_DTYPE_F16>(a, stream, held);
  }
}

template <int DT>
int launch_grad(const LossArgs& a, bool follows, cudaStream_t stream) {
  const int64_t per = int64_t(kGradThreads) * kGradVecs * Elem<DT>::E;    // shares differ by one vector at most
  const int chunks = int((a.vocab + per - 1) / per);
  const int64_t blocks = a.rows * chunks;
  if (blocks > 0x7FFFFFFF) return NS_ERR_INVALID_ARGUMENT;
  return launch(a.grad_entropy ? grad_kernel<DT, true> : grad_kernel<DT, false>, blocks, kGradThreads, 1, 0, follows,
                stream, a, chunks);
}

int gradient(const LossArgs& a, int dtype, bool follows, cudaStream_t stream) {
  switch (dtype) {
    case NS_DTYPE_F32: return launch_grad<NS_DTYPE_F32>(a, follows, stream);
    case NS_DTYPE_BF16: return launch_grad<NS_DTYPE_BF16>(a, follows, stream);
    default: return launch_grad<NS_DTYPE_F16>(a, follows, stream);
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

int policy_loss(const void* logits, int dtype, int64_t rows, int64_t vocab, int64_t row_stride,
                const int64_t* targets, const float* temperature, float temperature_all,
                const float* old_logprobs, const float* ref_logprobs, const float* advantages,
                const float* weights, float clip_low, float clip_high, float kl_coef, float entropy_coef,
                float* loss, float* row_loss, float* logprobs, float* entropy, float* kl, float* stats,
                float* row_grad, void* grad_logits, int64_t grad_stride, int64_t give_up, ns_stream_t stream) {
  if (const int rc = check_rows(dtype, rows, vocab, row_stride, temperature, temperature_all)) return rc;
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
  if (grad_logits && !grad_ok(logits, row_stride, grad_logits, grad_stride, vocab)) return NS_ERR_INVALID_ARGUMENT;
  LossArgs a = row_args(logits, rows, vocab, row_stride, targets, temperature, temperature_all);
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
  a.grad_logprobs = row_grad;
  a.grad_entropy = entropy_coef != 0.0f ? row_grad + rows : nullptr;
  a.grad_logits = grad_logits;
  a.grad_stride = grad_stride;
  a.give_up = give_up;
  bool held = false;
  if (grad_logits)
    if (const int rc = policy_held(a, dtype, s, &held)) return rc;
  if (!held) {
    if (const int rc = forward<kPolicy>(a, dtype, s)) return rc;
    if (grad_logits)
      if (const int rc = gradient(a, dtype, true, s)) return rc;
  }
  return launch(policy_sum_kernel, 1, 1024, 1, 0, true, s, a, loss);
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
  return ns::gradient(a, dtype, false, reinterpret_cast<cudaStream_t>(stream));
}

int ns_policy_loss(const void* logits, int dtype, int64_t rows, int64_t vocab, int64_t row_stride,
                   const int64_t* targets, const float* temperature, float temperature_all,
                   const float* old_logprobs, const float* ref_logprobs, const float* advantages,
                   const float* weights, float clip_low, float clip_high, float kl_coef, float entropy_coef,
                   float* loss, float* row_loss, float* logprobs, float* entropy, float* kl, float* stats,
                   float* row_grad, void* grad_logits, int64_t grad_stride, ns_stream_t stream) {
  return ns::policy_loss(logits, dtype, rows, vocab, row_stride, targets, temperature, temperature_all, old_logprobs,
                         ref_logprobs, advantages, weights, clip_low, clip_high, kl_coef, entropy_coef, loss, row_loss,
                         logprobs, entropy, kl, stats, row_grad, grad_logits, grad_stride, ns::kGiveUpNever, stream);
}

int ns_policy_loss_debug(const void* logits, int dtype, int64_t rows, int64_t vocab, int64_t row_stride,
                         const int64_t* targets, const float* temperature, float temperature_all,
                         const float* old_logprobs, const float* ref_logprobs, const float* advantages,
                         const float* weights, float clip_low, float clip_high, float kl_coef, float entropy_coef,
                         float* loss, float* row_loss, float* logprobs, float* entropy, float* kl, float* stats,
                         float* row_grad, void* grad_logits, int64_t grad_stride, int64_t give_up,
                         ns_stream_t stream) {
  if (give_up < 0) return NS_ERR_INVALID_ARGUMENT;
  return ns::policy_loss(logits, dtype, rows, vocab, row_stride, targets, temperature, temperature_all, old_logprobs,
                         ref_logprobs, advantages, weights, clip_low, clip_high, kl_coef, entropy_coef, loss, row_loss,
                         logprobs, entropy, kl, stats, row_grad, grad_logits, grad_stride, give_up, stream);
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
  if (const int rc = ns::launch(ns::pair_kernel, 1, 1024, 1, 0, rows > 0, s, a, beta, label_smoothing, average, loss,
                                pair_loss, rewards))
    return rc;
  if (!grad_logits || rows == 0) return NS_OK;
  a.grad_logprobs = row_grad;
  a.grad_logits = grad_logits;
  a.grad_stride = grad_stride;
  return ns::gradient(a, dtype, true, s);
}

}  // extern "C"
