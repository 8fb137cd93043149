// Log-probabilities of target tokens and the losses built on them.
//
//   logp_t = x_y - log sum_j exp(x_j)                     token_logprobs
//   policy:      r = exp(logp - old),  d = ref - logp
//                L = 1/N sum_t m_t (-min(r A, clip(r, 1 - lo, 1 + hi) A) + beta (e^d - 1 - d))
//   preference:  s_i = sum_t m_t (logp - ref),  h = beta (s_chosen - s_rejected)
//                L = mean over pairs of -((1 - e) log sigmoid(h) + e log sigmoid(-h))
//   gradient of any of them: dx_j = c_t ([j == y] - softmax(x)_j), c_t = dL / dlogp_t
//
// One pass over the logits forward (running maximum m and sum s per thread, joined over the
// row), one read and one write backward; policy_loss, whose coefficients hang on their own row
// only, writes the gradient with the loss and reads the logits once. The statistics kept between
// the two are (m, s) and not the log-sum-exp: exp(x - m) / s has no large terms that cancel, so
// its relative error does not grow with the size of the logits. What follows from a row's logp
// (ratio, KL estimate, their derivatives) is computed in 64 bits by the one thread that joins the
// row, from x_y - m and s: differences of log-probabilities nearly cancel, and rounding them first
// would be what is lost. Rows that do not count are not read.
//
// Bound by memory, with the exponentials (16 a cycle and SM) close behind: arithmetic is packed, two fp32 values to an
// instruction, and 16-bit logits are added to fp32 without unpacking. Measured on one B200 (6.45 TB/s copied), between
// events around queued calls, the launches' gaps and the small kernels among them:
//   scoring 4096 rows of 32000 bf16        48 us, 5.5 TB/s (262 MB); fp32 78 us, 6.7 TB/s
//   policy loss and gradient, 4096 rows of 128256 bf16, a quarter masked
//                                         364 us, 5.1 TB/s (1.84 GB; in two passes 418); 677 for a loss gradient that is not
//                                         1, for which the gradient is computed again
//   preference loss and gradient, 4096 rows of 32000 bf16, 40 % masked
//                                         113 us, 5.1 TB/s (577 MB: the logits are read twice, as a coefficient hangs on the
//                                         sums of both sequences); fp32 218 us
#include <ATen/ATen.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAException.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAGraphsC10Utils.h>
#include <cooperative_groups.h>

#include "train_ops.h"
#include "vec.cuh"

namespace dmb {
namespace {

namespace cg = cooperative_groups;

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLog2eUp = 1.4426951408386230f;  // the next larger fp32
// ex2.approx comes out low, by 2e-8 to 5e-8 of its value on average (measured). An exponent larger by 3.5e-8 takes that back:
// as the addend of the product that is the exponent it acts in the product's one rounding, and an exponent of 0 still gives 1.
// What is left of logp's mean error, for 64 to 128256 logits of a deviation of 0.5 to 2: at most 7e-9, where fp32 operations
// with expf throughout leave 6e-9 (16e-9 before, with the sum corrected afterwards).
constexpr float kLift = 3.5e-8f;
constexpr int kUnroll = 4;         // 8-element vectors that a thread takes at once
constexpr int kWarpRows = 4;       // rows of a CTA whose warps have one each

enum Mode { kLogprob, kPolicy, kPreference };

// A row's part of the policy loss. The loss is in 64 bits, as rows may cancel in the sum; 16 bytes for one load.
struct alignas(16) RowLoss {
  double loss;
  float kl;
  int clipped;
};

struct RowArgs {
  const void* logits;
  long long stride_b, stride_s;  // elements
  int seq;                       // rows per stride_b
  int rows, vocab;
  const int64_t* targets;
  const bool* mask;  // null: every row counts
  float* logp;
  float2* stats;  // (m, s) of each row
  int* error;
  // policy and preference
  const float *old_logp, *advantages, *ref_logp;
  double clip_low, clip_high, kl_coef;
  const int* count;  // rows that the mask keeps; null: all
  RowLoss* row_loss;
  float* coef;
  double* row_diff;
  void* grad;  // contiguous; null: no gradient
};

// Only of values that are at most 0, as they are taken against a maximum. Results below 2^-126 become 0: next to the
// maximum's own 1 they add nothing to a sum, and a probability that small is below what a gradient can hold.
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ F2 ex2(F2 x) {
  const float2 v = f2_values(x);
  return f2(ex2(v.x), ex2(v.y));
}

// What exponents are taken against: a row (or part) of nothing but -inf has no finite maximum.
__device__ __forceinline__ float anchor(float m) { return m == -INFINITY ? 0.f : m; }

// Joins two parts. expf and not ex2: what a sum is multiplied with again and again should not lean to one side. (With ex2 and
// kLift a row's logp comes out low by up to 4e-8: next to an exponent of 0 that is too much.)
__device__ __forceinline__ void join(float& m, float& s, float m2, float s2) {
  const float mx = fmaxf(m, m2), a = anchor(mx);
  s = (m == mx ? s : s * expf(m - a)) + (m2 == mx ? s2 : s2 * expf(m2 - a));
  m = mx;
}

// A warp's parts joined: the maximum first, so that each sum is scaled once. Every lane gets the result.
__device__ __forceinline__ void warp_join(float& m, float& s) {
  float mx = m;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(~0u, mx, o));
  s *= expf(m - anchor(mx));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(~0u, s, o);
  m = mx;
}

template <typename T>
__device__ __forceinline__ const T* row_of(const void* logits, long long stride_b, long long stride_s, int seq, int row) {
  const unsigned b = (unsigned)row / (unsigned)seq, s = row - b * seq;
  return static_cast<const T*>(logits) + b * stride_b + s * stride_s;
}

// Elements in front of a row's first 16-byte boundary.
template <typename T>
__device__ __forceinline__ int head_of(const T* p, int n) {
  const int h = (int)(((16 - (reinterpret_cast<uintptr_t>(p) & 15)) & 15) / sizeof(T));
  return min(h, n);
}

template <typename T>
__device__ __forceinline__ Raw8<T> raw_neg_inf() {
  Raw8<T> r;
  const uint32_t w = sizeof(T) == 4 ? 0xFF800000u : std::is_same<T, __nv_bfloat16>::value ? 0xFF80FF80u : 0xFC00FC00u;
#pragma unroll
  for (int i = 0; i < (int)sizeof(T) / 2; ++i) r.w[i] = make_uint4(w, w, w, w);
  return r;
}

// The largest of a thread's vectors; NaN is left out here and comes through the sum. 16-bit types two at a time.
template <typename T>
__device__ __forceinline__ float max_of(const Raw8<T> (&raw)[kUnroll]) {
  if constexpr (sizeof(T) == 4) {
    float mx = -INFINITY;
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      float f[8];
      unpack8<T>(raw[u], f);
#pragma unroll
      for (int k = 0; k < 8; ++k) mx = fmaxf(mx, f[k]);
    }
    return mx;
  } else {
    using T2 = std::conditional_t<std::is_same<T, __nv_bfloat16>::value, __nv_bfloat162, __half2>;
    T2 mx = reinterpret_cast<const T2&>(raw[0].w[0].x);
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const uint4& w = raw[u].w[0];
      mx = __hmax2(__hmax2(mx, __hmax2(reinterpret_cast<const T2&>(w.x), reinterpret_cast<const T2&>(w.y))),
                   __hmax2(reinterpret_cast<const T2&>(w.z), reinterpret_cast<const T2&>(w.w)));
    }
    const float lo = to_float(mx.x), hi = to_float(mx.y);
    return fmaxf(fmaxf(-INFINITY, lo), hi);
  }
}

// Adds kUnroll vectors of a thread to its maximum and sum.
template <typename T>
__device__ __forceinline__ void scan_vectors(const Raw8<T> (&raw)[kUnroll], float& m, float& s) {
  const float mx = fmaxf(m, max_of<T>(raw)), a = anchor(mx);
  if (mx != m) s *= expf(m - a);
  m = mx;
  // log2 e in 32 bits is 1.3e-8 of itself too small, which shifts every log-probability to the same side by that times its
  // distance from the mean logit; the next larger number is 6.9e-8 too large. One value in eight with that one leaves 3e-9.
  const F2 c = f2(kLog2e, kLog2e), up = f2(kLog2e, kLog2eUp), lift = f2(kLift, kLift);
  F2 sum[2] = {f2(0.f, 0.f), f2(0.f, 0.f)};
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) {
    F2 v[4];
    add_f2<T>(raw[u], -a, v);
#pragma unroll
    for (int k = 0; k < 4; ++k) sum[k & 1] = sum[k & 1] + ex2(fma2(v[k], k == 3 ? up : c, lift));
  }
  const float2 x = f2_values(sum[0] + sum[1]);
  s += x.x + x.y;
}

// kUnroll of a thread's vectors: at base, base + nt ..., -inf from v1 on.
template <typename T>
__device__ __forceinline__ void load_group(Raw8<T> (&raw)[kUnroll], const T* p, int base, int v1, int nt) {
#pragma unroll
  for (int u = 0; u < kUnroll; ++u) {
    const int v = base + u * nt;
    raw[u] = v < v1 ? load_raw8<T>(p + (long long)v * 8) : raw_neg_inf<T>();
  }
}

// Adds the vectors [v0, v1) of p, of which thread `tid` of `nt` takes every nt-th, to its maximum and sum.
template <typename T>
__device__ __forceinline__ void scan_row(const T* p, int v0, int v1, int tid, int nt, float& m, float& s) {
  for (int base = v0 + tid; base < v1; base += nt * kUnroll) {
    Raw8<T> raw[kUnroll];
    load_group<T>(raw, p, base, v1, nt);
    scan_vectors<T>(raw, m, s);
  }
}

// The values that no vector covers: `head` in front, and those behind the last of `vecs` vectors.
template <typename T>
__device__ __forceinline__ void scan_ends(const T* p, int n, int head, int vecs, int tid, int nt, float& m, float& s) {
  const int tail = head + vecs * 8;
  for (int j = tid; j < head + (n - tail); j += nt) join(m, s, to_float(p[j < head ? j : tail + j - head]), 1.f);
}

// What one thread does once a row's maximum and sum are known. Returns the derivative of the loss by logp, for kPolicy.
template <Mode MODE>
__device__ __forceinline__ float finish_row(const RowArgs& a, int row, float xy, float m, float s) {
  const double lp = ((double)xy - (double)anchor(m)) - log((double)s);
  a.logp[row] = (float)lp;
  a.stats[row] = make_float2(isnan(xy) ? xy : anchor(m), s);  // a target outside the vocabulary: NaN for the gradient too
  if constexpr (MODE == kPolicy) {
    const double adv = a.advantages[row], ratio = exp(lp - (double)a.old_logp[row]);
    const double held_ratio = ratio < 1.0 - a.clip_low ? 1.0 - a.clip_low : ratio > 1.0 + a.clip_high ? 1.0 + a.clip_high : ratio;
    const double open = ratio * adv, held = held_ratio * adv;
    const bool clipped = open > held;
    double loss = -(clipped ? held : open), coef = clipped ? 0.0 : -open, kl = 0.0;
    if (a.ref_logp) {
      const double d = (double)a.ref_logp[row] - lp, e = expm1(d);
      kl = e - d;
      if (a.kl_coef != 0) {
        loss += a.kl_coef * kl;
        coef -= a.kl_coef * e;
      }
    }
    a.row_loss[row] = RowLoss{loss, (float)kl, clipped};
    coef *= a.count ? (*a.count > 0 ? 1.0 / *a.count : 0.0) : 1.0 / a.rows;
    a.coef[row] = (float)coef;
    return (float)coef;
  }
  if constexpr (MODE == kPreference) a.row_diff[row] = lp - (double)a.ref_logp[row];
  return 0.f;
}

template <Mode MODE>
__device__ __forceinline__ void skip_row(const RowArgs& a, int row) {
  a.logp[row] = 0.f;
  a.stats[row] = make_float2(0.f, 1.f);
  if constexpr (MODE == kPolicy) {
    a.row_loss[row] = RowLoss{0.0, 0.f, 0};
    a.coef[row] = 0.f;
  }
  if constexpr (MODE == kPreference) a.row_diff[row] = 0.0;
}

template <typename T>
__device__ __forceinline__ float target_logit(const RowArgs& a, const T* p, int64_t y) {
  if (y < 0 || y >= a.vocab) {
    atomicExch(a.error, (int)kErrBadIndex);
    return NAN;
  }
  return to_float(p[y]);
}

// Gradient of one vector; `hot` is the target's place in it, if it has one in 0..7.
template <typename T>
__device__ __forceinline__ void grad_vector(const Raw8<T>& raw, T* to, bool aligned, float m, float neg, int hot, float c) {
  const F2 scale = f2(kLog2e, kLog2e), factor = f2(neg, neg);
  F2 f[4];
  add_f2<T>(raw, -m, f);
#pragma unroll
  for (int k = 0; k < 4; ++k) f[k] = factor * ex2(f[k] * scale);
  if ((unsigned)hot < 8u) {
#pragma unroll
    for (int k = 0; k < 4; ++k) f[k] = f[k] + f2(2 * k == hot ? c : 0.f, 2 * k + 1 == hot ? c : 0.f);
  }
  const Raw8<T> out = pack_f2<T>(f);
  if (aligned) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) reinterpret_cast<uint4*>(to)[i] = out.w[i];
  } else {  // the gradient's rows lie on other boundaries than the logits'
#pragma unroll
    for (int k = 0; k < 8; ++k) to[k] = reinterpret_cast<const T*>(&out)[k];
  }
}

// The ends that no vector covers.
template <typename T>
__device__ __forceinline__ void grad_ends(const T* p, T* g, int n, int head, int vecs, int tid, int nt, float m, float neg,
                                          int y, float c) {
  const int tail = head + vecs * 8;
  for (int i = tid; i < head + (n - tail); i += nt) {
    const int j = i < head ? i : tail + i - head;
    g[j] = from_float<T>(fmaf(neg, ex2((to_float(p[j]) - m) * kLog2e), j == y ? c : 0.f));
  }
}

// Zeros in a share of g[0, n).
template <typename T>
__device__ __forceinline__ void fill_zero(T* g, int n, int share, int shares, int tid, int nt) {
  const int head = head_of(g, n), vecs = (n - head) / 8, tail = head + vecs * 8;
  const float zero[8] = {};
  const int each = ((unsigned)vecs + shares - 1) / (unsigned)shares, v1 = min((share + 1) * each, vecs);
  for (int v = share * each + tid; v < v1; v += nt) store8t<T>(g + head + (long long)v * 8, zero);
  if (share == 0)
    for (int j = tid; j < head + (n - tail); j += nt) g[j < head ? j : tail + j - head] = from_float<T>(0.f);
}

// Gradient of the vectors [v0, v1) of p; `raw` holds the thread's first ones.
template <typename T>
__device__ __forceinline__ void grad_row(Raw8<T> (&raw)[kUnroll], const T* p, T* g, int v0, int v1, int tid, int nt, float m,
                                         float neg, int hot, float c) {
  const bool aligned = (reinterpret_cast<uintptr_t>(g) & 15) == 0;
  int base = v0 + tid;
  auto write = [&] {
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int v = base + u * nt;
      if (v < v1) grad_vector<T>(raw[u], g + (long long)v * 8, aligned, m, neg, hot - v * 8, c);
    }
  };
  write();
  for (base += nt * kUnroll; base < v1; base += nt * kUnroll) {
    load_group<T>(raw, p, base, v1, nt);
    write();
  }
}

// One warp per row, for short rows. With GRAD the row's gradient follows at once.
template <typename T, Mode MODE, bool GRAD>
__global__ void __launch_bounds__(32 * kWarpRows) warp_row_kernel(const RowArgs a) {
  const int row = blockIdx.x * kWarpRows + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (row >= a.rows) return;
  T* g = GRAD ? static_cast<T*>(a.grad) + (long long)row * a.vocab : nullptr;
  if (a.mask && !a.mask[row]) {
    if (lane == 0) skip_row<MODE>(a, row);
    if (GRAD) fill_zero<T>(g, a.vocab, 0, 1, lane, 32);
    return;
  }
  const T* p = row_of<T>(a.logits, a.stride_b, a.stride_s, a.seq, row);
  const int head = head_of(p, a.vocab), vecs = (a.vocab - head) / 8;
  const int64_t y = a.targets[row];
  const float xy = lane == 0 ? target_logit(a, p, y) : 0.f;
  float m = -INFINITY, s = 0.f;
  scan_row<T>(p + head, 0, vecs, lane, 32, m, s);
  scan_ends<T>(p, a.vocab, head, vecs, lane, 32, m, s);
  warp_join(m, s);
  float c = 0.f;
  if (lane == 0) c = finish_row<MODE>(a, row, xy, m, s);
  if constexpr (GRAD) {
    c = __shfl_sync(~0u, c, 0);
    if (c == 0.f) {
      fill_zero<T>(g, a.vocab, 0, 1, lane, 32);
      return;
    }
    const int hot = y >= 0 && y < a.vocab ? (int)y - head : -8;
    Raw8<T> raw[kUnroll];
    load_group<T>(raw, p + head, lane, vecs, 32);
    grad_row<T>(raw, p + head, g + head, 0, vecs, lane, 32, anchor(m), -c / s, hot, c);
    grad_ends<T>(p, g, a.vocab, head, vecs, lane, 32, anchor(m), -c / s, (int)y, c);
  }
}

constexpr int kRowThreads = 256;
// With GRAD a row is split until a part is no longer than this: fewer rows at once, which are still in the L2 when the
// gradient is written. 4096 rows of 128256 bf16 logits, a quarter of them masked, take 364 us in four parts, 443 in two, 480
// in one (each row then comes from memory twice), and 420 in eight, which have too little to do between two barriers.
constexpr int kGradPart = 80 * 1024;

// A cluster of CTAs per row, most often of one: with fewer rows than the GPU has room for a row is split, and the parts are
// joined through the first CTA's shared memory. With GRAD the row's gradient follows at once, while the row is in the L2.
// Registers for six CTAs to an SM, five for fp32, which the compiler does not come to by itself. With GRAD the rows above
// take 364 us so, 382 with four and 435 with eight (which spill); 4096 rows of 32000 take 48 us without GRAD, 49 with four and
// 51 with eight.
template <typename T, Mode MODE, bool GRAD>
__global__ void __launch_bounds__(kRowThreads, sizeof(T) == 2 ? 6 : 5) row_kernel(const RowArgs a) {
  constexpr int NT = kRowThreads;
  __shared__ float2 warps[NT / 32];
  __shared__ float2 parts[8];  // of the cluster's CTAs, in the first one
  __shared__ float3 known;     // m, -c / s and c, for GRAD
  cg::cluster_group cluster = cg::this_cluster();
  const unsigned split = cluster.num_blocks();
  const int rank = cluster.block_rank(), tid = threadIdx.x;
  const int row = blockIdx.x / split;
  T* g = GRAD ? static_cast<T*>(a.grad) + (long long)row * a.vocab : nullptr;
  if (a.mask && !a.mask[row]) {  // the whole cluster leaves
    if (GRAD) fill_zero<T>(g, a.vocab, rank, split, tid, NT);
    if (rank == 0 && tid == 0) skip_row<MODE>(a, row);
    return;
  }
  if (split > 1) cluster.barrier_arrive();  // waited for below: all have begun before one writes to another
  const T* p = row_of<T>(a.logits, a.stride_b, a.stride_s, a.seq, row);
  const int head = head_of(p, a.vocab), vecs = (a.vocab - head) / 8;
  const int each = (vecs + split - 1) / split, v0 = min(rank * each, vecs), v1 = min(v0 + each, vecs);
  if (GRAD && tid == 0 && v1 > v0)  // the whole part to the L2, at once: 383 to 364 us. (Without GRAD 48 become 49.)
    asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(p + head + (long long)v0 * 8),
                 "r"((uint32_t)(v1 - v0) * 8 * (uint32_t)sizeof(T))
                 : "memory");
  const int64_t y = a.targets[row];  // looked at once the row has been read
  float m = -INFINITY, s = 0.f;
  scan_row<T>(p + head, v0, v1, tid, NT, m, s);
  if (rank == 0) scan_ends<T>(p, a.vocab, head, vecs, tid, NT, m, s);
  Raw8<T> first[kUnroll];  // of the second pass, on their way while the row is joined
  if constexpr (GRAD) load_group<T>(first, p + head, v0 + tid, v1, NT);
  warp_join(m, s);
  if ((tid & 31) == 0) warps[tid >> 5] = make_float2(m, s);
  __syncthreads();
  if (tid < 32) {
    const float2 w = tid < NT / 32 ? warps[tid] : make_float2(-INFINITY, 0.f);
    m = w.x;
    s = w.y;
    warp_join(m, s);
  }
  if (split > 1) {
    cluster.barrier_wait();
    if (tid == 0) *cluster.map_shared_rank(&parts[rank], 0) = make_float2(m, s);
    cluster.sync();
    if (rank == 0 && tid == 0)
      for (int i = 1; i < (int)split; ++i) join(m, s, parts[i].x, parts[i].y);
  }
  if (rank == 0 && tid == 0) {
    const float c = finish_row<MODE>(a, row, target_logit(a, p, y), m, s);
    if constexpr (GRAD)
      for (int i = 0; i < (int)split; ++i) *cluster.map_shared_rank(&known, i) = make_float3(anchor(m), -c / s, c);
  }
  if constexpr (GRAD) {
    if (split > 1) cluster.sync();
    else __syncthreads();
    const float3 k = known;
    if (k.z == 0.f) {
      fill_zero<T>(g, a.vocab, rank, split, tid, NT);
      return;
    }
    const int hot = y >= 0 && y < a.vocab ? (int)y - head : -8;
    grad_row<T>(first, p + head, g + head, v0, v1, tid, NT, k.x, k.y, hot, k.z);
    if (rank == 0) grad_ends<T>(p, g, a.vocab, head, vecs, tid, NT, k.x, k.y, (int)y, k.z);
  }
}

struct GradArgs {
  const void* logits;
  long long stride_b, stride_s;
  int seq, rows, vocab, chunks;
  int rows_per_coef;
  const int64_t* targets;
  const bool* mask;
  const float* coef;
  const float* scale;  // null: 1
  const float2* stats;
  void* grad;  // contiguous
  bool ready;  // grad holds the gradient for a scale of 1 already
};

constexpr int kGradThreads = 256;

// dx_j = c ([j == y] - exp(x_j - m) / s). A group of NT threads (a CTA, or a warp for short rows) takes one of a row's
// `chunks` at a time. Rows with c = 0 are not read.
template <typename T, int NT>
__global__ void __launch_bounds__(kGradThreads) logprob_grad_kernel(const GradArgs a) {
  const float scale = a.scale ? *a.scale : 1.f;
  if (a.ready && scale == 1.f) return;
  constexpr unsigned kPer = kGradThreads / NT;
  const int tid = threadIdx.x % NT;
  for (unsigned unit = blockIdx.x * kPer + threadIdx.x / NT; unit < (unsigned)a.rows * a.chunks; unit += gridDim.x * kPer) {
    const int row = unit / (unsigned)a.chunks, chunk = unit - row * a.chunks;
    T* g = static_cast<T*>(a.grad) + (long long)row * a.vocab;
    float c = a.mask && !a.mask[row] ? 0.f : a.coef[(unsigned)row / (unsigned)a.rows_per_coef];
    if (c != 0.f) c *= scale;
    if (c == 0.f) {
      fill_zero<T>(g, a.vocab, chunk, a.chunks, tid, NT);
      continue;
    }
    const T* p = row_of<T>(a.logits, a.stride_b, a.stride_s, a.seq, row);
    const int head = head_of(p, a.vocab), vecs = (a.vocab - head) / 8;
    const int each = ((unsigned)vecs + a.chunks - 1) / (unsigned)a.chunks, v0 = min(chunk * each, vecs), v1 = min(v0 + each, vecs);
    Raw8<T> raw[kUnroll];
    load_group<T>(raw, p + head, v0 + tid, v1, NT);
    const float2 st = a.stats[row];
    const int64_t y = a.targets[row];
    const int hot = y >= 0 && y < a.vocab ? (int)y - head : -8;
    grad_row<T>(raw, p + head, g + head, v0, v1, tid, NT, st.x, -c / st.y, hot, c);
    if (chunk == 0) grad_ends<T>(p, g, a.vocab, head, vecs, tid, NT, st.x, -c / st.y, (int)y, c);
  }
}

constexpr int kReduceThreads = 1024;

// Sum over the CTA, the same order in every run; every thread gets it.
__device__ __forceinline__ double block_sum(double v, double* smem) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) smem[threadIdx.x >> 5] = v;
  __syncthreads();
  v = smem[threadIdx.x & 31];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
  return v;
}

// Rows that the mask keeps.
__global__ void __launch_bounds__(kReduceThreads) count_kernel(const bool* mask, int rows, int* count) {
  __shared__ double smem[32];
  double n = 0;
#pragma unroll 8
  for (int i = threadIdx.x; i < rows; i += kReduceThreads) n += mask[i] ? 1 : 0;
  n = block_sum(n, smem);
  if (threadIdx.x == 0) *count = (int)n;
}

// Means over the rows that count. One CTA: the rows' values are a vocabulary's size less than what the row kernel read.
__global__ void __launch_bounds__(kReduceThreads) policy_reduce_kernel(const RowArgs a, float* loss, float* kl, float* clipped) {
  __shared__ double smem[32];
  double l = 0, d = 0, c = 0;
#pragma unroll 4
  for (int i = threadIdx.x; i < a.rows; i += kReduceThreads) {
    const RowLoss r = a.row_loss[i];
    l += r.loss;
    d += r.kl;
    c += r.clipped;
  }
  l = block_sum(l, smem);
  d = block_sum(d, smem);
  c = block_sum(c, smem);
  if (threadIdx.x == 0) {
    const int n = a.count ? *a.count : a.rows;
    const double inv = n > 0 ? 1.0 / n : 0.0;
    *loss = (float)(l * inv);
    *kl = (float)(d * inv);
    *clipped = (float)(c * inv);
  }
}

// A warp sums each sequence, then a thread takes each pair. coef[i] is the derivative by each of sequence i's logp.
__global__ void __launch_bounds__(kReduceThreads) preference_reduce_kernel(const double* diff, int pairs, int seq, double beta,
                                                                          double smoothing, double* sums, float* loss,
                                                                          float* rewards, float* coef) {
  __shared__ double smem[32];
  const int lane = threadIdx.x & 31;
  for (int i = threadIdx.x >> 5; i < 2 * pairs; i += kReduceThreads / 32) {
    double v = 0;
#pragma unroll 8
    for (int t = lane; t < seq; t += 32) v += diff[(long long)i * seq + t];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
    if (lane == 0) {
      sums[i] = v;
      rewards[i] = (float)(beta * v);
    }
  }
  __syncthreads();
  double l = 0;
  for (int i = threadIdx.x; i < pairs; i += kReduceThreads) {
    const double h = beta * (sums[i] - sums[pairs + i]);
    const double tail = log1p(exp(-fabs(h)));  // log sigmoid(h) = min(h, 0) - tail
    const double up = fmin(h, 0.0) - tail, down = fmin(-h, 0.0) - tail;
    l -= (1.0 - smoothing) * up + smoothing * down;
    const double sig = h >= 0 ? 1.0 / (1.0 + exp(-h)) : exp(h) / (1.0 + exp(h));
    const double dh = smoothing * sig - (1.0 - smoothing) * (1.0 - sig);
    coef[i] = (float)(beta * dh / pairs);
    coef[pairs + i] = (float)(-beta * dh / pairs);
  }
  l = block_sum(l, smem);
  if (threadIdx.x == 0) *loss = (float)(l / pairs);
}

// ------------------------------------------------------------------ host

struct Rows {
  at::Tensor logits;  // [.., V], last stride 1; two or three dims
  long long stride_b, stride_s;
  int seq, rows, vocab;
};

Rows rows_of(const at::Tensor& logits, const at::Tensor& targets, const OptTensor& mask) {
  TORCH_CHECK_VALUE(logits.is_cuda(), "logits: CUDA tensor expected");
  const auto t = logits.scalar_type();
  TORCH_CHECK_VALUE(t == at::kFloat || t == at::kBFloat16 || t == at::kHalf, "logits: float32, bfloat16 or float16 expected, got ", t);
  TORCH_CHECK_VALUE(logits.dim() >= 2 && logits.size(-1) > 0, "logits: [..., vocab] with a vocabulary expected");
  TORCH_CHECK_VALUE(targets.scalar_type() == at::kLong && targets.device() == logits.device() &&
                        targets.sizes() == logits.sizes().slice(0, logits.dim() - 1),
                    "targets: int64 tensor of the logits' leading shape on their device expected");
  if (mask.has_value())
    TORCH_CHECK_VALUE(mask->scalar_type() == at::kBool && mask->device() == logits.device() && mask->sizes() == targets.sizes(),
                      "mask: bool tensor of the targets' shape on their device expected");
  const long long n = targets.numel(), v = logits.size(-1);
  TORCH_CHECK_VALUE(n < (1ll << 31) / 32 && v < (1ll << 30), "at most 2^26 rows of 2^30 logits expected, got ", n, " of ", v);
  Rows r;
  r.logits = logits;
  if (logits.dim() > 3) r.logits = logits.reshape({-1, v});
  if (r.logits.stride(-1) != 1 && v > 1) r.logits = r.logits.contiguous();
  const bool three = r.logits.dim() == 3;
  r.stride_b = three ? r.logits.stride(0) : 0;
  r.stride_s = r.logits.stride(-2);
  r.seq = (int)std::max<int64_t>(1, r.logits.size(-2));
  r.rows = (int)n;
  r.vocab = (int)v;
  return r;
}

void check_values(const at::Tensor& v, const at::Tensor& targets, const char* name) {
  TORCH_CHECK_VALUE(v.scalar_type() == at::kFloat && v.device() == targets.device() && v.sizes() == targets.sizes(), name,
                    ": float32 tensor of the targets' shape on their device expected");
}

// Whether rows go to a warp each: where they are short and many. Warp and CTA, log-probabilities and gradients of bf16 rows:
// 4096 of 1024 6 + 6 and 14 + 14 us, 16384 of 4096 29 + 47 and 63 + 66 us, 4096 of 8192 17 + 23 and 21 + 27 us, 1184 of 8192
// 8 + 10 and 8 + 8 us; 600 of 4096 6 + 6 us either way, 74 of 4096 6 + 6 and 4 + 4 us.
bool in_warps(const Rows& r) {
  return r.vocab <= 8192 && r.rows >= 8 * at::cuda::getCurrentDeviceProperties()->multiProcessorCount;
}

template <typename T, Mode MODE, bool GRAD>
void launch_row_kernel(const RowArgs& a, int split, cudaStream_t stream) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)a.rows * split);
  cfg.blockDim = dim3(kRowThreads);
  cfg.stream = stream;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim = {(unsigned)split, 1, 1};
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  C10_CUDA_CHECK(cudaLaunchKernelEx(&cfg, row_kernel<T, MODE, GRAD>, a));
}

template <Mode MODE>
void launch_rows(const Rows& r, RowArgs& a, cudaStream_t stream) {
  a.logits = r.logits.const_data_ptr();
  a.stride_b = r.stride_b;
  a.stride_s = r.stride_s;
  a.seq = r.seq;
  a.rows = r.rows;
  a.vocab = r.vocab;
  a.error = device_error_word(r.logits.device().index());
  if (r.rows == 0) return;
  with_element(r.logits.scalar_type(), [&](auto* tag) {
    using T = std::remove_pointer_t<decltype(tag)>;
    if (in_warps(r)) {
      const unsigned grid = (r.rows + kWarpRows - 1) / kWarpRows;
      bool done = false;
      if constexpr (MODE == kPolicy) {
        if ((done = a.grad != nullptr)) warp_row_kernel<T, MODE, true><<<grid, 32 * kWarpRows, 0, stream>>>(a);
      }
      if (!done) warp_row_kernel<T, MODE, false><<<grid, 32 * kWarpRows, 0, stream>>>(a);
      C10_CUDA_KERNEL_LAUNCH_CHECK();
      return;
    }
    // Few rows: split each until every SM has two CTAs or a part is down to two rounds of its CTA's loads. (Rows of 128256
    // bf16, split and whole: 4 of them 6 and 12 us, 64 8 and 12 us, 150 16 and 21 us.)
    const int sms = at::cuda::getCurrentDeviceProperties()->multiProcessorCount;
    int split = 1;
    while (split < 8 && (int64_t)r.rows * split < 2 * sms && r.vocab / split > 2 * kRowThreads * 8 * kUnroll) split *= 2;
    if constexpr (MODE == kPolicy) {
      if (a.grad) {
        while (split < 8 && (int64_t)r.vocab * sizeof(T) / split > kGradPart) split *= 2;
        return launch_row_kernel<T, MODE, true>(a, split, stream);
      }
    }
    launch_row_kernel<T, MODE, false>(a, split, stream);
  });
  count_launches(1);
}

}  // namespace

std::tuple<at::Tensor, at::Tensor> token_logprobs_fwd(const at::Tensor& logits, const at::Tensor& targets,
                                                      const OptTensor& mask) {
  const Rows r = rows_of(logits, targets, mask);
  const c10::cuda::CUDAGuard guard(logits.device());
  auto logp = new_empty(targets.sizes(), at::kFloat, logits), stats = new_empty({r.rows, 2}, at::kFloat, logits);
  const auto t = targets.contiguous();
  const auto m = mask.has_value() ? mask->contiguous() : at::Tensor();
  RowArgs a = {};
  a.targets = t.const_data_ptr<int64_t>();
  a.mask = m.defined() ? m.const_data_ptr<bool>() : nullptr;
  a.logp = logp.mutable_data_ptr<float>();
  a.stats = reinterpret_cast<float2*>(stats.mutable_data_ptr<float>());
  launch_rows<kLogprob>(r, a, at::cuda::getCurrentCUDAStream());
  return {logp, stats};
}

std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor> policy_loss_fwd(
    const at::Tensor& logits, const at::Tensor& targets, const at::Tensor& old_logp, const at::Tensor& advantages,
    const OptTensor& ref_logp, const OptTensor& mask, double clip_low, double clip_high, double kl_coef) {
  return policy_loss_fwd_grad(logits, targets, old_logp, advantages, ref_logp, mask, clip_low, clip_high, kl_coef, nullptr);
}

std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor> policy_loss_fwd_grad(
    const at::Tensor& logits, const at::Tensor& targets, const at::Tensor& old_logp, const at::Tensor& advantages,
    const OptTensor& ref_logp, const OptTensor& mask, double clip_low, double clip_high, double kl_coef, at::Tensor* grad) {
  const Rows r = rows_of(logits, targets, mask);
  TORCH_CHECK_VALUE(clip_low >= 0 && clip_low <= 1 && clip_high >= 0, "clip_low in [0, 1] and clip_high >= 0 expected, got ",
                    clip_low, " and ", clip_high);
  TORCH_CHECK_VALUE(kl_coef == 0 || ref_logp.has_value(), "kl_coef needs ref_logp");
  check_values(old_logp, targets, "old_logp");
  check_values(advantages, targets, "advantages");
  if (ref_logp.has_value()) check_values(*ref_logp, targets, "ref_logp");
  const c10::cuda::CUDAGuard guard(logits.device());
  const auto t = targets.contiguous(), old = old_logp.contiguous(), adv = advantages.contiguous();
  const auto ref = ref_logp.has_value() ? ref_logp->contiguous() : at::Tensor();
  const auto m = mask.has_value() ? mask->contiguous() : at::Tensor();
  auto loss = new_empty({}, at::kFloat, logits), kl = new_empty({}, at::kFloat, logits), clipped = new_empty({}, at::kFloat, logits);
  auto logp = new_empty(targets.sizes(), at::kFloat, logits), coef = new_empty(targets.sizes(), at::kFloat, logits);
  auto stats = new_empty({r.rows, 2}, at::kFloat, logits);
  // each row's part, and the number of rows that count
  auto work = new_empty({2 * (int64_t)r.rows + 1}, at::kDouble, logits);
  RowArgs a = {};
  a.targets = t.const_data_ptr<int64_t>();
  a.mask = m.defined() ? m.const_data_ptr<bool>() : nullptr;
  a.logp = logp.mutable_data_ptr<float>();
  a.stats = reinterpret_cast<float2*>(stats.mutable_data_ptr<float>());
  a.old_logp = old.const_data_ptr<float>();
  a.advantages = adv.const_data_ptr<float>();
  a.ref_logp = ref.defined() ? ref.const_data_ptr<float>() : nullptr;
  a.clip_low = clip_low;
  a.clip_high = clip_high;
  a.kl_coef = kl_coef;
  a.row_loss = reinterpret_cast<RowLoss*>(work.mutable_data_ptr<double>());
  int* count = reinterpret_cast<int*>(a.row_loss + r.rows);
  a.coef = coef.mutable_data_ptr<float>();
  const auto stream = at::cuda::getCurrentCUDAStream();
  if (a.mask) {
    a.count = count;
    count_kernel<<<1, kReduceThreads, 0, stream>>>(a.mask, r.rows, count);
    C10_CUDA_KERNEL_LAUNCH_CHECK();
    count_launches(1);
  }
  if (grad && r.rows > 0) {
    *grad = new_empty(logits.sizes(), logits.scalar_type(), logits);
    a.grad = grad->mutable_data_ptr();
  }
  launch_rows<kPolicy>(r, a, stream);
  policy_reduce_kernel<<<1, kReduceThreads, 0, stream>>>(a, loss.mutable_data_ptr<float>(), kl.mutable_data_ptr<float>(),
                                                        clipped.mutable_data_ptr<float>());
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  count_launches(1);
  return {loss, logp, kl, clipped, stats, coef};
}

std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor> preference_loss_fwd(
    const at::Tensor& logits, const at::Tensor& targets, const at::Tensor& ref_logp, const OptTensor& mask, double beta,
    double label_smoothing) {
  const Rows r = rows_of(logits, targets, mask);
  TORCH_CHECK_VALUE(targets.dim() == 2 && targets.size(0) > 0 && targets.size(0) % 2 == 0,
                    "targets: [2 * pairs, seq] expected, the chosen sequences in front of the rejected ones");
  TORCH_CHECK_VALUE(beta > 0 && label_smoothing >= 0 && label_smoothing < 0.5,
                    "beta > 0 and label_smoothing in [0, 0.5) expected, got ", beta, " and ", label_smoothing);
  check_values(ref_logp, targets, "ref_logp");
  const c10::cuda::CUDAGuard guard(logits.device());
  const auto t = targets.contiguous(), ref = ref_logp.contiguous();
  const auto m = mask.has_value() ? mask->contiguous() : at::Tensor();
  const int seqs = (int)targets.size(0), seq = (int)targets.size(1);
  auto loss = new_empty({}, at::kFloat, logits), rewards = new_empty({seqs}, at::kFloat, logits), coef = new_empty({seqs}, at::kFloat, logits);
  auto logp = new_empty(targets.sizes(), at::kFloat, logits), stats = new_empty({r.rows, 2}, at::kFloat, logits);
  auto wide = new_empty({r.rows + seqs}, at::kDouble, logits);
  RowArgs a = {};
  a.targets = t.const_data_ptr<int64_t>();
  a.mask = m.defined() ? m.const_data_ptr<bool>() : nullptr;
  a.logp = logp.mutable_data_ptr<float>();
  a.stats = reinterpret_cast<float2*>(stats.mutable_data_ptr<float>());
  a.ref_logp = ref.const_data_ptr<float>();
  a.row_diff = wide.mutable_data_ptr<double>();
  const auto stream = at::cuda::getCurrentCUDAStream();
  launch_rows<kPreference>(r, a, stream);
  preference_reduce_kernel<<<1, kReduceThreads, 0, stream>>>(a.row_diff, seqs / 2, seq, beta, label_smoothing,
                                                            a.row_diff + r.rows, loss.mutable_data_ptr<float>(),
                                                            rewards.mutable_data_ptr<float>(), coef.mutable_data_ptr<float>());
  C10_CUDA_KERNEL_LAUNCH_CHECK();
  count_launches(1);
  return {loss, logp, rewards, stats, coef};
}

at::Tensor token_logprobs_bwd(const at::Tensor& coef, const OptTensor& scale, const at::Tensor& logits,
                              const at::Tensor& targets, const at::Tensor& stats, const OptTensor& mask) {
  return token_logprobs_bwd_ready(coef, scale, logits, targets, stats, mask, at::Tensor());
}

at::Tensor token_logprobs_bwd_ready(const at::Tensor& coef, const OptTensor& scale, const at::Tensor& logits,
                                    const at::Tensor& targets, const at::Tensor& stats, const OptTensor& mask,
                                    const at::Tensor& ready) {
  const Rows r = rows_of(logits, targets, mask);
  TORCH_CHECK_VALUE(coef.scalar_type() == at::kFloat && coef.device() == logits.device() &&
                        (coef.sizes() == targets.sizes() || (targets.dim() == 2 && coef.dim() == 1 && coef.size(0) == targets.size(0))),
                    "coef: float32 per target or per sequence expected");
  TORCH_CHECK_VALUE(stats.scalar_type() == at::kFloat && stats.device() == logits.device() && stats.is_contiguous() &&
                        stats.dim() == 2 && stats.size(0) == r.rows && stats.size(1) == 2,
                    "stats: contiguous float32 [rows, 2] expected");
  if (scale.has_value())
    TORCH_CHECK_VALUE(scale->scalar_type() == at::kFloat && scale->device() == logits.device() && scale->numel() == 1,
                      "scale: one float32 value expected");
  const c10::cuda::CUDAGuard guard(logits.device());
  // A captured pass may be replayed with another scale, and then finds what the last one left: it computes all of it.
  const bool use_ready = ready.defined() && scale.has_value() &&
                         c10::cuda::currentStreamCaptureStatusMayInitCtx() == c10::cuda::CaptureStatus::None;
  auto grad = use_ready ? ready : new_empty(logits.sizes(), logits.scalar_type(), logits);
  if (r.rows == 0) return grad;
  const auto t = targets.contiguous(), cf = coef.contiguous();
  const auto m = mask.has_value() ? mask->contiguous() : at::Tensor();
  GradArgs a = {};
  a.logits = r.logits.const_data_ptr();
  a.stride_b = r.stride_b;
  a.stride_s = r.stride_s;
  a.seq = r.seq;
  a.rows = r.rows;
  a.vocab = r.vocab;
  a.rows_per_coef = (int)(r.rows / coef.numel());
  a.targets = t.const_data_ptr<int64_t>();
  a.mask = m.defined() ? m.const_data_ptr<bool>() : nullptr;
  a.coef = cf.const_data_ptr<float>();
  a.scale = scale.has_value() ? scale->const_data_ptr<float>() : nullptr;
  a.stats = reinterpret_cast<const float2*>(stats.const_data_ptr<float>());
  a.grad = grad.mutable_data_ptr();
  const bool warps = in_warps(r);  // else CTAs, in chunks of two rounds of their loads
  const int per = kGradThreads * 8 * kUnroll * 2;
  a.chunks = warps ? 1 : (r.vocab + per - 1) / per;
  TORCH_CHECK_VALUE((long long)a.chunks * r.rows < (1ll << 31), "logits: too many values for one call");
  a.ready = use_ready;
  // where there is likely nothing to do, no more CTAs than are resident
  const int sms = at::cuda::getCurrentDeviceProperties()->multiProcessorCount;
  const unsigned groups = warps ? kGradThreads / 32 : 1, all = ((unsigned)(a.chunks * r.rows) + groups - 1) / groups;
  const unsigned grid = use_ready ? std::min(all, (unsigned)sms * 4) : all;
  with_element(logits.scalar_type(), [&](auto* tag) {
    using T = std::remove_pointer_t<decltype(tag)>;
    const auto stream = at::cuda::getCurrentCUDAStream();
    if (warps) logprob_grad_kernel<T, 32><<<grid, kGradThreads, 0, stream>>>(a);
    else logprob_grad_kernel<T, kGradThreads><<<grid, kGradThreads, 0, stream>>>(a);
    C10_CUDA_KERNEL_LAUNCH_CHECK();
  });
  count_launches(1);
  return grad;
}

}  // namespace dmb
