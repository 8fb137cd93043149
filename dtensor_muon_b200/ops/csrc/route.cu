// Router of a sparse layer: top-k experts of each token with their gates, the number of tokens of
// each expert, the balance loss and the z loss.
//
//   p = softmax(l) over all E experts;  experts = the k greatest l, equal ones by index;  g = softmax(l[experts])
//   c_e = choices of e by the N tokens that count
//   balance = E / (N^2 k) sum_e c_e sum_t p_te   (1 where every expert gets the same),  z = 1/N sum_t lse_t^2
//   dl = g (dg - g.dg) at the chosen + p (dbalance E / (N^2 k) (c_e - c.p) + dz 2/N lse)
//
// Up to 64 experts a row lies on one to eight lanes, eight logits on each; above, on a warp, four to 16 logits on each
// lane. The choice takes k rounds of a maximum over the row by (value, index); on a warp the lanes sort their logits first,
// and a round is one redux over order-preserving integer keys and a ballot. Every group of lanes
// walks over rows and keeps its sums of p and of lse^2 in 32 bits and its counts in registers; a CTA joins them in a fixed
// order, in 32 bits too, and writes one part, and a second kernel sums the parts in 64 bits. The longest chain of 32-bit
// additions is a group's own rows, one in 592 CTAs times the groups of a CTA (4 of 65536 rows of 64 experts, 14 of 65536 rows
// of 128), then at most five over its warp and eight over the warps. Nothing that is rounded is summed by atomics, and a run
// gives the same bits each time. What bounds it: launches for small batches (16384 rows of 8, top 2: 16 us for three kernels),
// the instructions of the k rounds and latency for many experts (65536 bf16 rows, top 8, forward + backward: 8 experts 17 + 7
// us, 64 39 + 21 us, 128 47 + 25 us, 256 73 + 43 us, where the bytes alone take 1 to 12 us).
#include <ATen/ATen.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAException.h>
#include <c10/cuda/CUDAGuard.h>

#include "train_ops.h"
#include "vec.cuh"

namespace dmb {
namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxExperts = 512;
constexpr int kMaxTopK = 32;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

struct Args {
  const void* logits;
  long long stride;  // elements between rows
  bool vec, vec_out;  // logits, dlogits: rows of whole words, each lane's on its own boundary
  int tokens, experts, top_k;
  const bool* mask;  // null: every token counts
  // forward
  void* gates;
  int64_t* chosen;
  int64_t* counts;
  float* sum_p;  // [E + 1, CTAs]: sums of p, last the sum of lse^2
  int* sum_c;    // [E + 1, CTAs]: choices, last the tokens that count
  double* total_p;  // [E + 1]
  int* total_c;     // [E + 1]
  unsigned* ticket;
  // backward
  const void* dgates;                // null: none
  const float *dbalance, *dz;        // null: none
  void* dlogits;
};

constexpr int kPerLane = 8;  // logits next to each other on each lane, where a row lies on one to eight lanes

template <typename T>
__device__ __forceinline__ void load_row(const Args& a, int row, bool in, int lane, float (&x)[kPerLane]) {
  const T* p = static_cast<const T*>(a.logits) + (long long)row * a.stride;
  const int e = lane * kPerLane;
#pragma unroll
  for (int k = 0; k < kPerLane; ++k) x[k] = -INFINITY;
  if (in) {
    if (a.vec) {
      if (e < a.experts) load8t<T>(p + e, x);
    } else {
#pragma unroll
      for (int k = 0; k < kPerLane; ++k)
        if (e + k < a.experts) x[k] = to_float(p[e + k]);
    }
  }
}

template <int LPR>
__device__ __forceinline__ float group_max(float v) {
#pragma unroll
  for (int o = LPR / 2; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(~0u, v, o));
  return v;
}

template <int LPR>
__device__ __forceinline__ float group_sum(float v) {
#pragma unroll
  for (int o = LPR / 2; o > 0; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
  return v;
}

// Unsigned numbers in the order of the floats, NaN above all, both zeros alike, 0 below all.
__device__ __forceinline__ uint32_t order_key(float x) {
  if (x != x) return 0xFFFFFFFFu;
  const uint32_t u = __float_as_uint(x == 0.f ? 0.f : x);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

__device__ __forceinline__ float key_value(uint32_t k) {
  return __uint_as_float(k == 0xFFFFFFFFu ? 0x7FC00000u : k & 0x80000000u ? k & 0x7FFFFFFFu : ~k);
}

// Sums the warps' shares, [kWarps, width + 1] in shared memory, and writes the CTA's part. The first CTA also resets the
// ticket that route_join_kernel draws.
__device__ __forceinline__ void write_part(const Args& a, const float* join_p, const int* join_c, int width) {
  __syncthreads();
  for (int e = threadIdx.x; e <= a.experts; e += kThreads) {
    const int from = e < a.experts ? e : width;
    float p = 0.f;
    int c = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      p += join_p[w * (width + 1) + from];
      c += join_c[w * (width + 1) + from];
    }
    a.sum_p[(long long)e * gridDim.x + blockIdx.x] = p;
    a.sum_c[(long long)e * gridDim.x + blockIdx.x] = c;
  }
  if (blockIdx.x == 0 && threadIdx.x == 0) *a.ticket = 0;
}

template <typename T, int LPR>
__global__ void __launch_bounds__(kThreads) route_kernel(const Args a) {
  constexpr int VPL = kPerLane, kGroups = kThreads / LPR, kExperts = LPR * VPL;
  constexpr int kTop = kExperts < kMaxTopK ? kExperts : kMaxTopK;
  constexpr int kStash = 2 * kGroups * kTop, kJoin = 2 * kWarps * (kExperts + 1);
  __shared__ uint32_t smem[kStash > kJoin ? kStash : kJoin];
  const int lane = threadIdx.x % LPR, group = threadIdx.x / LPR;
  float* stash_e = reinterpret_cast<float*>(smem) + group * kTop;  // this row's exponentials and experts by rank
  int* stash_i = reinterpret_cast<int*>(smem) + kGroups * kTop + group * kTop;

  float sum_p[VPL] = {}, sum_z = 0.f;
  int sum_c[VPL] = {}, sum_n = 0;
  for (int base = blockIdx.x * kGroups; base < a.tokens; base += gridDim.x * kGroups) {
    const int row = base + group;
    const bool in = row < a.tokens;
    const bool valid = in && (!a.mask || a.mask[row]);
    float x[VPL];
    load_row<T>(a, row, in, lane, x);
    uint32_t key[VPL];
#pragma unroll
    for (int j = 0; j < VPL; ++j) key[j] = lane * VPL + j < a.experts ? order_key(x[j]) : 0u;
    uint32_t picked = 0;  // bit j: the lane's j-th expert is chosen
    float top = 0.f, total = 0.f;
    for (int i = 0; i < a.top_k; ++i) {
      uint32_t best = 0;
      int at = 0;
#pragma unroll
      for (int j = 0; j < VPL; ++j)
        if (key[j] > best) {  // within a lane, a later value has a higher index
          best = key[j];
          at = lane * VPL + j;
        }
#pragma unroll
      for (int o = LPR / 2; o > 0; o >>= 1) {
        const uint32_t other = __shfl_xor_sync(~0u, best, o);
        const int other_at = __shfl_xor_sync(~0u, at, o);
        if (other > best || (other == best && other_at < at)) {
          best = other;
          at = other_at;
        }
      }
#pragma unroll
      for (int j = 0; j < VPL; ++j)
        if (lane * VPL + j == at) {
          key[j] = 0;
          picked |= 1u << j;
        }
      const float v = key_value(best);
      if (i == 0) top = v;
      const float e = ex2((v - top) * kLog2e);
      total += e;
      if (lane == 0) {
        stash_e[i] = e;
        stash_i[i] = at;
      }
    }
    __syncwarp();
    if (in) {
      const float inv = 1.f / total;
      for (int i = lane; i < a.top_k; i += LPR) {
        static_cast<T*>(a.gates)[(long long)row * a.top_k + i] = from_float<T>(valid ? stash_e[i] * inv : 0.f);
        a.chosen[(long long)row * a.top_k + i] = stash_i[i];
      }
    }
    __syncwarp();
    // softmax over all experts; the row's maximum may be -inf
    float m = -INFINITY, s = 0.f;
#pragma unroll
    for (int j = 0; j < VPL; ++j) m = fmaxf(m, x[j]);
    m = group_max<LPR>(m);
    m = m == -INFINITY ? 0.f : m;
#pragma unroll
    for (int j = 0; j < VPL; ++j) {
      x[j] = ex2((x[j] - m) * kLog2e);
      s += x[j];
    }
    s = group_sum<LPR>(s);
    if (valid) {
      const float inv = 1.f / s, lse = m + __log2f(s) * kLn2;
      sum_n += 1;
      sum_z = fmaf(lse, lse, sum_z);
#pragma unroll
      for (int j = 0; j < VPL; ++j) {
        sum_p[j] = fmaf(x[j], inv, sum_p[j]);
        sum_c[j] += (picked >> j) & 1;
      }
    }
  }
  // join the groups of each warp, then the warps
#pragma unroll
  for (int o = LPR; o < 32; o <<= 1) {
#pragma unroll
    for (int j = 0; j < VPL; ++j) {
      sum_p[j] += __shfl_xor_sync(~0u, sum_p[j], o);
      sum_c[j] += __shfl_xor_sync(~0u, sum_c[j], o);
    }
    sum_z += __shfl_xor_sync(~0u, sum_z, o);
    sum_n += __shfl_xor_sync(~0u, sum_n, o);
  }
  __syncthreads();
  float* join_p = reinterpret_cast<float*>(smem);
  int* join_c = reinterpret_cast<int*>(smem) + kWarps * (kExperts + 1);
  const int warp = threadIdx.x >> 5;
  if ((threadIdx.x & 31) < LPR) {
#pragma unroll
    for (int j = 0; j < VPL; ++j) {
      join_p[warp * (kExperts + 1) + lane * VPL + j] = sum_p[j];
      join_c[warp * (kExperts + 1) + lane * VPL + j] = sum_c[j];
    }
    if (lane == 0) {
      join_p[warp * (kExperts + 1) + kExperts] = sum_z;
      join_c[warp * (kExperts + 1) + kExperts] = sum_n;
    }
  }
  write_part(a, join_p, join_c, kExperts);
}

// ------------------------------------------------------------------ a warp per row

// A lane's values as they lie in memory, in words of 16 bytes, or of 8 for four 16-bit values.
template <typename T, int VPL>
union LaneWords {
  using W = std::conditional_t<VPL * sizeof(T) == 8, uint2, uint4>;
  static constexpr int kWords = VPL * sizeof(T) / sizeof(W);
  W w[kWords];
  T t[VPL];
};

// VPL logits next to each other on each lane: lane order is index order.
template <typename T, int VPL>
__device__ __forceinline__ void load_lane(const Args& a, int row, int lane, float (&x)[VPL]) {
  const T* p = static_cast<const T*>(a.logits) + (long long)row * a.stride + lane * VPL;
  if (a.vec) {  // whole: the row ends with a lane, and every lane's share is on its own boundary
    LaneWords<T, VPL> u;
    if (lane * VPL < a.experts) {
#pragma unroll
      for (int i = 0; i < u.kWords; ++i) u.w[i] = __ldg(reinterpret_cast<const typename LaneWords<T, VPL>::W*>(p) + i);
    }
#pragma unroll
    for (int j = 0; j < VPL; ++j) x[j] = lane * VPL < a.experts ? to_float(u.t[j]) : -INFINITY;
  } else {
#pragma unroll
    for (int j = 0; j < VPL; ++j) x[j] = lane * VPL + j < a.experts ? to_float(p[j]) : -INFINITY;
  }
}

// Each lane first sorts its keys (by swaps of neighbours only, so that equal ones stay in order), and a round then takes the
// largest head of the lanes' lists: one redux, one ballot, and the winner's list moves up. The next row's logits are on
// their way meanwhile.
template <typename T, int VPL>
__global__ void __launch_bounds__(kThreads, VPL == 16 ? 2 : 4) route_warp_kernel(const Args a) {
  constexpr int kExperts = 32 * VPL;
  __shared__ float join_p[kWarps * (kExperts + 1)];
  __shared__ int join_c[kWarps * (kExperts + 1)];
  __shared__ uint2 stash[kWarps][kMaxTopK];  // a row's keys and experts by rank
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int* count = join_c + warp * (kExperts + 1);  // the warp's own
  for (int e = lane; e < kExperts; e += 32) count[e] = 0;
  __syncwarp();
  float sum_p[VPL] = {}, sum_z = 0.f;
  int sum_n = 0;
  const int step = gridDim.x * kWarps;
  int row = blockIdx.x * kWarps + warp;
  float next[VPL];
  bool next_valid = false;
  auto fetch = [&](int r) {
    if (r < a.tokens) {
      next_valid = !a.mask || a.mask[r];
      load_lane<T, VPL>(a, r, lane, next);
    }
  };
  fetch(row);
  for (; row < a.tokens; row += step) {
    const bool valid = next_valid;
    float x[VPL];
    uint32_t key[VPL], order[VPL];
#pragma unroll
    for (int j = 0; j < VPL; ++j) {
      x[j] = next[j];
      key[j] = lane * VPL + j < a.experts ? order_key(x[j]) : 0u;
      order[j] = j;
    }
    fetch(row + step);
#pragma unroll
    for (int i = 0; i < VPL - 1; ++i) {
#pragma unroll
      for (int j = VPL - 2; j >= i; --j) {
        const bool swap = key[j + 1] > key[j];
        const uint32_t hi = max(key[j], key[j + 1]), lo = min(key[j], key[j + 1]), t = order[j];
        order[j] = swap ? order[j + 1] : t;
        order[j + 1] = swap ? t : order[j + 1];
        key[j] = hi;
        key[j + 1] = lo;
      }
    }
    uint64_t list = 0;  // the sorted keys' places, four bits each
#pragma unroll
    for (int j = 0; j < VPL; ++j) list |= (uint64_t)order[j] << (4 * j);
    for (int i = 0; i < a.top_k; ++i) {
      const uint32_t top = __reduce_max_sync(~0u, key[0]);
      if (__ffs(__ballot_sync(~0u, key[0] == top)) - 1 == lane) {  // the first lane of those that have it
        stash[warp][i] = make_uint2(top, lane * VPL + ((uint32_t)list & 15u));
        list >>= 4;
#pragma unroll
        for (int j = 0; j < VPL - 1; ++j) key[j] = key[j + 1];
        key[VPL - 1] = 0;
      }
    }
    __syncwarp();
    // softmax over all experts; the row's maximum may be -inf
    const float top = key_value(stash[warp][0].x), m = top == -INFINITY ? 0.f : top;
    float s = 0.f, e = 0.f;
#pragma unroll
    for (int j = 0; j < VPL; ++j) {
      x[j] = ex2((x[j] - m) * kLog2e);
      s += x[j];
    }
    const bool mine = lane < a.top_k;
    const uint2 pick = stash[warp][lane];
    if (mine) e = ex2((key_value(pick.x) - top) * kLog2e);
    float total = e;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      s += __shfl_xor_sync(~0u, s, o);
      total += __shfl_xor_sync(~0u, total, o);
    }
    if (mine) {
      const long long out = (long long)row * a.top_k + lane;
      static_cast<T*>(a.gates)[out] = from_float<T>(valid ? e / total : 0.f);
      a.chosen[out] = pick.y;
      if (valid) count[pick.y] += 1;  // a row's experts differ
    }
    if (valid) {
      const float inv = 1.f / s, lse = m + __log2f(s) * kLn2;
      sum_n += 1;
      sum_z = fmaf(lse, lse, sum_z);
#pragma unroll
      for (int j = 0; j < VPL; ++j) sum_p[j] = fmaf(x[j], inv, sum_p[j]);
    }
    __syncwarp();
  }
#pragma unroll
  for (int j = 0; j < VPL; ++j) join_p[warp * (kExperts + 1) + lane * VPL + j] = sum_p[j];
  if (lane == 0) {
    join_p[warp * (kExperts + 1) + kExperts] = sum_z;
    count[kExperts] = sum_n;
  }
  write_part(a, join_p, join_c, kExperts);
}

constexpr int kJoinThreads = 512;

// A warp sums each expert's parts; the CTA that is done last takes the products, in the experts' order.
__global__ void __launch_bounds__(kJoinThreads) route_join_kernel(const Args a, int parts, float* balance, float* z) {
  __shared__ bool last;
  const int lane = threadIdx.x & 31;
  const int e = (blockIdx.x * kJoinThreads + threadIdx.x) >> 5;
  if (e <= a.experts) {
    double p = 0;
    int c = 0;
#pragma unroll 4
    for (int i = lane; i < parts; i += 32) {
      p += a.sum_p[(long long)e * parts + i];
      c += a.sum_c[(long long)e * parts + i];
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      p += __shfl_xor_sync(~0u, p, o);
      c += __shfl_xor_sync(~0u, c, o);
    }
    if (lane == 0) {
      a.total_p[e] = p;
      a.total_c[e] = c;
      if (e < a.experts) a.counts[e] = c;
      __threadfence();
    }
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    last = gridDim.x == 1 || atomicAdd(a.ticket, 1u) == gridDim.x - 1;
    __threadfence();
  }
  __syncthreads();
  if (!last || threadIdx.x >= 32) return;
  double dot = 0;
  for (int i = lane; i < a.experts; i += 32) dot += __ldcg(a.total_p + i) * __ldcg(a.total_c + i);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) dot += __shfl_xor_sync(~0u, dot, o);
  if (lane == 0) {
    const double n = __ldcg(a.total_c + a.experts);
    *balance = n > 0 ? (float)(dot * a.experts / (n * n * a.top_k)) : 0.f;
    *z = n > 0 ? (float)(__ldcg(a.total_p + a.experts) / n) : 0.f;
  }
}

// c_e / (N k) of each expert to shared memory, [0, width); returns the number of choices.
__device__ __forceinline__ int load_share(const Args& a, float* share, int* choices, int width) {
  if (threadIdx.x < 32) {
    int n = 0;
    for (int e = threadIdx.x; e < a.experts; e += 32) n += (int)a.counts[e];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) n += __shfl_xor_sync(~0u, n, o);
    if (threadIdx.x == 0) *choices = n;
  }
  __syncthreads();
  const int n = *choices;
  for (int e = threadIdx.x; e < width; e += kThreads)
    share[e] = e < a.experts && n > 0 ? (float)((double)a.counts[e] / n) : 0.f;
  __syncthreads();
  return n;
}

template <typename T, int VPL>
__global__ void __launch_bounds__(kThreads, VPL == 16 ? 2 : 4) route_warp_grad_kernel(const Args a) {
  constexpr int kExperts = 32 * VPL;
  __shared__ float share[kExperts];
  __shared__ int choices;
  // {dgate, 1} of the chosen experts of a warp's row, 0 elsewhere: each warp scatters to and gathers from its own
  __shared__ __align__(16) float2 picks[kWarps][kExperts];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (int e = threadIdx.x; e < kWarps * kExperts; e += kThreads) (&picks[0][0])[e] = make_float2(0.f, 0.f);
  const int count = load_share(a, share, &choices, kExperts);
  const float n = (float)(count / a.top_k);
  const float by_balance = a.dbalance && count > 0 ? *a.dbalance * a.experts / n : 0.f;
  const float by_z = a.dz && count > 0 ? *a.dz * 2.f / n : 0.f;
  float part[VPL];
#pragma unroll
  for (int j = 0; j < VPL; ++j) part[j] = share[lane * VPL + j];
  const int step = gridDim.x * kWarps;
  int row = blockIdx.x * kWarps + warp;
  float next[VPL], next_dg = 0.f;
  int next_at = -1;
  bool next_valid = false;
  auto fetch = [&](int r) {
    if (r >= a.tokens) return;
    next_valid = !a.mask || a.mask[r];
    load_lane<T, VPL>(a, r, lane, next);
    if (a.dgates && lane < a.top_k) {
      const int64_t e = a.chosen[(long long)r * a.top_k + lane];
      next_dg = to_float(static_cast<const T*>(a.dgates)[(long long)r * a.top_k + lane]);
      next_at = e >= 0 && e < a.experts ? (int)e : -1;
    }
  };
  fetch(row);
  for (; row < a.tokens; row += step) {
    T* out = static_cast<T*>(a.dlogits) + (long long)row * a.experts + lane * VPL;
    float x[VPL];
#pragma unroll
    for (int j = 0; j < VPL; ++j) x[j] = next[j];
    const int at = next_at;
    const float mine = next_dg;
    const bool valid = next_valid;
    fetch(row + step);
    if (valid) {
      if (at >= 0) picks[warp][at] = make_float2(mine, 1.f);
      float m = -INFINITY;
#pragma unroll
      for (int j = 0; j < VPL; ++j) m = fmaxf(m, x[j]);
      m = group_max<32>(m);
      m = m == -INFINITY ? 0.f : m;
      __syncwarp();
      // the chosen ones have the same maximum, so that one exponential serves both softmaxes
      float s = 0.f, s_top = 0.f, dot = 0.f, mix = 0.f, dg[VPL], in[VPL];
#pragma unroll
      for (int j = 0; j < VPL; ++j) {
        const float2 pick = picks[warp][lane * VPL + j];
        dg[j] = pick.x;
        in[j] = pick.y;
        x[j] = ex2((x[j] - m) * kLog2e);
        s += x[j];
        mix = fmaf(part[j], x[j], mix);
        if (in[j] != 0.f) {
          s_top += x[j];
          dot = fmaf(x[j], dg[j], dot);
        }
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        s += __shfl_xor_sync(~0u, s, o);
        mix += __shfl_xor_sync(~0u, mix, o);
        s_top += __shfl_xor_sync(~0u, s_top, o);
        dot += __shfl_xor_sync(~0u, dot, o);
      }
      if (at >= 0) picks[warp][at] = make_float2(0.f, 0.f);  // every lane has read: the shuffles lie between
      const float inv = 1.f / s, inv_top = 1.f / s_top;
      const float all = by_z * (m + __log2f(s) * kLn2) - by_balance * (mix * inv);
      dot *= inv_top;
#pragma unroll
      for (int j = 0; j < VPL; ++j) {
        float g = x[j] * inv * fmaf(by_balance, part[j], all);
        if (in[j] != 0.f) g = fmaf(x[j] * inv_top, dg[j] - dot, g);
        x[j] = g;
      }
      __syncwarp();
    } else {
#pragma unroll
      for (int j = 0; j < VPL; ++j) x[j] = 0.f;
    }
    if (a.vec_out) {
      LaneWords<T, VPL> u;
#pragma unroll
      for (int j = 0; j < VPL; ++j) u.t[j] = from_float<T>(x[j]);
      if (lane * VPL < a.experts) {
#pragma unroll
        for (int i = 0; i < u.kWords; ++i) reinterpret_cast<typename LaneWords<T, VPL>::W*>(out)[i] = u.w[i];
      }
    } else {
#pragma unroll
      for (int j = 0; j < VPL; ++j)
        if (lane * VPL + j < a.experts) out[j] = from_float<T>(x[j]);
    }
  }
}

template <typename T, int LPR>
__global__ void __launch_bounds__(kThreads) route_grad_kernel(const Args a) {
  constexpr int VPL = kPerLane, kGroups = kThreads / LPR, kExperts = LPR * VPL;
  __shared__ float share[kExperts];  // c_e / (N k)
  __shared__ int choices;
  const int lane = threadIdx.x % LPR, group = threadIdx.x / LPR;
  const int count = load_share(a, share, &choices, kExperts);
  const float n = (float)(count / a.top_k);
  const float by_balance = a.dbalance && count > 0 ? *a.dbalance * a.experts / n : 0.f;
  const float by_z = a.dz && count > 0 ? *a.dz * 2.f / n : 0.f;
  for (int base = blockIdx.x * kGroups; base < a.tokens; base += gridDim.x * kGroups) {
    const int row = base + group;
    const bool in = row < a.tokens;
    const bool valid = in && (!a.mask || a.mask[row]);
    float x[VPL];
    load_row<T>(a, row, valid, lane, x);
    uint32_t picked = 0;
    float dg[VPL] = {};
    if (valid && a.dgates) {
      for (int i = 0; i < a.top_k; ++i) {
        const long long at = (long long)row * a.top_k + i;
        const int64_t expert = a.chosen[at];
        const float d = to_float(static_cast<const T*>(a.dgates)[at]);
#pragma unroll
        for (int j = 0; j < VPL; ++j)
          if (lane * VPL + j == expert) {
            dg[j] = d;
            picked |= 1u << j;
          }
      }
    }
    float m = -INFINITY;
#pragma unroll
    for (int j = 0; j < VPL; ++j) m = fmaxf(m, x[j]);
    m = group_max<LPR>(m);
    m = m == -INFINITY ? 0.f : m;
    // the chosen ones have the same maximum, so that one exponential serves both softmaxes
    float s = 0.f, s_top = 0.f, dot = 0.f, mix = 0.f;
#pragma unroll
    for (int j = 0; j < VPL; ++j) {
      x[j] = ex2((x[j] - m) * kLog2e);
      s += x[j];
      mix = fmaf(share[lane * VPL + j], x[j], mix);
      if ((picked >> j) & 1) {
        s_top += x[j];
        dot = fmaf(x[j], dg[j], dot);
      }
    }
    s = group_sum<LPR>(s);
    mix = group_sum<LPR>(mix);
    s_top = group_sum<LPR>(s_top);
    dot = group_sum<LPR>(dot);
    const float inv = 1.f / s, inv_top = 1.f / s_top;
    const float all = by_z * (m + __log2f(s) * kLn2) - by_balance * (mix * inv);
    dot *= inv_top;
    if (!in) continue;
    T* out = static_cast<T*>(a.dlogits) + (long long)row * a.experts;
    const int e = lane * VPL;
#pragma unroll
    for (int j = 0; j < VPL; ++j) {
      float g = x[j] * inv * fmaf(by_balance, share[e + j], all);
      if ((picked >> j) & 1) g = fmaf(x[j] * inv_top, dg[j] - dot, g);
      x[j] = valid ? g : 0.f;
    }
    if (a.vec_out) {
      if (e < a.experts) store8t<T>(out + e, x);
    } else {
#pragma unroll
      for (int j = 0; j < VPL; ++j)
        if (e + j < a.experts) out[e + j] = from_float<T>(x[j]);
    }
  }
}

// ------------------------------------------------------------------ host

// f(T, LPR, VPL): up to 64 experts as few lanes per row as hold it at eight logits each, so that a warp has four rows or
// more at once; above a warp per row, whose rounds are cheaper and whose other work is dearer. 65536 bf16 rows forward +
// backward, on lanes and on a warp: 64 experts 24 + 14 and 37 + 25 us at top 2, 39 + 21 and 47 + 25 us at top 8; 128
// experts 37 + 23 and 37 + 25 us at top 2, 66 + 35 and 47 + 25 us at top 8.
template <typename F>
void with_layout(const at::Tensor& logits, F&& f) {
  with_element(logits.scalar_type(), [&](auto* t) {
    const int e = (int)logits.size(1);
    using std::integral_constant;
    if (e <= 8) f(t, integral_constant<int, 1>(), integral_constant<int, kPerLane>());
    else if (e <= 16) f(t, integral_constant<int, 2>(), integral_constant<int, kPerLane>());
    else if (e <= 32) f(t, integral_constant<int, 4>(), integral_constant<int, kPerLane>());
    else if (e <= 64) f(t, integral_constant<int, 8>(), integral_constant<int, kPerLane>());
    else if (e <= 128) f(t, integral_constant<int, 32>(), integral_constant<int, 4>());
    else if (e <= 256) f(t, integral_constant<int, 32>(), integral_constant<int, 8>());
    else f(t, integral_constant<int, 32>(), integral_constant<int, 16>());
  });
}

// Values that a lane has next to each other.
int per_lane(int experts) { return experts <= 64 ? kPerLane : experts <= 128 ? 4 : experts <= 256 ? 8 : 16; }

// Whether rows `stride` elements apart can be moved in a lane's whole words, of up to 16 bytes.
bool whole_words(const void* p, int64_t rows, int64_t stride, int experts, int64_t size) {
  const int64_t word = std::min<int64_t>(16, per_lane(experts) * size);
  return experts % per_lane(experts) == 0 && (rows <= 1 || stride * size % word == 0) && reinterpret_cast<uintptr_t>(p) % word == 0;
}

void check_route(const at::Tensor& logits, int64_t top_k, const OptTensor& mask) {
  TORCH_CHECK_VALUE(logits.is_cuda() && logits.dim() == 2, "logits: CUDA tensor [tokens, experts] expected");
  TORCH_CHECK_VALUE(logits.size(1) >= 1 && logits.size(1) <= kMaxExperts, "1 to ", kMaxExperts, " experts expected, got ", logits.size(1));
  const int64_t most = std::min<int64_t>(logits.size(1), kMaxTopK);
  TORCH_CHECK_VALUE(top_k >= 1 && top_k <= most, "top_k from 1 to ", most, " expected, got ", top_k);
  TORCH_CHECK_VALUE(logits.size(0) < (1ll << 30) / top_k, "logits: fewer than 2^30 choices expected");
  if (mask.has_value())
    TORCH_CHECK_VALUE(mask->scalar_type() == at::kBool && mask->device() == logits.device() && mask->dim() == 1 &&
                          mask->size(0) == logits.size(0),
                      "mask: bool [tokens] on the logits' device expected");
}

Args args_of(const at::Tensor& logits, const at::Tensor& mask, int64_t top_k) {
  Args a = {};
  a.logits = logits.const_data_ptr();
  a.stride = logits.stride(0);
  a.tokens = (int)logits.size(0);
  a.experts = (int)logits.size(1);
  a.top_k = (int)top_k;
  a.vec = whole_words(a.logits, a.tokens, a.stride, a.experts, logits.element_size());
  a.mask = mask.defined() ? mask.const_data_ptr<bool>() : nullptr;
  return a;
}

}  // namespace

std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor> route_fwd(const at::Tensor& logits,
                                                                                int64_t top_k, const OptTensor& mask) {
  check_route(logits, top_k, mask);
  const c10::cuda::CUDAGuard guard(logits.device());
  const auto x = logits.stride(1) == 1 || logits.size(1) == 1 ? logits : logits.contiguous();
  const auto m = mask.has_value() ? mask->contiguous() : at::Tensor();
  const int64_t t = x.size(0), e = x.size(1);
  auto gates = new_empty({t, top_k}, logits.scalar_type(), logits);
  auto chosen = new_empty({t, top_k}, at::kLong, logits), counts = new_empty({e}, at::kLong, logits);
  auto balance = new_empty({}, at::kFloat, logits), z = new_empty({}, at::kFloat, logits);
  if (t == 0) return {gates, chosen, counts.zero_(), balance.zero_(), z.zero_()};
  Args a = args_of(x, m, top_k);
  a.gates = gates.mutable_data_ptr();
  a.chosen = chosen.mutable_data_ptr<int64_t>();
  a.counts = counts.mutable_data_ptr<int64_t>();
  const auto stream = at::cuda::getCurrentCUDAStream();
  with_layout(x, [&](auto* tag, auto lanes, auto values) {
    using T = std::remove_pointer_t<decltype(tag)>;
    constexpr int L = decltype(lanes)::value, V = decltype(values)::value;
    const int groups = kThreads / L;  // rows of a CTA at once
    const int sms = at::cuda::getCurrentDeviceProperties()->multiProcessorCount;
    const int ctas = (int)std::min<int64_t>((t + groups - 1) / groups, (int64_t)sms * 4);
    // one workspace: the CTAs' parts, the totals and the ticket
    auto work = new_empty({(e + 1) * (2 * (int64_t)ctas + 3) + 2}, at::kFloat, logits);
    a.total_p = reinterpret_cast<double*>(work.template mutable_data_ptr<float>());
    a.total_c = reinterpret_cast<int*>(a.total_p + e + 1);
    a.ticket = reinterpret_cast<unsigned*>(a.total_c + e + 1);
    a.sum_p = reinterpret_cast<float*>(a.ticket + 2);
    a.sum_c = reinterpret_cast<int*>(a.sum_p + (e + 1) * ctas);
    if constexpr (L == 32) route_warp_kernel<T, V><<<ctas, kThreads, 0, stream>>>(a);
    else route_kernel<T, L><<<ctas, kThreads, 0, stream>>>(a);
    C10_CUDA_KERNEL_LAUNCH_CHECK();
    const int joins = (int)((e + 1 + kJoinThreads / 32 - 1) / (kJoinThreads / 32));
    route_join_kernel<<<joins, kJoinThreads, 0, stream>>>(a, ctas, balance.template mutable_data_ptr<float>(),
                                                      z.template mutable_data_ptr<float>());
    C10_CUDA_KERNEL_LAUNCH_CHECK();
    count_launches(2);
  });
  return {gates, chosen, counts, balance, z};
}

at::Tensor route_bwd(const OptTensor& dgates, const OptTensor& dbalance, const OptTensor& dz, const at::Tensor& logits,
                     const at::Tensor& experts, const at::Tensor& counts, const OptTensor& mask) {
  TORCH_CHECK_VALUE(experts.dim() == 2 && experts.scalar_type() == at::kLong && experts.device() == logits.device(),
                    "experts: int64 [tokens, top_k] expected");
  check_route(logits, experts.size(1), mask);
  TORCH_CHECK_VALUE(experts.size(0) == logits.size(0) && counts.dim() == 1 && counts.size(0) == logits.size(1) &&
                        counts.scalar_type() == at::kLong && counts.device() == logits.device(),
                    "counts: int64 [experts] expected");
  if (dgates.has_value())
    TORCH_CHECK_VALUE(dgates->sizes() == experts.sizes() && dgates->scalar_type() == logits.scalar_type() &&
                          dgates->device() == logits.device(),
                      "dgates: [tokens, top_k] in the logits' dtype expected");
  for (const auto* s : {&dbalance, &dz})
    if (s->has_value())
      TORCH_CHECK_VALUE((*s)->numel() == 1 && (*s)->scalar_type() == at::kFloat && (*s)->device() == logits.device(),
                        "dbalance, dz: one float32 value expected");
  const c10::cuda::CUDAGuard guard(logits.device());
  auto out = new_empty(logits.sizes(), logits.scalar_type(), logits);
  if (logits.size(0) == 0) return out;
  const auto x = logits.stride(1) == 1 || logits.size(1) == 1 ? logits : logits.contiguous();
  const auto m = mask.has_value() ? mask->contiguous() : at::Tensor();
  const auto chosen = experts.contiguous(), cnt = counts.contiguous();
  const auto dg = dgates.has_value() ? dgates->contiguous() : at::Tensor();
  Args a = args_of(x, m, experts.size(1));
  a.chosen = const_cast<int64_t*>(chosen.const_data_ptr<int64_t>());
  a.counts = const_cast<int64_t*>(cnt.const_data_ptr<int64_t>());
  a.dgates = dg.defined() ? dg.const_data_ptr() : nullptr;
  a.dbalance = dbalance.has_value() ? dbalance->const_data_ptr<float>() : nullptr;
  a.dz = dz.has_value() ? dz->const_data_ptr<float>() : nullptr;
  a.dlogits = out.mutable_data_ptr();
  a.vec_out = whole_words(a.dlogits, a.tokens, a.experts, a.experts, out.element_size());
  with_layout(x, [&](auto* tag, auto lanes, auto values) {
    using T = std::remove_pointer_t<decltype(tag)>;
    constexpr int L = decltype(lanes)::value, V = decltype(values)::value;
    const int groups = kThreads / L;
    const int sms = at::cuda::getCurrentDeviceProperties()->multiProcessorCount;
    const int ctas = (int)std::min<int64_t>((a.tokens + groups - 1) / groups, (int64_t)sms * (L == 32 ? 4 : 8));
    const auto stream = at::cuda::getCurrentCUDAStream();
    if constexpr (L == 32) route_warp_grad_kernel<T, V><<<ctas, kThreads, 0, stream>>>(a);
    else route_grad_kernel<T, L><<<ctas, kThreads, 0, stream>>>(a);
    C10_CUDA_KERNEL_LAUNCH_CHECK();
  });
  count_launches(1);
  return out;
}

}  // namespace dmb
