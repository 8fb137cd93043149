// Router of a sparse layer: top-k experts of each token with their gates, the number of tokens of
// each expert, the balance loss and the z loss.
//
//   p = softmax(l) over all E experts;  experts = the k greatest l, equal ones by index;  g = softmax(l[experts])
//   c_e = choices of e by the N tokens that count
//   balance = E / (N^2 k) sum_e c_e sum_t p_te   (1 where every expert gets the same),  z = 1/N sum_t lse_t^2
//   dl = g (dg - g.dg) at the chosen + p (dbalance E / (N^2 k) (c_e - c.p) + dz 2/N lse)
//
// A row lies on 1 to 32 lanes, eight logits (16 bytes of a 16-bit type) or two or four times that
// on each. The choice takes k rounds of a maximum over the row by (value, index). Every group of
// lanes walks over rows and keeps its sums of p and its counts in registers; a CTA joins them in a
// fixed order and writes one part, and a second kernel of one CTA sums the parts in 64 bits. So
// there are no atomics, and a run gives the same bits each time. What bounds it: launches for small
// batches, the k rounds for many experts; the logits are read once forward and once backward.
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
  bool vec;          // rows of whole 16-byte words on 16-byte boundaries
  int tokens, experts, top_k;
  const bool* mask;  // null: every token counts
  // forward
  void* gates;
  int64_t* chosen;
  int64_t* counts;
  float* sum_p;  // [E + 1, CTAs]: sums of p, last the sum of lse^2
  int* sum_c;    // [E + 1, CTAs]: choices, last the tokens that count
  // backward
  const void* dgates;                // null: none
  const float *dbalance, *dz;        // null: none
  void* dlogits;
};

// Expert of a lane's j-th value: whole 8-value words lie next to each other across the lanes.
template <int LPR>
__device__ __forceinline__ int expert_of(int lane, int j) { return (j >> 3) * LPR * 8 + lane * 8 + (j & 7); }

template <typename T, int LPR, int VPL>
__device__ __forceinline__ void load_row(const Args& a, int row, bool in, int lane, float (&x)[VPL]) {
  const T* p = static_cast<const T*>(a.logits) + (long long)row * a.stride;
#pragma unroll
  for (int j = 0; j < VPL; j += 8) {
    const int e = expert_of<LPR>(lane, j);
    float v[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = -INFINITY;
    if (in) {
      if (a.vec) {
        if (e < a.experts) load8t<T>(p + e, v);
      } else {
#pragma unroll
        for (int k = 0; k < 8; ++k)
          if (e + k < a.experts) v[k] = to_float(p[e + k]);
      }
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) x[j + k] = v[k];
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

template <typename T, int LPR, int VPL>
__global__ void __launch_bounds__(kThreads) route_kernel(const Args a) {
  constexpr int kGroups = kThreads / LPR, kExperts = LPR * VPL;
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
    load_row<T, LPR, VPL>(a, row, in, lane, x);
    uint32_t key[VPL];
#pragma unroll
    for (int j = 0; j < VPL; ++j) key[j] = expert_of<LPR>(lane, j) < a.experts ? order_key(x[j]) : 0u;
    uint32_t picked = 0;  // bit j: the lane's j-th expert is chosen
    float top = 0.f, total = 0.f;
    for (int i = 0; i < a.top_k; ++i) {
      uint32_t best = 0;
      int at = 0;
#pragma unroll
      for (int j = 0; j < VPL; ++j)
        if (key[j] > best) {  // within a lane, a later value has a higher index
          best = key[j];
          at = expert_of<LPR>(lane, j);
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
        if (expert_of<LPR>(lane, j) == at) {
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
      join_p[warp * (kExperts + 1) + expert_of<LPR>(lane, j)] = sum_p[j];
      join_c[warp * (kExperts + 1) + expert_of<LPR>(lane, j)] = sum_c[j];
    }
    if (lane == 0) {
      join_p[warp * (kExperts + 1) + kExperts] = sum_z;
      join_c[warp * (kExperts + 1) + kExperts] = sum_n;
    }
  }
  __syncthreads();
  for (int e = threadIdx.x; e <= a.experts; e += kThreads) {
    const int from = e < a.experts ? e : kExperts;
    float p = 0.f;
    int c = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      p += join_p[w * (kExperts + 1) + from];
      c += join_c[w * (kExperts + 1) + from];
    }
    a.sum_p[(long long)e * gridDim.x + blockIdx.x] = p;
    a.sum_c[(long long)e * gridDim.x + blockIdx.x] = c;
  }
}

constexpr int kJoinThreads = 512;

// A warp sums each expert's parts.
__global__ void __launch_bounds__(kJoinThreads) route_join_kernel(const Args a, int parts, float* balance, float* z) {
  __shared__ double sum_p[kMaxExperts + 1];
  __shared__ int sum_c[kMaxExperts + 1];
  const int lane = threadIdx.x & 31;
  for (int e = threadIdx.x >> 5; e <= a.experts; e += kJoinThreads / 32) {
    double p = 0;
    int c = 0;
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
      sum_p[e] = p;
      sum_c[e] = c;
    }
  }
  __syncthreads();
  for (int e = threadIdx.x; e < a.experts; e += kJoinThreads) a.counts[e] = sum_c[e];
  if (threadIdx.x < 32) {
    double dot = 0;
    for (int e = lane; e < a.experts; e += 32) dot += sum_p[e] * sum_c[e];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) dot += __shfl_xor_sync(~0u, dot, o);
    if (lane == 0) {
      const double n = sum_c[a.experts];
      *balance = n > 0 ? (float)(dot * a.experts / (n * n * a.top_k)) : 0.f;
      *z = n > 0 ? (float)(sum_p[a.experts] / n) : 0.f;
    }
  }
}

template <typename T, int LPR, int VPL>
__global__ void __launch_bounds__(kThreads) route_grad_kernel(const Args a) {
  constexpr int kGroups = kThreads / LPR, kExperts = LPR * VPL;
  __shared__ float share[kExperts];  // c_e / (N k)
  __shared__ int choices;
  const int lane = threadIdx.x % LPR, group = threadIdx.x / LPR;
  if (threadIdx.x < 32) {
    int n = 0;
    for (int e = threadIdx.x; e < a.experts; e += 32) n += (int)a.counts[e];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) n += __shfl_xor_sync(~0u, n, o);
    if (threadIdx.x == 0) choices = n;
  }
  __syncthreads();
  for (int e = threadIdx.x; e < kExperts; e += kThreads)
    share[e] = e < a.experts && choices > 0 ? (float)((double)a.counts[e] / choices) : 0.f;
  __syncthreads();
  const float n = (float)(choices / a.top_k);
  const float by_balance = a.dbalance && choices > 0 ? *a.dbalance * a.experts / n : 0.f;
  const float by_z = a.dz && choices > 0 ? *a.dz * 2.f / n : 0.f;
  for (int base = blockIdx.x * kGroups; base < a.tokens; base += gridDim.x * kGroups) {
    const int row = base + group;
    const bool in = row < a.tokens;
    const bool valid = in && (!a.mask || a.mask[row]);
    float x[VPL];
    load_row<T, LPR, VPL>(a, row, valid, lane, x);
    uint32_t picked = 0;
    float dg[VPL] = {};
    if (valid && a.dgates) {
      for (int i = 0; i < a.top_k; ++i) {
        const long long at = (long long)row * a.top_k + i;
        const int64_t expert = a.chosen[at];
        const float d = to_float(static_cast<const T*>(a.dgates)[at]);
#pragma unroll
        for (int j = 0; j < VPL; ++j)
          if (expert_of<LPR>(lane, j) == expert) {
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
      mix = fmaf(share[expert_of<LPR>(lane, j)], x[j], mix);
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
#pragma unroll
    for (int j = 0; j < VPL; j += 8) {
      const int e = expert_of<LPR>(lane, j);
      float v[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        float g = x[j + k] * inv * fmaf(by_balance, share[e + k], all);
        if ((picked >> (j + k)) & 1) g = fmaf(x[j + k] * inv_top, dg[j + k] - dot, g);
        v[k] = valid ? g : 0.f;
      }
      if (a.experts % 8 == 0) {
        if (e < a.experts) store8t<T>(out + e, v);
      } else {
#pragma unroll
        for (int k = 0; k < 8; ++k)
          if (e + k < a.experts) out[e + k] = from_float<T>(v[k]);
      }
    }
  }
}

// ------------------------------------------------------------------ host

// f(T, LPR, VPL): as few lanes per row as hold it at eight values each, then more values.
template <typename F>
void with_layout(const at::Tensor& logits, F&& f) {
  with_element(logits.scalar_type(), [&](auto* t) {
    const int e = (int)logits.size(1);
    using std::integral_constant;
    if (e <= 8) f(t, integral_constant<int, 1>(), integral_constant<int, 8>());
    else if (e <= 16) f(t, integral_constant<int, 2>(), integral_constant<int, 8>());
    else if (e <= 32) f(t, integral_constant<int, 4>(), integral_constant<int, 8>());
    else if (e <= 64) f(t, integral_constant<int, 8>(), integral_constant<int, 8>());
    else if (e <= 128) f(t, integral_constant<int, 16>(), integral_constant<int, 8>());
    else if (e <= 256) f(t, integral_constant<int, 32>(), integral_constant<int, 8>());
    else f(t, integral_constant<int, 32>(), integral_constant<int, 16>());
  });
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
  a.vec = a.experts % 8 == 0 && (a.tokens <= 1 || a.stride * logits.element_size() % 16 == 0) &&
          reinterpret_cast<uintptr_t>(a.logits) % 16 == 0;
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
  const auto f32 = logits.options().dtype(at::kFloat), i64 = logits.options().dtype(at::kLong);
  const int64_t t = x.size(0), e = x.size(1);
  auto gates = at::empty({t, top_k}, logits.options().memory_format(at::MemoryFormat::Contiguous));
  auto chosen = at::empty({t, top_k}, i64), counts = at::empty({e}, i64);
  auto balance = at::empty({}, f32), z = at::empty({}, f32);
  Args a = args_of(x, m, top_k);
  a.gates = gates.mutable_data_ptr();
  a.chosen = chosen.mutable_data_ptr<int64_t>();
  a.counts = counts.mutable_data_ptr<int64_t>();
  const auto stream = at::cuda::getCurrentCUDAStream();
  with_layout(x, [&](auto* tag, auto lanes, auto values) {
    using T = std::remove_pointer_t<decltype(tag)>;
    constexpr int L = decltype(lanes)::value, V = decltype(values)::value;
    const int groups = kThreads / L;
    const int sms = at::cuda::getCurrentDeviceProperties()->multiProcessorCount;
    const int ctas = (int)std::min<int64_t>((t + groups - 1) / groups, (int64_t)sms * 4);
    auto part_p = at::empty({e + 1, ctas}, f32), part_c = at::empty({e + 1, ctas}, f32.dtype(at::kInt));
    a.sum_p = part_p.template mutable_data_ptr<float>();
    a.sum_c = part_c.template mutable_data_ptr<int>();
    if (ctas) {
      route_kernel<T, L, V><<<ctas, kThreads, 0, stream>>>(a);
      C10_CUDA_KERNEL_LAUNCH_CHECK();
    }
    route_join_kernel<<<1, kJoinThreads, 0, stream>>>(a, ctas, balance.template mutable_data_ptr<float>(),
                                                      z.template mutable_data_ptr<float>());
    C10_CUDA_KERNEL_LAUNCH_CHECK();
    count_launches(ctas ? 2 : 1);
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
  auto out = at::empty(logits.sizes(), logits.options().memory_format(at::MemoryFormat::Contiguous));
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
  with_layout(x, [&](auto* tag, auto lanes, auto values) {
    using T = std::remove_pointer_t<decltype(tag)>;
    constexpr int L = decltype(lanes)::value, V = decltype(values)::value;
    const int groups = kThreads / L;
    const int sms = at::cuda::getCurrentDeviceProperties()->multiProcessorCount;
    const int ctas = (int)std::min<int64_t>((a.tokens + groups - 1) / groups, (int64_t)sms * 8);
    route_grad_kernel<T, L, V><<<ctas, kThreads, 0, at::cuda::getCurrentCUDAStream()>>>(a);
    C10_CUDA_KERNEL_LAUNCH_CHECK();
  });
  count_launches(1);
  return out;
}

}  // namespace dmb
