// RMS norm of each query and key head, its weight, and the position rotation, in one pass.
//
//   r = (mean_i x_i^2 + eps)^(-1/2),  n_i = x_i r w_i,
//   (y_2i, y_2i+1) = (n_2i cos - n_2i+1 sin, n_2i sin + n_2i+1 cos) at the token's position
//   backward: dn = the rotation by the negated angle of dy,  u = dn w,
//   dx = r u - r^3 x mean(u x),  dw = sum over tokens and heads of dn x r
//
// Bound by memory: two values moved per element forward, three backward (r is computed again from
// x, which the backward reads anyway). A row (one head of one token) lies on 8 to 32 lanes, eight
// values each, so that a row's sum takes three to five shuffles and every access is 16 bytes. A
// group of lanes keeps its token's cosines and sines in registers for several heads of that token.
// Queries and keys share one launch. All of it is computed in fp32 and rounded once.
#include <ATen/ATen.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAException.h>
#include <c10/cuda/CUDAGuard.h>

#include "train_ops.h"
#include "vec.cuh"

namespace dmb {
namespace {

constexpr int kThreads = 256;

// One of q and k: [B, S, H, D] with the last stride 1 and every row on a 16-byte boundary.
struct Heads {
  const void* x;
  long long xb, xs, xh;
  const void* dy;
  long long yb, ys, yh;
  void* out;  // contiguous: y forward, dx backward
  const void* weight;
  int heads, chunks;  // a token's heads are split into `chunks` runs
};

struct Args {
  Heads part[2];
  const float *cos, *sin;
  const void* positions;  // null: a token's place in its sequence
  bool wide_positions;    // int64, else int32
  int table;              // rows of cos and sin
  int seq, dim;
  unsigned tokens;
  float eps;
  int* error;
  float* partial;  // backward: [CTAs, 2, D], null where no weight needs a gradient
};

template <typename TW>
__device__ __forceinline__ void load_weight(const void* w, int at, float (&v)[8]) {
  const TW* p = static_cast<const TW*>(w) + at;  // a parameter may lie on any boundary
#pragma unroll
  for (int k = 0; k < 8; ++k) v[k] = to_float(p[k]);
}

template <int LPR>
__device__ __forceinline__ float row_sum(float v) {
#pragma unroll
  for (int o = LPR / 2; o > 0; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
  return v;
}

// The lane's four cosines and sines of a token. A position outside the table makes the token's rows NaN and is reported.
__device__ __forceinline__ void load_turn(const Args& a, unsigned token, int s, int at, bool active, float (&c)[4], float (&sn)[4]) {
  long long pos = s;
  if (a.positions) pos = a.wide_positions ? static_cast<const int64_t*>(a.positions)[token] : static_cast<const int*>(a.positions)[token];
  if (pos < 0 || pos >= a.table) {
    atomicExch(a.error, (int)kErrBadIndex);
#pragma unroll
    for (int k = 0; k < 4; ++k) c[k] = sn[k] = NAN;
    return;
  }
  if (!active) return;
  const long long row = pos * (a.dim / 2) + at / 2;
  const float4 cv = __ldg(reinterpret_cast<const float4*>(a.cos + row)), sv = __ldg(reinterpret_cast<const float4*>(a.sin + row));
  c[0] = cv.x; c[1] = cv.y; c[2] = cv.z; c[3] = cv.w;
  sn[0] = sv.x; sn[1] = sv.y; sn[2] = sv.z; sn[3] = sv.w;
}

// A run of up to HPG heads of one token, by one group of LPR lanes.
template <typename T, typename TW, int LPR, int HPG>
__global__ void __launch_bounds__(kThreads) fwd_kernel(const Args a) {
  const unsigned units_q = a.tokens * a.part[0].chunks, units = units_q + a.tokens * a.part[1].chunks;
  const unsigned group = blockIdx.x * (kThreads / LPR) + threadIdx.x / LPR;
  const int at = (threadIdx.x % LPR) * 8;
  const bool in = group < units, active = in && at < a.dim;
  const bool is_k = in && group >= units_q;
  const Heads& h = a.part[is_k];
  const unsigned unit = in ? group - (is_k ? units_q : 0) : 0;
  const unsigned token = unit / h.chunks, chunk = unit % h.chunks;
  const int h0 = (int)(chunk * HPG), n = in ? min(HPG, h.heads - h0) : 0;
  const long long b = token / a.seq, s = token % a.seq;
  const T* x = static_cast<const T*>(h.x) + b * h.xb + s * h.xs + h0 * h.xh + at;
  T* out = static_cast<T*>(h.out) + ((long long)token * h.heads + h0) * a.dim + at;
  Raw8<T> raw[HPG];
#pragma unroll
  for (int i = 0; i < HPG; ++i)
    if (active && i < n) raw[i] = load_raw8<T>(x + i * h.xh);
  float c[4] = {}, sn[4] = {}, w[8] = {};
  if (in) load_turn(a, token, (int)s, at, active, c, sn);
  if (active) load_weight<TW>(h.weight, at, w);
  const float inv_dim = 1.f / a.dim;
#pragma unroll
  for (int i = 0; i < HPG; ++i) {
    float v[8] = {};
    if (active && i < n) unpack8<T>(raw[i], v);
    float ss = 0.f;
#pragma unroll
    for (int k = 0; k < 8; ++k) ss = fmaf(v[k], v[k], ss);
    const float r = rsqrtf(row_sum<LPR>(ss) * inv_dim + a.eps);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float n0 = v[2 * k] * r * w[2 * k], n1 = v[2 * k + 1] * r * w[2 * k + 1];
      v[2 * k] = n0 * c[k] - n1 * sn[k];
      v[2 * k + 1] = n0 * sn[k] + n1 * c[k];
    }
    if (active && i < n) store8t<T>(out + (long long)i * a.dim, v);
  }
}

// Each group walks over runs of heads, first of the queries and then of the keys, and keeps its
// share of the weights' gradients in registers. The CTA joins its groups' shares in a fixed order.
template <typename T, typename TW, int LPR, int HPG>
__global__ void __launch_bounds__(kThreads) bwd_kernel(const Args a) {
  constexpr int kGroups = kThreads / LPR;
  const int at = (threadIdx.x % LPR) * 8;
  const bool lane_in = at < a.dim;
  const float inv_dim = 1.f / a.dim;
  __shared__ float share[kGroups][LPR * 8 + 4];
#pragma unroll 1
  for (int part = 0; part < 2; ++part) {
    const Heads& h = a.part[part];
    const unsigned units = a.tokens * h.chunks;
    float w[8] = {}, dw[8] = {};
    if (lane_in) load_weight<TW>(h.weight, at, w);
    for (unsigned base = blockIdx.x * kGroups; base < units; base += gridDim.x * kGroups) {
      const unsigned group = base + threadIdx.x / LPR;
      const bool in = group < units, active = in && lane_in;
      const unsigned unit = in ? group : 0;
      const unsigned token = unit / h.chunks, chunk = unit % h.chunks;
      const int h0 = (int)(chunk * HPG), n = in ? min(HPG, h.heads - h0) : 0;
      const long long b = token / a.seq, s = token % a.seq;
      const T* x = static_cast<const T*>(h.x) + b * h.xb + s * h.xs + h0 * h.xh + at;
      const T* dy = static_cast<const T*>(h.dy) + b * h.yb + s * h.ys + h0 * h.yh + at;
      T* out = static_cast<T*>(h.out) + ((long long)token * h.heads + h0) * a.dim + at;
      Raw8<T> rx[HPG], ry[HPG];
#pragma unroll
      for (int i = 0; i < HPG; ++i)
        if (active && i < n) {
          rx[i] = load_raw8<T>(x + i * h.xh);
          ry[i] = load_raw8<T>(dy + i * h.yh);
        }
      float c[4] = {}, sn[4] = {};
      if (in) load_turn(a, token, (int)s, at, active, c, sn);
#pragma unroll
      for (int i = 0; i < HPG; ++i) {
        float v[8] = {}, g[8] = {};
        if (active && i < n) {
          unpack8<T>(rx[i], v);
          unpack8<T>(ry[i], g);
        }
        float ss = 0.f, dot = 0.f;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float g0 = g[2 * k] * c[k] + g[2 * k + 1] * sn[k], g1 = g[2 * k + 1] * c[k] - g[2 * k] * sn[k];
          g[2 * k] = g0;
          g[2 * k + 1] = g1;
        }
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          ss = fmaf(v[k], v[k], ss);
          dot = fmaf(g[k] * w[k], v[k], dot);
        }
        ss = row_sum<LPR>(ss);
        dot = row_sum<LPR>(dot);
        const float r = rsqrtf(ss * inv_dim + a.eps), f = r * r * dot * inv_dim;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const float xr = v[k] * r;
          if (i < n) dw[k] = fmaf(g[k], xr, dw[k]);
          v[k] = r * (g[k] * w[k] - v[k] * f);
        }
        if (active && i < n) store8t<T>(out + (long long)i * a.dim, v);
      }
    }
    if (a.partial) {
#pragma unroll
      for (int k = 0; k < 8; ++k) share[threadIdx.x / LPR][at + k] = dw[k];
      __syncthreads();
      for (int j = threadIdx.x; j < a.dim; j += kThreads) {
        float sum = 0.f;
#pragma unroll
        for (int gr = 0; gr < kGroups; ++gr) sum += share[gr][j];
        a.partial[((long long)blockIdx.x * 2 + part) * a.dim + j] = sum;
      }
      __syncthreads();
    }
  }
}

// Sum of the CTAs' shares: 32 lanes for each of 8 columns... one warp per column, in a fixed order.
template <typename TW>
__global__ void __launch_bounds__(kThreads) weight_grad_kernel(const float* partial, int ctas, int dim, TW* dwq, TW* dwk) {
  __shared__ float smem[8][33];
  const int col = blockIdx.x * 32 + (threadIdx.x & 31), slice = threadIdx.x >> 5;
  float sum = 0.f;
  if (col < 2 * dim)
    for (int i = slice; i < ctas; i += 8) sum += partial[(long long)i * 2 * dim + col];
  smem[slice][threadIdx.x & 31] = sum;
  __syncthreads();
  if (slice == 0 && col < 2 * dim) {
#pragma unroll
    for (int i = 1; i < 8; ++i) sum += smem[i][threadIdx.x & 31];
    (col < dim ? dwq : dwk)[col < dim ? col : col - dim] = from_float<TW>(sum);
  }
}

// ------------------------------------------------------------------ host

// [B, S, H, D] as the kernels read it, copied only where a row does not lie on a 16-byte boundary.
at::Tensor rows16(const at::Tensor& t) {
  const int64_t size = t.element_size();
  bool ok = t.stride(3) == 1 && reinterpret_cast<uintptr_t>(t.const_data_ptr()) % 16 == 0;
  for (int i = 0; i < 3; ++i) ok = ok && (t.size(i) <= 1 || t.stride(i) * size % 16 == 0);
  if (ok) return t;
  return t.is_contiguous() ? t.clone(at::MemoryFormat::Contiguous) : t.contiguous();
}

void check_heads(const at::Tensor& q, const at::Tensor& k, const at::Tensor& qw, const at::Tensor& kw,
                 const at::Tensor& cos, const at::Tensor& sin, const OptTensor& positions) {
  TORCH_CHECK_VALUE(q.is_cuda() && k.device() == q.device(), "q, k: tensors of one CUDA device expected");
  TORCH_CHECK_VALUE(q.dim() == 4 && k.dim() == 4 && q.size(0) == k.size(0) && q.size(1) == k.size(1) && q.size(3) == k.size(3),
                    "q, k: [batch, seq, heads, head_dim] of one batch, seq and head_dim expected");
  TORCH_CHECK_VALUE(q.scalar_type() == k.scalar_type(), "q, k: one dtype expected");
  const int64_t d = q.size(3);
  TORCH_CHECK_VALUE(d % 8 == 0 && d >= 8 && d <= 256, "head_dim: a multiple of 8 up to 256 expected, got ", d);
  for (const auto* w : {&qw, &kw})
    TORCH_CHECK_VALUE(w->device() == q.device() && w->dim() == 1 && w->size(0) == d &&
                          (w->scalar_type() == q.scalar_type() || w->scalar_type() == at::kFloat) &&
                          w->scalar_type() == qw.scalar_type(),
                      "q_weight, k_weight: [head_dim] in the heads' dtype or both in float32 expected");
  for (const auto* t : {&cos, &sin})
    TORCH_CHECK_VALUE(t->device() == q.device() && t->scalar_type() == at::kFloat && t->dim() == 2 && t->size(1) == d / 2 &&
                          t->size(0) == cos.size(0) && (positions.has_value() || t->size(0) >= q.size(1)),
                      "cos, sin: float32 [positions, head_dim / 2] with a row for every position expected");
  if (positions.has_value())
    TORCH_CHECK_VALUE((positions->scalar_type() == at::kLong || positions->scalar_type() == at::kInt) &&
                          positions->device() == q.device() && positions->dim() == 2 && positions->size(0) == q.size(0) &&
                          positions->size(1) == q.size(1),
                      "positions: int64 or int32 [batch, seq] expected");
  TORCH_CHECK_VALUE(q.size(0) * q.size(1) * std::max(q.size(2), k.size(2)) < (1ll << 30), "q, k: at most 2^30 heads of tokens expected");
}

// A table on a 16-byte boundary (its rows are multiples of 16 bytes: head_dim is one of 8).
at::Tensor table16(const at::Tensor& t) {
  const auto c = t.contiguous();
  return reinterpret_cast<uintptr_t>(c.const_data_ptr()) % 16 ? c.clone() : c;
}

struct Kept {  // tensors that the launch reads from
  at::Tensor q, k, dq, dk, cos, sin, pos, qw, kw;
};

int lanes_per_row(int64_t d) { return d <= 64 ? 8 : d <= 128 ? 16 : 32; }

Args args_of(Kept& t, const at::Tensor& q, const at::Tensor& k, const at::Tensor& qw, const at::Tensor& kw,
             const at::Tensor& cos, const at::Tensor& sin, const OptTensor& positions, double eps, int hpg) {
  t.q = rows16(q);
  t.k = rows16(k);
  t.cos = table16(cos);
  t.sin = table16(sin);
  t.qw = qw.contiguous();
  t.kw = kw.contiguous();
  Args a = {};
  const at::Tensor* xs[2] = {&t.q, &t.k};
  const at::Tensor* ws[2] = {&t.qw, &t.kw};
  for (int i = 0; i < 2; ++i) {
    Heads& h = a.part[i];
    h.x = xs[i]->const_data_ptr();
    h.xb = xs[i]->stride(0);
    h.xs = xs[i]->stride(1);
    h.xh = xs[i]->stride(2);
    h.weight = ws[i]->const_data_ptr();
    h.heads = (int)xs[i]->size(2);
    h.chunks = std::max(1, (h.heads + hpg - 1) / hpg);
  }
  a.cos = t.cos.const_data_ptr<float>();
  a.sin = t.sin.const_data_ptr<float>();
  a.table = (int)cos.size(0);
  if (positions.has_value()) {
    t.pos = positions->contiguous();
    a.positions = t.pos.const_data_ptr();
    a.wide_positions = t.pos.scalar_type() == at::kLong;
  }
  a.seq = (int)std::max<int64_t>(1, q.size(1));
  a.dim = (int)q.size(3);
  a.tokens = (unsigned)(q.size(0) * q.size(1));
  a.eps = (float)eps;
  a.error = device_error_word(q.device().index());
  return a;
}

// Heads per group: four share a token's angles once there are enough of them to fill the GPU.
int heads_per_group(const at::Tensor& q, const at::Tensor& k) {
  const int64_t rows = q.size(0) * q.size(1) * (q.size(2) + k.size(2));
  const int64_t lanes = (int64_t)at::cuda::getCurrentDeviceProperties()->multiProcessorCount * 1024;
  return rows * lanes_per_row(q.size(3)) / 4 >= lanes ? 4 : 1;
}

// f(T, TW, LPR) with null pointers for the types
template <typename F>
void with_types(const at::Tensor& q, const at::Tensor& w, F&& f) {
  with_element(q.scalar_type(), [&](auto* t) {
    using T = std::remove_pointer_t<decltype(t)>;
    auto lanes = [&](auto* tw) {
      switch (lanes_per_row(q.size(3))) {
        case 8: return f(t, tw, std::integral_constant<int, 8>());
        case 16: return f(t, tw, std::integral_constant<int, 16>());
        default: return f(t, tw, std::integral_constant<int, 32>());
      }
    };
    if (w.scalar_type() == at::kFloat) return lanes(static_cast<float*>(nullptr));
    if constexpr (!std::is_same<T, float>::value) lanes(static_cast<T*>(nullptr));
  });
}

}  // namespace

std::tuple<at::Tensor, at::Tensor> qk_norm_rope_fwd(const at::Tensor& q, const at::Tensor& k, const at::Tensor& q_weight,
                                                    const at::Tensor& k_weight, const at::Tensor& cos,
                                                    const at::Tensor& sin, const OptTensor& positions, double eps) {
  check_heads(q, k, q_weight, k_weight, cos, sin, positions);
  const c10::cuda::CUDAGuard guard(q.device());
  auto qo = at::empty(q.sizes(), q.options().memory_format(at::MemoryFormat::Contiguous));
  auto ko = at::empty(k.sizes(), k.options().memory_format(at::MemoryFormat::Contiguous));
  if (q.numel() + k.numel() == 0) return {qo, ko};
  Kept t;
  const int hpg = heads_per_group(q, k);
  Args a = args_of(t, q, k, q_weight, k_weight, cos, sin, positions, eps, hpg);
  a.part[0].out = qo.mutable_data_ptr();
  a.part[1].out = ko.mutable_data_ptr();
  const int64_t units = (int64_t)a.tokens * (a.part[0].chunks + a.part[1].chunks);
  with_types(q, q_weight, [&](auto* tt, auto* tw, auto lanes) {
    using T = std::remove_pointer_t<decltype(tt)>;
    using TW = std::remove_pointer_t<decltype(tw)>;
    constexpr int L = decltype(lanes)::value;
    const unsigned grid = (unsigned)((units + kThreads / L - 1) / (kThreads / L));
    const auto stream = at::cuda::getCurrentCUDAStream();
    if (hpg == 4) fwd_kernel<T, TW, L, 4><<<grid, kThreads, 0, stream>>>(a);
    else fwd_kernel<T, TW, L, 1><<<grid, kThreads, 0, stream>>>(a);
    C10_CUDA_KERNEL_LAUNCH_CHECK();
  });
  count_launches(1);
  return {qo, ko};
}

std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor> qk_norm_rope_bwd(
    const at::Tensor& dq_out, const at::Tensor& dk_out, const at::Tensor& q, const at::Tensor& k,
    const at::Tensor& q_weight, const at::Tensor& k_weight, const at::Tensor& cos, const at::Tensor& sin,
    const OptTensor& positions, double eps, bool weight_grads) {
  check_heads(q, k, q_weight, k_weight, cos, sin, positions);
  TORCH_CHECK_VALUE(dq_out.sizes() == q.sizes() && dk_out.sizes() == k.sizes() && dq_out.scalar_type() == q.scalar_type() &&
                        dk_out.scalar_type() == k.scalar_type() && dq_out.device() == q.device() && dk_out.device() == q.device(),
                    "gradients of the heads' shapes, dtype and device expected");
  const c10::cuda::CUDAGuard guard(q.device());
  auto dq = at::empty(q.sizes(), q.options().memory_format(at::MemoryFormat::Contiguous));
  auto dk = at::empty(k.sizes(), k.options().memory_format(at::MemoryFormat::Contiguous));
  const auto wsize = weight_grads ? q.size(3) : 0;
  auto dwq = at::empty({wsize}, q_weight.options()), dwk = at::empty({wsize}, k_weight.options());
  if (q.numel() + k.numel() == 0) return {dq, dk, dwq.zero_(), dwk.zero_()};
  Kept t;
  t.dq = rows16(dq_out);
  t.dk = rows16(dk_out);
  const int hpg = heads_per_group(q, k) == 4 ? 2 : 1;
  Args a = args_of(t, q, k, q_weight, k_weight, cos, sin, positions, eps, hpg);
  const at::Tensor* dys[2] = {&t.dq, &t.dk};
  for (int i = 0; i < 2; ++i) {
    a.part[i].dy = dys[i]->const_data_ptr();
    a.part[i].yb = dys[i]->stride(0);
    a.part[i].ys = dys[i]->stride(1);
    a.part[i].yh = dys[i]->stride(2);
  }
  a.part[0].out = dq.mutable_data_ptr();
  a.part[1].out = dk.mutable_data_ptr();
  const int64_t units = (int64_t)a.tokens * std::max(a.part[0].chunks, a.part[1].chunks);
  const int groups = kThreads / lanes_per_row(q.size(3));
  const int sms = at::cuda::getCurrentDeviceProperties()->multiProcessorCount;
  const int ctas = (int)std::min<int64_t>((units + groups - 1) / groups, (int64_t)sms * 4);
  at::Tensor partial;
  if (weight_grads) {
    partial = at::empty({ctas, 2, q.size(3)}, q.options().dtype(at::kFloat));
    a.partial = partial.mutable_data_ptr<float>();
  }
  with_types(q, q_weight, [&](auto* tt, auto* tw, auto lanes) {
    using T = std::remove_pointer_t<decltype(tt)>;
    using TW = std::remove_pointer_t<decltype(tw)>;
    constexpr int L = decltype(lanes)::value;
    const auto stream = at::cuda::getCurrentCUDAStream();
    if (hpg == 2) bwd_kernel<T, TW, L, 2><<<ctas, kThreads, 0, stream>>>(a);
    else bwd_kernel<T, TW, L, 1><<<ctas, kThreads, 0, stream>>>(a);
    C10_CUDA_KERNEL_LAUNCH_CHECK();
    if (weight_grads) {
      weight_grad_kernel<TW><<<(2 * a.dim + 31) / 32, kThreads, 0, stream>>>(
          a.partial, ctas, a.dim, static_cast<TW*>(dwq.mutable_data_ptr()), static_cast<TW*>(dwk.mutable_data_ptr()));
      C10_CUDA_KERNEL_LAUNCH_CHECK();
    }
  });
  count_launches(weight_grads ? 2 : 1);
  return {dq, dk, dwq, dwk};
}

}  // namespace dmb
