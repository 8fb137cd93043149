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
// Queries and keys share one launch. All of it is computed in fp32 and rounded once. Unpacked
// arithmetic would take longer than the memory: the first and the second values of a lane's four
// rotated pairs lie in packed registers, two and two, so that nothing is shuffled between them.
// Measured on one B200, between events around queued calls: 4096 tokens of 32 + 8 heads of 128 bf16 take 18.5 us
// forward (84 MB, 4.5 TB/s) and 31 us backward (126 MB, 4.0 TB/s) with the 3 us for the sum of the weights' gradients
// over the CTAs; 16384 tokens 64 and 92 us (5.2 and 5.5 TB/s); 4096 tokens of fp32 32 and 66 us. An RMS norm and a
// rotation one after the other, each with its gradient, take 443 us for the 51 of the 4096 tokens here.
#include <ATen/ATen.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAException.h>
#include <c10/cuda/CUDAGuard.h>

#include "train_ops.h"
#include "vec.cuh"

namespace dmb {
namespace {

constexpr int kThreads = 256;

// n / d for n < 2^31 by a multiplication (Granlund and Montgomery): the kernels' rows are found by divisions that would
// otherwise stand in front of every load.
struct Divisor {
  unsigned d, mul, shift;
  Divisor(unsigned by = 1) : d(by), mul(0), shift(0) {
    while ((1ull << shift) < d) ++shift;
    mul = (unsigned)(((1ull << 32) * ((1ull << shift) - d)) / d + 1);
  }
  __device__ __forceinline__ unsigned div(unsigned n) const { return (__umulhi(n, mul) + n) >> shift; }
};

// One of q and k: [B, S, H, D] with the last stride 1 and every row on a 16-byte boundary.
struct Heads {
  const void* x;
  long long xb, xs, xh;
  const void* dy;
  long long yb, ys, yh;
  void* out;  // contiguous: y forward, dx backward
  const void* weight;
  int heads;
  Divisor chunks;  // a token's heads are split into so many runs
};

struct Args {
  Heads part[2];
  const float *cos, *sin;
  const void* positions;  // null: a token's place in its sequence
  bool wide_positions;    // int64, else int32
  int table;              // rows of cos and sin
  Divisor seq;
  int dim;
  unsigned tokens;
  float eps;
  int* error;
  float* partial;  // backward: [CTAs, 2, D], null where no weight needs a gradient
};

// A lane's eight values as four rotated pairs: a holds the pairs' first values (x0, x2), (x4, x6), b their second ones.
struct Pairs {
  F2 a[2], b[2];
};

template <typename T>
__device__ __forceinline__ Pairs to_pairs(const Raw8<T>& r) {
  float v[8];
  unpack8<T>(r, v);
  Pairs p;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    p.a[i] = f2(v[4 * i], v[4 * i + 2]);
    p.b[i] = f2(v[4 * i + 1], v[4 * i + 3]);
  }
  return p;
}

template <typename T>
__device__ __forceinline__ void store_pairs(T* to, const Pairs& p) {
  float v[8];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const float2 a = f2_values(p.a[i]), b = f2_values(p.b[i]);
    v[4 * i] = a.x;
    v[4 * i + 1] = b.x;
    v[4 * i + 2] = a.y;
    v[4 * i + 3] = b.y;
  }
  store8t<T>(to, v);
}

__device__ __forceinline__ Pairs no_pairs() {
  const F2 z = f2(0.f, 0.f);
  return Pairs{{z, z}, {z, z}};
}

// sum of x y over the lane's values
__device__ __forceinline__ float dot8(const Pairs& x, const Pairs& y) {
  const F2 s = fma2(x.b[1], y.b[1], fma2(x.a[1], y.a[1], fma2(x.b[0], y.b[0], x.a[0] * y.a[0])));
  const float2 v = f2_values(s);
  return v.x + v.y;
}

struct Turn {
  F2 cos[2], sin[2], minus[2];
};

// The rotation by the angle: first and second value of each pair; by the negated angle with sin and minus exchanged.
__device__ __forceinline__ Pairs rotate(const Pairs& x, const F2 (&c)[2], const F2 (&s)[2], const F2 (&minus)[2]) {
  Pairs y;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    y.a[i] = fma2(x.b[i], minus[i], x.a[i] * c[i]);
    y.b[i] = fma2(x.a[i], s[i], x.b[i] * c[i]);
  }
  return y;
}

template <int LPR>
__device__ __forceinline__ float row_sum(float v) {
#pragma unroll
  for (int o = LPR / 2; o > 0; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
  return v;
}

// The lane's four cosines and sines of a token. A position outside the table makes the token's rows NaN and is reported.
struct Angles {
  float4 cos, sin;
};

__device__ __forceinline__ Angles load_angles(const Args& a, unsigned token, unsigned s, int at, bool active) {
  Angles r;
  r.cos = r.sin = make_float4(0.f, 0.f, 0.f, 0.f);
  if (active) {
    long long pos = s;
    if (a.positions) pos = a.wide_positions ? static_cast<const int64_t*>(a.positions)[token] : static_cast<const int*>(a.positions)[token];
    if (pos < 0 || pos >= a.table) {
      atomicExch(a.error, (int)kErrBadIndex);
      r.cos = r.sin = make_float4(NAN, NAN, NAN, NAN);
    } else {
      const long long row = pos * (a.dim / 2) + at / 2;
      r.cos = __ldg(reinterpret_cast<const float4*>(a.cos + row));
      r.sin = __ldg(reinterpret_cast<const float4*>(a.sin + row));
    }
  }
  return r;
}

__device__ __forceinline__ Turn turn_of(const Angles& g) {
  return Turn{{f2(g.cos.x, g.cos.y), f2(g.cos.z, g.cos.w)},
              {f2(g.sin.x, g.sin.y), f2(g.sin.z, g.sin.w)},
              {f2(-g.sin.x, -g.sin.y), f2(-g.sin.z, -g.sin.w)}};
}

// A run of up to HPG heads of one token, by one group of LPR lanes.
template <typename T, typename TW, int LPR, int HPG>
__global__ void __launch_bounds__(kThreads) fwd_kernel(const Args a) {
  const unsigned units_q = a.tokens * a.part[0].chunks.d, units = units_q + a.tokens * a.part[1].chunks.d;
  const unsigned group = blockIdx.x * (kThreads / LPR) + threadIdx.x / LPR;
  const int at = (threadIdx.x % LPR) * 8;
  const bool active = group < units && at < a.dim;
  const bool is_k = group >= units_q;
  const Heads& h = a.part[is_k];
  const unsigned unit = group < units ? group - (is_k ? units_q : 0) : 0;
  const unsigned token = h.chunks.div(unit), chunk = unit - token * h.chunks.d;
  const int h0 = (int)(chunk * HPG), n = active ? min(HPG, h.heads - h0) : 0;
  const unsigned b = a.seq.div(token), s = token - b * a.seq.d;
  const T* x = static_cast<const T*>(h.x) + b * h.xb + s * h.xs + h0 * h.xh + at;
  T* out = static_cast<T*>(h.out) + ((long long)token * h.heads + h0) * a.dim + at;
  Raw8<T> raw[HPG];
#pragma unroll
  for (int i = 0; i < HPG; ++i)
    if (i < n) raw[i] = load_raw8<T>(x + i * h.xh);
  const Turn turn = turn_of(load_angles(a, token, s, at, active));
  Pairs w = no_pairs();
  if (active) w = to_pairs<TW>(load_raw8<TW>(static_cast<const TW*>(h.weight) + at));
  const float inv_dim = 1.f / a.dim;
#pragma unroll
  for (int i = 0; i < HPG; ++i) {
    Pairs v = no_pairs();
    if (i < n) v = to_pairs<T>(raw[i]);
    const float r = rsqrtf(row_sum<LPR>(dot8(v, v)) * inv_dim + a.eps);
    const F2 r2 = f2(r, r);
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      v.a[j] = v.a[j] * r2 * w.a[j];
      v.b[j] = v.b[j] * r2 * w.b[j];
    }
    if (i < n) store_pairs<T>(out + (long long)i * a.dim, rotate(v, turn.cos, turn.sin, turn.minus));
  }
}

// Each group walks over runs of heads, first of the queries and then of the keys, and keeps its share of the weights'
// gradients in registers; the CTA joins its groups' shares in a fixed order. While a lane computes, its next run's values
// are on their way into its own slots of shared memory, which take no registers and need no barrier.
template <typename T, typename TW, int LPR, int HPG>
__global__ void __launch_bounds__(kThreads, sizeof(T) == 4 ? 2 : 3) bwd_kernel(const Args a) {
  constexpr int kGroups = kThreads / LPR, kWords = sizeof(T) / 2;
  extern __shared__ __align__(16) uint4 slots[];  // [2][HPG][x, dy][kWords][kThreads]
  const int at = (threadIdx.x % LPR) * 8;
  const bool lane_in = at < a.dim;
  const float inv_dim = 1.f / a.dim;
  __shared__ float share[kGroups][LPR * 8 + 4];
#pragma unroll 1
  for (int part = 0; part < 2; ++part) {
    const Heads& h = a.part[part];
    const unsigned units = a.tokens * h.chunks.d, step = gridDim.x * kGroups;
    Pairs w = no_pairs(), dw = no_pairs();
    if (lane_in) w = to_pairs<TW>(load_raw8<TW>(static_cast<const TW*>(h.weight) + at));
    Angles angles;
    long long next_out = 0;
    int next_n = 0;
    auto fetch = [&](unsigned group, int slot) {
      const bool active = group < units && lane_in;
      const unsigned unit = group < units ? group : 0;
      const unsigned token = h.chunks.div(unit), chunk = unit - token * h.chunks.d;
      const int h0 = (int)(chunk * HPG);
      const unsigned b = a.seq.div(token), s = token - b * a.seq.d;
      next_n = active ? min(HPG, h.heads - h0) : 0;
      next_out = ((long long)token * h.heads + h0) * a.dim + at;
      const T* x = static_cast<const T*>(h.x) + b * h.xb + s * h.xs + h0 * h.xh + at;
      const T* dy = static_cast<const T*>(h.dy) + b * h.yb + s * h.ys + h0 * h.yh + at;
      const uint32_t to = smem_u32(slots + (slot * HPG * 2 * kWords) * kThreads + threadIdx.x);
#pragma unroll
      for (int i = 0; i < HPG; ++i)
        if (i < next_n) {
#pragma unroll
          for (int k = 0; k < kWords; ++k) {
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to + ((i * 2) * kWords + k) * kThreads * 16),
                         "l"(reinterpret_cast<const uint4*>(x + i * h.xh) + k)
                         : "memory");
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to + ((i * 2 + 1) * kWords + k) * kThreads * 16),
                         "l"(reinterpret_cast<const uint4*>(dy + i * h.yh) + k)
                         : "memory");
          }
        }
      asm volatile("cp.async.commit_group;" ::: "memory");
      angles = load_angles(a, token, s, at, active);
    };
    unsigned group = blockIdx.x * kGroups + threadIdx.x / LPR;
    int slot = 0;
    fetch(group, 0);
    for (unsigned base = blockIdx.x * kGroups; base < units; base += step, group += step, slot ^= 1) {
      const Turn turn = turn_of(angles);
      const int n = next_n;
      T* out = static_cast<T*>(h.out) + next_out;
      fetch(group + step, slot ^ 1);
      asm volatile("cp.async.wait_group 1;" ::: "memory");
      const uint4* from = slots + (slot * HPG * 2 * kWords) * kThreads + threadIdx.x;
#pragma unroll
      for (int i = 0; i < HPG; ++i) {
        Pairs v = no_pairs(), g = no_pairs(), u;
        if (i < n) {
          Raw8<T> rx, ry;
#pragma unroll
          for (int k = 0; k < kWords; ++k) {
            rx.w[k] = from[((i * 2) * kWords + k) * kThreads];
            ry.w[k] = from[((i * 2 + 1) * kWords + k) * kThreads];
          }
          v = to_pairs<T>(rx);
          g = rotate(to_pairs<T>(ry), turn.cos, turn.minus, turn.sin);
        }
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          u.a[j] = g.a[j] * w.a[j];
          u.b[j] = g.b[j] * w.b[j];
        }
        const float ss = row_sum<LPR>(dot8(v, v)), dot = row_sum<LPR>(dot8(u, v));
        const float r = rsqrtf(ss * inv_dim + a.eps), f = -(r * r * dot * inv_dim) * r;
        const F2 r2 = f2(r, r), ff = f2(f, f);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          if (i < n) {
            dw.a[j] = fma2(g.a[j], v.a[j] * r2, dw.a[j]);
            dw.b[j] = fma2(g.b[j], v.b[j] * r2, dw.b[j]);
          }
          v.a[j] = fma2(u.a[j], r2, v.a[j] * ff);
          v.b[j] = fma2(u.b[j], r2, v.b[j] * ff);
        }
        if (i < n) store_pairs<T>(out + (long long)i * a.dim, v);
      }
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    if (a.partial) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const float2 p = f2_values(dw.a[j]), q = f2_values(dw.b[j]);
        float* to = &share[threadIdx.x / LPR][at + 4 * j];
        to[0] = p.x;
        to[1] = q.x;
        to[2] = p.y;
        to[3] = q.y;
      }
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

// Sum of the CTAs' shares, in a fixed order: 32 threads for each of eight columns.
template <typename TW>
__global__ void __launch_bounds__(kThreads) weight_grad_kernel(const float* partial, int ctas, int dim, TW* dwq, TW* dwk) {
  __shared__ float smem[32][9];
  const int c = threadIdx.x & 7, col = blockIdx.x * 8 + c, slice = threadIdx.x >> 3;
  float sum = 0.f;
#pragma unroll 4
  for (int i = slice; i < ctas; i += 32) sum += partial[(long long)i * 2 * dim + col];
  smem[slice][c] = sum;
  __syncthreads();
  if (slice == 0) {
#pragma unroll
    for (int i = 1; i < 32; ++i) sum += smem[i][c];
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

// A table or weight on a 16-byte boundary (head_dim is a multiple of 8, so that its rows and vectors stay on one).
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
  t.qw = table16(qw);
  t.kw = table16(kw);
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
    h.chunks = Divisor(std::max(1, (h.heads + hpg - 1) / hpg));
  }
  a.cos = t.cos.const_data_ptr<float>();
  a.sin = t.sin.const_data_ptr<float>();
  a.table = (int)cos.size(0);
  if (positions.has_value()) {
    t.pos = positions->contiguous();
    a.positions = t.pos.const_data_ptr();
    a.wide_positions = t.pos.scalar_type() == at::kLong;
  }
  a.seq = Divisor((unsigned)std::max<int64_t>(1, q.size(1)));
  a.dim = (int)q.size(3);
  a.tokens = (unsigned)(q.size(0) * q.size(1));
  a.eps = (float)eps;
  a.error = device_error_word(q.device().index());
  return a;
}

// Heads per group: four share a token's angles (two in the backward pass) once they still fill half the GPU's lanes. 40
// heads of 128 bf16, forward and backward with one head and with four (two): 8 tokens 4.2 + 9.4 and 4.2 + 10.3 us, 512
// tokens 6.2 + 12.4 and 5.3 + 12.4 us, 1024 8.3 + 16.5 and 6.2 + 14.4 us, 4096 tokens 26 + 37 and 18.5 + 31 us.
int heads_per_group(const at::Tensor& q, const at::Tensor& k) {
  const int64_t rows = q.size(0) * q.size(1) * (q.size(2) + k.size(2));
  const int64_t lanes = (int64_t)at::cuda::getCurrentDeviceProperties()->multiProcessorCount * 512;
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

template <typename K>
void launch_bwd(K kernel, const Args& a, int ctas, size_t slots, cudaStream_t stream) {
  if (slots > 48 * 1024) C10_CUDA_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)slots));
  kernel<<<ctas, kThreads, slots, stream>>>(a);
}

}  // namespace

std::tuple<at::Tensor, at::Tensor> qk_norm_rope_fwd(const at::Tensor& q, const at::Tensor& k, const at::Tensor& q_weight,
                                                    const at::Tensor& k_weight, const at::Tensor& cos,
                                                    const at::Tensor& sin, const OptTensor& positions, double eps) {
  check_heads(q, k, q_weight, k_weight, cos, sin, positions);
  const c10::cuda::CUDAGuard guard(q.device());
  auto qo = new_empty(q.sizes(), q.scalar_type(), q);
  auto ko = new_empty(k.sizes(), k.scalar_type(), k);
  if (q.numel() + k.numel() == 0) return {qo, ko};
  Kept t;
  const int hpg = heads_per_group(q, k);
  Args a = args_of(t, q, k, q_weight, k_weight, cos, sin, positions, eps, hpg);
  a.part[0].out = qo.mutable_data_ptr();
  a.part[1].out = ko.mutable_data_ptr();
  const int64_t units = (int64_t)a.tokens * (a.part[0].chunks.d + a.part[1].chunks.d);
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
  auto dq = new_empty(q.sizes(), q.scalar_type(), q);
  auto dk = new_empty(k.sizes(), k.scalar_type(), k);
  const auto wsize = weight_grads ? q.size(3) : 0;
  auto dwq = new_empty({wsize}, q_weight.scalar_type(), q), dwk = new_empty({wsize}, k_weight.scalar_type(), q);
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
  const int64_t units = (int64_t)a.tokens * std::max(a.part[0].chunks.d, a.part[1].chunks.d);
  const int groups = kThreads / lanes_per_row(q.size(3));
  const int sms = at::cuda::getCurrentDeviceProperties()->multiProcessorCount;
  const int resident = sms * (q.scalar_type() == at::kFloat ? 2 : 3);  // as the kernel's launch bounds
  const int ctas = (int)std::min<int64_t>((units + groups - 1) / groups, resident);
  at::Tensor partial;
  if (weight_grads) {
    partial = new_empty({ctas, 2, q.size(3)}, at::kFloat, q);
    a.partial = partial.mutable_data_ptr<float>();
  }
  with_types(q, q_weight, [&](auto* tt, auto* tw, auto lanes) {
    using T = std::remove_pointer_t<decltype(tt)>;
    using TW = std::remove_pointer_t<decltype(tw)>;
    constexpr int L = decltype(lanes)::value;
    const auto stream = at::cuda::getCurrentCUDAStream();
    const size_t slots = 2 * (size_t)hpg * 2 * kThreads * 8 * sizeof(T);  // up to 64 KB, for fp32
    if (hpg == 2) launch_bwd(bwd_kernel<T, TW, L, 2>, a, ctas, slots, stream);
    else launch_bwd(bwd_kernel<T, TW, L, 1>, a, ctas, slots, stream);
    C10_CUDA_KERNEL_LAUNCH_CHECK();
    if (weight_grads) {
      weight_grad_kernel<TW><<<2 * a.dim / 8, kThreads, 0, stream>>>(
          a.partial, ctas, a.dim, static_cast<TW*>(dwq.mutable_data_ptr()), static_cast<TW*>(dwk.mutable_data_ptr()));
      C10_CUDA_KERNEL_LAUNCH_CHECK();
    }
  });
  count_launches(weight_grads ? 2 : 1);
  return {dq, dk, dwq, dwk};
}

}  // namespace dmb
