// 8-element vector access for the kernels that take fp32, bf16 and fp16 alike.
#pragma once

#include <ATen/core/Tensor.h>
#include <cuda_fp16.h>

#include "common.cuh"

namespace dmb {

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }

template <typename T>
__device__ __forceinline__ T from_float(float v);
template <>
__device__ __forceinline__ float from_float<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }

// Eight values as they lie in memory: one 16-byte word of a 16-bit type, two of fp32.
template <typename T>
struct Raw8 {
  uint4 w[sizeof(T) / 2];
};

template <typename T>
__device__ __forceinline__ Raw8<T> load_raw8(const T* p) {  // p is 16-byte aligned
  Raw8<T> r;
#pragma unroll
  for (int i = 0; i < (int)sizeof(T) / 2; ++i) r.w[i] = __ldg(reinterpret_cast<const uint4*>(p) + i);
  return r;
}

template <typename T>
__device__ __forceinline__ void unpack8(const Raw8<T>& r, float (&v)[8]) {
  if constexpr (sizeof(T) == 4) {
    const uint32_t w[8] = {r.w[0].x, r.w[0].y, r.w[0].z, r.w[0].w, r.w[1].x, r.w[1].y, r.w[1].z, r.w[1].w};
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = __uint_as_float(w[k]);
  } else {
    const uint32_t w[4] = {r.w[0].x, r.w[0].y, r.w[0].z, r.w[0].w};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if constexpr (std::is_same<T, __nv_bfloat16>::value) {
        v[2 * k] = __uint_as_float(w[k] << 16);
        v[2 * k + 1] = __uint_as_float(w[k] & 0xFFFF0000u);
      } else {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[k]));
        v[2 * k] = f.x;
        v[2 * k + 1] = f.y;
      }
    }
  }
}

template <typename T>
__device__ __forceinline__ void load8t(const T* p, float (&v)[8]) {
  unpack8<T>(load_raw8<T>(p), v);
}

template <typename T>
__device__ __forceinline__ Raw8<T> pack8(const float (&v)[8]) {
  Raw8<T> r;
  if constexpr (sizeof(T) == 4) {
    r.w[0] = make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
    r.w[1] = make_uint4(__float_as_uint(v[4]), __float_as_uint(v[5]), __float_as_uint(v[6]), __float_as_uint(v[7]));
  } else {
    uint32_t w[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if constexpr (std::is_same<T, __nv_bfloat16>::value) {
        w[k] = pack_bf16x2(v[2 * k], v[2 * k + 1]);
      } else {
        const __half2 h = __floats2half2_rn(v[2 * k], v[2 * k + 1]);
        w[k] = *reinterpret_cast<const uint32_t*>(&h);
      }
    }
    r.w[0] = make_uint4(w[0], w[1], w[2], w[3]);
  }
  return r;
}

template <typename T>
__device__ __forceinline__ void store8t(T* p, const float (&v)[8]) {  // p is 16-byte aligned
  const Raw8<T> r = pack8<T>(v);
#pragma unroll
  for (int i = 0; i < (int)sizeof(T) / 2; ++i) reinterpret_cast<uint4*>(p)[i] = r.w[i];
}

// Two fp32 values in a 64-bit register: Blackwell's packed arithmetic does both in one instruction.
struct F2 {
  unsigned long long v;
};

__device__ __forceinline__ F2 f2(float lo, float hi) {
  F2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ float2 f2_values(F2 a) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(a.v));
  return r;
}
__device__ __forceinline__ F2 operator*(F2 a, F2 b) {
  F2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ F2 operator+(F2 a, F2 b) {
  F2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
  F2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}

// Eight values as four pairs of neighbours.
template <typename T>
__device__ __forceinline__ void unpack_f2(const Raw8<T>& r, F2 (&v)[4]) {
  float f[8];
  unpack8<T>(r, f);
#pragma unroll
  for (int k = 0; k < 4; ++k) v[k] = f2(f[2 * k], f[2 * k + 1]);
}

// Eight values plus c, as four pairs of neighbours. 16-bit ones are added as they lie in their words, without unpacking.
template <typename T>
__device__ __forceinline__ void add_f2(const Raw8<T>& r, float c, F2 (&v)[4]) {
  if constexpr (sizeof(T) == 4) {
    unpack_f2<T>(r, v);
    const F2 cc = f2(c, c);
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] = v[k] + cc;
  } else {
    const uint32_t w[4] = {r.w[0].x, r.w[0].y, r.w[0].z, r.w[0].w};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      float lo, hi;
      if constexpr (std::is_same<T, __nv_bfloat16>::value) {
        asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tadd.rn.f32.bf16 %0, a, %3;\n\tadd.rn.f32.bf16 %1, b, %3;\n\t}"
            : "=f"(lo), "=f"(hi)
            : "r"(w[k]), "f"(c));
      } else {
        asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tadd.rn.f32.f16 %0, a, %3;\n\tadd.rn.f32.f16 %1, b, %3;\n\t}"
            : "=f"(lo), "=f"(hi)
            : "r"(w[k]), "f"(c));
      }
      v[k] = f2(lo, hi);
    }
  }
}

template <typename T>
__device__ __forceinline__ Raw8<T> pack_f2(const F2 (&v)[4]) {
  float f[8];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const float2 x = f2_values(v[k]);
    f[2 * k] = x.x;
    f[2 * k + 1] = x.y;
  }
  return pack8<T>(f);
}

// Calls f with a null pointer of the element type of a tensor (fp32, bf16 or fp16).
template <typename F>
void with_element(at::ScalarType t, F&& f) {
  switch (t) {
    case at::kFloat:
      return f(static_cast<float*>(nullptr));
    case at::kBFloat16:
      return f(static_cast<__nv_bfloat16*>(nullptr));
    case at::kHalf:
      return f(static_cast<__half*>(nullptr));
    default:
      TORCH_CHECK_VALUE(false, "float32, bfloat16 or float16 expected, got ", t);
  }
}

}  // namespace dmb
