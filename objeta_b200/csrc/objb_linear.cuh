// objb_linear.cuh -- the element types, activations and epilogue of the dense
// products of many tokens (linear.cu).
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>
#include <type_traits>

#include "../../include/objeta_b200.h"

namespace objb {
namespace dev {

__device__ __forceinline__ float load_elem(const void* p, int dtype, size_t i) {
  if (dtype == OBJB_DTYPE_F32) return static_cast<const float*>(p)[i];
  if (dtype == OBJB_DTYPE_BF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
  return __half2float(static_cast<const __half*>(p)[i]);
}
__device__ __forceinline__ void store_elem(void* p, int dtype, size_t i, float v) {
  if (dtype == OBJB_DTYPE_F32)
    static_cast<float*>(p)[i] = v;
  else if (dtype == OBJB_DTYPE_BF16)
    static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
  else
    static_cast<__half*>(p)[i] = __float2half_rn(v);
}

constexpr float kSqrt2OverPi = 0.79788456080286536f;
constexpr float kSqrtHalf = 0.70710678118654752f;
constexpr float kInvSqrt2Pi = 0.39894228040143268f;

// 1 / (1 + exp(-v)) without overflow on either side.
__device__ __forceinline__ float sigmoid(float v) {
  const float t = expf(-fabsf(v));
  const float r = 1.0f / (1.0f + t);
  return v >= 0.0f ? r : t * r;
}

__device__ __forceinline__ float act_value(int act, float v) {
  switch (act) {
    case OBJB_ACT_RELU: return v > 0.0f ? v : (v == v ? 0.0f : v);
    case OBJB_ACT_SILU: return v * sigmoid(v);
    case OBJB_ACT_GELU: return 0.5f * v * erfcf(-v * kSqrtHalf);  // exact tails
    case OBJB_ACT_GELU_TANH: return v * sigmoid(2.0f * kSqrt2OverPi * (v + 0.044715f * v * v * v));
    default: return v;
  }
}

// d act / d v.  gelu_tanh through tanh(u) = 2 sigmoid(2 u) - 1.
__device__ __forceinline__ float act_grad(int act, float v) {
  switch (act) {
    case OBJB_ACT_RELU: return v > 0.0f ? 1.0f : 0.0f;
    case OBJB_ACT_SILU: {
      const float s = sigmoid(v);
      return s * (1.0f + v * (1.0f - s));
    }
    case OBJB_ACT_GELU: return 0.5f * erfcf(-v * kSqrtHalf) + v * kInvSqrt2Pi * expf(-0.5f * v * v);
    case OBJB_ACT_GELU_TANH: {
      const float s = sigmoid(2.0f * kSqrt2OverPi * (v + 0.044715f * v * v * v));
      return s + 2.0f * v * s * (1.0f - s) * kSqrt2OverPi * (1.0f + 3.0f * 0.044715f * v * v);
    }
    default: return 1.0f;
  }
}

// The three bf16 parts of an f32: 8 bits of the significand each, cut off (not
// rounded), so that they sum to it exactly and none overflows.  A non-finite
// value is its first part alone.
__device__ __forceinline__ void split3(float v, __nv_bfloat16 (&p)[3]) {
  const float a = __uint_as_float(__float_as_uint(v) & 0xFFFF0000u);
  const bool finite = fabsf(v) < __int_as_float(0x7F800000);
  const float r = finite ? v - a : 0.0f;
  const float b = __uint_as_float(__float_as_uint(r) & 0xFFFF0000u);
  p[0] = __float2bfloat16_rn(finite ? a : v);
  p[1] = __float2bfloat16_rn(b);
  p[2] = __float2bfloat16_rn(r - b);
}

// What happens to the product's element (row m of A, row n of B), whose place
// in y, z and residual is [n][m]: + bias[m] -> z -> act -> + residual -> y.
struct LinearEpilogue {
  const void* bias = nullptr;
  const void* residual = nullptr;
  void* y = nullptr;
  void* z = nullptr;
  size_t ldr = 0, ldy = 0, ldz = 0;
  size_t plane = 0;  // put_planes: elements between y's planes
  int bias_dtype = 0, y_dtype = 0, act = 0;

  template <class T, int C>
  __device__ __forceinline__ void store(T* p, size_t ld, int m, long long n, long long N, const float (&v)[C]) const {
    p += static_cast<size_t>(n) * ld + m;
#pragma unroll
    for (int i = 0; i < C; ++i)
      if (n + i < N) {
        if constexpr (sizeof(T) == 4)
          p[i * ld] = v[i];
        else if constexpr (std::is_same<T, __half>::value)
          p[i * ld] = __float2half_rn(v[i]);
        else
          p[i * ld] = __float2bfloat16_rn(v[i]);
      }
  }
  template <class T, int C>
  __device__ __forceinline__ void add(const T* p, size_t ld, int m, long long n, long long N, float (&v)[C]) const {
    p += static_cast<size_t>(n) * ld + m;
    T r[C];
#pragma unroll
    for (int i = 0; i < C; ++i)
      if (n + i < N) r[i] = p[i * ld];
#pragma unroll
    for (int i = 0; i < C; ++i)
      if (n + i < N) v[i] += static_cast<float>(r[i]);
  }
  template <int C>
  __device__ __forceinline__ void store_any(void* p, size_t ld, int m, long long n, long long N,
                                            const float (&v)[C]) const {
    if (y_dtype == OBJB_DTYPE_F32)
      store(static_cast<float*>(p), ld, m, n, N, v);
    else if (y_dtype == OBJB_DTYPE_BF16)
      store(static_cast<__nv_bfloat16*>(p), ld, m, n, N, v);
    else
      store(static_cast<__half*>(p), ld, m, n, N, v);
  }

  // C neighbouring n of one m (those below N).
  template <int C>
  __device__ __forceinline__ void put_columns(int m, long long n, long long N, float (&v)[C]) const {
    if (n >= N) return;
    if (bias) {
      const float b = load_elem(bias, bias_dtype, m);
#pragma unroll
      for (int i = 0; i < C; ++i) v[i] += b;
    }
    if (z) store_any(z, ldz, m, n, N, v);
    switch (act) {
#define OBJB_ACT_CASE(A)                                          \
  case A:                                                         \
    _Pragma("unroll") for (int i = 0; i < C; ++i) v[i] = act_value(A, v[i]); \
    break
      OBJB_ACT_CASE(OBJB_ACT_RELU);
      OBJB_ACT_CASE(OBJB_ACT_SILU);
      OBJB_ACT_CASE(OBJB_ACT_GELU);
      OBJB_ACT_CASE(OBJB_ACT_GELU_TANH);
#undef OBJB_ACT_CASE
      default: break;
    }
    if (residual) {
      if (y_dtype == OBJB_DTYPE_F32)
        add(static_cast<const float*>(residual), ldr, m, n, N, v);
      else if (y_dtype == OBJB_DTYPE_BF16)
        add(static_cast<const __nv_bfloat16*>(residual), ldr, m, n, N, v);
      else
        add(static_cast<const __half*>(residual), ldr, m, n, N, v);
    }
    store_any(y, ldy, m, n, N, v);
  }

  // One f32 value as the three planes of the next product's operand.
  __device__ __forceinline__ void put_planes(int m, long long n, float v) const {
    __nv_bfloat16 p[3];
    split3(v, p);
    __nv_bfloat16* o = static_cast<__nv_bfloat16*>(y) + static_cast<size_t>(n) * ldy + m;
    o[0] = p[0];
    o[plane] = p[1];
    o[2 * plane] = p[2];
  }
};

}  // namespace dev
}  // namespace objb
