// objb_linear.cuh -- the element types, activations and epilogue of the dense
// products of many tokens (linear.cu).
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>

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

// What happens to the product's element (row m of A, row n of B), whose place
// in y, z and residual is [n][m]: + bias[m] -> z -> act -> + residual -> y.
struct LinearEpilogue {
  const void* bias = nullptr;
  const void* residual = nullptr;
  void* y = nullptr;
  void* z = nullptr;
  size_t ldr = 0, ldy = 0, ldz = 0;
  int bias_dtype = 0, y_dtype = 0, act = 0;

  __device__ __forceinline__ void put(int m, size_t n, float v) const {
    if (bias) v += load_elem(bias, bias_dtype, m);
    if (z) store_elem(z, y_dtype, n * ldz + m, v);
    v = act_value(act, v);
    if (residual) v += load_elem(residual, y_dtype, n * ldr + m);
    store_elem(y, y_dtype, n * ldy + m, v);
  }
};

}  // namespace dev
}  // namespace objb
