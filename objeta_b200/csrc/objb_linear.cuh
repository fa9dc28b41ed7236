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

// exp2 and 1 / v by the special-function unit (2 ulp and 1 ulp).
__device__ __forceinline__ float ex2_sfu(float v) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
__device__ __forceinline__ float rcp_sfu(float v) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
// 1 / (1 + exp(-v)): five instructions, since a tile's epilogue is not hidden
// behind its MMAs (the IEEE division alone takes twenty).  Overflow of the
// exponential gives the right 0.
__device__ __forceinline__ float sigmoid(float v) { return rcp_sfu(1.0f + ex2_sfu(v * -1.4426950408889634f)); }

__device__ __forceinline__ float act_value(int act, float v) {
  switch (act) {
    case OBJB_ACT_RELU: return v > 0.0f ? v : (v == v ? 0.0f : v);
    case OBJB_ACT_SILU: return v * sigmoid(v);
    case OBJB_ACT_GELU: return 0.5f * v * erfcf(-v * kSqrtHalf);  // exact tails
    case OBJB_ACT_GELU_TANH: return v * sigmoid(v * fmaf(v * v, 2.0f * kSqrt2OverPi * 0.044715f, 2.0f * kSqrt2OverPi));
    default: return v;
  }
}

// d act / d v.  gelu_tanh through tanh(u) = 2 sigmoid(2 u) - 1.  Past 128 (in
// f32 already before) every one is its limit; a larger v, whose powers
// overflow, would make 0 * inf of it.
__device__ __forceinline__ float act_grad(int act, float v) {
  v = fabsf(v) > 128.0f ? copysignf(128.0f, v) : v;  // (NaN stays)
  switch (act) {
    case OBJB_ACT_RELU: return v > 0.0f ? 1.0f : 0.0f;
    case OBJB_ACT_SILU: {
      const float s = sigmoid(v);
      return s * fmaf(v, 1.0f - s, 1.0f);
    }
    case OBJB_ACT_GELU:
      return 0.5f * erfcf(-v * kSqrtHalf) + v * kInvSqrt2Pi * ex2_sfu(v * v * (-0.5f * 1.4426950408889634f));
    case OBJB_ACT_GELU_TANH: {
      const float q = v * v;
      const float s = sigmoid(v * fmaf(q, 2.0f * kSqrt2OverPi * 0.044715f, 2.0f * kSqrt2OverPi));
      const float d = v * (1.0f - s) * fmaf(q, 6.0f * kSqrt2OverPi * 0.044715f, 2.0f * kSqrt2OverPi);
      return fmaf(s, d, s);
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

// The same of two neighbours, part j of both in u[j] (v0 in its lower half).  By
// byte permutations: the conversion to bf16 takes four times an add's slots.
__device__ __forceinline__ void split3_pair(float v0, float v1, uint32_t (&u)[3]) {
  auto rest = [](float v) {  // v without its upper half; 0 for a non-finite v
    const float r = v - __uint_as_float(__float_as_uint(v) & 0xFFFF0000u);
    return r == r ? r : 0.0f;
  };
  auto upper = [](float a, float b) { return __byte_perm(__float_as_uint(a), __float_as_uint(b), 0x7632); };
  u[0] = upper(v0 == v0 ? v0 : __int_as_float(0x7FFFFFFF), v1 == v1 ? v1 : __int_as_float(0x7FFFFFFF));
  v0 = rest(v0), v1 = rest(v1);
  u[1] = upper(v0, v1);
  v0 -= __uint_as_float(__float_as_uint(v0) & 0xFFFF0000u);
  v1 -= __uint_as_float(__float_as_uint(v1) & 0xFFFF0000u);
  u[2] = upper(v0, v1);
}

// What happens to the product's element (row m of A, row n of B), whose place
// in y, z and residual is [n][m]: + bias[m] -> z -> act -> + residual -> y.
struct LinearEpilogue {
  const void* bias = nullptr;
  const void* residual = nullptr;
  void* y = nullptr;
  void* z = nullptr;
  uint32_t ldr = 0, ldy = 0, ldz = 0;
  size_t plane = 0;  // put_planes: elements between y's planes
  int bias_dtype = 0, y_dtype = 0, act = 0;

  __device__ __forceinline__ float bias_of(int m) const { return bias ? load_elem(bias, bias_dtype, m) : 0.0f; }

  // FULL: all C columns exist.
  template <class T, int C, bool FULL>
  __device__ __forceinline__ static void store(T* p, uint32_t ld, int m, long long n, int left, const float (&v)[C],
                                               uint32_t lane = 0) {
    char* at = reinterpret_cast<char*>(p + n * ld + m);
    const uint32_t off = lane * static_cast<uint32_t>(sizeof(T));
    const uint32_t pitch = ld * static_cast<uint32_t>(sizeof(T));
#pragma unroll
    for (int i = 0; i < C; ++i)
      if (FULL || i < left) {
        T* q = reinterpret_cast<T*>(at + static_cast<uint64_t>(pitch) * i + off);
        if constexpr (sizeof(T) == 4)
          *q = v[i];
        else if constexpr (std::is_same<T, __half>::value)
          *q = __float2half_rn(v[i]);
        else
          *q = __float2bfloat16_rn(v[i]);
      }
  }
  template <class T, int C, bool FULL>
  __device__ __forceinline__ static void add(const T* p, uint32_t ld, int m, long long n, int left, float (&v)[C],
                                             uint32_t lane = 0) {
    const char* at = reinterpret_cast<const char*>(p + n * ld + m + lane);
    const uint32_t pitch = ld * static_cast<uint32_t>(sizeof(T));
    T r[C];
#pragma unroll
    for (int i = 0; i < C; ++i)
      if (FULL || i < left) r[i] = *reinterpret_cast<const T*>(at + static_cast<uint64_t>(pitch) * i);
#pragma unroll
    for (int i = 0; i < C; ++i)
      if (FULL || i < left) v[i] += static_cast<float>(r[i]);
  }
  template <class T, int C, bool FULL>
  __device__ __forceinline__ void put_typed(int m, long long n, int left, float (&v)[C], uint32_t lane) const {
    if (z) store<T, C, FULL>(static_cast<T*>(z), ldz, m, n, left, v, lane);
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
    if (residual) add<T, C, FULL>(static_cast<const T*>(residual), ldr, m, n, left, v, lane);
    store<T, C, FULL>(static_cast<T*>(y), ldy, m, n, left, v, lane);
  }
  template <class T, int C>
  __device__ __forceinline__ void put_left(int m, long long n, int left, float (&v)[C], uint32_t lane) const {
    if (left >= C)
      put_typed<T, C, true>(m, n, left, v, lane);
    else
      put_typed<T, C, false>(m, n, left, v, lane);
  }

  // C neighbouring n of one m, those below n_end; b = bias_of(m).  Where a warp
  // has 32 neighbouring m, m is the first of them and `lane` the rest: the
  // addresses but for the lane are the warp's.
  template <int C>
  __device__ __forceinline__ void put_columns(int m, long long n, long long n_end, float b, float (&v)[C],
                                              uint32_t lane = 0) const {
    if (n >= n_end) return;
    const int left = n_end - n < C ? static_cast<int>(n_end - n) : C;
#pragma unroll
    for (int i = 0; i < C; ++i) v[i] += b;
    if (y_dtype == OBJB_DTYPE_F32)
      put_left<float>(m, n, left, v, lane);
    else if (y_dtype == OBJB_DTYPE_BF16)
      put_left<__nv_bfloat16>(m, n, left, v, lane);
    else
      put_left<__half>(m, n, left, v, lane);
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
