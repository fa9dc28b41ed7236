// objb_router.cuh -- what the router-training kernels share: teams of threads
// that hold a token's experts, the scores, sequences and arguments.
#pragma once

#include <cuda_runtime.h>

#include <type_traits>

#include "objb_common.h"
#include "objb_host_launch.cuh"
#include "objb_launch.h"
#include "objb_pipe.cuh"

namespace objb {
namespace dev {

// A token belongs to a team of L threads: 8 up to 64 experts, 16 up to 128, a
// warp up to 1024, a block of 8 warps up to 8192; a thread holds EPL of its
// experts in registers.  Small teams share a warp's instructions between two
// or four tokens and reduce in fewer shuffles (32768 tokens of 64 experts, the
// first pass of the loss and the gradient: 24 and 22 us with a warp per token,
// 7 and 11 now).  With V4 (rows of whole
// 16-byte quads) a thread's experts come in quads.  Teams of a warp run in
// step: every lane takes part in every shuffle.
constexpr int kTeamWarps = 8;  // warps of a block-wide team

template <int LANES, int E_PER_LANE, bool V4>
struct Team {
  static constexpr int L = LANES, EPL = E_PER_LANE;
  static constexpr bool kBlock = L > 32, kQuads = V4;
  static __device__ __forceinline__ int rank() { return kBlock ? threadIdx.x : threadIdx.x & (L - 1); }
  static __device__ __forceinline__ int expert(int i, int r) {
    return V4 ? (i >> 2) * (4 * L) + r * 4 + (i & 3) : i * L + r;
  }
  static __device__ __forceinline__ void sync() {
    if (kBlock)
      __syncthreads();
    else
      __syncwarp();
  }
  // The lanes of this thread's team in its warp.
  static __device__ __forceinline__ unsigned lanes() {
    return L >= 32 ? 0xFFFFFFFFu : ((1u << (L & 31)) - 1u) << (threadIdx.x & 31 & ~(L - 1));
  }
  // v of every lane becomes the team's maximum / sum (fixed order).
  static __device__ __forceinline__ float max(float v, float* red) {
#pragma unroll
    for (int o = (kBlock ? 32 : L) / 2; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xFFFFFFFFu, v, o));
    if (kBlock) {
      __syncthreads();
      if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
      __syncthreads();
      v = red[0];
      for (int w = 1; w < kTeamWarps; ++w) v = fmaxf(v, red[w]);
    }
    return v;
  }
  static __device__ __forceinline__ float sum(float v, float* red) {
#pragma unroll
    for (int o = (kBlock ? 32 : L) / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
    if (kBlock) {
      __syncthreads();
      if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
      __syncthreads();
      v = red[0];
      for (int w = 1; w < kTeamWarps; ++w) v += red[w];
    }
    return v;
  }
  // Experts past E read as `fill`.
  static __device__ __forceinline__ void load(const float* row, int E, float fill, float (&l)[EPL]) {
    const int r = rank();
    if constexpr (V4) {
#pragma unroll
      for (int i = 0; i < EPL; i += 4) {
        const int e = expert(i, r);
        float4 q = make_float4(fill, fill, fill, fill);
        if (e < E) q = *reinterpret_cast<const float4*>(row + e);
        l[i] = q.x, l[i + 1] = q.y, l[i + 2] = q.z, l[i + 3] = q.w;
      }
    } else {
#pragma unroll
      for (int i = 0; i < EPL; ++i) {
        const int e = expert(i, r);
        l[i] = e < E ? row[e] : fill;
      }
    }
  }
};

enum { kSoftmax = 0, kSigmoid = 1, kSqrtSoftplus = 2 };

__device__ __forceinline__ float neg_inf() { return -__int_as_float(0x7F800000); }

// exp by the special-function unit: 2 ulp, plus |x| half steps from the product.
__device__ __forceinline__ float exp_sfu(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x * 1.4426950408889634f));
  return r;
}
__device__ __forceinline__ float rcp_sfu(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// The gate's sigmoid and sqrt-softplus scores and their derivatives.  The
// sqrt-softplus keeps the gate's branches, log1p(exp(-l)) below -20 among
// them, so the derivative is that of the score as it is computed.  Below about
// -88.7 that exponential leaves f32 and the gate's score is no number that
// shares could be made of: such a logit (-inf and the lowest f32, which masks
// are made of, among them) has score 0 and derivative 0, as under the other two.
__device__ __forceinline__ float score_of(int func, float l, float* d) {
  if (func == kSigmoid) {
    const float t = expf(-fabsf(l));  // (of few scores, or of far logits: their exponents are not rounded at |l|)
    const float r = rcp_sfu(1.0f + t);
    *d = t * r * r;
    return l >= 0.0f ? r : t * r;
  }
  if (l > 20.0f) {
    const float s = sqrtf(l);
    *d = 0.5f / s;
    return s;
  }
  // (below -20, log1p(exp(-l)) is -l to 1e-10 of it, and its sigmoid 1)
  const bool low = l < -20.0f, lost = l < -88.72283f;
  const float ex = expf(l);
  const float s = sqrtf(low ? -l : log1pf(ex));
  const float sg = low ? -0.5f : 0.5f * ex / (1.0f + ex);
  *d = lost ? 0.0f : sg / s;
  return lost ? 0.0f : s;
}

// ex = exp(l - base) of a token's logits; returns their sum.  The first try has
// base 0: its sum says whether the largest logits are within 11.5 of it (1e5,
// 1e-5), and only else (few trained routers) is there a maximum to find.  An
// exponent is rounded at |l - base|, so that with base 0 a probability is off
// by up to 5e-7 instead of 1e-7 (logits around 60: 3e-6, hence the bounds).
// *direct: base is 0 and the exponentials serve the sigmoid too.
template <class TM>
__device__ __forceinline__ float exponentials(const float (&l)[TM::EPL], float (&ex)[TM::EPL], float* red, float* base,
                                              bool* direct) {
  float sum = 0.0f;
#pragma unroll
  for (int i = 0; i < TM::EPL; ++i) {
    ex[i] = exp_sfu(l[i]);
    sum += ex[i];
  }
  sum = TM::sum(sum, red);
  *base = 0.0f;
  *direct = sum > 1e-5f && sum < 1e5f;
  if (TM::kBlock ? !*direct : !__all_sync(0xFFFFFFFFu, *direct)) {
    float m = neg_inf();
#pragma unroll
    for (int i = 0; i < TM::EPL; ++i) m = fmaxf(m, l[i]);
    m = TM::max(m, red);
    if (!*direct) *base = m > neg_inf() ? m : 0.0f;  // a row of -inf: every exponential is 0
    sum = 0.0f;
#pragma unroll
    for (int i = 0; i < TM::EPL; ++i) {
      ex[i] = exp_sfu(l[i] - *base);
      sum += ex[i];
    }
    sum = TM::sum(sum, red);
  }
  return sum;
}

// The sequence of token t: -1 before the first, S behind the last.  Offsets
// off[0..S] ascend; without a table every token is of sequence 0.
__device__ __forceinline__ int sequence_of(const int32_t* off, int S, long long t) {
  if (!off) return 0;
  int lo = -1, hi = S + 1;  // off[lo] <= t < off[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (off[mid] <= t)
      lo = mid;
    else
      hi = mid;
  }
  return lo;
}

struct BalanceArgs {
  const float* logits;
  size_t ld;
  const int32_t* ids;
  const uint8_t* mask;
  const int32_t* off;
  int S;
  long long T;
  int E, k, func;
  long long chunk;  // tokens per block
  // partial rows, one per (block, sequence it meets): index block + sequence,
  // which is its own for every pair (both only ascend along the tokens)
  float* part_p;       // [rows][E] sums of p
  int32_t* part_c;     // [rows][E] selections
  double* part_z;      // [rows] sums of lse^2
  int32_t* part_n;     // [rows] counted tokens
  unsigned* ticket;
};

// Who folds the partial rows: a grid launched behind them; the one block that
// made them all; the kFinishCluster blocks of one cluster that did.
enum { kFinishGrid = 0, kFinishAlone = 1, kFinishInCluster = 2 };
constexpr int kFinishCluster = 8;

struct BalanceFinishArgs {
  BalanceArgs a;
  int groups;          // 32-expert groups
  int mode;            // kFinishGrid: a launch of its own; else by the blocks of the partial pass
  double* bal_part;    // [S][groups] sum_e c P
  double* seq_z;       // [S]
  int32_t* counts;     // [S][E]
  int32_t* tokens;     // [S]
  float* losses;       // balance, z
  float* scales;       // [S + 1]: E / (k n_q^2 S'), then 2 / N
};

struct RouterBackwardArgs {
  const float* logits;
  size_t ld;
  const int32_t* ids;
  const float* dw;        // may be null
  const uint8_t* mask;
  const int32_t* off;
  int S;
  const int32_t* counts;  // null: no losses
  const float* scales;
  long long T;
  int E, k, func, renorm;
  float route_scale, balance_grad, z_grad;
  float* out;
  size_t ld_out;
  int per_team;           // consecutive tokens of a team
};

}  // namespace dev

// f(Team) for E experts; v4: rows of whole aligned quads.  WIDE: the lanes of 129
// to 256 experts (16, or 32 where registers run short).
template <int WIDE, class F>
int with_team(size_t E, bool v4, F&& f) {
  if (E <= 8) return f(dev::Team<8, 1, false>{});
  if (E <= 16) return f(dev::Team<8, 2, false>{});
  if (E <= 32) return f(dev::Team<8, 4, false>{});
  if (E <= 64) return v4 ? f(dev::Team<8, 8, true>{}) : f(dev::Team<8, 8, false>{});
  if (E <= 128) return v4 ? f(dev::Team<16, 8, true>{}) : f(dev::Team<16, 8, false>{});
  if (E <= 256) return v4 ? f(dev::Team<WIDE, 256 / WIDE, true>{}) : f(dev::Team<WIDE, 256 / WIDE, false>{});
  if (E <= 512) return v4 ? f(dev::Team<32, 16, true>{}) : f(dev::Team<32, 16, false>{});
  if (E <= 1024) return f(dev::Team<32, 32, false>{});
  return f(dev::Team<32 * dev::kTeamWarps, 32, false>{});
}

template <class F>
int with_func(int func, F&& f) {
  using std::integral_constant;
  if (func == dev::kSoftmax) return f(integral_constant<int, dev::kSoftmax>{});
  if (func == dev::kSigmoid) return f(integral_constant<int, dev::kSigmoid>{});
  return f(integral_constant<int, dev::kSqrtSoftplus>{});
}

// router_partial.cu, router_backward.cu
int launch_balance_partial(const dev::BalanceFinishArgs& f, int grid, bool v4, cudaStream_t st);
int launch_router_backward(dev::RouterBackwardArgs a, bool v4, const DeviceProps& props, cudaStream_t st);

}  // namespace objb
