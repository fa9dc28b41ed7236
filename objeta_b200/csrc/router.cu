// router.cu -- what training a router on frozen experts takes: per-expert
// counts with the balance and z losses of packed sequences, the gradient of
// the router's logits (through the routing weights and both losses in one
// pass) and the gradient of the routing weights of the top-k combine.  No
// counterpart in the reference, which only routes; the scores are those of
// its router and gate (crates/objeta-cuda/src/bin/deepseek_single_layer_moe.rs:
// 720-740, 768-881).
//
// With s_i = score(l_i), p = s / sum s, lse = log sum exp l, per sequence q of
// n_q counted tokens (S' sequences have any, N tokens in all):
//   balance = 1/S' sum_q sum_e (E c[q,e] / (k n_q)) (1/n_q sum_t p[t,e])
//   z       = 1/N sum_t lse_t^2
//   dl      = ds/dl ( dL/ds of the routing weights
//                     + (B - sum_m B_m p_m) / sum s ),  B_e = E c[q,e] / (k n_q^2 S')
//             + 2/N lse softmax(l)
// where c counts the selections (token, slot), which carry no gradient.
#include <cuda_runtime.h>

#include <algorithm>
#include <string>

#include "objb_common.h"
#include "objb_host_launch.cuh"
#include "objb_launch.h"
#include "objb_pipe.cuh"

namespace objb {
namespace dev {

// A token belongs to a team: one warp up to 1024 experts, a block of 8 warps
// up to 8192.  Each thread holds EPL experts of the token in registers.  With
// V4 (EPL >= 4, rows of whole 16-byte quads) a thread's experts come in quads.
constexpr int kTeamWarps = 8;  // warps of a block-wide team

template <int EPL, int WPT, bool V4>
struct Team {
  static constexpr int kThreads = 32 * WPT;
  static __device__ __forceinline__ int rank() { return WPT == 1 ? (threadIdx.x & 31) : threadIdx.x; }
  static __device__ __forceinline__ int expert(int i, int r) {
    return V4 ? (i >> 2) * (4 * kThreads) + r * 4 + (i & 3) : i * kThreads + r;
  }
  static __device__ __forceinline__ void sync() {
    if (WPT == 1)
      __syncwarp();
    else
      __syncthreads();
  }
  // v of every lane becomes the team's maximum / sum (fixed order).
  static __device__ __forceinline__ float max(float v, float* red) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xFFFFFFFFu, v, o));
    if (WPT > 1) {
      __syncthreads();
      if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
      __syncthreads();
      v = red[0];
      for (int w = 1; w < WPT; ++w) v = fmaxf(v, red[w]);
    }
    return v;
  }
  static __device__ __forceinline__ float sum(float v, float* red) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
    if (WPT > 1) {
      __syncthreads();
      if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
      __syncthreads();
      v = red[0];
      for (int w = 1; w < WPT; ++w) v += red[w];
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
// them, so the derivative is that of the score as it is computed.
__device__ __forceinline__ float score_of(int func, float l, float* d) {
  if (func == kSigmoid) {
    const float t = exp_sfu(-fabsf(l));
    const float r = rcp_sfu(1.0f + t);
    *d = t * r * r;
    return l >= 0.0f ? r : t * r;
  }
  if (l > 20.0f) {
    const float s = sqrtf(l);
    *d = 0.5f / s;
    return s;
  }
  const bool low = l < -20.0f;
  const float ex = expf(low ? -l : l);
  const float s = sqrtf(log1pf(ex));
  const float sg = low ? 1.0f / (1.0f + expf(l)) : ex / (1.0f + ex);
  *d = (low ? -0.5f : 0.5f) * sg / s;
  return s;
}

// A token's logits l become exp(l - base); returns their sum.  Where none is
// above 64 and one above -64 (every trained router), base is 0: no maximum has
// to be found first, and the exponentials serve the sigmoid too (*direct).
template <class TM, int EPL>
__device__ __forceinline__ float exponentials(float (&l)[EPL], float* red, float* base, bool* direct) {
  *base = 0.0f;
  *direct = false;
  if (TM::kThreads == 32) {
    float m = l[0];
#pragma unroll
    for (int i = 1; i < EPL; ++i) m = fmaxf(m, l[i]);
    *direct = !__any_sync(0xFFFFFFFFu, m > 64.0f) && __any_sync(0xFFFFFFFFu, m > -64.0f);
  }
  if (!*direct) {
    float m = neg_inf();
#pragma unroll
    for (int i = 0; i < EPL; ++i) m = fmaxf(m, l[i]);
    m = TM::max(m, red);
    *base = m > neg_inf() ? m : 0.0f;  // a row of -inf: every exponential is 0
  }
  float sum = 0.0f;
#pragma unroll
  for (int i = 0; i < EPL; ++i) {
    l[i] = exp_sfu(l[i] - *base);
    sum += l[i];
  }
  return TM::sum(sum, red);
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

struct BalanceFinishArgs {
  BalanceArgs a;
  int groups;          // 32-expert groups
  bool alone;          // one block does the partial pass and this one
  double* bal_part;    // [S][groups] sum_e c P
  double* seq_z;       // [S]
  int32_t* counts;     // [S][E]
  int32_t* tokens;     // [S]
  float* losses;       // balance, z
  float* scales;       // [S + 1]: E / (k n_q^2 S'), then 2 / N
};

// Sums of up to four values per thread over the block, in a fixed order.
template <int N>
__device__ __forceinline__ void block_sums(double (&v)[N], double (*red)[32]) {
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, warps = blockDim.x >> 5;
#pragma unroll
  for (int i = 0; i < N; ++i)
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v[i] += __shfl_xor_sync(0xFFFFFFFFu, v[i], o);
  __syncthreads();
#pragma unroll
  for (int i = 0; i < N; ++i)
    if (lane == 0) red[i][w] = v[i];
  __syncthreads();
#pragma unroll
  for (int i = 0; i < N; ++i) {
    v[i] = 0.0;
    for (int j = 0; j < warps; ++j) v[i] += red[i][j];
  }
}

struct FinishSmem {
  double p[16][32];
  int c[16][32];
  double red[4][32];
  bool last;
};

// One (sequence, 32 experts) item per block and turn: the partial rows of the
// sequence are summed in block order (interleaved over the warps, the runs
// folded in order), in double.  The block that finishes last (`alone`: the
// only one) folds the sequences' sums into the losses.
__device__ __forceinline__ void balance_finish(const BalanceFinishArgs& f, FinishSmem& sm, bool alone) {
  const BalanceArgs& a = f.a;
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, warps = blockDim.x >> 5;
  for (int item = alone ? 0 : blockIdx.x; item < a.S * f.groups; item += alone ? 1 : gridDim.x) {
    const int q = item / f.groups, g = item - q * f.groups;
    const int e = g * 32 + lane;
    long long b = a.off ? a.off[q] : 0, end = a.off ? a.off[q + 1] : a.T;
    b = b > 0 ? b : 0;
    end = end < a.T ? end : a.T;
    const int c0 = static_cast<int>(b / a.chunk), c1 = end > b ? static_cast<int>((end - 1) / a.chunk) : c0 - 1;
    double p = 0.0;
    int c = 0;
    if (e < a.E) {
      const float* pp = a.part_p + (static_cast<size_t>(c0) + q) * a.E + e;
      const int32_t* pc = a.part_c + (static_cast<size_t>(c0) + q) * a.E + e;
#pragma unroll 8
      for (int i = w; i <= c1 - c0; i += warps) {
        p += pp[static_cast<size_t>(i) * a.E];
        c += pc[static_cast<size_t>(i) * a.E];
      }
    }
    sm.p[w][lane] = p;
    sm.c[w][lane] = c;
    if (g == 0) {
      double zn[2] = {};
      for (int i = c0 + threadIdx.x; i <= c1; i += blockDim.x) {
        zn[0] += a.part_z[static_cast<size_t>(i) + q];
        zn[1] += a.part_n[static_cast<size_t>(i) + q];
      }
      block_sums(zn, sm.red);
      if (threadIdx.x == 0) {
        f.seq_z[q] = zn[0];
        f.tokens[q] = static_cast<int32_t>(zn[1]);
      }
    }
    __syncthreads();
    if (w == 0) {
      for (int i = 1; i < warps; ++i) p += sm.p[i][lane], c += sm.c[i][lane];
      if (e < a.E) f.counts[static_cast<size_t>(q) * a.E + e] = c;
      double v = p * c;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
      if (lane == 0) f.bal_part[item] = v;
    }
    __syncthreads();
  }
  if (!alone) {
    if (threadIdx.x == 0) {
      __threadfence();
      sm.last = atomicAdd(a.ticket, 1u) == gridDim.x - 1;
      __threadfence();
    }
    __syncthreads();
    if (!sm.last) return;
  }
  double t[4] = {};  // S', N, sum of z, sum of the sequences' balances
  for (int i = threadIdx.x; i < a.S; i += blockDim.x) {
    const int n = __ldcg(f.tokens + i);
    if (n == 0) continue;
    t[0] += 1.0;
    t[1] += n;
    t[2] += __ldcg(f.seq_z + i);
    double v = 0.0;
    for (int j = 0; j < f.groups; ++j) v += __ldcg(f.bal_part + static_cast<size_t>(i) * f.groups + j);
    t[3] += v * a.E / (static_cast<double>(a.k) * n * n);
  }
  block_sums(t, sm.red);
  for (int i = threadIdx.x; i < a.S; i += blockDim.x) {
    const double n = __ldcg(f.tokens + i);
    f.scales[i] = n > 0.0 ? static_cast<float>(a.E / (a.k * n * n * t[0])) : 0.0f;
  }
  if (threadIdx.x == 0) {
    f.losses[0] = t[0] > 0.0 ? static_cast<float>(t[3] / t[0]) : 0.0f;
    f.losses[1] = t[1] > 0.0 ? static_cast<float>(t[2] / t[1]) : 0.0f;
    f.scales[a.S] = t[1] > 0.0 ? static_cast<float>(2.0 / t[1]) : 0.0f;
  }
}

__global__ void __launch_bounds__(256) balance_finish_kernel(const BalanceFinishArgs f) {
  __shared__ FinishSmem sm;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  balance_finish(f, sm, false);
}

template <int EPL, int WPT, bool V4, int THREADS>
__global__ void __launch_bounds__(THREADS, EPL <= 8 ? 3 : 1) balance_partial_kernel(const BalanceFinishArgs f) {
  using TM = Team<EPL, WPT, V4>;
  constexpr int kTeams = THREADS / TM::kThreads;
  extern __shared__ __align__(16) uint8_t router_smem[];
  const BalanceArgs& a = f.a;
  int32_t* hist = reinterpret_cast<int32_t*>(router_smem);             // [E]
  float* acc_sm = reinterpret_cast<float*>(hist + (a.E + 3) / 4 * 4);  // [kTeams][E], warp teams
  __shared__ float red[kTeamWarps];
  __shared__ double z_sm[kTeams];
  __shared__ int n_sm[kTeams];
  __shared__ FinishSmem fin;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (blockIdx.x == 0 && threadIdx.x == 0) *a.ticket = 0;
  const int E = a.E, r = TM::rank();
  const int team = WPT == 1 ? threadIdx.x >> 5 : 0;
  const long long t0 = blockIdx.x * a.chunk;
  const long long t1 = t0 + a.chunk < a.T ? t0 + a.chunk : a.T;
  long long pos = t0;
  while (pos < t1) {
    const int q = sequence_of(a.off, a.S, pos);
    if (q >= a.S) break;
    if (q < 0) {
      pos = a.off[0];
      continue;
    }
    long long end = a.off ? a.off[q + 1] : t1;
    end = end < t1 ? end : t1;
    for (int e = threadIdx.x; e < E; e += THREADS) hist[e] = 0;
    __syncthreads();
    float acc[EPL];
#pragma unroll
    for (int i = 0; i < EPL; ++i) acc[i] = 0.0f;
    double z = 0.0;
    int n = 0;
    float nxt[EPL];
    int id_nxt = -1;  // slot r of the team's next token
    bool in_nxt = false;
    auto fetch = [&](long long t) {
      if (t >= end) return;
      TM::load(a.logits + t * a.ld, E, neg_inf(), nxt);
      id_nxt = r < a.k ? a.ids[t * a.k + r] : -1;
      in_nxt = !a.mask || a.mask[t];
    };
    fetch(pos + team);
    for (long long t = pos + team; t < end; t += kTeams) {
      float l[EPL];
#pragma unroll
      for (int i = 0; i < EPL; ++i) l[i] = nxt[i];
      const int id = id_nxt;
      const bool in = in_nxt;
      fetch(t + kTeams);
      if (!in) continue;
      ++n;
      if (id >= 0 && id < E) atomicAdd(&hist[id], 1);
      for (int j = r + TM::kThreads; j < a.k; j += TM::kThreads) {
        const int e = a.ids[t * a.k + j];
        if (e >= 0 && e < E) atomicAdd(&hist[e], 1);
      }
      float base, s[EPL];
      bool direct;
      if (a.func != kSoftmax) {
#pragma unroll
        for (int i = 0; i < EPL; ++i) s[i] = l[i];
      }
      const float sum = exponentials<TM, EPL>(l, red, &base, &direct);
      float ssum = sum;
      if (a.func != kSoftmax) {
        ssum = 0.0f;
        if (a.func == kSigmoid && direct) {
#pragma unroll
          for (int i = 0; i < EPL; ++i) {
            s[i] = l[i] * rcp_sfu(1.0f + l[i]);
            ssum += s[i];
          }
        } else {
#pragma unroll
          for (int i = 0; i < EPL; ++i) {
            float d;
            s[i] = TM::expert(i, r) < E ? score_of(a.func, s[i], &d) : 0.0f;
            ssum += s[i];
          }
        }
        ssum = TM::sum(ssum, red);
      } else {
#pragma unroll
        for (int i = 0; i < EPL; ++i) s[i] = l[i];
      }
      const float inv = ssum == 0.0f ? 0.0f : 1.0f / ssum;  // nothing to share out: p = 0
#pragma unroll
      for (int i = 0; i < EPL; ++i) acc[i] = fmaf(s[i], inv, acc[i]);
      if (r == 0 && sum != 0.0f) {
        const float lse = base + logf(sum);
        z += static_cast<double>(lse) * lse;
      }
    }
    const size_t row = static_cast<size_t>(blockIdx.x) + q;
    if (r == 0) {
      z_sm[team] = z;
      n_sm[team] = n;
    }
    if (WPT == 1) {
#pragma unroll
      for (int i = 0; i < EPL; ++i) {
        const int e = TM::expert(i, r);
        if (e < E) acc_sm[team * E + e] = acc[i];
      }
    }
    __syncthreads();
    float* pr = a.part_p + row * E;
    int32_t* cr = a.part_c + row * E;
    if (WPT == 1) {
      for (int e = threadIdx.x; e < E; e += THREADS) {
        float v = 0.0f;
#pragma unroll
        for (int w = 0; w < kTeams; ++w) v += acc_sm[w * E + e];
        pr[e] = v;
      }
    } else {
#pragma unroll
      for (int i = 0; i < EPL; ++i) {
        const int e = TM::expert(i, r);
        if (e < E) pr[e] = acc[i];
      }
    }
    for (int e = threadIdx.x; e < E; e += THREADS) cr[e] = hist[e];
    if (threadIdx.x == 0) {
      double zz = 0.0;
      int nn = 0;
      for (int w = 0; w < kTeams; ++w) zz += z_sm[w], nn += n_sm[w];
      a.part_z[row] = zz;
      a.part_n[row] = nn;
    }
    __syncthreads();
    pos = end;
  }
  if (f.alone) balance_finish(f, fin, true);  // its own rows are all there are
}

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
  long long per_team;     // consecutive tokens of a team
};

template <int EPL, int WPT, bool V4>
__global__ void __launch_bounds__(256, EPL <= 8 ? 3 : 1) router_backward_kernel(const RouterBackwardArgs a) {
  using TM = Team<EPL, WPT, V4>;
  extern __shared__ __align__(16) uint8_t router_smem[];
  __shared__ float red[kTeamWarps];
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int E = a.E, r = TM::rank();
  const int team = WPT == 1 ? threadIdx.x >> 5 : 0;
  const int Epad = (E + 3) / 4 * 4;
  float* g = reinterpret_cast<float*>(router_smem) + static_cast<size_t>(team) * Epad;  // dL/ds of the selected experts
  for (int e = r; e < Epad; e += TM::kThreads) g[e] = 0.0f;
  TM::sync();
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const long long t0 = (static_cast<long long>(blockIdx.x) * (256 / TM::kThreads) + team) * a.per_team;
  const long long t1 = t0 + a.per_team < a.T ? t0 + a.per_team : a.T;
  float B[EPL];
#pragma unroll
  for (int i = 0; i < EPL; ++i) B[i] = 0.0f;
  const bool losses = a.counts != nullptr;
  const float zc = losses && a.z_grad != 0.0f ? a.z_grad * a.scales[a.S] : 0.0f;
  // the team's next token: its logits, and its slot r
  float nxt[EPL], w_nxt = 0.0f;
  int id_nxt = -1;
  bool in_nxt = false;
  auto fetch = [&](long long t) {
    if (t >= t1) return;
    TM::load(a.logits + t * a.ld, E, neg_inf(), nxt);
    in_nxt = !a.mask || a.mask[t];
    if (a.dw) {
      id_nxt = r < a.k ? a.ids[t * a.k + r] : -1;
      w_nxt = r < a.k ? a.dw[t * a.k + r] : 0.0f;
    }
  };
  fetch(t0);
  int q = -1;
  long long q_end = t0;  // where the sequence q ends
  for (long long t = t0; t < t1; ++t) {
    float l[EPL], s[EPL], d[EPL];
#pragma unroll
    for (int i = 0; i < EPL; ++i) l[i] = nxt[i];
    const int id0 = id_nxt >= 0 && id_nxt < E ? id_nxt : -1;
    const float w0 = w_nxt;
    const bool in = in_nxt;
    const float le0 = a.dw && id0 >= 0 ? a.logits[t * a.ld + id0] : 0.0f;
    fetch(t + 1);
    if (t >= q_end) {
      q = sequence_of(a.off, a.S, t);
      q_end = !a.off || q >= a.S ? a.T : a.off[q < 0 ? 0 : q + 1];
      const bool some = losses && q >= 0 && q < a.S;
      const float c = some ? a.balance_grad * a.scales[q] : 0.0f;
#pragma unroll
      for (int i = 0; i < EPL; ++i) {
        const int e = TM::expert(i, r);
        B[i] = some && e < E ? c * static_cast<float>(a.counts[static_cast<size_t>(q) * E + e]) : 0.0f;
      }
    }
    float dl[EPL];
#pragma unroll
    for (int i = 0; i < EPL; ++i) dl[i] = 0.0f;
    if (in && q >= 0 && q < a.S) {
      // exponentials, where the score or the z loss wants them
      float base = 0.0f, inv = 0.0f, lse = 0.0f;
      bool direct = false;
      const bool exps = a.func != kSqrtSoftplus || zc != 0.0f;
#pragma unroll
      for (int i = 0; i < EPL; ++i) s[i] = l[i];
      if (exps) {
        const float sum = exponentials<TM, EPL>(l, red, &base, &direct);
        inv = sum == 0.0f ? 0.0f : 1.0f / sum;  // a row of -inf: no probabilities, no gradient
        if (zc != 0.0f) lse = sum == 0.0f ? 0.0f : base + logf(sum);
      }
      // scores and their derivatives
      if (a.func == kSigmoid) {
        if (direct) {
#pragma unroll
          for (int i = 0; i < EPL; ++i) {
            const float rc = rcp_sfu(1.0f + l[i]);
            s[i] = l[i] * rc;
            d[i] = s[i] * rc;
          }
        } else {
#pragma unroll
          for (int i = 0; i < EPL; ++i) s[i] = score_of(kSigmoid, s[i], &d[i]);
        }
      } else if (a.func == kSqrtSoftplus) {
#pragma unroll
        for (int i = 0; i < EPL; ++i) {
          d[i] = 0.0f;
          s[i] = TM::expert(i, r) < E ? score_of(kSqrtSoftplus, s[i], &d[i]) : 0.0f;
        }
      }
      // dL/ds of the selected experts, scattered into g
      if (a.dw) {
        auto score_at = [&](float le) {
          float dd;
          return a.func == kSoftmax ? exp_sfu(le - base) * inv : score_of(a.func, le, &dd);
        };
        float c = a.route_scale, mean = 0.0f;
        if (a.renorm) {
          float Q = 0.0f, GQ = 0.0f;
          if (id0 >= 0) {
            Q = score_at(le0);
            GQ = w0 * Q;
          }
          for (int j = r + TM::kThreads; j < a.k; j += TM::kThreads) {
            const int e = a.ids[t * a.k + j];
            if (e >= 0 && e < E) {
              const float v = score_at(a.logits[t * a.ld + e]);
              Q += v;
              GQ = fmaf(a.dw[t * a.k + j], v, GQ);
            }
          }
          Q = TM::sum(Q, red);
          GQ = TM::sum(GQ, red);
          if (Q > 0.0f) {  // as the gate: a sum of 0 divides nothing
            const float iq = 1.0f / Q;
            c *= iq;
            mean = GQ * iq;
          }
        }
        // 32 slots at a time; equal ids of a group are added in slot order
        if (WPT == 1 || threadIdx.x < 32) {
          const int lane = threadIdx.x & 31;
          for (int j0 = 0; j0 < a.k; j0 += 32) {
            int e = id0;
            float v = w0;
            if (j0) {
              const int j = j0 + lane;
              e = j < a.k ? a.ids[t * a.k + j] : -1;
              if (e < 0 || e >= E) e = -1;
              v = e >= 0 ? a.dw[t * a.k + j] : 0.0f;
            }
            v = c * (v - mean);
            const unsigned same = __match_any_sync(0xFFFFFFFFu, e);
            if (__all_sync(0xFFFFFFFFu, (same & (same - 1)) == 0 || e < 0)) {
              if (e >= 0) g[e] += v;
            } else {
              for (int i = 0; i < 32; ++i) {
                if (lane == i && e >= 0) g[e] += v;
                __syncwarp();
              }
            }
            __syncwarp();
          }
        }
        TM::sync();
#pragma unroll
        for (int i = 0; i < EPL; ++i) {
          const int e = TM::expert(i, r);
          dl[i] = e < E ? g[e] : 0.0f;
        }
        TM::sync();
        if (id0 >= 0) g[id0] = 0.0f;  // back to zero
        for (int j = r + TM::kThreads; j < a.k; j += TM::kThreads) {
          const int e = a.ids[t * a.k + j];
          if (e >= 0 && e < E) g[e] = 0.0f;
        }
        TM::sync();
      }
      if (a.func == kSoftmax) {
        float dot = 0.0f;
#pragma unroll
        for (int i = 0; i < EPL; ++i) {
          dl[i] += B[i];
          dot = fmaf(dl[i], l[i], dot);
        }
        dot = TM::sum(dot, red) * inv;
        const float shift = zc * lse - dot;
#pragma unroll
        for (int i = 0; i < EPL; ++i) dl[i] = l[i] * inv * (dl[i] + shift);
      } else {
        if (losses) {
          float ssum = 0.0f, bsum = 0.0f;
#pragma unroll
          for (int i = 0; i < EPL; ++i) {
            ssum += s[i];
            bsum = fmaf(B[i], s[i], bsum);
          }
          ssum = TM::sum(ssum, red);
          bsum = TM::sum(bsum, red);
          const float is = ssum == 0.0f ? 0.0f : 1.0f / ssum;
          const float mean = bsum * is;
#pragma unroll
          for (int i = 0; i < EPL; ++i) dl[i] = fmaf(B[i] - mean, is, dl[i]);
        }
        const float zl = zc * lse * inv;
#pragma unroll
        for (int i = 0; i < EPL; ++i) {
          dl[i] *= d[i];
          if (zc != 0.0f) dl[i] = fmaf(zl, l[i], dl[i]);
        }
      }
    }
    float* o = a.out + t * a.ld_out;
    if constexpr (V4) {
#pragma unroll
      for (int i = 0; i < EPL; i += 4) {
        const int e = TM::expert(i, r);
        if (e < E) *reinterpret_cast<float4*>(o + e) = make_float4(dl[i], dl[i + 1], dl[i + 2], dl[i + 3]);
      }
    } else {
#pragma unroll
      for (int i = 0; i < EPL; ++i) {
        const int e = TM::expert(i, r);
        if (e < E) o[e] = dl[i];
      }
    }
  }
}

// dw[t, j] = sum_o dout[t, o] v[slot_row[t, j], o]: WPS warps per slot, each
// lane four partial sums (the quads of its columns), folded in a fixed order.
template <int WPS, bool V4>
__global__ void __launch_bounds__(256) combine_backward_kernel(const float* __restrict__ dout,
                                                               const float* __restrict__ v, long long v_rows,
                                                               const int32_t* __restrict__ slot_row, long long slots,
                                                               int k, int O, float* __restrict__ dw, unsigned* err) {
  __shared__ float red[8];
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int w = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long long slot = static_cast<long long>(blockIdx.x) * (8 / WPS) + w / WPS;
  const int part = (w % WPS) * 32 + lane;
  float s = 0.0f;
  if (slot < slots) {
    long long row = slot_row[slot];
    if (row < 0 || row >= v_rows) {
      if (part == 0 && err) atomicOr(err, kErrBadExpertId);
      row = 0;
    }
    const float* d = dout + slot / k * static_cast<long long>(O);
    const float* x = v + row * O;
    if constexpr (V4) {
      float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 8
      for (int o = part * 4; o < O; o += WPS * 128) {
        const float4 a = *reinterpret_cast<const float4*>(d + o);
        const float4 b = __ldcs(reinterpret_cast<const float4*>(x + o));
        acc.x = fmaf(a.x, b.x, acc.x);
        acc.y = fmaf(a.y, b.y, acc.y);
        acc.z = fmaf(a.z, b.z, acc.z);
        acc.w = fmaf(a.w, b.w, acc.w);
      }
      s = (acc.x + acc.y) + (acc.z + acc.w);
    } else {
#pragma unroll 8
      for (int o = part; o < O; o += WPS * 32) s = fmaf(d[o], x[o], s);
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xFFFFFFFFu, s, o);
  if (WPS > 1) {
    if (lane == 0) red[w] = s;
    __syncthreads();
    s = red[w / WPS * WPS];
    for (int i = 1; i < WPS; ++i) s += red[w / WPS * WPS + i];
  }
  if (slot < slots && part == 0) dw[slot] = s;
}

}  // namespace dev

namespace {

constexpr size_t kMaxExperts = 8192;  // as the router and the gate

struct BalancePlan {
  long long chunk;
  size_t chunks, rows, groups;
  size_t p, c, z, n, bal, seqz, ticket, total;  // offsets into the workspace
};

int check_router(const char* action, size_t T, size_t E, size_t k, size_t S, int func, const void* off) {
  if (T > (1u << 30) || E == 0 || E > kMaxExperts || k == 0 || k > E)
    return OBJB_FAIL(OBJB_ERR_INVALID_INPUT, action,
                     "need num_tokens <= 2^30 and 1 <= top_k <= num_experts <= 8192 (got top_k " + std::to_string(k) +
                         ", num_experts " + std::to_string(E) + ", num_tokens " + std::to_string(T) + ")");
  if (func < 0 || func > 2)
    return OBJB_FAIL(OBJB_ERR_INVALID_INPUT, action, "score_func must be 0 (softmax), 1 (sigmoid) or 2");
  if (S == 0 || S > (1u << 24) || (S != 1 && !off))
    return OBJB_FAIL(OBJB_ERR_INVALID_INPUT, action,
                     "need 1 <= num_seqs <= 2^24, and num_seqs 1 without sequence offsets");
  return OBJB_OK;
}

// Blocks of the partial pass: three per SM at most (what its registers allow).
// Up to 128 tokens one block does it, and, with few experts and sequences, the
// finish too (no second launch); beyond, 16 tokens or more in each.
BalancePlan plan_balance(size_t T, size_t E, size_t S, int sms) {
  BalancePlan p;
  const size_t most = static_cast<size_t>(3) * sms;
  const size_t want = T <= 128 ? 1 : std::min(most, (T + 15) / 16);
  p.chunk = static_cast<long long>(std::max<size_t>(1, (T + want - 1) / want));
  p.chunks = (T + p.chunk - 1) / p.chunk;
  p.rows = p.chunks + S;
  p.groups = (E + 31) / 32;
  size_t at = 0;
  auto take = [&](size_t bytes) {
    const size_t o = at;
    at += (bytes + 255) / 256 * 256;
    return o;
  };
  p.ticket = take(4);
  p.p = take(p.rows * E * 4);
  p.c = take(p.rows * E * 4);
  p.z = take(p.rows * 8);
  p.n = take(p.rows * 4);
  p.bal = take(S * p.groups * 8);
  p.seqz = take(S * 8);
  p.total = at;
  return p;
}

int plan_balance_here(size_t T, size_t E, size_t S, BalancePlan* p) {
  int device = 0;
  OBJB_TRY(current_device(&device));
  DeviceProps props;
  OBJB_TRY(device_props(device, &props));
  *p = plan_balance(T, E, S, props.sm_count);
  return OBJB_OK;
}

// f(EPL, WPT, V4) for E experts; v4: rows of whole aligned quads.
template <class F>
int with_team(size_t E, bool v4, F&& f) {
  using std::integral_constant;
#define OBJB_TEAM(EPL, WPT, V) f(integral_constant<int, EPL>{}, integral_constant<int, WPT>{}, integral_constant<bool, V>{})
  if (E <= 32) return OBJB_TEAM(1, 1, false);
  if (E <= 64) return OBJB_TEAM(2, 1, false);
  if (E <= 128) return v4 ? OBJB_TEAM(4, 1, true) : OBJB_TEAM(4, 1, false);
  if (E <= 256) return v4 ? OBJB_TEAM(8, 1, true) : OBJB_TEAM(8, 1, false);
  if (E <= 512) return v4 ? OBJB_TEAM(16, 1, true) : OBJB_TEAM(16, 1, false);
  if (E <= 1024) return v4 ? OBJB_TEAM(32, 1, true) : OBJB_TEAM(32, 1, false);
  return OBJB_TEAM(32, dev::kTeamWarps, false);
#undef OBJB_TEAM
}

}  // namespace
}  // namespace objb

using namespace objb;

extern "C" {

int objb_balance_loss_scratch_bytes(size_t num_tokens, size_t num_experts, size_t num_seqs, size_t* bytes) {
  clear_error();
  if (!bytes) return OBJB_FAIL(OBJB_ERR_INVALID_INPUT, "objb_balance_loss_scratch_bytes", "null output pointer");
  OBJB_TRY(check_router("objb_balance_loss_scratch_bytes", num_tokens, num_experts, 1, num_seqs, 0, bytes));
  BalancePlan p;
  OBJB_TRY(plan_balance_here(num_tokens, num_experts, num_seqs, &p));
  *bytes = p.total;
  return OBJB_OK;
}

int objb_balance_loss_device(const float* d_logits, size_t logits_stride, const int32_t* d_ids,
                             const uint8_t* d_token_mask, const int32_t* d_seq_offsets, size_t num_seqs,
                             size_t num_tokens, size_t num_experts, size_t top_k, int score_func, int32_t* d_counts,
                             int32_t* d_seq_tokens, float* d_losses, float* d_scales, void* d_scratch,
                             size_t scratch_bytes, objb_stream_t stream) {
  clear_error();
  const char* action = "objb_balance_loss_device";
  OBJB_TRY(check_router(action, num_tokens, num_experts, top_k, num_seqs, score_func, d_seq_offsets));
  if ((num_tokens && (!d_logits || !d_ids)) || !d_counts || !d_seq_tokens || !d_losses || !d_scales)
    return OBJB_FAIL(OBJB_ERR_INVALID_INPUT, action, "null device pointer");
  const size_t ld = logits_stride ? logits_stride : num_experts;
  if (ld < num_experts) return OBJB_FAIL(OBJB_ERR_INVALID_INPUT, action, "logits_stride is below num_experts");
  BalancePlan p;
  OBJB_TRY(plan_balance_here(num_tokens, num_experts, num_seqs, &p));
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  void* ws = d_scratch;
  if (ws) {
    if (scratch_bytes < p.total || (reinterpret_cast<uintptr_t>(ws) & 255u))
      return OBJB_FAIL(OBJB_ERR_INVALID_INPUT, action,
                       "scratch needs " + std::to_string(p.total) + " bytes, 256-byte aligned (got " +
                           std::to_string(scratch_bytes) + ")");
  } else {
    int device = 0;
    OBJB_TRY(current_device(&device));
    OBJB_TRY(workspace_get(device, st, p.total, &ws));
  }
  uint8_t* b = static_cast<uint8_t*>(ws);
  dev::BalanceFinishArgs f;
  dev::BalanceArgs& a = f.a;
  a.logits = d_logits;
  a.ld = ld;
  a.ids = d_ids;
  a.mask = d_token_mask;
  a.off = d_seq_offsets;
  a.S = static_cast<int>(num_seqs);
  a.T = static_cast<long long>(num_tokens);
  a.E = static_cast<int>(num_experts);
  a.k = static_cast<int>(top_k);
  a.func = score_func;
  a.chunk = p.chunk;
  a.ticket = reinterpret_cast<unsigned*>(b + p.ticket);
  a.part_p = reinterpret_cast<float*>(b + p.p);
  a.part_c = reinterpret_cast<int32_t*>(b + p.c);
  a.part_z = reinterpret_cast<double*>(b + p.z);
  a.part_n = reinterpret_cast<int32_t*>(b + p.n);
  f.groups = static_cast<int>(p.groups);
  f.alone = p.chunks <= 1 && num_seqs * p.groups <= 8;
  f.bal_part = reinterpret_cast<double*>(b + p.bal);
  f.seq_z = reinterpret_cast<double*>(b + p.seqz);
  f.counts = d_counts;
  f.tokens = d_seq_tokens;
  f.losses = d_losses;
  f.scales = d_scales;
  const bool v4 = aligned16(d_logits) && ld % 4 == 0 && num_experts % 4 == 0;
  const int grid = static_cast<int>(std::max<size_t>(1, p.chunks));
  OBJB_TRY(with_team(num_experts, v4, [&](auto epl, auto wpt, auto v) {
    constexpr int EPL = decltype(epl)::value, WPT = decltype(wpt)::value;
    constexpr int THREADS = 256;
    const size_t teams = WPT == 1 ? THREADS / 32 : 0;
    const size_t smem = ((num_experts + 3) / 4 * 4 + teams * num_experts) * 4;
    return launch_pdl(dev::balance_partial_kernel<EPL, WPT, decltype(v)::value, THREADS>, grid, THREADS, smem, st, f);
  }));
  if (f.alone) return OBJB_OK;
  return launch_pdl(dev::balance_finish_kernel, static_cast<int>(num_seqs * p.groups), 256, 0, st, f);
}

int objb_router_backward_device(const float* d_logits, size_t logits_stride, const int32_t* d_ids,
                                const float* d_dweights, const uint8_t* d_token_mask, const int32_t* d_seq_offsets,
                                size_t num_seqs, const int32_t* d_counts, const float* d_scales, size_t num_tokens,
                                size_t num_experts, size_t top_k, int score_func, int renormalize, float route_scale,
                                float balance_grad, float z_grad, float* d_dlogits, size_t dlogits_stride,
                                objb_stream_t stream) {
  clear_error();
  const char* action = "objb_router_backward_device";
  OBJB_TRY(check_router(action, num_tokens, num_experts, top_k, num_seqs, score_func, d_seq_offsets));
  if (num_tokens == 0) return OBJB_OK;
  if (!d_logits || !d_ids || !d_dlogits) return OBJB_FAIL(OBJB_ERR_INVALID_INPUT, action, "null device pointer");
  if (!d_counts != !d_scales)
    return OBJB_FAIL(OBJB_ERR_INVALID_INPUT, action, "counts and scales of the balance loss come together");
  if (!d_counts && (balance_grad != 0.0f || z_grad != 0.0f))
    return OBJB_FAIL(OBJB_ERR_INVALID_INPUT, action, "a loss gradient needs the counts and scales of the balance loss");
  if (!d_counts && !d_dweights)
    return OBJB_FAIL(OBJB_ERR_INVALID_INPUT, action, "neither routing-weight gradients nor losses are given");
  const size_t ld = logits_stride ? logits_stride : num_experts;
  const size_t ldo = dlogits_stride ? dlogits_stride : num_experts;
  if (ld < num_experts || ldo < num_experts)
    return OBJB_FAIL(OBJB_ERR_INVALID_INPUT, action, "a row stride is below num_experts");
  if (d_logits == d_dlogits && ld != ldo)
    return OBJB_FAIL(OBJB_ERR_INVALID_INPUT, action, "in place needs equal row strides");
  int device = 0;
  OBJB_TRY(current_device(&device));
  DeviceProps props;
  OBJB_TRY(device_props(device, &props));
  dev::RouterBackwardArgs a;
  a.logits = d_logits;
  a.ld = ld;
  a.ids = d_ids;
  a.dw = d_dweights;
  a.mask = d_token_mask;
  a.off = d_seq_offsets;
  a.S = static_cast<int>(num_seqs);
  a.counts = d_counts;
  a.scales = d_scales;
  a.T = static_cast<long long>(num_tokens);
  a.E = static_cast<int>(num_experts);
  a.k = static_cast<int>(top_k);
  a.func = score_func;
  a.renorm = renormalize != 0;
  a.route_scale = route_scale;
  a.balance_grad = balance_grad;
  a.z_grad = z_grad;
  a.out = d_dlogits;
  a.ld_out = ldo;
  const bool v4 = aligned16(d_logits) && aligned16(d_dlogits) && ld % 4 == 0 && ldo % 4 == 0 && num_experts % 4 == 0;
  return with_team(num_experts, v4, [&](auto epl, auto wpt, auto v) {
    constexpr int EPL = decltype(epl)::value, WPT = decltype(wpt)::value;
    const size_t teams = 8 / WPT;
    // up to three blocks per SM (what the registers allow), each team a run of consecutive tokens
    const size_t most = static_cast<size_t>(EPL <= 8 ? 3 : 1) * props.sm_count * teams;
    a.per_team = static_cast<long long>((num_tokens + most - 1) / most);
    const size_t per_block = teams * a.per_team;
    const size_t smem = teams * ((num_experts + 3) / 4 * 4) * 4;
    return launch_pdl(dev::router_backward_kernel<EPL, WPT, decltype(v)::value>,
                      static_cast<int>((num_tokens + per_block - 1) / per_block), 256, smem,
                      static_cast<cudaStream_t>(stream), a);
  });
}

int objb_moe_combine_backward_device(const float* d_dout, const float* d_v, size_t v_rows, const int32_t* d_slot_row,
                                     size_t num_tokens, size_t top_k, size_t out_dim, float* d_dweights,
                                     objb_stream_t stream) {
  clear_error();
  const char* action = "objb_moe_combine_backward_device";
  if (num_tokens > (1u << 24) || top_k == 0 || top_k > 1024 || out_dim == 0 || out_dim > (1u << 24) ||
      v_rows > (1u << 30) || num_tokens * top_k > (1u << 30))
    return OBJB_FAIL(OBJB_ERR_INVALID_INPUT, action,
                     "need num_tokens <= 2^24, 1 <= top_k <= 1024, num_tokens * top_k <= 2^30, 1 <= out_dim <= 2^24");
  if (num_tokens == 0) return OBJB_OK;
  if (!d_dout || !d_v || !d_slot_row || !d_dweights || v_rows == 0)
    return OBJB_FAIL(OBJB_ERR_INVALID_INPUT, action, "null device pointer or no value rows");
  int device = 0;
  OBJB_TRY(current_device(&device));
  DeviceProps props;
  OBJB_TRY(device_props(device, &props));
  unsigned* err = nullptr;
  OBJB_TRY(device_error_word(device, &err));
  const long long slots = static_cast<long long>(num_tokens * top_k);
  const bool v4 = aligned16(d_dout) && aligned16(d_v) && out_dim % 4 == 0;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  auto go = [&](auto wps, auto v) {
    constexpr int WPS = decltype(wps)::value;
    const int grid = static_cast<int>((slots + 8 / WPS - 1) / (8 / WPS));
    return launch_pdl(dev::combine_backward_kernel<WPS, decltype(v)::value>, grid, 256, 0, st, d_dout, d_v,
                      static_cast<long long>(v_rows), d_slot_row, slots, static_cast<int>(top_k),
                      static_cast<int>(out_dim), d_dweights, err);
  };
  using std::integral_constant;
  // a warp per slot once the slots alone fill the SMs, else a block per slot
  const bool many = slots >= static_cast<long long>(props.sm_count) * 16;
  if (many)
    return v4 ? go(integral_constant<int, 1>{}, integral_constant<bool, true>{})
              : go(integral_constant<int, 1>{}, integral_constant<bool, false>{});
  return v4 ? go(integral_constant<int, 8>{}, integral_constant<bool, true>{})
            : go(integral_constant<int, 8>{}, integral_constant<bool, false>{});
}

}  // extern "C"
