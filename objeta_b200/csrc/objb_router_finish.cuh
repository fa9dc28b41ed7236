// objb_router_finish.cuh -- the partial rows of the balance loss folded into
// counts, losses and gradient factors.
#pragma once

#include "objb_router.cuh"
#include "objb_tc.cuh"

namespace objb {
namespace dev {

template <int WARPS>
struct FinishSmem {
  double p[WARPS][32];
  int c[WARPS][32];
  double z[WARPS];
  int n[WARPS];
  double red[4][WARPS];
  bool last;
};

__device__ __forceinline__ double warp_sum(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
  return v;
}

// One (sequence, 32 experts) item per block and turn: the partial rows of the
// sequence are summed in block order (interleaved over the warps, the runs
// folded in order), in double.  The block that finishes last (of a cluster the
// first, behind its barrier; alone the only one) folds the sequences' sums into
// the losses.
template <int WARPS>
__device__ __forceinline__ void balance_finish(const BalanceFinishArgs& f, FinishSmem<WARPS>& sm, int mode) {
  const BalanceArgs& a = f.a;
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  const int items = a.S * f.groups;
  for (int item = mode == kFinishAlone ? 0 : blockIdx.x; item < items;
       item += mode == kFinishAlone ? 1 : gridDim.x) {
    const int q = item / f.groups, g = item - q * f.groups;
    const int e = g * 32 + lane;
    long long b = a.off ? a.off[q] : 0, end = a.off ? a.off[q + 1] : a.T;
    b = b > 0 ? b : 0;
    end = end < a.T ? end : a.T;
    const int c0 = static_cast<int>(b / a.chunk), c1 = end > b ? static_cast<int>((end - 1) / a.chunk) : c0 - 1;
    const size_t row0 = static_cast<size_t>(c0) + q;
    double p = 0.0;
    int c = 0;
    if (e < a.E) {
      const float* pp = a.part_p + row0 * a.E + e;
      const int32_t* pc = a.part_c + row0 * a.E + e;
#pragma unroll 8
      for (int i = w; i <= c1 - c0; i += WARPS) {
        p += pp[static_cast<size_t>(i) * a.E];
        c += pc[static_cast<size_t>(i) * a.E];
      }
    }
    sm.p[w][lane] = p;
    sm.c[w][lane] = c;
    if (g == 0) {
      double z = 0.0;
      int n = 0;
      for (int i = threadIdx.x; i <= c1 - c0; i += 32 * WARPS) z += a.part_z[row0 + i], n += a.part_n[row0 + i];
      z = warp_sum(z);
      n = __reduce_add_sync(0xFFFFFFFFu, n);
      if (lane == 0) sm.z[w] = z, sm.n[w] = n;
    }
    __syncthreads();
    if (w == 0) {
      for (int i = 1; i < WARPS; ++i) p += sm.p[i][lane], c += sm.c[i][lane];
      if (e < a.E) f.counts[static_cast<size_t>(q) * a.E + e] = c;
      const double v = warp_sum(p * c);
      if (lane == 0) f.bal_part[item] = v;
    } else if (w == 1 && g == 0) {
      const double z = warp_sum(lane < WARPS ? sm.z[lane] : 0.0);
      const int n = __reduce_add_sync(0xFFFFFFFFu, lane < WARPS ? sm.n[lane] : 0);
      if (lane == 0) {
        f.seq_z[q] = z;
        f.tokens[q] = n;
      }
    }
    __syncthreads();
  }
  if (mode == kFinishInCluster) {
    cluster_sync_all();
    if (blockIdx.x != 0) return;
  } else if (mode == kFinishGrid) {
    if (threadIdx.x == 0) {
      __threadfence();
      sm.last = atomicAdd(a.ticket, 1u) == gridDim.x - 1;
      __threadfence();
    }
    __syncthreads();
    if (!sm.last) return;
  }
  double t[4] = {};  // S', N, sum of z, sum of the sequences' balances
  for (int i = threadIdx.x; i < a.S; i += 32 * WARPS) {
    const int n = __ldcg(f.tokens + i);
    const double z = __ldcg(f.seq_z + i);
    double v = 0.0;
    for (int j = 0; j < f.groups; ++j) v += __ldcg(f.bal_part + static_cast<size_t>(i) * f.groups + j);
    if (n == 0) continue;
    t[0] += 1.0;
    t[1] += n;
    t[2] += z;
    t[3] += v * a.E / (static_cast<double>(a.k) * n * n);
  }
  const bool one = a.S <= 32;  // all in warp 0: no block sum
  if (one && w > 0) return;
#pragma unroll
  for (int i = 0; i < 4; ++i) t[i] = warp_sum(t[i]);
  if (!one) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (lane == 0) sm.red[i][w] = t[i];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      t[i] = 0.0;
      for (int j = 0; j < WARPS; ++j) t[i] += sm.red[i][j];
    }
  }
  for (int i = threadIdx.x; i < a.S; i += one ? 32 : 32 * WARPS) {
    const double n = __ldcg(f.tokens + i);
    f.scales[i] = n > 0.0 ? static_cast<float>(a.E / (a.k * n * n * t[0])) : 0.0f;
  }
  if (threadIdx.x == 0) {
    f.losses[0] = t[0] > 0.0 ? static_cast<float>(t[3] / t[0]) : 0.0f;
    f.losses[1] = t[1] > 0.0 ? static_cast<float>(t[2] / t[1]) : 0.0f;
    f.scales[a.S] = t[1] > 0.0 ? static_cast<float>(2.0 / t[1]) : 0.0f;
  }
}

}  // namespace dev
}  // namespace objb
