// router_partial.cu -- the first pass of the balance loss: each block's tokens,
// sequence by sequence, into partial sums of the scores' shares, selections,
// lse^2 and counted tokens.  Bound by its instructions (about 200 per token
// and warp at 256 experts, 24 warps an SM), not by the 4 bytes per logit:
// 32768 x 256 takes 12.4 us (softmax) or 15.8 (sigmoid), 63 % of an active SM's
// issue slots, where the logits alone take 5.2.  Logits further than 11.5 from 0
// take their maximum first (a call of both launches 19 -> 22 and 21 -> 29 us).
#include "objb_router.cuh"
#include "objb_router_finish.cuh"

namespace objb {
namespace dev {

template <class TM, int FUNC, int THREADS>
__global__ void __launch_bounds__(THREADS, TM::EPL <= 8 ? 3 : TM::EPL <= 16 ? 2 : 1) balance_partial_kernel(const BalanceFinishArgs f) {
  constexpr int EPL = TM::EPL, L = TM::L;
  constexpr int kTeams = THREADS / L;
  extern __shared__ __align__(16) uint8_t router_smem[];
  const BalanceArgs& a = f.a;
  int32_t* hist = reinterpret_cast<int32_t*>(router_smem);             // [E]
  float* acc_sm = reinterpret_cast<float*>(hist + (a.E + 3) / 4 * 4);  // [kTeams][E], teams within a warp
  __shared__ float red[kTeamWarps];
  __shared__ double z_sm[kTeams];
  __shared__ int n_sm[kTeams];
  __shared__ FinishSmem<THREADS / 32> fin;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (blockIdx.x == 0 && threadIdx.x == 0) *a.ticket = 0;
  const int E = a.E, r = TM::rank();
  const int team = TM::kBlock ? 0 : threadIdx.x / L;
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
      in_nxt = t < end && (!a.mask || a.mask[t]);
      id_nxt = -1;
      if (t < end) {
        TM::load(a.logits + t * a.ld, E, neg_inf(), nxt);
        if (r < a.k) id_nxt = a.ids[t * a.k + r];
      } else {
#pragma unroll
        for (int i = 0; i < EPL; ++i) nxt[i] = 0.0f;
      }
    };
    fetch(pos + team);
    for (long long t = pos + team; t - team < end; t += kTeams) {  // the teams of a warp in step
      float l[EPL], s[EPL];
#pragma unroll
      for (int i = 0; i < EPL; ++i) l[i] = nxt[i];
      const int id = id_nxt;
      const bool in = in_nxt;
      fetch(t + kTeams);
      if (in) {
        if (id >= 0 && id < E) atomicAdd(&hist[id], 1);
        for (int j = r + L; j < a.k; j += L) {
          const int e = a.ids[t * a.k + j];
          if (e >= 0 && e < E) atomicAdd(&hist[e], 1);
        }
      }
      float base;
      bool direct;
      const float sum = exponentials<TM>(l, s, red, &base, &direct);
      float ssum = sum;
      if (FUNC != kSoftmax) {
        ssum = 0.0f;
        if (FUNC == kSigmoid && direct) {
#pragma unroll
          for (int i = 0; i < EPL; ++i) {
            s[i] *= rcp_sfu(1.0f + s[i]);
            ssum += s[i];
          }
        } else {
#pragma unroll
          for (int i = 0; i < EPL; ++i) {
            float d;
            s[i] = TM::expert(i, r) < E ? score_of(FUNC, l[i], &d) : 0.0f;
            ssum += s[i];
          }
        }
        __syncwarp();
        ssum = TM::sum(ssum, red);
      }
      const float inv = !in || ssum == 0.0f ? 0.0f : rcp_sfu(ssum);  // nothing to share out: p = 0
      if (in) {
#pragma unroll
        for (int i = 0; i < EPL; ++i) acc[i] = fmaf(s[i], inv, acc[i]);
        ++n;
        if (r == 0 && sum != 0.0f) {
          const float lse = base + __logf(sum);
          z += static_cast<double>(lse) * lse;
        }
      }
    }
    const size_t row = static_cast<size_t>(blockIdx.x) + q;
    if (r == 0) {
      z_sm[team] = z;
      n_sm[team] = n;
    }
    if (!TM::kBlock) {
#pragma unroll
      for (int i = 0; i < EPL; ++i) {
        const int e = TM::expert(i, r);
        if (e < E) acc_sm[team * E + e] = acc[i];
      }
    }
    __syncthreads();
    float* pr = a.part_p + row * E;
    int32_t* cr = a.part_c + row * E;
    if (!TM::kBlock) {
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
#pragma unroll
      for (int w = 0; w < kTeams; ++w) zz += z_sm[w], nn += n_sm[w];
      a.part_z[row] = zz;
      a.part_n[row] = nn;
    }
    __syncthreads();
    pos = end;
  }
  if (f.mode == kFinishInCluster) cluster_sync_all();  // the other blocks' rows are in place
  if (f.mode != kFinishGrid) balance_finish(f, fin, f.mode);
}

}  // namespace dev

int launch_balance_partial(const dev::BalanceFinishArgs& f, int grid, bool v4, cudaStream_t st) {
  return with_team<32>(f.a.E, v4, [&](auto tm) {
    return with_func(f.a.func, [&](auto func) -> int {
      using TM = decltype(tm);
      constexpr int THREADS = 256;
      const size_t teams = TM::kBlock ? 0 : THREADS / TM::L;
      const size_t smem = (static_cast<size_t>(f.a.E + 3) / 4 * 4 + teams * f.a.E) * 4;
      auto kernel = dev::balance_partial_kernel<TM, decltype(func)::value, THREADS>;
      if (f.mode != dev::kFinishInCluster) return launch_pdl(kernel, grid, THREADS, smem, st, f);
      cudaLaunchConfig_t cfg = {};
      cfg.gridDim = dim3(grid);
      cfg.blockDim = dim3(THREADS);
      cfg.dynamicSmemBytes = smem;
      cfg.stream = st;
      cudaLaunchAttribute attr[2];
      attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
      attr[0].val.programmaticStreamSerializationAllowed = 1;
      attr[1].id = cudaLaunchAttributeClusterDimension;
      attr[1].val.clusterDim.x = static_cast<unsigned>(grid);
      attr[1].val.clusterDim.y = 1;
      attr[1].val.clusterDim.z = 1;
      cfg.attrs = attr;
      cfg.numAttrs = 2;
      OBJB_CUDA(cudaLaunchKernelEx(&cfg, kernel, f), "launch balance loss");
      return OBJB_OK;
    });
  });
}

}  // namespace objb
