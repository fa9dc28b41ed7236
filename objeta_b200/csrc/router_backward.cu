// router_backward.cu -- the gradient of the router's logits, through the
// routing weights and the balance and z losses, in one pass over the logits.
// 32768 x 256: 22 us (softmax) or 24 (sigmoid) where reading and writing 67 MB
// takes 10.4 (issue slots 44 and 52 %): the reductions of a token (its
// exponentials' sum, the weights', the losses') follow one another, in 16 to 24
// warps an SM that 80 to 128 registers leave room for.
#include "objb_router.cuh"

namespace objb {
namespace dev {

// A token whose renormalised weights' scores (nearly) underflow: given ids need
// not be the largest.  With q = exp(l - top) relative to the largest selected (a
// sigmoid is its exponential there) w = q / sum q and dl = w (dw - mean), not by
// way of the scores, down to scores of exp(-128), which f32 has long lost; a
// mask is far below.  One at a time, behind the team's ordinary tokens: beside
// them its registers would cost those 12 % (32768 x 256), a call of its own
// 25 % where they fill the registers (2000 experts, sigmoid).  `mine`: the team
// has one (the teams of a warp run in step).  g: zeros, and left as such.
template <class TM, int FUNC>
__device__ __forceinline__ void far_token(const RouterBackwardArgs& a, long long t, bool mine, float* g, float* red) {
  const int r = TM::rank(), E = mine ? a.E : 0, k = mine ? a.k : 0;
  if (!mine) t = 0;
  const float* l = a.logits + t * a.ld;
  const int32_t* ids = a.ids + t * a.k;
  const float* dw = a.dw + t * a.k;
  auto selected = [&](auto f) {
    for (int j = r; j < k; j += TM::L) {
      const int e = ids[j];
      if (e >= 0 && e < E) f(l[e], dw[j]);
    }
    __syncwarp();
  };
  auto experts = [&](auto f) {
    for (int e = r; e < E; e += TM::L) f(e, l[e]);
    __syncwarp();
  };
  // the row's statistics
  float m = neg_inf(), sum = 0.0f;
  experts([&](int, float v) { m = fmaxf(m, v); });
  m = TM::max(m, red);
  const float base = m > neg_inf() ? m : 0.0f;
  experts([&](int, float v) { sum += exp_sfu(v - base); });
  sum = TM::sum(sum, red);
  const float inv = sum == 0.0f ? 0.0f : rcp_sfu(sum), lse = sum == 0.0f ? 0.0f : base + __logf(sum);
  // the weights
  float top = neg_inf(), q = 0.0f, wq = 0.0f, rest = 0.0f;
  selected([&](float v, float) { top = fmaxf(top, v); });
  top = TM::max(top, red);
  const bool some = top - (FUNC == kSoftmax ? lse : 0.0f) > -128.0f;
  selected([&](float v, float w) {
    const float x = some ? exp_sfu(v - top) : 0.0f;
    q += x;
    wq = fmaf(x, w, wq);
  });
  q = TM::sum(q, red);
  const float iq = some ? rcp_sfu(q) : 0.0f;
  const float mean = TM::sum(wq, red) * iq;
  selected([&](float v, float w) { rest = some ? fmaf(exp_sfu(v - top), w - mean, rest) : 0.0f; });
  rest = TM::sum(rest, red) * iq;
  if (r == 0 && some)
    for (int j = 0; j < k; ++j) {
      const int e = ids[j];
      if (e >= 0 && e < E) g[e] += a.route_scale * (exp_sfu(l[e] - top) * iq * ((dw[j] - mean) - rest));
    }
  // the losses
  const int seq = mine ? sequence_of(a.off, a.S, t) : 0;
  const float zc = a.counts && a.z_grad != 0.0f ? a.z_grad * a.scales[a.S] : 0.0f;
  const float c = a.counts ? a.balance_grad * a.scales[seq] : 0.0f;
  auto B = [&](int e) { return a.counts ? c * static_cast<float>(a.counts[static_cast<size_t>(seq) * E + e]) : 0.0f; };
  float ssum = 0.0f, bsum = 0.0f, d;
  experts([&](int e, float v) {
    const float s = FUNC == kSoftmax ? exp_sfu(v - base) * inv : score_of(FUNC, v, &d);
    ssum += s;
    bsum = fmaf(B(e), s, bsum);
  });
  ssum = TM::sum(ssum, red);
  bsum = TM::sum(bsum, red);
  const float is = FUNC == kSoftmax ? 1.0f : ssum == 0.0f ? 0.0f : rcp_sfu(ssum);
  TM::sync();
  experts([&](int e, float v) {
    const float p = exp_sfu(v - base) * inv;
    d = p;
    if (FUNC != kSoftmax) score_of(FUNC, v, &d);
    float dl = g[e];
    if (a.counts) dl += d * (B(e) * is - bsum * is * is);
    if (zc != 0.0f) dl += zc * lse * p;
    a.out[t * a.ld_out + e] = dl;
    g[e] = 0.0f;
  });
  TM::sync();
}

template <class TM, int FUNC>
__global__ void __launch_bounds__(256, TM::EPL <= 8 ? 3 : TM::EPL <= 16 ? 2 : 1)
    router_backward_kernel(const RouterBackwardArgs a) {
  constexpr int EPL = TM::EPL, L = TM::L;
  extern __shared__ __align__(16) uint8_t router_smem[];
  __shared__ float red[kTeamWarps];
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int E = a.E, r = TM::rank();
  const int team = TM::kBlock ? 0 : threadIdx.x / L;
  const int Epad = (E + 3) / 4 * 4;
  float* g = reinterpret_cast<float*>(router_smem) + static_cast<size_t>(team) * Epad;  // dL/ds of the selected experts
  auto far_steps = [&]() {  // a bit per step of the team: its far tokens
    return reinterpret_cast<unsigned*>(router_smem) + 256 / L * ((a.E + 3) / 4 * 4) +
           (TM::kBlock ? 0 : threadIdx.x / L) * ((a.per_team + 31) >> 5);
  };
  for (int e = r; e < Epad; e += L) g[e] = 0.0f;
  for (int i = r; i < (a.per_team + 31) >> 5; i += L) far_steps()[i] = 0;
  TM::sync();
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const long long t0 = (static_cast<long long>(blockIdx.x) * (256 / L) + team) * a.per_team;
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
    in_nxt = t < t1 && (!a.mask || a.mask[t]);
    id_nxt = -1;
    w_nxt = 0.0f;
    if (t < t1) {
      TM::load(a.logits + t * a.ld, E, neg_inf(), nxt);
      if (a.dw && r < a.k) {
        id_nxt = a.ids[t * a.k + r];
        w_nxt = a.dw[t * a.k + r];
      }
    } else {
#pragma unroll
      for (int i = 0; i < EPL; ++i) nxt[i] = 0.0f;
    }
  };
  fetch(t0);
  int q = -1;
  long long q_end = t0;  // where the sequence q ends
  for (int step = 0; step < a.per_team; ++step) {  // the teams of a warp in step
    const long long t = t0 + step;
    const bool here = t < t1;
    float l[EPL], ex[EPL], s[EPL], d[EPL];
#pragma unroll
    for (int i = 0; i < EPL; ++i) l[i] = nxt[i];
    const int id0 = id_nxt >= 0 && id_nxt < E ? id_nxt : -1;
    const float w0 = w_nxt;
    bool in = in_nxt;
    const float le0 = id0 >= 0 ? a.logits[t * a.ld + id0] : 0.0f;
    fetch(t + 1);
    if (here && t >= q_end) {
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
    in = in && q >= 0 && q < a.S;
    bool far = false;
    float dl[EPL];
    if (TM::kBlock ? in : __any_sync(0xFFFFFFFFu, in)) {
      // exponentials, where the score or the z loss wants them
      float base = 0.0f, inv = 0.0f, lse = 0.0f;
      bool direct = false;
      if (FUNC != kSqrtSoftplus || zc != 0.0f) {
        const float sum = exponentials<TM>(l, ex, red, &base, &direct);
        inv = sum == 0.0f ? 0.0f : rcp_sfu(sum);  // a row of -inf: no probabilities, no gradient
        if (zc != 0.0f) lse = sum == 0.0f ? 0.0f : base + __logf(sum);
      }
      // scores and their derivatives
      if (FUNC == kSigmoid && direct) {
#pragma unroll
        for (int i = 0; i < EPL; ++i) {
          const float rc = rcp_sfu(1.0f + ex[i]);
          s[i] = ex[i] * rc;
          d[i] = s[i] * rc;
        }
      } else if (FUNC != kSoftmax) {
#pragma unroll
        for (int i = 0; i < EPL; ++i) {
          d[i] = 0.0f;
          s[i] = TM::expert(i, r) < E ? score_of(FUNC, l[i], &d[i]) : 0.0f;
        }
      }
      __syncwarp();
      // dL/ds of the selected experts, scattered into g
      if (a.dw) {
        auto score_at = [&](float le) {
          float dd;
          return FUNC == kSoftmax ? exp_sfu(le - base) * inv : score_of(FUNC, le, &dd);
        };
        float c = a.route_scale, mean = 0.0f, rest = 0.0f;
        if (a.renorm) {
          // less the weights' mean by score, and less the mean of what that
          // leaves: what all slots have alike cancels before it is rounded
          // (one slot: to nothing, beside the small gradients of the losses)
          const float q0 = id0 >= 0 ? score_at(le0) : 0.0f;
          auto sums = [&](float less, float* Q) {
            float q = q0, wq = id0 >= 0 ? q0 * (w0 - less) : 0.0f;
            for (int j = r + L; j < a.k; j += L) {
              const int e = here ? a.ids[t * a.k + j] : -1;
              if (e >= 0 && e < E) {
                const float v = score_at(a.logits[t * a.ld + e]);
                q += v;
                wq = fmaf(a.dw[t * a.k + j] - less, v, wq);
              }
            }
            __syncwarp();
            if (Q) *Q = TM::sum(q, red);
            return TM::sum(wq, red);
          };
          float Q;
          const float wq = sums(0.0f, &Q);
          const float iq = Q > 0.0f ? rcp_sfu(Q) : 0.0f;  // as the gate: a sum of 0 divides nothing
          mean = wq * iq;
          rest = sums(mean, nullptr) * iq;
          if (Q > 0.0f) c *= iq;
          far = FUNC != kSqrtSoftplus && in && Q < 1e-30f;
        }
        // a team's (a block's first warp's) slots at a time; equal ids among them are added in slot order
        constexpr int W = TM::kBlock ? 32 : L;
        if (!TM::kBlock || threadIdx.x < 32) {
          const int slot = threadIdx.x & (W - 1);
          for (int j0 = 0; j0 < a.k; j0 += W) {
            int e = id0;
            float v = w0;
            if (j0) {
              const int j = j0 + slot;
              e = here && j < a.k ? a.ids[t * a.k + j] : -1;
              if (e < 0 || e >= E) e = -1;
              v = e >= 0 ? a.dw[t * a.k + j] : 0.0f;
            }
            v = c * ((v - mean) - rest);
            const unsigned same = __match_any_sync(0xFFFFFFFFu, e) & TM::lanes();
            if (__all_sync(0xFFFFFFFFu, (same & (same - 1)) == 0 || e < 0)) {
              if (e >= 0) g[e] += v;
            } else {
              for (int i = 0; i < W; ++i) {
                if (slot == i && e >= 0) g[e] += v;
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
        for (int j = r + L; j < a.k; j += L) {
          const int e = here ? a.ids[t * a.k + j] : -1;
          if (e >= 0 && e < E) g[e] = 0.0f;
        }
        TM::sync();
      } else {
#pragma unroll
        for (int i = 0; i < EPL; ++i) dl[i] = 0.0f;
      }
      if (FUNC == kSoftmax) {
        float dot = 0.0f;
#pragma unroll
        for (int i = 0; i < EPL; ++i) {
          dl[i] += B[i];
          dot = fmaf(dl[i], ex[i], dot);
        }
        dot = TM::sum(dot, red) * inv;
        const float shift = fmaf(zc, lse, -dot);
#pragma unroll
        for (int i = 0; i < EPL; ++i) dl[i] = ex[i] * inv * (dl[i] + shift);
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
          const float is = ssum == 0.0f ? 0.0f : rcp_sfu(ssum);
          const float less = bsum * is * is;
#pragma unroll
          for (int i = 0; i < EPL; ++i) dl[i] += fmaf(B[i], is, -less);
        }
        if (zc != 0.0f) {
          const float zl = zc * lse * inv;
#pragma unroll
          for (int i = 0; i < EPL; ++i) dl[i] = fmaf(dl[i], d[i], zl * ex[i]);
        } else {
#pragma unroll
          for (int i = 0; i < EPL; ++i) dl[i] *= d[i];
        }
      }
    }
    if (!in) {
#pragma unroll
      for (int i = 0; i < EPL; ++i) dl[i] = 0.0f;
    }
    if (here && !far) {
      float* o = a.out + t * a.ld_out;
      if constexpr (TM::kQuads) {
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
    if (far && TM::rank() == 0) far_steps()[step >> 5] |= 1u << (step & 31);
  }
  if (FUNC != kSqrtSoftplus) {
    TM::sync();
    for (int step = 0; step < a.per_team; step += 32) {
      const unsigned word = far_steps()[step >> 5];
      if (TM::kBlock ? word != 0 : __any_sync(0xFFFFFFFFu, word))
        for (int i = 0; i < 32; ++i) {
          const bool mine = word >> i & 1;
          if (TM::kBlock ? mine : __any_sync(0xFFFFFFFFu, mine)) far_token<TM, FUNC>(a, t0 + step + i, mine, g, red);
        }
    }
  }
}

}  // namespace dev

int launch_router_backward(dev::RouterBackwardArgs a, bool v4, const DeviceProps& props, cudaStream_t st) {
  return with_team<16>(a.E, v4, [&](auto tm) {
    return with_func(a.func, [&](auto func) {
      using TM = decltype(tm);
      const size_t teams = 256 / TM::L;
      // up to three blocks per SM (what the registers allow), each team a run of consecutive tokens
      const size_t most = static_cast<size_t>(TM::EPL <= 8 ? 3 : TM::EPL <= 16 ? 2 : 1) * props.sm_count * teams;
      // of 1024 at most (a bit of shared memory each), in rounds of even length
      const size_t rounds = (static_cast<size_t>(a.T) + most * 1024 - 1) / (most * 1024);
      a.per_team = static_cast<int>((static_cast<size_t>(a.T) + most * rounds - 1) / (most * rounds));
      const size_t per_block = teams * a.per_team;
      const size_t smem = teams * ((static_cast<size_t>(a.E) + 3) / 4 * 4 + (a.per_team + 31) / 32) * 4;
      return launch_pdl(dev::router_backward_kernel<TM, decltype(func)::value>,
                        static_cast<int>((static_cast<size_t>(a.T) + per_block - 1) / per_block), 256, smem, st, a);
    });
  });
}

}  // namespace objb
