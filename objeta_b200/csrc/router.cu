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

#include "objb_router.cuh"
#include "objb_router_finish.cuh"

namespace objb {
namespace dev {

// About 6 us of latencies (its launch, the partial rows, the fence and ticket of
// the last block, the losses), whatever the sizes.
constexpr int kFinishWarps = 32;

__global__ void __launch_bounds__(32 * kFinishWarps) balance_finish_kernel(const BalanceFinishArgs f) {
  __shared__ FinishSmem<kFinishWarps> sm;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  balance_finish(f, sm, kFinishGrid);
}

// dw[t, j] = sum_o dout[t, o] v[slot_row[t, j], o]: WPS warps per slot, each
// lane four partial sums (the quads of its columns), folded in a fixed order.
// Bound by the value rows: 4096 tokens x 8 of 2048 take 48 to 49 us, 6.2 TB/s.
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
  int mode;
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
  if (S * ((E + 31) / 32) > (1u << 30))
    return OBJB_FAIL(OBJB_ERR_INVALID_INPUT, action, "num_seqs * num_experts is above 2^35");
  return OBJB_OK;
}

// Blocks of the partial pass: three per SM at most (what its registers allow),
// 16 tokens or more in each (4 in up to 128 blocks that are one team each: 8192
// experts, 16 tokens 40 -> 28 us).  Few tokens of few experts and sequences need
// no second launch: one block does the finish too (64 experts: 5.7 us), or a
// cluster of eight does both while a thread team has at most 16 tokens of 8
// experts a lane (256 experts, 16 tokens: 6.1 us, alone 10.5; a call's time with
// 4096 tokens of 64: 13.0, in two launches 16.9; 2048 of 256: 20.9 and 16.4).
BalancePlan plan_balance(size_t T, size_t E, size_t S, int sms) {
  BalancePlan p;
  const size_t most = static_cast<size_t>(3) * sms;
  const size_t items = S * ((E + 31) / 32), cluster = dev::kFinishCluster;
  const size_t team = E <= 64 ? 8 : E <= 128 ? 16 : E <= 1024 ? 32 : 256;         // threads of a token
  const size_t lane = E <= 256 ? 8 : E <= 512 ? 16 : 32;                          // experts of a thread
  const bool few = T * lane * team <= 16 * 8 * 256 * cluster && items <= 8 * cluster;
  p.mode = T <= 128 && items <= 2 ? dev::kFinishAlone : few ? dev::kFinishInCluster : dev::kFinishGrid;
  size_t blocks = (T + 15) / 16;
  if (team == 256) blocks = std::max(blocks, std::min<size_t>(128, (T + 3) / 4));
  const size_t want = p.mode == dev::kFinishAlone ? 1 : p.mode == dev::kFinishInCluster ? cluster : std::min(most, blocks);
  p.chunk = static_cast<long long>(std::max<size_t>(1, T ? (T + want - 1) / want : 0));
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
  f.mode = p.mode;
  f.bal_part = reinterpret_cast<double*>(b + p.bal);
  f.seq_z = reinterpret_cast<double*>(b + p.seqz);
  f.counts = d_counts;
  f.tokens = d_seq_tokens;
  f.losses = d_losses;
  f.scales = d_scales;
  const bool v4 = aligned16(d_logits) && ld % 4 == 0 && num_experts % 4 == 0;
  const int grid = p.mode == dev::kFinishInCluster ? dev::kFinishCluster : static_cast<int>(std::max<size_t>(1, p.chunks));
  OBJB_TRY(launch_balance_partial(f, grid, v4, st));
  if (f.mode != dev::kFinishGrid) return OBJB_OK;
  return launch_pdl(dev::balance_finish_kernel, static_cast<int>(num_seqs * p.groups), 32 * dev::kFinishWarps, 0, st, f);
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
  {
    const size_t T = num_tokens, E = num_experts, slots = T * top_k * 4, nc = num_seqs * E * 4, ns = (num_seqs + 1) * 4;
    const Rows out{d_dlogits, T, E * 4, ldo * 4};
    if ((d_logits != d_dlogits && overlap(out, {d_logits, T, E * 4, ld * 4})) || overlap(out, {d_ids, 1, slots, slots}) ||
        overlap(out, {d_dweights, 1, slots, slots}) || overlap(out, {d_counts, 1, nc, nc}) ||
        overlap(out, {d_scales, 1, ns, ns}) || overlap(out, {d_seq_offsets, 1, ns, ns}) || overlap(out, {d_token_mask, 1, T, T}))
      return OBJB_FAIL(OBJB_ERR_INVALID_INPUT, action, "dlogits overlaps an operand without being the logits");
  }
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
  return launch_router_backward(a, v4, props, static_cast<cudaStream_t>(stream));
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
  {
    const size_t n = num_tokens * top_k * 4, o = num_tokens * out_dim * 4, v = v_rows * out_dim * 4;
    const Rows out{d_dweights, 1, n, n};
    if (overlap(out, {d_dout, 1, o, o}) || overlap(out, {d_v, 1, v, v}) || overlap(out, {d_slot_row, 1, n, n}))
      return OBJB_FAIL(OBJB_ERR_INVALID_INPUT, action, "dweights overlaps an operand");
  }
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
