// linear.cu -- dense products of many tokens: y = act(x w^T + b) + r, its
// gradients, and the bf16 SwiGLU FFN (shared expert) built on it.
//
// Every product is D[n][m] = sum_k A(m, k) B(n, k), D row-major with m
// innermost:
//   y  [t][o]: A = w [o][i],       B = x  [t][i],       k = i
//   dx [t][i]: A = w^T (k rows),   B = dz [t][o],       k = o
//   dw [o][i]: A = x^T (k rows),   B = dz^T (k rows),   k = t
#include <cuda_runtime.h>

#include <algorithm>
#include <string>

#include "objb_common.h"
#include "objb_host_launch.cuh"
#include "objb_launch.h"
#include "objb_linear.cuh"
#include "objb_moe.cuh"

namespace objb {
namespace dev {

// An operand in memory: element (row, k) at row * ld + k, or k * ld + row
// where k runs over the memory's rows.
struct Operand {
  const void* p;
  size_t ld;
  int dtype;
  bool k_rows;
};

__device__ __forceinline__ float operand_at(const Operand& o, size_t row, size_t k) {
  return load_elem(o.p, o.dtype, o.k_rows ? k * o.ld + row : row * o.ld + k);
}

// 64 x 64 tile, 16 x 16 threads of 4 x 4 elements, 16 of k at a time.
__global__ void __launch_bounds__(256) gemm_kernel(const Operand A, const Operand B, int M, long long N, long long K,
                                                   const LinearEpilogue epi) {
  __shared__ float as[16][65], bs[16][65];
  const int m0 = blockIdx.x * 64;
  const long long n0 = static_cast<long long>(blockIdx.y) * 64;
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  float acc[4][4] = {};
  for (long long k0 = 0; k0 < K; k0 += 16) {
    for (int i = threadIdx.x; i < 64 * 16; i += 256) {
      const int ra = A.k_rows ? i & 63 : i >> 4, ka = A.k_rows ? i >> 6 : i & 15;
      const int rb = B.k_rows ? i & 63 : i >> 4, kb = B.k_rows ? i >> 6 : i & 15;
      as[ka][ra] = m0 + ra < M && k0 + ka < K ? operand_at(A, m0 + ra, k0 + ka) : 0.0f;
      bs[kb][rb] = n0 + rb < N && k0 + kb < K ? operand_at(B, n0 + rb, k0 + kb) : 0.0f;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 16; ++k)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(as[k][tx + 16 * j], bs[k][ty + 16 * i], acc[i][j]);
    __syncthreads();
  }
  for (int i = 0; i < 4; ++i)
    for (int j = 0; j < 4; ++j) {
      const int m = m0 + tx + 16 * j;
      const long long n = n0 + ty + 16 * i;
      if (m < M && n < N) epi.put(m, n, acc[i][j]);
    }
}

// dz = dy act'(z), rounded to dz's type, and column sums of runs of rows.
__global__ void __launch_bounds__(256) dz_kernel(const void* dy, size_t ldy, const void* z, size_t ldz, int dtype,
                                                 int act, long long T, int N, void* dz, int dz_dtype,
                                                 long long rows_per, float* part) {
  const int c = blockIdx.x * 256 + threadIdx.x;
  if (c >= N) return;
  const long long r0 = blockIdx.y * rows_per, r1 = r0 + rows_per < T ? r0 + rows_per : T;
  float s = 0.0f;
  for (long long r = r0; r < r1; ++r) {
    float v = load_elem(dy, dtype, r * ldy + c);
    if (act != OBJB_ACT_NONE) v *= act_grad(act, load_elem(z, dtype, r * ldz + c));
    if (dz) store_elem(dz, dz_dtype, r * N + c, v);
    s += v;
  }
  if (part) part[static_cast<size_t>(blockIdx.y) * N + c] = s;
}

__global__ void __launch_bounds__(256) dbias_kernel(const float* part, int parts, int N, float* db, int accumulate) {
  const int c = blockIdx.x * 256 + threadIdx.x;
  if (c >= N) return;
  float s = 0.0f;
  for (int i = 0; i < parts; ++i) s += part[static_cast<size_t>(i) * N + c];
  db[c] = accumulate ? db[c] + s : s;
}

__global__ void __launch_bounds__(256) swiglu_kernel(const float* g, const float* u, float* act, size_t n,
                                                     float limit) {
  const size_t i = static_cast<size_t>(blockIdx.x) * 256 + threadIdx.x;
  if (i < n) act[i] = swiglu(g[i], u[i], limit);
}

}  // namespace dev

namespace {

constexpr size_t kMaxSize = size_t{1} << 24;    // in / out features
constexpr size_t kMaxTokens = size_t{1} << 30;

size_t r256(size_t b) { return (b + 255) / 256 * 256; }
size_t elem_bytes(int dtype) { return dtype == OBJB_DTYPE_F32 ? 4 : 2; }

int gemm(const dev::Operand& A, const dev::Operand& B, size_t M, size_t N, size_t K, const dev::LinearEpilogue& e,
         cudaStream_t st) {
  const dim3 grid(static_cast<unsigned>((M + 63) / 64), static_cast<unsigned>((N + 63) / 64));
  dev::gemm_kernel<<<grid, 256, 0, st>>>(A, B, static_cast<int>(M), static_cast<long long>(N),
                                         static_cast<long long>(K), e);
  OBJB_CUDA(cudaGetLastError(), "launch dense product");
  return OBJB_OK;
}

int check_sizes(const char* action, size_t T, size_t K, size_t N, int act) {
  if (T > kMaxTokens || K == 0 || K > kMaxSize || N == 0 || N > kMaxSize)
    return OBJB_FAIL(OBJB_ERR_INVALID_INPUT, action,
                     "need tokens <= 2^30 and 1 <= in_features, out_features <= 2^24 (got " + std::to_string(T) +
                         ", " + std::to_string(K) + ", " + std::to_string(N) + ")");
  if (act < OBJB_ACT_NONE || act > OBJB_ACT_GELU_TANH)
    return OBJB_FAIL(OBJB_ERR_INVALID_INPUT, action, "unknown activation " + std::to_string(act));
  return OBJB_OK;
}

// x and w both bf16, both f16, f32 with bf16, or both f32; y f32 or x's type.
int check_types(const char* action, int x, int w, int y, const char* y_name) {
  const bool half = x == OBJB_DTYPE_BF16 || x == OBJB_DTYPE_F16;
  const bool ok = half ? w == x : x == OBJB_DTYPE_F32 && (w == OBJB_DTYPE_F32 || w == OBJB_DTYPE_BF16);
  if (!ok)
    return OBJB_FAIL(OBJB_ERR_UNSUPPORTED, action,
                     "x and w are both bf16, both f16, f32 with bf16, or both f32 (got dtypes " + std::to_string(x) +
                         " and " + std::to_string(w) + ")");
  if (y != OBJB_DTYPE_F32 && !(half && y == x))
    return OBJB_FAIL(OBJB_ERR_UNSUPPORTED, action, std::string(y_name) + " is f32, or x's type where that has 16 bits");
  return OBJB_OK;
}

int check_stride(const char* action, const char* name, size_t stride, size_t cols, size_t* out) {
  *out = stride ? stride : cols;
  if (*out < cols)
    return OBJB_FAIL(OBJB_ERR_INVALID_INPUT, action, std::string(name) + " is below the row's " + std::to_string(cols) +
                                                         " elements");
  return OBJB_OK;
}

// The caller's scratch, or the stream's workspace.
int take_scratch(const char* action, void* d_scratch, size_t have, size_t need, cudaStream_t st, uint8_t** out) {
  void* ws = d_scratch;
  if (ws) {
    if (have < need || (reinterpret_cast<uintptr_t>(ws) & 255u))
      return OBJB_FAIL(OBJB_ERR_INVALID_INPUT, action,
                       "scratch needs " + std::to_string(need) + " bytes, 256-byte aligned (got " +
                           std::to_string(have) + ")");
  } else {
    int device = 0;
    OBJB_TRY(current_device(&device));
    OBJB_TRY(workspace_get(device, st, need, &ws));
  }
  *out = static_cast<uint8_t*>(ws);
  return OBJB_OK;
}

int check_linear(const char* action, const objb_linear_desc* d) {
  if (!d) return OBJB_FAIL(OBJB_ERR_INVALID_INPUT, action, "null descriptor");
  if (d->reserved) return OBJB_FAIL(OBJB_ERR_INVALID_INPUT, action, "reserved must be 0");
  OBJB_TRY(check_sizes(action, d->tokens, d->in_features, d->out_features, d->activation));
  return check_types(action, d->x_dtype, d->w_dtype, d->y_dtype, "y");
}

int check_backward(const char* action, const objb_linear_backward_desc* d) {
  if (!d) return OBJB_FAIL(OBJB_ERR_INVALID_INPUT, action, "null descriptor");
  if (d->reserved) return OBJB_FAIL(OBJB_ERR_INVALID_INPUT, action, "reserved must be 0");
  OBJB_TRY(check_sizes(action, d->tokens, d->in_features, d->out_features, d->activation));
  OBJB_TRY(check_types(action, d->x_dtype, d->w_dtype, d->dy_dtype, "dy"));
  if (d->x_dtype == OBJB_DTYPE_F16 && d->dy_dtype == OBJB_DTYPE_F32)
    return OBJB_FAIL(OBJB_ERR_UNSUPPORTED, action, "f32 dy with f16 x");
  if (d->dw_dtype != OBJB_DTYPE_F32 && d->dw_dtype != d->w_dtype)
    return OBJB_FAIL(OBJB_ERR_UNSUPPORTED, action, "dw is f32 or w's type");
  if ((d->outputs & ~7) || !d->outputs)
    return OBJB_FAIL(OBJB_ERR_INVALID_INPUT, action, "outputs must name at least one of dx, dw and dbias");
  return OBJB_OK;
}

struct BackwardPlan {
  int parts;
  long long rows_per;
  size_t dz, part, total;
  int dz_dtype;
};
BackwardPlan plan_backward(const objb_linear_backward_desc* d) {
  BackwardPlan p;
  p.parts = static_cast<int>(std::max<size_t>(1, std::min<size_t>(64, (d->tokens + 63) / 64)));
  p.rows_per = static_cast<long long>((d->tokens + p.parts - 1) / p.parts);
  p.dz_dtype = d->dw_dtype == OBJB_DTYPE_F32 ? OBJB_DTYPE_F32 : d->dy_dtype;
  p.dz = 0;
  p.part = r256(d->tokens * d->out_features * elem_bytes(p.dz_dtype));
  p.total = p.part + r256(static_cast<size_t>(p.parts) * d->out_features * 4);
  return p;
}

}  // namespace
}  // namespace objb

using namespace objb;

extern "C" {

int objb_linear_scratch_bytes(const objb_linear_desc* desc, size_t* bytes) {
  clear_error();
  OBJB_TRY(check_linear("objb_linear_scratch_bytes", desc));
  if (!bytes) return OBJB_FAIL(OBJB_ERR_INVALID_INPUT, "objb_linear_scratch_bytes", "null output pointer");
  *bytes = 0;
  return OBJB_OK;
}

int objb_linear_device(const objb_linear_desc* desc, const void* d_x, const void* d_w, const void* d_bias,
                       const void* d_residual, void* d_y, void* d_z, void* d_scratch, size_t scratch_bytes,
                       objb_stream_t stream) {
  clear_error();
  const char* action = "objb_linear_device";
  OBJB_TRY(check_linear(action, desc));
  const objb_linear_desc& d = *desc;
  if (d_bias && d.bias_dtype != OBJB_DTYPE_F32 && d.bias_dtype != d.w_dtype)
    return OBJB_FAIL(OBJB_ERR_UNSUPPORTED, action, "bias is f32 or w's type");
  size_t ldx, ldw, ldy, ldr, ldz;
  OBJB_TRY(check_stride(action, "x_stride", d.x_stride, d.in_features, &ldx));
  OBJB_TRY(check_stride(action, "w_stride", d.w_stride, d.in_features, &ldw));
  OBJB_TRY(check_stride(action, "y_stride", d.y_stride, d.out_features, &ldy));
  OBJB_TRY(check_stride(action, "residual_stride", d.residual_stride, d.out_features, &ldr));
  OBJB_TRY(check_stride(action, "z_stride", d.z_stride, d.out_features, &ldz));
  if (d.tokens == 0) return OBJB_OK;
  if (!d_x || !d_w || !d_y) return OBJB_FAIL(OBJB_ERR_INVALID_INPUT, action, "null device pointer");
  if (d_residual == d_y && ldr != ldy)
    return OBJB_FAIL(OBJB_ERR_INVALID_INPUT, action, "a residual in place needs y's stride");
  (void)d_scratch;
  (void)scratch_bytes;
  dev::LinearEpilogue e;
  e.bias = d_bias;
  e.bias_dtype = d.bias_dtype;
  e.residual = d_residual;
  e.ldr = ldr;
  e.y = d_y;
  e.ldy = ldy;
  e.z = d_z;
  e.ldz = ldz;
  e.y_dtype = d.y_dtype;
  e.act = d.activation;
  return gemm({d_w, ldw, d.w_dtype, false}, {d_x, ldx, d.x_dtype, false}, d.out_features, d.tokens, d.in_features, e,
              static_cast<cudaStream_t>(stream));
}

int objb_linear_backward_scratch_bytes(const objb_linear_backward_desc* desc, size_t* bytes) {
  clear_error();
  OBJB_TRY(check_backward("objb_linear_backward_scratch_bytes", desc));
  if (!bytes) return OBJB_FAIL(OBJB_ERR_INVALID_INPUT, "objb_linear_backward_scratch_bytes", "null output pointer");
  *bytes = plan_backward(desc).total;
  return OBJB_OK;
}

int objb_linear_backward_device(const objb_linear_backward_desc* desc, const void* d_dy, const void* d_z,
                                const void* d_x, const void* d_w, void* d_dx, void* d_dw, float* d_dbias,
                                void* d_scratch, size_t scratch_bytes, objb_stream_t stream) {
  clear_error();
  const char* action = "objb_linear_backward_device";
  OBJB_TRY(check_backward(action, desc));
  const objb_linear_backward_desc& d = *desc;
  const bool want_dx = d.outputs & OBJB_LINEAR_DX, want_dw = d.outputs & OBJB_LINEAR_DW,
             want_db = d.outputs & OBJB_LINEAR_DBIAS, has_act = d.activation != OBJB_ACT_NONE;
  size_t lddy, ldz, ldx, ldw, lddx, lddw;
  OBJB_TRY(check_stride(action, "dy_stride", d.dy_stride, d.out_features, &lddy));
  OBJB_TRY(check_stride(action, "z_stride", d.z_stride, d.out_features, &ldz));
  OBJB_TRY(check_stride(action, "x_stride", d.x_stride, d.in_features, &ldx));
  OBJB_TRY(check_stride(action, "w_stride", d.w_stride, d.in_features, &ldw));
  OBJB_TRY(check_stride(action, "dx_stride", d.dx_stride, d.in_features, &lddx));
  OBJB_TRY(check_stride(action, "dw_stride", d.dw_stride, d.in_features, &lddw));
  if ((want_dw && !d_dw) || (want_db && !d_dbias) ||
      (d.tokens && (!d_dy || (has_act && !d_z) || (want_dw && !d_x) || (want_dx && (!d_w || !d_dx)))))
    return OBJB_FAIL(OBJB_ERR_INVALID_INPUT, action, "null device pointer");
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (d.tokens == 0) {  // sums over nothing
    if (want_dw && !d.accumulate)
      OBJB_CUDA(cudaMemset2DAsync(d_dw, lddw * elem_bytes(d.dw_dtype), 0, d.in_features * elem_bytes(d.dw_dtype),
                                  d.out_features, st),
                "clear dw");
    if (want_db && !d.accumulate) OBJB_CUDA(cudaMemsetAsync(d_dbias, 0, d.out_features * 4, st), "clear dbias");
    return OBJB_OK;
  }
  const BackwardPlan p = plan_backward(desc);
  uint8_t* ws = nullptr;
  OBJB_TRY(take_scratch(action, d_scratch, scratch_bytes, p.total, st, &ws));
  const int N = static_cast<int>(d.out_features);
  const unsigned cols = (N + 255) / 256;
  dev::dz_kernel<<<dim3(cols, p.parts), 256, 0, st>>>(d_dy, lddy, d_z, ldz, d.dy_dtype, d.activation,
                                                      static_cast<long long>(d.tokens), N, ws + p.dz, p.dz_dtype,
                                                      p.rows_per, reinterpret_cast<float*>(ws + p.part));
  OBJB_CUDA(cudaGetLastError(), "launch dz");
  if (want_db) {
    dev::dbias_kernel<<<cols, 256, 0, st>>>(reinterpret_cast<float*>(ws + p.part), p.parts, N, d_dbias, d.accumulate);
    OBJB_CUDA(cudaGetLastError(), "launch dbias");
  }
  if (want_dx) {
    dev::LinearEpilogue e;
    e.y = d_dx;
    e.ldy = lddx;
    e.y_dtype = d.x_dtype;
    OBJB_TRY(gemm({d_w, ldw, d.w_dtype, true}, {ws + p.dz, d.out_features, p.dz_dtype, false}, d.in_features,
                  d.tokens, d.out_features, e, st));
  }
  if (want_dw) {
    dev::LinearEpilogue e;
    e.y = d_dw;
    e.ldy = lddw;
    e.y_dtype = d.dw_dtype;
    if (d.accumulate) e.residual = d_dw, e.ldr = lddw;
    OBJB_TRY(gemm({d_x, ldx, d.x_dtype, true}, {ws + p.dz, d.out_features, p.dz_dtype, true}, d.in_features,
                  d.out_features, d.tokens, e, st));
  }
  return OBJB_OK;
}

static int check_ffn(const char* action, size_t T, size_t H, size_t I, size_t O) {
  OBJB_TRY(check_sizes(action, T, H, I, 0));
  return check_sizes(action, T, I, O, 0);
}

int objb_ffn_bf16_tokens_scratch_bytes(size_t num_tokens, size_t hidden, size_t intermediate, size_t out_dim,
                                       size_t* bytes) {
  clear_error();
  OBJB_TRY(check_ffn("objb_ffn_bf16_tokens_scratch_bytes", num_tokens, hidden, intermediate, out_dim));
  if (!bytes) return OBJB_FAIL(OBJB_ERR_INVALID_INPUT, "objb_ffn_bf16_tokens_scratch_bytes", "null output pointer");
  *bytes = 2 * r256(num_tokens * intermediate * 4);
  return OBJB_OK;
}

int objb_ffn_bf16_tokens_device(const void* d_gate, const void* d_up, const void* d_down, size_t hidden,
                                size_t intermediate, size_t out_dim, const float* d_x, size_t num_tokens,
                                const float* d_residual, float* d_out, float swiglu_limit, void* d_scratch,
                                size_t scratch_bytes, objb_stream_t stream) {
  clear_error();
  const char* action = "objb_ffn_bf16_tokens_device";
  OBJB_TRY(check_ffn(action, num_tokens, hidden, intermediate, out_dim));
  if (num_tokens == 0) return OBJB_OK;
  if (!d_gate || !d_up || !d_down || !d_x || !d_out)
    return OBJB_FAIL(OBJB_ERR_INVALID_INPUT, action, "null device pointer");
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  uint8_t* ws = nullptr;
  const size_t half = r256(num_tokens * intermediate * 4);
  OBJB_TRY(take_scratch(action, d_scratch, scratch_bytes, 2 * half, st, &ws));
  float* g = reinterpret_cast<float*>(ws);
  float* u = reinterpret_cast<float*>(ws + half);
  dev::LinearEpilogue e;
  e.y_dtype = OBJB_DTYPE_F32;
  e.ldy = intermediate;
  const dev::Operand x{d_x, hidden, OBJB_DTYPE_F32, false};
  e.y = g;
  OBJB_TRY(gemm({d_gate, hidden, OBJB_DTYPE_BF16, false}, x, intermediate, num_tokens, hidden, e, st));
  e.y = u;
  OBJB_TRY(gemm({d_up, hidden, OBJB_DTYPE_BF16, false}, x, intermediate, num_tokens, hidden, e, st));
  const size_t n = num_tokens * intermediate;
  dev::swiglu_kernel<<<static_cast<unsigned>((n + 255) / 256), 256, 0, st>>>(g, u, g, n, swiglu_limit);
  OBJB_CUDA(cudaGetLastError(), "launch SwiGLU");
  e.y = d_out;
  e.ldy = out_dim;
  e.residual = d_residual;
  e.ldr = out_dim;
  return gemm({d_down, intermediate, OBJB_DTYPE_BF16, false}, {g, intermediate, OBJB_DTYPE_F32, false}, out_dim,
              num_tokens, intermediate, e, st);
}

}  // extern "C"
