// linear.cu -- dense products of many tokens: y = act(x w^T + b) + r, its
// gradients, and the bf16 SwiGLU FFN (shared expert) built on it.
//
// Every product is D[n][m] = sum_k A(m, k) B(n, k), D row-major with m
// innermost:
//   y  [t][o]: A = w [o][i],       B = x  [t][i],       k = i
//   dx [t][i]: A = w^T (k rows),   B = dz [t][o],       k = o
//   dw [o][i]: A = x^T (k rows),   B = dz^T (k rows),   k = t
#include <cuda.h>
#include <cudaTypedefs.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <mutex>
#include <string>

#include "objb_common.h"
#include "objb_host_launch.cuh"
#include "objb_launch.h"
#include "objb_linear_gemm.cuh"

namespace objb {
namespace dev {

// 8 neighbouring elements as f32; VEC: their address is 16-byte aligned.
template <bool VEC>
__device__ __forceinline__ void load8(const void* p, int dtype, size_t at, int n, float (&v)[8]) {
  if constexpr (VEC) {
    if (n >= 8) {
      if (dtype == OBJB_DTYPE_F32) {
        const float4* q = reinterpret_cast<const float4*>(static_cast<const float*>(p) + at);
        const float4 a = q[0], b = q[1];
        v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
      } else {
        const uint4 q = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p) + at);
        const uint32_t u[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const uint16_t h = static_cast<uint16_t>(u[i >> 1] >> (16 * (i & 1)));
          v[i] = dtype == OBJB_DTYPE_BF16 ? __uint_as_float(static_cast<uint32_t>(h) << 16)
                                          : __half2float(__ushort_as_half(h));
        }
      }
      return;
    }
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = i < n ? load_elem(p, dtype, at + i) : 0.0f;
}

// 8 elements of an image row (its pitch is a whole number of 16-byte quads):
// one plane of `dtype`, or the first `planes` bf16 parts.
__device__ __forceinline__ void store_image8(uint16_t* img, size_t plane, size_t at, int planes, int dtype,
                                             const float (&v)[8]) {
  uint32_t u[3][4] = {};
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    uint16_t h[3] = {};
    if (planes == 1) {
      h[0] = dtype == OBJB_DTYPE_F16 ? __half_as_ushort(__float2half_rn(v[i]))
                                     : __bfloat16_as_ushort(__float2bfloat16_rn(v[i]));
    } else {
      __nv_bfloat16 b[3];
      split3(v[i], b);
#pragma unroll
      for (int j = 0; j < 3; ++j) h[j] = __bfloat16_as_ushort(b[j]);
    }
#pragma unroll
    for (int j = 0; j < 3; ++j) u[j][i >> 1] |= static_cast<uint32_t>(h[j]) << (16 * (i & 1));
  }
#pragma unroll
  for (int j = 0; j < 3; ++j)
    if (j < planes)
      *reinterpret_cast<uint4*>(img + j * plane + at) = make_uint4(u[j][0], u[j][1], u[j][2], u[j][3]);
}

// An operand laid out for the copy engine: rows of `pitch` elements (a multiple
// of 8), f32 in planes.  8 elements per thread.
template <bool VEC>
__global__ void __launch_bounds__(256) image_kernel(const void* src, int dtype, size_t ld, long long rows, int cols,
                                                    uint16_t* img, int pitch, int planes) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int quads = pitch / 8;
  const long long n = rows * quads;
  for (long long i = blockIdx.x * 256LL + threadIdx.x; i < n; i += gridDim.x * 256LL) {
    const long long r = i / quads;
    const int c = static_cast<int>(i - r * quads) * 8;
    float v[8];
    load8<VEC>(src, dtype, r * ld + c, cols - c, v);
    store_image8(img, rows * static_cast<size_t>(pitch), r * static_cast<size_t>(pitch) + c, planes, dtype, v);
  }
}

// dz = dy act'(z) as an image (may be null: only its sums), and the column
// sums of each run of rows.  A block: 256 columns (8 per thread), 8 rows at a
// time; the 8 row lanes are folded in order.
template <bool VEC>
__global__ void __launch_bounds__(256) dz_kernel(const void* dy, size_t ldy, const void* z, size_t ldz, int dtype,
                                                 int act, long long T, int N, uint16_t* img, int pitch, int planes,
                                                 long long rows_per, float* part) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  __shared__ float sm[8][256];
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  const int c = blockIdx.x * 256 + tx * 8;
  const long long r0 = blockIdx.y * rows_per, r1 = r0 + rows_per < T ? r0 + rows_per : T;
  float s[8] = {};
  if (c < N) {
    for (long long r = r0 + ty; r < r1; r += 8) {
      float v[8];
      load8<VEC>(dy, dtype, r * ldy + c, N - c, v);
      if (act != OBJB_ACT_NONE) {
        float zz[8];
        load8<VEC>(z, dtype, r * ldz + c, N - c, zz);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] *= act_grad(act, zz[i]);
      }
      if (img) store_image8(img, T * static_cast<size_t>(pitch), r * static_cast<size_t>(pitch) + c, planes, dtype, v);
#pragma unroll
      for (int i = 0; i < 8; ++i) s[i] += v[i];
    }
  }
  if (!part) return;
#pragma unroll
  for (int i = 0; i < 8; ++i) sm[ty][tx * 8 + i] = s[i];
  __syncthreads();
  const int col = blockIdx.x * 256 + threadIdx.x;
  if (col >= N) return;
  float sum = 0.0f;
#pragma unroll
  for (int i = 0; i < 8; ++i) sum += sm[i][threadIdx.x];
  part[static_cast<size_t>(blockIdx.y) * N + col] = sum;
}

__global__ void __launch_bounds__(256) dbias_kernel(const float* part, int parts, int N, float* db, int accumulate) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int c = blockIdx.x * 256 + threadIdx.x;
  if (c >= N) return;
  float s = 0.0f;
#pragma unroll 8
  for (int i = 0; i < parts; ++i) s += part[static_cast<size_t>(i) * N + c];
  db[c] = accumulate ? db[c] + s : s;
}

}  // namespace dev

namespace {

constexpr size_t kMaxSize = size_t{1} << 24;    // in / out features
constexpr size_t kMaxTokens = size_t{1} << 30;

size_t r256(size_t b) { return (b + 255) / 256 * 256; }
size_t elem_bytes(int dtype) { return dtype == OBJB_DTYPE_F32 ? 4 : 2; }

// A 16-bit matrix as the copy engine reads it: 16-byte aligned, rows of `ld`
// elements (a multiple of 8), `planes` of them `rows * ld` apart.
struct Image {
  const void* p = nullptr;
  size_t ld = 0, rows = 0, cols = 0;
  int planes = 1;
  int dtype = 0;  // OBJB_DTYPE_BF16 or F16
};

// How an operand becomes an image: as it lies, or laid out in the scratch.
struct ImagePlan {
  bool direct = false;
  int planes = 1;
  size_t pitch = 0, bytes = 0;
};
ImagePlan plan_image(const void* p, int dtype, size_t ld, size_t rows, size_t cols, int planes) {
  ImagePlan i;
  i.planes = planes;
  i.direct = planes == 1 && dtype != OBJB_DTYPE_F32 && aligned16(p) && ld % 8 == 0;
  i.pitch = i.direct ? ld : (cols + 7) / 8 * 8;
  i.bytes = i.direct ? 0 : r256(static_cast<size_t>(planes) * rows * i.pitch * 2);
  return i;
}

int make_image(const ImagePlan& pl, const void* p, int dtype, size_t ld, size_t rows, size_t cols, void* scratch,
               const DeviceProps& props, cudaStream_t st, Image* out) {
  out->rows = rows;
  out->cols = cols;
  out->planes = pl.planes;
  out->ld = pl.pitch;
  out->dtype = pl.planes > 1 || dtype == OBJB_DTYPE_F32 ? OBJB_DTYPE_BF16 : dtype;
  if (pl.direct) {
    out->p = p;
    return OBJB_OK;
  }
  out->p = scratch;
  const size_t n = rows * (pl.pitch / 8);
  const int grid = static_cast<int>(std::min<size_t>((n + 255) / 256, static_cast<size_t>(props.sm_count) * 16));
  const bool vec = aligned16(p) && ld % 8 == 0;
  auto k = vec ? dev::image_kernel<true> : dev::image_kernel<false>;
  return launch_pdl(k, grid, 256, 0, st, p, dtype, ld, static_cast<long long>(rows), static_cast<int>(cols),
                    static_cast<uint16_t*>(scratch), static_cast<int>(pl.pitch), pl.planes);
}

// The tensor map of an image: box of 64 elements by `box_rows` rows.
int encode(CUtensorMap* map, const Image& im, int box_rows) {
  static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q = cudaDriverEntryPointSymbolNotFound;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
  });
  if (!fn) return OBJB_FAIL(OBJB_ERR_DRIVER, "dense product", "cuTensorMapEncodeTiled is not available");
  const cuuint64_t dims[3] = {im.cols, im.rows, static_cast<cuuint64_t>(im.planes)};
  const cuuint64_t strides[2] = {im.ld * 2, im.rows * im.ld * 2};
  const cuuint32_t box[3] = {64, static_cast<cuuint32_t>(box_rows), 1};
  const cuuint32_t estr[3] = {1, 1, 1};
  const CUresult r =
      fn(map, im.dtype == OBJB_DTYPE_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3,
         const_cast<void*>(im.p), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
         CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS)
    return OBJB_FAIL(OBJB_ERR_DRIVER, "dense product", "cuTensorMapEncodeTiled failed (" + std::to_string(r) + ")");
  return OBJB_OK;
}

struct Product {
  int maj = dev::kMajKK;
  Image a, a2, b;  // a2: the up rows of a gated product
  bool gated = false;
  size_t M = 0, N = 0, K = 0;
  dev::LinearEpilogue epi;
  float swiglu_limit = 0.0f;
};

constexpr size_t kLinRing = 216 * 1024;  // bytes of stages: three of f32 x f32 pair tiles

// A product's tile: rm rows per accumulator, mt accumulators and bn columns
// per CTA or pair, k split over a cluster.
struct Tile {
  int rm = 128, bn = 0, split = 1, chunk_kb = 0;
  size_t ring = kLinRing;
};

template <int MAJ, int BN, int CG, int MT, bool GATED, bool PROMOTE>
int launch_gemm(const Product& p, const Tile& tile, int device, const DeviceProps& props, cudaStream_t st) {
  dev::GemmArgs g;
  g.M = static_cast<int>(p.M);
  g.N = static_cast<long long>(p.N);
  g.nkb = static_cast<int>((p.K + 63) / 64);
  g.pa = p.a.planes;
  g.pb = p.b.planes;
  g.rm = tile.rm;
  g.bn = tile.bn;
  g.split = tile.split;
  g.chunk_kb = PROMOTE ? tile.chunk_kb : g.nkb;
  g.swiglu_limit = p.swiglu_limit;
  g.epi = p.epi;
  OBJB_TRY(device_error_word(device, &g.err));
  const size_t mt = static_cast<size_t>(GATED ? 64 : MT * tile.rm) * CG;
  g.tiles_m = static_cast<int>((p.M + mt - 1) / mt);
  g.tiles_n = static_cast<int>((p.N + tile.bn - 1) / tile.bn);
  const size_t stage = static_cast<size_t>(g.pa) * MT * dev::kLinABlock + static_cast<size_t>(g.pb) * (tile.bn / CG) * 128;
  g.nstages = static_cast<int>(std::max<size_t>(2, std::min<size_t>(dev::kLinStagesMax, tile.ring / stage)));
  size_t smem = g.nstages * stage;
  if (GATED || tile.split > 1) smem = std::max(smem, static_cast<size_t>(MT) * BN * 512);  // the partial tile
  smem += 1024;
  const uint32_t half = p.a.dtype == OBJB_DTYPE_F16 ? 0 : 1;
  g.idesc = (1u << 4) | (half << 7) | (half << 10) | (static_cast<uint32_t>(MAJ != dev::kMajKK) << 15) |
            (static_cast<uint32_t>(MAJ == dev::kMajMN) << 16) | (static_cast<uint32_t>(tile.bn >> 3) << 17) |
            (static_cast<uint32_t>(128 * CG >> 4) << 24);
  CUtensorMap ma, ma2, mb;
  OBJB_TRY(encode(&ma, p.a, MAJ == dev::kMajKK && !GATED ? tile.rm : 64));
  if (GATED)
    OBJB_TRY(encode(&ma2, p.a2, 64));
  else
    ma2 = ma;
  OBJB_TRY(encode(&mb, p.b, MAJ == dev::kMajMN ? 64 : tile.bn / CG));
  auto kernel = dev::lin_gemm_kernel<MAJ, BN, CG, MT, GATED, PROMOTE>;
  OBJB_TRY(ensure_smem_attr(kernel, device, smem));
  const long long tiles = static_cast<long long>(g.tiles_m) * g.tiles_n;
  const int csize = CG == 2 ? 2 : tile.split;
  const bool one_each = GATED || tile.split > 1;
  const long long clusters = one_each ? tiles : std::min<long long>(tiles, props.sm_count / csize);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(clusters * csize));
  cfg.blockDim = dim3(dev::lin_threads(PROMOTE));
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = csize;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = csize > 1 ? 2 : 1;
  OBJB_CUDA(cudaLaunchKernelEx(&cfg, kernel, ma, ma2, mb, g), "launch dense product");
  return OBJB_OK;
}

size_t ceil_div(size_t a, size_t b) { return (a + b - 1) / b; }

// Columns of a pair's tile, 256 or fewer: the count (a multiple of 16) whose
// rounds of the grid take the fewest columns in all.
int pair_columns(size_t tiles_m, size_t N, int most, int step, int pairs) {
  int best = most;
  size_t cost = ~size_t{0};
  for (int bn = most; bn >= most / 2; bn -= step) {
    const size_t c = ceil_div(tiles_m * ceil_div(N, bn), pairs) * bn;
    if (c < cost) cost = c, best = bn;
  }
  return best;
}

// Which tile a product takes.  CTA pairs where their tiles fill most of the
// SMs: 512 x 256 straight from tensor memory for a 16-bit result of one-plane
// operands, else 256 x 128 with promoted accumulators.  Otherwise single CTAs
// of 128 rows by N up to 128, a tile's k split over a cluster while that
// leaves SMs free.
int gemm(const Product& p, int device, const DeviceProps& props, cudaStream_t st) {
  const size_t sms = static_cast<size_t>(props.sm_count);
  const int pairs = props.sm_count / 2;
  const size_t nkb = ceil_div(p.K, 64);
  const bool y16 = !p.gated && p.epi.y_dtype != OBJB_DTYPE_F32;
  const bool plain = p.a.planes == 1 && p.b.planes == 1;
  Tile t;
#define OBJB_GEMM(MAJ, BN, CG, MT, GATED, PROMOTE) return launch_gemm<MAJ, BN, CG, MT, GATED, PROMOTE>(p, t, device, props, st)
  if (y16 && plain && ceil_div(p.M, 512) * ceil_div(p.N, 256) * 4 >= sms) {
    t.bn = pair_columns(ceil_div(p.M, 512), p.N, 256, p.maj == dev::kMajMN ? 128 : 16, pairs);
    switch (p.maj) {
      case dev::kMajKK: OBJB_GEMM(dev::kMajKK, 256, 2, 2, false, false);
      case dev::kMajMK: OBJB_GEMM(dev::kMajMK, 256, 2, 2, false, false);
      default: OBJB_GEMM(dev::kMajMN, 256, 2, 2, false, false);
    }
  }
  t.chunk_kb = y16 ? 16 : 4;
  const size_t pair_m = ceil_div(p.M, p.gated ? 128 : 256);
  if (pair_m * ceil_div(p.N, 128) * 4 >= sms) {
    t.bn = p.maj == dev::kMajMN ? 128 : pair_columns(pair_m, p.N, 128, 16, pairs);
    if (p.gated) OBJB_GEMM(dev::kMajKK, 128, 2, 1, true, true);
    switch (p.maj) {
      case dev::kMajKK: OBJB_GEMM(dev::kMajKK, 128, 2, 1, false, true);
      case dev::kMajMK: OBJB_GEMM(dev::kMajMK, 128, 2, 1, false, true);
      default: OBJB_GEMM(dev::kMajMN, 128, 2, 1, false, true);
    }
  }
  int bn = p.maj == dev::kMajMN ? 64 : 16;
  while (bn < 128 && static_cast<size_t>(bn) < p.N) bn *= 2;
  t.bn = p.maj == dev::kMajMN ? bn : static_cast<int>(std::min<size_t>(bn, ceil_div(p.N, 16) * 16));
  const size_t tiles = ceil_div(p.M, p.gated ? 64 : 128) * ceil_div(p.N, t.bn);
  while (t.split < 8 && tiles * t.split * 2 <= sms && nkb >= static_cast<size_t>(t.split) * 8 && bn / (t.split * 2) >= 2)
    t.split *= 2;
  if (p.gated) {
    switch (bn) {
      case 16: OBJB_GEMM(dev::kMajKK, 16, 1, 1, true, true);
      case 32: OBJB_GEMM(dev::kMajKK, 32, 1, 1, true, true);
      case 64: OBJB_GEMM(dev::kMajKK, 64, 1, 1, true, true);
      default: OBJB_GEMM(dev::kMajKK, 128, 1, 1, true, true);
    }
  }
  switch (p.maj) {
    case dev::kMajKK:
      switch (bn) {
        case 16: OBJB_GEMM(dev::kMajKK, 16, 1, 1, false, true);
        case 32: OBJB_GEMM(dev::kMajKK, 32, 1, 1, false, true);
        case 64: OBJB_GEMM(dev::kMajKK, 64, 1, 1, false, true);
        default: OBJB_GEMM(dev::kMajKK, 128, 1, 1, false, true);
      }
    case dev::kMajMK:
      switch (bn) {
        case 16: OBJB_GEMM(dev::kMajMK, 16, 1, 1, false, true);
        case 32: OBJB_GEMM(dev::kMajMK, 32, 1, 1, false, true);
        case 64: OBJB_GEMM(dev::kMajMK, 64, 1, 1, false, true);
        default: OBJB_GEMM(dev::kMajMK, 128, 1, 1, false, true);
      }
    default:
      if (bn == 64) OBJB_GEMM(dev::kMajMN, 64, 1, 1, false, true);
      OBJB_GEMM(dev::kMajMN, 128, 1, 1, false, true);
  }
#undef OBJB_GEMM
}

int device_here(int* device, DeviceProps* props) {
  OBJB_TRY(current_device(device));
  return device_props(*device, props);
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
  if (need == 0) {
    ws = nullptr;
  } else if (ws) {
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
  if (d->dw_dtype != OBJB_DTYPE_F32 && d->dw_dtype != d->w_dtype)
    return OBJB_FAIL(OBJB_ERR_UNSUPPORTED, action, "dw is f32 or w's type");
  if ((d->outputs & ~7) || !d->outputs)
    return OBJB_FAIL(OBJB_ERR_INVALID_INPUT, action, "outputs must name at least one of dx, dw and dbias");
  return OBJB_OK;
}

struct LinearPlan {
  ImagePlan x, w;
  size_t total;
};
LinearPlan plan_linear(const objb_linear_desc& d, size_t ldx, size_t ldw, const void* x, const void* w) {
  LinearPlan p;
  p.x = plan_image(x, d.x_dtype, ldx, d.tokens, d.in_features, d.x_dtype == OBJB_DTYPE_F32 ? 3 : 1);
  p.w = plan_image(w, d.w_dtype, ldw, d.out_features, d.in_features, d.w_dtype == OBJB_DTYPE_F32 ? 3 : 1);
  p.total = p.x.bytes + p.w.bytes;
  return p;
}

// dz enters the two products in dy's 16-bit type, or in three bf16 planes (f32
// dy; f32 dw behind an activation); then f16 operands become two bf16 planes,
// which hold their 11 bits exactly.
struct BackwardPlan {
  bool has_act, want_dx, want_dw, want_db, dz_direct;
  int parts;
  long long rows_per;
  ImagePlan x, w, dz;
  size_t part_bytes, total;
};
BackwardPlan plan_backward(const objb_linear_backward_desc& d, size_t lddy, size_t ldx, size_t ldw, const void* dy,
                           const void* x, const void* w, int sms) {
  BackwardPlan p;
  p.want_dx = d.outputs & OBJB_LINEAR_DX;
  p.want_dw = d.outputs & OBJB_LINEAR_DW;
  p.want_db = d.outputs & OBJB_LINEAR_DBIAS;
  p.has_act = d.activation != OBJB_ACT_NONE;
  const bool wide = d.dy_dtype == OBJB_DTYPE_F32 || (p.has_act && p.want_dw && d.dw_dtype == OBJB_DTYPE_F32);
  p.dz = plan_image(dy, d.dy_dtype, lddy, d.tokens, d.out_features, wide ? 3 : 1);
  p.dz_direct = !p.has_act && p.dz.direct;
  if (p.has_act && p.dz.direct) p.dz = plan_image(nullptr, OBJB_DTYPE_F32, 0, d.tokens, d.out_features, 1);
  if (!p.want_dx && !p.want_dw) p.dz.bytes = 0;
  auto planes = [&](int dtype) { return dtype == OBJB_DTYPE_F32 ? 3 : dtype == OBJB_DTYPE_F16 && wide ? 2 : 1; };
  p.x = plan_image(x, d.x_dtype, ldx, d.tokens, d.in_features, planes(d.x_dtype));
  p.w = plan_image(w, d.w_dtype, ldw, d.out_features, d.in_features, planes(d.w_dtype));
  if (!p.want_dw) p.x.bytes = 0;
  if (!p.want_dx) p.w.bytes = 0;
  // runs of rows of the column sums: enough blocks to fill the SMs, 32 rows or more in each
  const size_t cols = (d.out_features + 255) / 256;
  const size_t want = std::max<size_t>(1, (static_cast<size_t>(sms) * 4 + cols - 1) / cols);
  p.parts = static_cast<int>(std::max<size_t>(1, std::min(want, (d.tokens + 31) / 32)));
  p.rows_per = static_cast<long long>((d.tokens + p.parts - 1) / p.parts);
  p.part_bytes = p.want_db ? r256(static_cast<size_t>(p.parts) * d.out_features * 4) : 0;
  p.total = p.x.bytes + p.w.bytes + p.dz.bytes + p.part_bytes;
  return p;
}

struct FfnPlan {
  ImagePlan gate, up, down, x, act;
  size_t total;
};
FfnPlan plan_ffn(size_t T, size_t H, size_t I, size_t O, const void* gate, const void* up, const void* down) {
  FfnPlan p;
  p.gate = plan_image(gate, OBJB_DTYPE_BF16, H, I, H, 1);
  p.up = plan_image(up, OBJB_DTYPE_BF16, H, I, H, 1);
  p.down = plan_image(down, OBJB_DTYPE_BF16, I, O, I, 1);
  p.x = plan_image(nullptr, OBJB_DTYPE_F32, H, T, H, 3);
  p.act = plan_image(nullptr, OBJB_DTYPE_F32, I, T, I, 3);
  p.total = p.gate.bytes + p.up.bytes + p.down.bytes + p.x.bytes + p.act.bytes;
  return p;
}

}  // namespace
}  // namespace objb

using namespace objb;

extern "C" {

int objb_linear_scratch_bytes(const objb_linear_desc* desc, const void* d_x, const void* d_w, size_t* bytes) {
  clear_error();
  const char* action = "objb_linear_scratch_bytes";
  OBJB_TRY(check_linear(action, desc));
  if (!bytes) return OBJB_FAIL(OBJB_ERR_INVALID_INPUT, action, "null output pointer");
  size_t ldx, ldw;
  OBJB_TRY(check_stride(action, "x_stride", desc->x_stride, desc->in_features, &ldx));
  OBJB_TRY(check_stride(action, "w_stride", desc->w_stride, desc->in_features, &ldw));
  *bytes = plan_linear(*desc, ldx, ldw, d_x, d_w).total;
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
  int device = 0;
  DeviceProps props;
  OBJB_TRY(device_here(&device, &props));
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  const LinearPlan pl = plan_linear(d, ldx, ldw, d_x, d_w);
  uint8_t* ws = nullptr;
  OBJB_TRY(take_scratch(action, d_scratch, scratch_bytes, pl.total, st, &ws));
  Product p;
  OBJB_TRY(make_image(pl.w, d_w, d.w_dtype, ldw, d.out_features, d.in_features, ws, props, st, &p.a));
  OBJB_TRY(make_image(pl.x, d_x, d.x_dtype, ldx, d.tokens, d.in_features, ws + pl.w.bytes, props, st, &p.b));
  p.M = d.out_features;
  p.N = d.tokens;
  p.K = d.in_features;
  dev::LinearEpilogue& e = p.epi;
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
  return gemm(p, device, props, st);
}

static int backward_strides(const char* action, const objb_linear_backward_desc& d, size_t* lddy, size_t* ldz,
                            size_t* ldx, size_t* ldw, size_t* lddx, size_t* lddw) {
  OBJB_TRY(check_stride(action, "dy_stride", d.dy_stride, d.out_features, lddy));
  OBJB_TRY(check_stride(action, "z_stride", d.z_stride, d.out_features, ldz));
  OBJB_TRY(check_stride(action, "x_stride", d.x_stride, d.in_features, ldx));
  OBJB_TRY(check_stride(action, "w_stride", d.w_stride, d.in_features, ldw));
  OBJB_TRY(check_stride(action, "dx_stride", d.dx_stride, d.in_features, lddx));
  return check_stride(action, "dw_stride", d.dw_stride, d.in_features, lddw);
}

int objb_linear_backward_scratch_bytes(const objb_linear_backward_desc* desc, const void* d_dy, const void* d_x,
                                       const void* d_w, size_t* bytes) {
  clear_error();
  const char* action = "objb_linear_backward_scratch_bytes";
  OBJB_TRY(check_backward(action, desc));
  if (!bytes) return OBJB_FAIL(OBJB_ERR_INVALID_INPUT, action, "null output pointer");
  size_t lddy, ldz, ldx, ldw, lddx, lddw;
  OBJB_TRY(backward_strides(action, *desc, &lddy, &ldz, &ldx, &ldw, &lddx, &lddw));
  int device = 0;
  DeviceProps props;
  OBJB_TRY(device_here(&device, &props));
  *bytes = plan_backward(*desc, lddy, ldx, ldw, d_dy, d_x, d_w, props.sm_count).total;
  return OBJB_OK;
}

int objb_linear_backward_device(const objb_linear_backward_desc* desc, const void* d_dy, const void* d_z,
                                const void* d_x, const void* d_w, void* d_dx, void* d_dw, float* d_dbias,
                                void* d_scratch, size_t scratch_bytes, objb_stream_t stream) {
  clear_error();
  const char* action = "objb_linear_backward_device";
  OBJB_TRY(check_backward(action, desc));
  const objb_linear_backward_desc& d = *desc;
  size_t lddy, ldz, ldx, ldw, lddx, lddw;
  OBJB_TRY(backward_strides(action, d, &lddy, &ldz, &ldx, &ldw, &lddx, &lddw));
  const bool want_dx = d.outputs & OBJB_LINEAR_DX, want_dw = d.outputs & OBJB_LINEAR_DW,
             want_db = d.outputs & OBJB_LINEAR_DBIAS;
  if ((want_dw && !d_dw) || (want_db && !d_dbias) ||
      (d.tokens && (!d_dy || (d.activation != OBJB_ACT_NONE && !d_z) || (want_dw && !d_x) ||
                    (want_dx && (!d_w || !d_dx)))))
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
  int device = 0;
  DeviceProps props;
  OBJB_TRY(device_here(&device, &props));
  const BackwardPlan pl = plan_backward(d, lddy, ldx, ldw, d_dy, d_x, d_w, props.sm_count);
  uint8_t* ws = nullptr;
  OBJB_TRY(take_scratch(action, d_scratch, scratch_bytes, pl.total, st, &ws));
  uint8_t *ws_dz = ws, *ws_x = ws_dz + pl.dz.bytes, *ws_w = ws_x + pl.x.bytes, *ws_part = ws_w + pl.w.bytes;
  const int N = static_cast<int>(d.out_features);
  const bool products = want_dx || want_dw;
  Image dz;
  dz.p = pl.dz_direct ? d_dy : ws_dz;
  dz.ld = pl.dz.pitch;
  dz.rows = d.tokens;
  dz.cols = d.out_features;
  dz.planes = pl.dz.planes;
  dz.dtype = pl.dz.planes > 1 ? OBJB_DTYPE_BF16 : d.dy_dtype;
  const bool image = products && !pl.dz_direct;
  if (image || want_db) {
    const bool vec = aligned16(d_dy) && lddy % 8 == 0 && (!pl.has_act || (aligned16(d_z) && ldz % 8 == 0));
    const dim3 grid((N + 255) / 256, pl.parts);
    auto k = vec ? dev::dz_kernel<true> : dev::dz_kernel<false>;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(256);
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    float* part = want_db ? reinterpret_cast<float*>(ws_part) : nullptr;
    OBJB_CUDA(cudaLaunchKernelEx(&cfg, k, d_dy, lddy, d_z, ldz, static_cast<int>(d.dy_dtype),
                                 static_cast<int>(d.activation), static_cast<long long>(d.tokens), N,
                                 image ? reinterpret_cast<uint16_t*>(ws_dz) : nullptr, static_cast<int>(pl.dz.pitch),
                                 pl.dz.planes, pl.rows_per, part),
              "launch dz");
    if (want_db)
      OBJB_TRY(launch_pdl(dev::dbias_kernel, (N + 255) / 256, 256, 0, st, static_cast<const float*>(part), pl.parts, N,
                          d_dbias, static_cast<int>(d.accumulate)));
  }
  if (want_dx) {
    Product p;
    p.maj = dev::kMajMK;
    OBJB_TRY(make_image(pl.w, d_w, d.w_dtype, ldw, d.out_features, d.in_features, ws_w, props, st, &p.a));
    p.b = dz;
    p.M = d.in_features;
    p.N = d.tokens;
    p.K = d.out_features;
    p.epi.y = d_dx;
    p.epi.ldy = lddx;
    p.epi.y_dtype = d.x_dtype;
    OBJB_TRY(gemm(p, device, props, st));
  }
  if (want_dw) {
    Product p;
    p.maj = dev::kMajMN;
    OBJB_TRY(make_image(pl.x, d_x, d.x_dtype, ldx, d.tokens, d.in_features, ws_x, props, st, &p.a));
    p.b = dz;
    p.M = d.in_features;
    p.N = d.out_features;
    p.K = d.tokens;
    p.epi.y = d_dw;
    p.epi.ldy = lddw;
    p.epi.y_dtype = d.dw_dtype;
    if (d.accumulate) p.epi.residual = d_dw, p.epi.ldr = lddw;
    OBJB_TRY(gemm(p, device, props, st));
  }
  return OBJB_OK;
}

static int check_ffn(const char* action, size_t T, size_t H, size_t I, size_t O) {
  OBJB_TRY(check_sizes(action, T, H, I, 0));
  return check_sizes(action, T, I, O, 0);
}

int objb_ffn_bf16_tokens_scratch_bytes(const void* d_gate, const void* d_up, const void* d_down, size_t hidden,
                                       size_t intermediate, size_t out_dim, size_t num_tokens, size_t* bytes) {
  clear_error();
  const char* action = "objb_ffn_bf16_tokens_scratch_bytes";
  OBJB_TRY(check_ffn(action, num_tokens, hidden, intermediate, out_dim));
  if (!bytes) return OBJB_FAIL(OBJB_ERR_INVALID_INPUT, action, "null output pointer");
  *bytes = plan_ffn(num_tokens, hidden, intermediate, out_dim, d_gate, d_up, d_down).total;
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
  int device = 0;
  DeviceProps props;
  OBJB_TRY(device_here(&device, &props));
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  const FfnPlan pl = plan_ffn(num_tokens, hidden, intermediate, out_dim, d_gate, d_up, d_down);
  uint8_t* ws = nullptr;
  OBJB_TRY(take_scratch(action, d_scratch, scratch_bytes, pl.total, st, &ws));
  const int bf = OBJB_DTYPE_BF16;
  Product gu;
  gu.gated = true;
  OBJB_TRY(make_image(pl.gate, d_gate, bf, hidden, intermediate, hidden, ws, props, st, &gu.a));
  ws += pl.gate.bytes;
  OBJB_TRY(make_image(pl.up, d_up, bf, hidden, intermediate, hidden, ws, props, st, &gu.a2));
  ws += pl.up.bytes;
  Product dn;
  OBJB_TRY(make_image(pl.down, d_down, bf, intermediate, out_dim, intermediate, ws, props, st, &dn.a));
  ws += pl.down.bytes;
  OBJB_TRY(make_image(pl.x, d_x, OBJB_DTYPE_F32, hidden, num_tokens, hidden, ws, props, st, &gu.b));
  ws += pl.x.bytes;
  gu.M = intermediate;
  gu.N = num_tokens;
  gu.K = hidden;
  gu.swiglu_limit = swiglu_limit;
  gu.epi.y = ws;  // the activations, as the planes that the down product reads
  gu.epi.ldy = pl.act.pitch;
  gu.epi.plane = num_tokens * pl.act.pitch;
  OBJB_TRY(gemm(gu, device, props, st));
  dn.b.p = ws;
  dn.b.ld = pl.act.pitch;
  dn.b.rows = num_tokens;
  dn.b.cols = intermediate;
  dn.b.planes = 3;
  dn.b.dtype = bf;
  dn.M = out_dim;
  dn.N = num_tokens;
  dn.K = intermediate;
  dn.epi.y = d_out;
  dn.epi.ldy = out_dim;
  dn.epi.residual = d_residual;
  dn.epi.ldr = out_dim;
  dn.epi.y_dtype = OBJB_DTYPE_F32;
  return gemm(dn, device, props, st);
}

}  // extern "C"
