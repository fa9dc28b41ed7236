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
#include <cmath>
#include <map>
#include <mutex>
#include <string>

#include "objb_common.h"
#include "objb_host_launch.cuh"
#include "objb_launch.h"
#include "objb_linear_launch.cuh"

namespace objb {
namespace dev {

// 8 neighbouring elements in flight; T: float, __nv_bfloat16 or __half.  VEC:
// their address is 16-byte aligned and all 8 exist.
template <class T, bool VEC>
struct Oct {
  uint4 q[sizeof(T) / 2];
  T e[VEC ? 1 : 8];
  __device__ __forceinline__ void load(const T* p, int n) {
    if constexpr (VEC) {
      const uint4* s = reinterpret_cast<const uint4*>(p);
#pragma unroll
      for (int i = 0; i < static_cast<int>(sizeof(T) / 2); ++i) q[i] = __ldg(s + i);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) e[i] = i < n ? p[i] : T(0.0f);
    }
  }
  __device__ __forceinline__ void values(float (&v)[8]) const {
    if constexpr (!VEC) {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = static_cast<float>(e[i]);
    } else if constexpr (sizeof(T) == 4) {
      v[0] = __uint_as_float(q[0].x), v[1] = __uint_as_float(q[0].y), v[2] = __uint_as_float(q[0].z);
      v[3] = __uint_as_float(q[0].w), v[4] = __uint_as_float(q[1].x), v[5] = __uint_as_float(q[1].y);
      v[6] = __uint_as_float(q[1].z), v[7] = __uint_as_float(q[1].w);
    } else {
      const uint32_t u[4] = {q[0].x, q[0].y, q[0].z, q[0].w};
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint16_t h = static_cast<uint16_t>(u[i >> 1] >> (16 * (i & 1)));
        if constexpr (std::is_same<T, __half>::value)
          v[i] = __half2float(__ushort_as_half(h));
        else
          v[i] = __uint_as_float(static_cast<uint32_t>(h) << 16);
      }
    }
  }
};

// f(T, VEC) for an element type; vec: rows of aligned octs.
template <class F>
auto with_elements(int dtype, bool vec, F&& f) {
  using std::integral_constant;
  if (dtype == OBJB_DTYPE_F32)
    return vec ? f(float{}, integral_constant<bool, true>{}) : f(float{}, integral_constant<bool, false>{});
  if (dtype == OBJB_DTYPE_BF16)
    return vec ? f(__nv_bfloat16{}, integral_constant<bool, true>{})
               : f(__nv_bfloat16{}, integral_constant<bool, false>{});
  return vec ? f(__half{}, integral_constant<bool, true>{}) : f(__half{}, integral_constant<bool, false>{});
}

// 8 elements of an image row (its pitch is a whole number of 16-byte quads):
// one plane of `dtype`, or the first `planes` bf16 parts.
__device__ __forceinline__ void store_image8(uint16_t* img, size_t plane, size_t at, int planes, int dtype,
                                             const float (&v)[8]) {
  uint32_t u[4][3] = {};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (planes > 1) {
      split3_pair(v[2 * i], v[2 * i + 1], u[i]);
    } else if (dtype == OBJB_DTYPE_F16) {
      const __half2 h = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
      u[i][0] = *reinterpret_cast<const uint32_t*>(&h);
    } else {
      const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
      u[i][0] = *reinterpret_cast<const uint32_t*>(&h);
    }
  }
#pragma unroll
  for (int j = 0; j < 3; ++j)
    if (j < planes)
      *reinterpret_cast<uint4*>(img + j * plane + at) = make_uint4(u[0][j], u[1][j], u[2][j], u[3][j]);
}

// Up to two operands laid out for the copy engine in one launch: rows of
// `pitch` elements (a multiple of 8), f32 in planes.  8 elements per thread; a
// block takes 256 >> log_width rows at a time, two in flight.
struct ImageJob {
  const void* src;
  uint16_t* img;
  size_t ld;
  long long rows;
  int cols, pitch, planes, dtype, vec, log_width;
};
template <class T, bool VEC>
__device__ __forceinline__ void image_run(const ImageJob& j, int block, int blocks) {
  const int width = 1 << j.log_width, per = 256 >> j.log_width;
  const int tx = threadIdx.x & (width - 1), ty = threadIdx.x >> j.log_width;
  const size_t plane = j.rows * static_cast<size_t>(j.pitch);
  const T* src = static_cast<const T*>(j.src);
  for (long long r = static_cast<long long>(block) * per * 2 + ty; r < j.rows;
       r += static_cast<long long>(blocks) * per * 2) {
    const bool two = r + per < j.rows;
    for (int c = tx * 8; c < j.pitch; c += width * 8) {
      Oct<T, VEC> a, b;
      float v[8];
      a.load(src + r * j.ld + c, j.cols - c);
      if (two) b.load(src + (r + per) * j.ld + c, j.cols - c);
      a.values(v);
      store_image8(j.img, plane, r * static_cast<size_t>(j.pitch) + c, j.planes, j.dtype, v);
      if (two) {
        b.values(v);
        store_image8(j.img, plane, (r + per) * static_cast<size_t>(j.pitch) + c, j.planes, j.dtype, v);
      }
    }
  }
}
__device__ __forceinline__ void image_block(const ImageJob& j, int block, int blocks) {
  if (j.dtype == OBJB_DTYPE_F32)
    j.vec ? image_run<float, true>(j, block, blocks) : image_run<float, false>(j, block, blocks);
  else if (j.dtype == OBJB_DTYPE_BF16)
    j.vec ? image_run<__nv_bfloat16, true>(j, block, blocks) : image_run<__nv_bfloat16, false>(j, block, blocks);
  else
    j.vec ? image_run<__half, true>(j, block, blocks) : image_run<__half, false>(j, block, blocks);
}
__global__ void __launch_bounds__(256) image_kernel(const ImageJob first, const ImageJob second) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  image_block(blockIdx.y ? second : first, blockIdx.x, gridDim.x);
}

// dz = dy act'(z) as an image (may be null: only its sums), and the column
// sums of each run of rows (of one run: dbias itself).  A block: 256 columns (8
// per thread), 8 row lanes with two rows in flight; the lanes are folded in
// order.  The blocks behind dz's lay out the other operands, in the same launch.
// Bound by its bytes: 4096 x 14336 bf16 with SiLU 51.8 us (352 MB), 2048 x 4096
// f16 with tanh-GELU 12.6 with the fold of the sums.  (Four rows in flight take
// 80 registers, three blocks an SM: 61 and 13.9; four blocks of 64 registers
// with as many rows spill so much that they take 101.  The 16-bit kernels as
// they are spill 32 bytes a thread, 96 where rows are not aligned.)
struct DzJob {
  const void *dy, *z;
  size_t ldy, ldz;
  long long rows, rows_per;
  int N, dtype, act, pitch, planes;
  int cols, blocks;  // blocks of 256 columns, of all
  uint16_t* img;
  float* part;
  bool add;          // one run: part += the sums
};
template <class T, bool VEC>
__global__ void __launch_bounds__(256, sizeof(T) == 4 ? 3 : 4) dz_kernel(const DzJob d, const ImageJob first, const ImageJob second,
                                                 int image_blocks) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  __shared__ float sm[8][256];
  if (static_cast<int>(blockIdx.x) >= d.blocks) {
    const int b = blockIdx.x - d.blocks;
    image_block(b < image_blocks ? first : second, b < image_blocks ? b : b - image_blocks, image_blocks);
    return;
  }
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  const int run = blockIdx.x / d.cols, col0 = (blockIdx.x - run * d.cols) * 256;
  const int c = col0 + tx * 8, N = d.N, act = d.act;
  const T *dy = static_cast<const T*>(d.dy), *z = static_cast<const T*>(d.z);
  const long long r0 = run * d.rows_per, r1 = r0 + d.rows_per < d.rows ? r0 + d.rows_per : d.rows;
  float s[8] = {};
  if (c < N) {
    constexpr int R = 2;
    for (long long r = r0 + ty; r < r1; r += 8 * R) {
      Oct<T, VEC> g[R], a[R];
#pragma unroll
      for (int q = 0; q < R; ++q)
        if (r + 8 * q < r1) {
          g[q].load(dy + (r + 8 * q) * d.ldy + c, N - c);
          if (act != OBJB_ACT_NONE) a[q].load(z + (r + 8 * q) * d.ldz + c, N - c);
        }
#pragma unroll
      for (int q = 0; q < R; ++q)
        if (r + 8 * q < r1) {
          float v[8];
          g[q].values(v);
          if (act != OBJB_ACT_NONE) {
            float zz[8];
            a[q].values(zz);
            switch (act) {
#define OBJB_GRAD_CASE(A) \
  case A:                 \
    _Pragma("unroll") for (int i = 0; i < 8; ++i) v[i] *= act_grad(A, zz[i]); \
    break
              OBJB_GRAD_CASE(OBJB_ACT_RELU);
              OBJB_GRAD_CASE(OBJB_ACT_SILU);
              OBJB_GRAD_CASE(OBJB_ACT_GELU);
              OBJB_GRAD_CASE(OBJB_ACT_GELU_TANH);
#undef OBJB_GRAD_CASE
              default: break;
            }
          }
          if (d.img)
            store_image8(d.img, d.rows * static_cast<size_t>(d.pitch),
                         (r + 8 * q) * static_cast<size_t>(d.pitch) + c, d.planes, d.dtype, v);
#pragma unroll
          for (int i = 0; i < 8; ++i) s[i] += v[i];
        }
    }
  }
  if (!d.part) return;
#pragma unroll
  for (int i = 0; i < 8; ++i) sm[ty][tx * 8 + i] = s[i];
  __syncthreads();
  const int col = col0 + threadIdx.x;
  if (col >= N) return;
  float sum = 0.0f;
#pragma unroll
  for (int i = 0; i < 8; ++i) sum += sm[i][threadIdx.x];
  float* to = d.part + static_cast<size_t>(run) * N + col;
  *to = d.add ? *to + sum : sum;
}

// The runs' sums folded: 32 columns per block, 32 interleaved runs, those in order.
__global__ void __launch_bounds__(1024) dbias_kernel(const float* part, int parts, int N, float* db, int accumulate) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
  __shared__ float sm[32][33];
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + tx;
  float s = 0.0f;
  if (c < N) {
#pragma unroll 4
    for (int i = ty; i < parts; i += 32) s += part[static_cast<size_t>(i) * N + c];
  }
  sm[ty][tx] = s;
  __syncthreads();
  s = sm[tx][ty];  // column ty, run tx
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xFFFFFFFFu, s, o);
  const int col = blockIdx.x * 32 + ty;
  if (tx == 0 && col < N) db[col] = accumulate ? db[col] + s : s;
}

}  // namespace dev

namespace {

constexpr size_t kMaxSize = size_t{1} << 24;    // in / out features
constexpr size_t kMaxTokens = size_t{1} << 30;
constexpr size_t kMaxStride = size_t{1} << 28;

size_t r256(size_t b) { return (b + 255) / 256 * 256; }
size_t elem_bytes(int dtype) { return dtype == OBJB_DTYPE_F32 ? 4 : 2; }

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

// The images of up to two operands, laid out by one launch where they are not
// direct.
class Images {
 public:
  Image take(const ImagePlan& pl, const void* p, int dtype, size_t ld, size_t rows, size_t cols, void* scratch) {
    Image im;
    im.rows = rows;
    im.cols = cols;
    im.planes = pl.planes;
    im.ld = pl.pitch;
    im.dtype = pl.planes > 1 || dtype == OBJB_DTYPE_F32 ? OBJB_DTYPE_BF16 : dtype;
    im.p = pl.direct ? p : scratch;
    if (!pl.direct) {
      dev::ImageJob& j = jobs_[n_++];
      j.src = p;
      j.img = static_cast<uint16_t*>(scratch);
      j.ld = ld;
      j.rows = static_cast<long long>(rows);
      j.cols = static_cast<int>(cols);
      j.pitch = static_cast<int>(pl.pitch);
      j.planes = pl.planes;
      j.dtype = dtype;
      j.vec = aligned16(p) && ld % 8 == 0 && cols % 8 == 0;
      j.log_width = 0;
      while (j.log_width < 8 && (8u << j.log_width) < pl.pitch) ++j.log_width;
      blocks_ = std::max(blocks_, ceil_div(rows, size_t{512} >> j.log_width));
    }
    return im;
  }
  int launch(const DeviceProps& props, cudaStream_t st) {
    if (!n_) return OBJB_OK;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(blocks(props)), static_cast<unsigned>(n_));
    cfg.blockDim = dim3(256);
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    OBJB_CUDA(cudaLaunchKernelEx(&cfg, dev::image_kernel, jobs_[0], jobs_[1]), "launch operand image");
    clear();
    return OBJB_OK;
  }
  // for a launch that does them beside its own work
  int count() const { return n_; }
  int blocks(const DeviceProps& props) const {
    return n_ ? static_cast<int>(std::min(blocks_, static_cast<size_t>(props.sm_count) * 8)) : 0;
  }
  const dev::ImageJob& job(int i) const { return jobs_[i]; }
  void clear() { n_ = 0, blocks_ = 0; }

 private:
  dev::ImageJob jobs_[2] = {};
  int n_ = 0;
  size_t blocks_ = 0;
};

// The tensor map of an image: box of 64 elements by `box_rows` rows, all planes.
}  // namespace

int linear_encode(CUtensorMap* map, const Image& im, int box_rows) {
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
  const bool f32 = im.dtype == OBJB_DTYPE_F32;
  const cuuint32_t planes = f32 ? 1 : im.planes;
  const size_t pitch = im.ld * (f32 ? 4 : 2);
  const cuuint64_t dims[3] = {im.cols, im.rows, planes};
  const cuuint64_t strides[2] = {pitch, im.rows * pitch};
  const cuuint32_t box[3] = {64, static_cast<cuuint32_t>(box_rows), planes};
  const cuuint32_t estr[3] = {1, 1, 1};
  const CUresult r =
      fn(map,
         f32                             ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
         : im.dtype == OBJB_DTYPE_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                         : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16,
         3, const_cast<void*>(im.p), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
         f32 ? CU_TENSOR_MAP_SWIZZLE_NONE : CU_TENSOR_MAP_SWIZZLE_128B,
         CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS)
    return OBJB_FAIL(OBJB_ERR_DRIVER, "dense product", "cuTensorMapEncodeTiled failed (" + std::to_string(r) + ")");
  return OBJB_OK;
}

namespace {

struct Choice {
  TileKind kind = kSingle;
  Tile tile;
};

// Clusters of 1, 2, 4 and 8 single CTAs that the device holds at once, one and
// two CTAs per SM (clusters do not straddle its SM groups, so that four or
// eight CTAs leave SMs over).
struct Room {
  int clusters[2][4] = {};
};

// A product's time by a model whose parts were measured apart on B200.  It ranks
// tiles; its sums do not hold as times (4096^3: 78 us, measured 99; 4096 x 4096 x
// 14336: 267 and 395; f32 split inside at 16 x 4096 x 16384: 55 and 98).  A
// producer iteration (wait, expected bytes) 145 and a copy 35; an MMA of 16 of
// k 20 or bn / 2 clocks, a stage's wait and commit 150; 131 bytes taken in per
// SM from L2; 1000 (direct: 1500) to drain a tile; launch, set-up and exit
// 3000, a fold over a cluster 2200.
double nanoseconds(const Product& p, TileKind kind, const Tile& t, size_t sms, const Room& room) {
  const size_t cg = kind == kSingle ? 1 : 2, mt = kind == kDirect ? 2 : 1;
  const bool two = t.ring == kLinRingTwo;
  const size_t rows = p.gated ? 64 : mt * t.rm;
  const double tiles = static_cast<double>(ceil_div(p.M, rows * cg)) * ceil_div(p.N, t.bn);
  const int log_split = t.split == 1 ? 0 : t.split == 2 ? 1 : t.split == 4 ? 2 : 3;
  const double width = kind == kSingle ? room.clusters[two][log_split] : sms / 2;
  const double share = two ? std::min(2.0, std::max(1.0, tiles * t.split / sms)) : 1.0;  // CTAs at work per SM
  // clocks of a k-step's MMAs: side by side (N 3 bn, 2 bn, bn), or one per pair of planes
  const int pa = p.a.planes, pb = p.b.planes;
  auto one = [](double n) { return std::max(39.0, n / 2); };
  double clocks = mt * one(t.bn);
  if (pb > 1 && kind == kSingle)
    clocks = one(3.0 * t.bn) + (pa > 1 ? one(2.0 * t.bn) : 0.0) + (pa > 2 ? one(t.bn) : 0.0);
  else if (pb > 1)
    clocks = (pa == 1 ? 3 : pa == 2 ? 5 : 6) * one(t.bn);
  const double mma = 4.0 * clocks / 1.7;
  const double copies = mt * (p.maj == dev::kMajKK && !p.gated ? 1 : 2) +
                        (p.raw ? 0 : p.maj == dev::kMajMN ? ceil_div(t.bn / cg, 64) : 1);
  const double bytes = 128.0 * (p.a.planes * (p.gated ? 128 : mt * t.rm) + p.b.planes * t.bn / cg);
  // splitting an f32 operand's rows
  const double convert = p.raw ? 150.0 / t.unit + 5.0 * ((p.raw == 2 ? t.rm : 0) + t.bn) : 0.0;
  const double kb = std::max(convert, std::max(std::max(145.0 / t.unit + 35.0 * copies, std::max(mma * share, 150.0 / t.unit + mma / 2)),
                             bytes / (kind == kSingle ? 125.0 : 90.0) * share));
  const double kbs = std::ceil(static_cast<double>(ceil_div(p.K, 64)) / t.split);
  return std::ceil(tiles / width) * (kbs * kb + (kind == kDirect ? 1500.0 : 1000.0)) + 3000.0 +
         (t.split > 1 ? 2200.0 : 0.0);
}

// Which tile a product takes: the one of the fewest nanoseconds() among
//   * direct: pairs, 512 x up to 256 columns, for 16-bit results of one-plane operands (k up to direct_k);
//   * pairs of 256 rows x up to 128 columns;
//   * single CTAs of 128 rows x up to 128 columns, k split over a cluster, one
//     per SM or (up to 64 columns) two.
// Rows below 128 (K-major A) and columns below the most even out the rounds;
// stages of several k-blocks save the producer's and the MMA warp's turns.
Choice choose_tile(const Product& p, bool y16, size_t sms, const Room& room) {
  const size_t nkb = ceil_div(p.K, 64);
  const bool mn = p.maj == dev::kMajMN, rows_free = p.maj == dev::kMajKK && !p.gated;
  Choice best;
  double least = 1e300;
  auto consider = [&](TileKind k, const Tile& c) {
    const double v = nanoseconds(p, k, c, sms, room);
    if (v < least) {
      least = v;
      best.kind = k;
      best.tile = c;
    }
  };
  // columns: what N needs, rounded to a step of the layout, at most `most` and then down to `least_bn`
  auto each_bn = [&](int most, int step, int least_bn, auto f) {
    const int need = static_cast<int>(std::min<size_t>(most, ceil_div(p.N, step) * step));
    for (int bn = need; bn >= std::min(need, least_bn); bn -= step) f(bn);
  };
  // rows, and units whose stages leave the ring at least three (two of one k-block)
  auto each_row_unit = [&](TileKind k, Tile c, int cg) {
    for (c.rm = 128; c.rm >= (rows_free ? 64 : 128); c.rm -= 8) {
      const size_t kb = 128 * (p.a.planes * (rows_free ? c.rm : 128) + p.b.planes * c.bn / cg) +
                        (p.raw ? 256 * ((p.raw == 2 ? c.rm : 0) + c.bn) : 0);
      for (c.unit = 1; c.unit <= 4; c.unit *= 2)
        if (kb * c.unit * (c.unit == 1 ? 2 : 3) <= c.ring) consider(k, c);
    }
  };
  Tile c;
  if (p.raw) {
    each_bn(single_columns(p.maj, 3), 16, 16, [&](int bn) {
      c.bn = bn;
      for (c.split = 1; c.split <= 8 && nkb >= static_cast<size_t>(c.split); c.split *= 2)
        each_row_unit(kSingle, c, 1);
    });
    return best;
  }
  if (y16 && p.a.planes == 1 && p.b.planes == 1 && p.K <= dev::direct_k(p.a.dtype == OBJB_DTYPE_F16))
    each_bn(256, mn ? 128 : 16, 144, [&](int bn) {
      c.bn = bn;
      consider(kDirect, c);
    });
  each_bn(128, mn ? 128 : 16, 80, [&](int bn) {
    c.bn = bn;
    each_row_unit(kPair, c, 2);
  });
  each_bn(single_columns(p.maj, p.b.planes), mn ? 64 : 16, 16, [&](int bn) {
    c.bn = bn;
    for (c.split = 1; c.split <= 8 && nkb >= static_cast<size_t>(c.split); c.split *= 2)
      for (size_t ring : {kLinRing, kLinRingTwo}) {
        if (ring == kLinRingTwo && bn > two_columns(p.maj, p.b.planes)) continue;
        c.ring = ring;
        each_row_unit(kSingle, c, 1);
      }
  });
  return best;
}

int room_of(int device, size_t sms, Room* out) {
  static std::mutex mu;
  static std::map<int, Room> rooms;
  std::lock_guard<std::mutex> lk(mu);
  auto it = rooms.find(device);
  if (it == rooms.end()) {
    auto kernel = dev::lin_gemm_kernel<dev::kMajKK, 32, 1, 1, false, true, 1, 0>;
    Room r;
    for (int two = 0; two < 2; ++two) {
      const size_t smem = (two ? kLinRingTwo : kLinRing) + 1024;
      OBJB_TRY(ensure_smem_attr(kernel, device, smem));
      for (int i = 0; i < 4; ++i) {
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(static_cast<unsigned>(8 * sms));
        cfg.blockDim = dim3(dev::lin_threads(true));
        cfg.dynamicSmemBytes = smem;
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = 1u << i;
        attr[0].val.clusterDim.y = 1;
        attr[0].val.clusterDim.z = 1;
        cfg.attrs = attr;
        cfg.numAttrs = 1;
        OBJB_CUDA(cudaOccupancyMaxActiveClusters(&r.clusters[two][i], kernel, &cfg), "query clusters per device");
        r.clusters[two][i] = std::max(1, r.clusters[two][i]);
      }
    }
    it = rooms.emplace(device, r).first;
  }
  *out = it->second;
  return OBJB_OK;
}

// The choice is a function of these alone; trying all tiles takes the host
// several microseconds, so each thread keeps its last choices.
struct ChoiceKey {
  size_t M, N, K, sms;  // (devices of one process with as many SMs are alike)
  int maj, pa, pb, flags;
  bool operator==(const ChoiceKey& o) const {
    return M == o.M && N == o.N && K == o.K && sms == o.sms && maj == o.maj && pa == o.pa && pb == o.pb &&
           flags == o.flags;
  }
};

int gemm(const Product& p, int device, const DeviceProps& props, cudaStream_t st) {
  const bool y16 = !p.gated && p.epi.y_dtype != OBJB_DTYPE_F32;
  const ChoiceKey key{p.M, p.N, p.K, static_cast<size_t>(props.sm_count), p.maj, p.a.planes, p.b.planes,
                      (y16 ? 1 : 0) | (p.gated ? 2 : 0) | p.raw << 2 | (p.a.dtype == OBJB_DTYPE_F16 ? 16 : 0)};
  struct Kept {
    ChoiceKey key{};
    Choice choice;
  };
  thread_local Kept kept[64];
  Kept& k = kept[(p.M * 31 + p.N * 7 + p.K * 3 + static_cast<size_t>(p.maj)) % 64];
  if (!(k.key == key)) {
    Room room;
    OBJB_TRY(room_of(device, key.sms, &room));
    k.choice = choose_tile(p, y16, key.sms, room);
    k.key = key;
  }
  const TileKind kind = k.choice.kind;
  Tile t = k.choice.tile;
  // An MMA into an accumulator takes 2e-8 (bf16) or 8e-8 (f16) of a sum of one sign away: 8 k-blocks (32 MMAs) keep an
  // f32 result within 7e-7 or 2.5e-6 of it, where f32 sums of 4096 products are off by 8e-7 (relative norm, 1024 x 4096
  // x 2048); of mixed signs, 4.8e-7 and 6.5e-7 against 6e-7 to 1.1e-6.  (4 k-blocks: half of it, 16: twice; a chunk's
  // end costs some 400 ns.)  A gated product multiplies two such results: 4.  16-bit results: 2.4e-5 of f16's 4.9e-4.
  t.chunk_kb = y16 ? 64 : p.gated ? 4 : 8;
  switch (p.maj) {
    case dev::kMajKK: return launch_kk(p, kind, t, device, props, st);
    case dev::kMajMK: return launch_mk(p, kind, t, device, props, st);
    default: return launch_mn(p, kind, t, device, props, st);
  }
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
  if (*out > kMaxStride)
    return OBJB_FAIL(OBJB_ERR_INVALID_INPUT, action, std::string(name) + " is above 2^28 elements");
  if (*out < cols)
    return OBJB_FAIL(OBJB_ERR_INVALID_INPUT, action, std::string(name) + " is below the row's " + std::to_string(cols) +
                                                         " elements");
  return OBJB_OK;
}

Rows rows_of(const void* p, size_t rows, size_t cols, size_t ld, int dtype) {
  return {p, rows, cols * elem_bytes(dtype), ld * elem_bytes(dtype)};
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

// Which products split their f32 operands themselves (RAW: no launch before, no
// scratch, an f32 w read once), where the copy engine can read them as they lie.
// Every row tile splits x anew and every column tile w, so it pays
//   * for an f32 w of one narrow column tile (16384 x 4096, 16 tokens: 98 us,
//     laid out first 182; 64 tokens 180 and 187; 128 tokens 326 and 193; the
//     border between 16 and 64 was not searched);
//   * for results so small that the launch saved counts (250 tokens by 256 of
//     2048: 14.1 us a call, laid out first 15.7, launches bound; 512 tokens 18.6
//     and 15.7; 2^16 results lie between the two).  A column tile has 16 columns
//     at least (bf16 w of 16384 x 4096, one token: 30.8 and 27.8 us).
bool raw_pays(size_t T, size_t N, bool w_f32) {
  return (w_f32 && T <= 32) || std::max<size_t>(T, 16) * N <= (size_t{1} << 16);
}
// The same for the gated product (4096 x 2048, 16 tokens: 25.9 and 26.7 us with
// the down product and one launch less, 64 tokens 35.6 and 31.7; the border in
// between was not searched).
constexpr size_t kRawTokensFfn = 16;

bool raw_fits(const void* p, size_t ld) { return aligned16(p) && ld % 4 == 0; }
Image raw_image(const void* p, size_t ld, size_t rows, size_t cols) {
  Image im;
  im.p = p;
  im.ld = ld;
  im.rows = rows;
  im.cols = cols;
  im.planes = 3;
  im.dtype = OBJB_DTYPE_F32;
  return im;
}

struct LinearPlan {
  ImagePlan x, w;
  int raw = 0;
  size_t total;
};
LinearPlan plan_linear(const objb_linear_desc& d, size_t ldx, size_t ldw, const void* x, const void* w) {
  LinearPlan p;
  p.x = plan_image(x, d.x_dtype, ldx, d.tokens, d.in_features, d.x_dtype == OBJB_DTYPE_F32 ? 3 : 1);
  p.w = plan_image(w, d.w_dtype, ldw, d.out_features, d.in_features, d.w_dtype == OBJB_DTYPE_F32 ? 3 : 1);
  if (d.x_dtype == OBJB_DTYPE_F32 && raw_pays(d.tokens, d.out_features, d.w_dtype == OBJB_DTYPE_F32) &&
      raw_fits(x, ldx) && (d.w_dtype != OBJB_DTYPE_F32 || raw_fits(w, ldw))) {
    p.raw = d.w_dtype == OBJB_DTYPE_F32 ? 2 : 1;
    p.x.bytes = 0;
    if (p.raw == 2) p.w.bytes = 0;
  }
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
  // runs of rows of the column sums: 16 blocks per SM to even out the rounds, 32 rows or more in each; up to 256 rows are one
  // run, whose sums need no folding launch
  const size_t cols = (d.out_features + 255) / 256;
  const size_t want = std::max<size_t>(1, (static_cast<size_t>(sms) * 16 + cols - 1) / cols);
  p.parts = d.tokens <= 256 ? 1 : static_cast<int>(std::max<size_t>(1, std::min(want, (d.tokens + 31) / 32)));
  p.rows_per = static_cast<long long>((d.tokens + p.parts - 1) / p.parts);
  p.part_bytes = p.want_db && p.parts > 1 ? r256(static_cast<size_t>(p.parts) * d.out_features * 4) : 0;
  p.total = p.x.bytes + p.w.bytes + p.dz.bytes + p.part_bytes;
  return p;
}

struct FfnPlan {
  ImagePlan gate, up, down, x, act;
  bool raw;
  size_t total;
};
FfnPlan plan_ffn(size_t T, size_t H, size_t I, size_t O, const void* gate, const void* up, const void* down,
                 const void* x) {
  FfnPlan p;
  p.raw = T <= kRawTokensFfn && x && raw_fits(x, H);
  p.gate = plan_image(gate, OBJB_DTYPE_BF16, H, I, H, 1);
  p.up = plan_image(up, OBJB_DTYPE_BF16, H, I, H, 1);
  p.down = plan_image(down, OBJB_DTYPE_BF16, I, O, I, 1);
  p.x = plan_image(nullptr, OBJB_DTYPE_F32, H, T, H, 3);
  p.act = plan_image(nullptr, OBJB_DTYPE_F32, I, T, I, 3);
  if (p.raw) p.x.bytes = 0;
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
  if (d_z == d_y) return OBJB_FAIL(OBJB_ERR_INVALID_INPUT, action, "z and y are the same array");
  const size_t eb = elem_bytes(d.y_dtype), N = d.out_features;
  const Rows x = rows_of(d_x, d.tokens, d.in_features, ldx, d.x_dtype), w = rows_of(d_w, N, d.in_features, ldw, d.w_dtype);
  const Rows bias{d_bias, 1, N * elem_bytes(d.bias_dtype), N * elem_bytes(d.bias_dtype)};
  const Rows y{d_y, d.tokens, N * eb, ldy * eb}, z{d_z, d.tokens, N * eb, ldz * eb};
  const Rows res{d_residual, d.tokens, N * eb, ldr * eb};
  if (overlap(y, x) || overlap(y, w) || overlap(y, bias) || overlap(y, z) || (d_residual != d_y && overlap(y, res)) ||
      overlap(z, x) || overlap(z, w) || overlap(z, bias) || overlap(z, res))
    return OBJB_FAIL(OBJB_ERR_INVALID_INPUT, action, "y or z overlaps an operand or the other");
  int device = 0;
  DeviceProps props;
  OBJB_TRY(device_here(&device, &props));
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  const LinearPlan pl = plan_linear(d, ldx, ldw, d_x, d_w);
  uint8_t* ws = nullptr;
  OBJB_TRY(take_scratch(action, d_scratch, scratch_bytes, pl.total, st, &ws));
  Product p;
  Images images;
  p.raw = pl.raw;
  if (pl.raw == 2) {
    p.a = raw_image(d_w, ldw, d.out_features, d.in_features);
  } else {
    p.a = images.take(pl.w, d_w, d.w_dtype, ldw, d.out_features, d.in_features, ws);
  }
  if (pl.raw) {
    p.b = raw_image(d_x, ldx, d.tokens, d.in_features);
  } else {
    p.b = images.take(pl.x, d_x, d.x_dtype, ldx, d.tokens, d.in_features, ws + pl.w.bytes);
  }
  OBJB_TRY(images.launch(props, st));
  p.M = d.out_features;
  p.N = d.tokens;
  p.K = d.in_features;
  dev::LinearEpilogue& e = p.epi;
  e.bias = d_bias;
  e.bias_dtype = d.bias_dtype;
  e.residual = d_residual;
  e.ldr = static_cast<uint32_t>(ldr);
  e.y = d_y;
  e.ldy = static_cast<uint32_t>(ldy);
  e.z = d_z;
  e.ldz = static_cast<uint32_t>(ldz);
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
  {
    const size_t T = d.tokens, K = d.in_features, N = d.out_features;
    const Rows out[3] = {rows_of(want_dx ? d_dx : nullptr, T, K, lddx, d.x_dtype),
                         rows_of(want_dw ? d_dw : nullptr, N, K, lddw, d.dw_dtype),
                         rows_of(want_db ? d_dbias : nullptr, 1, N, N, OBJB_DTYPE_F32)};
    // (what the call reads)
    const Rows in[4] = {rows_of(d_dy, T, N, lddy, d.dy_dtype),
                        rows_of(d.activation != OBJB_ACT_NONE ? d_z : nullptr, T, N, ldz, d.dy_dtype),
                        rows_of(want_dw ? d_x : nullptr, T, K, ldx, d.x_dtype),
                        rows_of(want_dx ? d_w : nullptr, N, K, ldw, d.w_dtype)};
    bool bad = overlap(out[0], out[1]) || overlap(out[0], out[2]) || overlap(out[1], out[2]);
    for (const Rows& o : out)
      for (const Rows& i : in) bad = bad || overlap(o, i);
    if (bad) return OBJB_FAIL(OBJB_ERR_INVALID_INPUT, action, "a gradient overlaps an operand or another gradient");
  }
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
  dev::BiasFold fold;
  Images images;
  Image w, x;
  if (want_dx) w = images.take(pl.w, d_w, d.w_dtype, ldw, d.out_features, d.in_features, ws_w);
  if (want_dw) x = images.take(pl.x, d_x, d.x_dtype, ldx, d.tokens, d.in_features, ws_x);
  if (image || want_db) {
    dev::DzJob j;
    j.dy = d_dy;
    j.z = d_z;
    j.ldy = lddy;
    j.ldz = ldz;
    j.rows = static_cast<long long>(d.tokens);
    j.rows_per = pl.rows_per;
    j.N = N;
    j.dtype = d.dy_dtype;
    j.act = d.activation;
    j.pitch = static_cast<int>(pl.dz.pitch);
    j.planes = pl.dz.planes;
    j.cols = (N + 255) / 256;
    j.blocks = j.cols * pl.parts;
    j.img = image ? reinterpret_cast<uint16_t*>(ws_dz) : nullptr;
    j.part = !want_db ? nullptr : pl.parts > 1 ? reinterpret_cast<float*>(ws_part) : d_dbias;
    j.add = pl.parts == 1 && d.accumulate;
    const bool vec = aligned16(d_dy) && lddy % 8 == 0 && N % 8 == 0 && (!pl.has_act || (aligned16(d_z) && ldz % 8 == 0));
    const int image_blocks = images.blocks(props);
    OBJB_TRY(dev::with_elements(d.dy_dtype, vec, [&](auto elem, auto v) -> int {
      return launch_pdl(dev::dz_kernel<decltype(elem), decltype(v)::value>, j.blocks + images.count() * image_blocks, 256,
                        0, st, j, images.job(0), images.job(1), image_blocks);
    }));
    images.clear();
    if (want_db && pl.parts > 1 && products && pl.parts <= dev::kFoldParts)
      fold = {j.part, d_dbias, pl.parts, N, d.accumulate != 0};
    else if (want_db && pl.parts > 1)
      OBJB_TRY(launch_pdl(dev::dbias_kernel, (N + 31) / 32, 1024, 0, st, static_cast<const float*>(j.part), pl.parts, N,
                          d_dbias, static_cast<int>(d.accumulate)));
  }
  OBJB_TRY(images.launch(props, st));
  if (want_dx) {
    Product p;
    p.maj = dev::kMajMK;
    p.a = w;
    p.b = dz;
    p.M = d.in_features;
    p.N = d.tokens;
    p.K = d.out_features;
    p.epi.y = d_dx;
    p.epi.ldy = static_cast<uint32_t>(lddx);
    p.epi.y_dtype = d.x_dtype;
    p.fold = fold;
    p.next_apart = want_dw;
    fold.part = nullptr;
    OBJB_TRY(gemm(p, device, props, st));
  }
  if (want_dw) {
    Product p;
    p.maj = dev::kMajMN;
    p.a = x;
    p.b = dz;
    p.M = d.in_features;
    p.N = d.out_features;
    p.K = d.tokens;
    p.epi.y = d_dw;
    p.epi.ldy = static_cast<uint32_t>(lddw);
    p.epi.y_dtype = d.dw_dtype;
    p.apart = want_dx;  // beside dx
    p.fold = fold;
    if (d.accumulate) p.epi.residual = d_dw, p.epi.ldr = static_cast<uint32_t>(lddw);
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
  // (x is not named here: room for its planes in any case)
  *bytes = plan_ffn(num_tokens, hidden, intermediate, out_dim, d_gate, d_up, d_down, nullptr).total;
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
  // (out may lie over x, which is read before the first result is written)
  const Rows out = rows_of(d_out, 1, num_tokens * out_dim, num_tokens * out_dim, OBJB_DTYPE_F32);
  auto weight = [](const void* p, size_t n) { return rows_of(p, 1, n, n, OBJB_DTYPE_BF16); };
  if (overlap(out, weight(d_gate, intermediate * hidden)) || overlap(out, weight(d_up, intermediate * hidden)) ||
      overlap(out, weight(d_down, out_dim * intermediate)) ||
      (d_residual != d_out && overlap(out, rows_of(d_residual, 1, num_tokens * out_dim, num_tokens * out_dim, OBJB_DTYPE_F32))))
    return OBJB_FAIL(OBJB_ERR_INVALID_INPUT, action, "out overlaps a weight, or the residual without being it");
  int device = 0;
  DeviceProps props;
  OBJB_TRY(device_here(&device, &props));
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  const FfnPlan pl = plan_ffn(num_tokens, hidden, intermediate, out_dim, d_gate, d_up, d_down, d_x);
  uint8_t* ws = nullptr;
  OBJB_TRY(take_scratch(action, d_scratch, scratch_bytes, pl.total, st, &ws));
  const int bf = OBJB_DTYPE_BF16;
  Product gu;
  gu.gated = true;
  Images images;
  gu.a = images.take(pl.gate, d_gate, bf, hidden, intermediate, hidden, ws);
  ws += pl.gate.bytes;
  gu.a2 = images.take(pl.up, d_up, bf, hidden, intermediate, hidden, ws);
  ws += pl.up.bytes;
  OBJB_TRY(images.launch(props, st));
  Product dn;
  dn.a = images.take(pl.down, d_down, bf, intermediate, out_dim, intermediate, ws);
  ws += pl.down.bytes;
  if (pl.raw) {
    gu.raw = 1;
    gu.b = raw_image(d_x, hidden, num_tokens, hidden);
    // the down weights come while the gated product ends and the next one starts (26.2 -> 25.5 us at 4096 x 2048)
    if (pl.down.direct) gu.ahead = d_down, gu.ahead_bytes = out_dim * intermediate * 2;
  } else {
    gu.b = images.take(pl.x, d_x, OBJB_DTYPE_F32, hidden, num_tokens, hidden, ws);
    ws += pl.x.bytes;
  }
  OBJB_TRY(images.launch(props, st));
  gu.M = intermediate;
  gu.N = num_tokens;
  gu.K = hidden;
  gu.swiglu_limit = swiglu_limit;
  gu.epi.y = ws;  // the activations, as the planes that the down product reads
  gu.epi.ldy = static_cast<uint32_t>(pl.act.pitch);
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
  dn.epi.ldy = static_cast<uint32_t>(out_dim);
  dn.epi.residual = d_residual;
  dn.epi.ldr = static_cast<uint32_t>(out_dim);
  dn.epi.y_dtype = OBJB_DTYPE_F32;
  return gemm(dn, device, props, st);
}

}  // extern "C"
