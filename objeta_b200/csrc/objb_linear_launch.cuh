// objb_linear_launch.cuh -- host side of the tensor-core product: operands as
// the copy engine reads them, tiles, and the launch of one (instantiated per
// operand layout in linear_kk.cu, linear_mk.cu and linear_mn.cu).
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>

#include <algorithm>

#include "objb_common.h"
#include "objb_host_launch.cuh"
#include "objb_launch.h"
#include "objb_linear_gemm.cuh"

namespace objb {

// A 16-bit matrix as the copy engine reads it: 16-byte aligned, rows of `ld`
// elements (a multiple of 8), `planes` of them `rows * ld` apart; or an f32 one
// as it lies (OBJB_DTYPE_F32, `planes` those it is split into).
struct Image {
  const void* p = nullptr;
  size_t ld = 0, rows = 0, cols = 0;
  int planes = 1;
  int dtype = 0;  // OBJB_DTYPE_*
};

// The tensor map of an image: box of 64 elements by `box_rows` rows, all planes.
int linear_encode(CUtensorMap* map, const Image& im, int box_rows);

// One product: A (a2: the up rows of a gated one), B, D's epilogue.
struct Product {
  int maj = dev::kMajKK;
  Image a, a2, b;
  int raw = 0;  // 1: b is f32 as it lies (three planes in the stages), 2: a too
  const void* ahead = nullptr;  // what the next product reads
  size_t ahead_bytes = 0;
  dev::BiasFold fold;
  bool next_apart = false, apart = false;  // GemmArgs
  bool gated = false;
  size_t M = 0, N = 0, K = 0;
  dev::LinearEpilogue epi;
  float swiglu_limit = 0.0f;
};

constexpr size_t kLinRing = 216 * 1024;    // bytes of stages: three of f32 x f32 pair tiles
constexpr size_t kLinRingTwo = 104 * 1024;  // the same with two CTAs per SM

inline size_t ceil_div(size_t a, size_t b) { return (a + b - 1) / b; }

// A product's tile: rm rows per accumulator, mt accumulators and bn columns
// per CTA or pair, k split over a cluster.
struct Tile {
  int rm = 128, bn = 0, split = 1, chunk_kb = 0, unit = 1;
  size_t ring = kLinRing;
};

enum TileKind { kDirect, kPair, kSingle };

template <int MAJ, int BN, int CG, int MT, bool GATED, bool PROMOTE, int PB, int RAW = 0>
int launch_gemm(const Product& p, const Tile& tile, int device, const DeviceProps& props, cudaStream_t st) {
  using SH = dev::LinShape<MAJ, BN, CG, MT, GATED, PROMOTE, PB, RAW>;
  dev::GemmArgs g;
  g.M = static_cast<int>(p.M);
  g.N = static_cast<long long>(p.N);
  g.nkb = static_cast<int>((p.K + 63) / 64);
  g.pa = p.a.planes;
  g.rm = tile.rm;
  g.bn = tile.bn;
  g.split = tile.split;
  g.chunk_kb = PROMOTE ? tile.chunk_kb : g.nkb;
  g.swiglu_limit = p.swiglu_limit;
  g.epi = p.epi;
  g.fold = p.fold;
  g.next_apart = p.next_apart;
  g.apart = p.apart;
  g.ahead = static_cast<const uint8_t*>(p.ahead);
  g.ahead_bytes = p.ahead_bytes;
  OBJB_TRY(device_error_word(device, &g.err));
  const size_t mt = static_cast<size_t>(GATED ? 64 : MT * tile.rm) * CG;
  g.tiles_m = static_cast<int>((p.M + mt - 1) / mt);
  g.tiles_n = static_cast<int>((p.N + tile.bn - 1) / tile.bn);
  const size_t a_rows = static_cast<size_t>(MT) * (MAJ != dev::kMajKK || GATED ? 128 : tile.rm);
  g.unit = PROMOTE ? tile.unit : 1;
  const size_t stage = g.unit * 128 * (g.pa * a_rows + static_cast<size_t>(PB) * (tile.bn / CG));
  const size_t raw = RAW ? g.unit * 256 * ((RAW == 2 ? tile.rm : 0) + static_cast<size_t>(tile.bn)) : 0;
  const long long tiles = static_cast<long long>(g.tiles_m) * g.tiles_n;
  const int csize = CG == 2 ? 2 : tile.split;
  const long long at_once = static_cast<long long>(props.sm_count) * (tile.ring == kLinRingTwo ? 2 : 1) / csize;
  // A tile in f32, exchanged over the stages or, where another tile is on its way into them, behind (1000 tokens of
  // 4096 x 2048, replayed from a graph: 139 -> 131 us the whole FFN, 149 as a call among others; with one tile per CTA
  // the stages are worth more: 250 tokens 66.6, over them 61.4).
  const size_t partial = static_cast<size_t>(tile.bn) * 512;
  const bool behind = GATED && tile.split == 1 && tiles > at_once;
  const size_t room = tile.ring - (behind ? partial : 0);
  g.nstages = static_cast<int>(std::max<size_t>(2, std::min<size_t>(dev::kLinStagesMax, room / (stage + raw))));
  // A group keeps to its own stages (a wait for a phase that is not the next one of its barrier falls through), so
  // that they are a multiple of the groups.
  g.conv_groups = g.nstages >= dev::kConvWarps ? dev::kConvWarps : g.nstages >= 4 ? 4 : 2;
  if (RAW) g.nstages -= g.nstages % g.conv_groups;
  size_t smem = g.nstages * (stage + raw);
  g.exchange = behind ? static_cast<uint32_t>(smem) : 0;
  if (GATED || tile.split > 1) smem = std::max(smem, g.exchange + partial);
  smem += 1024 + (128 - tile.rm) * 128;  // an MMA reads 128 rows, those past rm for nothing
  // A kernel that takes all of tensor memory leaves no room for another of these on its SM (the least take 78 KB): of
  // two clusters that share SMs, each might hold what the other waits for.
  if (SH::kCols == 512) smem = std::max(smem, size_t{152} * 1024);
  const uint32_t half = p.a.dtype == OBJB_DTYPE_F16 ? 0 : 1;
  g.idesc = (1u << 4) | (half << 7) | (half << 10) | (static_cast<uint32_t>(MAJ != dev::kMajKK) << 15) |
            (static_cast<uint32_t>(MAJ == dev::kMajMN) << 16) | (static_cast<uint32_t>(tile.bn >> 3) << 17) |
            (static_cast<uint32_t>(128 * CG >> 4) << 24);
  CUtensorMap ma, ma2, mb;
  OBJB_TRY(linear_encode(&ma, p.a, MAJ == dev::kMajKK && !GATED ? tile.rm : 64));
  if (GATED)
    OBJB_TRY(linear_encode(&ma2, p.a2, 64));
  else
    ma2 = ma;
  OBJB_TRY(linear_encode(&mb, p.b, MAJ == dev::kMajMN ? 64 : tile.bn / CG));
  auto kernel = dev::lin_gemm_kernel<MAJ, BN, CG, MT, GATED, PROMOTE, PB, RAW>;
  OBJB_TRY(ensure_smem_attr(kernel, device, smem));
  const bool one_each = tile.split > 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>((one_each ? tiles : std::min(tiles, at_once)) * csize));
  cfg.blockDim = dim3(SH::kThreads);
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

// The kernel that a tile of this layout takes (linear_kk.cu, linear_mk.cu, linear_mn.cu).
int launch_kk(const Product& p, TileKind kind, const Tile& t, int device, const DeviceProps& props, cudaStream_t st);
int launch_mk(const Product& p, TileKind kind, const Tile& t, int device, const DeviceProps& props, cudaStream_t st);
int launch_mn(const Product& p, TileKind kind, const Tile& t, int device, const DeviceProps& props, cudaStream_t st);

// Most columns of a single CTA's tile, and with two CTAs on an SM.
inline int single_columns(int maj, int pb) { return pb == 1 ? 128 : maj == dev::kMajMN ? 64 : 80; }
inline int two_columns(int maj, int pb) { return pb == 1 ? 64 : maj == dev::kMajMN ? 0 : 32; }

}  // namespace objb
