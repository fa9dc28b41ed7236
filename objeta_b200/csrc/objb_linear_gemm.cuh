// objb_linear_gemm.cuh -- the tensor-core product under the dense operators
// (linear.cu): D[n][m] = sum_k A(m, k) B(n, k), f32 accumulation.
//
// A and B are 16-bit matrices in memory ("images"), each either with k along
// its rows' elements (K-major) or with k along its rows (the transposed read
// of the gradients, MN-major); an f32 operand has three bf16 planes (the upper,
// middle and lower 8 bits of its significand), whose products are taken pair
// by pair.  Rows of A are the rows m of a tcgen05.mma, rows of B its N, so a
// tensor-memory lane is a row m and a warp's 32 lanes store 32 neighbouring
// elements of D's row n: no transposition on the way out.
//
// One warp issues TMA copies into a ring of 128-byte-swizzled stages (`unit`
// k-blocks of 64, all planes), one warp the MMAs, the others the epilogue.
// A turn of the producer costs about 145 ns and a copy 35 more, a turn of the
// MMA warp 150, whatever the tile: small tiles take several k-blocks per stage
// (16.4 -> 11.6 us for one token by 4096 x 4096 in 64 CTAs).  Accumulators:
//   * PROMOTE.  The tensor core adds into its f32 accumulators with
//     truncation, so their error grows with the number of MMAs in one
//     accumulator; the epilogue warps therefore take the accumulators into
//     registers every chunk_kb k-blocks (two buffers) and add there, rounded
//     to nearest.  Products of planes i and j are 2^-8 (i + j) of the main one;
//     those of i + j > 2 are below f32 and left out.
//     CG 1, planes side by side: B's planes lie behind one another, so one MMA
//     of N = 3 bn takes a plane of A against all of them, plane 1 against two
//     of them into columns bn.. (the products of i + j = 1 and 2), plane 2
//     against one into columns 2 bn..; an MMA takes 39 clocks or more, so a
//     third (half) of the MMAs is what counts up to bn 64.
//     CG 2: one MMA per pair of planes, the cross products into two buffers of
//     their own, each read once per kCrossChunks chunks (their sum is 2^-8 of
//     the main one, so 16 times the MMAs err less); twice the columns per tile.
//   * else straight from tensor memory into the epilogue, which rounds to 16
//     bits: two accumulators of 256 columns, all of tensor memory, for k up to
//     65536 (bf16) or 16384 (f16; direct_k).  The ring goes on filling while a
//     tile is drained.
// CTA pairs (CG 2, cta_group::2) share each MMA: M 256, half of B's rows from
// each CTA's shared memory.  MT accumulators per CTA (rows m0 + a * rm) share
// B's stage.  An L2-fed SM takes in about 64 bytes per clock, an MMA of 128 x
// 256 x 64 per CTA pair half lasts 512 clocks: 512 x 256 tiles (48 KB a
// k-block and CTA, 1024 clocks) are fed in time, 256 x 256 ones (32 KB, 512
// clocks) were not (140 against 98 us at 4096^3).
//   * Few tiles (CG 1): `split` CTAs of a cluster share a tile's k-blocks and
//     fold their partial tiles through distributed shared memory in rank
//     order: one launch, no atomics, no scratch.
//   * RAW: an f32 operand of few tokens is not laid out in planes by a launch
//     of its own: a second producer copies it as it lies, eight more warps
//     split it into the planes of the stages (RAW 1: B; 2: both).  (Copies by
//     the splitting warps themselves, into registers or shared memory, cost
//     a memory latency per k-block: the proxy fence waits for them.)
//   * GATED: A is 64 rows of the gate and the same 64 rows of up; the epilogue
//     pairs lanes i and i + 64 through shared memory (behind the stages, where
//     a CTA has more than one tile, so that the next one's MMAs go on).
//
// What it comes to (bf16, 4096 x 4096 x 4096, 20 launches replayed from a graph):
// 99 us, 1389 TFLOP/s, tensor pipe 95 % busy in the main loop (alone, with cold
// caches, 108 us and 70 % over the launch); the library's product 95 us.  In long
// runs both are bound by power (117 and 110 us at 1.48 GHz).
// f32 results: 256 x 128 pair tiles 53 to 55 % busy, bound by the planes that
// an SM takes in.  Few tokens: bound by w (37 x 2048 x 151936: 6.0 TB/s).
// Registers are capped to what the CTAs on an SM leave, and some kernels spill:
// the direct 512 x 256 tiles 88 to 92 bytes a thread at 96 registers, two CTAs of
// 64 columns on an SM 296 at 80 (32 columns: 84), the splitting ones 16 to 72 at
// 96; the promoted pair and 128- and 80-column tiles none.
#pragma once

#include <cuda.h>

#include "objb_linear.cuh"
#include "objb_moe.cuh"
#include "objb_pipe.cuh"
#include "objb_tc.cuh"

namespace objb {
namespace dev {

enum { kMajKK = 0, kMajMK = 1, kMajMN = 2 };  // A, B: K-major both; A MN-major; both MN-major

constexpr int kLinBK = 64;        // k of a stage: 128 bytes, one swizzle row
constexpr int kLinStagesMax = 12;
constexpr int kCrossChunks = 16;  // chunks of a cross product's buffer
// Longest k of one accumulator that is not promoted: what truncation takes from a sum of one sign stays below a fifth of
// the result's half step.  f16 (2^-11, 4.9e-4): 8.9e-5 at 16384, 3.9e-4 at 65536; bf16 (2^-9 at least, 2e-3), whose
// products need fewer bits: 1.2e-4 at 65536.
constexpr size_t direct_k(bool f16) { return f16 ? 16384 : 65536; }
constexpr int kConvWarps = 8;
// producer, MMA, eight (PROMOTE) or sixteen epilogue warps, second MMA warp (RAW: producer of raw k-blocks), RAW: the
// converting warps
constexpr int lin_threads(bool promote, bool raw = false) { return promote ? 352 + (raw ? 32 * kConvWarps : 0) : 608; }

// The column sums of dz's runs of rows (dz_kernel), folded by the epilogue warps
// while they wait for their first tile: a launch less.
struct BiasFold {
  const float* part = nullptr;  // [parts][n], or null
  float* to = nullptr;
  int parts = 0, n = 0;
  bool add = false;
};
constexpr int kFoldParts = 128;  // beyond, the fold would outlast that wait

// Group w of 32 columns: a lane's runs in order.
__device__ __forceinline__ void fold_bias(const BiasFold& f, int w) {
  const int c = w * 32 + (threadIdx.x & 31);
  if (c >= f.n) return;
  float s = 0.0f;
  for (int i = 0; i < f.parts; i += 16) {
    float v[16];
#pragma unroll
    for (int u = 0; u < 16; ++u) v[u] = i + u < f.parts ? f.part[static_cast<size_t>(i + u) * f.n + c] : 0.0f;
#pragma unroll
    for (int u = 0; u < 16; ++u) s += v[u];
  }
  f.to[c] = f.add ? f.to[c] + s : s;
}

struct GemmArgs {
  int M;                  // rows of A (GATED: features)
  long long N;            // rows of B
  int nkb;                // k-blocks
  int tiles_m, tiles_n;
  int rm;                 // rows of an accumulator in use (128, or fewer to even out the rounds of the grid)
  int bn;                 // columns of a tile in use (at most BN)
  int pa;                 // planes of A
  int split;              // CTAs of a cluster per tile (CG 1)
  int chunk_kb;           // k-blocks per accumulator chunk, a multiple of unit
  int nstages, unit;      // stages of `unit` k-blocks
  uint32_t exchange;      // GATED, split: where in the stages' memory a tile is exchanged
  int conv_groups;        // RAW: groups of converting warps, which take the stages in turn; divides nstages
  uint32_t idesc;
  // Two launches that do not read each other's results run side by side: the
  // first lets the next one start only when what came before it is complete
  // (next_apart); the second does not wait but at its end, so that what comes
  // behind it finds both done (apart).
  bool next_apart, apart;
  float swiglu_limit;
  unsigned* err;
  LinearEpilogue epi;
  BiasFold fold;
  const uint8_t* ahead;  // bytes that the next product reads, brought into L2 behind this one's own (16-byte
  size_t ahead_bytes;    // aligned, whole 16-byte quads); may be null
};

// An oct of 8 f32, and its three planes, `plane` bytes apart.
__device__ __forceinline__ void raw_take(uint32_t from, float (&v)[8]) {
#pragma unroll
  for (int h = 0; h < 2; ++h)
    asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];"
                 : "=f"(v[4 * h]), "=f"(v[4 * h + 1]), "=f"(v[4 * h + 2]), "=f"(v[4 * h + 3])
                 : "r"(from + h * 16)
                 : "memory");
}
__device__ __forceinline__ void raw_split(const float (&v)[8], uint32_t to, uint32_t plane) {
  uint32_t u[4][3];
#pragma unroll
  for (int i = 0; i < 4; ++i) split3_pair(v[2 * i], v[2 * i + 1], u[i]);
#pragma unroll
  for (int j = 0; j < 3; ++j)
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(to + j * plane), "r"(u[0][j]), "r"(u[1][j]),
                 "r"(u[2][j]), "r"(u[3][j])
                 : "memory");
}

// swiglu's clamps (fminf, fmaxf, as the reference has them) turn NaN into the limit: a bad token would come out finite.
__device__ __forceinline__ float swiglu_keeping_nan(float g, float u, float limit) {
  const float v = swiglu(g, u, limit);
  return g == g && u == u ? v : g + u;
}

// SWIZZLE_128B operand tiles, without their address.  K-major: rows of 128
// bytes, 8-row groups 1024 bytes apart.  MN-major: 64 rows x 64 k as 64 k rows
// of 128 bytes; 8-k groups 1024 bytes apart (stride offset), the next 64 rows
// behind this chunk's planes (leading offset).
template <bool MN>
__device__ __forceinline__ uint64_t lin_desc(int planes) {
  uint64_t d = static_cast<uint64_t>((MN ? 8192 * planes : 16) >> 4) << 16;
  d |= static_cast<uint64_t>(1024 >> 4) << 32;
  d |= static_cast<uint64_t>(1) << 46;
  d |= static_cast<uint64_t>(2) << 61;
  return d;
}

template <int CG>
__device__ __forceinline__ void lin_mma(uint32_t d_tmem, uint64_t a, uint64_t b, uint32_t idesc, bool accumulate) {
  if constexpr (CG == 1)
    asm volatile(
        "{\n\t.reg .pred p, e;\n\telect.sync _|e, 0xffffffff;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d_tmem),
        "l"(a), "l"(b), "r"(idesc), "r"(accumulate ? 1u : 0u));
  else
    asm volatile(
        "{\n\t.reg .pred p, e;\n\telect.sync _|e, 0xffffffff;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "@e tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d_tmem),
        "l"(a), "l"(b), "r"(idesc), "r"(accumulate ? 1u : 0u));
}

// 3-D tiled load (x along a row, row; the box holds all planes).  x is a multiple of 64 elements.
// With CG 2 the bytes are counted on the even CTA's barrier.
template <int CG>
__device__ __forceinline__ void lin_tma(uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint32_t bar) {
  if constexpr (CG == 1)
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], "
        "[%5];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(bar)
        : "memory");
  else
    asm volatile(
        "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, "
        "{%2, %3, %4}], [%5];" ::"r"(dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(bar)
        : "memory");
}

__device__ __forceinline__ uint32_t lin_mapa(uint32_t addr, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
__device__ __forceinline__ float lin_ld_cluster(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}

__device__ __forceinline__ void tmem_ld32(uint32_t taddr, float (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,"
      "%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=f"(r[0]), "=f"(r[1]), "=f"(r[2]), "=f"(r[3]), "=f"(r[4]), "=f"(r[5]), "=f"(r[6]), "=f"(r[7]), "=f"(r[8]),
        "=f"(r[9]), "=f"(r[10]), "=f"(r[11]), "=f"(r[12]), "=f"(r[13]), "=f"(r[14]), "=f"(r[15]), "=f"(r[16]),
        "=f"(r[17]), "=f"(r[18]), "=f"(r[19]), "=f"(r[20]), "=f"(r[21]), "=f"(r[22]), "=f"(r[23]), "=f"(r[24]),
        "=f"(r[25]), "=f"(r[26]), "=f"(r[27]), "=f"(r[28]), "=f"(r[29]), "=f"(r[30]), "=f"(r[31])
      : "r"(taddr));
}
template <int G>
__device__ __forceinline__ void tmem_ldf(uint32_t taddr, float (&r)[G]) {
  if constexpr (G == 32) {
    tmem_ld32(taddr, r);
  } else {
    uint32_t u[G];
    if constexpr (G == 16)
      tmem_ld16(taddr, u);
    else
      tmem_ld8(taddr, u);
#pragma unroll
    for (int i = 0; i < G; ++i) r[i] = __uint_as_float(u[i]);
  }
}

// Whether phase `parity` of a barrier is over, without waiting.
__device__ __forceinline__ bool lin_test(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\tmbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(smem_u32(bar)), "r"(parity)
      : "memory");
  return __all_sync(0xFFFFFFFFu, ok != 0);
}

// mbar_wait_bounded by a whole warp: all lanes go on or all give up.
__device__ __forceinline__ bool lin_wait(uint64_t* bar, uint32_t parity, unsigned* err, unsigned code,
                                         unsigned* abort) {
  return __all_sync(0xFFFFFFFFu, mbar_wait_bounded(bar, parity, err, code, abort));
}

// Tile t of the grid, in bands of 8 tiles of n: the tiles that run together
// share few rows of A and of B.
__device__ __forceinline__ void lin_tile(const GemmArgs& g, int t, int* tm, int* tn) {
  const int band = 8 * g.tiles_m;
  const int b = t / band, r = t - b * band;
  const int width = g.tiles_n - b * 8 < 8 ? g.tiles_n - b * 8 : 8;
  *tm = r / width;
  *tn = b * 8 + r - *tm * width;
}

// BN: columns of a tile at most; PB: planes of B.
template <int MAJ, int BN, int CG, int MT, bool GATED, bool PROMOTE, int PB, int RAW>
struct LinShape {
  static constexpr bool kWideB = CG == 1 && PB > 1;         // planes side by side in N
  static constexpr int kSet = MT * BN * (kWideB ? PB : 1);  // accumulator columns of one set
  static constexpr int kUsed = PROMOTE ? (CG == 2 && PB > 1 ? 4 : 2) * kSet : kSet;
  static constexpr int pow2(int v) { return v <= 32 ? 32 : v <= 64 ? 64 : v <= 128 ? 128 : v <= 256 ? 256 : 512; }
  static constexpr int kCols = pow2(kUsed);
  static constexpr int kThreads = lin_threads(PROMOTE, RAW != 0);
  static constexpr bool kCross = PROMOTE && CG == 2 && PB > 1;  // cross products in their own accumulators
  static constexpr bool kTwoIssue = !PROMOTE || kCross;         // a second warp issues MMAs
  static constexpr int kBlocks = PROMOTE && CG == 1 && BN <= 64 && kCols <= 256 && !RAW ? 2 : 1;  // CTAs an SM has room for
  static_assert(kUsed <= 512, "tensor memory columns");
  static_assert(!GATED || (MAJ == kMajKK && MT == 1 && PROMOTE), "gated products are K-major, one accumulator");
  static_assert(!RAW || (MAJ == kMajKK && CG == 1 && PROMOTE && PB == 3 && !(GATED && RAW == 2)), "raw operands");
  static_assert(!(kWideB && MAJ == kMajMN) || BN < 128, "planes side by side of one 64-row chunk");
  static_assert(PROMOTE ? MT == 1 : CG == 2 && MT == 2 && PB == 1, "one promoted accumulator, or a pair of two direct ones");
};

template <int MAJ, int BN, int CG, int MT, bool GATED, bool PROMOTE, int PB, int RAW>
__global__ void __launch_bounds__(LinShape<MAJ, BN, CG, MT, GATED, PROMOTE, PB, RAW>::kThreads,
                                  LinShape<MAJ, BN, CG, MT, GATED, PROMOTE, PB, RAW>::kBlocks)
    lin_gemm_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_a2,
                    const __grid_constant__ CUtensorMap map_b, const GemmArgs g) {
  using SH = LinShape<MAJ, BN, CG, MT, GATED, PROMOTE, PB, RAW>;
  constexpr bool A_MN = MAJ != kMajKK, B_MN = MAJ == kMajMN;
  constexpr int kWarps = PROMOTE ? 8 : 16;        // epilogue warps
  constexpr int HN = MT * BN * 4 / kWarps;        // columns of each
  constexpr int G = HN % 32 == 0 ? 32 : HN % 16 == 0 ? 16 : 8;  // of one tensor-memory load
  constexpr int P = G < 16 ? G : 16;              // of one step of the epilogue
  constexpr int kSet = SH::kSet;
  constexpr uint32_t kCols = SH::kCols;

  extern __shared__ uint8_t lin_smem[];
  __shared__ alignas(8) uint64_t full[kLinStagesMax], empty[kLinStagesMax], t_full[2], t_empty[2], c_full[2], c_empty[2];
  __shared__ alignas(8) uint64_t raw_full[RAW ? kLinStagesMax : 1], raw_empty[RAW ? kLinStagesMax : 1];
  __shared__ uint32_t s_tmem;
  __shared__ unsigned s_abort;
  uint8_t* stages = lin_smem + ((1024u - (smem_u32(lin_smem) & 1023u)) & 1023u);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = CG == 2 || g.split > 1 ? cluster_ctarank() : 0;
  const int csize = CG == 2 ? 2 : g.split;

  if (warp == 0 && lane == 0) {
    for (int i = 0; i < g.nstages; ++i) mbar_init(&full[i], (RAW < 2 ? 1 : 0) + (RAW ? kConvWarps / g.conv_groups : 0)), mbar_init(&empty[i], SH::kTwoIssue ? 2 : 1);
    if (RAW)
      for (int i = 0; i < g.nstages; ++i) mbar_init(&raw_full[i], 1), mbar_init(&raw_empty[i], kConvWarps / g.conv_groups);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&t_full[i], 1);
      mbar_init(&t_empty[i], 8 * CG);  // PROMOTE: all epilogue warps; else the eight of accumulator i
      mbar_init(&c_full[i], 1);
      mbar_init(&c_empty[i], 8 * CG);
    }
    s_abort = 0;
    fence_mbar_init();
  }
  if (warp == 1) {
    if constexpr (CG == 1)
      tmem_alloc(&s_tmem, kCols);
    else
      tmem_alloc_pair(&s_tmem, kCols);
  }
  tc_fence_before_sync();
  __syncthreads();
  if (csize > 1) cluster_sync_all();  // the peers' barriers exist before any arrival
  tc_fence_after_sync();
  const uint32_t tmem = s_tmem;
  if (!g.next_apart) asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (!g.apart) asm volatile("griddepcontrol.wait;" ::: "memory");
  if (g.next_apart) asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  const int ntiles = g.tiles_m * g.tiles_n;
  const int first = blockIdx.x / csize, step = gridDim.x / csize;
  const int krank = CG == 1 ? static_cast<int>(rank) : 0;
  const int kb0 = static_cast<int>(static_cast<long long>(g.nkb) * krank / g.split);
  const int kb1 = static_cast<int>(static_cast<long long>(g.nkb) * (krank + 1) / g.split);
  // A k-block of a stage: A's accumulators (all planes of each: K-major planes
  // of rm rows; MN-major two 64-row chunks of planes), then B's planes.
  const uint32_t b_rows = g.bn / CG;  // of B in this CTA's shared memory
  const uint32_t a_plane = A_MN || GATED ? 8192 : g.rm * 128, b_plane = B_MN ? 8192 : b_rows * 128;
  const uint32_t a_acc = g.pa * (A_MN || GATED ? 16384 : a_plane);
  const uint32_t b_at = MT * a_acc, kb_bytes = b_at + PB * b_rows * 128, stage_bytes = g.unit * kb_bytes;
  const uint32_t raw_kb_bytes = ((RAW == 2 ? g.rm : 0) + b_rows) * 256;  // behind the stages
  const uint32_t raw_at = smem_u32(stages) + g.nstages * stage_bytes;
  // first row of A of this CTA's part of tile row tm
  const int cta_rows = GATED ? 64 : MT * g.rm;
  auto row0 = [&](int tm) { return (tm * CG + (CG == 2 ? static_cast<int>(rank) : 0)) * cta_rows; };

  if (warp == 0) {
    if (lane == 0 && RAW < 2) {
      // ---- producer
      int issued = 0, st = 0;
      uint32_t phase = 1;  // of empty[st]: the first round finds every stage free
      bool ok = true;
      for (int t = first; t < ntiles && ok; t += step) {
        int tm, tn;
        lin_tile(g, t, &tm, &tn);
        const int m0 = row0(tm);
        const int n0 = tn * g.bn + (CG == 2 ? rank * b_rows : 0);
        for (int kb = kb0; kb < kb1;) {
          if (!mbar_wait_bounded(&empty[st], phase, g.err, kErrEmptyWaitTimeout, &s_abort)) {
            ok = false;
            break;
          }
          uint32_t bar = smem_u32(&full[st]);
          const int n = kb1 - kb < g.unit ? kb1 - kb : g.unit;
          if (rank == 0 || CG == 1) mbar_arrive_expect_tx(&full[st], CG * n * (RAW ? b_at : kb_bytes));
          if (CG == 2) bar = lin_mapa(bar, 0);
          uint32_t dst = smem_u32(stages) + st * stage_bytes;
          for (const int end = kb + n; kb < end; ++kb, dst += kb_bytes) {
#pragma unroll
            for (int a = 0; a < MT; ++a) {
              const uint32_t to = dst + a * a_acc;
              if constexpr (GATED) {
                lin_tma<CG>(to, &map_a, kb * 64, m0, 0, bar);
                lin_tma<CG>(to + 8192, &map_a2, kb * 64, m0, 0, bar);
              } else if constexpr (A_MN) {
                lin_tma<CG>(to, &map_a, m0 + a * 128, kb * 64, 0, bar);
                lin_tma<CG>(to + g.pa * 8192, &map_a, m0 + a * 128 + 64, kb * 64, 0, bar);
              } else {
                lin_tma<CG>(to, &map_a, kb * 64, m0 + a * g.rm, 0, bar);
              }
            }
            if constexpr (RAW != 0) {
            } else if constexpr (B_MN) {
              for (uint32_t c = 0; c < b_rows; c += 64)
                lin_tma<CG>(dst + b_at + c * 128 * PB, &map_b, n0 + c, kb * 64, 0, bar);
            } else {
              lin_tma<CG>(dst + b_at, &map_b, kb * 64, n0, 0, bar);
            }
          }
          ++issued;
          if (++st == g.nstages) st = 0, phase ^= 1;
        }
      }
      if (*reinterpret_cast<volatile unsigned*>(&s_abort)) {
        // a wait ran out: let the copies in flight land before shared memory goes
        for (int i = issued > g.nstages ? issued - g.nstages : 0; i < issued && (CG == 1 || rank == 0); ++i)
          if (!mbar_wait_bounded(&full[i % g.nstages], (i / g.nstages) & 1, g.err, kErrDrainTimeout)) break;
      }
      if (g.ahead) {
        constexpr uint32_t kPiece = 4096;
        for (size_t at = static_cast<size_t>(blockIdx.x) * kPiece; at < g.ahead_bytes; at += gridDim.x * size_t{kPiece}) {
          const uint32_t n = g.ahead_bytes - at < kPiece ? static_cast<uint32_t>(g.ahead_bytes - at) : kPiece;
          asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(g.ahead + at), "r"(n) : "memory");
        }
      }
    }
    __syncwarp();
  } else if (RAW && warp == 10) {
    if (lane == 0) {
      // ---- producer of raw k-blocks: A's rows (RAW 2), then B's, 256 bytes each
      int issued = 0, st = 0;
      uint32_t phase = 1;
      bool ok = true;
      for (int t = first; t < ntiles && ok; t += step) {
        int tm, tn;
        lin_tile(g, t, &tm, &tn);
        for (int kb = kb0; kb < kb1;) {
          if (!mbar_wait_bounded(&raw_empty[st], phase, g.err, kErrEmptyWaitTimeout, &s_abort)) {
            ok = false;
            break;
          }
          const uint32_t bar = smem_u32(&raw_full[st]);
          const int n = kb1 - kb < g.unit ? kb1 - kb : g.unit;
          mbar_arrive_expect_tx(&raw_full[st], n * raw_kb_bytes);
          uint32_t dst = raw_at + st * g.unit * raw_kb_bytes;
          for (const int end = kb + n; kb < end; ++kb, dst += raw_kb_bytes) {
            if (RAW == 2) lin_tma<1>(dst, &map_a, kb * 64, row0(tm), 0, bar);
            lin_tma<1>(dst + (RAW == 2 ? g.rm * 256 : 0), &map_b, kb * 64, tn * g.bn, 0, bar);
          }
          ++issued;
          if (++st == g.nstages) st = 0, phase ^= 1;
        }
      }
      if (*reinterpret_cast<volatile unsigned*>(&s_abort))
        for (int i = issued > g.nstages ? issued - g.nstages : 0; i < issued; ++i)
          mbar_wait_bounded(&raw_full[i % g.nstages], (i / g.nstages) & 1, g.err, kErrDrainTimeout);
    }
    __syncwarp();
  } else if (RAW && warp > 10) {
    // ---- converter: the octs of 8 elements of every conv_groups-th stage, a
    // thread's kConvGroup at a time.  A stage takes about 0.6 us from its
    // arrival on (waits, splitting, proxy fence), whatever its size: so several
    // are under way at once.
    constexpr int kConvGroup = 4;
    const int kThreads = 32 * kConvWarps / g.conv_groups;
    const int tid = (threadIdx.x - 352) & (kThreads - 1);
    const int a_octs = RAW == 2 ? g.rm * 8 : 0, octs = a_octs + static_cast<int>(b_rows) * 8;
    const int at0 = tid / octs, oct0 = tid - at0 * octs;
    int st = 0, turn = (threadIdx.x - 352) / kThreads;  // stages until this group's next
    uint32_t phase = 0;                                 // of raw_full[st]
    bool ok = true;
    for (int t = first; t < ntiles && ok; t += step)
      for (int kb = kb0; kb < kb1; kb += g.unit) {
        if (turn-- > 0) {
          if (++st == g.nstages) st = 0, phase ^= 1;
          continue;
        }
        turn = g.conv_groups - 1;
        if (!lin_wait(&raw_full[st], phase, g.err, kErrFullWaitTimeout, &s_abort) ||
            !lin_wait(&empty[st], phase ^ 1, g.err, kErrEmptyWaitTimeout, &s_abort)) {
          ok = false;
          break;
        }
        const int n = kb1 - kb < g.unit ? kb1 - kb : g.unit;
        const uint32_t from = raw_at + st * g.unit * raw_kb_bytes, to = smem_u32(stages) + st * stage_bytes;
        int at = at0, oct = oct0;  // this thread's next oct: k-block of the stage, place in it
        while (at < n) {
          float v[kConvGroup][8];
          uint32_t dst[kConvGroup], plane[kConvGroup];
          bool have[kConvGroup];
#pragma unroll
          for (int u = 0; u < kConvGroup; ++u) {
            have[u] = at < n;
            if (!have[u]) continue;
            raw_take(from + at * raw_kb_bytes + oct * 32, v[u]);
            const bool of_a = oct < a_octs;
            const int i = of_a ? oct : oct - a_octs, r = i >> 3;
            dst[u] = to + at * kb_bytes + (of_a ? 0 : b_at) + r * 128 + (((i ^ r) & 7) << 4);
            plane[u] = of_a ? a_plane : b_plane;
            oct += kThreads;
            while (oct >= octs) oct -= octs, ++at;
          }
#pragma unroll
          for (int u = 0; u < kConvGroup; ++u)
            if (have[u]) raw_split(v[u], dst[u], plane[u]);
        }
        fence_async_shared();
        __syncwarp();
        if (lane == 0) mbar_arrive(&full[st]), mbar_arrive(&raw_empty[st]);
        if (++st == g.nstages) st = 0, phase ^= 1;
      }
  } else if (warp == 1 || (!RAW && warp == SH::kThreads / 32 - 1)) {
    const int role = warp == 1 ? 0 : 1;
    if ((CG == 1 || rank == 0) && (role == 0 || SH::kTwoIssue)) {
      // ---- MMA issue.  The tensor core takes an MMA when the one before it is
      // nearly done, so whatever a warp does between two MMAs beyond that time
      // idles it (a turn's 260 clocks of waits, addresses and branches).  So
      // two warps issue, each for accumulators of its own (the second: direct
      // accumulator 1, or the cross products), and the next k-block's
      // bookkeeping is done between this one's MMAs.
      int st = 0, cc = 0, tt = 0;
      uint32_t phase = 0;  // of full[st]
      bool ok = true;
      constexpr uint32_t kStepA = (A_MN ? 2048 : 32) >> 4, kStepB = (B_MN ? 2048 : 32) >> 4;
      const uint64_t base_a = lin_desc<A_MN>(g.pa), base_b = lin_desc<B_MN>(SH::kWideB ? 1 : PB);
      // (side by side, an MN-major B is one 64-row chunk and its planes are the next rows)
      const uint32_t plane_a = a_plane >> 4, plane_b = b_plane >> 4;
      const uint32_t n_step = static_cast<uint32_t>(g.bn >> 3) << 17;  // bn columns in the instruction descriptor
      const uint32_t ring = smem_u32(stages) & 0x3FFFFu;  // (in a cluster a shared address carries the CTA's rank
                                                          // above the 18 bits a descriptor has room for)
      const uint32_t a_at = PROMOTE ? 0 : role * a_acc;
      uint32_t sa = ring, head = ring;  // this k-block's place, its stage's
      int left = g.unit;                // k-blocks left in its stage
      bool ready = false;               // its stage is known to be full
      const int chunk = !PROMOTE ? g.nkb : role == 0 ? g.chunk_kb : kCrossChunks * g.chunk_kb;
      uint64_t* const chunk_full = role == 0 ? t_full : c_full;
      uint64_t* const chunk_empty = role == 0 ? t_empty : c_empty;
      const uint32_t d0 = tmem + (PROMOTE ? 2 * kSet : BN) * role;
      for (int t = first; t < ntiles && ok; t += step, ++tt) {
        if (!PROMOTE && tt >= 1)  // the accumulator is drained of the tile before
          ok = lin_wait(&t_empty[role], (tt - 1) & 1, g.err, kErrEmptyWaitTimeout, &s_abort);
        for (int kb = kb0; kb < kb1 && ok; ++cc) {
          // PROMOTE: chunk cc into buffer cc & 1; else the tile into accumulator `role`
          const int buf = PROMOTE ? cc & 1 : 0;
          if (PROMOTE && cc >= 2 &&
              !lin_wait(&chunk_empty[buf], ((cc >> 1) - 1) & 1, g.err, kErrEmptyWaitTimeout, &s_abort)) {
            ok = false;
            break;
          }
          tc_fence_after_sync();
          const uint32_t d = d0 + buf * kSet;
          const int end = kb + chunk < kb1 ? kb + chunk : kb1;
          bool acc = false;
          while (kb < end) {
            if (!ready && !lin_wait(&full[st], phase, g.err, kErrFullWaitTimeout, &s_abort)) {
              ok = false;
              break;
            }
            tc_fence_after_sync();
            const uint64_t da = base_a + ((sa + a_at) >> 4), db = base_b + ((sa + b_at) >> 4);
            // the k-block after this one: in this stage, or at the head of the next
            int next_st = st;
            uint32_t next_phase = phase, next_sa = sa;
            bool stage_end = false;
            auto look_ahead = [&]() {
              ++kb;
              stage_end = --left == 0 || kb == kb1;
              if (stage_end) {
                left = g.unit;
                next_st = st + 1;
                head += stage_bytes;
                if (next_st == g.nstages) next_st = 0, next_phase ^= 1, head = ring;
                next_sa = head;
                ready = lin_test(&full[next_st], next_phase);
              } else {
                next_sa = sa + kb_bytes;
                ready = true;
              }
              asm volatile("" : "+r"(next_sa), "+r"(next_st), "+r"(next_phase));  // here, not behind the MMAs
            };
            auto four = [&](uint32_t to, uint64_t a, uint64_t b, uint32_t idesc, bool into) {
#pragma unroll
              for (int k = 0; k < 4; ++k) lin_mma<CG>(to, a + k * kStepA, b + k * kStepB, idesc, into || k > 0);
            };
            auto four_ahead = [&](uint32_t to, uint64_t a, uint64_t b, uint32_t idesc, bool into) {
              lin_mma<CG>(to, a, b, idesc, into);
              look_ahead();
#pragma unroll
              for (int k = 1; k < 4; ++k) lin_mma<CG>(to, a + k * kStepA, b + k * kStepB, idesc, true);
            };
            if constexpr (SH::kWideB) {
              // plane i of A against B's planes 0 .. PB - 1 - i, into the columns of i + j
              const uint32_t wide = g.idesc + (PB - 1) * n_step;
              four_ahead(d, da, db, wide, acc);
              if (g.pa > 1) four(d + g.bn, da + plane_a, db, wide - n_step, true);
              if (g.pa > 2) four(d + 2 * g.bn, da + 2 * plane_a, db, g.idesc, true);
            } else if (role == 0 || !SH::kCross) {
              four_ahead(d, da, db, g.idesc, acc);
            } else {
              four_ahead(d, da, db + plane_b, g.idesc, acc);
              four(d, da, db + 2 * plane_b, g.idesc, true);
              if (g.pa > 1) {
                four(d, da + plane_a, db, g.idesc, true);
                four(d, da + plane_a, db + plane_b, g.idesc, true);
              }
              if (g.pa > 2) four(d, da + 2 * plane_a, db, g.idesc, true);
            }
            acc = true;
            if (stage_end) {
              if constexpr (CG == 1)
                umma_commit(&empty[st]);
              else
                umma_commit_pair(&empty[st]);
            }
            st = next_st;
            phase = next_phase;
            sa = next_sa;
          }
          uint64_t* done = PROMOTE ? &chunk_full[buf] : &t_full[role];
          if constexpr (CG == 1)
            umma_commit(done);
          else
            umma_commit_pair(done);
        }
      }
    }
  } else {
    // ---- epilogue
    const int warp_u = __shfl_sync(0xFFFFFFFFu, warp, 0);  // (known to be the warp's)
    const int quarter = warp_u & 3;                        // tensor-memory lanes 32 quarter ..
    const int part = (warp_u - 2) >> 2;                    // of the columns
    // PROMOTE: half of the tile's bn columns; else HN columns of accumulator a
    const int a = PROMOTE ? 0 : part * HN / BN;
    const int half = PROMOTE ? g.bn / 2 : HN;
    const int col0 = part * half - a * BN;
    const uint32_t t_lane = tmem + (static_cast<uint32_t>(quarter * 32) << 16) + part * half;
    const int row = quarter * 32 + lane;
    if (g.fold.part)
      for (int w = blockIdx.x + gridDim.x * (warp - 2); w * 32 < g.fold.n; w += gridDim.x * kWarps) fold_bias(g.fold, w);
    int cc = 0, xc = 0, tt = 0;
    bool ok = true;
    auto release = [&](uint64_t* bar) {
      tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) {
        if constexpr (CG == 1)
          mbar_arrive(bar);
        else
          mbar_arrive_cta_relaxed(bar, 0);
      }
    };
    // (a gated tile's warps meet at a barrier, in every tile, whatever runs out)
    for (int t = first; t < ntiles && (ok || GATED); t += step, ++tt) {
      int tm, tn;
      lin_tile(g, t, &tm, &tn);
      const long long n0 = static_cast<long long>(tn) * g.bn;
      long long n_end = n0 + g.bn < g.N ? n0 + g.bn : g.N;
      const int m_warp = GATED ? 0 : row0(tm) + a * g.rm + quarter * 32, m = m_warp + lane;
      const bool m_ok = row < g.rm && m < g.M;
      const float bias = !GATED && m_ok ? g.epi.bias_of(m) : 0.0f;
      if constexpr (PROMOTE) {
        // (columns past the half hold other columns or nothing: never stored)
        if (n_end > n0 + col0 + half) n_end = n0 + col0 + half;
        float acc[HN];
#pragma unroll
        for (int i = 0; i < HN; ++i) acc[i] = 0.0f;
        auto take = [&](uint32_t at) {
#pragma unroll
          for (int c = 0; c < HN; c += G) {
            float v[G];
            tmem_ldf<G>(at + c, v);
            tmem_wait_ld();
#pragma unroll
            for (int i = 0; i < G; ++i) acc[c + i] += v[i];
          }
        };
        for (int kb = kb0, left = kCrossChunks; kb < kb1; kb += g.chunk_kb, ++cc) {
          const int buf = cc & 1;
          if (!ok) break;
          if (!lin_wait(&t_full[buf], (cc >> 1) & 1, g.err, kErrFullWaitTimeout, &s_abort)) {
            ok = false;
            break;
          }
          tc_fence_after_sync();
          if constexpr (SH::kWideB) {
#pragma unroll 1
            for (int j = PB - 1; j >= 0; --j) take(t_lane + buf * kSet + j * g.bn);
          } else {
            take(t_lane + buf * kSet);
          }
          release(&t_empty[buf]);
          if constexpr (SH::kCross) {
            if (--left && kb + g.chunk_kb < kb1) continue;
            left = kCrossChunks;
            if (!lin_wait(&c_full[xc & 1], (xc >> 1) & 1, g.err, kErrFullWaitTimeout, &s_abort)) {
              ok = false;
              break;
            }
            tc_fence_after_sync();
            take(t_lane + (2 + (xc & 1)) * kSet);
            release(&c_empty[xc & 1]);
            ++xc;
          }
        }
        if (GATED || g.split > 1) {
          // as [column][row]; where there is one tile per CTA, over its stages, which are done with
          float* ex = reinterpret_cast<float*>(stages + g.exchange) + part * half * 128 + row;
#pragma unroll
          for (int i = 0; i < HN; ++i)
            if (i < half) ex[i * 128] = acc[i];
          if (GATED && g.split == 1) {
            // gate and up of a feature are 64 lanes apart: they meet here, while the next tile's MMAs run
            asm volatile("bar.sync 1, 256;" ::: "memory");
            const int tid = threadIdx.x - 64, f = tid & 63, mf = row0(tm) + f;
            const float* e = reinterpret_cast<const float*>(stages + g.exchange) + f;
            const long long tile_end = n0 + g.bn < g.N ? n0 + g.bn : g.N;
            if (ok && mf < g.M)
              for (int c = tid >> 6; n0 + c < tile_end; c += 4)
                g.epi.put_planes(mf, n0 + c, swiglu_keeping_nan(e[c * 128], e[c * 128 + 64], g.swiglu_limit));
            asm volatile("bar.sync 1, 256;" ::: "memory");
          }
        } else if (ok && m_ok) {
#pragma unroll
          for (int c = 0; c < HN; c += P) {
            float v[P];
#pragma unroll
            for (int i = 0; i < P; ++i) v[i] = acc[c + i];
            g.epi.put_columns<P>(m_warp, n0 + col0 + c, n_end, bias, v, lane);
          }
        }
      } else {
        if (!lin_wait(&t_full[a], tt & 1, g.err, kErrFullWaitTimeout, &s_abort)) {
          ok = false;
          break;
        }
        tc_fence_after_sync();
#pragma unroll 1
        for (int c = 0; c < HN; c += P) {
          float v[P];
          tmem_ldf<P>(t_lane + c, v);
          tmem_wait_ld();
          if (c + P == HN) release(&t_empty[a]);  // read: the next tile may have the accumulator
          if (m_ok) g.epi.put_columns<P>(m_warp, n0 + col0 + c, n_end, bias, v, lane);
        }
      }
    }
  }

  if (CG == 1 && g.split > 1) {
    __syncthreads();
    cluster_sync_all();  // every partial tile is in place
    if (warp >= 2 && warp < 2 + kWarps) {
      int tm, tn;
      lin_tile(g, first, &tm, &tn);
      const uint32_t ex = smem_u32(stages);
      const long long n0 = static_cast<long long>(tn) * g.bn;
      const long long n_end = n0 + g.bn < g.N ? n0 + g.bn : g.N;
      const int krank_cols = g.bn / g.split, c0 = krank * krank_cols;
      if constexpr (GATED) {
        const int tid = threadIdx.x - 64, f = tid & 63, m = row0(tm) + f;
        for (int c = c0 + (tid >> 6); c < c0 + krank_cols; c += 4) {
          if (m >= g.M || n0 + c >= n_end) continue;
          float gate = 0.0f, up = 0.0f;
          for (int s = 0; s < g.split; ++s) {
            const uint32_t at = lin_mapa(ex, s) + (c * 128 + f) * 4;
            gate += lin_ld_cluster(at);
            up += lin_ld_cluster(at + 256);
          }
          g.epi.put_planes(m, n0 + c, swiglu_keeping_nan(gate, up, g.swiglu_limit));
        }
      } else {
        // threads of 128 rows by two halves of this CTA's columns
        const int tid = threadIdx.x - 64, row = tid & 127;
        auto fold = [&](auto cnt) {
          constexpr int C = decltype(cnt)::value;
          for (int c = c0 + (tid >> 7) * C; c < c0 + krank_cols; c += 2 * C) {
            const int m = row0(tm) + row;
            const long long n = n0 + c;
            if (row >= g.rm || m >= g.M || n >= n_end) continue;
            float v[C];
#pragma unroll
            for (int i = 0; i < C; ++i) v[i] = 0.0f;
            for (int s = 0; s < g.split; ++s) {
              const uint32_t at = lin_mapa(ex, s) + (c * 128 + row) * 4;
#pragma unroll
              for (int i = 0; i < C; ++i) v[i] += lin_ld_cluster(at + i * 512);
            }
            g.epi.put_columns<C>(m, n, n_end, g.epi.bias_of(m), v);
          }
        };
        if (krank_cols % 8 == 0)
          fold(std::integral_constant<int, 4>{});
        else
          fold(std::integral_constant<int, 1>{});
      }
    }
  }
  tc_fence_before_sync();
  __syncthreads();
  if (csize > 1) cluster_sync_all();  // no CTA leaves while a peer may still signal or read it
  tc_fence_after_sync();
  if (warp == 1) {
    if constexpr (CG == 1)
      tmem_dealloc(tmem, kCols);
    else
      tmem_dealloc_pair(tmem, kCols);
  }
  if (g.apart) asm volatile("griddepcontrol.wait;" ::: "memory");
}

}  // namespace dev
}  // namespace objb
