// linear_kk.cu -- the dense products with both operands K-major: y = x w^T and the gated gate / up product.
#include "objb_linear_launch.cuh"

namespace objb {

#define OBJB_GEMM(...) launch_gemm<dev::kMajKK, __VA_ARGS__>(p, t, device, props, st)
int launch_kk(const Product& p, TileKind kind, const Tile& t, int device, const DeviceProps& props, cudaStream_t st) {
  if (p.raw == 1)  // few tokens, f32
    return p.gated      ? OBJB_GEMM(32, 1, 1, true, true, 3, 1)  // (of 16 tokens at most)
           : t.bn <= 32 ? OBJB_GEMM(32, 1, 1, false, true, 3, 1) : OBJB_GEMM(80, 1, 1, false, true, 3, 1);
  if (p.raw == 2) return t.bn <= 32 ? OBJB_GEMM(32, 1, 1, false, true, 3, 2) : OBJB_GEMM(80, 1, 1, false, true, 3, 2);
  if (p.gated) {
    if (kind == kPair) return OBJB_GEMM(128, 2, 1, true, true, 3);
    return t.bn <= 32 ? OBJB_GEMM(32, 1, 1, true, true, 3) : OBJB_GEMM(80, 1, 1, true, true, 3);
  }
  if (kind == kDirect) return OBJB_GEMM(256, 2, 2, false, false, 1);
  if (p.b.planes == 1) {
    if (kind == kPair) return OBJB_GEMM(128, 2, 1, false, true, 1);
    return t.bn <= 32 ? OBJB_GEMM(32, 1, 1, false, true, 1)
           : t.bn <= 64 ? OBJB_GEMM(64, 1, 1, false, true, 1) : OBJB_GEMM(128, 1, 1, false, true, 1);
  }
  if (kind == kPair) return OBJB_GEMM(128, 2, 1, false, true, 3);
  return t.bn <= 32 ? OBJB_GEMM(32, 1, 1, false, true, 3) : OBJB_GEMM(80, 1, 1, false, true, 3);
}
#undef OBJB_GEMM

}  // namespace objb
