// linear_mn.cu -- the dense products with both transposed in memory: dw = dz^T x.
#include "objb_linear_launch.cuh"

namespace objb {

#define OBJB_GEMM(...) launch_gemm<dev::kMajMN, __VA_ARGS__>(p, t, device, props, st)
int launch_mn(const Product& p, TileKind kind, const Tile& t, int device, const DeviceProps& props, cudaStream_t st) {
  if (kind == kDirect) return OBJB_GEMM(256, 2, 2, false, false, 1);
  if (p.b.planes == 1) {
    if (kind == kPair) return OBJB_GEMM(128, 2, 1, false, true, 1);
    return t.bn <= 64 ? OBJB_GEMM(64, 1, 1, false, true, 1) : OBJB_GEMM(128, 1, 1, false, true, 1);
  }
  if (kind == kPair) return OBJB_GEMM(128, 2, 1, false, true, 3);
  return OBJB_GEMM(80, 1, 1, false, true, 3);
}
#undef OBJB_GEMM

}  // namespace objb
