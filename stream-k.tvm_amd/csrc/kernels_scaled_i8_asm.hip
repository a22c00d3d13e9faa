// The four-wave 256 x 256 int8 tiles with scales, for one product and for groups.
#include "scaled_launch.h"
#include "sk_persistent.h"
#include "tile_scaled_i8_asm.h"

namespace sk {

constexpr int ASM_I8_ID = 84;   // (kernel_table.h: SK_TILE_ASM8_KERNELS)

template <class P, bool FIXUP>
__global__ __launch_bounds__(P::NT, P::WAVES_PER_EU) void sk_scaled_asm_kernel(typename P::Args a, DevPlan plan, Workspace ws, const void *bias) {
  __shared__ __attribute__((aligned(16))) char smem[P::LDS_BYTES];
  run_persistent<P, FIXUP, true>(a, plan, ws, smem, bias);
}

bool has_scaled_i8_asm(int id) { return id == ASM_I8_ID; }

int launch_scaled_i8_asm(int id, const GemmArgs &g, const Scales &sc, const DevPlan &p, const Workspace &ws, hipStream_t s, const void *bias) {
  if (id != ASM_I8_ID) return (int)hipErrorInvalidValue;
  ScaledAsm::Args a;
  static_cast<GemmArgs &>(a) = g;
  a.s = sc;
  if (p.sk_tiles == 0)
    hipLaunchKernelGGL((sk_scaled_asm_kernel<ScaledAsm, false>), dim3(p.grid), dim3(ScaledAsm::NT), 0, s, a, p, ws, bias);
  else
    hipLaunchKernelGGL((sk_scaled_asm_kernel<ScaledAsm, true>), dim3(p.grid), dim3(ScaledAsm::NT), 0, s, a, p, ws, bias);
  return (int)hipGetLastError();
}

int occupancy_scaled_i8_asm(int id) {
  int occ = 0;
  if (id != ASM_I8_ID) return 0;
  return hipOccupancyMaxActiveBlocksPerMultiprocessor(&occ, sk_scaled_asm_kernel<ScaledAsm, true>, ScaledAsm::NT, 0) == hipSuccess ? occ : -1;
}

}  // namespace sk
