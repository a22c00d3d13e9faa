// Products of microscaled 4-bit operands on tiles whose waves stream K on their own (tile_mx.h) or share the tile (tile_mx_shared.h), by expert
// or of one matrix.
#include "grouped_launch.h"
#include "grouped_mx.h"
#include "kernel_table.h"
#include "tile_mx_shared.h"

namespace sk {

template <class P>
struct MxWithZero : P {
  static __device__ __forceinline__ void zero_sums(typename P::Acc &acc) {
#pragma unroll
    for (int u = 0; u < P::NQ; ++u) acc.c[u] = typename P::AccV{0, 0, 0, 0};
  }
};
template <class P, bool DENSE>
__global__ __launch_bounds__(P::NT, P::WAVES_PER_EU) void sk_mx_kernel(MxGrouped<DENSE> g, int ipt, Workspace ws) {
  __shared__ __attribute__((aligned(1024))) char smem[P::LDS_BYTES];
  run_grouped_sk<P>(g, ipt, ws, smem);
}

template <class P, bool DENSE>
static int launch(const MxOperands &operands, const GroupedShape &h, const Workspace &ws, hipStream_t s) {
  MxGrouped<DENSE> g;
  static_cast<MxOperands &>(g) = operands;
  g.tiles_n = (g.N + P::BN - 1) / P::BN;
  const int ipt = (g.K + P::BK - 1) / P::BK;
  if (grouped_tiles(h, P::BM) * g.tiles_n * ipt >= 0x7fffffff) return (int)hipErrorNotSupported;   // (iterations are numbered in 32 bits)
  g.grid = h.cus * P::CTAS_PER_CU;
  hipLaunchKernelGGL((sk_mx_kernel<P, DENSE>), dim3(g.grid), dim3(P::NT), 0, s, g, ipt, ws);
  return (int)hipGetLastError();
}

template <bool BF16, int FM, int FN>
using MxWaveK = MxWithZero<TileWaveKMx<BF16, FM, FN>>;
template <bool BF16, int FM, int FN>
using MxWaveK2 = MxWithZero<TileWaveKMx<BF16, FM, FN, 2>>;

// variant -> policy (BF16: C's type):  X(variant, policy)
#define MX_TILES(X)                                                 \
  X(GV_WAVEK16, MxWaveK<BF16, 1, 4>)                              \
  X(GV_WAVEK32, MxWaveK<BF16, 2, 4>)                              \
  X(GV_WAVEK64, MxWaveK<BF16, 4, 4>)                              \
  X(10, MxWaveK2<BF16, 1, 4>) \
  X(11, MxWaveK2<BF16, 2, 4>) \
  X(12, MxWaveK2<BF16, 4, 4>) \
  X(18, TileMxShared<BF16, 64, 64, 2, 2, 4, 2>) \
  X(GV_SHARED256, TileMxShared<BF16, 256, 128, 2, 2, 3>) \
  X(13, TileMxShared<BF16, 64, 128, 2, 2, 3, 2>) \
  X(14, TileMxShared<BF16, 128, 64, 2, 2, 3, 2>) \
  X(15, TileMxShared<BF16, 128, 128, 2, 2, 2, 2>) \
  X(16, MxWaveK2<BF16, 1, 1>) \
  X(17, MxWaveK2<BF16, 1, 2>) \
   X(GV_SHARED64, TileMxShared<BF16, 64, 128, 2, 2, 4>)            \
  X(GV_TILE128, TileMxShared<BF16, 128, 128, 2, 2, 4>)
int mx_variant(const GroupedShape &h) {
  if (h.variant != GV_RULE) return h.variant;
  const int64_t rows = (h.R + h.E - 1) / h.E;
  if (rows > 512) return GV_ASM256;
  return rows <= 16 ? GV_WAVEK16 : (rows <= 32 ? GV_WAVEK32 : GV_WAVEK64);
}
size_t mx_workspace(const GroupedShape &h) {
  constexpr bool BF16 = false;
  const int v = mx_variant(h);
  if (v == GV_ASM256) return mx_asm_workspace(h.cus);
#define X(V, ...) \
  if (v == V) return (size_t)WS_PART_OFF + (size_t)2 * h.cus * __VA_ARGS__::CTAS_PER_CU * __VA_ARGS__::TILE_ELEMS * 4;
  MX_TILES(X)
#undef X
  return 0;
}
// (rows of exponents that are no words apart cannot be read 16 bytes at a time)
bool mx_needs_tiled(const GroupedShape &h) { return h.K % 128 != 0 || mx_variant(h) == GV_ASM256; }
bool mx_wants_tiled(const GroupedShape &h) { return mx_needs_tiled(h); }
template <bool BF16, bool DENSE>
static int launch_by_variant(const MxOperands &g, const GroupedShape &h, const Workspace &ws, hipStream_t s) {
#define X(V, ...) \
  if (h.variant == V) return launch<__VA_ARGS__, DENSE>(g, h, ws, s);
  MX_TILES(X)
#undef X
  return (int)hipErrorNotSupported;
}
int launch_mx(const MxOperands &g, const GroupedShape &h, bool bf16, const Workspace &ws, hipStream_t s) {
  if (h.variant == GV_ASM256) return launch_mx_asm(g, h, bf16, ws, s);
  if (g.offsets == nullptr) return bf16 ? launch_by_variant<true, true>(g, h, ws, s) : launch_by_variant<false, true>(g, h, ws, s);
  return bf16 ? launch_by_variant<true, false>(g, h, ws, s) : launch_by_variant<false, false>(g, h, ws, s);
}

}  // namespace sk
