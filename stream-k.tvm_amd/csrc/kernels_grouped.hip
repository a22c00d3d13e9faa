// Products grouped by expert and the gradient of the experts' weights (grouped.h, tile_tn.h): kernel entries and launchers.
#include "grouped.h"
#include "grouped_launch.h"
#include "tile_tn.h"

namespace sk {

template <class P>
__global__ __launch_bounds__(P::NT, P::WAVES_PER_EU) void sk_grouped_kernel(GroupedArgs g, int ipt) {
  __shared__ __attribute__((aligned(1024))) char smem[P::LDS_BYTES];
  run_grouped<P>(g, ipt, smem);
}

int grouped_variant(const GroupedShape &h) {
  if (h.variant != GV_RULE) return h.variant;
  const int64_t experts = h.E < h.R ? h.E : h.R, rows = h.R / experts;   // of an expert that has any, about
  if (!h.nn) {
    if (rows <= 8) return GV_WAVEK16;
    if (rows <= 20) return GV_WAVEK32;
    if (rows <= 40) return GV_WAVEK64;
    if (rows <= 80) return GV_WAVEK64W;
  }
  return grouped_asm_takes(h) && rows >= 128 ? GV_ASM256 : GV_TILE128;
}
size_t grouped_workspace(const GroupedShape &h) {
  const int v = grouped_variant(h);
  return v == GV_ASM256 ? grouped_asm_workspace(h.cus) : grouped_wavek_workspace(v, h.cus);
}

template <class P>
static int launch_grouped_policy(GroupedArgs g, const GroupedShape &h, hipStream_t s) {
  g.tiles_n = (g.N + P::BN - 1) / P::BN;
  const int64_t most = grouped_tiles(h, P::BM) * g.tiles_n;   // whatever the groups' sizes
  if (most > 0x7fffffff) return (int)hipErrorInvalidValue;
  g.grid = (int)(most < (int64_t)h.cus * P::CTAS_PER_CU ? most : (int64_t)h.cus * P::CTAS_PER_CU);
  hipLaunchKernelGGL((sk_grouped_kernel<P>), dim3(g.grid), dim3(P::NT), 0, s, g, (g.K + P::BK - 1) / P::BK);
  return (int)hipGetLastError();
}

int launch_grouped(const GroupedArgs &g, const GroupedShape &h, const Workspace &ws, hipStream_t s) {
  GroupedShape with = h;
  with.variant = grouped_variant(h);
  if (with.variant >= GV_WAVEK16) return h.nn ? (int)hipErrorNotSupported : launch_grouped_wavek(g, with, ws, s);
  if (with.variant == GV_ASM256) return grouped_asm_takes(h) ? launch_grouped_asm(g, h, ws, s) : (int)hipErrorNotSupported;
  if (h.type == GT_I8) return launch_grouped_policy<ScaledDma<TileF16NTDma<128, 128, 2, 2, false, 64, true, false, 3>>>(g, h, s);
  if (h.nn) {
    if (h.type == GT_BF16) return launch_grouped_policy<TileF16NTDma<128, 128, 2, 2, true, 64, true, true>>(g, h, s);
    return launch_grouped_policy<TileF16NTDma<128, 128, 2, 2, true, 64, true, false>>(g, h, s);
  }
  if (h.type == GT_BF16) return launch_grouped_policy<TileF16NTDma<128, 128, 2, 2, false, 64, true, true>>(g, h, s);
  return launch_grouped_policy<TileF16NTDma<128, 128, 2, 2, false, 64, true, false>>(g, h, s);
}

// ---- dW[e] = dC[rows of e]^T A[rows of e] ----
template <class P>
__global__ __launch_bounds__(P::NT, P::WAVES_PER_EU) void sk_grouped_wgrad_kernel(WgradArgs g) {
  __shared__ __attribute__((aligned(1024))) char smem[P::LDS_BYTES];
  typename P::Acc acc;
  const int per_expert = g.tiles_m * g.tiles_n, total = g.E * per_expert;
  for (int tile = grouped_pid(g.grid); tile < total; tile += g.grid) {
    const int e = tile / per_expert;
    const int lo = min(max(g.offsets[e], 0), g.R), rows = min(max(g.offsets[e + 1], lo), g.R) - lo;
    int pm, pn;
    group_raster(tile - e * per_expert, g.tiles_m, g.tiles_n, pm, pn);
    typename P::Args a;
    a.A = g.dC + (int64_t)lo * g.lddc;
    a.B = g.A + (int64_t)lo * g.lda;
    a.C = g.dW + (int64_t)e * g.N * g.K;
    a.M = g.N;
    a.N = g.K;
    a.K = rows;
    a.lda = g.lddc;
    a.ldb = g.lda;
    a.ldc = g.K;
    a.width_a = g.width;
    a.width_b = g.K;
    P::mac(a, acc, pm, pn, 0, (rows + P::BK - 1) / P::BK, smem);   // (no rows: no iterations, and zeros are stored)
    P::store_c(a, acc, pm, pn, smem, nullptr);
  }
}

template <class P>
static int launch_wgrad_policy(WgradArgs g, int cus, hipStream_t s) {
  g.tiles_m = (g.N + P::BM - 1) / P::BM;
  g.tiles_n = (g.K + P::BN - 1) / P::BN;
  const int64_t total = (int64_t)g.E * g.tiles_m * g.tiles_n;
  if (total > 0x7fffffff) return (int)hipErrorInvalidValue;
  g.grid = (int)(total < (int64_t)cus * P::CTAS_PER_CU ? total : (int64_t)cus * P::CTAS_PER_CU);
  hipLaunchKernelGGL((sk_grouped_wgrad_kernel<P>), dim3(g.grid), dim3(P::NT), 0, s, g);
  return (int)hipGetLastError();
}

int launch_wgrad(const WgradArgs &g, bool bf16, int cus, int variant, hipStream_t s) {
  if (variant > GV_ASM256 || (variant == GV_ASM256 && !wgrad_asm_takes(g))) return (int)hipErrorNotSupported;
  if (variant == GV_ASM256 || (variant == GV_RULE && wgrad_asm_takes(g) && g.R >= 64 * g.E)) return launch_wgrad_asm(g, bf16, cus, s);
  return bf16 ? launch_wgrad_policy<TileTN<128, 128, 2, 2, true>>(g, cus, s) : launch_wgrad_policy<TileTN<128, 128, 2, 2, false>>(g, cus, s);
}

}  // namespace sk
