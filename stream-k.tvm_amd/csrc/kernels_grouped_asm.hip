// The four-wave 256 x 256 tiles whose K loop is assembly (tile_f16_asm.h, tile_tn_asm.h), for products grouped by expert and for the
// gradient of the experts' weights.  The first loads of a CTA's next tile go out before this one is stored, across experts too.
#include "grouped.h"
#include "grouped_launch.h"
#include "tile_scaled_i8_asm.h"
#include "tile_tn_asm.h"

namespace sk {

template <class P>
__global__ __launch_bounds__(P::NT, P::WAVES_PER_EU) void sk_grouped_asm_kernel(GroupedArgs g, int ipt) {
  GroupWalk<P::BM> walk(g.offsets, g.E, g.R, g.tiles_n);
  typename P::Acc acc;
  GroupTile t, next;
  int tile = grouped_pid(g.grid);
  bool have = walk.find(tile, t), requested = false;
  while (have) {
    const bool owned = t.group != 0 && t.group != g.E + 1;
    const typename P::Args a = expert_args<P>(g, t);
    const void *epi = expert_epilogue(g, t);
    if (owned) P::mac(a, acc, t.pm, t.pn, 0, ipt, nullptr, requested);
    requested = false;
    tile += g.grid;
    have = walk.find(tile, next);
    if (have && owned && next.group != 0 && next.group != g.E + 1 && P::epilogue_lds_free(a, t.pn, epi)) {
      P::prefetch_first_stage(expert_args<P>(g, next), next.pm, next.pn, 0, ipt);
      requested = true;
    }
    if (owned) P::store_c(a, acc, t.pm, t.pn, nullptr, epi);
    else zero_tile<P>(g, t);
    t = next;
  }
}

template <class P>
static int launch_asm(GroupedArgs g, const GroupedShape &h, int ipt, hipStream_t s) {
  g.tiles_n = (g.N + P::BN - 1) / P::BN;
  const int64_t most = grouped_tiles(h, P::BM) * g.tiles_n;
  if (most > 0x7fffffff) return (int)hipErrorInvalidValue;
  g.grid = (int)(most < h.cus ? most : h.cus);
  hipLaunchKernelGGL((sk_grouped_asm_kernel<P>), dim3(g.grid), dim3(P::NT), 0, s, g, ipt);
  return (int)hipGetLastError();
}

bool grouped_asm_takes(const GroupedShape &h) { return h.K % (h.type == GT_I8 ? 128 : 64) == 0; }

int launch_grouped_asm(const GroupedArgs &g, const GroupedShape &h, hipStream_t s) {
  const int ipt = (int)(h.K / (h.type == GT_I8 ? 128 : 64));
  if (h.type == GT_I8) return launch_asm<ScaledAsm>(g, h, ipt, s);
  if (h.nn) return h.type == GT_BF16 ? launch_asm<TileF16Asm<1, true>>(g, h, ipt, s) : launch_asm<TileF16Asm<0, true>>(g, h, ipt, s);
  return h.type == GT_BF16 ? launch_asm<TileF16Asm<1, false>>(g, h, ipt, s) : launch_asm<TileF16Asm<0, false>>(g, h, ipt, s);
}

// ---- dW[e] = dC[rows of e]^T A[rows of e] ----
struct WgradTile {
  int expert, lo, rows, pm, pn;
};
template <class P>
__device__ __forceinline__ bool wgrad_tile(const WgradArgs &g, int tile, WgradTile &t) {
  const int per_expert = g.tiles_m * g.tiles_n;
  if (tile >= g.E * per_expert) return false;
  t.expert = (int)((unsigned)tile / (unsigned)per_expert);
  const int local = tile - t.expert * per_expert;
  t.lo = min(max(g.offsets[t.expert], 0), g.R);
  t.rows = min(max(g.offsets[t.expert + 1], t.lo), g.R) - t.lo;
  group_raster(local, g.tiles_m, g.tiles_n, t.pm, t.pn);
  return true;
}
template <class P>
__device__ __forceinline__ TnArgs wgrad_args(const WgradArgs &g, const WgradTile &t) {
  TnArgs a;
  a.A = g.dC + (int64_t)t.lo * g.lddc;
  a.B = g.A + (int64_t)t.lo * g.lda;
  a.C = g.dW + (int64_t)t.expert * g.N * g.K;
  a.M = g.N;
  a.N = g.K;
  a.K = t.rows;
  a.lda = g.lddc;
  a.ldb = g.lda;
  a.ldc = g.K;
  a.alpha = 1.f;
  a.scales = nullptr;
  a.zero = a.groups = 0;
  a.width_a = g.width;
  a.width_b = g.K;
  return a;
}
template <class P>
__device__ __forceinline__ void zero_block(const TnArgs &a, int pm, int pn) {
  for (int i = threadIdx.x; i < P::BM * P::BN; i += P::NT) {
    const int row = pm * P::BM + i / P::BN, col = pn * P::BN + i % P::BN;
    if (row < a.M && col < a.N) a.C[(int64_t)row * a.ldc + col] = (half_t)0.f;
  }
}
template <class P>
__global__ __launch_bounds__(P::NT, P::WAVES_PER_EU) void sk_grouped_wgrad_asm_kernel(WgradArgs g) {
  typename P::Acc acc;
  WgradTile t, next;
  int tile = grouped_pid(g.grid);
  bool have = wgrad_tile<P>(g, tile, t), requested = false;
  while (have) {
    const TnArgs a = wgrad_args<P>(g, t);
    if (t.rows > 0) P::mac(a, acc, t.pm, t.pn, 0, (t.rows + 63) / 64, nullptr, requested);
    requested = false;
    tile += g.grid;
    have = wgrad_tile<P>(g, tile, next);
    if (have && t.rows > 0 && next.rows > 0 && P::epilogue_lds_free(a, t.pn, nullptr)) {
      P::prefetch_first_stage(wgrad_args<P>(g, next), next.pm, next.pn, 0, (next.rows + 63) / 64);
      requested = true;
    }
    if (t.rows > 0) P::store_c(a, acc, t.pm, t.pn, nullptr, nullptr);
    else zero_block<P>(a, t.pm, t.pn);
    t = next;
  }
}
template <class P>
static int launch_wgrad_asm_policy(WgradArgs g, int cus, hipStream_t s) {
  g.tiles_m = (g.N + P::BM - 1) / P::BM;
  g.tiles_n = (g.K + P::BN - 1) / P::BN;
  const int64_t total = (int64_t)g.E * g.tiles_m * g.tiles_n;
  if (total > 0x7fffffff) return (int)hipErrorInvalidValue;
  g.grid = (int)(total < cus ? total : cus);
  hipLaunchKernelGGL((sk_grouped_wgrad_asm_kernel<P>), dim3(g.grid), dim3(P::NT), 0, s, g);
  return (int)hipGetLastError();
}

bool wgrad_asm_takes(const WgradArgs &g) {
  // one expert may have all rows, and its descriptors reach to the last of them
  const int64_t ld = g.lddc > g.lda ? g.lddc : g.lda;
  return ((int64_t)g.R + 64) * ld * 2 < (int64_t)1 << 31;
}
int launch_wgrad_asm(const WgradArgs &g, bool bf16, int cus, hipStream_t s) {
  return bf16 ? launch_wgrad_asm_policy<TileTNAsm<true>>(g, cus, s) : launch_wgrad_asm_policy<TileTNAsm<false>>(g, cus, s);
}

}  // namespace sk
