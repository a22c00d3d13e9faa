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

// The host knows the rows and the experts, not who has how many: an expert is taken to have R / E rows, spread by half a tile.
//
// Up to 8 and 20 rows the 16- and 32-row tiles, whose rings hold the most weights: us, 8 experts of 11008 x 4096 and 64 of 2048 x
// 4096, fp16, 16- / 32- / 64-row tiles: 8 rows each 127 / 130 / 133 and 181 / 180 / 184, 16 rows 134 / 131 / 135, 32 rows 176 / 142 /
// 140.  Above, the tile with the least estimated time: the rounds of the CUs that the tiles make, each of tau iterations of K (128 bytes
// of a row) and o for a tile's beginning and end, against the weights' and rows' way from memory at the rate the tile reaches.
// Estimated / measured us of 64 x 64, 64 x 128, 128 x 128, 256 x 256 tiles: 8 experts, 11008 x 4096, 48 rows each 166 / 145, 165 / 140,
// 192 / 192, 209 / 196; 187 rows 306 / 297, 260 / 264, 240 / 240, 196 / 220; 1024 rows (bfloat16) the last 530 / 565; 64 experts,
// 2048 x 4096, 64 rows 246 / 241, 244 / 232, 278 / 282, 304 / 262, 128 rows 352 / 347, 302 / 314, 282 / 271, 308 / 289.
struct TileCost {
  int variant, bm, bn, per_cu;
  double tau, o, rate;   // us per 64 iterations of a CU's tiles, us, bytes per us
};
static const TileCost TILE_COSTS[] = {{GV_WAVEK64, 64, 64, 1, 13.0, 2.5, 5.2e6},
                                      {GV_WAVEK64W, 64, 128, 1, 22.0, 3.5, 5.2e6},
                                      {GV_TILE128, 128, 128, 2, 69.0, 3.0, 4.3e6},
                                      {GV_ASM256, 256, 256, 1, 75.0, 7.0, 3.9e6}};
static double estimate(const GroupedShape &h, const TileCost &c) {
  const double experts = (double)(h.E < h.R ? h.E : h.R), rows = h.R / experts, bytes = h.type == GT_I8 ? 1.0 : 2.0;
  const double high = h.E == 1 ? (double)((h.R + c.bm - 1) / c.bm) : rows / c.bm + 0.5;
  const double tiles = experts * (high > 1.0 ? high : 1.0) * (double)((h.N + c.bn - 1) / c.bn);
  const double iters = h.K * bytes / 8192.0, round = c.tau * iters + c.o, slots = (double)h.cus * c.per_cu;
  const double whole = (double)(int64_t)(tiles / slots), rest = tiles / slots - whole;
  double busy = whole * round;
  if (c.variant == GV_WAVEK64 || c.variant == GV_WAVEK64W) {
    busy += rest * round + (whole > 0 ? 5.0 : 10.0);            // (cut evenly)
  } else if (rest > 0 && c.variant == GV_TILE128) {
    busy += rest <= 0.5 ? 0.58 * c.tau * iters + c.o : round;   // (a tile that has its CU for itself)
  } else if (rest > 0) {
    const int parts = iters < 0.5 ? 1 : (rest <= 0.25 ? 4 : (rest <= 0.5 ? 2 : 1));
    busy += parts == 1 ? round : c.tau * iters / parts + c.o + 20.0;
  }
  const double memory = (experts * h.N * h.K * bytes + h.R * (h.K * bytes + 2.0 * h.N)) / c.rate;
  return busy > memory ? busy + 0.15 * memory : memory + 0.15 * busy;   // (they overlap but for a part)
}
int grouped_variant(const GroupedShape &h) {
  if (h.variant != GV_RULE) return h.variant;
  const int64_t experts = h.E < h.R ? h.E : h.R, rows = h.R / experts;
  if (!h.nn && rows <= 20) return rows <= 8 ? GV_WAVEK16 : GV_WAVEK32;
  int best = GV_TILE128;
  double least = 0;
  for (const TileCost &c : TILE_COSTS) {
    if ((h.nn && c.variant >= GV_WAVEK16) || (c.variant == GV_ASM256 && !grouped_asm_takes(h))) continue;
    const double t = estimate(h, c);
    if (least == 0 || t < least) {
      least = t;
      best = c.variant;
    }
  }
  return best;
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
