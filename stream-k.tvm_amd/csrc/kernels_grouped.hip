// Products grouped by expert and the gradient of the experts' weights (grouped.h, tile_tn.h): kernel entries and launchers.
#include <cmath>

#include "grouped.h"
#include "grouped_launch.h"
#include "tile_tn.h"

namespace sk {

template <class P>
__global__ __launch_bounds__(P::NT, P::WAVES_PER_EU) void sk_grouped_kernel(GroupedArgs g, int ipt) {
  __shared__ __attribute__((aligned(1024))) char smem[P::LDS_BYTES];
  run_grouped<P>(g, ipt, smem);
}

// The tile with the least estimated time.  The host knows the rows and the experts, not who has how many: the rows are taken to fall on
// the experts by chance, spread by half a tile.
//     time = 2 + sqrt(busy^2 + memory^2)
//   busy    the rounds of the CUs that the tiles make, each of `tau` for 8 KB of K and `o` for a tile's beginning and end; what whole
//           rounds leave costs its share and `cut` (tiles of waves that stream K: cut evenly, pieces of four iterations at least), `cut` of
//           tau (128 x 128, a tile with its CU for itself), or a part of a round and `cut` (256 x 256, cut in two or four)
//   memory  the weights of the experts that have rows, and the rows, once at `rate`
// Fitted to 1150 products (1 to 64 experts, 1 to 2000 rows to an expert, N 256 to 12288, K 64 to 12288, even and skewed; mean |log error|
// 6 to 12 %).  On 600 others its choice takes 1.02 of the fastest tile's time on average, 1.5 at worst, and more than 1.1 in 35.
struct TileCost {
  int variant, bm, bn, per_cu;
  double tau, o, rate, cut;   // us, us, bytes per us, see above
};
static const TileCost COSTS_16[6] = {{GV_WAVEK16, 16, 64, 1, 9.7, 1.25, 6.13e6, 5.62},
                                     {GV_WAVEK32, 32, 64, 1, 11.3, 1.44, 6.18e6, 6.30},
                                     {GV_WAVEK64, 64, 64, 1, 13.7, 1.98, 6.17e6, 7.32},
                                     {GV_WAVEK64W, 64, 128, 1, 22.7, 3.43, 5.67e6, 10.29},
                                     {GV_TILE128, 128, 128, 2, 64.2, 2.53, 6.46e6, 0.71},
                                     {GV_ASM256, 256, 256, 1, 74.6, 5.49, 8.00e6, 18.10}};
static const TileCost COSTS_NN[3] = {{GV_WAVEK64, 64, 64, 1, 17.1, 2.03, 5.72e6, 7.73},
                                     {GV_TILE128, 128, 128, 2, 66.0, 2.57, 6.15e6, 0.69},
                                     {GV_ASM256, 256, 256, 1, 78.0, 6.09, 6.01e6, 19.82}};
static const TileCost COSTS_I8[6] = {{GV_WAVEK16, 16, 64, 1, 9.2, 1.58, 5.63e6, 6.41},
                                     {GV_WAVEK32, 32, 64, 1, 11.3, 1.78, 5.70e6, 7.00},
                                     {GV_WAVEK64, 64, 64, 1, 14.3, 2.32, 5.91e6, 7.53},
                                     {GV_WAVEK64W, 64, 128, 1, 22.5, 4.50, 4.99e6, 10.10},
                                     {GV_TILE128, 128, 128, 2, 61.7, 3.52, 5.17e6, 0.67},
                                     {GV_ASM256, 256, 256, 1, 72.5, 9.01, 7.49e6, 17.71}};
static double estimate(const GroupedShape &h, double experts, const TileCost &c) {
  const double bytes = h.type == GT_I8 ? 1.0 : 2.0, rows = h.R / experts;
  const double high = h.E == 1 ? (double)((h.R + c.bm - 1) / c.bm) : rows / c.bm + 0.5;
  const double tiles = experts * (high > 1.0 ? high : 1.0) * (double)((h.N + c.bn - 1) / c.bn);
  const double iters = h.K * bytes / 8192.0, round = c.tau * iters + c.o, slots = (double)h.cus * c.per_cu;
  const double whole = (double)(int64_t)(tiles / slots), rest = tiles / slots - whole;
  double busy = whole * round;
  if (rest > 0 && c.variant >= GV_WAVEK16) {
    const double least = iters < 0.25 ? iters : 0.25;
    busy += c.tau * (rest * iters > least ? rest * iters : least) + c.o + c.cut;
  } else if (rest > 0 && c.variant == GV_TILE128) {
    busy += rest <= 0.5 ? c.cut * c.tau * iters + c.o : round;
  } else if (rest > 0) {
    const int parts = iters < 0.5 ? 1 : (rest <= 0.25 ? 4 : (rest <= 0.5 ? 2 : 1));
    busy += parts == 1 ? round : c.tau * iters / parts + c.o + c.cut;
  }
  const double memory = (experts * h.N * h.K * bytes + h.R * (h.K * bytes + 2.0 * h.N)) / c.rate;
  return 2.0 + sqrt(busy * busy + memory * memory);
}
int grouped_variant(const GroupedShape &h) {
  if (h.variant != GV_RULE) return h.variant;
  const double experts = h.E == 1 ? 1.0 : h.E * (1 - pow(1 - 1.0 / h.E, (double)h.R));   // that have a row
  int best = GV_TILE128;
  double least = 0;
  auto consider = [&](const TileCost &c) {
    // (many low tiles, beyond what the constants were fitted to: the higher ones are as fast from 8 and 30 rows on)
    if ((c.variant == GV_WAVEK16 && h.R > 40 * h.E) || (c.variant == GV_WAVEK32 && h.R > 150 * h.E) || (c.variant == GV_ASM256 && !grouped_asm_takes(h)))
      return;
    const double t = estimate(h, experts, c);
    if (least == 0 || t < least) {
      least = t;
      best = c.variant;
    }
  };
  if (h.type == GT_I8) {
    for (const TileCost &c : COSTS_I8) consider(c);
  } else if (h.nn) {
    for (const TileCost &c : COSTS_NN) consider(c);
  } else {
    for (const TileCost &c : COSTS_16) consider(c);
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
  if (h.variant >= GV_WAVEK16) return launch_grouped_wavek(g, h, ws, s);
  if (h.variant == GV_ASM256) return grouped_asm_takes(h) ? launch_grouped_asm(g, h, ws, s) : (int)hipErrorNotSupported;
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

// A round of 256 x 256 tiles, one to a CU, takes 1.1 to 1.5 times as long as one of 128 x 128 tiles, two to a CU: they pay where there are
// fewer rounds of them, and rows enough for their longer beginning and end.  bfloat16, times of 256 x 256 tiles by those of 128 x 128:
//   one round against one    1 x 2048 x 2048, 8192 rows 1.49; 1 x 4096 x 2048, 128 rows 1.31, 8192 rows 1.11
//   one against two, two     64 rows an expert .94 to 1.08, 128 rows .91 to 1.06, 512 rows .77 to .91, 8192 rows .60 to .75
//   against four
//   two against three        128 rows 1.11 to 1.22, 512 rows .98 to 1.05, 2048 rows .92 to .94
//   four and six             24 rows 1.00 to 1.13, 64 rows .90 to 1.03, 512 rows .75 to .84
//   eight and more           16 rows .80 to .92, 1024 rows .65 to .75
//   nine against thirteen    712 rows .82
// On 84 random sizes (1 to 64 experts, 8 to 4000 rows each) the choice takes 1.00 of the faster tiles' time on average, 1.1 at worst
// (256 x 256 from 64 rows an expert on, whatever their number: 1.10 and 1.9).
static bool wgrad_asm_pays(const WgradArgs &g, int cus) {
  const auto rounds = [&](int64_t b, int per_cu) { return (g.E * ((g.N + b - 1) / b) * ((g.K + b - 1) / b) + cus * per_cu - 1) / (cus * per_cu); };
  const int64_t large = rounds(256, 1), small = rounds(128, 2);
  if (4 * small < 7 * large) return 5 * small >= 7 * large && g.R >= (int64_t)512 * g.E;
  return g.R >= (int64_t)(large < 4 ? 128 : (large < 8 ? 64 : 0)) * g.E;
}
int launch_wgrad(const WgradArgs &g, bool bf16, int cus, int variant, hipStream_t s) {
  if (variant > GV_ASM256 || (variant == GV_ASM256 && !wgrad_asm_takes(g))) return (int)hipErrorNotSupported;
  if (variant == GV_ASM256 || (variant == GV_RULE && wgrad_asm_takes(g) && wgrad_asm_pays(g, cus))) return launch_wgrad_asm(g, bf16, cus, s);
  return bf16 ? launch_wgrad_policy<TileTN<128, 128, 2, 2, true>>(g, cus, s) : launch_wgrad_policy<TileTN<128, 128, 2, 2, false>>(g, cus, s);
}

}  // namespace sk
