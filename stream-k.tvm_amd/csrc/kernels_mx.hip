// Products of microscaled 4-bit operands on tiles whose waves stream K on their own (tile_mx.h) or share the tile (tile_mx_shared.h), by expert
// or of one matrix.
#include <cmath>

#include "grouped_cut.h"
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

// (two tiles to a CU -- one stores or waits for its first rows while the other computes -- but for 64 x 64, whose registers fill it)
template <bool BF16, int FM, int FN, bool WORDS, int CTAS = 2>
using MxWaveK = MxWithZero<TileWaveKMx<BF16, FM, FN, CTAS, WORDS>>;

// variant -> policy (BF16: C's type; WORDS: tile_mx.h):  X(variant, policy)
#define MX_ROWS(X)                                            \
  X(GV_MX16X16, MxWaveK<BF16, 1, 1, WORDS>)                   \
  X(GV_MX16X32, MxWaveK<BF16, 1, 2, WORDS>)                   \
  X(GV_WAVEK16, MxWaveK<BF16, 1, 4, WORDS>)                   \
  X(GV_WAVEK32, MxWaveK<BF16, 2, 4, WORDS>)                   \
  X(GV_WAVEK64, MxWaveK<BF16, 4, 4, WORDS, 1>)
#define MX_TILES(X)                                           \
  X(GV_WAVEK64W, TileMxShared<BF16, 64, 128, 2, 2, 3, 2>)     \
  X(GV_TILE128, TileMxShared<BF16, 128, 128, 2, 2, 2, 2>)     \
  X(GV_MX128X256, TileMxShared<BF16, 128, 256, 2, 4, 3, 1>)

// (rows of exponents that are no words apart cannot be read where these tiles read them)
static bool takes_tiled(int64_t K, int variant) {
  const bool shared = variant == GV_WAVEK64W || variant == GV_TILE128 || variant == GV_MX128X256;
  return variant == GV_ASM256 || (K % 128 != 0 && shared);
}
// The tile with the least estimated time, for rows that fall on the experts by chance.
//     time = start + max(busy, memory) + hidden min(busy, memory), and where exponents are tiled 3.5 us and their bytes twice at 4 TB/s
//   busy    iterations of `bk` values of the CU that has most -- whole rounds of tiles, and of those that are left their share and `cut`, or
//           whole tiles where that is less (256 x 256: what Cuts takes) -- each of `alone` or, of `per_cu` tiles at a time, `shared`, and more
//           by `astray` where rows do not begin at 128 bytes (at 64: half of it), so that a chunk's are in two lines;
//           `end` for a tile's beginning and end, `join` for a cut
//   memory  the operands of the experts that have rows, and C, once at 6 TB/s
// Fitted to 993 products (none to 256 experts, 1 to 16384 rows, N 20 to 28672, K 256 to 16384, of which half no multiples of 128; mean
// |log error| 7 to 13 %).  On 750 others its choice takes 1.020 of the fastest tile's time on average, 1.7 at worst, and more than 1.1 in 40.
struct MxCost {
  int variant, bm, bn, bk, per_cu, cut;
  double start, alone, shared, end, join, hidden, astray;   // us (hidden, astray: parts)
};
static const MxCost COSTS[9] = {{GV_MX16X16, 16, 16, 2048, 2, 3, 4.11, 0.44, 0.26, 1.37, 6.57, 0.25, 1.62},
                                {GV_MX16X32, 16, 32, 2048, 2, 3, 3.95, 0.56, 0.37, 1.32, 5.48, 0.34, 1.79},
                                {GV_WAVEK16, 16, 64, 2048, 2, 3, 4.12, 0.92, 0.67, 1.06, 4.34, 0.55, 1.51},
                                {GV_WAVEK32, 32, 64, 2048, 2, 3, 4.27, 1.19, 0.87, 1.26, 4.70, 0.50, 1.30},
                                {GV_WAVEK64, 64, 64, 2048, 1, 3, 3.76, 1.39, 0.00, 2.80, 4.69, 0.33, 1.03},
                                {GV_WAVEK64W, 64, 128, 512, 2, 8, 3.51, 0.71, 0.71, 1.76, 11.85, 0.42, 0.11},
                                {GV_TILE128, 128, 128, 512, 2, 8, 4.80, 1.14, 1.04, 1.25, 19.16, 0.54, 0.10},
                                {GV_MX128X256, 128, 256, 512, 1, 8, 3.65, 1.89, 0.00, 2.90, 20.00, 0.48, 0.14},
                                {GV_ASM256, 256, 256, 256, 1, 0, 1.00, 0.88, 0.00, 11.22, 18.72, 0.69, 0.26}};
static double estimate(const GroupedShape &h, double experts, const MxCost &c) {
  const double rows = h.R / experts;
  double high = h.E == 1 ? (double)((h.R + c.bm - 1) / c.bm) : experts * fmax(1.0, 0.5 + rows / c.bm);
  if (c.variant == GV_ASM256) {   // (a last tile of up to 128 rows counts 0.6)
    const int64_t rest = h.R % 256;
    high = h.E == 1 ? (double)(h.R / 256) + (rest == 0 ? 0.0 : (rest <= 128 ? 0.6 : 1.0)) : experts * fmax(0.6, 0.3 + rows / 256);
  }
  const double tiles = ceil(high * (double)((h.N + c.bn - 1) / c.bn) - 1e-9), slots = (double)h.cus * c.per_cu;
  const double ipt = (double)((h.K + c.bk - 1) / c.bk), whole = floor(tiles / slots), rest = tiles - whole * slots;
  double iters = whole * ipt, at_once = whole > 0 ? c.per_cu : ceil(rest / h.cus);
  bool joined = false;
  if (rest > 0 && c.variant == GV_ASM256) {
    const int parts = Cuts::parts_of((int64_t)rest, h.cus, (int64_t)ipt);
    joined = parts > 1;
    iters += ipt / parts;
  } else if (rest > 0) {
    const double run = ceil(rest * ipt / slots);
    joined = run + c.cut < ipt;
    iters += joined ? run : ipt;
    if (joined) at_once = c.per_cu;
  }
  const double astray = 1.0 + (h.K % 256 == 0 ? 0.0 : (h.K % 128 == 0 ? 0.5 : 1.0)) * c.astray;
  const double busy = iters * fmax(c.alone, at_once * c.shared) * astray + (whole + (rest > 0)) * c.end + (joined ? c.join : 0.0);
  const double memory = ((experts * h.N + h.R) * h.K * (17.0 / 32) + 2.0 * h.R * h.N) / 6e6;
  const bool tiled = takes_tiled(h.K, c.variant);
  return c.start + fmax(busy, memory) + c.hidden * fmin(busy, memory) + (tiled ? 3.5 + (double)(h.E * h.N + h.R) * h.K / 32 * 2 / 4e6 : 0.0);
}
int mx_variant(const GroupedShape &h) {
  if (h.variant != GV_RULE) return h.variant;
  const double experts = h.E == 1 ? 1.0 : h.E * (1 - pow(1 - 1.0 / h.E, (double)h.R));   // that have a row
  int best = 0;
  double least = 0;
  for (const MxCost &c : COSTS) {
    if (takes_tiled(h.K, c.variant) && !mx_tiled_fits(h)) continue;   // (64 x 64 and smaller tiles take any size)
    const double t = estimate(h, experts, c);
    if (best == 0 || t < least) {
      least = t;
      best = c.variant;
    }
  }
  return best;
}
size_t mx_workspace(const GroupedShape &h) {
  constexpr bool BF16 = false, WORDS = false;
  const int v = mx_variant(h);
  if (v == GV_ASM256) return mx_asm_workspace(h.cus);
#define X(V, ...) \
  if (v == V) return (size_t)WS_PART_OFF + (size_t)2 * h.cus * __VA_ARGS__::CTAS_PER_CU * __VA_ARGS__::TILE_ELEMS * 4;
  MX_ROWS(X)
  MX_TILES(X)
#undef X
  return 0;
}
bool mx_needs_tiled(const GroupedShape &h) { return takes_tiled(h.K, mx_variant(h)); }
template <bool BF16, bool DENSE, bool WORDS>
static int launch_rows(const MxOperands &g, const GroupedShape &h, const Workspace &ws, hipStream_t s) {
#define X(V, ...) \
  if (h.variant == V) return launch<__VA_ARGS__, DENSE>(g, h, ws, s);
  MX_ROWS(X)
#undef X
  return (int)hipErrorNotSupported;
}
template <bool BF16, bool DENSE>
static int launch_by_variant(const MxOperands &g, const GroupedShape &h, const Workspace &ws, hipStream_t s) {
#define X(V, ...) \
  if (h.variant == V) return launch<__VA_ARGS__, DENSE>(g, h, ws, s);
  MX_TILES(X)
#undef X
  const bool words = ((g.ea.pitch | g.eb.pitch) & 3) == 0;   // (the arrays begin at words)
  return words ? launch_rows<BF16, DENSE, true>(g, h, ws, s) : launch_rows<BF16, DENSE, false>(g, h, ws, s);
}
int launch_mx(const MxOperands &g, const GroupedShape &h, bool bf16, const Workspace &ws, hipStream_t s) {
  if (h.variant == GV_ASM256) return launch_mx_asm(g, h, bf16, ws, s);
  if (g.offsets == nullptr) return bf16 ? launch_by_variant<true, true>(g, h, ws, s) : launch_by_variant<false, true>(g, h, ws, s);
  return bf16 ? launch_by_variant<true, false>(g, h, ws, s) : launch_by_variant<false, false>(g, h, ws, s);
}

}  // namespace sk
