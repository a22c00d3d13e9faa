// The four-wave 256 x 256 tiles on microscaled 4-bit operands (tile_mx_asm.h), by expert or of one matrix.  The first loads of a CTA's next tile
// go out before this one is stored.  A row tile of at most 128 rows is a low one, as in kernels_grouped_asm.hip: half the MFMAs, three quarters of
// the loads; 2100 x 8192 x 8192 94 us, so 83, 100 x 28672 x 8192 51 and 44, 8 experts of 11008 x 4096, 8192 rows 221 and 218.
#include "grouped_cut.h"
#include "grouped_launch.h"
#include "grouped_mx.h"
#include "kernel_table.h"
#include "tile_mx_asm.h"

namespace sk {

template <class P, bool DENSE>
__global__ __launch_bounds__(P::NT, P::WAVES_PER_EU) void sk_mx_asm_kernel(MxGrouped<DENSE> g, int ipt, Workspace ws) {
  GroupWalk<P::BM, false, DENSE> walk(g.offsets, g.E, g.R, g.tiles_n);
  const int pid = grouped_pid(g.grid);
  int front, back;
  const int tiles = walk.total_tiles(front, back);
  if constexpr (!DENSE) zero_unowned(g, pid, P::NT, front, back);
  const Cuts cuts(tiles, g.grid, ipt);
  struct Segment {
    GroupTile t;
    int cut, part, k0, n;   // (cut: number among the cut tiles, or -1)
    bool last, low;
  };
  const int items = cuts.whole + (tiles - cuts.whole) * cuts.parts, pairs = (ipt + 1) >> 1;
  auto segment = [&](int item, Segment &s) {
    if (item >= items) return false;
    s.cut = -1;
    s.k0 = 0;
    int end = pairs, tile = item;
    if (item >= cuts.whole) {
      const int rest = item - cuts.whole;
      s.cut = cuts.parts == 4 ? rest >> 2 : rest >> 1;
      s.part = rest - s.cut * cuts.parts;
      s.k0 = 2 * (s.part * pairs / cuts.parts);
      end = (s.part + 1) * pairs / cuts.parts;
      tile = cuts.whole + s.cut;
    }
    s.n = min(2 * end, ipt) - s.k0;
    s.last = s.k0 + s.n == ipt;
    walk.find(tile, s.t);
    s.low = s.t.rows - s.t.pm * P::BM <= P::BM / 2;
    return true;
  };
  typename P::Acc acc;
  Segment s, next;
  int item = pid;
  bool have = segment(item, s), requested = false;
  while (have) {
    const typename P::Args a = expert_args<P>(g, s.t);
    const void *epi = expert_epilogue(g, s.t);
    if (s.low) P::template mac<true>(a, s.t.pm, s.t.pn, s.k0, s.n, s.last, requested);
    else P::template mac<false>(a, s.t.pm, s.t.pn, s.k0, s.n, s.last, requested);
    item += g.grid;
    have = requested = segment(item, next);
    if (have) {
      const typename P::Args b = expert_args<P>(g, next.t);
      if (next.low) P::template prefetch_first_stage<true>(b, next.t.pm, next.t.pn, next.k0, next.n, next.last);
      else P::template prefetch_first_stage<false>(b, next.t.pm, next.t.pn, next.k0, next.n, next.last);
    }
    if (s.cut < 0 || join_parts<P>(acc, s.cut, s.part, cuts.parts, g.grid, g.spin_limit, ws, s.low)) {
      if (s.low) P::template store_c<true>(a, s.t.pm, s.t.pn, epi);
      else P::template store_c<false>(a, s.t.pm, s.t.pn, epi);
    }
    s = next;
  }
}

template <class P, bool DENSE>
static int launch(const MxOperands &operands, const GroupedShape &h, const Workspace &ws, hipStream_t s) {
  MxGrouped<DENSE> g;
  static_cast<MxOperands &>(g) = operands;
  g.tiles_n = (g.N + P::BN - 1) / P::BN;
  if (grouped_tiles(h, P::BM) * g.tiles_n > 0x7fffffff) return (int)hipErrorNotSupported;
  g.grid = h.cus;
  hipLaunchKernelGGL((sk_mx_asm_kernel<P, DENSE>), dim3(g.grid), dim3(P::NT), 0, s, g, (g.K + P::BK - 1) / P::BK, ws);
  return (int)hipGetLastError();
}

size_t mx_asm_workspace(int cus) { return (size_t)WS_PART_OFF + (size_t)cus * TileMxAsm<false>::TILE_ELEMS * 4; }
int launch_mx_asm(const MxOperands &g, const GroupedShape &h, bool bf16, const Workspace &ws, hipStream_t s) {
  if (g.offsets == nullptr) return bf16 ? launch<TileMxAsm<true>, true>(g, h, ws, s) : launch<TileMxAsm<false>, true>(g, h, ws, s);
  return bf16 ? launch<TileMxAsm<true>, false>(g, h, ws, s) : launch<TileMxAsm<false>, false>(g, h, ws, s);
}

}  // namespace sk
