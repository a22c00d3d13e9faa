// The four-wave 256 x 256 tiles whose K loop is assembly (tile_f16_asm.h, tile_tn_asm.h), for products grouped by expert and for the
// gradient of the experts' weights.  The first loads of a CTA's next tile go out before this one is stored, across experts too.
// 8 experts of 11008 x 4096, 8192 rows, bfloat16: 554 us (1.33 PFLOP/s), the rows' gradient 568, the weights' 625; the matrix pipes are busy
// 80, 80 and 67 % of the time, at a clock that the power limit sets.
#include "grouped.h"
#include "grouped_launch.h"
#include "kernel_table.h"
#include "tile_scaled_i8_asm.h"
#include "tile_tn_asm.h"

namespace sk {

// The 16-bit policies with an end that leaves the stages alone whatever the tile's columns and epilogue are
template <bool BF16, bool NN>
struct GroupedAsm16 : TileF16Asm<BF16 ? 1 : 0, NN> {
  typedef TileF16Asm<BF16 ? 1 : 0, NN> P;
  static __device__ __forceinline__ void store_rows(const typename P::Args &a, int pm, int pn, const void *epi, int i1) {
    const int wave = threadIdx.x >> 6, row0 = pm * P::BM + (wave >> 1) * P::WTM, col0 = pn * P::BN + (wave & 1) * P::WTN;
    by_epilogue(epi, [&](auto e) {
      AsmEnd<P, false, BF16, decltype(e)::value>::store(a.C, a.ldc, a.M, a.N, row0, col0, nullptr, nullptr, epi_bias(epi), 0, i1);
    });
  }
  static __device__ __forceinline__ void store_c(const typename P::Args &a, const typename P::Acc &, int pm, int pn, char *, const void *epi) {
    if (P::direct_store_ok(a, pn, epi)) P::template store_c_direct<-1>(a, pm, pn);
    else store_rows(a, pm, pn, epi, P::FM);
  }
  static __device__ __forceinline__ void store_c_half(const typename P::Args &a, const typename P::Acc &, int pm, int pn, char *, const void *epi, int) {
    if (P::direct_store_ok(a, pn, epi)) P::template store_c_direct<0>(a, pm, pn);
    else store_rows(a, pm, pn, epi, P::FM / 2);
  }
};

// How the tiles that are left when every CTA has had its whole rounds are cut: K in `parts` equal parts, one to a CTA.  (Aligned cuts: the
// CTAs stay at the same K of their tiles and share rows and weights in the L2s.  Runs of equal length that begin anywhere, as for the
// small tiles in grouped.h, write 90 MB of sums and cost 100 us here: 8 x 11008 x 4096, 3000 rows, bfloat16 307 us, whole tiles 284.)
struct Cuts {
  int whole, parts;
  __device__ __forceinline__ Cuts(int tiles, int grid, int ipt) {
    const int rest = (int)((unsigned)tiles % (unsigned)grid);
    parts = ipt < CUT_LEAST || rest == 0 ? 1 : (rest * 4 <= grid ? 4 : (rest * 2 <= grid ? 2 : 1));
    whole = parts > 1 ? tiles - rest : tiles;
  }
  static constexpr int CUT_LEAST = 32;   // iterations of a tile from which the exchange, some 20 us, pays
};

// The end of a part of a cut tile.  Each CTA of the tile takes a ticket; all but the last put their sums into the workspace and raise a
// flag, the last one -- the others are past their loops by then and wait for nobody, so the wait is a short one whatever else the
// device does -- adds them to its own in the order of the parts, which is the same on every launch.  True: acc has the tile's sums.
// flags: [grid] of the CTAs, then a counter for each cut tile; all zero before and after.  A wait that gives up after spin_limit polls says
// so in the workspace's status and leaves tile, flags and counter as they are, for a late part may still raise its flag: the next
// launch must not count on zeros, and is refused once sk_workspace_status has seen it.  (With a count in place of the wait, every part
// put down and the last to have done so adding up, 8 x 11008 x 4096, 800 rows take 160 us and not 154: a third more, or twice as many,
// sums go through memory at the same time.)
// (low: the lower half of the accumulators)
template <class P>
__device__ __forceinline__ bool join_parts(typename P::Acc &acc, int tile, int part, int parts, int grid, int spin_limit, const Workspace &ws, bool low) {
  int *ticket = ws.flags + grid + tile, *flags = ws.flags + tile * parts, *word = reinterpret_cast<int *>(P::lds() + 2 * P::STAGE_BYTES);
  auto slot = [&](int q) { return ws.partials + (size_t)(tile * parts + q) * P::TILE_ELEMS; };
  if (threadIdx.x == 0) *word = __hip_atomic_fetch_add(ticket, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  __syncthreads();
  const bool last = *word == parts - 1;
  __syncthreads();
  if (!last) {
    if (low) P::store_partial_half(acc, slot(part), 0);
    else P::store_partial(acc, slot(part));
    signal_partial_ready<true>(flags + part, ws.status + WS_DIRTY, (int)(((size_t)(tile * parts + part + 1) * P::TILE_ELEMS * 4 + 255) >> 8));
    return false;
  }
  bool ok = true;
  if (threadIdx.x < 64) {
    for (int q = 0; q < parts; ++q) {
      if (q == part) continue;
      int got = 0;
      for (int spin = 0; spin < spin_limit && !got; ++spin) {
        got = __hip_atomic_load(flags + q, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        if (!got) __builtin_amdgcn_s_sleep(1);
      }
      ok = ok && got;
    }
    if (threadIdx.x == 0) *word = ok;
  }
  __syncthreads();
  const bool complete = *word != 0;
  __syncthreads();   // (the patches of the tile's end overlap the word)
  if (!complete) {
    if (threadIdx.x == 0) ws.status[WS_STATUS] = -8;   // SK_ERR_TIMEOUT
    return false;
  }
  // eight groups at a time: the parts in front of this one, this one, the parts behind it
  constexpr int BATCH = 8;
  const uint32_t off = (uint32_t)pin_here((int)threadIdx.x) * 16;
  static_for<0, P::NV4 / BATCH>([&](auto b) {
    constexpr int base = decltype(b)::value * BATCH;
    if (base >= P::NV4 / 2 && low) return;
    typedef typename std::conditional<P::I8, typename P::intx4, floatx4>::type Sum;
    Sum sum[BATCH];
    for (int q = 0; q < parts; ++q) {
      const BufferRsrc r = make_rsrc(slot(q), P::TILE_ELEMS * 4);
      Sum x[BATCH];
      if (q == part) {
        static_for<0, BATCH>([&](auto i) { x[decltype(i)::value] = __builtin_bit_cast(Sum, agpr_read4<(base + decltype(i)::value) * 4>()); });
      } else {
        static_for<0, BATCH>([&](auto i) {
          x[decltype(i)::value] = __builtin_bit_cast(Sum, ld_coherent16(r, off, (uint32_t)(base + decltype(i)::value) * P::NT * 16));
        });
      }
#pragma unroll
      for (int i = 0; i < BATCH; ++i) sum[i] = q == 0 ? x[i] : sum[i] + x[i];
    }
    static_for<0, BATCH>([&](auto i) { agpr_write4<(base + decltype(i)::value) * 4>(__builtin_bit_cast(floatx4, sum[decltype(i)::value])); });
  });
  if (threadIdx.x < parts) __hip_atomic_store(flags + threadIdx.x, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  if (threadIdx.x == 0) __hip_atomic_store(ticket, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  return true;
}

// A row tile of at most 128 rows -- the last of half of the groups -- is a low one: half the MFMAs, three quarters of the
// loads; 8 experts of 11008 x 4096, 800 rows, 179 -> 154 us with them and the starts below, 16 of 4096 x 4096, 1900 int8 rows 76 -> 62.
// It keeps its place among its expert's tiles, which share the weights: behind all others 64 experts of 2048 x 4096, 16384 rows, take 356 us
// and not 347.  (Tiles drawn from a counter as CTAs become free, and not dealt out: 356.)
template <class P, bool NN>
__global__ __launch_bounds__(P::NT, P::WAVES_PER_EU) void sk_grouped_asm_kernel(GroupedArgs g, int ipt, Workspace ws) {
  constexpr auto LOW = P::LOW_TILE, FULL = NN ? P::WHOLE_TILE : P::WRAPPED_TILE;
  GroupWalk<P::BM, false> walk(g.offsets, g.E, g.R, g.tiles_n);
  const int pid = grouped_pid(g.grid);
  int front, back;
  const int tiles = walk.total_tiles(front, back);
  zero_unowned(g, pid, P::NT, front, back);
  const Cuts cuts(tiles, g.grid, ipt);
  struct Segment {
    GroupTile t;
    int cut, part, k0, n;   // (cut: number among the cut tiles, or -1)
    bool low;
  };
  const int items = cuts.whole + (tiles - cuts.whole) * cuts.parts;
  auto find = [&](int tile, Segment &s) {
    walk.find(tile, s.t);
    s.low = s.t.rows - s.t.pm * P::BM <= P::BM / 2;
  };
  // Weights come straight from memory where few tiles share them, and all CTAs at the same K of rows whose pitch is a large power of two
  // meet in the same channels (see rotation_of): 128 rows against 65536 x 4096 135 us, with these starts 101.  Eight neighbours of a row
  // tile, which share its rows in an L2, and all tiles that share weights are at the same K; the next eight, and other experts, elsewhere
  // (every tile one iteration from the one beside it: up to 3 % slower).  [K, N] weights: neighbouring tiles read neighbouring
  // pieces of the same rows.
  auto rot_of = [&](const Segment &s) { return NN ? 0 : __builtin_amdgcn_readfirstlane((int)((unsigned)(5 * (s.t.pn >> 3) + 11 * s.t.group) % (unsigned)s.n)); };
  auto segment = [&](int item, Segment &s) {
    if (item >= items) return false;
    s.cut = -1;
    s.k0 = 0;
    s.n = ipt;
    int tile = item;
    if (item >= cuts.whole) {
      const int rest = item - cuts.whole;
      s.cut = cuts.parts == 4 ? rest >> 2 : rest >> 1;
      s.part = rest - s.cut * cuts.parts;
      s.k0 = s.part * ipt / cuts.parts;
      s.n = (s.part + 1) * ipt / cuts.parts - s.k0;
      tile = cuts.whole + s.cut;
    }
    find(tile, s);
    return true;
  };
  typename P::Acc acc;
  Segment s, next;
  int item = pid;
  bool have = segment(item, s), requested = false;
  while (have) {
    typename P::Args a = expert_args<P>(g, s.t);
    const void *epi = expert_epilogue(g, s.t);
    if (s.low) P::template mac<LOW>(a, acc, s.t.pm, s.t.pn, s.k0, s.n, nullptr, requested, rot_of(s));
    else P::template mac<FULL>(a, acc, s.t.pm, s.t.pn, s.k0, s.n, nullptr, requested, rot_of(s));
    requested = false;
    item += g.grid;
    have = segment(item, next);
    if (have) {   // (every end here leaves the stages alone)
      const typename P::Args b = expert_args<P>(g, next.t);
      if (next.low) P::template prefetch_first_stage<LOW>(b, next.t.pm, next.t.pn, next.k0, next.n, rot_of(next));
      else P::template prefetch_first_stage<FULL>(b, next.t.pm, next.t.pn, next.k0, next.n, rot_of(next));
      requested = true;
    }
    if (s.cut < 0 || join_parts<P>(acc, s.cut, s.part, cuts.parts, g.grid, g.spin_limit, ws, s.low)) {
      if (s.low) {
        // the lower half of each wave's 128 rows; the second wave's are the tile's rows 64 .., not 128 ..: C moved back by 64
        const int back = (threadIdx.x >> 7) * (P::WTM / 2);
        a.C -= (int64_t)back * a.ldc;
        a.M += back;
        if constexpr (is_scaled<typename P::Args>::value) a.s.a -= back;
        P::store_c_half(a, acc, s.t.pm, s.t.pn, nullptr, epi, 0);
      } else {
        P::store_c(a, acc, s.t.pm, s.t.pn, nullptr, epi);
      }
    }
    s = next;
  }
}

template <class P, bool NN = false>
static int launch_asm(GroupedArgs g, const GroupedShape &h, int ipt, const Workspace &ws, hipStream_t s) {
  g.tiles_n = (g.N + P::BN - 1) / P::BN;
  if (grouped_tiles(h, P::BM) * g.tiles_n > 0x7fffffff) return (int)hipErrorNotSupported;
  g.grid = h.cus;
  hipLaunchKernelGGL((sk_grouped_asm_kernel<P, NN>), dim3(g.grid), dim3(P::NT), 0, s, g, ipt, ws);
  return (int)hipGetLastError();
}

size_t grouped_asm_workspace(int cus) { return (size_t)WS_PART_OFF + (size_t)cus * ScaledAsm::TILE_ELEMS * 4; }

bool grouped_asm_takes(const GroupedShape &h) { return h.K % (h.type == GT_I8 ? 128 : 64) == 0; }

int launch_grouped_asm(const GroupedArgs &g, const GroupedShape &h, const Workspace &ws, hipStream_t s) {
  const int ipt = (int)(h.K / (h.type == GT_I8 ? 128 : 64));
  if (h.type == GT_I8) return launch_asm<ScaledAsm>(g, h, ipt, ws, s);
  if (h.nn) return h.type == GT_BF16 ? launch_asm<GroupedAsm16<true, true>, true>(g, h, ipt, ws, s) : launch_asm<GroupedAsm16<false, true>, true>(g, h, ipt, ws, s);
  return h.type == GT_BF16 ? launch_asm<GroupedAsm16<true, false>>(g, h, ipt, ws, s) : launch_asm<GroupedAsm16<false, false>>(g, h, ipt, ws, s);
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
