// Products grouped by expert: rows offsets[e] <= r < offsets[e + 1] of A times the weights of expert e, groups of any size.
//
// The offsets are in device memory (a router has just written them), so the host knows neither how many tiles there are nor whose
// they are.  A launch is persistent: every CTA derives the list of tiles from the offsets itself -- lane g of a wave holds group
// 64 c + g, a prefix sum over the lanes numbers the tiles, a ballot finds the group of a tile -- and takes tiles pid, pid + grid, ...
// An expert without rows has no tile, and no weights of it are read.  The lookup is two loads and some thirty instructions a chunk
// of 64 groups, done once where there are no more (the tiles of a CTA come in ascending order).
//
// Groups 0 and E + 1 are the rows in front of offsets[0] and behind offsets[E], which no expert owns: zeros are stored for them, so
// that every row of C is written.  Offsets are clamped to 0 .. R and none counts that is below one in front of it: whatever they hold, the
// groups lie side by side, no access leaves the operands, and there are no more tiles than the host reckons with.
//
// The tiles themselves are those of the ordinary products, each with its arguments moved to the expert's operands.
#pragma once
#include "sk_device.h"
#include "sk_persistent.h"
#include "tile_scaled_i8.h"

namespace sk {

struct GroupedArgs {
  const half_t *A, *B;
  half_t *C;
  const int *offsets;
  const half_t *bias;            // [E, N] in C's type, or null
  Scales s;                      // int8: of A's rows [R], of the weights' rows [E, N]
  int64_t lda, ldb, ldc, expert_b;   // expert_b: elements of B from one expert to the next
  int E, R, N, K;                // one-byte operands: K, lda, ldb, expert_b in pairs
  int act, tiles_n, grid;
  int spin_limit;                // polls of a wait for the other parts of a tile (kernels_grouped_asm.hip)
};

struct GroupTile {
  int group, lo, rows, pm, pn;   // (group: 0 and E + 1 are no expert's)
};

// tile number `local` of a group of tm x tn: eight tiles down, then one to the right, so that CTAs which run together share rows of A
// and of the weights
__device__ __forceinline__ void group_raster(int local, int tm, int tn, int &pm, int &pn) {
  if (tm == 1) {
    pm = 0;
    pn = local;
    return;
  }
  const int q = (int)((unsigned)local / (unsigned)(8 * tn)), r = local - q * 8 * tn;
  const int high = min(8, tm - 8 * q), c = (int)((unsigned)r / (unsigned)high);
  pm = 8 * q + r - c * high;
  pn = c;
}

// UNOWNED: groups 0 and E + 1 have tiles too.  DENSE: no offsets, one expert has all rows.
template <int BM, bool UNOWNED = true, bool DENSE = false>
struct GroupWalk {
  const int *offsets;
  int E, R, tiles_n;
  int chunk, before;             // groups 64 chunk .. + 63 are in the lanes; tiles of the groups in front of them
  int reached;                   // the largest offset of this chunk and those in front of it
  int lo, rows, ends;            // this lane's group: first row, rows, tiles of the chunk up to its last one

  __device__ __forceinline__ GroupWalk(const int *o, int E_, int R_, int tn) : offsets(o), E(E_), R(R_), tiles_n(tn), before(0) { load(0); }
  __device__ __forceinline__ void load(int c) {
    chunk = c;
    if constexpr (DENSE) {
      const int lane = threadIdx.x & 63;
      lo = lane > 1 ? R : 0;
      rows = lane == 1 ? R : 0;
      ends = lane >= 1 ? (int)((unsigned)(R + BM - 1) / BM) * tiles_n : 0;
      reached = R;
      return;
    }
    const int lane = threadIdx.x & 63, g = 64 * c + lane, before_chunk = c == 0 ? 0 : reached;
    // this group's end, and the one in front of it (from the lane below: 0x138)
    const int end = max((int)wave_max_up_to((uint32_t)min(max(offsets[min(g, E)], 0), R)), before_chunk);
    lo = __builtin_amdgcn_update_dpp(before_chunk, end, 0x138, 0xf, 0xf, false);
    rows = UNOWNED ? (g == E + 1 ? R : end) - lo : (g == 0 ? 0 : end - lo);   // (behind E: end is lo)
    reached = __builtin_amdgcn_readlane(end, 63);
    int x = (int)((unsigned)(rows + BM - 1) / BM) * tiles_n;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
      const int y = __shfl_up(x, d, 64);
      if (lane >= d) x += y;
    }
    ends = x;
  }
  // tiles of all groups (before the first find); front, back: the rows in front of all experts' and behind them begin and end there
  __device__ __forceinline__ int total_tiles(int &front, int &back) {
    int sum = __builtin_amdgcn_readlane(ends, 63);
    front = __builtin_amdgcn_readlane(lo, 1);
    back = reached;
    if (E + 1 < 64) return sum;
    for (int c = 1; 64 * c <= E + 1; ++c) {
      load(c);
      sum += __builtin_amdgcn_readlane(ends, 63);
    }
    back = reached;
    load(0);
    return sum;
  }
  // the tile of this number, or false past the last one; numbers are asked for in ascending order
  __device__ __forceinline__ bool find(int tile, GroupTile &t) {
    for (;;) {
      const int total = __builtin_amdgcn_readlane(ends, 63);
      if (tile - before < total) break;
      if (64 * (chunk + 1) > E + 1) return false;
      before += total;
      load(chunk + 1);
    }
    const int n = tile - before;
    const int i = __builtin_popcountll(__builtin_amdgcn_ballot_w64(ends <= n));
    const int first = i > 0 ? __builtin_amdgcn_readlane(ends, i - 1) : 0;
    t.group = 64 * chunk + i;
    t.lo = __builtin_amdgcn_readlane(lo, i);
    t.rows = __builtin_amdgcn_readlane(rows, i);
    group_raster(n - first, (int)((unsigned)(t.rows + BM - 1) / BM), tiles_n, t.pm, t.pn);
    return true;
  }
};

// the arguments of an expert's product
template <class Args>
struct is_scaled { static constexpr bool value = false; };
template <class Base>
struct is_scaled<ScaledArgs<Base>> { static constexpr bool value = true; };
__device__ __forceinline__ void set_operands(GemmArgs &a, const GroupedArgs &g, const half_t *B) {
  a.B = B;
  a.ldb = g.ldb;
  a.alpha = 1.f;
  a.scales = nullptr;
  a.zero = a.groups = 0;
}
__device__ __forceinline__ void set_operands(WaveKArgs &a, const GroupedArgs &g, const half_t *B) {
  set_operands(static_cast<GemmArgs &>(a), g, B);
  a.start_scale = 0xffffffffu / (unsigned)g.tiles_n;   // an eighth of the columns start at an eighth of K each
}
template <class P>
__device__ __forceinline__ typename P::Args expert_args(const GroupedArgs &g, const GroupTile &t) {
  typename P::Args a;
  const int e = t.group - 1;
  set_operands(a, g, g.B + (int64_t)e * g.expert_b);
  a.A = g.A + (int64_t)t.lo * g.lda;
  a.C = g.C + (int64_t)t.lo * g.ldc;
  a.M = t.rows;
  a.N = g.N;
  a.K = g.K;
  a.lda = g.lda;
  a.ldc = g.ldc;
  if constexpr (is_scaled<typename P::Args>::value) a.s = Scales{g.s.a + t.lo, g.s.b + (int64_t)e * g.N, g.s.bf16};
  return a;
}
__device__ __forceinline__ const void *expert_epilogue(const GroupedArgs &g, const GroupTile &t) {
  return epi_word(g.bias ? g.bias + (int64_t)(t.group - 1) * g.N : nullptr, g.act);
}

template <class P>
__device__ __forceinline__ void zero_tile(const GroupedArgs &g, const GroupTile &t) {
  half_t *C = g.C + (int64_t)t.lo * g.ldc;
  for (int i = threadIdx.x; i < P::BM * P::BN; i += P::NT) {
    const int row = t.pm * P::BM + i / P::BN, col = t.pn * P::BN + i % P::BN;
    if (row < t.rows && col < g.N) C[(int64_t)row * g.ldc + col] = (half_t)0.f;
  }
}

// XCD x (the workgroups x, x + 8, ..) takes a contiguous range of numbers, as in logical_pid
__device__ __forceinline__ int grouped_pid(int grid) {
  const int b = blockIdx.x, x = b & 7;
  return x * (grid >> 3) + min(x, grid & 7) + (b >> 3);
}

// what a policy fetches ahead of a tile's loop
template <class P>
__device__ __forceinline__ void prefetch_epilogue(const typename P::Args &a, typename P::Acc &acc, const GroupTile &t, const void *epi) {
  if constexpr (has_prefetch_bias<P>::value) {
    if (epi != nullptr) P::prefetch_bias(a, acc, t.pn, epi);
  }
  if constexpr (has_prefetch_scales<P>::value) P::prefetch_scales(a, acc, t.pm, t.pn, epi);
}

template <class P>
__device__ __forceinline__ void run_grouped(const GroupedArgs &g, int ipt, char *smem) {
  GroupWalk<P::BM> walk(g.offsets, g.E, g.R, g.tiles_n);
  typename P::Acc acc;
  GroupTile t;
  for (int tile = grouped_pid(g.grid); walk.find(tile, t); tile += g.grid) {
    if (t.group == 0 || t.group == g.E + 1) {
      zero_tile<P>(g, t);
      continue;
    }
    const typename P::Args a = expert_args<P>(g, t);
    const void *epi = expert_epilogue(g, t);
    prefetch_epilogue<P>(a, acc, t, epi);
    P::mac(a, acc, t.pm, t.pn, 0, ipt, smem);
    P::store_c(a, acc, t.pm, t.pn, smem, epi);
  }
}

// ---- Stream-K over the groups ----
// As long as there is a tile for every CTA each takes one -- neighbouring tiles at a time, which share rows and weights in the L2s --
// and the iterations of the tiles that are left, fewer than CTAs, are numbered through and dealt out in equal runs.  A tile that lies
// in one run is stored as it is.  Of one that is cut, every CTA with a part leaves its sums in the workspace, two slots to a CTA:
// slot 1 for the tile whose start it has, slot 0 for the one that it enters in the middle.  When its run is over a CTA adds its
// iterations to the tile's counter (kept at the CTA that has the tile's start, and zero before and after); who completes the count
// adds up the parts in the order of the CTAs, which is the same on every launch, and stores.  Nobody waits for another CTA.
struct SkRuns {
  int total, ctas, each, extra;   // iterations, CTAs that have some, of each CTA, CTAs with one more
  // least: iterations of a run, that its fix-up is worth
  __device__ __forceinline__ SkRuns(int total_, int grid, int least) : total(total_) { deal(min(grid, max(1, total / least))); }
  // tiles whole, or cut where that saves more than `cost` iterations
  __device__ __forceinline__ SkRuns(int tiles, int ipt, int grid, int cost) : total(tiles * ipt) {
    const int run = (int)((unsigned)(total + grid - 1) / (unsigned)grid);
    deal(run + cost < ipt ? min(grid, total) : max(1, tiles));
  }
  __device__ __forceinline__ void deal(int ctas_) {
    ctas = ctas_;
    each = (int)((unsigned)total / (unsigned)ctas);
    extra = total - each * ctas;
  }
  __device__ __forceinline__ int start(int pid) const { return pid * each + min(pid, extra); }
  __device__ __forceinline__ int length(int pid) const { return each + (pid < extra ? 1 : 0); }
  __device__ __forceinline__ int cta_of(int at) const {
    const int boundary = extra * (each + 1);
    return at < boundary ? (int)((unsigned)at / (unsigned)(each + 1)) : extra + (int)((unsigned)(at - boundary) / (unsigned)each);
  }
};
// rows without an expert become zeros, shared out over the grid
__device__ __forceinline__ void zero_unowned(const GroupedArgs &g, int pid, int threads, int front, int back) {
  const int rows = front + g.R - back;
  for (int r = pid; r < rows; r += g.grid) {
    half_t *C = g.C + (int64_t)(r < front ? r : back + r - front) * g.ldc;
    for (int col = threadIdx.x; col < g.N; col += threads) C[col] = (half_t)0.f;
  }
}

// What a cut costs, in iterations, where a policy says so: tiles that are left stay whole, one to a CTA, unless runs are shorter than a tile
// by more than that.  (0: all are cut, into runs of four iterations at least)
template <class P, class = void>
struct cut_cost { static constexpr int value = 0; };
template <class P>
struct cut_cost<P, std::void_t<decltype(P::CUT_COST)>> { static constexpr int value = P::CUT_COST; };
// arguments of one product without groups (dense, below): a member of that name
template <class G, class = void>
struct is_dense { static constexpr bool value = false; };
template <class G>
struct is_dense<G, std::void_t<decltype(G::DENSE)>> { static constexpr bool value = G::DENSE; };

// P: a policy whose partial tiles are coherent (store_partial, add_partial) and whose LDS is dead between two calls of mac.  G: GroupedArgs,
// or what is derived from it and has expert_args of its own
template <class P, class G>
__device__ __forceinline__ void run_grouped_sk(const G &g, int ipt, const Workspace &ws, char *smem) {
  static_assert(P::COHERENT_PARTIALS && P::FIXUP_WORD_IN_LDS, "see above");
  GroupWalk<P::BM, false, is_dense<G>::value> walk(g.offsets, g.E, g.R, g.tiles_n);
  const int pid = grouped_pid(g.grid);
  int front, back;
  const int tiles = walk.total_tiles(front, back), whole = tiles - (int)((unsigned)tiles % (unsigned)g.grid);
  zero_unowned(g, pid, P::NT, front, back);
  auto slot = [&](int p, int which) { return ws.partials + (size_t)(2 * p + which) * P::TILE_ELEMS; };
  typename P::Acc acc;
  GroupTile t;
  for (int tile = pid; tile < whole; tile += g.grid) {
    walk.find(tile, t);
    const typename P::Args a = expert_args<P>(g, t);
    const void *epi = expert_epilogue(g, t);
    prefetch_epilogue<P>(a, acc, t, epi);
    P::mac(a, acc, t.pm, t.pn, 0, ipt, smem);
    P::store_c(a, acc, t.pm, t.pn, smem, epi);
  }
  const SkRuns runs = cut_cost<P>::value > 0 ? SkRuns(tiles - whole, ipt, g.grid, cut_cost<P>::value) : SkRuns((tiles - whole) * ipt, g.grid, 4);   // (a cut costs about as much as two iterations)
  // (runs that are fewer than CTAs go to the workgroups that begin first, which stand on all CUs and XCDs)
  const int run = cut_cost<P>::value == 0 ? pid : ((int)blockIdx.x < runs.ctas ? grouped_pid(runs.ctas) : runs.ctas);
  if (run >= runs.ctas || runs.total == 0) return;
  int at = runs.start(run), left = runs.length(run);
  int cut_tile[2] = {-1, -1}, cut_n[2];   // [0]: entered in the middle, [1]: its start is here
  GroupTile cut[2];
  while (left > 0) {
    const int tile = (int)((unsigned)at / (unsigned)ipt), k0 = at - tile * ipt, n = min(ipt - k0, left);
    walk.find(whole + tile, t);
    const typename P::Args a = expert_args<P>(g, t);
    const void *epi = expert_epilogue(g, t);
    prefetch_epilogue<P>(a, acc, t, epi);
    P::mac(a, acc, t.pm, t.pn, k0, n, smem);
    if (n == ipt) {
      P::store_c(a, acc, t.pm, t.pn, smem, epi);
    } else {
      P::store_partial(acc, slot(run, k0 == 0));
      if (k0 == 0) {
        cut_tile[1] = tile;
        cut_n[1] = n;
        cut[1] = t;
      } else {
        cut_tile[0] = tile;
        cut_n[0] = n;
        cut[0] = t;
      }
    }
    at += n;
    left -= n;
  }
  if (cut_tile[0] < 0 && cut_tile[1] < 0) return;
  wait_own_memory_ops();
  __syncthreads();
  int *word = reinterpret_cast<int *>(smem);
  if (threadIdx.x == 0)
    __hip_atomic_fetch_max(ws.status + WS_DIRTY, (int)(((size_t)(2 * run + 2) * P::TILE_ELEMS * 4 + 255) >> 8), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    if (cut_tile[c] < 0) continue;   // (uniform)
    const int p0 = runs.cta_of(cut_tile[c] * ipt), p1 = runs.cta_of(cut_tile[c] * ipt + ipt - 1);
    if (threadIdx.x == 0) {
      const int have = __hip_atomic_fetch_add(ws.flags + p0, cut_n[c], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) + cut_n[c];
      if (have == ipt) __hip_atomic_store(ws.flags + p0, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      *word = have == ipt;
    }
    __syncthreads();
    const bool complete = *word != 0;
    __syncthreads();
    if (!complete) continue;
    const typename P::Args a = expert_args<P>(g, cut[c]);
    const void *epi = expert_epilogue(g, cut[c]);
    prefetch_epilogue<P>(a, acc, cut[c], epi);
    P::zero_sums(acc);
    for (int p = p0; p <= p1; ++p) P::add_partial(acc, slot(p, p == p0));
    P::store_c(a, acc, cut[c].pm, cut[c].pn, smem, epi);
  }
}

}  // namespace sk
