// Products grouped by expert: rows offsets[e] <= r < offsets[e + 1] of A times the weights of expert e, groups of any size.
//
// The offsets are in device memory (a router has just written them), so the host knows neither how many tiles there are nor whose
// they are.  A launch is persistent: every CTA derives the list of tiles from the offsets itself -- lane g of a wave holds group
// 64 c + g, a prefix sum over the lanes numbers the tiles, a ballot finds the group of a tile -- and takes tiles pid, pid + grid, ...
// An expert without rows has no tile, and no weights of it are read.  The lookup is two loads and some thirty instructions a chunk
// of 64 groups, done once where there are no more (the tiles of a CTA come in ascending order).
//
// Groups 0 and E + 1 are the rows in front of offsets[0] and behind offsets[E], which no expert owns: zeros are stored for them, so
// that every row of C is written.  Offsets are clamped to 0 <= lo <= hi <= R, whatever they hold: no access leaves the operands.
//
// The tiles themselves are those of the ordinary products, each with its arguments moved to the expert's operands.
#pragma once
#include "sk_device.h"
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

// UNOWNED: groups 0 and E + 1 have tiles too
template <int BM, bool UNOWNED = true>
struct GroupWalk {
  const int *offsets;
  int E, R, tiles_n;
  int chunk, before;             // groups 64 chunk .. + 63 are in the lanes; tiles of the groups in front of them
  int lo, rows, ends;            // this lane's group: first row, rows, tiles of the chunk up to its last one

  __device__ __forceinline__ GroupWalk(const int *o, int E_, int R_, int tn) : offsets(o), E(E_), R(R_), tiles_n(tn), before(0) { load(0); }
  __device__ __forceinline__ void load(int c) {
    chunk = c;
    const int lane = threadIdx.x & 63, g = 64 * c + lane;
    lo = rows = 0;
    if (g <= E + 1) {
      lo = g == 0 ? 0 : min(max(offsets[g - 1], 0), R);
      rows = (g == E + 1 ? R : min(max(offsets[g], lo), R)) - lo;
      if (!UNOWNED && (g == 0 || g == E + 1)) rows = 0;
    }
    int x = (int)((unsigned)(rows + BM - 1) / BM) * tiles_n;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
      const int y = __shfl_up(x, d, 64);
      if (lane >= d) x += y;
    }
    ends = x;
  }
  // tiles of all groups (before the first find)
  __device__ __forceinline__ int total_tiles() {
    int sum = __builtin_amdgcn_readlane(ends, 63);
    if (E + 1 < 64) return sum;
    for (int c = 1; 64 * c <= E + 1; ++c) {
      load(c);
      sum += __builtin_amdgcn_readlane(ends, 63);
    }
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
__device__ __forceinline__ void set_operands(SkinnyArgs &a, const GroupedArgs &g, const half_t *B) {
  a.W = B;
  a.ldw = g.ldb;
  a.scales = a.zeros = nullptr;
  a.zero = a.groups = 0;
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
    P::mac(a, acc, t.pm, t.pn, 0, ipt, smem);
    P::store_c(a, acc, t.pm, t.pn, smem, expert_epilogue(g, t));
  }
}

}  // namespace sk
