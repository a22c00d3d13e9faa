// Tiles of the grouped products that several CTAs share along K, a part each: which are cut, and how the parts are joined.
#pragma once
#include "grouped.h"
#include "tile_f16_asm.h"

namespace sk {

// How the tiles that are left when every CTA has had its whole rounds are cut: K in `parts` equal parts, one to a CTA.  (Aligned cuts: the
// CTAs stay at the same K of their tiles and share rows and weights in the L2s.  Runs of equal length that begin anywhere, as for the
// small tiles in grouped.h, write 90 MB of sums and cost 100 us here: 8 x 11008 x 4096, 3000 rows, bfloat16 307 us, whole tiles 284.)
struct Cuts {
  int whole, parts;
  __device__ __forceinline__ Cuts(int tiles, int grid, int ipt) {
    const int rest = (int)((unsigned)tiles % (unsigned)grid);
    parts = parts_of(rest, grid, ipt);
    whole = parts > 1 ? tiles - rest : tiles;
  }
  static constexpr int CUT_LEAST = 32;   // iterations of a tile from which the exchange, some 20 us, pays
  // (the rule of kernels_mx.hip counts on the same parts)
  template <class Int>
  static __host__ __device__ __forceinline__ constexpr int parts_of(Int rest, int grid, Int ipt) {
    return ipt < CUT_LEAST || rest == 0 ? 1 : (rest * 4 <= grid ? 4 : (rest * 2 <= grid ? 2 : 1));
  }
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
  int *ticket = ws.flags + grid + tile, *flags = ws.flags + tile * parts, *word = reinterpret_cast<int *>(P::lds() + P::PATCHES_AT);
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

}  // namespace sk
