// Products grouped by expert on the tiles whose waves stream K on their own (tile_wavek.h): few rows to an expert, bound by the weights'
// way from memory, of which a CTA's rings hold up to 160 KB.  8 experts of 11008 x 4096, fp16: 2 rows (two experts' weights) 38 us, 128
// rows 131 us, 5.5 TB/s.  [K, N] weights, 8 of 1024 x 2048, 500 rows: 18 us (128 x 128 tiles 24).
#include "grouped.h"
#include "grouped_launch.h"
#include "kernel_table.h"

namespace sk {

template <class P>
struct WithZero : P {
  static __device__ __forceinline__ void zero_sums(typename P::Acc &acc) {
#pragma unroll
    for (int u = 0; u < P::NQ; ++u) acc.c[u] = typename P::AccV{0, 0, 0, 0};
  }
};
template <class P>
__global__ __launch_bounds__(P::NT, P::WAVES_PER_EU) void sk_grouped_wavek_kernel(GroupedArgs g, int ipt, Workspace ws) {
  __shared__ __attribute__((aligned(1024))) char smem[P::LDS_BYTES];
  run_grouped_sk<WithZero<P>>(g, ipt, ws, smem);
}

template <class P>
static int launch(GroupedArgs g, const GroupedShape &h, const Workspace &ws, hipStream_t s) {
  g.tiles_n = (g.N + P::BN - 1) / P::BN;
  const int ipt = (g.K + P::BK - 1) / P::BK;
  if (grouped_tiles(h, P::BM) * g.tiles_n * ipt >= 0x7fffffff) return (int)hipErrorNotSupported;   // (iterations are numbered in 32 bits)
  g.grid = h.cus;
  hipLaunchKernelGGL((sk_grouped_wavek_kernel<P>), dim3(g.grid), dim3(P::NT), 0, s, g, ipt, ws);
  return (int)hipGetLastError();
}

// variant -> blocks of 16 rows, of 16 columns:  X(variant, FM, FN)
#define GROUP_WAVEKS(X)  \
  X(GV_WAVEK16, 1, 4)    \
  X(GV_WAVEK32, 2, 4)    \
  X(GV_WAVEK64, 4, 4)    \
  X(GV_WAVEK64W, 4, 8)

size_t grouped_wavek_workspace(int variant, int cus) {
#define X(V, FM, FN) \
  if (variant == V) return (size_t)WS_PART_OFF + (size_t)2 * cus * (16 * FM) * (16 * FN) * 4;
  GROUP_WAVEKS(X)
#undef X
  return 0;
}
template <int FM, int FN>
static int launch_by_type(const GroupedArgs &g, const GroupedShape &h, const Workspace &ws, hipStream_t s) {
  if (h.nn) {
    // (the lower ones are behind 64 x 64 from one row on: 100 rows, 8 experts of 4096 x 11008 158, 157 and 148 us; of 64 x 128 the ring
    // would hold one chunk only)
    if constexpr (FM == 4 && FN == 4) return h.type == GT_BF16 ? launch<TileWaveK<WK_BF16, FM, FN, true>>(g, h, ws, s) : launch<TileWaveK<WK_F16, FM, FN, true>>(g, h, ws, s);
    return (int)hipErrorNotSupported;
  }
  if (h.type == GT_I8) return launch<ScaledWaveK<TileWaveK<WK_I8, FM, FN, false>>>(g, h, ws, s);
  return h.type == GT_BF16 ? launch<TileWaveK<WK_BF16, FM, FN, false>>(g, h, ws, s) : launch<TileWaveK<WK_F16, FM, FN, false>>(g, h, ws, s);
}
int launch_grouped_wavek(const GroupedArgs &g, const GroupedShape &h, const Workspace &ws, hipStream_t s) {
#define X(V, FM, FN) \
  if (h.variant == V) return launch_by_type<FM, FN>(g, h, ws, s);
  GROUP_WAVEKS(X)
#undef X
  return (int)hipErrorNotSupported;
}

}  // namespace sk
