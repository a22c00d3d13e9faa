// Products grouped by expert with few rows each (tile_group_stream.h).
#include "grouped_launch.h"
#include "kernel_table.h"
#include "tile_group_stream.h"

namespace sk {

template <class P>
__global__ __launch_bounds__(P::NT, P::WAVES_PER_EU) void sk_grouped_stream_kernel(GroupedArgs g, int ipt, Workspace ws) {
  __shared__ __attribute__((aligned(1024))) char smem[P::LDS_BYTES];
  P::run(g, ipt, ws, smem);
}

// variant -> tile, types alike:  X(variant, MB, WM, WN, WD, AD)
#define GROUP_STREAMS(X)            \
  X(GV_STREAM16, 1, 1, 4, 4, 3)     \
  X(GV_STREAM32, 2, 1, 4, 3, 3)     \
  X(GV_STREAM64, 2, 2, 2, 3, 3)

// iterations of all tiles are numbered in 32 bits
template <class P>
static bool takes(const GroupedShape &h, const GroupedArgs &g) {
  return grouped_tiles(h, P::BM) * ((g.N + P::BN - 1) / P::BN) * ((g.K + P::BK - 1) / P::BK) < 0x7fffffff;
}
template <class P>
static int launch(GroupedArgs g, const GroupedShape &h, const Workspace &ws, hipStream_t s) {
  if (!takes<P>(h, g)) return (int)hipErrorNotSupported;
  g.tiles_n = (g.N + P::BN - 1) / P::BN;
  g.grid = h.cus;
  hipLaunchKernelGGL((sk_grouped_stream_kernel<P>), dim3(g.grid), dim3(P::NT), 0, s, g, (g.K + P::BK - 1) / P::BK, ws);
  return (int)hipGetLastError();
}

size_t grouped_stream_workspace(int variant, int cus) {
#define X(V, MB, WM, WN, WD, AD) \
  if (variant == V) return (size_t)WS_PART_OFF + (size_t)2 * cus * GroupStream<MB, WM, WN, WD, AD, GE_F16>::SLOT_BYTES;
  GROUP_STREAMS(X)
#undef X
  return 0;
}
int launch_grouped_stream(const GroupedArgs &g, const GroupedShape &h, const Workspace &ws, hipStream_t s) {
#define X(V, MB, WM, WN, WD, AD)                                                                          \
  if (h.variant == V) {                                                                                   \
    if (h.type == GT_I8) return launch<GroupStream<MB, WM, WN, WD, AD, GE_I8>>(g, h, ws, s);              \
    if (h.type == GT_BF16) return launch<GroupStream<MB, WM, WN, WD, AD, GE_BF16>>(g, h, ws, s);          \
    return launch<GroupStream<MB, WM, WN, WD, AD, GE_F16>>(g, h, ws, s);                                  \
  }
  GROUP_STREAMS(X)
#undef X
  return (int)hipErrorNotSupported;
}

}  // namespace sk
