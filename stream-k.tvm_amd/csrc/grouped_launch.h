// Between the C ABI and the units that hold the grouped kernels.
#pragma once
#include <hip/hip_runtime.h>

#include "grouped.h"

namespace sk {

enum GroupedType { GT_F16 = 0, GT_BF16 = 1, GT_I8 = 2 };
struct GroupedShape {
  int type;      // GroupedType
  bool nn;       // weights [E, K, N]
  int64_t E, R, N, K;   // (K in elements)
  int cus;
  int variant;   // GroupedVariant
};
// which tiles (0: by the rule in kernels_grouped.hip; launches know theirs)
enum GroupedVariant { GV_RULE = 0, GV_TILE128 = 1, GV_ASM256 = 2, GV_WAVEK16 = 3, GV_WAVEK32 = 4, GV_WAVEK64 = 5, GV_WAVEK64W = 6 };
// the variant that a call takes (never GV_RULE; what a caller asked for, if anything), and the workspace it needs
int grouped_variant(const GroupedShape &h);
size_t grouped_workspace(const GroupedShape &h);
// the most row tiles that R rows in E groups (and the two of rows without an expert) can make: every group has one tile that is not
// full, and no tile is without a row
static inline int64_t grouped_tiles(const GroupedShape &h, int bm) {
  const int64_t by_size = h.R / bm + h.E + 2;
  return by_size < h.R ? by_size : h.R;
}
// hipError_t as int; hipErrorNotSupported: h.variant does not exist or does not take the problem
int launch_grouped(const GroupedArgs &g, const GroupedShape &h, const Workspace &ws, hipStream_t s);
// up to some dozen rows to an expert (kernels_grouped_wavek.hip)
size_t grouped_wavek_workspace(int variant, int cus);
int launch_grouped_wavek(const GroupedArgs &g, const GroupedShape &h, const Workspace &ws, hipStream_t s);

struct WgradArgs {
  const half_t *dC, *A;   // [R, N] (width readable columns), [R, K]
  half_t *dW;             // [E, N, K]
  const int *offsets;
  int64_t lddc, lda;
  int E, R, N, K, width;
  int tiles_m, tiles_n, grid;
};
int launch_wgrad(const WgradArgs &g, bool bf16, int cus, int variant, hipStream_t s);

// the 256 x 256 tiles (kernels_grouped_asm.hip), and what they take
bool grouped_asm_takes(const GroupedShape &h);
size_t grouped_asm_workspace(int cus);
int launch_grouped_asm(const GroupedArgs &g, const GroupedShape &h, const Workspace &ws, hipStream_t s);
bool wgrad_asm_takes(const WgradArgs &g);
int launch_wgrad_asm(const WgradArgs &g, bool bf16, int cus, hipStream_t s);

}  // namespace sk
