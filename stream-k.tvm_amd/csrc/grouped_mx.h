// Products of microscaled 4-bit operands by expert, and of one matrix (DENSE): the walk over groups of grouped.h with exponents beside
// the operands.
#pragma once
#include "grouped.h"
#include "tile_mx.h"

namespace sk {

struct MxOperands : GroupedArgs {   // (K, lda, ldb, expert_b in pairs of bytes, four values)
  MxExponents ea, eb;               // of A's rows [R], of the weights' rows [E, N]
};
template <bool DENSE_>
struct MxGrouped : MxOperands {
  static constexpr bool DENSE = DENSE_;
};

template <class P, bool DENSE>
__device__ __forceinline__ typename P::Args expert_args(const MxGrouped<DENSE> &g, const GroupTile &t) {
  typename P::Args a;
  const int e = DENSE ? 0 : t.group - 1, lo = DENSE ? 0 : t.lo;
  set_operands(a, g, g.B + (int64_t)e * g.expert_b);
  a.A = g.A + (int64_t)lo * g.lda;
  a.C = g.C + (int64_t)lo * g.ldc;
  a.M = t.rows;
  a.N = g.N;
  a.K = g.K;
  a.lda = g.lda;
  a.ldc = g.ldc;
  a.ea = g.ea.row(lo);
  a.eb = g.eb.row((int64_t)e * g.N);
  return a;
}

}  // namespace sk
