// The four-wave 256 x 256 int8 tiles with scales (tile_scaled_i8.h): the end goes through the patch behind the stages, so that the
// first loads of the next tile are on their way while this one is stored.  4096 x 8192 x 8192: 191 us, 2.88 POPS.
#pragma once
#include "tile_asm_epilogue.h"

namespace sk {

struct ScaledAsm : TileF16Asm<2, false> {
  typedef TileF16Asm<2, false> P;
  typedef ScaledArgs<GemmArgs> Args;
  // rows 16 i0 .. 16 i1 - 1 of every wave's 128
  static __device__ __forceinline__ void store_rows(const Args &a, int pm, int pn, const void *epi, int i0, int i1) {
    const int wave = threadIdx.x >> 6, row0 = pm * P::BM + (wave >> 1) * P::WTM, col0 = pn * P::BN + (wave & 1) * P::WTN;
    by_epilogue(epi, [&](auto e) {
      constexpr int EPI = decltype(e)::value;
      if (a.s.bf16) AsmEnd<P, true, true, EPI>::store(a.C, a.ldc, a.M, a.N, row0, col0, a.s.a, a.s.b, epi_bias(epi), i0, i1);
      else AsmEnd<P, true, false, EPI>::store(a.C, a.ldc, a.M, a.N, row0, col0, a.s.a, a.s.b, epi_bias(epi), i0, i1);
    });
  }
  static __device__ __forceinline__ void store_c(const Args &a, const Acc &, int pm, int pn, char *, const void *epi) {
    store_rows(a, pm, pn, epi, 0, P::FM);
  }
  static __device__ __forceinline__ void store_c_half(const Args &a, const Acc &, int pm, int pn, char *, const void *epi, int h) {
    store_rows(a, pm, pn, epi, h * (P::FM / 2), (h + 1) * (P::FM / 2));
  }
};

}  // namespace sk
