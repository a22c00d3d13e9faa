// The four-wave 256 x 256 int8 tiles with scales (tile_scaled_i8.h): the end goes through the patch behind the stages, so that the
// first loads of the next tile are on their way while this one is stored.  4096 x 8192 x 8192: 191 us, 2.88 POPS.
#pragma once
#include "tile_f16_asm.h"
#include "tile_scaled_i8.h"

namespace sk {

struct ScaledAsm : TileF16Asm<2, false> {
  typedef TileF16Asm<2, false> P;
  typedef ScaledArgs<GemmArgs> Args;
  static constexpr int HALF = P::FN / 2;   // 64 columns at a time: the scales and biases of 128 do not fit beside the fix-up's addresses
  typedef BlockPatch<P::FM, HALF> Patch;
  static_assert(Patch::BYTES <= P::FAST_PATCH_BYTES, "a wave's patch behind the stages");
  template <int I0, int I1>
  static __device__ __forceinline__ void store_rows(const Args &a, int pm, int pn, const void *epi) {
    const int wave = threadIdx.x >> 6, wm = wave >> 1, wn = wave & 1;
    const int row0 = pm * P::BM + wm * P::WTM, col0 = pn * P::BN + wn * P::WTN;
    by_result(a.s.bf16 != 0, epi, [&](auto bf16, auto with_epi) {
      static_for<0, 2>([&](auto half) {
        constexpr int j0 = decltype(half)::value * HALF;
        const ScaleRegs<P::FM, HALF, decltype(bf16)::value, decltype(with_epi)::value> r(a, row0, col0 + 16 * j0, epi);
        Patch::store<I0, I1>(a.C, a.ldc, a.M, a.N, row0, col0 + 16 * j0, P::lds() + 2 * P::STAGE_BYTES + wave * P::FAST_PATCH_BYTES,
                             [&](auto i, auto j) {
                               constexpr int ii = decltype(i)::value, jj = decltype(j)::value;
                               return r.template values<ii, jj>(__builtin_bit_cast(intx4_s, agpr_read4<(ii * P::FN + j0 + jj) * 4>()));
                             });
      });
    });
  }
  static __device__ __forceinline__ void store_c(const Args &a, const Acc &, int pm, int pn, char *, const void *epi) {
    store_rows<0, P::FM>(a, pm, pn, epi);
  }
  static __device__ __forceinline__ void store_c_half(const Args &a, const Acc &, int pm, int pn, char *, const void *epi, int h) {
    if (h == 0) store_rows<0, P::FM / 2>(a, pm, pn, epi);
    else store_rows<P::FM / 2, P::FM>(a, pm, pn, epi);
  }
};

}  // namespace sk
