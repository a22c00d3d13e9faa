// int8 products with scales (tile_scaled_i8.h): an instance for each int8 kernel that operator calls take, under that kernel's id.
#include "launch.h"
#include "sk_persistent.h"
#include "scaled_launch.h"
#include "tile_scaled_i8.h"
#include "wavek_launch.h"

namespace sk {

// K of an iteration of a CTA
template <class P, class = void>
struct has_bkc { static constexpr bool value = false; };
template <class P>
struct has_bkc<P, std::void_t<decltype(P::BKC)>> { static constexpr bool value = true; };
template <class P>
__host__ __device__ constexpr int iteration_k() {
  if constexpr (has_bkc<P>::value) return P::BKC;
  else return P::BK;
}

template <class P, bool FIXUP>
__global__ __launch_bounds__(P::NT, P::WAVES_PER_EU) void sk_scaled_kernel(typename P::Args a, DevPlan plan, Workspace ws, const void *bias) {
  __shared__ __attribute__((aligned(1024))) char smem[P::LDS_BYTES];
  run_persistent<P, FIXUP, true>(a, plan, ws, smem, bias);
}

// One round of whole tiles: scalar arguments that are preloaded into scalar registers, and no plan (wavek_launch.h has the reasons).
// 1 x 4096 x 4096 6.3 us (with the plan 7.4), 100 x 11008 x 4096 with bias and SiLU 16.2.
template <class P>
__global__ __launch_bounds__(P::NT, P::WAVES_PER_EU) void sk_scaled_flat_kernel(const half_t *A, const half_t *B, int M, int N, int K, int lda, int ldb,
                                                                                int tiles_m, uint32_t start_scale, int ldc, half_t *C, Scales scales,
                                                                                const void *epi) {
  __shared__ __attribute__((aligned(1024))) char smem[P::LDS_BYTES];
  typename P::Args a;
  if constexpr (std::is_base_of<SkinnyArgs, typename P::Args>::value) {
    a.W = B;
    a.ldw = ldb;
    a.scales = a.zeros = nullptr;
  } else {
    a.B = B;
    a.ldb = ldb;
    a.alpha = 1.f;
    a.scales = nullptr;
    a.start_scale = start_scale;
  }
  a.zero = a.groups = 0;
  a.A = A;
  a.C = C;
  a.M = M;
  a.N = N;
  a.K = K;
  a.lda = lda;
  a.ldc = ldc;
  a.s = scales;
  const FlatTile t = flat_tile(tiles_m, (N + P::BN - 1) / P::BN);
  typename P::Acc acc;
  P::prefetch_scales(a, acc, t.pm, t.pn, epi);
  P::mac(a, acc, t.pm, t.pn, 0, (K + iteration_k<P>() - 1) / iteration_k<P>(), smem);
  P::store_c(a, acc, t.pm, t.pn, smem, epi);
}

// F(id, policy)
#define SCALED_STREAM(id, MB, WM, WN, RK, DEPTH, NB, AD, PAD, KH) \
  F((id + 20), (ScaledStream<TileStreamPairs<MB, WM, WN, RK, DEPTH, false, NB, AD, PAD, KH, 3>>))
#define SCALED_WAVEK(T, id, FM, FN) F((id), (ScaledWaveK<TileWaveK<T, FM, FN, false>>))
#define SCALED_DMA(id, BM, BN, WM, WN) F((id), (ScaledDma<TileF16NTDma<BM, BN, WM, WN, false, 64, true, false, 3>>))
#define SCALED_DMA_BK64(id, BM, BN, WM, WN) F((id), (ScaledDma<TileF16NTDma<BM, BN, WM, WN, false, 32, true, false, 3>>))
#define FOR_SCALED_KERNELS                                       \
  SK_STREAM_BYTES_KERNELS(SCALED_STREAM)                         \
  SK_TILE_WAVEK_KERNELS(SCALED_WAVEK, WK_I8, wavek_base(WK_I8))  \
  SK_TILE_I8_KERNELS(SCALED_DMA)                                 \
  SK_TILE_I8_BK64_KERNELS(SCALED_DMA_BK64)

template <class T>
struct unparen;
template <class R, class P>
struct unparen<R(P)> { typedef P type; };

template <class Args>
static inline void set_operands_of(Args &a, const GemmArgs &g, const DevPlan &p) {
  if constexpr (std::is_base_of<SkinnyArgs, Args>::value) {
    static_cast<SkinnyArgs &>(a) = SkinnyArgs{g.A, g.B, nullptr, g.C, g.M, g.N, g.K, g.lda, g.ldb, g.ldc, 0, 0, nullptr};
  } else {
    static_cast<GemmArgs &>(a) = g;
    if constexpr (std::is_base_of<WaveKArgs, Args>::value) a.start_scale = start_scale(p);
  }
}

template <class P>
static int launch_scaled_policy(const GemmArgs &g, const Scales &sc, const DevPlan &p, const Workspace &ws, hipStream_t s, const void *bias) {
  typename P::Args a;
  set_operands_of(a, g, p);
  a.s = sc;
  if constexpr (has_prefetch_scales<P>::value) {
    if (flat_plan(g, p, iteration_k<P>())) {
      hipLaunchKernelGGL((sk_scaled_flat_kernel<P>), dim3(p.grid), dim3(P::NT), 0, s, g.A, g.B, g.M, g.N, g.K, (int)g.lda, (int)g.ldb, p.tiles_m,
                         start_scale(p), (int)g.ldc, g.C, sc, bias);
      return (int)hipGetLastError();
    }
  }
  if (p.sk_tiles == 0)
    hipLaunchKernelGGL((sk_scaled_kernel<P, false>), dim3(p.grid), dim3(P::NT), 0, s, a, p, ws, bias);
  else
    hipLaunchKernelGGL((sk_scaled_kernel<P, true>), dim3(p.grid), dim3(P::NT), 0, s, a, p, ws, bias);
  return (int)hipGetLastError();
}

bool has_scaled_i8(int id) {
  switch (id) {
#define F(ID, P) case ID:
    FOR_SCALED_KERNELS
#undef F
    return true;
  }
  return has_scaled_i8_asm(id);
}

int launch_scaled_i8(int id, const GemmArgs &a, const Scales &sc, const DevPlan &p, const Workspace &ws, hipStream_t s, const void *bias) {
  switch (id) {
#define F(ID, P) case ID: return launch_scaled_policy<unparen<void P>::type>(a, sc, p, ws, s, bias);
    FOR_SCALED_KERNELS
#undef F
  }
  return launch_scaled_i8_asm(id, a, sc, p, ws, s, bias);
}

int occupancy_scaled_i8(int id) {
  int occ = 0;
  switch (id) {
#define F(ID, P)                                                                                                                            \
  case ID: {                                                                                                                                \
    typedef unparen<void P>::type Q;                                                                                                        \
    return hipOccupancyMaxActiveBlocksPerMultiprocessor(&occ, sk_scaled_kernel<Q, true>, Q::NT, 0) == hipSuccess ? occ : -1;                \
  }
    FOR_SCALED_KERNELS
#undef F
  }
  return occupancy_scaled_i8_asm(id);
}

}  // namespace sk
