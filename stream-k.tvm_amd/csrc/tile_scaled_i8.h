// int8 products with a scale for each row of A (token) and each row of the weights (output channel):
//   C[m][n] = act(sa[m] * sb[n] * sum_k A[m][k] B[n][k] + bias[n]),  C in fp16 or bfloat16.
//
// The int8 policies with another end: sums, Stream-K segments and partial tiles stay int32, exact in every order, and the CTA that
// stores a tile converts its sums to fp32 (one rounding where a sum needs more than 24 bits), multiplies by the row's scale and the
// column's, adds the bias, applies the activation and rounds once.  C is half the bytes of the int32 result, and no second kernel
// reads it back.
#pragma once
#include "sk_device.h"
#include "tile_epilogue.h"
#include "tile_f16_dma.h"
#include "tile_stream_pairs.h"
#include "tile_wavek.h"

namespace sk {

struct Scales {
  const float *a, *b;   // of A's rows, of the weights' rows
  int bf16;             // C's type
};
template <class Base>
struct ScaledArgs : Base {
  Scales s;
};

typedef int intx4_s __attribute__((ext_vector_type(4)));

// four scales of consecutive columns (zero past N)
__device__ __forceinline__ floatx4 scale4_at(const float *s, int col, int N) {
  floatx4 r = {0.f, 0.f, 0.f, 0.f};
  if (col + 4 <= N && (reinterpret_cast<uintptr_t>(s) & 15) == 0) return *reinterpret_cast<const floatx4 *>(s + col);
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (col + e < N) r[e] = s[col + e];
  return r;
}
// activate() with the reciprocal (one ulp) in place of the division, which takes as long as all the rest of a value's way: 16 int8 experts
// of 4096 x 2048, 3000 rows, SiLU 82 and 74 us.  (No contraction here and below: every kernel gives the same bits.)
__device__ __forceinline__ float activate_by_rcp(float x, int act) {
#pragma clang fp contract(off)
  if (act == 2) return x * __builtin_amdgcn_rcpf(1.f + __expf(-2.f * (0.7978845608028654f * (x + 0.044715f * x * x * x))));
  if (act == 3) return x * __builtin_amdgcn_rcpf(1.f + __expf(-x));
  return activate(x, act);
}
// a value of C ahead of its rounding to 16 bits
template <bool EPI>
__device__ __forceinline__ float scaled_value(int x, float sa, float sb, float bias, int act) {
#pragma clang fp contract(off)
  const float y = (float)x * sa * sb;
  if constexpr (!EPI) return y;
  return activate_by_rcp(y + bias, act);
}
// EPI: bias and activation.  The instances differ in C's type and in EPI, and the store code is compiled for each: chosen by element,
// the 256 x 256 tiles' end took 30 us.
template <bool BF16, bool EPI>
__device__ __forceinline__ half4v scaled4(intx4_s x, float sa, floatx4 sb, floatx4 bias, int act) {
  floatx4 y;
#pragma unroll
  for (int e = 0; e < 4; ++e) y[e] = scaled_value<EPI>(x[e], sa, sb[e], bias[e], act);
  return round4<BF16>(y);
}
// f(BF16, EPI) as constants
template <class F>
__device__ __forceinline__ void by_result(bool bf16, const void *epi, F &&f) {
  if (epi == nullptr) {
    if (bf16) f(std::true_type{}, std::false_type{});
    else f(std::false_type{}, std::false_type{});
  } else {
    if (bf16) f(std::true_type{}, std::true_type{});
    else f(std::false_type{}, std::true_type{});
  }
}

// Four bias values of C's type as they lie in memory (zeros without a bias)
__device__ __forceinline__ half4v raw_bias4_at(const half_t *bias, int col, int N) {
  half4v r = {0, 0, 0, 0};
  if (bias == nullptr) return r;
  if (col + 4 <= N && (reinterpret_cast<uintptr_t>(bias) & 7) == 0) return *reinterpret_cast<const half4v *>(bias + col);
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (col + e < N) r[e] = bias[col + e];
  return r;
}
template <bool BF16>
__device__ __forceinline__ floatx4 widen4(half4v h) {
  floatx4 r;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const half_t x = h[e];
    if constexpr (BF16) r[e] = __builtin_bit_cast(float, (uint32_t)__builtin_bit_cast(uint16_t, x) << 16);
    else r[e] = (float)x;
  }
  return r;
}

// What the columns of a wave's FN blocks and the rows of its FM blocks bring along.  All of it is requested before any is looked at, and
// columns inside the matrix without a branch of their own: each wait for memory costs a launch of one round of tiles a microsecond.
template <int FM, int FN, bool BF16, bool EPI>
struct ScaleRegs {
  floatx4 sb[FN];
  half4v bias[EPI ? FN : 1];
  float sa[FM];
  int act;
  template <class Args>
  __device__ __forceinline__ ScaleRegs(const Args &a, int row0, int col0, const void *epi) {
    const int lane = pin_here((int)threadIdx.x) & 63, col = col0 + 4 * (lane >> 4);
    act = EPI ? epi_act(epi) : 0;
    const half_t *b = EPI ? epi_bias(epi) : nullptr;
#pragma unroll
    for (int i = 0; i < FM; ++i) sa[i] = a.s.a[min(row0 + 16 * i + (lane & 15), a.M - 1)];
    if (col0 + 16 * FN <= a.N && (reinterpret_cast<uintptr_t>(a.s.b) & 15) == 0 && (reinterpret_cast<uintptr_t>(b) & 7) == 0) {
#pragma unroll
      for (int j = 0; j < FN; ++j) sb[j] = *reinterpret_cast<const floatx4 *>(a.s.b + col + 16 * j);
      if constexpr (EPI) {
#pragma unroll
        for (int j = 0; j < FN; ++j) bias[j] = half4v{0, 0, 0, 0};
        if (b != nullptr) {
#pragma unroll
          for (int j = 0; j < FN; ++j) bias[j] = *reinterpret_cast<const half4v *>(b + col + 16 * j);
        }
      }
    } else {
#pragma unroll
      for (int j = 0; j < FN; ++j) {
        sb[j] = scale4_at(a.s.b, col + 16 * j, a.N);
        if constexpr (EPI) bias[j] = raw_bias4_at(b, col + 16 * j, a.N);
      }
    }
  }
  template <int I, int J>
  __device__ __forceinline__ half4v values(intx4_s x) const {
    floatx4 b = {0.f, 0.f, 0.f, 0.f};
    if constexpr (EPI) b = widen4<BF16>(bias[J]);
    return scaled4<BF16, EPI>(x, sa[I], sb[J], b, act);
  }
};

// LDS-tiled kernels (128 x 128 and relatives)
template <class P>
struct ScaledDma : P {
  static_assert(P::I8, "int8 tiles");
  typedef ScaledArgs<GemmArgs> Args;
  typedef typename P::Acc Acc;
  typedef BlockPatch<P::FM, P::FN> Patch;
  static_assert(P::NW * Patch::BYTES <= P::STAGE_BYTES, "the patches fit a stage");
  template <int I0, int I1>
  static __device__ __forceinline__ void store_rows(const Args &a, const Acc &acc, int pm, int pn, const void *epi) {
    const int wave = threadIdx.x >> 6, wm = wave / P::WN, wn = wave % P::WN;
    const int row0 = pm * P::BM + wm * P::WTM, col0 = pn * P::BN + wn * P::WTN;
    by_result(a.s.bf16 != 0, epi, [&](auto bf16, auto with_epi) {
      const ScaleRegs<P::FM, P::FN, decltype(bf16)::value, decltype(with_epi)::value> r(a, row0, col0, epi);
      Patch::template store<I0, I1>(a.C, a.ldc, a.M, a.N, row0, col0, P::stage(0) + wave * Patch::BYTES, [&](auto i, auto j) {
        return r.template values<decltype(i)::value, decltype(j)::value>(acc.v[i][j]);
      });
    });
    __syncthreads();   // the patches overlap the stages of the next tile
  }
  static __device__ __forceinline__ void store_c(const Args &a, const Acc &acc, int pm, int pn, char *, const void *epi) {
    store_rows<0, P::FM>(a, acc, pm, pn, epi);
  }
  static __device__ __forceinline__ void store_c_half(const Args &a, const Acc &acc, int pm, int pn, char *, const void *epi, int h) {
    if (h == 0) store_rows<0, P::FM / 2>(a, acc, pm, pn, epi);
    else store_rows<P::FM / 2, P::FM>(a, acc, pm, pn, epi);
  }
};

// tiles whose waves stream K on their own: a thread holds pieces of four columns of one row.  Their scales and biases are requested
// before the tile's loop; behind it their way from memory would be waited for (2 to 5 us of a launch).  Tiles of 64 x 128 have no
// registers left for that; theirs are read at the end.
template <class P>
struct ScaledWaveK : P {
  typedef ScaledArgs<WaveKArgs> Args;
  static constexpr bool SCALES_AHEAD = P::BM * P::BN < 64 * 128;
  static constexpr int COLS = P::ONE_COL ? 1 : P::PIECES;   // (pieces below each other share their columns' scales)
  struct Ends {
    floatx4 sb[COLS];
    half4v b4[COLS];
    float sa[P::PIECES];
  };
  struct Nothing {};
  struct Acc : P::Acc {
    std::conditional_t<SCALES_AHEAD, Ends, Nothing> ends;
  };
  static __device__ __forceinline__ void fetch(const Args &a, Ends &ends, int pm, int pn, const void *epi, int tid) {
#pragma unroll
    for (int u = 0; u < P::PIECES; ++u) {
      const int row = pm * P::BM + P::piece_row(u, tid), col = pn * P::BN + P::piece_col(u, tid) * 4;
      ends.sa[u] = a.s.a[min(row, a.M - 1)];
      if (u < COLS) {
        ends.sb[u] = scale4_at(a.s.b, col, a.N);
        ends.b4[u] = raw_bias4_at(epi_bias(epi), col, a.N);
      }
    }
  }
  static __device__ __forceinline__ void prefetch_scales(const Args &a, Acc &acc, int pm, int pn, const void *epi) {
    if constexpr (SCALES_AHEAD) fetch(a, acc.ends, pm, pn, epi, threadIdx.x);
  }
  static __device__ __forceinline__ void store_c(const Args &a, const Acc &acc, int pm, int pn, char *, const void *epi) {
    const int tid = pin_here((int)threadIdx.x);
    if constexpr (SCALES_AHEAD) {
      store_by_type(a, acc, acc.ends, pm, pn, epi, tid);
    } else {
      Ends ends;
      fetch(a, ends, pm, pn, epi, tid);
      store_by_type(a, acc, ends, pm, pn, epi, tid);
    }
  }
  static __device__ __forceinline__ void store_by_type(const Args &a, const Acc &acc, const Ends &ends, int pm, int pn, const void *epi, int tid) {
    by_result(a.s.bf16 != 0, epi, [&](auto bf16, auto with_epi) { store<decltype(bf16)::value, decltype(with_epi)::value>(a, acc, ends, pm, pn, epi, tid); });
  }
  template <bool BF16, bool EPI>
  static __device__ __forceinline__ void store(const Args &a, const Acc &acc, const Ends &ends, int pm, int pn, const void *epi, int tid) {
    const int act = EPI ? epi_act(epi) : 0;
    const bool vec_ok = (a.ldc & 3) == 0 && (reinterpret_cast<uintptr_t>(a.C) & 7) == 0;
#pragma unroll
    for (int u = 0; u < P::PIECES; ++u) {
      const int row = pm * P::BM + P::piece_row(u, tid), col = pn * P::BN + P::piece_col(u, tid) * 4;
      if (row >= a.M || col >= a.N) continue;
      const half4v h = scaled4<BF16, EPI>(acc.c[u], ends.sa[u], ends.sb[u % COLS], widen4<BF16>(ends.b4[u % COLS]), act);
      half_t *dst = a.C + (int64_t)row * a.ldc + col;
      if (vec_ok && col + 4 <= a.N) {
        *reinterpret_cast<half4v *>(dst) = h;
      } else {
        for (int e = 0; e < 4 && col + e < a.N; ++e) dst[e] = h[e];
      }
    }
  }
};

// up to 64 rows, the weights streaming through LDS: the same
template <class P>
struct ScaledStream : P {
  typedef ScaledArgs<SkinnyArgs> Args;
  static constexpr bool SCALES_AHEAD = true;
  struct Acc : P::Acc {
    floatx4 sb[P::NB];
    half4v b4[P::NB];
    float sa[P::MB];
  };
  static __device__ __forceinline__ void origin(int pm, int pn, int &row0, int &col0) {
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, wm = wave % P::WM, wn = wave / P::WM % P::WN;
    row0 = pm * P::BM + wm * P::MB * 16 + (lane & 15);
    col0 = pn * P::BN + wn * P::NB * 16 + 4 * (lane >> 4);
  }
  static __device__ __forceinline__ void prefetch_scales(const Args &a, Acc &acc, int pm, int pn, const void *epi) {
    int row0, col0;
    origin(pm, pn, row0, col0);
#pragma unroll
    for (int i = 0; i < P::MB; ++i) acc.sa[i] = a.s.a[min(row0 + 16 * i, a.M - 1)];
#pragma unroll
    for (int j = 0; j < P::NB; ++j) {
      acc.sb[j] = scale4_at(a.s.b, col0 + 16 * j, a.N);
      acc.b4[j] = raw_bias4_at(epi_bias(epi), col0 + 16 * j, a.N);
    }
  }
  static __device__ __forceinline__ void store_c(const Args &a, const Acc &acc, int pm, int pn, char *, const void *epi) {
    if ((int)(threadIdx.x >> 6) >= P::WM * P::WN) return;
    int row0, col0;
    origin(pm, pn, row0, col0);
    const int act = epi_act(epi);
    const bool vec_ok = (a.ldc & 3) == 0 && (reinterpret_cast<uintptr_t>(a.C) & 7) == 0;
    by_result(a.s.bf16 != 0, epi, [&](auto bf16, auto with_epi) {
      static_for<0, P::MB>([&](auto i) {
        static_for<0, P::NB>([&](auto j) {
          const int row = row0 + 16 * i, col = col0 + 16 * j;
          if (row >= a.M || col >= a.N) return;
          const half4v h = scaled4<decltype(bf16)::value, decltype(with_epi)::value>(acc.c[i][j], acc.sa[i], acc.sb[j],
                                                                                     widen4<decltype(bf16)::value>(acc.b4[j]), act);
          half_t *dst = a.C + (int64_t)row * a.ldc + col;
          if (vec_ok && col + 4 <= a.N) {
            *reinterpret_cast<half4v *>(dst) = h;
          } else {
            for (int e = 0; e < 4 && col + e < a.N; ++e) dst[e] = h[e];
          }
        });
      });
    });
  }
};

}  // namespace sk
