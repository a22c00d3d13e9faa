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
__device__ __forceinline__ half4v scaled4(intx4_s x, float sa, floatx4 sb, floatx4 bias, int act, bool bf16) {
  floatx4 y;
#pragma unroll
  for (int e = 0; e < 4; ++e) y[e] = activate((float)x[e] * sa * sb[e] + bias[e], act);
  return round4(y, bf16);
}

// what the columns of a wave's FN blocks and the rows of its FM blocks bring along
template <int FM, int FN>
struct ScaleRegs {
  floatx4 sb[FN], bias[FN];
  float sa[FM];
  int act;
  bool bf16;
  template <class Args>
  __device__ __forceinline__ void load(const Args &a, int row0, int col0, const void *epi) {
    const int lane = pin_here((int)threadIdx.x) & 63;
    const half_t *b = epi_bias(epi);
    act = epi_act(epi);
    bf16 = a.s.bf16 != 0;
#pragma unroll
    for (int i = 0; i < FM; ++i) {
      const int row = row0 + 16 * i + (lane & 15);
      sa[i] = row < a.M ? a.s.a[row] : 0.f;
    }
#pragma unroll
    for (int j = 0; j < FN; ++j) {
      const int col = col0 + 16 * j + 4 * (lane >> 4);
      sb[j] = scale4_at(a.s.b, col, a.N);
      bias[j] = bias4_of(b, col, a.N, bf16);
    }
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
    ScaleRegs<P::FM, P::FN> r;
    r.load(a, row0, col0, epi);
    Patch::template store<I0, I1>(a.C, a.ldc, a.M, a.N, row0, col0, P::stage(0) + wave * Patch::BYTES, [&](auto i, auto j) {
      return scaled4(acc.v[i][j], r.sa[i], r.sb[j], r.bias[j], r.act, r.bf16);
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

// tiles whose waves stream K on their own: a thread holds pieces of four columns of one row
template <class P>
struct ScaledWaveK : P {
  typedef ScaledArgs<WaveKArgs> Args;
  typedef typename P::Acc Acc;
  static __device__ __forceinline__ void store_c(const Args &a, const Acc &acc, int pm, int pn, char *, const void *epi) {
    const int tid = pin_here((int)threadIdx.x), act = epi_act(epi);
    const half_t *bias = epi_bias(epi);
    const bool bf16 = a.s.bf16 != 0, vec_ok = (a.ldc & 3) == 0 && (reinterpret_cast<uintptr_t>(a.C) & 7) == 0;
    floatx4 sb[P::PIECES], b4[P::PIECES];
    float sa[P::PIECES];
#pragma unroll
    for (int u = 0; u < P::PIECES; ++u) {   // all loads at once
      const int row = pm * P::BM + P::piece_row(u, tid), col = pn * P::BN + P::piece_col(u, tid) * 4;
      sa[u] = row < a.M ? a.s.a[row] : 0.f;
      sb[u] = scale4_at(a.s.b, col, a.N);
      b4[u] = bias4_of(bias, col, a.N, bf16);
    }
#pragma unroll
    for (int u = 0; u < P::PIECES; ++u) {
      const int row = pm * P::BM + P::piece_row(u, tid), col = pn * P::BN + P::piece_col(u, tid) * 4;
      if (row >= a.M || col >= a.N) continue;
      const half4v h = scaled4(acc.c[u], sa[u], sb[u], b4[u], act, bf16);
      half_t *dst = a.C + (int64_t)row * a.ldc + col;
      if (vec_ok && col + 4 <= a.N) {
        *reinterpret_cast<half4v *>(dst) = h;
      } else {
        for (int e = 0; e < 4 && col + e < a.N; ++e) dst[e] = h[e];
      }
    }
  }
};

// up to 64 rows, the weights streaming through LDS
template <class P>
struct ScaledStream : P {
  typedef ScaledArgs<SkinnyArgs> Args;
  typedef typename P::Acc Acc;
  static __device__ __forceinline__ void store_c(const Args &a, const Acc &acc, int pm, int pn, char *, const void *epi) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    if (wave >= P::WM * P::WN) return;
    const int wm = wave % P::WM, wn = wave / P::WM;
    const int row0 = pm * P::BM + wm * P::MB * 16, col0 = pn * P::BN + wn * P::NB * 16;
    const bool vec_ok = (a.ldc & 3) == 0 && (reinterpret_cast<uintptr_t>(a.C) & 7) == 0;
    ScaleRegs<P::MB, P::NB> r;
    r.load(a, row0, col0, epi);
#pragma unroll
    for (int i = 0; i < P::MB; ++i) {
      const int row = row0 + 16 * i + (lane & 15);
#pragma unroll
      for (int j = 0; j < P::NB; ++j) {
        const int col = col0 + 16 * j + 4 * (lane >> 4);
        if (row >= a.M || col >= a.N) continue;
        const half4v h = scaled4(acc.c[i][j], r.sa[i], r.sb[j], r.bias[j], r.act, r.bf16);
        half_t *dst = a.C + (int64_t)row * a.ldc + col;
        if (vec_ok && col + 4 <= a.N) {
          *reinterpret_cast<half4v *>(dst) = h;
        } else {
          for (int e = 0; e < 4 && col + e < a.N; ++e) dst[e] = h[e];
        }
      }
    }
  }
};

}  // namespace sk
