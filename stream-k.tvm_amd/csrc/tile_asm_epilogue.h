// The end of a tile of the assembly-loop kernels (tile_f16_asm.h: block (i, j) of a wave's 128 x 128 in a[(8 i + j) 4 .. + 3]) with bias,
// activation or scales, through the wave's patch behind the stages, which it leaves alone.
//
// 16 rows x 64 columns at a time go into the patch as they are, 32 bits a value, and come back as rows: lane l has columns
// 8 (l % 8) .. + 7 of rows l / 8 and l / 8 + 8.  So a lane's columns are the same for all rows, their scales and biases are read once a
// tile, and all that depends on a register's number is its copy: the arithmetic is a loop, for one activation at a time.  Written
// out for every block -- 64 times four activations -- it was the fetching of instructions that took the time, 20 to 30 us a tile: 8 experts of
// 11008 x 4096, 8192 rows, bias and SiLU, bfloat16 743 us, without them 565; int8 461 and 321.  Now 617 and 578, 358 and 333.
#pragma once
#include "tile_epilogue.h"
#include "tile_f16_asm.h"
#include "tile_scaled_i8.h"

namespace sk {

// P: the policy; BF16: C's type; EPI: -1 nothing, else bias and the activation of this number
template <class P, bool SCALED, bool BF16, int EPI>
struct AsmEnd {
  static constexpr int STRIDE = P::PATCH_STRIDE;
  static_assert(STRIDE == 64 * 4 + 16 && P::FN == 8 && P::WTN == 128, "16 rows of 64 values and a pad against bank conflicts");
  template <int HALF, int II>
  static __device__ __forceinline__ void copy_block_row(char *to) {
    static_for<0, 4>([&](auto j) {
      constexpr int jj = decltype(j)::value;
      *reinterpret_cast<floatx4 *>(to + jj * 64) = agpr_read4<(II * 8 + HALF * 4 + jj) * 4>();
    });
  }
  template <int HALF>
  static __device__ __forceinline__ void copy_row(int ii, char *to) {   // (ii: uniform)
    switch (ii) {
      case 0: return copy_block_row<HALF, 0>(to);
      case 1: return copy_block_row<HALF, 1>(to);
      case 2: return copy_block_row<HALF, 2>(to);
      case 3: return copy_block_row<HALF, 3>(to);
      case 4: return copy_block_row<HALF, 4>(to);
      case 5: return copy_block_row<HALF, 5>(to);
      case 6: return copy_block_row<HALF, 6>(to);
      default: return copy_block_row<HALF, 7>(to);
    }
  }
  static __device__ __forceinline__ void sync() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
  }
  struct Columns {
    floatx4 scale[SCALED ? 2 : 1];
    half4v bias[EPI >= 0 ? 2 : 1];
    __device__ __forceinline__ void load(const float *s, const half_t *b, int col, int N) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        if constexpr (SCALED) scale[h] = scale4_at(s, col + 4 * h, N);
        if constexpr (EPI >= 0) bias[h] = raw_bias4_at(b, col + 4 * h, N);
      }
    }
  };
  // rows row0 + 16 i0 .. of the wave's block that stands at (row0, col0)
  static __device__ __forceinline__ void store(half_t *C, int64_t ldc, int M, int N, int row0, int col0, const float *sa, const float *sb, const half_t *bias,
                                               int i0, int i1) {
    const int lane = pin_here((int)threadIdx.x) & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    char *patch = P::lds() + 2 * P::STAGE_BYTES + wave * P::FAST_PATCH_BYTES;
    char *to = patch + (lane & 15) * STRIDE + (lane >> 4) * 16;
    const char *from = patch + (lane >> 3) * STRIDE + (lane & 7) * 32;
    const int col = col0 + (lane & 7) * 8;
    const bool vec_ok = (ldc & 7) == 0 && (reinterpret_cast<uintptr_t>(C) & 15) == 0;
    float sa_lo = 0.f, sa_hi = 0.f;   // of rows row0 + lane and row0 + 64 + lane
    if constexpr (SCALED) {
      sa_lo = sa[min(row0 + lane, M - 1)];
      sa_hi = sa[min(row0 + 64 + lane, M - 1)];
    }
    Columns columns[2];
    columns[0].load(sb, bias, col, N);
    columns[1].load(sb, bias, col + 64, N);
    auto emit = [&](int ii, int half) {
#pragma unroll
      for (int pass = 0; pass < 2; ++pass) {
        const int r = 16 * ii + 8 * pass + (lane >> 3), row = row0 + r, c0 = col + 64 * half;
        float s = 0.f;
        if constexpr (SCALED) s = __shfl(ii < 4 ? sa_lo : sa_hi, r & 63, 64);
        half4v h[2];
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          floatx4 y = *reinterpret_cast<const floatx4 *>(from + pass * 8 * STRIDE + q * 16);
          floatx4 b = {0.f, 0.f, 0.f, 0.f};
          if constexpr (EPI >= 0) b = widen4<BF16>(columns[half].bias[q]);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            if constexpr (SCALED) y[e] = scaled_value<EPI >= 0>(__builtin_bit_cast(intx4_s, y)[e], s, columns[half].scale[q][e], b[e], EPI);
            else if constexpr (EPI >= 0) y[e] = activate_by_rcp(y[e] + b[e], EPI);
          }
          h[q] = round4<BF16>(y);
        }
        if (row < M && c0 < N) {
          half_t *dst = C + (int64_t)row * ldc + c0;
          if (vec_ok && c0 + 8 <= N) {
            struct alignas(16) Eight { half4v h[2]; };
            *reinterpret_cast<Eight *>(dst) = Eight{{h[0], h[1]}};
          } else {
#pragma unroll
            for (int e = 0; e < 8; ++e)
              if (c0 + e < N) dst[e] = h[e / 4][e % 4];
          }
        }
      }
      sync();
    };
#pragma unroll 1
    for (int ii = i0; ii < i1; ++ii) {
      copy_row<0>(ii, to);
      sync();
      emit(ii, 0);
      copy_row<1>(ii, to);
      sync();
      emit(ii, 1);
    }
  }
};
// f(std::integral_constant<int, EPI>)
template <class F>
__device__ __forceinline__ void by_epilogue(const void *epi, F &&f) {
  if (epi == nullptr) return f(std::integral_constant<int, -1>{});
  switch (epi_act(epi)) {
    case 1: return f(std::integral_constant<int, 1>{});
    case 2: return f(std::integral_constant<int, 2>{});
    case 3: return f(std::integral_constant<int, 3>{});
    default: return f(std::integral_constant<int, 0>{});
  }
}

}  // namespace sk
