// Epilogue pieces of the kernels whose result is formed from accumulator blocks of 16 x 16 (lane l of block (i, j) holds
// C[16 i + l % 16][16 j + 4 (l / 16) + e]): rounding to C's 16-bit type, bias, and stores of whole row pieces.
#pragma once
#include "sk_device.h"

namespace sk {

// four fp32 values, rounded to bfloat16 or fp16 (C and the patches carry 16-bit patterns).  The conversion is an instruction of its own: the
// compiler may merge one to fp16 with the multiplication in front of it, which rounds once where another kernel rounds twice.
template <bool BF16>
__device__ __forceinline__ half4v round4(floatx4 x) {
  union { uint32_t w[2]; half4v h; } r;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    if constexpr (BF16) asm("v_cvt_pk_bf16_f32 %0, %1, %2" : "=v"(r.w[i]) : "v"(x[2 * i]), "v"(x[2 * i + 1]));
    else asm("v_cvt_pk_f16_f32 %0, %1, %2" : "=v"(r.w[i]) : "v"(x[2 * i]), "v"(x[2 * i + 1]));
  }
  return r.h;
}

// 16 bytes anywhere in a row of C: the hardware takes them at any multiple of 2 bytes.
typedef uint4v AnyPiece __attribute__((aligned(2)));

// Stores FM x FN blocks of a wave, the first of which stands at (row0, col0) of C, through a patch of LDS of the wave's own
// (16 rows of FN * 32 + 16 bytes: the padding keeps the 8-byte writes and the 16-byte reads on different banks), one row of
// blocks at a time: 16-byte stores along rows of C instead of 8-byte ones down them.  block(ii, jj) gives the lane's four
// values; ii and jj are compile-time constants.
template <int FM, int FN>
struct BlockPatch {
  static constexpr int STRIDE = FN * 32 + 16, BYTES = 16 * STRIDE, PPR = FN * 2;   // PPR pieces of 16 bytes make a row
  static_assert((16 * PPR) % 64 == 0, "the lanes share out the pieces of a row of blocks evenly");
  template <int I0 = 0, int I1 = FM, class Block>
  static __device__ __forceinline__ void store(half_t *C, int64_t ldc, int M, int N, int row0, int col0, char *patch, Block &&block) {
    const int lane = pin_here((int)threadIdx.x) & 63;
    static_for<I0, I1>([&](auto bi) {
      constexpr int ii = decltype(bi)::value;
      static_for<0, FN>([&](auto bj) {
        constexpr int jj = decltype(bj)::value;
        *reinterpret_cast<half4v *>(patch + (lane & 15) * STRIDE + jj * 32 + (lane >> 4) * 8) = block(bi, bj);
      });
      __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
      __builtin_amdgcn_wave_barrier();
      __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
      uint4v v[16 * PPR / 64];
#pragma unroll
      for (int s = 0; s < 16 * PPR / 64; ++s) {
        const int idx = s * 64 + lane;
        v[s] = *reinterpret_cast<const uint4v *>(patch + (idx / PPR) * STRIDE + (idx % PPR) * 16);
      }
#pragma unroll
      for (int s = 0; s < 16 * PPR / 64; ++s) {
        const int idx = s * 64 + lane, row = row0 + 16 * ii + idx / PPR, col = col0 + (idx % PPR) * 8;
        if (row < M && col < N) {
          half_t *dst = C + (int64_t)row * ldc + col;
          if (col + 8 <= N) {
            *reinterpret_cast<AnyPiece *>(dst) = v[s];
          } else {
            union { uint4v q; half_t h[8]; } u;
            u.q = v[s];
#pragma unroll
            for (int e = 0; e < 8; ++e)
              if (col + e < N) dst[e] = u.h[e];
          }
        }
      }
      __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
      __builtin_amdgcn_wave_barrier();
      __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    });
  }
};

}  // namespace sk
