// Microscaled 4-bit floating point: 32 neighbours of a row share a power of two X = 2^(floor(log2 max|x|) - 2) (at least 2^-127), kept as its
// biased exponent in a byte, and each becomes x / X to the nearest e2m1 number (0, .5, 1, 1.5, 2, 3, 4, 6; ties to the even code), at most 6.
// Value 2 i of a row is the low half of byte i.  A block with an infinity or a NaN has scale 255, the format's NaN, and codes 0.
//
// Both directions are one pass over memory, 16 bits and 17/32 of a byte a value, and what bounds them is that: a thread has eight values
// (the conversions of this target take two at a time), four neighbours a block, whose maximum is two steps within a quad.  28672 x 8192: 6.3
// and 6.9 TB/s; of 32 bits 5.1 and 6.2 (a copy of 0.5 to 1 GB reaches 5.1 to 5.3).
#include <hip/hip_runtime.h>

#include "sk_device.h"
#include "streamk.h"
#include "wide_grid.h"

using namespace sk;

namespace {

// Arrays of values above half of the last cache's bytes (256 MB) pass it by, which leaves room for codes: 28672 x 8192 of 16 bits 104 us (5.7 TB/s),
// so 94, back 105 and 86; 14336 rows 54 and 50, 51 and 45.  One that fits may be there: 4096 rows 16 us, past the caches 18.
constexpr int64_t CACHED = (int64_t)128 << 20;
constexpr int THREADS = 256, PIECES = 4;   // pieces of eight values that a thread has in flight
enum { EL_F16 = 0, EL_BF16 = 1, EL_F32 = 2 };
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));

template <int EL>
struct Eight {
  uint32_t w[EL == EL_F32 ? 8 : 4];
};

// the largest magnitude as the bits of a float: infinities and NaN are above every number
template <int EL>
__device__ __forceinline__ uint32_t largest(const Eight<EL> &v) {
  if constexpr (EL == EL_F32) {
    uint32_t most = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) most = max(most, v.w[i] & 0x7fffffffu);
    return most;
  } else {
    typedef uint16_t ushort2v __attribute__((ext_vector_type(2)));
    ushort2v pair = {0, 0};
#pragma unroll
    for (int i = 0; i < 4; ++i) pair = __builtin_elementwise_max(pair, __builtin_bit_cast(ushort2v, v.w[i] & 0x7fff7fffu));
    const uint32_t most = max((uint32_t)pair[0], (uint32_t)pair[1]);
    if constexpr (EL == EL_BF16) return most << 16;
    const float f = (float)__builtin_bit_cast(half_t, (uint16_t)most);   // (exact, infinities and NaN as well)
    return __builtin_bit_cast(uint32_t, f);
  }
}
// of the four threads of a block
__device__ __forceinline__ uint32_t quad_max(uint32_t x) {
  x = max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0xb1, 0xf, 0xf, true));   // lanes 1 0 3 2
  return max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x4e, 0xf, 0xf, true));   // lanes 2 3 0 1
}
__device__ __forceinline__ uint32_t scale_byte(uint32_t most) {
  const uint32_t field = most >> 23;   // floor(log2) + 127, 0 below the normal numbers
  return field == 255 ? 255 : (field < 2 ? 0 : field - 2);
}
// 2^(byte - 127)
__device__ __forceinline__ float scale_value(uint32_t byte) { return __builtin_bit_cast(float, byte == 0 ? 0x00400000u : byte << 23); }

template <int EL>
__device__ __forceinline__ uint32_t encode(const Eight<EL> &v, uint32_t byte) {
  const float x = scale_value(byte);
  uint32_t q = 0;
  if constexpr (EL == EL_F32) {
    const float *f = reinterpret_cast<const float *>(v.w);
    q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, f[0], f[1], x, 0);
    q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, f[2], f[3], x, 1);
    q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, f[4], f[5], x, 2);
    q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, f[6], f[7], x, 3);
  } else if constexpr (EL == EL_BF16) {
    q = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(q, __builtin_bit_cast(bf16x2, v.w[0]), x, 0);
    q = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(q, __builtin_bit_cast(bf16x2, v.w[1]), x, 1);
    q = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(q, __builtin_bit_cast(bf16x2, v.w[2]), x, 2);
    q = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(q, __builtin_bit_cast(bf16x2, v.w[3]), x, 3);
  } else {
    q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(q, __builtin_bit_cast(half2v, v.w[0]), x, 0);
    q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(q, __builtin_bit_cast(half2v, v.w[1]), x, 1);
    q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(q, __builtin_bit_cast(half2v, v.w[2]), x, 2);
    q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(q, __builtin_bit_cast(half2v, v.w[3]), x, 3);
  }
  return byte == 255 ? 0 : q;
}

// Rows of `pieces` pieces, `blocks` workgroups to a row.  (Rows without a gap between them are one row.)
// VEC: 16-byte loads; PAST: past the caches
template <int EL, bool VEC, bool PAST>
__global__ __launch_bounds__(THREADS) void quantize_kernel(const char *X, int64_t rows, int64_t pieces, int64_t ldx_bytes, int64_t blocks, uint32_t *Q,
                                                           uint8_t *scales) {
  constexpr int BYTES = EL == EL_F32 ? 32 : 16;
  const int64_t block = wide_block(), row = block / blocks;
  if (row >= rows) return;
  const int64_t first = (block - row * blocks) * (THREADS * PIECES) + threadIdx.x;
  const char *x = X + row * ldx_bytes;
  Eight<EL> v[PIECES];
#pragma unroll
  for (int i = 0; i < PIECES; ++i) {
    const int64_t p = first + i * THREADS;
    if (p >= pieces) continue;   // (a block's four threads all or none: pieces is a multiple of four)
    if constexpr (VEC) {
      const uint4v *from = reinterpret_cast<const uint4v *>(x + p * BYTES);
#pragma unroll
      for (int h = 0; h < BYTES / 16; ++h) {
        const uint4v w = PAST ? __builtin_nontemporal_load(from + h) : from[h];
#pragma unroll
        for (int e = 0; e < 4; ++e) v[i].w[4 * h + e] = w[e];
      }
    } else {
      typedef typename std::conditional<EL == EL_F32, uint32_t, uint16_t>::type Word;
      const Word *from = reinterpret_cast<const Word *>(x + p * BYTES);
      Word *to = reinterpret_cast<Word *>(v[i].w);
#pragma unroll
      for (int e = 0; e < 8; ++e) to[e] = from[e];
    }
  }
#pragma unroll
  for (int i = 0; i < PIECES; ++i) {
    const int64_t p = first + i * THREADS;
    if (p >= pieces) continue;
    const uint32_t byte = scale_byte(quad_max(largest<EL>(v[i])));
    Q[row * pieces + p] = encode<EL>(v[i], byte);
    if ((threadIdx.x & 3) == 0) scales[(row * pieces + p) >> 2] = (uint8_t)byte;
  }
}

// A thread has 16 bytes of values a piece: eight or, of 32 bits, four.
template <int EL, bool VEC, bool PAST>
__global__ __launch_bounds__(THREADS) void dequantize_kernel(const char *Q, const uint8_t *scales, int64_t pieces, char *X) {
  constexpr int VALUES = EL == EL_F32 ? 4 : 8, MORE = PIECES * 8 / VALUES;
  typedef typename std::conditional<EL == EL_F32, uint16_t, uint32_t>::type Codes;
  const int64_t first = wide_block() * (THREADS * MORE) + threadIdx.x;
  uint32_t q[MORE], byte[MORE];
#pragma unroll
  for (int i = 0; i < MORE; ++i) {
    const int64_t p = first + i * THREADS;
    q[i] = byte[i] = 0;
    if (p < pieces) {
      q[i] = reinterpret_cast<const Codes *>(Q)[p];
      byte[i] = scales[p / (32 / VALUES)];
    }
  }
#pragma unroll
  for (int i = 0; i < MORE; ++i) {
    const int64_t p = first + i * THREADS;
    if (p >= pieces) continue;
    const float x = byte[i] == 255 ? __builtin_nanf("") : scale_value(byte[i]);
    float f[8];   // (the code's number is exact, and so is its product unless it is NaN, or infinite)
    auto two = [&](int at, auto pair) {
      f[at] = pair[0] * x;
      f[at + 1] = pair[1] * x;
    };
    two(0, __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q[i], 1.f, 0));
    two(2, __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q[i], 1.f, 1));
    if constexpr (VALUES == 8) {
      two(4, __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q[i], 1.f, 2));
      two(6, __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q[i], 1.f, 3));
    }
    typedef typename std::conditional<EL == EL_F32, uint32_t, uint16_t>::type Word;
    union { Word h[VALUES]; uint4v w; } o;
#pragma unroll
    for (int e = 0; e < VALUES; ++e) {
      if constexpr (EL == EL_F32) o.h[e] = __builtin_bit_cast(uint32_t, f[e]);
      else if constexpr (EL == EL_BF16) o.h[e] = __builtin_bit_cast(uint16_t, (__bf16)f[e]);
      else o.h[e] = __builtin_bit_cast(uint16_t, (half_t)f[e]);
    }
    if constexpr (VEC) {
      uint4v *to = reinterpret_cast<uint4v *>(X) + p;
      if constexpr (PAST) __builtin_nontemporal_store(o.w, to);
      else *to = o.w;
    } else {
#pragma unroll
      for (int e = 0; e < VALUES; ++e) reinterpret_cast<Word *>(X)[VALUES * p + e] = o.h[e];
    }
  }
}

// Scales as the tiles with many rows read them: 16 bytes for 512 values of a row, those of all rows together, pair by pair of 256 values,
// with zeros behind the last.  A workgroup turns 64 rows of up to 256 bytes through LDS; two arrays in one launch.
struct TileScales {
  const uint8_t *from;
  uint8_t *to;
  int64_t rows;
};
struct __attribute__((packed)) AnyBytes { uint4v w; };   // (the hardware takes 16 bytes at any address)
__global__ __launch_bounds__(THREADS) void tile_scales_kernel(TileScales a, TileScales b, int64_t blocks_a, int blocks) {
  constexpr int EACH = 64 * 16 / THREADS;
  __shared__ uint4v part[64][17];   // [row][16 bytes], a column of padding
  const bool second = (int64_t)blockIdx.x >= blocks_a;
  const TileScales &t = second ? b : a;
  const int64_t row0 = ((int64_t)blockIdx.x - (second ? blocks_a : 0)) * 64;
  const int pieces = (blocks + 15) / 16, p0 = (int)blockIdx.y * 16;
  uint4v w[EACH];
#pragma unroll
  for (int q = 0; q < EACH; ++q) {
    const int i = threadIdx.x + q * THREADS, p = p0 + i % 16, n = blocks - 16 * p;   // (n: bytes from here to the row's end)
    const int64_t row = row0 + i / 16;
    w[q] = uint4v{0, 0, 0, 0};
    if (row >= t.rows || n <= 0) continue;
    const uint8_t *from = t.from + row * blocks + 16 * p;
    if (n >= 16 || row + 16 < t.rows) {   // (a row has a byte at least)
      w[q] = reinterpret_cast<const AnyBytes *>(from)->w;
    } else {
      union { uint8_t c[16]; uint4v w; } o;
      o.w = w[q];
#pragma unroll
      for (int e = 0; e < 15; ++e)
        if (e < n) o.c[e] = from[e];
      w[q] = o.w;
    }
  }
#pragma unroll
  for (int q = 0; q < EACH; ++q) {
    const int i = threadIdx.x + q * THREADS, n = blocks - 16 * (p0 + i % 16);
#pragma unroll
    for (int e = 0; e < 4; ++e) {   // (what is behind the row)
      const int left = n - 4 * e;
      w[q][e] &= left >= 4 ? ~0u : (left <= 0 ? 0u : (1u << (8 * left)) - 1);
    }
    part[i / 16][i % 16] = w[q];
  }
  __syncthreads();
  for (int i = threadIdx.x; i < 64 * 16; i += THREADS) {
    const int64_t row = row0 + i % 64;
    const int p = p0 + i / 64;
    if (row < t.rows && p < pieces) *reinterpret_cast<uint4v *>(t.to + (p * t.rows + row) * 16) = part[i % 64][i / 64];
  }
}

int element_of(int dtype) { return dtype == SK_F16 ? EL_F16 : (dtype == SK_BF16 ? EL_BF16 : (dtype == SK_F32 ? EL_F32 : -1)); }
bool misaligned(const void *p, uintptr_t mask) { return (reinterpret_cast<uintptr_t>(p) & mask) != 0; }
// rows and values of a launch: every index counts in 64 bits, blocks in those of a launch
bool fits(int64_t M, int64_t K) { return M > 0 && K > 0 && M <= ((int64_t)1 << 40) && K <= ((int64_t)1 << 31) && M <= ((int64_t)1 << 45) / K; }

}  // namespace

extern "C" int sk_quantize_mxfp4(const void *X, int dtype, int64_t M, int64_t K, int64_t ldx, void *Q, void *scales, void *stream) {
  const int el = element_of(dtype);
  if (el < 0) return SK_ERR_CONFIG;
  if (!X || !Q || !scales) return SK_ERR_NULL;
  if (!fits(M, K) || ldx < K || ldx > ((int64_t)1 << 40)) return SK_ERR_SHAPE;
  const int size = el == EL_F32 ? 4 : 2;
  if (K % 32 || misaligned(X, size - 1) || misaligned(Q, 3)) return SK_ERR_ALIGN;
  const bool vec = !misaligned(X, 15) && (M == 1 || ldx * size % 16 == 0);
  int64_t rows = M, pieces = K / 8;
  if (ldx == K || M == 1) {   // one row
    pieces *= M;
    rows = 1;
  }
  const int64_t blocks = (pieces + THREADS * PIECES - 1) / (THREADS * PIECES);
  const bool past = vec && M * K * size > CACHED;
#define SK_QUANTIZE(EL, VEC, PAST)                                                                                                                \
  hipLaunchKernelGGL((quantize_kernel<EL, VEC, PAST>), wide_grid(rows * blocks), dim3(THREADS), 0, (hipStream_t)stream, (const char *)X, rows, pieces, \
                     ldx * size, blocks, (uint32_t *)Q, (uint8_t *)scales)
#define SK_QUANTIZE_OF(EL)                    \
  if (past) SK_QUANTIZE(EL, true, true);      \
  else if (vec) SK_QUANTIZE(EL, true, false); \
  else SK_QUANTIZE(EL, false, false)
  if (el == EL_F16) {
    SK_QUANTIZE_OF(EL_F16);
  } else if (el == EL_BF16) {
    SK_QUANTIZE_OF(EL_BF16);
  } else {
    SK_QUANTIZE_OF(EL_F32);
  }
#undef SK_QUANTIZE_OF
#undef SK_QUANTIZE
  return hipGetLastError() == hipSuccess ? SK_OK : SK_ERR_LAUNCH;
}

extern "C" int sk_dequantize_mxfp4(const void *Q, const void *scales, int64_t M, int64_t K, int dtype, void *X, void *stream) {
  const int el = element_of(dtype);
  if (el < 0) return SK_ERR_CONFIG;
  if (!X || !Q || !scales) return SK_ERR_NULL;
  if (!fits(M, K)) return SK_ERR_SHAPE;
  if (K % 32 || misaligned(X, el == EL_F32 ? 3 : 1) || misaligned(Q, 3)) return SK_ERR_ALIGN;
  const int64_t bytes = M * K * (el == EL_F32 ? 4 : 2), pieces = bytes / 16;
  const dim3 grid = wide_grid((M * (K / 8) + THREADS * PIECES - 1) / (THREADS * PIECES));
  const bool vec = !misaligned(X, 15), past = vec && bytes > CACHED;
#define SK_DEQUANTIZE(EL, VEC, PAST) \
  hipLaunchKernelGGL((dequantize_kernel<EL, VEC, PAST>), grid, dim3(THREADS), 0, (hipStream_t)stream, (const char *)Q, (const uint8_t *)scales, pieces, (char *)X)
#define SK_DEQUANTIZE_OF(EL)                    \
  if (past) SK_DEQUANTIZE(EL, true, true);      \
  else if (vec) SK_DEQUANTIZE(EL, true, false); \
  else SK_DEQUANTIZE(EL, false, false)
  if (el == EL_F16) {
    SK_DEQUANTIZE_OF(EL_F16);
  } else if (el == EL_BF16) {
    SK_DEQUANTIZE_OF(EL_BF16);
  } else {
    SK_DEQUANTIZE_OF(EL_F32);
  }
#undef SK_DEQUANTIZE_OF
#undef SK_DEQUANTIZE
  return hipGetLastError() == hipSuccess ? SK_OK : SK_ERR_LAUNCH;
}

extern "C" int sk_tile_mx_scales(const void *a, int64_t rows_a, void *tiled_a, const void *b, int64_t rows_b, void *tiled_b, int64_t blocks, void *stream) {
  if (!a || !tiled_a || !b || !tiled_b) return SK_ERR_NULL;
  if (!fits(rows_a, blocks) || !fits(rows_b, blocks) || rows_a > 0x7fffffff || rows_b > 0x7fffffff || blocks > (1 << 24)) return SK_ERR_SHAPE;
  if (misaligned(tiled_a, 15) || misaligned(tiled_b, 15)) return SK_ERR_ALIGN;
  const int64_t blocks_a = (rows_a + 63) / 64, all = blocks_a + (rows_b + 63) / 64;
  const dim3 grid((unsigned)all, (unsigned)((blocks + 255) / 256));
  if (grid.y > 65535) return SK_ERR_SHAPE;
  const TileScales ta{(const uint8_t *)a, (uint8_t *)tiled_a, rows_a}, tb{(const uint8_t *)b, (uint8_t *)tiled_b, rows_b};
  hipLaunchKernelGGL(tile_scales_kernel, grid, dim3(THREADS), 0, (hipStream_t)stream, ta, tb, blocks_a, (int)blocks);
  return hipGetLastError() == hipSuccess ? SK_OK : SK_ERR_LAUNCH;
}
