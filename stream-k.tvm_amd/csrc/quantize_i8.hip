// Row quantiser of 16-bit activations: s = max |x| / 127 of a row in fp32, q = x / s rounded to the nearest integer (ties to even).
//
// One workgroup per row, which it reads once (a thread keeps up to eight pieces of eight values in registers; of rows beyond 16384
// values the rest is read again).  What bounds it is memory, 2 bytes in and 1 out per value, as long as the arithmetic stays at some
// seven instructions a value: 4096 x 8192 23 us, 4.35 TB/s (29 us with a rounding, a clamp and a conversion to each); one row of 4096 2.9.
#include <hip/hip_runtime.h>

#include "sk_device.h"
#include "streamk.h"
#include "wide_grid.h"

using namespace sk;

namespace {

constexpr int THREADS = 256, KEPT = 8;   // pieces of a row that a thread keeps

template <bool BF16>
__device__ __forceinline__ float widen(uint16_t bits) {
  if constexpr (BF16) return __builtin_bit_cast(float, (uint32_t)bits << 16);
  return (float)__builtin_bit_cast(half_t, bits);
}

// x / s to the nearest integer: the product with the reciprocal is at most one off, and the remainder, exact in an fma, says so.
// (Cheaper than the division, and no double rounding where x / s lies next to a tie.)
__device__ __forceinline__ int quantise(float x, float s, float inv) {
  float q = rintf(x * inv);
  const float r = fmaf(-q, s, x), h = 0.5f * s, m = fabsf(r);
  if (m > h || (m == h && ((int)q & 1))) q += copysignf(1.f, r);
  return (int)fminf(fmaxf(q, -127.f), 127.f);
}

// Eight values: x times the reciprocal plus 1.5 * 2^23 in one fma leaves the rounded quotient in the sum's low bits, in two's complement.
// Whether it is the nearest integer the remainder says as in quantise(), which takes over where it is not, or where x / s is a tie.
typedef uint16_t ushort8v __attribute__((ext_vector_type(8)));
template <bool BF16>
__device__ __forceinline__ uint64_t quantise8(ushort8v v, float s, float inv) {
  constexpr float MAGIC = 12582912.f;
  uint32_t t[8];
  const float h = 0.5f * s;
  bool off = false;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float x = widen<BF16>(v[e]), sum = fmaf(x, inv, MAGIC);
    t[e] = __builtin_bit_cast(uint32_t, sum);
    off = off || !(fabsf(fmaf(-(sum - MAGIC), s, x)) < h);
  }
  if (off) {
#pragma unroll
    for (int e = 0; e < 8; ++e) t[e] = (uint32_t)quantise(widen<BF16>(v[e]), s, inv);
  }
  uint32_t w[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint32_t lo = __builtin_amdgcn_perm(t[4 * i + 1], t[4 * i], 0x0c0c0400u), hi = __builtin_amdgcn_perm(t[4 * i + 3], t[4 * i + 2], 0x0c0c0400u);
    w[i] = lo | hi << 16;
  }
  return (uint64_t)w[1] << 32 | w[0];
}

template <bool BF16>
__global__ __launch_bounds__(THREADS) void quantize_i8_kernel(const uint16_t *X, int M, int K, int64_t ldx, int8_t *Q, int64_t ldq,
                                                              float *scales, int vec) {
  const int64_t row = wide_block();
  if (row >= M) return;
  const uint16_t *x = X + row * ldx;
  int8_t *q = Q + row * ldq;
  const int pieces = (K + 7) / 8, tid = threadIdx.x;
  auto load = [&](int p) {
    ushort8v v = {0, 0, 0, 0, 0, 0, 0, 0};
    if (vec) {   // rows of whole aligned pieces
      v = *reinterpret_cast<const ushort8v *>(x + 8 * (int64_t)p);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (8 * p + e < K) v[e] = x[8 * p + e];
    }
    return v;
  };
  // the largest magnitude as bits, of pairs of values: infinities and NaN are above every number
  typedef uint16_t ushort2v __attribute__((ext_vector_type(2)));
  ushort8v kept[KEPT];
  ushort2v pair = {0, 0};
  auto look = [&](ushort8v v) {
#pragma unroll
    for (int e = 0; e < 8; e += 2) pair = __builtin_elementwise_max(pair, ushort2v{(uint16_t)(v[e] & 0x7fff), (uint16_t)(v[e + 1] & 0x7fff)});
  };
#pragma unroll
  for (int i = 0; i < KEPT; ++i) {
    kept[i] = ushort8v{0, 0, 0, 0, 0, 0, 0, 0};
    if (tid + i * THREADS < pieces) kept[i] = load(tid + i * THREADS);
  }
#pragma unroll
  for (int i = 0; i < KEPT; ++i)
    if (i * THREADS < pieces) look(kept[i]);   // (uniform)
  for (int p = tid + KEPT * THREADS; p < pieces; p += THREADS) look(load(p));
  __shared__ uint32_t of_wave[THREADS / 64];
  const uint32_t wave_most = wave_max(max((uint32_t)pair[0], (uint32_t)pair[1]));
  if ((tid & 63) == 0) of_wave[tid >> 6] = wave_most;
  __syncthreads();
  uint32_t most = 0;
#pragma unroll
  for (int w = 0; w < THREADS / 64; ++w) most = max(most, of_wave[w]);

  // a row with an infinity or a NaN has no scale: NaN, so that whatever is made of it is NaN too
  const bool finite = most < (BF16 ? 0x7f80u : 0x7c00u);
  const float s = finite ? widen<BF16>((uint16_t)most) / 127.f : __builtin_nanf("");
  if (tid == 0) scales[row] = s;
  const bool any = s > 0.f, small = s < 1e-37f;   // (the reciprocal of a smaller scale overflows)
  const float inv = any && !small ? 1.f / s : 0.f;
  auto store = [&](int p, ushort8v v) {
    union { int8_t b[8]; uint64_t w; } o;
    o.w = 0;
    if (any && !small) {
      o.w = quantise8<BF16>(v, s, inv);
    } else if (small) {
#pragma unroll
      for (int e = 0; e < 8; ++e) o.b[e] = any ? (int8_t)fminf(fmaxf(rintf(widen<BF16>(v[e]) / s), -127.f), 127.f) : 0;
    }
    if (vec) {
      *reinterpret_cast<uint64_t *>(q + 8 * (int64_t)p) = o.w;
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (8 * p + e < K) q[8 * p + e] = o.b[e];
    }
  };
#pragma unroll
  for (int i = 0; i < KEPT; ++i)
    if (tid + i * THREADS < pieces) store(tid + i * THREADS, kept[i]);
  for (int p = tid + KEPT * THREADS; p < pieces; p += THREADS) store(p, load(p));
}

}  // namespace

extern "C" int sk_quantize_i8(const void *X, int dtype, int64_t M, int64_t K, int64_t ldx, void *Q, int64_t ldq, void *scales, void *stream) {
  if (dtype != SK_F16 && dtype != SK_BF16) return SK_ERR_CONFIG;
  if (!X || !Q || !scales) return SK_ERR_NULL;
  if (M <= 0 || K <= 0 || M > 0x7fffffff || K > 0x7fffff00 || ldx < K || ldq < K) return SK_ERR_SHAPE;
  if ((reinterpret_cast<uintptr_t>(X) & 1) || (reinterpret_cast<uintptr_t>(scales) & 3)) return SK_ERR_ALIGN;
  const int vec = K % 8 == 0 && ldx % 8 == 0 && ldq % 8 == 0 && (reinterpret_cast<uintptr_t>(X) & 15) == 0 && (reinterpret_cast<uintptr_t>(Q) & 7) == 0;
  if (dtype == SK_BF16)
    hipLaunchKernelGGL((quantize_i8_kernel<true>), wide_grid(M), dim3(THREADS), 0, (hipStream_t)stream, (const uint16_t *)X, (int)M, (int)K, ldx,
                       (int8_t *)Q, ldq, (float *)scales, vec);
  else
    hipLaunchKernelGGL((quantize_i8_kernel<false>), wide_grid(M), dim3(THREADS), 0, (hipStream_t)stream, (const uint16_t *)X, (int)M, (int)K, ldx,
                       (int8_t *)Q, ldq, (float *)scales, vec);
  return hipGetLastError() == hipSuccess ? SK_OK : SK_ERR_LAUNCH;
}
