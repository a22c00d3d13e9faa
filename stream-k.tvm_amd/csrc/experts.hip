// What stands before and behind the products of a mixture of experts: the experts of each token, the tokens' rows in the experts'
// order, the experts' rows added up for each token, and the gradients of all three.
//
//   route     the k largest logits of each token (ties: the lower number first; -inf and NaN are never chosen), their softmax
//             w = exp(z - max) / sum, and the T k slots (token t's j-th expert is slot t k + j) sorted by expert, stably:
//             order[p] is the slot of sorted row p (-1 behind the last), place[slot] its row (-1 without an expert)
//   dispatch  rows[p] = x[order[p] / k], zeros where order[p] < 0
//   combine   out[t] = sum_j w[t][j] y[place[t][j]]
// All sums in fp32 and in a fixed order: the same bits on every launch.  Everything but the routing of few tokens is bound by memory.
#include <hip/hip_runtime.h>

#include "sk_device.h"
#include "streamk.h"
#include "wide_grid.h"

using namespace sk;

namespace {

constexpr int MAX_EXPERTS = 1024, MAX_CHOSEN = 64;
enum { EL_F16 = 0, EL_BF16 = 1, EL_F32 = 2 };

template <int EL>
__device__ __forceinline__ float load_el(const void *p, int64_t i) {
  if constexpr (EL == EL_F32) return static_cast<const float *>(p)[i];
  const uint16_t b = static_cast<const uint16_t *>(p)[i];
  if constexpr (EL == EL_BF16) return __builtin_bit_cast(float, (uint32_t)b << 16);
  return (float)__builtin_bit_cast(half_t, b);
}
template <int EL>
__device__ __forceinline__ void store_el(void *p, int64_t i, float x) {
  if constexpr (EL == EL_F32) {
    static_cast<float *>(p)[i] = x;
  } else if constexpr (EL == EL_BF16) {
    static_cast<__bf16 *>(p)[i] = (__bf16)x;
  } else {
    static_cast<half_t *>(p)[i] = (half_t)x;
  }
}

__device__ __forceinline__ float wave_sum(float x) {
#pragma unroll
  for (int d = 32; d > 0; d /= 2) x += __shfl_xor(x, d, 64);
  return x;
}

// logits as unsigned numbers in the same order; 0: not to be chosen
__device__ __forceinline__ uint32_t order_key(float z) {
  z += 0.f;   // (-0 is 0)
  const uint32_t b = __builtin_bit_cast(uint32_t, z);
  if (!(z > -__builtin_inff())) return 0;
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}

// The k experts of token t by one wave: S x 64 logits, S in each lane.  Lane j < k returns the j-th expert (-1: none) and weight.
template <int EL, int S>
__device__ __forceinline__ void choose(const void *logits, int64_t ld, int t, int E, int k, int &expert, float &weight) {
  const int lane = threadIdx.x & 63;
  uint32_t key[S];
#pragma unroll
  for (int s = 0; s < S; ++s) key[s] = 64 * s + lane < E ? order_key(load_el<EL>(logits, t * ld + 64 * s + lane)) : 0;
  expert = -1;
  uint32_t mine = 0, first = 0;
  for (int j = 0; j < k; ++j) {
    uint32_t best = key[0];
#pragma unroll
    for (int s = 1; s < S; ++s) best = max(best, key[s]);
    best = wave_max(best);
    if (best == 0) break;
    if (j == 0) first = best;
    bool found = false;
#pragma unroll
    for (int s = 0; s < S; ++s) {   // the lowest number with it
      const uint64_t at = __builtin_amdgcn_ballot_w64(key[s] == best);
      if (!found && at != 0) {
        found = true;
        const int l = __builtin_ctzll(at);
        if (lane == l) key[s] = 0;
        if (lane == j) {
          expert = 64 * s + l;
          mine = best;
        }
      }
    }
  }
  auto value = [](uint32_t b) { return __builtin_bit_cast(float, b & 0x80000000u ? b ^ 0x80000000u : ~b); };
  // (a logit of +inf: the differences of such a token are NaN, as the softmax's)
  const float e = expert >= 0 ? expf(value(mine) - value(first)) : 0.f;
  const float sum = wave_sum(e);
  weight = expert >= 0 ? e / sum : 0.f;
}

struct RouteArgs {
  const void *logits;
  int64_t ld;
  int T, E, k;
  float *weights;                          // [T, k]
  int *experts, *offsets, *order, *place;  // [T, k], [E + 1], [T k], [T k]
  int *counts;                             // [blocks, E]: slots of a block's tokens by expert
  int tokens;                              // of a block
};

// The slots of a range, in order, 64 at a time by each of the block's waves, which own consecutive parts of it: start[e] + slots with
// expert e in front.  have: LDS, [waves][E] counts of the waves' parts, replaced by where their rows go.
template <int WAVES>
__device__ __forceinline__ void place_slots(const RouteArgs &a, const int *experts, int slot0, int n, int *have) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int part = (n + 64 * WAVES - 1) / (64 * WAVES) * 64, from = wave * part, to = min(n, from + part);
  int *mine = have + wave * a.E;
  int bits = 1;
  while ((1 << bits) < a.E + 1) ++bits;
  for (int i0 = from; i0 < to; i0 += 64) {
    const int i = i0 + lane;
    const int e = i < to ? experts[i] : -1;
    uint64_t same = __builtin_amdgcn_ballot_w64(e >= 0);
    for (int b = 0; b < bits; ++b) {
      const uint64_t set = __builtin_amdgcn_ballot_w64(((e >> b) & 1) != 0);
      same &= (e >> b) & 1 ? set : ~set;
    }
    if (i < to) {
      int p = -1;
      if (e >= 0) {
        const int rank = __builtin_popcountll(same & ((1ull << lane) - 1));
        p = mine[e] + rank;
        a.order[p] = slot0 + i;
      }
      a.place[slot0 + i] = p;
    }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    // (the first lane of an expert counts its rows; every lane has read the count it needs)
    if (e >= 0 && (same & ((1ull << lane) - 1)) == 0) mine[e] += __builtin_popcountll(same);
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
  }
}
// slots of the waves' parts by expert, into have[waves][E] (LDS atomics: counts, whose order does not matter)
template <int WAVES>
__device__ __forceinline__ void count_parts(const int *experts, int n, int E, int *have) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int part = (n + 64 * WAVES - 1) / (64 * WAVES) * 64, from = wave * part, to = min(n, from + part);
  for (int i = threadIdx.x; i < WAVES * E; i += 64 * WAVES) have[i] = 0;
  __syncthreads();
  for (int i = from + lane; i < to; i += 64)
    if (experts[i] >= 0) atomicAdd(&have[wave * E + experts[i]], 1);
  __syncthreads();
}
// exclusive sums over the experts of total[E] (LDS), by the first wave; returns the sum of all in every thread
__device__ __forceinline__ int scan_experts(int *total, int E, int *word) {
  if (threadIdx.x < 64) {
    const int lane = threadIdx.x;
    int before = 0;
    for (int e0 = 0; e0 < E; e0 += 64) {
      const int own = e0 + lane < E ? total[e0 + lane] : 0;
      int x = own;
#pragma unroll
      for (int d = 1; d < 64; d *= 2) {
        const int y = __shfl_up(x, d, 64);
        if (lane >= d) x += y;
      }
      if (e0 + lane < E) total[e0 + lane] = before + x - own;
      before += __builtin_amdgcn_readlane(x, 63);
    }
    if (lane == 0) *word = before;
  }
  __syncthreads();
  return *word;
}

constexpr int FEW_TOKENS = 64, FEW_EXPERTS = 256, FEW_WAVES = 16;   // one workgroup does it all
// (two launches take about 4 us more than one; 64 tokens are four for each wave of the workgroup)

template <int EL, int S>
__global__ __launch_bounds__(64 * FEW_WAVES) void route_few_kernel(RouteArgs a) {
  extern __shared__ int lds[];
  int *experts = lds, *have = lds + FEW_TOKENS * a.k, *total = have + FEW_WAVES * a.E, *word = total + a.E;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, n = a.T * a.k;
  for (int t = wave; t < a.T; t += FEW_WAVES) {
    int e;
    float w;
    choose<EL, S>(a.logits, a.ld, t, a.E, a.k, e, w);
    if (lane < a.k) {
      experts[t * a.k + lane] = e;
      a.experts[t * a.k + lane] = e;
      a.weights[t * a.k + lane] = w;
    }
  }
  __syncthreads();
  count_parts<FEW_WAVES>(experts, n, a.E, have);
  for (int e = threadIdx.x; e < a.E; e += 64 * FEW_WAVES) {
    int sum = 0;
    for (int w = 0; w < FEW_WAVES; ++w) sum += have[w * a.E + e];
    total[e] = sum;
  }
  __syncthreads();
  const int used = scan_experts(total, a.E, word);
  for (int e = threadIdx.x; e < a.E; e += 64 * FEW_WAVES) {
    int at = total[e];
    a.offsets[e] = at;
    for (int w = 0; w < FEW_WAVES; ++w) {
      const int c = have[w * a.E + e];
      have[w * a.E + e] = at;
      at += c;
    }
  }
  if (threadIdx.x == 0) a.offsets[a.E] = used;
  for (int p = used + threadIdx.x; p < n; p += 64 * FEW_WAVES) a.order[p] = -1;
  __syncthreads();
  place_slots<FEW_WAVES>(a, experts, 0, n, have);
}

// More tokens: choice and counts by blocks, then places.  8192 tokens, 8 of 64 experts: 4 and 9 us (four waves a block for the choice 28 us:
// a token is a chain of k reductions).
constexpr int WAVES = 4, CHOOSE_WAVES = 16;
template <int EL, int S>
__global__ __launch_bounds__(64 * CHOOSE_WAVES) void route_choose_kernel(RouteArgs a) {
  extern __shared__ int lds[];   // [E] counts of the block
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, t0 = blockIdx.x * a.tokens, t1 = min(a.T, t0 + a.tokens);
  for (int e = threadIdx.x; e < a.E; e += 64 * CHOOSE_WAVES) lds[e] = 0;
  __syncthreads();
  for (int t = t0 + wave; t < t1; t += CHOOSE_WAVES) {
    int e;
    float w;
    choose<EL, S>(a.logits, a.ld, t, a.E, a.k, e, w);
    if (lane < a.k) {
      a.experts[(int64_t)t * a.k + lane] = e;
      a.weights[(int64_t)t * a.k + lane] = w;
      if (e >= 0) atomicAdd(&lds[e], 1);
    }
  }
  __syncthreads();
  for (int e = threadIdx.x; e < a.E; e += 64 * CHOOSE_WAVES) a.counts[(int64_t)blockIdx.x * a.E + e] = lds[e];
}
// every block adds up the counts of all blocks, and of those in front of it, by itself
__global__ __launch_bounds__(64 * WAVES) void route_place_kernel(RouteArgs a) {
  extern __shared__ int lds[];
  int *have = lds, *total = have + WAVES * a.E, *front = total + a.E, *word = front + a.E;
  const int t0 = blockIdx.x * a.tokens, t1 = min(a.T, t0 + a.tokens), slot0 = t0 * a.k, n = (t1 - t0) * a.k;
  const int *experts = a.experts + slot0;
  for (int e = threadIdx.x; e < a.E; e += 64 * WAVES) total[e] = front[e] = 0;
  __syncthreads();
  // (SHARE threads to an expert, eight counts in flight each)
  constexpr int SHARE = 16;
  for (int i = threadIdx.x; i < SHARE * a.E; i += 64 * WAVES) {
    const int e = (int)((unsigned)i % (unsigned)a.E), share = (int)((unsigned)i / (unsigned)a.E), blocks = (int)gridDim.x;
    int sum = 0, before = 0;
    for (int b0 = share; b0 < blocks; b0 += 8 * SHARE) {
      int c[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) c[j] = b0 + j * SHARE < blocks ? a.counts[(int64_t)(b0 + j * SHARE) * a.E + e] : 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        sum += c[j];
        before += b0 + j * SHARE < (int)blockIdx.x ? c[j] : 0;
      }
    }
    atomicAdd(&total[e], sum);
    atomicAdd(&front[e], before);
  }
  __syncthreads();
  count_parts<WAVES>(experts, n, a.E, have);
  const int used = scan_experts(total, a.E, word);
  for (int e = threadIdx.x; e < a.E; e += 64 * WAVES) {
    int at = total[e] + front[e];
    if (blockIdx.x == 0) a.offsets[e] = total[e];
    for (int w = 0; w < WAVES; ++w) {
      const int c = have[w * a.E + e];
      have[w * a.E + e] = at;
      at += c;
    }
  }
  if (blockIdx.x == 0 && threadIdx.x == 0) a.offsets[a.E] = used;
  for (int p = used + blockIdx.x * 64 * WAVES + threadIdx.x; p < a.T * a.k; p += gridDim.x * 64 * WAVES) a.order[p] = -1;
  __syncthreads();
  place_slots<WAVES>(a, experts, slot0, n, have);
}

constexpr int MOST_BLOCKS = 256;   // (each of which reads all blocks' counts)
int route_tokens(int64_t T) {
  int64_t tokens = (T + MOST_BLOCKS - 1) / MOST_BLOCKS;
  if (tokens < 16) tokens = 16;
  return (int)tokens;
}
int route_blocks(int64_t T, int64_t E) {
  return T <= FEW_TOKENS && E <= FEW_EXPERTS ? 0 : (int)((T + route_tokens(T) - 1) / route_tokens(T));
}

template <int EL, int S>
int launch_route(const RouteArgs &a, int blocks, hipStream_t s) {
  if (blocks == 0) {
    const size_t lds = sizeof(int) * (FEW_TOKENS * a.k + (FEW_WAVES + 1) * a.E + 1);
    hipLaunchKernelGGL((route_few_kernel<EL, S>), dim3(1), dim3(64 * FEW_WAVES), lds, s, a);
    return (int)hipGetLastError();
  }
  hipLaunchKernelGGL((route_choose_kernel<EL, S>), dim3(blocks), dim3(64 * CHOOSE_WAVES), sizeof(int) * a.E, s, a);
  if (hipGetLastError() != hipSuccess) return 1;
  hipLaunchKernelGGL(route_place_kernel, dim3(blocks), dim3(64 * WAVES), sizeof(int) * ((WAVES + 2) * a.E + 1), s, a);
  return (int)hipGetLastError();
}
template <int EL>
int launch_route_of(const RouteArgs &a, int blocks, hipStream_t s) {
  if (a.E <= 64) return launch_route<EL, 1>(a, blocks, s);
  if (a.E <= 128) return launch_route<EL, 2>(a, blocks, s);
  if (a.E <= 256) return launch_route<EL, 4>(a, blocks, s);
  return launch_route<EL, 16>(a, blocks, s);
}

// d logits[t][e_j] = w_j (dw_j - sum_i w_i dw_i); one wave per token (8192 tokens, 64 experts: 5 us)
template <int EL>
__global__ __launch_bounds__(64 * WAVES) void route_backward_kernel(const float *weights, const int *experts, const float *dweights, int T,
                                                                    int E, int k, void *dlogits) {
  extern __shared__ float row_lds[];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t t = wide_block() * WAVES + wave;
  float *row = row_lds + wave * E;
  if (t < T) {
    for (int e = lane; e < E; e += 64) row[e] = 0.f;
    const float w = lane < k ? weights[t * k + lane] : 0.f, dw = lane < k ? dweights[t * k + lane] : 0.f;
    const int e = lane < k ? experts[t * k + lane] : -1;
    const float sum = wave_sum(e >= 0 ? w * dw : 0.f);
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    if (e >= 0 && e < E) row[e] = w * (dw - sum);
  }
  __syncthreads();
  if (t < T)
    for (int e = lane; e < E; e += 64) store_el<EL>(dlogits, t * E + e, row[e]);
}

// rows[p] = x[order[p] / k]: one wave per row, pieces of UNIT bytes
template <class Unit>
__global__ __launch_bounds__(64 * WAVES) void dispatch_kernel(const Unit *x, int64_t ldx, const int *order, int T, int k, int64_t rows, int units,
                                                              Unit *out) {
  const int lane = threadIdx.x & 63;
  const int64_t p = wide_block() * WAVES + (threadIdx.x >> 6);
  if (p >= rows) return;
  const int slot = order[p], t = slot >= 0 ? (int)((unsigned)slot / (unsigned)k) : -1;
  Unit *dst = out + p * units;
  if (t < 0 || t >= T) {
    for (int i = lane; i < units; i += 64) dst[i] = Unit{};
    return;
  }
  const Unit *src = x + t * ldx;
  int i = lane;
  for (; i + 192 < units; i += 256) {
    const Unit u0 = src[i], u1 = src[i + 64], u2 = src[i + 128], u3 = src[i + 192];
    dst[i] = u0;
    dst[i + 64] = u1;
    dst[i + 128] = u2;
    dst[i + 192] = u3;
  }
  for (; i < units; i += 64) dst[i] = src[i];
}

// The same by tokens: one wave reads a token's row once and stores it to each of its places; the waves also clear the rows without a
// slot.  8192 tokens of 4 KB to 65536 rows: 47 us (6.4 TB/s), by rows 71.
template <class Unit>
__global__ __launch_bounds__(64 * WAVES) void dispatch_tokens_kernel(const Unit *x, int64_t ldx, const int *order, const int *place, int T, int k,
                                                                     int units, Unit *out) {
  const int lane = threadIdx.x & 63;
  const int64_t t = wide_block() * WAVES + __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), rows = (int64_t)T * k;
  if (t >= T) return;
  const Unit *src = x + t * ldx;
  const int mine = lane < k ? place[t * k + lane] : -1, at = lane < k ? order[t * k + lane] : 0;   // (k <= 64)
  for (int i0 = 0; i0 < units; i0 += 256) {
    Unit u[4];
#pragma unroll
    for (int q = 0; q < 4; ++q)
      if (i0 + 64 * q + lane < units) u[q] = src[i0 + 64 * q + lane];
    for (int j = 0; j < k; ++j) {
      const int p = __builtin_amdgcn_readlane(mine, j);
      if (p >= 0 && p < rows) {
        Unit *dst = out + (int64_t)p * units + i0 + lane;
#pragma unroll
        for (int q = 0; q < 4; ++q)
          if (i0 + 64 * q + lane < units) dst[64 * q] = u[q];
      }
      if (__builtin_amdgcn_readlane(at, j) < 0) {
        Unit *dst = out + (t * k + j) * units + i0 + lane;
#pragma unroll
        for (int q = 0; q < 4; ++q)
          if (i0 + 64 * q + lane < units) dst[64 * q] = Unit{};
      }
    }
  }
}

typedef uint16_t ushort8v __attribute__((ext_vector_type(8)));
template <bool BF16>
__device__ __forceinline__ float widen(uint16_t bits) {
  if constexpr (BF16) return __builtin_bit_cast(float, (uint32_t)bits << 16);
  return (float)__builtin_bit_cast(half_t, bits);
}
template <bool BF16>
__device__ __forceinline__ uint16_t narrow(float x) {
  if constexpr (BF16) return __builtin_bit_cast(uint16_t, (__bf16)x);
  return __builtin_bit_cast(uint16_t, (half_t)x);
}
// eight values from column c on (zeros past H)
template <bool VEC>
__device__ __forceinline__ ushort8v load8(const uint16_t *row, int c, int H) {
  if constexpr (VEC) return *reinterpret_cast<const ushort8v *>(row + c);
  ushort8v v = {0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
  for (int e = 0; e < 8; ++e)
    if (c + e < H) v[e] = row[c + e];
  return v;
}
template <bool VEC>
__device__ __forceinline__ void store8(uint16_t *row, int c, int H, ushort8v v) {
  if constexpr (VEC) {
    *reinterpret_cast<ushort8v *>(row + c) = v;
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (c + e < H) row[c + e] = v[e];
  }
}

// out[t] = sum_j w[t][j] y[place[t][j]] (weights null: 1), j ascending; a wave takes 512 columns of a token, a thread eight.  8192 tokens,
// 8 rows of 4 KB each: 57 us, 5.3 TB/s (rows in the tokens' order 54).
template <bool BF16, bool VEC>
__global__ __launch_bounds__(64 * WAVES) void combine_kernel(const uint16_t *y, const int *place, const float *weights, int k, int H, int64_t T,
                                                             uint16_t *out, int pieces) {
  const int64_t item = wide_block() * WAVES + __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), t = item / pieces, rows = T * k;
  if (t >= T) return;
  const int c = ((int)(item - t * pieces) * 64 + (threadIdx.x & 63)) * 8;
  if (c < H) {
    float sum[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    // eight rows in flight; a slot without an expert reads row 0, whose values are not used
    for (int j0 = 0; j0 < k; j0 += 8) {
      ushort8v v[8];
      float w[8];
      bool used[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int p = j0 + j < k ? place[t * k + j0 + j] : -1;   // (uniform)
        used[j] = p >= 0 && p < rows;
        w[j] = used[j] && weights ? weights[t * k + j0 + j] : 1.f;
        if (j0 + j < k) v[j] = load8<VEC>(y + (int64_t)(used[j] ? p : 0) * H, c, H);
      }
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (used[j]) {
#pragma unroll
          for (int e = 0; e < 8; ++e) sum[e] = fmaf(w[j], widen<BF16>(v[j][e]), sum[e]);
        }
    }
    ushort8v o;
#pragma unroll
    for (int e = 0; e < 8; ++e) o[e] = narrow<BF16>(sum[e]);
    store8<VEC>(out + t * H, c, H, o);
  }
}

// dy[p] = w d_out[t], dw[slot] = <d_out[t], y[p]> for the slot of p; one wave per slot.  Row number `slot` without a slot: zeros.
// 8192 tokens, 8 rows of 4 KB each: 98 us, 5.8 TB/s.
template <bool BF16, bool VEC>
__global__ __launch_bounds__(64 * WAVES) void combine_backward_kernel(const uint16_t *d_out, const uint16_t *y, const int *order, const int *place,
                                                                      const float *weights, int k, int H, int64_t rows, uint16_t *dy, float *dw) {
  const int lane = threadIdx.x & 63;
  const int64_t slot = wide_block() * WAVES + (threadIdx.x >> 6);
  if (slot >= rows) return;
  if (order[slot] < 0)
    for (int c = lane * 8; c < H; c += 512) store8<VEC>(dy + slot * H, c, H, ushort8v{0, 0, 0, 0, 0, 0, 0, 0});
  const int p = place[slot];
  if (p < 0 || p >= rows) {
    if (lane == 0) dw[slot] = 0.f;
    return;
  }
  const float w = weights[slot];
  const uint16_t *g = d_out + slot / k * H, *row = y + (int64_t)p * H;
  float dot = 0.f;
  for (int c = lane * 8; c < H; c += 512) {
    const ushort8v a = load8<VEC>(g, c, H), b = load8<VEC>(row, c, H);
    ushort8v o;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float x = widen<BF16>(a[e]);
      dot = fmaf(x, widen<BF16>(b[e]), dot);
      o[e] = narrow<BF16>(w * x);
    }
    store8<VEC>(dy + (int64_t)p * H, c, H, o);
  }
  dot = wave_sum(dot);
  if (lane == 0) dw[slot] = dot;
}

bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
int check_route_shape(int64_t T, int64_t E, int64_t k) {
  return T > 0 && E > 0 && E <= MAX_EXPERTS && k > 0 && k <= E && k <= MAX_CHOSEN && T * k <= 0x7fffffff / 2 ? SK_OK : SK_ERR_SHAPE;
}
int element_of(int dtype) { return dtype == SK_F16 ? EL_F16 : (dtype == SK_BF16 ? EL_BF16 : (dtype == SK_F32 ? EL_F32 : -1)); }
int launched() { return hipGetLastError() == hipSuccess ? SK_OK : SK_ERR_LAUNCH; }

}  // namespace

extern "C" size_t sk_route_workspace_bytes(int64_t T, int64_t E, int64_t k) {
  return check_route_shape(T, E, k) == SK_OK ? sizeof(int) * (size_t)route_blocks(T, E) * (size_t)E : 0;
}

extern "C" int sk_route_experts(const void *logits, int dtype, int64_t T, int64_t E, int64_t k, int64_t ld, void *weights, void *experts,
                                void *offsets, void *order, void *place, void *ws, size_t ws_bytes, void *stream) {
  if (element_of(dtype) < 0) return SK_ERR_CONFIG;
  if (int rc = check_route_shape(T, E, k)) return rc;
  if (!logits || !weights || !experts || !offsets || !order || !place) return SK_ERR_NULL;
  if (ld < E) return SK_ERR_SHAPE;
  const int blocks = route_blocks(T, E);
  if (ws_bytes < sk_route_workspace_bytes(T, E, k) || (blocks > 0 && !ws)) return SK_ERR_WORKSPACE;
  if (reinterpret_cast<uintptr_t>(ws) & 3) return SK_ERR_ALIGN;
  RouteArgs a{logits, ld, (int)T, (int)E, (int)k, (float *)weights, (int *)experts, (int *)offsets, (int *)order, (int *)place, (int *)ws,
              route_tokens(T)};
  hipStream_t s = (hipStream_t)stream;
  const int el = element_of(dtype);
  const int herr = el == EL_F16 ? launch_route_of<EL_F16>(a, blocks, s) : (el == EL_BF16 ? launch_route_of<EL_BF16>(a, blocks, s) : launch_route_of<EL_F32>(a, blocks, s));
  return herr == 0 ? SK_OK : SK_ERR_LAUNCH;
}

extern "C" int sk_route_backward(const void *weights, const void *experts, const void *dweights, int64_t T, int64_t E, int64_t k, int dtype,
                                 void *dlogits, void *stream) {
  if (element_of(dtype) < 0) return SK_ERR_CONFIG;
  if (int rc = check_route_shape(T, E, k)) return rc;
  if (!weights || !experts || !dweights || !dlogits) return SK_ERR_NULL;
  const dim3 grid = wide_grid((T + WAVES - 1) / WAVES), block(64 * WAVES);
  const size_t lds = sizeof(float) * WAVES * E;
#define SK_ROUTE_BACKWARD(EL)                                                                                                            \
  hipLaunchKernelGGL((route_backward_kernel<EL>), grid, block, lds, (hipStream_t)stream, (const float *)weights, (const int *)experts,    \
                     (const float *)dweights, (int)T, (int)E, (int)k, dlogits)
  if (dtype == SK_F16) SK_ROUTE_BACKWARD(EL_F16);
  else if (dtype == SK_BF16) SK_ROUTE_BACKWARD(EL_BF16);
  else SK_ROUTE_BACKWARD(EL_F32);
#undef SK_ROUTE_BACKWARD
  return launched();
}

extern "C" int sk_dispatch_rows(const void *x, int64_t row_bytes, int64_t x_pitch, const void *order, const void *place, int64_t T, int64_t k, void *rows,
                                void *stream) {
  if (!x || !order || !rows) return SK_ERR_NULL;
  if (T <= 0 || k <= 0 || T * k > 0x7fffffff / 2 || row_bytes <= 0 || row_bytes > 0x7fffffff || x_pitch < row_bytes) return SK_ERR_SHAPE;
  const int64_t n = T * k;
  const dim3 grid = wide_grid((n + WAVES - 1) / WAVES), block(64 * WAVES);
  const uint64_t all = reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(rows) | (uint64_t)row_bytes | (uint64_t)x_pitch;
  // (many tokens: fewer waves than rows fill the device)
  const bool by_tokens = place && k <= MAX_CHOSEN && T >= 2048;
  const dim3 tokens_grid = wide_grid((T + WAVES - 1) / WAVES);
#define SK_DISPATCH(UNIT)                                                                                                            \
  if (by_tokens)                                                                                                                     \
    hipLaunchKernelGGL((dispatch_tokens_kernel<UNIT>), tokens_grid, block, 0, (hipStream_t)stream, (const UNIT *)x,                   \
                       x_pitch / (int64_t)sizeof(UNIT), (const int *)order, (const int *)place, (int)T, (int)k,                       \
                       (int)(row_bytes / (int64_t)sizeof(UNIT)), (UNIT *)rows);                                                       \
  else                                                                                                                               \
    hipLaunchKernelGGL((dispatch_kernel<UNIT>), grid, block, 0, (hipStream_t)stream, (const UNIT *)x, x_pitch / (int64_t)sizeof(UNIT), \
                       (const int *)order, (int)T, (int)k, n, (int)(row_bytes / (int64_t)sizeof(UNIT)), (UNIT *)rows)
  if (all % 16 == 0) {
    SK_DISPATCH(uint4v);
  } else if (all % 4 == 0) {
    SK_DISPATCH(uint32_t);
  } else {
    SK_DISPATCH(uint8_t);
  }
#undef SK_DISPATCH
  return launched();
}

extern "C" int sk_combine_rows(const void *y, int dtype, const void *place, const void *weights, int64_t T, int64_t k, int64_t H, void *out,
                               void *stream) {
  if (dtype != SK_F16 && dtype != SK_BF16) return SK_ERR_CONFIG;
  if (!y || !place || !out) return SK_ERR_NULL;
  if (T <= 0 || k <= 0 || H <= 0 || T * k > 0x7fffffff / 2 || H > 0x7fffff00) return SK_ERR_SHAPE;
  const int pieces = (int)((H + 511) / 512);
  const int64_t blocks = (T * pieces + WAVES - 1) / WAVES;
  if (blocks > 0x7fffffff) return SK_ERR_SHAPE;
  const bool vec = H % 8 == 0 && aligned16(y) && aligned16(out);
#define SK_COMBINE(BF, VEC)                                                                                                            \
  hipLaunchKernelGGL((combine_kernel<BF, VEC>), wide_grid(blocks), dim3(64 * WAVES), 0, (hipStream_t)stream, (const uint16_t *)y,   \
                     (const int *)place, (const float *)weights, (int)k, (int)H, T, (uint16_t *)out, pieces)
  if (dtype == SK_BF16) {
    if (vec) SK_COMBINE(true, true);
    else SK_COMBINE(true, false);
  } else {
    if (vec) SK_COMBINE(false, true);
    else SK_COMBINE(false, false);
  }
#undef SK_COMBINE
  return launched();
}

extern "C" int sk_combine_backward(const void *d_out, const void *y, int dtype, const void *order, const void *place, const void *weights, int64_t T,
                                   int64_t k, int64_t H, void *dy, void *dweights, void *stream) {
  if (dtype != SK_F16 && dtype != SK_BF16) return SK_ERR_CONFIG;
  if (!d_out || !y || !order || !place || !weights || !dy || !dweights) return SK_ERR_NULL;
  if (T <= 0 || k <= 0 || H <= 0 || T * k > 0x7fffffff / 2 || H > 0x7fffff00) return SK_ERR_SHAPE;
  const bool vec = H % 8 == 0 && aligned16(d_out) && aligned16(y) && aligned16(dy);
  const dim3 grid = wide_grid((T * k + WAVES - 1) / WAVES), block(64 * WAVES);
#define SK_COMBINE_BACKWARD(BF, VEC)                                                                                                  \
  hipLaunchKernelGGL((combine_backward_kernel<BF, VEC>), grid, block, 0, (hipStream_t)stream, (const uint16_t *)d_out, (const uint16_t *)y, \
                     (const int *)order, (const int *)place, (const float *)weights, (int)k, (int)H, T * k, (uint16_t *)dy, (float *)dweights)
  if (dtype == SK_BF16) {
    if (vec) SK_COMBINE_BACKWARD(true, true);
    else SK_COMBINE_BACKWARD(true, false);
  } else {
    if (vec) SK_COMBINE_BACKWARD(false, true);
    else SK_COMBINE_BACKWARD(false, false);
  }
#undef SK_COMBINE_BACKWARD
  return launched();
}
