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

constexpr int MAX_EXPERTS = 1024, MAX_CHOSEN = 64, MAX_GROUPS = 64;
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

// ---- scores, a bias for balance, groups ----
//   s = sigmoid(z), or softmax(z) over all experts;  c = s + bias
//   of `groups` equal groups of experts, neighbours in number, the chosen_groups with the largest sum of their two largest c stay open;
//   the k largest c among the open (without a bias: the k largest z, in whose order the scores are), ties to the lower number;
//   weights = s of the chosen, divided by their sum if renormalised, times a factor.
// Two experts' c may differ by less than 32 bits tell, and the choice is a whole number that two programs should agree on: scores, sums and
// comparisons are in 64 bits.  What bounds the kernel is its instructions, about a thousand to a token of 256 experts: some seventy for each
// logit of a lane, fifty for each of the k, a hundred for the groups, which are all compared at once.  (One after the other, two
// reductions over the wave to each: 16 tokens, 8 of 256 experts in 4 of 8 groups 18 us, so 13; 8192 tokens 71 us, with that and the scan of
// counts below 28.)
struct Scores {
  const float *bias;   // [E] or null
  double scale;
  int groups, chosen_groups, size, lanes;   // size: of a group; lanes: that hold it (set by the launch)
  bool sigmoid, renormalize;
};

// doubles as unsigned numbers in the same order; 0: not to be chosen
__device__ __forceinline__ uint64_t order_key64(double c) {
  c += 0.;
  const uint64_t b = __builtin_bit_cast(uint64_t, c);
  if (!(c > -__builtin_inf())) return 0;
  return b >> 63 ? ~b : b | 1ull << 63;
}
__device__ __forceinline__ double read_lane(double x, int lane) {   // (lane: uniform)
  const uint64_t b = __builtin_bit_cast(uint64_t, x);
  const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)b, lane), hi = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(b >> 32), lane);
  return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
// (no NaN comes here: the builtins make sure of a signalling one's result first, two more instructions each)
__device__ __forceinline__ double larger(double a, double b) {
  double r;
  asm("v_max_f64 %0, %1, %2" : "=v"(r) : "v"(a), "v"(b));
  return r;
}
__device__ __forceinline__ double smaller(double a, double b) {
  double r;
  asm("v_min_f64 %0, %1, %2" : "=v"(r) : "v"(a), "v"(b));
  return r;
}
// (the order of wave_max_up_to: within rows of 16 lanes, then from row to row)
__device__ __forceinline__ double wave_sum(double x) {
#define SK_SUM_STEP(CTRL, ROWS)                                                                                        \
  {                                                                                                                    \
    const uint64_t b = __builtin_bit_cast(uint64_t, x);                                                                \
    const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)b, CTRL, ROWS, 0xf, false);            \
    const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(b >> 32), CTRL, ROWS, 0xf, false);    \
    x += __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);                                                          \
  }
  SK_SUM_STEP(0x111, 0xf);
  SK_SUM_STEP(0x112, 0xf);
  SK_SUM_STEP(0x114, 0xf);
  SK_SUM_STEP(0x118, 0xf);
  SK_SUM_STEP(0x142, 0xa);
  SK_SUM_STEP(0x143, 0xc);
#undef SK_SUM_STEP
  return read_lane(x, 63);
}
// the largest of all lanes, and the first lane that has it: most often the upper halves tell
__device__ __forceinline__ uint64_t wave_max64(uint64_t x, int &lane) {
  const uint32_t hi = (uint32_t)(x >> 32), top = wave_max(hi);
  uint64_t at = __builtin_amdgcn_ballot_w64(hi == top);
  uint32_t low = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)x, __builtin_ctzll(at));
  if (at & (at - 1)) {   // (uniform)
    low = wave_max(hi == top ? (uint32_t)x : 0);
    at = __builtin_amdgcn_ballot_w64(hi == top && (uint32_t)x == low);
  }
  lane = __builtin_ctzll(at);
  return (uint64_t)top << 32 | low;
}
__device__ __forceinline__ double sigmoid64(double z) { return 1. / (1. + exp(-z)); }
// e^(z - m); infinities of both as the limit
__device__ __forceinline__ double exp_from(double z, double m) { return z == m ? 1. : exp(z - m); }

// The weights of the lanes' chosen experts, whose logits are z (expert < 0: none); most, sum: of all experts (softmax not renormalised).
// share: before the factor.
__device__ __forceinline__ double chosen_share(const Scores &p, int expert, float z, double most, double sum) {
  if (!p.renormalize) return expert < 0 ? 0. : (p.sigmoid ? sigmoid64(z) : exp_from(z, most) / sum);
  // scores that underflow have quotients all the same: sigmoid(z) = e^(z - m) / (1 + e^z) times e^m
  const uint32_t top = wave_max(expert < 0 ? 0 : order_key(z));
  const double m = __builtin_bit_cast(float, top & 0x80000000u ? top ^ 0x80000000u : ~top);
  double s = 0.;
  if (expert >= 0) s = p.sigmoid ? (m < -600. ? exp_from(z, m) / (1. + exp((double)z)) : sigmoid64(z)) : exp_from(z, m);
  const double all = wave_sum(s);
  return expert < 0 ? 0. : s / all;
}

// The experts that a lane holds: S neighbours, of one group; a group has `lanes` lanes, neighbours too, so that the first of the lanes with
// a score has the lowest number.
struct Span {
  int first, n, group, in_group;   // (in_group: number of the lane among its group's)
  __device__ __forceinline__ Span(const Scores &p, int S) {
    const int lane = threadIdx.x & 63;
    group = (int)((unsigned)lane / (unsigned)p.lanes);
    in_group = lane - group * p.lanes;
    first = group * p.size + in_group * S;
    n = group < p.groups ? min(S, p.size - in_group * S) : 0;
  }
};
// As choose(), by scores.
template <int EL, int S>
__device__ __forceinline__ void choose_scored(const void *logits, int64_t ld, int t, int k, const Scores &p, const Span &own, int &expert, float &weight) {
  constexpr double NONE = -__builtin_inf();
  const int lane = threadIdx.x & 63;
  float z[S];
  bool there[S];
#pragma unroll
  for (int s = 0; s < S; ++s) {
    z[s] = s < own.n ? load_el<EL>(logits, t * ld + own.first + s) : -__builtin_inff();
    there[s] = z[s] > -__builtin_inff();   // (neither -inf nor NaN)
  }
  double most = 0., sum = 1.;
  if (!p.sigmoid && (p.bias || p.groups > 1 || !p.renormalize)) {
    uint32_t top = 0;
#pragma unroll
    for (int s = 0; s < S; ++s) top = max(top, order_key(z[s]));
    top = wave_max(top);
    most = __builtin_bit_cast(float, top & 0x80000000u ? top ^ 0x80000000u : ~top);
    double part = 0.;
#pragma unroll
    for (int s = 0; s < S; ++s) part += there[s] ? exp_from(z[s], most) : 0.;
    sum = wave_sum(part);
  }
  double c[S];
#pragma unroll
  for (int s = 0; s < S; ++s) c[s] = (double)z[s];
  if (p.bias || p.groups > 1) {   // (uniform)
#pragma unroll
    for (int s = 0; s < S; ++s) {
      c[s] = p.sigmoid ? sigmoid64(z[s]) : exp_from(z[s], most) / sum;
      if (p.bias && there[s]) c[s] += (double)p.bias[own.first + s];
      there[s] = there[s] && c[s] > NONE;
    }
  }
  bool open = true;
  if (p.groups > 1) {
    double first = NONE, second = NONE;
#pragma unroll
    for (int s = 0; s < S; ++s) {
      const double x = there[s] ? c[s] : NONE;
      second = larger(second, smaller(first, x));
      first = larger(first, x);
    }
    // after step d a lane has those of the 2 d lanes from it on, as far as they are its group's
    for (int d = 1; d < p.lanes; d *= 2) {
      const double f = __shfl_down(first, d, 64), g = __shfl_down(second, d, 64);
      if (own.in_group + d < p.lanes) {
        second = larger(smaller(first, f), larger(second, g));
        first = larger(first, f);
      }
    }
    const double both = __shfl(first + (second > NONE ? second : 0.), lane - own.in_group, 64);
    int above = 0;   // groups in front of this lane's
    for (int g = 0; g < p.groups; ++g) {
      const double x = read_lane(both, g * p.lanes);
      above += x > both || (x == both && g < own.group);
    }
    open = above < p.chosen_groups;
    if (!p.bias) {
#pragma unroll
      for (int s = 0; s < S; ++s) c[s] = (double)z[s];
    }
  }
  uint64_t key[S];
#pragma unroll
  for (int s = 0; s < S; ++s) key[s] = there[s] && open ? order_key64(c[s]) : 0;
  expert = -1;
  for (int j = 0; j < k; ++j) {
    uint64_t best = key[0];
    int which = 0;
#pragma unroll
    for (int s = 1; s < S; ++s)
      if (key[s] > best) {
        best = key[s];
        which = s;
      }
    int at;
    if (wave_max64(best, at) == 0) break;
    const int e = __builtin_amdgcn_readlane(own.first + which, at);
#pragma unroll
    for (int s = 0; s < S; ++s)
      if (own.first + s == e) key[s] = 0;
    if (lane == j) expert = e;
  }
  const float chosen = expert >= 0 ? load_el<EL>(logits, t * ld + expert) : 0.f;
  weight = (float)(p.scale * chosen_share(p, expert, chosen, most, sum));
}

struct RouteArgs {
  const void *logits;
  int64_t ld;
  int T, E, k;
  float *weights;                          // [T, k]
  int *experts, *offsets, *order, *place;  // [T, k], [E + 1], [T k], [T k]
  int *counts, *totals;                    // [blocks, E]: slots of a block's tokens by expert, then those in front of the block; [E]: of all
  int tokens;                              // of a block
  Scores scores;
};
// SCORED: by scores, bias and groups
template <int EL, int S, bool SCORED>
__device__ __forceinline__ void choose_by(const RouteArgs &a, const Span &own, int t, int &expert, float &weight) {
  if constexpr (SCORED) choose_scored<EL, S>(a.logits, a.ld, t, a.k, a.scores, own, expert, weight);
  else choose<EL, S>(a.logits, a.ld, t, a.E, a.k, expert, weight);
}

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

// One workgroup does it all.  A second launch takes 1 to 2 us more, more tokens than waves take turns of k reductions each: 56 tokens, 2 of 8
// experts 6.1 us in one and 6.3 in two, 64 tokens 6.7 and 6.5, 32 tokens, 6 of 64, 6.6 and 7.0, 40 tokens 7.2 and 6.8, 8 of 64, 24 tokens 6.6 and
// 7.0, 32 tokens 7.0 and 6.6; by scores and groups, 8 of 256 experts, 12 tokens 11.5 and 11.7, 32 tokens 21 and 11.6.
constexpr int MAX_SPAN = 32, FEW_TOKENS = 64, FEW_EXPERTS = 256, FEW_WAVES = 16;
// the most experts that a lane has where the groups' lanes, whole ones, are no more than a wave's (launch_route_of) and experts are up to `most`
constexpr int span_of(int most) {
  int span = 1;
  for (int groups = 1; groups <= MAX_GROUPS; ++groups)
    for (int size = 1; groups * size <= most; ++size)
      while (groups * ((size + span - 1) / span) > 64) span *= 2;
  return span;
}
constexpr int FEW_SPAN = span_of(FEW_EXPERTS);   // (3 groups of 85 experts: 8 to a lane, where 256 experts without groups are 4)
static_assert(FEW_SPAN == 8 && span_of(MAX_EXPERTS) <= MAX_SPAN, "instances of launch_route_of");

template <int EL, int S, bool SCORED>
__global__ __launch_bounds__(64 * FEW_WAVES) void route_few_kernel(RouteArgs a) {
  extern __shared__ int lds[];
  int *experts = lds, *have = lds + FEW_TOKENS * a.k, *total = have + FEW_WAVES * a.E, *word = total + a.E;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, n = a.T * a.k;
  const Span own(a.scores, S);
  for (int t = wave; t < a.T; t += FEW_WAVES) {
    int e;
    float w;
    choose_by<EL, S, SCORED>(a, own, t, e, w);
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

// More tokens: choice and counts by blocks, sums of the counts in front of each block, then places.  8192 tokens, 8 of 256 experts: 17 us (every
// block adding up the counts of all by itself 50), by scores 28.
// (sixteen scores in 64 bits to a lane do not fit the registers of sixteen waves)
constexpr int WAVES = 4;
template <int S, bool SCORED>
constexpr int choose_threads = SCORED && S >= 16 ? 512 : 1024;
template <int EL, int S, bool SCORED>
__global__ __launch_bounds__((choose_threads<S, SCORED>)) void route_choose_kernel(RouteArgs a) {
  extern __shared__ int lds[];   // [E] counts of the block
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, t0 = blockIdx.x * a.tokens, t1 = min(a.T, t0 + a.tokens);
  const Span own(a.scores, S);
  for (int e = threadIdx.x; e < a.E; e += blockDim.x) lds[e] = 0;
  __syncthreads();
  for (int t = t0 + wave; t < t1; t += blockDim.x / 64) {
    int e;
    float w;
    choose_by<EL, S, SCORED>(a, own, t, e, w);
    if (lane < a.k) {
      a.experts[(int64_t)t * a.k + lane] = e;
      a.weights[(int64_t)t * a.k + lane] = w;
      if (e >= 0) atomicAdd(&lds[e], 1);
    }
  }
  __syncthreads();
  for (int e = threadIdx.x; e < a.E; e += blockDim.x) a.counts[(int64_t)blockIdx.x * a.E + e] = lds[e];
}
// the counts of SCAN_EXPERTS experts: 64 threads to an expert, each with up to SHARE blocks
constexpr int MOST_BLOCKS = 256, SHARE = MOST_BLOCKS / 64, SCAN_EXPERTS = 16;
__global__ __launch_bounds__(64 * SCAN_EXPERTS) void route_scan_kernel(int *counts, int *totals, int blocks, int E) {
  __shared__ int parts[64][SCAN_EXPERTS + 1];
  const int e = blockIdx.x * SCAN_EXPERTS + threadIdx.x % SCAN_EXPERTS, share = threadIdx.x / SCAN_EXPERTS, b0 = share * SHARE;
  int c[SHARE], sum = 0;
#pragma unroll
  for (int j = 0; j < SHARE; ++j) c[j] = e < E && b0 + j < blocks ? counts[(b0 + j) * E + e] : 0;
#pragma unroll
  for (int j = 0; j < SHARE; ++j) sum += c[j];
  parts[share][threadIdx.x % SCAN_EXPERTS] = sum;
  __syncthreads();
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, part = parts[lane][wave];
  int x = part;
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const int y = __shfl_up(x, d, 64);
    if (lane >= d) x += y;
  }
  parts[lane][wave] = x - part;
  if (lane == 63 && blockIdx.x * SCAN_EXPERTS + wave < E) totals[blockIdx.x * SCAN_EXPERTS + wave] = x;
  __syncthreads();
  int before = parts[share][threadIdx.x % SCAN_EXPERTS];
#pragma unroll
  for (int j = 0; j < SHARE; ++j) {
    if (e < E && b0 + j < blocks) counts[(b0 + j) * E + e] = before;
    before += c[j];
  }
}
// threads to an expert where a block adds up the counts of all blocks by itself, and the blocks up to which that is less than the scan: 512
// tokens, 2 of 8 experts 6.5 us, with it 8.5, 8 of 64 experts 8.2 and 9.9; by scores, 8 of 256 experts, 256 tokens in 64 blocks 13.9 and 14.3
constexpr int shares_of(int E) { return E < 64 * WAVES ? 64 * WAVES / E : 1; }
constexpr int unscanned_blocks(int E) { return shares_of(E) > 2 ? 32 * shares_of(E) : 64; }
// SCANNED: the kernel above has run; of a few blocks every block adds up the counts by itself
template <bool SCANNED>
__global__ __launch_bounds__(64 * WAVES) void route_place_kernel(RouteArgs a) {
  extern __shared__ int lds[];
  int *have = lds, *total = have + WAVES * a.E, *front = total + a.E, *word = front + a.E;
  const int t0 = blockIdx.x * a.tokens, t1 = min(a.T, t0 + a.tokens), slot0 = t0 * a.k, n = (t1 - t0) * a.k;
  const int *experts = a.experts + slot0;
  // (eight counts are on their way together)
  const int blocks = (int)gridDim.x, shares = SCANNED || blocks <= 8 ? 1 : shares_of(a.E), step = 8 * shares;
  if (SCANNED || shares > 1)
    for (int e = threadIdx.x; e < a.E; e += 64 * WAVES) {
      total[e] = SCANNED ? a.totals[e] : 0;
      front[e] = SCANNED ? a.counts[(int64_t)blockIdx.x * a.E + e] : 0;
    }
  if constexpr (!SCANNED) {
    if (shares > 1) __syncthreads();   // (uniform)
    for (int i = threadIdx.x; i < shares * a.E; i += 64 * WAVES) {
      const int share = (int)((unsigned)i / (unsigned)a.E), e = i - share * a.E;
      int sum = 0, before = 0;
      auto eight = [&](auto all, int b0) {
        int c[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) c[j] = decltype(all)::value || b0 + j * shares < blocks ? a.counts[(b0 + j * shares) * a.E + e] : 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          sum += c[j];
          before += b0 + j * shares < (int)blockIdx.x ? c[j] : 0;
        }
      };
      int b0 = share;
      for (; b0 + 7 * shares < blocks; b0 += step) eight(std::true_type{}, b0);
      if (b0 < blocks) eight(std::false_type{}, b0);
      if (shares == 1) {
        total[e] = sum;
        front[e] = before;
      } else {   // (sums of whole numbers, whose order does not matter)
        atomicAdd(&total[e], sum);
        atomicAdd(&front[e], before);
      }
    }
  }
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

// tokens of a block (256 tokens, 8 of 64 experts, four to a block 8.1 us, eight 7.5; by scores, 128 tokens, 8 of 256, 12.5 and 13.0)
int route_tokens(int64_t T, bool scored) {
  const int64_t tokens = (T + MOST_BLOCKS - 1) / MOST_BLOCKS, least = scored ? 4 : 8;
  return (int)(tokens < least ? least : tokens);
}
bool few_tokens(int64_t T, int64_t E, int64_t k, bool scored) {
  return E <= FEW_EXPERTS && (T <= FEW_WAVES || (!scored && T <= FEW_TOKENS && T * (k + 2) <= 256));
}
int route_blocks(int64_t T, int64_t E, int64_t k, bool scored) {
  return few_tokens(T, E, k, scored) ? 0 : (int)((T + route_tokens(T, scored) - 1) / route_tokens(T, scored));
}

template <int EL, int S, bool SCORED>
int launch_route(RouteArgs a, int blocks, hipStream_t s) {
  a.scores.lanes = (a.scores.size + S - 1) / S;
  if constexpr (S <= FEW_SPAN) {
    if (blocks == 0) {
      const size_t lds = sizeof(int) * (FEW_TOKENS * a.k + (FEW_WAVES + 1) * a.E + 1);
      hipLaunchKernelGGL((route_few_kernel<EL, S, SCORED>), dim3(1), dim3(64 * FEW_WAVES), lds, s, a);
      return (int)hipGetLastError();
    }
  }
  const int waves = a.tokens * 64 < choose_threads<S, SCORED> ? a.tokens : choose_threads<S, SCORED> / 64;
  hipLaunchKernelGGL((route_choose_kernel<EL, S, SCORED>), dim3(blocks), dim3(64 * waves), sizeof(int) * a.E, s, a);
  if (hipGetLastError() != hipSuccess) return 1;
  const size_t lds = sizeof(int) * ((WAVES + 2) * a.E + 1);
  if (blocks <= unscanned_blocks(a.E)) {
    hipLaunchKernelGGL(route_place_kernel<false>, dim3(blocks), dim3(64 * WAVES), lds, s, a);
    return (int)hipGetLastError();
  }
  hipLaunchKernelGGL(route_scan_kernel, dim3((a.E + SCAN_EXPERTS - 1) / SCAN_EXPERTS), dim3(64 * SCAN_EXPERTS), 0, s, a.counts, a.totals, blocks, a.E);
  if (hipGetLastError() != hipSuccess) return 1;
  hipLaunchKernelGGL(route_place_kernel<true>, dim3(blocks), dim3(64 * WAVES), lds, s, a);
  return (int)hipGetLastError();
}
// experts to a lane so that the groups' lanes, whole ones, are no more than a wave's (MAX_SPAN always do)
bool fits_wave(const Scores &p, int S) { return p.groups * ((p.size + S - 1) / S) <= 64; }
template <int EL, bool SCORED>
int launch_route_of(const RouteArgs &a, int blocks, hipStream_t s) {
  if constexpr (SCORED) {
    if (fits_wave(a.scores, 1)) return launch_route<EL, 1, true>(a, blocks, s);
    if (fits_wave(a.scores, 2)) return launch_route<EL, 2, true>(a, blocks, s);
    if (fits_wave(a.scores, 4)) return launch_route<EL, 4, true>(a, blocks, s);
    if (fits_wave(a.scores, 8)) return launch_route<EL, 8, true>(a, blocks, s);
    return fits_wave(a.scores, 16) ? launch_route<EL, 16, true>(a, blocks, s) : launch_route<EL, MAX_SPAN, true>(a, blocks, s);
  } else {
    if (a.E <= 64) return launch_route<EL, 1, false>(a, blocks, s);
    if (a.E <= 128) return launch_route<EL, 2, false>(a, blocks, s);
    if (a.E <= 256) return launch_route<EL, 4, false>(a, blocks, s);
    return launch_route<EL, 16, false>(a, blocks, s);
  }
}
template <bool SCORED>
int launch_route_by(int el, const RouteArgs &a, int blocks, hipStream_t s) {
  return el == EL_F16 ? launch_route_of<EL_F16, SCORED>(a, blocks, s)
                      : (el == EL_BF16 ? launch_route_of<EL_BF16, SCORED>(a, blocks, s) : launch_route_of<EL_F32, SCORED>(a, blocks, s));
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

// The same with scores: with g = factor * dw, r the shares and s the scores of the chosen, by the scores' own formula
//   sigmoid   g_j s_j (1 - s_j), renormalised r_j (1 - s_j) (g_j - sum r g)
//   softmax   s_e (g_e - sum s g) for every expert of the token (g is 0 for the others), renormalised r_j (g_j - sum r g)
// computed again from the logits in 64 bits: differences of nearly equal gradients keep their digits.
template <int EL, int S>
__global__ __launch_bounds__(64 * WAVES) void route_scored_backward_kernel(const void *logits, int64_t ld, const int *experts, const float *dweights, int T, int E,
                                                                           int k, Scores p, void *dlogits) {
  extern __shared__ float row_lds[];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t t = wide_block() * WAVES + wave;
  if (t >= T) return;   // (a wave's rows are its own: no barrier)
  float *row = row_lds + wave * E;
  double most = 0., sum = 1.;
  float z[S];
  const bool all = !p.sigmoid && !p.renormalize;
  if (all) {
    uint32_t top = 0;
#pragma unroll
    for (int s = 0; s < S; ++s) {
      z[s] = 64 * s + lane < E ? load_el<EL>(logits, t * ld + 64 * s + lane) : -__builtin_inff();
      top = max(top, order_key(z[s]));
    }
    top = wave_max(top);
    most = __builtin_bit_cast(float, top & 0x80000000u ? top ^ 0x80000000u : ~top);
    double part = 0.;
#pragma unroll
    for (int s = 0; s < S; ++s) part += z[s] > -__builtin_inff() ? exp_from(z[s], most) : 0.;
    sum = wave_sum(part);
  }
  const int e = lane < k ? experts[t * k + lane] : -1;
  const bool mine = e >= 0 && e < E;
  const float own = mine ? load_el<EL>(logits, t * ld + e) : 0.f;
  const double g = mine ? p.scale * (double)dweights[t * k + lane] : 0.;
  const double r = chosen_share(p, mine ? e : -1, own, most, sum);
  double d;
  if (p.sigmoid && !p.renormalize) {
    d = g * r * (1. / (1. + exp((double)own)));
  } else {
    const double dot = wave_sum(r * g);
    d = r * (g - dot);
    if (p.sigmoid) d *= 1. / (1. + exp((double)own));
    if (all) {
#pragma unroll
      for (int s = 0; s < S; ++s)
        if (64 * s + lane < E) row[64 * s + lane] = z[s] > -__builtin_inff() ? (float)(-(exp_from(z[s], most) / sum) * dot) : 0.f;
    }
  }
  if (!all)
    for (int i = lane; i < E; i += 64) row[i] = 0.f;
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
  if (mine) row[e] = (float)d;
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
  for (int i = lane; i < E; i += 64) store_el<EL>(dlogits, t * E + i, row[i]);
}
template <int EL>
int launch_scored_backward(const void *logits, int64_t ld, const int *experts, const float *dweights, int T, int E, int k, const Scores &p, void *dlogits,
                           hipStream_t s) {
  const dim3 grid = wide_grid((T + WAVES - 1) / WAVES), block(64 * WAVES);
  const size_t lds = sizeof(float) * WAVES * E;
#define SK_SCORED_BACKWARD(S) \
  hipLaunchKernelGGL((route_scored_backward_kernel<EL, S>), grid, block, lds, s, logits, ld, experts, dweights, T, E, k, p, dlogits)
  if (E <= 64) SK_SCORED_BACKWARD(1);
  else if (E <= 256) SK_SCORED_BACKWARD(4);
  else SK_SCORED_BACKWARD(16);
#undef SK_SCORED_BACKWARD
  return (int)hipGetLastError();
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
  if (check_route_shape(T, E, k) != SK_OK) return 0;
  const int blocks = route_blocks(T, E, k, true);   // (whichever takes more)
  return blocks > 0 ? sizeof(int) * (size_t)(blocks + 1) * (size_t)E : 0;
}

// p: null for the plain route
static int route(const void *logits, int dtype, int64_t T, int64_t E, int64_t k, int64_t ld, const Scores *p, void *weights, void *experts, void *offsets, void *order,
                 void *place, void *ws, size_t ws_bytes, void *stream) {
  if (element_of(dtype) < 0) return SK_ERR_CONFIG;
  if (int rc = check_route_shape(T, E, k)) return rc;
  if (!logits || !weights || !experts || !offsets || !order || !place) return SK_ERR_NULL;
  if (ld < E) return SK_ERR_SHAPE;
  const int blocks = route_blocks(T, E, k, p != nullptr);
  if (ws_bytes < sk_route_workspace_bytes(T, E, k) || (blocks > 0 && !ws)) return SK_ERR_WORKSPACE;
  if (reinterpret_cast<uintptr_t>(ws) & 3) return SK_ERR_ALIGN;
  RouteArgs a{logits, ld, (int)T, (int)E, (int)k, (float *)weights, (int *)experts, (int *)offsets, (int *)order, (int *)place, (int *)ws,
              (int *)ws + (int64_t)blocks * E, route_tokens(T, p != nullptr), p ? *p : Scores{nullptr, 1., 1, 1, (int)E, 1, false, true}};
  const int herr = p ? launch_route_by<true>(element_of(dtype), a, blocks, (hipStream_t)stream) : launch_route_by<false>(element_of(dtype), a, blocks, (hipStream_t)stream);
  return herr == 0 ? SK_OK : SK_ERR_LAUNCH;
}
// fills p; sk_status
static int check_scores(const sk_route_scores *s, int64_t E, int64_t k, Scores *p) {
  if (!s) return SK_ERR_NULL;
  if ((s->scores != SK_SCORES_SOFTMAX && s->scores != SK_SCORES_SIGMOID) || !(s->scale > -__builtin_inf() && s->scale < __builtin_inf())) return SK_ERR_CONFIG;
  if (s->groups < 1 || s->groups > MAX_GROUPS || E % s->groups || s->chosen_groups < 1 || s->chosen_groups > s->groups || k > E / s->groups * s->chosen_groups)
    return SK_ERR_SHAPE;
  if (reinterpret_cast<uintptr_t>(s->bias) & 3) return SK_ERR_ALIGN;
  // (all groups open: none is asked)
  const int groups = s->chosen_groups == s->groups ? 1 : s->groups;
  *p = Scores{(const float *)s->bias, s->scale, groups, s->chosen_groups, (int)(E / groups), 1, s->scores == SK_SCORES_SIGMOID, s->renormalize != 0};
  return SK_OK;
}

extern "C" int sk_route_experts(const void *logits, int dtype, int64_t T, int64_t E, int64_t k, int64_t ld, void *weights, void *experts,
                                void *offsets, void *order, void *place, void *ws, size_t ws_bytes, void *stream) {
  return route(logits, dtype, T, E, k, ld, nullptr, weights, experts, offsets, order, place, ws, ws_bytes, stream);
}

extern "C" int sk_route_scored(const void *logits, int dtype, int64_t T, int64_t E, int64_t k, int64_t ld, const sk_route_scores *scores, void *weights,
                               void *experts, void *offsets, void *order, void *place, void *ws, size_t ws_bytes, void *stream) {
  if (int rc = check_route_shape(T, E, k)) return rc;
  Scores p;
  if (int rc = check_scores(scores, E, k, &p)) return rc;
  return route(logits, dtype, T, E, k, ld, &p, weights, experts, offsets, order, place, ws, ws_bytes, stream);
}

extern "C" int sk_route_scored_backward(const void *logits, int dtype, int64_t T, int64_t E, int64_t k, int64_t ld, const sk_route_scores *scores,
                                        const void *experts, const void *dweights, void *dlogits, void *stream) {
  if (element_of(dtype) < 0) return SK_ERR_CONFIG;
  if (int rc = check_route_shape(T, E, k)) return rc;
  Scores p;
  if (int rc = check_scores(scores, E, k, &p)) return rc;
  if (!logits || !experts || !dweights || !dlogits) return SK_ERR_NULL;
  if (ld < E) return SK_ERR_SHAPE;
  const int el = element_of(dtype);
  const auto launch = el == EL_F16 ? launch_scored_backward<EL_F16> : (el == EL_BF16 ? launch_scored_backward<EL_BF16> : launch_scored_backward<EL_F32>);
  return launch(logits, ld, (const int *)experts, (const float *)dweights, (int)T, (int)E, (int)k, p, dlogits, (hipStream_t)stream) == 0 ? SK_OK : SK_ERR_LAUNCH;
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
