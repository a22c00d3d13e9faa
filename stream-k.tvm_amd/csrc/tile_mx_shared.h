// Microscaled 4-bit products (tile_mx.h) on tiles that a CTA's four or eight waves share: WM x WN waves, each with its part of the tile, operands through
// a ring of LDS that all of them fill and read.
//
// A chunk is 256 values of K, 128 bytes a row; the exponents of two chunks come together, 16 bytes a row.  Each wave fetches its part
// of a chunk's rows.  A chunk is multiplied in two steps of 128: beside the MFMAs of the first stand the reads of the second's fragments, then
// one barrier -- everybody has read this chunk, and the next one has landed --, and beside those of the second the reads of the next
// chunk's and the loads of the chunk that takes this one's place.  So STAGES - 1 chunks are on their way or waiting.
//
// Eight waves for 128 x 256: 1024 x 8192 x 8192 43 us where 128 x 128, two to a CU, take 55 and 256 x 256 47, 2048 x 4096 x 4096 24.5 and 25.3 (36).  One
// 128 x 128 tile to a CU, in four stages: 58 us with four waves and 57 with eight.
//
// Against tile_mx.h's 64 x 64 tiles a 128 x 128 tile takes in half the bytes for each product, which is what bounds those with many
// rows (a CU takes in 50 to 100 GB/s); against 256 x 256 tiles it fills the CUs from a quarter of the rows on.
#pragma once
#include "tile_asm_epilogue.h"
#include "tile_epilogue.h"
#include "tile_mx.h"
#include "tile_scaled_i8.h"

namespace sk {

template <bool BF16_, int BM_, int BN_, int WM_, int WN_, int STAGES_, int CTAS_>
struct TileMxShared {
  typedef MxArgs Args;
  typedef int intx4 __attribute__((ext_vector_type(4)));
  typedef int intx8 __attribute__((ext_vector_type(8)));
  static constexpr bool COHERENT_PARTIALS = true, FIXUP_WORD_IN_LDS = true, BF16 = BF16_;
  static constexpr int BM = BM_, BN = BN_, WM = WM_, WN = WN_, STAGES = STAGES_, WAVES = WM_ * WN_, NT = 64 * WAVES;
  static constexpr int WTM = BM / WM, WTN = BN / WN, FM = WTM / 16, FN = WTN / 16, NB = FM * FN, TILE_ELEMS = BM * BN;
  static constexpr int KV = 64, BK = 2 * KV;                   // pairs of bytes: of a chunk, of an iteration
  static constexpr int LW = (BM + BN) / (8 * WAVES);           // a wave's loads of a chunk, 8 rows each
  static constexpr int LE = (BM + BN + NT - 1) / NT;           // and of two chunks' exponents, 64 rows each
  static constexpr int CHUNK = (BM + BN) * 128, PAIR = (BM + BN) * 16, PAIRS = (STAGES + 2) / 2;   // bytes; pairs of chunks whose exponents are kept
  static constexpr int EXPONENTS = STAGES * CHUNK, LDS_BYTES = EXPONENTS + PAIRS * PAIR, CTAS_PER_CU = CTAS_, WAVES_PER_EU = CTAS_ * WAVES / 4, CUT_COST = 8;
  static_assert(BM % (8 * WAVES) == 0 && BN % (8 * WAVES) == 0 && CTAS_ * LDS_BYTES <= 160 * 1024, "see above");
  typedef BlockPatch<FM, FN> Patch;
  static_assert(WAVES * Patch::BYTES <= LDS_BYTES, "the patches fit the ring");

  struct Acc {
    floatx4 c[NB];
  };
  static __device__ __forceinline__ void zero_sums(Acc &acc) {
    static_for<0, NB>([&](auto v) { acc.c[v] = floatx4{0.f, 0.f, 0.f, 0.f}; });
  }
  static constexpr int loads(int parity) { return LW + (parity == 0 ? LE : 0); }
  static constexpr int loads_behind(int P, int behind) { return behind == 0 ? 0 : loads_behind(P, behind - 1) + loads((P + behind) & 1); }
  // a chunk of parity P has landed, behind which `behind` chunks have been requested (at most MOST)
  template <int P, int MOST>
  static __device__ __forceinline__ void wait_chunk(int behind) {
    if (behind >= MOST) wavek_wait_loads<loads_behind(P, MOST)>();
    else if (behind == 0) wavek_wait_loads<0>();
    else if (behind == 1) wavek_wait_loads<loads_behind(P, 1)>();
    else wavek_wait_loads<loads_behind(P, 2)>();
  }
  struct Frags {
    intx4 a[FM], b[FN];
  };
  struct Exponents {
    int a[FM], b[FN];   // byte of the step
  };

  static __device__ __forceinline__ void mac(const Args &a, Acc &acc, int pm, int pn, int k0, int n, char *smem) {
    const int tid = pin_here((int)threadIdx.x), lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), wm = wave / WN, wn = wave % WN;
    zero_sums(acc);
    const uint32_t lda_bytes = (uint32_t)a.lda * 2, ldb_bytes = (uint32_t)a.ldb * 2;
    const int rows_a = min(BM, a.M - pm * BM), rows_b = min(BN, a.N - pn * BN);
    // rows past M / N lie beyond the descriptors' ranges and read as zero
    const uint4v rsrc_a = uniform_rsrc(make_rsrc_words(a.A + (int64_t)pm * BM * a.lda, (uint32_t)rows_a * lda_bytes));
    const uint4v rsrc_b = uniform_rsrc(make_rsrc_words(a.B + (int64_t)pn * BN * a.ldb, (uint32_t)rows_b * ldb_bytes));
    const uint4v rsrc_ea = uniform_rsrc(a.ea.row((int64_t)pm * BM).rsrc()), rsrc_eb = uniform_rsrc(a.eb.row((int64_t)pn * BN).rsrc());
    // load x of a chunk: rows 8 (wave + WAVES x) .. + 7 of A's and then the weights', lane's row lane / 8; piece p (16 bytes, 32 values) of row r stands
    // at position p ^ ((r >> 1) & 7)
    const int row8 = lane >> 3, fi = lane & 15, fg = mx_group(lane), kp = ((lane & 7) ^ (4 * (wave & 1) + (row8 >> 1))) * 8;
    const uint32_t off_a = (uint32_t)row8 * lda_bytes + (uint32_t)kp * 2, off_b = (uint32_t)row8 * ldb_bytes + (uint32_t)kp * 2;
    const uint32_t off_ea = (uint32_t)(lane * a.ea.pitch), off_eb = (uint32_t)(lane * a.eb.pitch);
    const uint32_t ring = lds_address(smem) + (uint32_t)wave * 1024;
    const int rot = rotation_of(pn, n), chunks = 2 * n;
    auto left_of = [&](int t) { return t < chunks ? a.K - ((k0 + rotated_iteration(t >> 1, rot, n)) * 2 + (t & 1)) * KV : 0; };
    struct Chunk {
      uint32_t kbytes, base, pair;   // base, pair: LDS addresses
      int left;
    };
    auto chunk = [&](int t, int slot, int pair) {
      const int left = left_of(t);
      const uint32_t kbytes = (uint32_t)__builtin_amdgcn_readfirstlane(left > 0 ? (a.K - left) * 2 : 0);
      return Chunk{kbytes, ring + (uint32_t)slot * CHUNK, ring - (uint32_t)wave * 1024 + EXPONENTS + (uint32_t)pair * PAIR, left};
    };
    auto issue = [&](auto xi, const Chunk &q) {
      constexpr int x = decltype(xi)::value;
      constexpr bool A = x < BM / (8 * WAVES);
      const uint32_t rows = q.kbytes + (uint32_t)(8 * (wave + WAVES * (A ? x : x - BM / (8 * WAVES)))) * (A ? lda_bytes : ldb_bytes);
      wavek_dma_16<x * WAVES * 1024>(A ? rsrc_a : rsrc_b, q.base, kp < q.left ? (A ? off_a : off_b) : OOB_OFFSET, rows);
    };
    // (rows 64 (wave + WAVES y) ..; the exponents of a row's end and of what lies behind it arrive together, see mask_exponents)
    auto issue_exponents = [&](const Chunk &q) {
      static_for<0, LE>([&](auto yi) {
        constexpr int y = decltype(yi)::value;
        const int first = min(64 * (wave + WAVES * y), BM + BN - 64);   // (waves behind the last rows fetch these again)
        const bool of_a = first < BM, any = q.left > 0;
        const int at = (int)q.kbytes / 256;
        const uint32_t rows = (uint32_t)(any ? (of_a ? at * a.ea.step + first * a.ea.pitch : at * a.eb.step + (first - BM) * a.eb.pitch) : 0);
        wavek_dma_16<0>(uniform_rsrc(of_a ? rsrc_ea : rsrc_eb), q.pair + (uint32_t)first * 16, any ? (of_a ? off_ea : off_eb) : OOB_OFFSET,
                        (uint32_t)__builtin_amdgcn_readfirstlane((int)rows));
      });
    };
    static_for<0, STAGES>([&](auto t) {
      if (t < chunks) {
        const Chunk q = chunk(t, t, t / 2 % PAIRS);
        if constexpr (t % 2 == 0) issue_exponents(q);
        static_for<0, LW>([&](auto x) { issue(x, q); });
      }
    });
    // fragments: lane (i, g) takes piece 2 g + s of its row for step s
    const uint32_t pos0 = (uint32_t)((2 * fg) ^ ((fi >> 1) & 7)) * 16;
    const char *rd_a = smem + (wm * WTM + fi) * 128 + pos0, *rd_b = smem + (BM + wn * WTN + fi) * 128 + pos0;
    const char *rd_a1 = smem + (wm * WTM + fi) * 128 + (pos0 ^ 16), *rd_b1 = smem + (BM + wn * WTN + fi) * 128 + (pos0 ^ 16);
    const char *rd_ea = smem + EXPONENTS + (wm * WTM + fi) * 16 + 2 * fg, *rd_eb = smem + EXPONENTS + (BM + wn * WTN + fi) * 16 + 2 * fg;
    auto read = [&](auto ri, auto step, Frags &f, int slot) {
      constexpr int r = decltype(ri)::value, s = decltype(step)::value;
      if constexpr (r < FN) f.b[r] = *reinterpret_cast<const intx4 *>((s ? rd_b1 : rd_b) + slot * CHUNK + r * 2048);
      else f.a[r - FN] = *reinterpret_cast<const intx4 *>((s ? rd_a1 : rd_a) + slot * CHUNK + (r - FN) * 2048);
    };
    auto read_exponent = [&](auto ri, auto parity, Exponents &e, int pair) {
      constexpr int r = decltype(ri)::value, P = decltype(parity)::value;
      if constexpr (r < FN) e.b[r] = *reinterpret_cast<const uint16_t *>(rd_eb + pair * PAIR + r * 256 + 8 * P);
      else e.a[r - FN] = *reinterpret_cast<const uint16_t *>(rd_ea + pair * PAIR + (r - FN) * 256 + 8 * P);
    };
    // the last chunk of K: blocks behind K are zeros, and their exponents, which are another row's, have to be numbers
    auto mask_exponents = [&](int left, Exponents &e) {
      const int mask = (16 * fg < left ? 0xff : 0) | (16 * fg + 8 < left ? 0xff00 : 0);
#pragma unroll
      for (int i = 0; i < FM; ++i) e.a[i] &= mask;
#pragma unroll
      for (int j = 0; j < FN; ++j) e.b[j] &= mask;
    };
    auto mfma = [&](auto vi, auto step, const Frags &f, const Exponents &e) {
      constexpr int v = decltype(vi)::value, s = decltype(step)::value, i = v / FN, j = i % 2 ? FN - 1 - v % FN : v % FN;
      const intx8 b = __builtin_shufflevector(f.b[j], f.b[j], 0, 1, 2, 3, -1, -1, -1, -1), x = __builtin_shufflevector(f.a[i], f.a[i], 0, 1, 2, 3, -1, -1, -1, -1);
      acc.c[i * FN + j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(b, x, acc.c[i * FN + j], 4, 4, s, e.b[j], s, e.a[i]);   // (4: e2m1)
    };
    constexpr std::integral_constant<int, 0> zero;
    constexpr std::integral_constant<int, 1> one;
    constexpr int READS = FM + FN;
    int slot = 0, pair = 0;   // of chunk t
    Frags f0, f1;             // of the steps
    // REFILL: chunk t + STAGES is requested; MORE: there is a chunk t + 1.  (The loops below say which: with the choice inside, the compiler
    // moves the accumulators between its register files for every MFMA.)
    auto body = [&](int t, auto parity, auto refill, auto more, const Exponents &e, Exponents &en) {
      constexpr int P = decltype(parity)::value;
      constexpr bool REFILL = decltype(refill)::value, MORE = decltype(more)::value, FIRST = ((P + STAGES) & 1) == 0;
      const int next = slot + 1 == STAGES ? 0 : slot + 1, next_pair = P == 0 ? pair : (pair + 1 == PAIRS ? 0 : pair + 1);
      static_for<0, NB>([&](auto v) {
        mfma(v, zero, f0, e);
        static_for<v * READS / NB, (v + 1) * READS / NB>([&](auto r) { read(r, one, f1, slot); });
        __builtin_amdgcn_sched_barrier(0);
      });
      if constexpr (REFILL) wavek_wait_loads<loads_behind(1 - P, STAGES - 2)>();
      else if constexpr (MORE) wait_chunk<1 - P, STAGES - 2>(chunks - 2 - t);
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
      Chunk q;
      if constexpr (REFILL) {
        q = chunk(t + STAGES, slot, ((t + STAGES) >> 1) % PAIRS);
        if constexpr (FIRST) issue_exponents(q);
      }
      static_for<0, NB>([&](auto v) {
        mfma(v, one, f1, e);
        if constexpr (REFILL) static_for<v * LW / NB, (v + 1) * LW / NB>([&](auto x) { issue(x, q); });
        if constexpr (MORE)
          static_for<v * READS / NB, (v + 1) * READS / NB>([&](auto r) {
            read(r, zero, f0, next);
            read_exponent(r, std::integral_constant<int, 1 - P>{}, en, next_pair);
          });
        __builtin_amdgcn_sched_barrier(0);
      });
      if constexpr (MORE) {
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        mask_exponents(left_of(t + 1), en);
      }
      slot = next;
      pair = next_pair;
    };
    Exponents x, y;
    wait_chunk<0, STAGES - 1>(chunks - 1);
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    static_for<0, READS>([&](auto r) {
      read(r, zero, f0, 0);
      read_exponent(r, zero, x, 0);
    });
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    mask_exponents(left_of(0), x);
    constexpr std::true_type yes;
    constexpr std::false_type no;
    int t = 0;
    for (; t + 1 + STAGES < chunks; t += 2) {
      body(t, zero, yes, yes, x, y);
      body(t + 1, one, yes, yes, y, x);
    }
    if constexpr (STAGES % 2 == 1)
      if (t + STAGES < chunks) {
        body(t, zero, yes, yes, x, y);
        body(t + 1, one, no, yes, y, x);
        t += 2;
      }
    for (; t + 2 < chunks; t += 2) {
      body(t, zero, no, yes, x, y);
      body(t + 1, one, no, yes, y, x);
    }
    body(t, zero, no, yes, x, y);
    body(t + 1, one, no, no, y, x);
    wavek_wait_loads<0>();
    __syncthreads();   // the ring may be used for something else
  }

  // (one activation at a time: with the choice at every value a tile of 100 x 11008 x 4096, ReLU, took 1.2 us longer than without any)
  static __device__ __forceinline__ void store_c(const Args &a, const Acc &acc, int pm, int pn, char *smem, const void *epi) {
    by_epilogue(epi, [&](auto e) { store_by<decltype(e)::value>(a, acc, pm, pn, smem, epi); });
    __syncthreads();   // the patches overlap the ring
  }
  // EPI: -1 nothing, else bias and the activation of this number
  template <int EPI>
  static __device__ __forceinline__ void store_by(const Args &a, const Acc &acc, int pm, int pn, char *smem, const void *epi) {
    const int tid = pin_here((int)threadIdx.x), lane = tid & 63, wave = tid >> 6;
    const int row0 = pm * BM + wave / WN * WTM, col0 = pn * BN + wave % WN * WTN;
    half4v bias[EPI >= 0 ? FN : 1];
    if constexpr (EPI >= 0) static_for<0, FN>([&](auto j) { bias[j] = raw_bias4_at(epi_bias(epi), col0 + 16 * j + 4 * (lane >> 4), a.N); });
    Patch::store(a.C, a.ldc, a.M, a.N, row0, col0, smem + wave * Patch::BYTES, [&](auto i, auto j) {
      floatx4 v = acc.c[i * FN + j];
      if constexpr (EPI >= 0) {
        const floatx4 b = widen4<BF16>(bias[j]);
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = activate_by_rcp(v[e] + b[e], EPI);
      }
      return round4<BF16>(v);
    });
  }

  static __device__ __forceinline__ void store_partial(const Acc &acc, float *dst) {
    const BufferRsrc r = make_rsrc(dst, TILE_ELEMS * 4);
    const uint32_t off = (uint32_t)pin_here((int)threadIdx.x) * 16;
#pragma unroll
    for (int u = 0; u < NB; ++u) st_coherent16(r, off, u * NT * 16, __builtin_bit_cast(uint4v, acc.c[u]));
  }
  static __device__ __forceinline__ void add_partial(Acc &acc, const float *src) {
    const BufferRsrc r = make_rsrc(src, TILE_ELEMS * 4);
    const uint32_t off = (uint32_t)pin_here((int)threadIdx.x) * 16;
    constexpr int BATCH = NB < 16 ? NB : 16;
    static_assert(NB % BATCH == 0, "whole batches");
    static_for<0, NB / BATCH>([&](auto g) {
      floatx4 x[BATCH];
#pragma unroll
      for (int u = 0; u < BATCH; ++u) x[u] = __builtin_bit_cast(floatx4, ld_coherent16(r, off, (g * BATCH + u) * NT * 16));
#pragma unroll
      for (int u = 0; u < BATCH; ++u) acc.c[g * BATCH + u] += x[u];
    });
  }
};

}  // namespace sk
