// Products of microscaled 4-bit operands (rows of e2m1 pairs, a power of two for each 32 of K) on tiles whose waves stream K on their own:
//   C[m][n] = sum over blocks b of 2^(sa[m][b] + sb[n][b] - 254) sum over the block's 32 k of A[m][k] B[n][k]
// v_mfma_scale_f32_16x16x128_f8f6f4 takes both scales with the operands: lane (i, g) has 32 values of row i -- one block -- in 16 bytes and
// the block's exponent in a byte of a register.  Which block of a chunk that is does not matter as long as both operands agree: a lane group
// takes blocks 2 g (step 0) and 2 g + 1 (step 1) of a chunk's eight (mx_group), so that its two exponents are neighbours in memory.
//
// The rings, the order of loads, reads and refills, the sums over the waves and the end are those of tile_wavek.h.  A wave takes two
// neighbouring chunks of 256 values of an iteration's eight, and fetches their exponents together, 16 bytes to a row.  (Two bytes to
// a lane with every 16 rows: 12 more loads beside the 32 of a 64 x 64 tile's two chunks, 1024 x 8192 x 8192 114 us and, without any exponents
// but wrong, 78.)  What bounds it with few rows is the weights' way from memory, with many what a CU takes in.
#pragma once
#include "tile_wavek.h"

namespace sk {

// Exponents come 16 bytes to a row, for 512 values of K (two chunks): those of row r and pair of chunks q stand at r * pitch + q * step --
// rows as they are, K / 32 bytes apart, and 16 from pair to pair; or tiled, 16 bytes from row to row and all rows of a pair together, with zeros
// behind K.  Descriptors reach to the array's end: a row behind the tile's brings numbers or NaN to rows and columns that are not stored.
struct MxExponents {
  const uint8_t *at, *end;
  int pitch, step;
  __device__ __forceinline__ MxExponents row(int64_t r) const { return MxExponents{at + r * pitch, end, pitch, step}; }
  // from the word that it begins in to the word that the array ends in; loads take whole words
  __device__ __forceinline__ uint4v rsrc() const {
    const uint8_t *from = at - shift();
    const int64_t n = (end - from + 3) & ~(int64_t)3;
    return make_rsrc_words(from, (uint32_t)(n > 0x7ffffffc ? 0x7ffffffc : n));
  }
  __device__ __forceinline__ int shift() const { return (int)(reinterpret_cast<uintptr_t>(at) & 3); }
};
// The pair of a chunk's pieces that lane group l / 16 takes, 2 g and 2 g + 1.  The 16 lanes that the LDS serves together in a 16-byte read are
// rows 0-3 and 12-15 of one group and rows 4-11 of the next; pieces of groups 0 and 1, and 2 and 3, that differ in two bits of their
// position keep these apart, pairs in the groups' order do not (half the cycles of the reads were conflicts).
__device__ __forceinline__ int mx_group(int lane) { return (3 * (lane >> 4)) & 3; }
struct MxArgs : WaveKArgs {      // (K, lda, ldb in pairs of bytes, four values)
  MxExponents ea, eb;            // of A's rows and of the weights'
};

// WORDS: rows of exponents begin at words (K a multiple of 128, or tiled).  Others are fetched from the word that they begin in, 16 bytes for each
// chunk, and read at their bytes: 3 to 9 % slower than two chunks' in one load, and rows that are laid out anew first cost 7 us and more.
template <bool BF16_, int FM_, int FN_, int CTAS_, bool WORDS>
struct TileWaveKMx : WaveKTile<BF16_ ? WK_BF16 : WK_F16, FM_, FN_> {
  typedef WaveKTile<BF16_ ? WK_BF16 : WK_F16, FM_, FN_> Base;
  typedef MxArgs Args;
  typedef typename Base::Acc Acc;
  typedef typename Base::AccV AccV;
  typedef int intx4 __attribute__((ext_vector_type(4)));
  typedef int intx8 __attribute__((ext_vector_type(8)));
  static constexpr int FM = FM_, FN = FN_, BM = Base::BM, BN = Base::BN, WAVES = Base::WAVES, NT = Base::NT, NB = Base::NB;
  static constexpr int KV = 64, BK = 2 * KV * WAVES;  // pairs of bytes: of a chunk, of an iteration
  static constexpr int L = FM + FN;                   // blocks of a chunk, of two loads each
  static constexpr int CHUNK = L * 2048, EXPS = 2 * 1024, PAIR = WORDS ? EXPS : 2 * EXPS;   // bytes: of a chunk, of exponents in one load and of two chunks (64 rows of A and of the weights)
  static constexpr int MOST = 40 * 1024 / CTAS_;      // a wave's share of the LDS
  static constexpr int S = (MOST - 2 * PAIR) / CHUNK >= 3 ? 3 : (MOST - 2 * PAIR) / CHUNK, PAIRS = 2;   // chunks, pairs in the ring
  static constexpr int EXPONENTS = S * CHUNK, RING = EXPONENTS + PAIRS * PAIR, LDS_BYTES = WAVES * RING, LDS_TOTAL = LDS_BYTES;
  static_assert(RING <= MOST, "LDS of a CU");
  static constexpr int CTAS_PER_CU = CTAS_, WAVES_PER_EU = CTAS_, CUT_COST = 3;
  static constexpr int NMFMA = 2 * NB;                // of a chunk
  static constexpr int H = NB, HR = H == 1 ? 1 : H - (H + 3) / 4;  // of a phase, of those that have fragments read beside them

  // loads of a chunk of this parity, and of the `behind` chunks that follow one of parity P
  static constexpr int loads(int parity) { return 2 * L + (parity == 0 ? (WORDS ? 2 : 4) : 0); }
  static constexpr int loads_behind(int P, int behind) { return behind == 0 ? 0 : loads_behind(P, behind - 1) + loads((P + behind) & 1); }
  // a chunk of parity P behind which `left` more chunks of the segment follow
  template <int P>
  static __device__ __forceinline__ void wait_chunk(int left) {
    if (left >= S - 1) wavek_wait_loads<loads_behind(P, S - 1)>();
    else if (left == 0) wavek_wait_loads<0>();
    else wavek_wait_loads<loads_behind(P, 1)>();
  }
  struct Frags {
    intx4 v[L][2];   // [step]; A's blocks, then the weights'
    int e[L];        // exponents: byte `step`
  };
  // MFMA m of a chunk
  template <int m>
  static __device__ __forceinline__ void mfma(AccV (&c)[NB], const Frags &f) {
    constexpr int v = m % NB, s = m / NB, i = v / FN, j = FM + v % FN;
    const intx8 b = __builtin_shufflevector(f.v[j][s], f.v[j][s], 0, 1, 2, 3, -1, -1, -1, -1);
    const intx8 a = __builtin_shufflevector(f.v[i][s], f.v[i][s], 0, 1, 2, 3, -1, -1, -1, -1);
    c[v] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(b, a, c[v], 4, 4, s, f.e[j], s, f.e[i]);   // (4: e2m1)
  }

  static __device__ __forceinline__ void mac(const Args &a, Acc &acc, int pm, int pn, int k0, int n, char *smem) {
    const int lane = threadIdx.x & 63, wave = Base::wave_id();
    AccV c[NB];
    static_for<0, NB>([&](auto v) { c[v] = AccV{0, 0, 0, 0}; });
    // ---- descriptors: rows past M / N read as zero ----
    const uint32_t lda_bytes = (uint32_t)a.lda * 2, ldb_bytes = (uint32_t)a.ldb * 2;
    const int rows_a = min(BM, a.M - pm * BM), rows_b = min(BN, a.N - pn * BN);
    const uint4v rsrc_a = uniform_rsrc(make_rsrc_words(a.A + (int64_t)pm * BM * a.lda, (uint32_t)rows_a * lda_bytes));
    const uint4v rsrc_b = uniform_rsrc(make_rsrc_words(a.B + (int64_t)pn * BN * a.ldb, (uint32_t)rows_b * ldb_bytes));
    const uint4v rsrc_ea = uniform_rsrc(a.ea.row((int64_t)pm * BM).rsrc()), rsrc_eb = uniform_rsrc(a.eb.row((int64_t)pn * BN).rsrc());
    // load e of a block: its rows 8 e .. 8 e + 7, lane's row lane / 8, piece p (16 bytes, 32 values) of row r of a block at position
    // p ^ ((r >> 1) & 7); exponents: lane's row, 16 bytes
    const int row8 = lane >> 3, fi = lane & 15, fg = mx_group(lane);
    uint32_t off_a[2], off_b[2];
    int kp[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      kp[e] = ((lane & 7) ^ (4 * e + (row8 >> 1))) * 8;
      off_a[e] = (uint32_t)(8 * e + row8) * lda_bytes + (uint32_t)kp[e] * 2;
      off_b[e] = (uint32_t)(8 * e + row8) * ldb_bytes + (uint32_t)kp[e] * 2;
    }
    // (from the word that they begin in)
    const int shift_a = WORDS ? 0 : a.ea.row((int64_t)pm * BM).shift(), shift_b = WORDS ? 0 : a.eb.row((int64_t)pn * BN).shift();
    const uint32_t off_ea = lane < BM ? (uint32_t)(shift_a + lane * a.ea.pitch) & (WORDS ? ~0u : ~3u) : OOB_OFFSET;
    const uint32_t off_eb = lane < BN ? (uint32_t)(shift_b + lane * a.eb.pitch) & (WORDS ? ~0u : ~3u) : OOB_OFFSET;
    const uint32_t ring = (uint32_t)__builtin_amdgcn_readfirstlane((int)lds_address(smem) + wave * RING);
    // one row of tiles: see rotation_of.  Several: the CTAs of an XCD share A as well as the weights and stay on the same K
    const int rot = a.M <= BM ? rotation_of(pn, n) : Base::start_of(a, pn, n);
    const int chunks = 2 * n;
    // a chunk that starts kbytes into the rows and `left` pairs of bytes before K's end.  (Pieces past K fetch nothing: zeros arrive and
    // the wait counts stay exact; a chunk past K or past the segment must not carry its offset either.)
    auto left_of = [&](int t) { return t < chunks ? a.K - (((k0 + rotated_iteration(t >> 1, rot, n)) * WAVES + wave) * 2 + (t & 1)) * KV : 0; };
    struct Chunk {
      uint32_t kbytes, base, pair;   // base, pair: LDS addresses
      int left;
    };
    auto chunk = [&](int t, int slot, int pair) {
      const int left = left_of(t);
      const uint32_t kbytes = (uint32_t)__builtin_amdgcn_readfirstlane(left > 0 ? (a.K - left) * 2 : 0);
      return Chunk{kbytes, ring + (uint32_t)slot * CHUNK, ring + EXPONENTS + (uint32_t)pair * PAIR, left};
    };
    auto issue = [&](auto li, const Chunk &q) {
      constexpr int l = decltype(li)::value;
      constexpr bool A = l < FM;
      const bool whole = q.left >= KV;
      const uint32_t rows = q.kbytes + (A ? l * 16 * lda_bytes : (l - FM) * 16 * ldb_bytes);
      wavek_dma_16<l * 2048>(A ? rsrc_a : rsrc_b, q.base, whole || kp[0] < q.left ? (A ? off_a : off_b)[0] : OOB_OFFSET, rows);
      wavek_dma_16<l * 2048 + 1024>(A ? rsrc_a : rsrc_b, q.base, whole || kp[1] < q.left ? (A ? off_a : off_b)[1] : OOB_OFFSET, rows);
    };
    // (the exponents of a row's end and of what lies behind it arrive together; see read_exponents.  WORDS: of the pair that a chunk is in)
    auto issue_exponents = [&](const Chunk &q) {
      const int at = __builtin_amdgcn_readfirstlane((int)q.kbytes / (WORDS ? 256 : 128)), to = __builtin_amdgcn_readfirstlane((int)q.pair);
      const int at_a = WORDS ? at * a.ea.step : at * 8, at_b = WORDS ? at * a.eb.step : at * 8;
      wavek_dma_16<0>(rsrc_ea, (uint32_t)to, q.left > 0 ? off_ea : OOB_OFFSET, (uint32_t)at_a);
      wavek_dma_16<1024>(rsrc_eb, (uint32_t)to, q.left > 0 ? off_eb : OOB_OFFSET, (uint32_t)at_b);
      if constexpr (WORDS) return;
      wavek_dma_16<EXPS>(rsrc_ea, (uint32_t)to, q.left > 0 ? off_ea : OOB_OFFSET, (uint32_t)(at_a + 8));
      wavek_dma_16<EXPS + 1024>(rsrc_eb, (uint32_t)to, q.left > 0 ? off_eb : OOB_OFFSET, (uint32_t)(at_b + 8));
    };
#pragma unroll
    for (int t = 0; t < S; ++t)
      if (t < chunks) {
        const Chunk q = chunk(t, t, t >> 1);
        if (t % 2 == 0) issue_exponents(q);
        static_for<0, L>([&](auto l) { issue(l, q); });
      }

    // fragments: lane (i, g) takes piece 2 g + s of its row for step s
    const char *mine = smem + wave * RING;
    const char *rd0 = mine + fi * 128 + ((2 * fg) ^ ((fi >> 1) & 7)) * 16, *rd1 = mine + fi * 128 + ((2 * fg + 1) ^ ((fi >> 1) & 7)) * 16;
    struct __attribute__((packed, aligned(WORDS ? 2 : 1))) Two { uint16_t e; };
    const char *rd_ea = mine + EXPONENTS + fi * 16 + 2 * fg + (WORDS ? 0 : (shift_a + fi * a.ea.pitch) & 3);   // (the same for row fi + 16, ..)
    const char *rd_eb = mine + EXPONENTS + 1024 + fi * 16 + 2 * fg + (WORDS ? 0 : (shift_b + fi * a.eb.pitch) & 3);
    constexpr int READS = 3 * L;
    int slot = 0, pair = 0;   // of the chunk that is read next
    // read r of a chunk of parity P: the fragments of step 0 and the exponents, block by block, then the fragments of step 1
    auto read = [&](auto ri, auto parity, Frags &f) {
      constexpr int r = decltype(ri)::value, what = r < 2 * L ? r % 2 : 2, b = r < 2 * L ? r / 2 : r - 2 * L;
      if constexpr (what == 1) f.e[b] = reinterpret_cast<const Two *>((b < FM ? rd_ea : rd_eb) + pair * PAIR + (b < FM ? b : b - FM) * 256 + (WORDS ? 8 : EXPS) * decltype(parity)::value)->e;
      else f.v[b][what / 2] = *reinterpret_cast<const intx4 *>((what ? rd1 : rd0) + slot * CHUNK + b * 2048);
    };
    // the last chunk of K: blocks behind K are zeros, and their exponents, which are another row's, have to be numbers
    auto mask_exponents = [&](int left, Frags &f) {
      const int mask = (16 * fg < left ? 0xff : 0) | (16 * fg + 8 < left ? 0xff00 : 0);
#pragma unroll
      for (int b = 0; b < L; ++b) f.e[b] &= mask;
    };
    // X: fragments of chunk t (parity P), Y: of chunk t + 1, read while the first half of chunk t is multiplied; their place is refilled
    // during the second half with chunk t + 1 + S.  REFILL: it is requested; MORE: there is a chunk t + 1.  (The loops below say which: with the
    // choice inside, the compiler moves the accumulators between its register files for every MFMA.)
    auto body = [&](int t, auto parity, auto refill, auto more, const Frags &x, Frags &y) {
      constexpr int P = decltype(parity)::value;
      constexpr bool REFILL = decltype(refill)::value, MORE = decltype(more)::value, FIRST = ((P + 1 + S) & 1) == 0;
      if constexpr (REFILL) wavek_wait_loads<loads_behind(1 - P, S - 1)>();
      else if constexpr (MORE) wait_chunk<1 - P>(chunks - 2 - t);
      static_for<0, H>([&](auto m) {
        mfma<m>(c, x);
        // (none beside the last MFMAs: they are waited for behind those)
        if constexpr (MORE)
          static_for<(m * READS / HR < READS ? m * READS / HR : READS), ((m + 1) * READS / HR < READS ? (m + 1) * READS / HR : READS)>(
              [&](auto r) { read(r, std::integral_constant<int, 1 - P>{}, y); });
        __builtin_amdgcn_sched_barrier(0);
      });
      if constexpr (MORE) {
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        mask_exponents(left_of(t + 1), y);
      }
      Chunk q;
      if constexpr (REFILL) {   // (chunk t + 1 is of the pair `pair`)
        q = chunk(t + 1 + S, slot, P == 1 ? (pair + S / 2) % PAIRS : (pair + 1 + S / 2) % PAIRS);
        if constexpr (FIRST) issue_exponents(q);
      }
      static_for<0, NMFMA - H>([&](auto m) {
        mfma<H + m>(c, x);
        if constexpr (REFILL) static_for<m * L / (NMFMA - H), (m + 1) * L / (NMFMA - H)>([&](auto l) { issue(l, q); });
        __builtin_amdgcn_sched_barrier(0);
      });
      slot = slot + 1 == S ? 0 : slot + 1;
      if constexpr (P == 0) pair ^= 1;   // (chunk t + 2 begins the next pair)
    };
    Frags x, y;
    constexpr std::integral_constant<int, 0> even;
    constexpr std::integral_constant<int, 1> odd;
    wait_chunk<0>(chunks - 1);
    static_for<0, READS>([&](auto r) { read(r, even, x); });
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    mask_exponents(left_of(0), x);
    if (S < chunks) {
      const Chunk q = chunk(S, 0, S / 2 % PAIRS);
      if constexpr (S % 2 == 0) issue_exponents(q);
      static_for<0, L>([&](auto l) { issue(l, q); });
    }
    slot = S > 1 ? 1 : 0;
    constexpr std::true_type yes;
    constexpr std::false_type no;
    int t = 0;
    for (; t + 2 + S < chunks; t += 2) {
      body(t, even, yes, yes, x, y);
      body(t + 1, odd, yes, yes, y, x);
    }
    if constexpr (S % 2 == 0)
      if (t + 1 + S < chunks) {
        body(t, even, yes, yes, x, y);
        body(t + 1, odd, no, yes, y, x);
        t += 2;
      }
    for (; t + 2 < chunks; t += 2) {
      body(t, even, no, yes, x, y);
      body(t + 1, odd, no, yes, y, x);
    }
    body(t, even, no, yes, x, y);
    body(t + 1, odd, no, no, y, x);
    wavek_wait_loads<0>();
    Base::template add_waves<RING>(c, acc, smem);
  }
};

}  // namespace sk
