// Products of microscaled 4-bit operands (rows of e2m1 pairs, a power of two for each 32 of K) on tiles whose waves stream K on their own:
//   C[m][n] = sum over blocks b of 2^(sa[m][b] + sb[n][b] - 254) sum over the block's 32 k of A[m][k] B[n][k]
// v_mfma_scale_f32_16x16x128_f8f6f4 takes both scales with the operands: lane (i, g) has 32 values of row i -- one block -- in 16 bytes and
// the block's exponent in a byte of a register.  Which block of a chunk that is does not matter as long as both operands agree: lane group g
// takes blocks 2 g (step 0) and 2 g + 1 (step 1) of a chunk's eight, so that its two exponents are neighbours in memory.
//
// The rings, the order of loads, reads and refills, the sums over the waves and the end are those of tile_wavek.h.  Here a ring's unit is a
// block of 16 rows: two loads of 8 rows x 128 bytes, 256 values a row, and one of a row's exponents, two bytes to a lane (64 x 4 bytes of
// LDS).  What bounds it with few rows is the weights' way from memory, with many what a CU takes in.
#pragma once
#include "tile_wavek.h"

namespace sk {

struct MxArgs : WaveKArgs {      // (K, lda, ldb in pairs of bytes, four values)
  const uint8_t *sa, *sb;        // exponents of A's rows and of the weights'
  int pitch_a, pitch_b;          // bytes from row to row
};

template <bool BF16_, int FM_, int FN_>
struct TileWaveKMx : WaveKTile<BF16_ ? WK_BF16 : WK_F16, FM_, FN_> {
  typedef WaveKTile<BF16_ ? WK_BF16 : WK_F16, FM_, FN_> Base;
  typedef MxArgs Args;
  typedef typename Base::Acc Acc;
  typedef typename Base::AccV AccV;
  typedef int intx4 __attribute__((ext_vector_type(4)));
  typedef int intx8 __attribute__((ext_vector_type(8)));
  static constexpr int FM = FM_, FN = FN_, BM = Base::BM, BN = Base::BN, WAVES = Base::WAVES, NT = Base::NT, NB = Base::NB;
  static constexpr int KV = 64, BK = KV * WAVES;      // pairs of bytes: of a chunk, of an iteration
  static constexpr int L = FM + FN, LOADS = 3;        // blocks of a chunk, loads of a block
  static constexpr int MOST = 17;                     // blocks that a wave's quarter of the LDS holds
  static constexpr int R = L > MOST / 2 ? MOST : (4 * L < MOST ? 4 * L : MOST / L * L), S = R / L, PART = R % L;
  static_assert(S >= 1, "a chunk fits the ring");
  static constexpr int EXPONENTS = R * 2048, RING = R * (2048 + 256), LDS_BYTES = WAVES * RING, LDS_TOTAL = LDS_BYTES;
  static_assert(LDS_BYTES <= 160 * 1024, "LDS of a CU");
  static constexpr int CTAS_PER_CU = 1, WAVES_PER_EU = 1;
  static constexpr int NMFMA = 2 * NB;                // of a chunk
  static constexpr int H = NB, HR = H - (H + 3) / 4;  // of a phase, of those that have fragments read beside them
  static_assert(LOADS * ((S - 1) * L + PART) < 64, "the wait counter's range");

  // the loads of a chunk behind which `left` more chunks of the segment follow (the last PART blocks of a segment fetch nothing)
  static __device__ __forceinline__ void wait_chunk(int left) {
    if (left >= S - 1) wavek_wait_loads<LOADS *(R - L)>();
    else if (left == 0) wavek_wait_loads<LOADS * PART>();
    else if (left == 1) wavek_wait_loads<LOADS *(L + PART)>();
    else wavek_wait_loads<LOADS *(2 * L + PART)>();
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
    const uint4v rsrc_ea = uniform_rsrc(make_rsrc_words(a.sa + (int64_t)pm * BM * a.pitch_a, (uint32_t)rows_a * a.pitch_a));
    const uint4v rsrc_eb = uniform_rsrc(make_rsrc_words(a.sb + (int64_t)pn * BN * a.pitch_b, (uint32_t)rows_b * a.pitch_b));
    // load e of a block: its rows 8 e .. 8 e + 7, lane's row lane / 8, piece p (16 bytes, 32 values) of row r of a block at position
    // p ^ ((r >> 1) & 7); exponents: lane (i, g) those of pieces 2 g and 2 g + 1 of row i
    const int row8 = lane >> 3, fi = lane & 15, fg = lane >> 4;
    // (the block is in the uniform part of the address)
    uint32_t off_a[2], off_b[2];
    int kp[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      kp[e] = ((lane & 7) ^ (4 * e + (row8 >> 1))) * 8;
      off_a[e] = (uint32_t)(8 * e + row8) * lda_bytes + (uint32_t)kp[e] * 2;
      off_b[e] = (uint32_t)(8 * e + row8) * ldb_bytes + (uint32_t)kp[e] * 2;
    }
    const uint32_t off_ea = (uint32_t)(fi * a.pitch_a + 2 * fg), off_eb = (uint32_t)(fi * a.pitch_b + 2 * fg);
    const uint32_t ring = (uint32_t)__builtin_amdgcn_readfirstlane((int)lds_address(smem) + wave * RING);
    // one row of tiles: see rotation_of.  Several: the CTAs of an XCD share A as well as the weights and stay on the same K
    const int rot = a.M <= BM ? rotation_of(pn, n) : Base::start_of(a, pn, n);
    // a chunk that starts kbytes into the rows and `left` pairs of bytes before K's end, pos: where it starts in the ring, in blocks.
    // (Pieces past K fetch nothing: zeros arrive and the wait counts stay exact.)
    struct Chunk {
      uint32_t kbytes;
      int left, pos;
      uint32_t base, base_e;   // LDS addresses of block 0, were the ring long enough
    };
    auto chunk = [&](int t, int pos) {
      const int kk = ((k0 + rotated_iteration(t, rot, n)) * WAVES + wave) * KV, left = t < n ? a.K - kk : 0;
      // (a chunk past K or past the segment must not carry its offset either)
      const uint32_t kbytes = (uint32_t)__builtin_amdgcn_readfirstlane(left > 0 ? kk * 2 : 0);
      return Chunk{kbytes, left, pos, ring + (uint32_t)pos * 2048, ring + EXPONENTS + (uint32_t)pos * 256};
    };
    auto issue = [&](auto li, const Chunk &q) {
      constexpr int l = decltype(li)::value;
      uint32_t base = q.base, base_e = q.base_e;
      if (R % L != 0 && q.pos >= R - l) {
        base -= R * 2048;
        base_e -= R * 256;
      }
      const bool whole = q.left >= KV;
      constexpr bool A = l < FM;
      const uint32_t rows = q.kbytes + (A ? l * 16 * lda_bytes : (l - FM) * 16 * ldb_bytes);
      const uint32_t rows_e = q.kbytes / 16 + (A ? l * 16 * (uint32_t)a.pitch_a : (l - FM) * 16 * (uint32_t)a.pitch_b);
      wavek_dma_16<l * 2048>(A ? rsrc_a : rsrc_b, base, whole || kp[0] < q.left ? (A ? off_a : off_b)[0] : OOB_OFFSET, rows);
      wavek_dma_16<l * 2048 + 1024>(A ? rsrc_a : rsrc_b, base, whole || kp[1] < q.left ? (A ? off_a : off_b)[1] : OOB_OFFSET, rows);
      wavek_dma_2<l * 256>(A ? rsrc_ea : rsrc_eb, base_e, whole || 16 * fg < q.left ? (A ? off_ea : off_eb) : OOB_OFFSET, rows_e);
    };
#pragma unroll
    for (int t = 0; t < S; ++t)
      if (t < n) {
        const Chunk q = chunk(t, t * L);
        static_for<0, L>([&](auto l) { issue(l, q); });
      }
    {
      const Chunk q = chunk(S, S * L);
      static_for<0, PART>([&](auto l) { issue(l, q); });
    }

    // fragments: lane (i, g) takes piece 2 g + s of its row for step s
    const char *mine = smem + wave * RING;
    const char *rd0 = mine + fi * 128 + ((2 * fg) ^ ((fi >> 1) & 7)) * 16, *rd1 = mine + fi * 128 + ((2 * fg + 1) ^ ((fi >> 1) & 7)) * 16;
    const char *rd_e = mine + EXPONENTS + lane * 4;
    constexpr int READS = LOADS * L;
    // read r of a chunk: the fragments of step 0 and the exponents, block by block, then the fragments of step 1
    auto read = [&](auto ri, Frags &f, int pos) {
      constexpr int r = decltype(ri)::value, what = r < 2 * L ? r % 2 : 2, b = r < 2 * L ? r / 2 : r - 2 * L;
      int p = pos;
      if (R % L != 0 && pos >= R - b) p -= R;
      if constexpr (what == 1) f.e[b] = *reinterpret_cast<const int *>(rd_e + p * 256 + b * 256);
      else f.v[b][what / 2] = *reinterpret_cast<const intx4 *>((what ? rd1 : rd0) + p * 2048 + b * 2048);
    };
    int pos = 0;   // of the chunk that is read next
    auto advance = [&] {
      pos += L;
      if (pos >= R) pos -= R;
    };
    // the place of the chunk just read (t) takes the rest of chunk t + S and the first PART blocks of chunk t + S + 1
    Chunk q0, q1;
    auto refill_begin = [&](int t) {
      int p = pos + S * L;
      if (p >= R) p -= R;
      q0 = chunk(t + S, p);
      p += L;
      if (p >= R) p -= R;
      if (PART > 0) q1 = chunk(t + S + 1, p);
    };
    auto refill = [&](auto xi) {
      constexpr int x = decltype(xi)::value;
      if constexpr (x < L - PART) issue(std::integral_constant<int, x + PART>{}, q0);
      else issue(std::integral_constant<int, x - (L - PART)>{}, q1);
    };
    // X: fragments of chunk t, Y: of chunk t + 1, read while the first half of chunk t is multiplied; their place is refilled
    // during the second half
    auto body = [&](int t, const Frags &x, Frags &y) {
      if (t + 1 < n) {
        wait_chunk(n - 2 - t);
        static_for<0, H>([&](auto m) {
          mfma<m>(c, x);
          // (none beside the last MFMAs: they are waited for behind those)
          static_for<(m * READS / HR < READS ? m * READS / HR : READS), ((m + 1) * READS / HR < READS ? (m + 1) * READS / HR : READS)>([&](auto r) { read(r, y, pos); });
          __builtin_amdgcn_sched_barrier(0);
        });
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      } else {
        static_for<0, H>([&](auto m) { mfma<m>(c, x); });
      }
      if (t + 1 + S < n) {
        refill_begin(t + 1);
        static_for<0, NMFMA - H>([&](auto m) {
          mfma<H + m>(c, x);
          static_for<m * L / (NMFMA - H), (m + 1) * L / (NMFMA - H)>([&](auto l) { refill(l); });
          __builtin_amdgcn_sched_barrier(0);
        });
      } else {
        static_for<H, NMFMA>([&](auto m) { mfma<m>(c, x); });
      }
      advance();
    };
    Frags x, y;
    wait_chunk(n - 1);
    static_for<0, READS>([&](auto r) { read(r, x, pos); });
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    if (S < n) {
      refill_begin(0);
      static_for<0, L>([&](auto l) { refill(l); });
    }
    advance();
    for (int t = 0;;) {
      body(t, x, y);
      if (++t == n) break;
      body(t, y, x);
      if (++t == n) break;
    }
    wavek_wait_loads<0>();   // the loads past the segment write LDS too
    Base::template add_waves<RING>(c, acc, smem);
  }
};

}  // namespace sk
