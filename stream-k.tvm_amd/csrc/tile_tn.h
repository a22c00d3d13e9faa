// fp16 / bfloat16 tiles of C[M, N] = A^T B with A [K, M] and B [K, N] row-major ("TN"): the gradient of a layer's weights, K being
// the rows of a batch.
//
// K runs down the columns of both operands, and an MFMA wants runs of K: a stage holds 64 rows of K of BM (A) and BN (B) columns as
// they lie in memory (direct global -> LDS loads of 16 bytes per lane, 16-byte piece c of row k at position
// c ^ 4 (k & 3) ^ 2 ((k >> 3) & 1)), and the fragments come back with ds_read_b64_tr_b16, which hands each lane four K of one column:
// two such reads make the eight K-values of a lane's operand.  Rows past K lie beyond the descriptors and read as zero, so any
// number of rows will do; columns past M / N are masked per lane (M and N as the operands' rows have them: multiples of 8).
// Two stages; the loads of an iteration are on their way while the one before is multiplied.  Batches of few rows, where the result's
// way to memory bounds it: 8 experts of 2048 x 1024, 500 rows, fp16 12 us (33 MB written).
#pragma once
#include "sk_device.h"
#include "tile_epilogue.h"
#include "tile_f16.h"

namespace sk {

// widths of the operands as they lie in memory; C has M x N (M may be cut off inside the last piece of A's rows)
struct TnArgs : GemmArgs {
  int width_a, width_b;   // columns of A and B that may be read: multiples of 8
};

template <int BM_, int BN_, int WM_, int WN_, bool BF16_>
struct TileTN {
  typedef TnArgs Args;
  static constexpr int BM = BM_, BN = BN_, BK = 64, WM = WM_, WN = WN_, NW = WM * WN, NT = 64 * NW;
  static constexpr int WTM = BM / WM, WTN = BN / WN, FM = WTM / 16, FN = WTN / 16;
  static constexpr int A_ROW = 2 * BM, B_ROW = 2 * BN, A_BYTES = BK * A_ROW, B_BYTES = BK * B_ROW, STAGE = A_BYTES + B_BYTES;
  static constexpr int LDS_BYTES = 2 * STAGE;
  static constexpr int LA = A_BYTES / 1024 / NW, LB = B_BYTES / 1024 / NW;   // loads per wave and stage
  static constexpr int CTAS_PER_CU = (160 * 1024) / LDS_BYTES > 2 ? 2 : (160 * 1024) / LDS_BYTES, WAVES_PER_EU = CTAS_PER_CU * NW / 4;
  static_assert((1024 / A_ROW * NW) % 16 == 0 && (1024 / B_ROW * NW) % 16 == 0, "the swizzle of a lane's row must not depend on the load");
  typedef BlockPatch<FM, FN> Patch;
  static_assert(NW * Patch::BYTES <= STAGE, "patches");

  struct Acc {
    floatx4 v[FM][FN];
  };

  // lane's piece of a load of rows of ROW bytes: row inside the load's group, byte offset in the row (or out of range)
  template <int ROW>
  static __device__ __forceinline__ uint32_t load_offset(int wave, int lane, int64_t ld, int cols) {
    const int row_in = (lane * 16) / ROW, pos = ((lane * 16) % ROW) / 16, k = (1024 / ROW) * wave + row_in;
    const int piece = pos ^ (4 * (k & 3)) ^ (2 * ((k >> 3) & 1));
    return piece * 8 < cols ? (uint32_t)(row_in * ld + piece * 8) * 2 : OOB_OFFSET;
  }

  static __device__ __forceinline__ void mac(const Args &a, Acc &acc, int pm, int pn, int k0, int n, char *smem) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int wm = wave / WN, wn = wave % WN;
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
      for (int j = 0; j < FN; ++j) acc.v[i][j] = floatx4{0.f, 0.f, 0.f, 0.f};
    const int cols_a = min(BM, a.width_a - pm * BM), cols_b = min(BN, a.width_b - pn * BN);
    const uint32_t voff_a = load_offset<A_ROW>(wave, lane, a.lda, cols_a), voff_b = load_offset<B_ROW>(wave, lane, a.ldb, cols_b);
    const uint32_t grp_a = (uint32_t)(1024 / A_ROW * a.lda * 2), grp_b = (uint32_t)(1024 / B_ROW * a.ldb * 2);
    const uint32_t base = lds_address(smem);
    // (the descriptors move along with K -- a batch of rows may be longer than 32-bit offsets reach -- and end with the tile's last
    // element of row K - 1)
    auto request = [&](int stage, int kt) {
      const int64_t k = (int64_t)kt * BK;
      const int last = min(BK, a.K - (int)k) - 1;
      const uint4v rsrc_a = make_rsrc_words(a.A + k * a.lda + (int64_t)pm * BM, (uint32_t)((last * a.lda + cols_a) * 2));
      const uint4v rsrc_b = make_rsrc_words(a.B + k * a.ldb + (int64_t)pn * BN, (uint32_t)((last * a.ldb + cols_b) * 2));
#pragma unroll
      for (int x = 0; x < LA; ++x) {
        const int g = wave + x * NW;
        dma_load_16(rsrc_a, base + stage * STAGE + g * 1024, voff_a, g * grp_a);
      }
#pragma unroll
      for (int x = 0; x < LB; ++x) {
        const int g = wave + x * NW;
        dma_load_16(rsrc_b, base + stage * STAGE + A_BYTES + g * 1024, voff_b, g * grp_b);
      }
    };
    // lane group g = lane / 16 takes K-rows 8 g .. 8 g + 7 of a 16-column block: rows 8 g + (lane % 16) / 4, and four further on
    const int kl = 8 * (lane >> 4) + ((lane & 15) >> 2), swz = (4 * (kl & 3)) ^ (2 * ((kl >> 3) & 1));
    int rd_a[FM], rd_b[FN];
#pragma unroll
    for (int i = 0; i < FM; ++i) {
      const int col = wm * WTM + i * 16 + 4 * (lane & 3);
      rd_a[i] = kl * A_ROW + ((col >> 3) ^ swz) * 16 + (col & 7) * 2;
    }
#pragma unroll
    for (int j = 0; j < FN; ++j) {
      const int col = wn * WTN + j * 16 + 4 * (lane & 3);
      rd_b[j] = A_BYTES + kl * B_ROW + ((col >> 3) ^ swz) * 16 + (col & 7) * 2;
    }
    typedef short short4v __attribute__((ext_vector_type(4)));
    typedef __attribute__((address_space(3))) short4v *lds_s4;
    auto fragment = [&](const char *p, int row_bytes) {
      union { short4v s[2]; half8v h; } u;
      u.s[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4)p);
      u.s[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4)(p + 4 * row_bytes));
      return u.h;
    };
    if (n > 0) request(0, k0);
    for (int it = 0; it < n; ++it) {
      // own loads of this stage have landed, then everybody's; everybody has read the other stage
      asm volatile("s_waitcnt vmcnt(0)\n\ts_barrier" ::: "memory");
      if (it + 1 < n) request((it + 1) & 1, k0 + it + 1);
      const char *st = smem + (it & 1) * STAGE;
#pragma unroll
      for (int kk = 0; kk < 2; ++kk) {
        half8v fa[FM], fb[FN];
#pragma unroll
        for (int i = 0; i < FM; ++i) fa[i] = fragment(st + rd_a[i] + kk * 32 * A_ROW, A_ROW);
#pragma unroll
        for (int j = 0; j < FN; ++j) fb[j] = fragment(st + rd_b[j] + kk * 32 * B_ROW, B_ROW);
#pragma unroll
        for (int i = 0; i < FM; ++i)
#pragma unroll
          for (int j = 0; j < FN; ++j) {
            if constexpr (BF16_) {
              typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
              acc.v[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, fb[j]), __builtin_bit_cast(bf16x8, fa[i]),
                                                                    acc.v[i][j], 0, 0, 0);
            } else {
              acc.v[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(fb[j], fa[i], acc.v[i][j], 0, 0, 0);
            }
          }
      }
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // the fragments are in registers before the next barrier
    }
    __syncthreads();
  }

  static __device__ __forceinline__ void store_c(const Args &a, const Acc &acc, int pm, int pn, char *smem, const void *) {
    const int wave = threadIdx.x >> 6, wm = wave / WN, wn = wave % WN;
    Patch::template store<0, FM>(a.C, a.ldc, a.M, a.N, pm * BM + wm * WTM, pn * BN + wn * WTN, smem + wave * Patch::BYTES,
                                 [&](auto i, auto j) { return round4<BF16_>(acc.v[i][j]); });
    __syncthreads();   // the patches overlap the stages of the next tile
  }
};

}  // namespace sk
