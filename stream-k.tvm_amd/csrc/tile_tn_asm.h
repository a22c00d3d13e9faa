// The four-wave 256 x 256 tiles of C[M, N] = A^T B, A [K, M], B [K, N] (see tile_tn.h for the layout's terms): the kernels of
// tile_f16_asm.h with both halves of a stage in the [K, ..] form (gen_tile_asm.py, SK_TILE_ASM_LOOP_TN).  Rows past K read as zero
// on both sides, so any K will do that 32-bit byte offsets reach ((K - 1) ld elements below 2 GiB).
// 8 experts of 11008 x 4096, 8192 rows, bfloat16: 625 us, 1.18 PFLOP/s; one of 8192 x 8192, 4096 rows 1.5.  What is between them is the
// end of a tile, 9 us, every 1024 rows of K.
#pragma once
#include "tile_f16_asm.h"
#include "tile_tn.h"

namespace sk {

template <bool BF16_>
struct TileTNAsm : TileF16Asm<BF16_ ? 1 : 0, false> {
  typedef TileF16Asm<BF16_ ? 1 : 0, false> P;
  typedef TnArgs Args;
  typedef typename P::Acc Acc;

  struct Ctx {
    uint4v rsrc_a, rsrc_b;
    uint32_t voff_a, voff_a1, voff_b, voff_b1;   // of even and odd row groups
    uint32_t goff_a, goff_b, gstep_a, gstep_b, kstep_a, kstep_b;
    uint32_t lds_wave;
    uint32_t rat[8], rbt[8];
  };
  static __device__ __forceinline__ Ctx make_ctx(const Args &a, int pm, int pn) {
    Ctx c;
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), wm = wave >> 1, wn = wave & 1;
    const int cols_a = min(P::BM, a.width_a - pm * P::BM), cols_b = min(P::BN, a.width_b - pn * P::BN);
    c.rsrc_a = make_rsrc_words(a.A + (int64_t)pm * P::BM, (uint32_t)(((int64_t)(a.K - 1) * a.lda + cols_a) * 2));
    c.rsrc_b = make_rsrc_words(a.B + (int64_t)pn * P::BN, (uint32_t)(((int64_t)(a.K - 1) * a.ldb + cols_b) * 2));
    // as the NN form's B in tile_f16_asm.h: row group g = wave + 4 x holds K-rows 2 g, 2 g + 1, piece p of row k at position
    // p ^ 4 (k & 3) ^ 2 ((k >> 3) & 1)
    const int row_in = lane >> 5, k_bits = 2 * wave + row_in;
    const int piece0 = (lane & 31) ^ (4 * (k_bits & 3)), piece1 = piece0 ^ 2;
    c.voff_a = piece0 * 8 < cols_a ? (uint32_t)(row_in * a.lda + piece0 * 8) * 2 : OOB_OFFSET;
    c.voff_a1 = piece1 * 8 < cols_a ? (uint32_t)(row_in * a.lda + piece1 * 8) * 2 : OOB_OFFSET;
    c.voff_b = piece0 * 8 < cols_b ? (uint32_t)(row_in * a.ldb + piece0 * 8) * 2 : OOB_OFFSET;
    c.voff_b1 = piece1 * 8 < cols_b ? (uint32_t)(row_in * a.ldb + piece1 * 8) * 2 : OOB_OFFSET;
    c.kstep_a = (uint32_t)(128 * a.lda);   // 64 K-rows
    c.kstep_b = (uint32_t)(128 * a.ldb);
    c.goff_a = (uint32_t)(wave * 4 * a.lda);
    c.goff_b = (uint32_t)(wave * 4 * a.ldb);
    c.gstep_a = (uint32_t)(16 * a.lda);
    c.gstep_b = (uint32_t)(16 * a.ldb);
    const uint32_t base = lds_address(P::lds());
    c.lds_wave = base + wave * 1024;
    const int k_lane = 8 * (lane >> 4) + ((lane & 15) >> 2), swz = (4 * (k_lane & 3)) ^ (2 * ((k_lane >> 3) & 1));
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int col_a = wm * P::WTM + j * 16 + 4 * (lane & 3), col_b = wn * P::WTN + j * 16 + 4 * (lane & 3);
      c.rat[j] = base + (uint32_t)(k_lane * 512 + (((col_a >> 3) ^ swz) * 16) + (col_a & 7) * 2);
      c.rbt[j] = base + P::A_BYTES + (uint32_t)(k_lane * 512 + (((col_b >> 3) ^ swz) * 16) + (col_b & 7) * 2);
    }
    return c;
  }
  template <bool EARLY_ONLY>
  static __device__ __forceinline__ void stage_loads(const Ctx &c, int stage, int n) {
    const uint32_t oob = stage < n ? 0u : OOB_OFFSET;
    const uint32_t voa = c.voff_a | oob, voa1 = c.voff_a1 | oob, vob = c.voff_b | oob, vob1 = c.voff_b1 | oob;
    const uint32_t ga = c.goff_a + (uint32_t)stage * c.kstep_a, gb = c.goff_b + (uint32_t)stage * c.kstep_b;
    const uint32_t lds_stage = c.lds_wave + (uint32_t)stage * P::STAGE_BYTES;
#define SK_ASM_TN_LOAD_OPERANDS                                                                                              \
  : : [rsa] "s"(c.rsrc_a), [rsb] "s"(c.rsrc_b), [voa] "v"(voa), [voa1] "v"(voa1), [vob] "v"(vob), [vob1] "v"(vob1), [ga] "s"(ga), \
      [gb] "s"(gb), [gas] "s"(c.gstep_a), [gbs] "s"(c.gstep_b), [lds] "s"(lds_stage)                                          \
  : "memory", "m0", "scc", "s83"
    if constexpr (EARLY_ONLY) {
      asm volatile(SK_TILE_ASM_LOADS_EARLY_TN SK_ASM_TN_LOAD_OPERANDS);
    } else {
      asm volatile(SK_TILE_ASM_LOADS_TN SK_ASM_TN_LOAD_OPERANDS);
    }
#undef SK_ASM_TN_LOAD_OPERANDS
  }
  static __device__ __forceinline__ void prefetch_first_stage(const Args &a, int pm, int pn, int, int n) {
    const Ctx c = make_ctx(a, pm, pn);
    stage_loads<false>(c, 0, n);
  }
  // all n > 0 iterations of a tile (k0 is 0)
  static __device__ __forceinline__ void mac(const Args &a, Acc &, int pm, int pn, int, int n, char *, bool first_stage_requested = false) {
    Ctx c = make_ctx(a, pm, pn);
    if (!first_stage_requested) stage_loads<false>(c, 0, n);
    stage_loads<true>(c, 1, n);   // (directly ahead of the loop, whose first wait counts on these being the youngest operations)
    const uint32_t iters = (uint32_t)n;
#define SK_ASM_TN_OPERANDS                                                                                                 \
  : [rat0] "+v"(c.rat[0]), [rat1] "+v"(c.rat[1]), [rat2] "+v"(c.rat[2]), [rat3] "+v"(c.rat[3]), [rat4] "+v"(c.rat[4]),       \
    [rat5] "+v"(c.rat[5]), [rat6] "+v"(c.rat[6]), [rat7] "+v"(c.rat[7]), [rbt0] "+v"(c.rbt[0]), [rbt1] "+v"(c.rbt[1]),       \
    [rbt2] "+v"(c.rbt[2]), [rbt3] "+v"(c.rbt[3]), [rbt4] "+v"(c.rbt[4]), [rbt5] "+v"(c.rbt[5]), [rbt6] "+v"(c.rbt[6]),       \
    [rbt7] "+v"(c.rbt[7])                                                                                                  \
  : [rsa] "s"(c.rsrc_a), [rsb] "s"(c.rsrc_b), [voa] "v"(c.voff_a), [voa1] "v"(c.voff_a1), [vob] "v"(c.voff_b),               \
    [vob1] "v"(c.voff_b1), [ga0] "s"(c.goff_a), [gb0] "s"(c.goff_b), [gas] "s"(c.gstep_a), [gas4] "s"(4 * c.gstep_a),        \
    [gbs] "s"(c.gstep_b), [gbs4] "s"(4 * c.gstep_b), [kas] "s"(c.kstep_a), [kbs] "s"(c.kstep_b), [n] "s"(iters),             \
    [lds] "s"(c.lds_wave)                                                                                                  \
  : "memory", "m0", "scc", SK_TILE_ASM_CLOBBERS
    if constexpr (BF16_) {
      asm volatile(SK_TILE_ASM_LOOP_TN("v_mfma_f32_16x16x32_bf16") SK_ASM_TN_OPERANDS);
    } else {
      asm volatile(SK_TILE_ASM_LOOP_TN("v_mfma_f32_16x16x32_f16") SK_ASM_TN_OPERANDS);
    }
#undef SK_ASM_TN_OPERANDS
    __syncthreads();   // (see TileF16Asm::mac)
  }
};

}  // namespace sk
