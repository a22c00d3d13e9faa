// The four-wave 256 x 256 tiles whose K loop is assembly (tile_f16_asm.h) for microscaled 4-bit operands (tile_mx.h has the product): an
// iteration is 256 values of K, 128 bytes a row, as in the 16-bit loop, whose loads, stages and schedule this one has; a block of 16 x 16 x 128
// takes the 16 cycles that one of 16 x 16 x 32 takes in 16 bits.  Lane group g takes chunks 2 g and 2 g + 1 of a row, so that its two exponents
// are neighbours, and exponents come 16 bytes to a row for two iterations at a time.  gen_tile_asm.py has the register plan.
//
// The exponents are tiled (MxExponents), 1 KB behind each other for a wave's load of 64 rows: as rows of K / 32 bytes they are 64 lines of the L2,
// as many as half of the operands' own, and 8192^3 takes 265 us and not 250.  Zeros from K on multiply the zeros that the last
// iteration's lanes behind K fetch.  A segment starts at an even iteration.
#pragma once
#include "tile_asm_epilogue.h"
#include "tile_mx.h"
#include "tile_mx_asm_gen.h"

namespace sk {

template <bool BF16>
struct TileMxAsm : TileF16Asm<BF16 ? 6 : 5, false> {
  typedef TileF16Asm<BF16 ? 6 : 5, false> P;
  typedef MxArgs Args;
  typedef typename P::Acc Acc;
  static constexpr int EXPONENTS_AT = 2 * P::STAGE_BYTES, PAIR_BYTES = 2 * P::BM * 16;   // of two iterations: A's rows, then the weights'
  static_assert(EXPONENTS_AT + PAIR_BYTES <= P::PATCHES_AT, "the first pair of the next segment is on its way while the patches are in use");
  static_assert(EXPONENTS_AT + 2 * PAIR_BYTES <= P::LDS_TOTAL && (EXPONENTS_AT & (2 * PAIR_BYTES - 1)) == 0, "the pairs' addresses differ in one bit");

  struct Ctx {
    uint4v rsrc_a, rsrc_b, rsrc_ea, rsrc_eb;
    uint32_t voff_a, voff_b, voff_ea, voff_e, tail;
    uint32_t goff_a, goff_b, goff_ea, goff_eb, gstep_a, gstep_b, step_ea, step_eb;
    uint32_t lds_wave, lds_e;
    uint32_t ra0, rb0, rda, rdb;   // where the lane reads fragments and exponents
  };
  // LOW: at most 128 rows, 64 to a wave (TileF16Asm::LOW_TILE): the second wave row's 64 stand where a whole tile has rows 128 ..
  template <bool LOW>
  static __device__ __forceinline__ Ctx make_ctx(const Args &a, int pm, int pn, int k0) {
    Ctx c;
    // (pinned: no address is held through the loop, which leaves the compiler 88 registers)
    const int tid = pin_here((int)threadIdx.x), lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), wm = wave >> 1, wn = wave & 1;
    const int rows_a = min(P::BM, a.M - pm * P::BM), rows_b = min(P::BN, a.N - pn * P::BN);
    // rows past the matrix edge lie beyond the descriptors' ranges and read as zero
    c.rsrc_a = make_rsrc_words(a.A + (int64_t)pm * P::BM * a.lda, (uint32_t)(rows_a * a.lda * 2));
    c.rsrc_b = make_rsrc_words(a.B + (int64_t)pn * P::BN * a.ldb, (uint32_t)(rows_b * a.ldb * 2));
    c.rsrc_ea = a.ea.row((int64_t)pm * P::BM).rsrc();
    c.rsrc_eb = a.eb.row((int64_t)pn * P::BN).rsrc();
    // (loads and swizzle as in TileF16Asm::make_ctx)
    const int my_chunk = (lane & 7) ^ (((wave & 1) << 2) | (lane >> 4)), my_row = lane >> 3;
    c.voff_a = (uint32_t)(my_row * a.lda + my_chunk * 8) * 2;
    c.voff_b = (uint32_t)(my_row * a.ldb + my_chunk * 8) * 2;
    c.tail = my_chunk * 8 < a.K - (a.K - 1) / P::BK * P::BK ? 0u : OOB_OFFSET;
    c.goff_a = (uint32_t)k0 * (P::BK * 2) + (uint32_t)(wave * 16 * a.lda);
    c.goff_b = (uint32_t)k0 * (P::BK * 2) + (uint32_t)(wave * 16 * a.ldb);
    c.gstep_a = (uint32_t)(64 * a.lda);
    c.gstep_b = (uint32_t)(64 * a.ldb);
    c.voff_e = (uint32_t)((wave * 64 + lane) * 16);
    c.voff_ea = c.voff_e - (LOW && wave >= 2 ? 64 * 16 : 0);
    c.goff_ea = (uint32_t)(k0 >> 1) * (uint32_t)a.ea.step;
    c.goff_eb = (uint32_t)(k0 >> 1) * (uint32_t)a.eb.step;
    c.step_ea = (uint32_t)a.ea.step;
    c.step_eb = (uint32_t)a.eb.step;
    const uint32_t base = lds_address(P::lds());
    c.lds_wave = base + wave * 1024;
    c.lds_e = base + EXPONENTS_AT + wave * 1024;
    // fragments: lane (r = l % 16, g = mx_group(l)) reads row r of a 16-row block, chunk 2 g + kk at position (2 g + kk) ^ ((r >> 1) & 7): K-step 1
    // is K-step 0 with address bit 4 flipped
    const int g = mx_group(lane);
    const uint32_t pos0 = (uint32_t)((2 * g) ^ ((lane >> 1) & 7)) * 16;
    c.ra0 = base + (uint32_t)(wm * P::WTM + (lane & 15)) * P::ROW_BYTES + pos0;
    c.rb0 = base + P::A_BYTES + (uint32_t)(wn * P::WTN + (lane & 15)) * P::ROW_BYTES + pos0;
    c.rda = base + EXPONENTS_AT + (uint32_t)(wm * P::WTM + (lane & 15)) * 16 + 2 * g;
    c.rdb = base + EXPONENTS_AT + P::BM * 16 + (uint32_t)(wn * P::WTN + (lane & 15)) * 16 + 2 * g;
    return c;
  }
  template <bool LOW, bool EARLY_ONLY>
  static __device__ __forceinline__ void stage_loads(const Ctx &c, int stage, int n, bool last) {
    const uint32_t oob = stage < n ? 0u : OOB_OFFSET, tail = last && stage == n - 1 ? c.tail : 0u;
    const uint32_t voa = c.voff_a | oob | tail, vob = c.voff_b | oob | tail;
    const uint32_t ga = c.goff_a + (uint32_t)stage * 128, gb = c.goff_b + (uint32_t)stage * 128, lds_stage = c.lds_wave + (uint32_t)stage * P::STAGE_BYTES;
#define SK_MX_LOAD_OPERANDS                                                                                              \
  : : [rsa] "s"(c.rsrc_a), [rsb] "s"(c.rsrc_b), [voa] "v"(voa), [vob] "v"(vob), [ga] "s"(ga), [gb] "s"(gb),               \
      [gas] "s"(c.gstep_a), [gas2] "s"(2 * c.gstep_a), [gas3] "s"(3 * c.gstep_a), [gbs] "s"(c.gstep_b),                   \
      [gbs2] "s"(2 * c.gstep_b), [gbs3] "s"(3 * c.gstep_b), [lds] "s"(lds_stage)                                          \
  : "memory", "m0", "scc", "s83"
    if constexpr (LOW && EARLY_ONLY) asm volatile(SK_TILE_ASM_LOADS_EARLY_LOW SK_MX_LOAD_OPERANDS);
    else if constexpr (LOW) asm volatile(SK_TILE_ASM_LOADS_LOW SK_MX_LOAD_OPERANDS);
    else if constexpr (EARLY_ONLY) asm volatile(SK_TILE_ASM_LOADS_EARLY SK_MX_LOAD_OPERANDS);
    else asm volatile(SK_TILE_ASM_LOADS SK_MX_LOAD_OPERANDS);
#undef SK_MX_LOAD_OPERANDS
  }
  template <bool LOW>
  static __device__ __forceinline__ void first_loads(const Ctx &c, int n, bool last) {
    dma_load_16(c.rsrc_ea, c.lds_e, c.voff_ea, c.goff_ea);
    dma_load_16(c.rsrc_eb, c.lds_e + P::BM * 16, c.voff_e, c.goff_eb);
    stage_loads<LOW, false>(c, 0, n, last);
  }
  // last: the segment ends with K
  template <bool LOW>
  static __device__ __forceinline__ void prefetch_first_stage(const Args &a, int pm, int pn, int k0, int n, bool last) {
    first_loads<LOW>(make_ctx<LOW>(a, pm, pn, k0), n, last);
  }
  template <bool LOW>
  static __device__ __forceinline__ void mac(const Args &a, int pm, int pn, int k0, int n, bool last, bool first_stage_requested) {
    Ctx c = make_ctx<LOW>(a, pm, pn, k0);
    if (!first_stage_requested) first_loads<LOW>(c, n, last);
    // (directly ahead of the loop, whose first wait counts on these being the youngest operations)
    stage_loads<LOW, true>(c, 1, n, last);
#define SK_MX_LOOP_OPERANDS(...) \
  : [ra0] "+v"(c.ra0), [rb0] "+v"(c.rb0) \
  : [rsa] "s"(c.rsrc_a), [rsb] "s"(c.rsrc_b), [rea] "s"(c.rsrc_ea), [reb] "s"(c.rsrc_eb), [voa] "v"(c.voff_a), [vob] "v"(c.voff_b), \
  [ve] "v"(c.voff_e), __VA_ARGS__ [tail] "v"(last ? c.tail : 0u), [rda] "v"(c.rda), [rdb] "v"(c.rdb), [ga0] "s"(c.goff_a), \
  [gb0] "s"(c.goff_b), [gas] "s"(c.gstep_a), [gas2] "s"(2 * c.gstep_a), [gas3] "s"(3 * c.gstep_a), [gbs] "s"(c.gstep_b), \
  [gbs2] "s"(2 * c.gstep_b), [gbs3] "s"(3 * c.gstep_b), [n] "s"((uint32_t)n), [lds] "s"(c.lds_wave), [eka] "s"(c.goff_ea + c.step_ea), \
  [ekb] "s"(c.goff_eb + c.step_eb), [esa] "s"(c.step_ea), [esb] "s"(c.step_eb), \
  [el] "s"(c.lds_e + PAIR_BYTES) \
  : "memory", "m0", "scc", SK_TILE_ASM_CLOBBERS_MX
    if constexpr (LOW) asm volatile(SK_TILE_ASM_LOOP_MX_LOW SK_MX_LOOP_OPERANDS([vea] "v"(c.voff_ea),));
    else asm volatile(SK_TILE_ASM_LOOP_MX SK_MX_LOOP_OPERANDS());
#undef SK_MX_LOOP_OPERANDS
    // every wave has left the loop and its own loads have landed: the stages are free
    __syncthreads();
  }
  // LOW: the lower half of each wave's 128 rows; the second wave row's are the tile's rows 64 .., not 128 ..: C moved back by 64
  template <bool LOW>
  static __device__ __forceinline__ void store_c(Args a, int pm, int pn, const void *epi) {
    if constexpr (LOW) {
      const int back = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 7) * (P::WTM / 2);
      a.C -= (int64_t)back * a.ldc;
      a.M += back;
    }
    if (P::direct_store_ok(a, pn, epi)) {
      P::template store_c_direct<LOW ? 0 : -1>(a, pm, pn);
      return;
    }
    const int wave = threadIdx.x >> 6, row0 = pm * P::BM + (wave >> 1) * P::WTM, col0 = pn * P::BN + (wave & 1) * P::WTN;
    by_epilogue(epi, [&](auto e) {
      AsmEnd<TileMxAsm, false, BF16, decltype(e)::value, true>::store(a.C, a.ldc, a.M, a.N, row0, col0, nullptr, nullptr, epi_bias(epi), 0, LOW ? P::FM / 2 : P::FM);
    });
  }
};

}  // namespace sk
