// Few rows to an expert: the weights of all experts that have rows as ONE stream.
//
// With up to a few dozen rows an expert's product is its weights' way from HBM.  A tile of 64 weight rows and K = 4096 is half a
// megabyte, some 20 us of a CU's share of the memory, and a kernel that fills its pipeline anew for every tile, or has 344 tiles for
// 256 CUs, loses a third of it.  Here the iterations of all tiles -- 256 K-values (int8: 512) of WN * 16 * NB weight rows -- are
// numbered through, over the experts, and every CTA takes an equal run of them (Stream-K over the groups): its ring of loads never
// drains between tiles, and all CTAs end together.
//
//  * Data movement as in tile_stream_pairs.h: four waves, WM along the rows by WN along the weights; a load instruction reads two
//    rows of 512 contiguous bytes into LDS (pairs of rows padded to 1056 bytes, the odd row's neighbouring pieces swapped); rings of
//    WD slots of weights and AD of the rows; one wait and one barrier an iteration; tiles walk K from different starts (rotation_of).
//    What is new: the loads run ahead of the arithmetic across tiles and experts, each side with a cursor of its own.
//  * A tile that one CTA has whole is stored from the accumulators.  A tile cut by the end of a CTA's run leaves fp32 sums (int8:
//    int32) in the workspace, two slots to a CTA: slot 1 for the tile whose start it has, slot 0 for the one that it enters in the
//    middle.  When its run is over a CTA adds its iterations to the tile's counter (kept at the CTA that has the tile's start); who
//    completes the count adds the sums in the order of the CTAs, which is the same on every launch, and stores.  Nobody waits for
//    another CTA.
#pragma once
#include "grouped.h"
#include "tile_scaled_i8.h"

namespace sk {

enum GroupElement { GE_F16 = 0, GE_BF16 = 1, GE_I8 = 2 };

// MB blocks of 16 rows to each of WM waves along the rows, one block of 16 weight rows to each of WN waves
template <int MB_, int WM_, int WN_, int WD_, int AD_, int TYPE_>
struct GroupStream {
  static constexpr int MB = MB_, WM = WM_, WN = WN_, WD = WD_, AD = AD_, TYPE = TYPE_, NT = 256;
  static constexpr bool I8 = TYPE_ == GE_I8, BF16 = TYPE_ == GE_BF16;
  static_assert(WM * WN == 4 && WD >= AD && AD >= 2, "four waves; the barrier of an iteration frees the slots read an iteration earlier");
  typedef int intx4 __attribute__((ext_vector_type(4)));
  typedef typename std::conditional<I8, intx4, floatx4>::type AccV;
  static constexpr int BM = 16 * MB * WM, BN = 16 * WN, BK = 256;   // (K in 16-bit units)
  static constexpr int PAIR = 1056, W_SLOT = 8 * PAIR, A_PAIRS = 8 * MB * WM, A_SLOT = A_PAIRS * PAIR;
  static constexpr int LDS_W = WN * WD * W_SLOT, LDS_BYTES = LDS_W + AD * A_SLOT;
  static_assert(LDS_BYTES <= 160 * 1024 - 64, "LDS of a CU");
  static constexpr int CTAS_PER_CU = (160 * 1024) / (LDS_BYTES + 64), WAVES_PER_EU = CTAS_PER_CU;
  static constexpr int LOADS_W = 8 / WM, LOADS_A = A_PAIRS / 4;     // per wave and iteration
  static_assert(A_PAIRS % 4 == 0, "the loads are shared out evenly");
  static constexpr int OUTSTANDING = (WD > AD ? LOADS_W : 0) + (AD - 2) * (LOADS_W + LOADS_A);   // (see tile_stream_pairs.h)
  static constexpr int SLOT_BYTES = BM * BN * 4;                    // a partial tile

  // where one side of the pipeline stands: iteration i of a tile, in the order of the tile's rotation
  struct Cursor {
    GroupWalk<BM, false> walk;
    GroupTile t;
    int tile, i, rot;
    uint4v rsrc;         // the side's operand
    __device__ __forceinline__ Cursor(const GroupedArgs &g) : walk(g.offsets, g.E, g.R, g.tiles_n) {}
    // (number of the iteration; ipt iterations to a tile)
    template <bool W>
    __device__ __forceinline__ void seek(const GroupedArgs &g, int at, int ipt) {
      tile = (int)((unsigned)at / (unsigned)ipt);
      i = at - tile * ipt;
      open<W>(g, ipt);
    }
    template <bool W>
    __device__ __forceinline__ void open(const GroupedArgs &g, int ipt) {
      if (!walk.find(tile, t)) return;   // (behind the last tile: nothing is asked for any more)
      rot = rotation_of(t.pn, ipt);
      if constexpr (W) {
        const int row0 = t.pn * BN;
        rsrc = uniform_rsrc(make_rsrc_words(g.B + (int64_t)(t.group - 1) * g.expert_b + (int64_t)row0 * g.ldb, (uint32_t)min(BN, g.N - row0) * (uint32_t)(g.ldb * 2)));
      } else {
        const int row0 = t.pm * BM;
        rsrc = uniform_rsrc(make_rsrc_words(g.A + (int64_t)(t.lo + row0) * g.lda, (uint32_t)min(BM, t.rows - row0) * (uint32_t)(g.lda * 2)));
      }
    }
    template <bool W>
    __device__ __forceinline__ void advance(const GroupedArgs &g, int ipt) {
      if (++i == ipt) {
        i = 0;
        ++tile;
        open<W>(g, ipt);
      }
    }
    __device__ __forceinline__ int k(int ipt) const { return rotated_iteration(i, rot, ipt) * BK; }
  };

  static __device__ __forceinline__ void store_tile(const GroupedArgs &g, const GroupTile &t, const AccV (&acc)[MB], int wm, int wn, int lane) {
    const int col = t.pn * BN + wn * 16 + (lane >> 4) * 4;
    if (col >= g.N) return;
    const int e = t.group - 1;
    const half_t *bias = g.bias ? g.bias + (int64_t)e * g.N : nullptr;
    const bool bf16 = I8 ? g.s.bf16 != 0 : BF16;
    const floatx4 b4 = bias4_of(bias, col, g.N, bf16);
    floatx4 sb;
    if constexpr (I8) sb = scale4_at(g.s.b + (int64_t)e * g.N, col, g.N);
    half_t *C = g.C + (int64_t)t.lo * g.ldc;
    const bool vec_ok = (g.ldc & 3) == 0 && (reinterpret_cast<uintptr_t>(C) & 7) == 0;
#pragma unroll
    for (int i = 0; i < MB; ++i) {
      const int row = t.pm * BM + (wm * MB + i) * 16 + (lane & 15);
      if (row >= t.rows) continue;
      half4v h;
      if constexpr (I8) {
        h = scaled4(acc[i], g.s.a[t.lo + row], sb, b4, g.act, bf16);
      } else {
        floatx4 y;
#pragma unroll
        for (int q = 0; q < 4; ++q) y[q] = activate(acc[i][q] + b4[q], g.act);
        h = round4(y, BF16);
      }
      half_t *dst = C + (int64_t)row * g.ldc + col;
      if (vec_ok && col + 4 <= g.N) {
        *reinterpret_cast<half4v *>(dst) = h;
      } else {
        for (int q = 0; q < 4 && col + q < g.N; ++q) dst[q] = h[q];
      }
    }
  }

  // ws: flags (a counter per CTA, zero before and after) and partials (two slots per CTA)
  static __device__ __forceinline__ void run(const GroupedArgs &g, int ipt, const Workspace &ws, char *smem) {
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wave % WM, wn = wave / WM;

    // ---- this CTA's run of iterations ----
    Cursor w(g), a(g), c(g);
    const int total = w.walk.total_tiles() * ipt;
    // (at least MIN_RUN iterations each: a cut costs about as much as two)
    constexpr int MIN_RUN = 4;
    const int ctas = min(g.grid, max(1, total / MIN_RUN)), pid = grouped_pid(g.grid);
    zero_unowned(g, pid);
    if (pid >= ctas || total == 0) return;
    const int each = (int)((unsigned)total / (unsigned)ctas), extra = total - each * ctas;
    const int start = pid * each + min(pid, extra), n = each + (pid < extra ? 1 : 0);

    // ---- loads: see tile_stream_pairs.h ----
    const uint32_t ldw_bytes = (uint32_t)g.ldb * 2, lda_bytes = (uint32_t)g.lda * 2;
    const int odd = lane >> 5, piece = (lane & 31) ^ odd;
    const int fi = lane & 15, fg = lane >> 4;
    const int frag0 = (fi >> 1) * PAIR + (fi & 1) * 512 + ((fg ^ (fi & 1)) * 16);
    const uint32_t base = lds_address(smem);
    const uint32_t w_ring = (uint32_t)__builtin_amdgcn_readfirstlane((int)(base + (uint32_t)wn * (WD * W_SLOT)));
    const uint32_t a_ring = (uint32_t)__builtin_amdgcn_readfirstlane((int)(base + (uint32_t)LDS_W));
    const char *w_ptr = smem + wn * (WD * W_SLOT) + frag0, *a_ptr = smem + LDS_W + wm * (8 * MB * PAIR) + frag0;
    auto issue_w = [&](int t, int slot) {
      const int kk = w.k(ipt);
      const uint32_t kbytes = (uint32_t)__builtin_amdgcn_readfirstlane(kk * 2);
      const uint32_t off = t < n && kk + piece * 8 < g.K ? (uint32_t)odd * ldw_bytes + (uint32_t)piece * 16 : OOB_OFFSET;
#pragma unroll
      for (int jj = 0; jj < LOADS_W; ++jj) {
        const int j = wm * LOADS_W + jj;
        dma_load_16(w.rsrc, w_ring + (uint32_t)(slot * W_SLOT + j * PAIR), off, kbytes + (uint32_t)(16 * wn + 2 * j) * ldw_bytes);
      }
      if (t + 1 < n) w.template advance<true>(g, ipt);
    };
    auto issue_a = [&](int t, int slot) {
      const int kk = a.k(ipt);
      const uint32_t kbytes = (uint32_t)__builtin_amdgcn_readfirstlane(kk * 2);
      const uint32_t off = t < n && kk + piece * 8 < g.K ? (uint32_t)odd * lda_bytes + (uint32_t)piece * 16 : OOB_OFFSET;
#pragma unroll
      for (int j = 0; j < LOADS_A; ++j) {
        const int q = wave * LOADS_A + j;
        dma_load_16(a.rsrc, a_ring + (uint32_t)(slot * A_SLOT + q * PAIR), off, kbytes + (uint32_t)(2 * q) * lda_bytes);
      }
      if (t + 1 < n) a.template advance<false>(g, ipt);
    };
    w.template seek<true>(g, start, ipt);
    a.template seek<false>(g, start, ipt);
    c.template seek<false>(g, start, ipt);
#pragma unroll
    for (int j = 1 - WD; j < 0; ++j) {
      if (j + AD - 1 >= 0) issue_a(j + AD - 1, j + AD - 1);
      issue_w(j + WD - 1, j + WD - 1);
    }

    // ---- the run ----
    AccV acc[MB];
#pragma unroll
    for (int i = 0; i < MB; ++i) acc[i] = AccV{0, 0, 0, 0};
    int first_i = c.i;            // where the segment of the current tile began
    int head_tile = -1, head_n = 0, tail_tile = -1, tail_n = 0;   // tiles that this run has parts of
    GroupTile head_t, tail_t;
    int wslot = 0, aslot = 0;
    for (int t = 0; t < n; ++t) {
      asm volatile("s_waitcnt vmcnt(%0)" ::"n"(OUTSTANDING) : "memory");
      __syncthreads();
      issue_a(t + AD - 1, aslot == 0 ? AD - 1 : aslot - 1);
      issue_w(t + WD - 1, wslot == 0 ? WD - 1 : wslot - 1);
      const char *wp = w_ptr + wslot * W_SLOT, *ap = a_ptr + aslot * A_SLOT;
      half8v fw[8], fa[MB][8];
#pragma unroll
      for (int s = 0; s < 8; ++s) {
        fw[s] = *reinterpret_cast<const half8v *>(wp + s * 64);
#pragma unroll
        for (int i = 0; i < MB; ++i) fa[i][s] = *reinterpret_cast<const half8v *>(ap + i * 8 * PAIR + s * 64);
      }
#pragma unroll
      for (int s = 0; s < 8; ++s)
#pragma unroll
        for (int i = 0; i < MB; ++i) {
          if constexpr (I8) {
            acc[i] = __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(intx4, fw[s]), __builtin_bit_cast(intx4, fa[i][s]), acc[i], 0, 0, 0);
          } else if constexpr (BF16) {
            typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
            acc[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, fw[s]), __builtin_bit_cast(bf16x8, fa[i][s]), acc[i], 0, 0, 0);
          } else {
            acc[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(fw[s], fa[i][s], acc[i], 0, 0, 0);
          }
        }
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // the fragments are in registers before the next barrier frees their slots
      wslot = wslot + 1 == WD ? 0 : wslot + 1;
      aslot = aslot + 1 == AD ? 0 : aslot + 1;
      if (c.i + 1 == ipt || t + 1 == n) {   // the end of a segment
        const int length = c.i + 1 - first_i;
        if (length == ipt) {
          store_tile(g, c.t, acc, wm, wn, lane);
        } else {
          const int which = first_i == 0 ? 1 : 0;
          const BufferRsrc r = make_rsrc(reinterpret_cast<char *>(ws.partials) + (size_t)(2 * pid + which) * SLOT_BYTES, SLOT_BYTES);
#pragma unroll
          for (int i = 0; i < MB; ++i) st_coherent16(r, (uint32_t)tid * 16, (uint32_t)i * NT * 16, __builtin_bit_cast(uint4v, acc[i]));
          if (which) {
            tail_tile = c.tile;
            tail_n = length;
            tail_t = c.t;
          } else {
            head_tile = c.tile;
            head_n = length;
            head_t = c.t;
          }
        }
#pragma unroll
        for (int i = 0; i < MB; ++i) acc[i] = AccV{0, 0, 0, 0};
        first_i = 0;
      }
      if (t + 1 < n) c.template advance<false>(g, ipt);
    }
    wait_own_memory_ops();   // (the last loads fetch nothing but write LDS; the partial sums are in memory)
    __syncthreads();
    if (head_tile < 0 && tail_tile < 0) return;

    // ---- tiles that more than one CTA has a part of ----
    int *word = reinterpret_cast<int *>(smem);
    auto cta_of = [&](int at) {
      const int boundary = extra * (each + 1);
      return at < boundary ? (int)((unsigned)at / (unsigned)(each + 1)) : extra + (int)((unsigned)(at - boundary) / (unsigned)each);
    };
    auto finish = [&](int tile, int length, const GroupTile &tt) {
      if (tile < 0) return;   // (uniform)
      const int p0 = cta_of(tile * ipt), p1 = cta_of(tile * ipt + ipt - 1);
      if (tid == 0) {
        const int old = __hip_atomic_fetch_add(ws.flags + p0, length, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        *word = old + length == ipt;
        if (old + length == ipt) __hip_atomic_store(ws.flags + p0, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      }
      __syncthreads();
      const bool complete = *word != 0;
      __syncthreads();
      if (!complete) return;
#pragma unroll
      for (int i = 0; i < MB; ++i) acc[i] = AccV{0, 0, 0, 0};
      for (int p = p0; p <= p1; ++p) {
        const BufferRsrc r = make_rsrc(reinterpret_cast<char *>(ws.partials) + (size_t)(2 * p + (p == p0 ? 1 : 0)) * SLOT_BYTES, SLOT_BYTES);
#pragma unroll
        for (int i = 0; i < MB; ++i) acc[i] += __builtin_bit_cast(AccV, ld_coherent16(r, (uint32_t)tid * 16, (uint32_t)i * NT * 16));
      }
      store_tile(g, tt, acc, wm, wn, lane);
    };
    if (tid == 0)
      __hip_atomic_fetch_max(ws.status + WS_DIRTY, (int)(((size_t)(2 * pid + 2) * SLOT_BYTES + 255) >> 8), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    finish(head_tile, head_n, head_t);
    finish(tail_tile, tail_n, tail_t);
  }

  // rows without an expert
  static __device__ __forceinline__ void zero_unowned(const GroupedArgs &g, int pid) {
    const int front = min(max(g.offsets[0], 0), g.R), back = min(max(g.offsets[g.E], front), g.R);
    const int rows = front + g.R - back;
    for (int r = pid; r < rows; r += g.grid) {
      half_t *C = g.C + (int64_t)(r < front ? r : back + r - front) * g.ldc;
      for (int col = threadIdx.x; col < g.N; col += NT) C[col] = (half_t)0.f;
    }
  }
};

}  // namespace sk
