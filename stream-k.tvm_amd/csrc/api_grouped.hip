// C ABI of the grouped products: argument checking and launch.
#include <hip/hip_runtime.h>

#include "grouped_launch.h"
#include "grouped_mx.h"
#include "launch.h"
#include "streamk.h"

using namespace sk;

namespace {
bool misaligned(const void *p, uintptr_t mask) { return (reinterpret_cast<uintptr_t>(p) & mask) != 0; }
constexpr int64_t MAX_INT = 0x7fffff00;
// (a variant that does not exist or does not take the problem)
int status_of(int herr) { return herr == 0 ? SK_OK : (herr == (int)hipErrorNotSupported ? SK_ERR_CONFIG : SK_ERR_LAUNCH); }
}  // namespace

// everything but the operands' addresses; fills h
static int check_shape(const sk_grouped *g, GroupedShape *h) {
  const bool i8 = g->dtype == SK_I8, mx = g->dtype == SK_MXFP4, nn = g->layout == SK_LAYOUT_NN;
  if (!i8 && !mx && g->dtype != SK_F16 && g->dtype != SK_BF16) return SK_ERR_CONFIG;
  if ((!nn && g->layout != SK_LAYOUT_NT) || (nn && (i8 || mx))) return SK_ERR_CONFIG;
  if (i8 || mx ? g->out_dtype != SK_F16 && g->out_dtype != SK_BF16 : g->out_dtype != g->dtype) return SK_ERR_CONFIG;
  if (g->activation < SK_ACT_NONE || g->activation > SK_ACT_SILU || g->variant < 0) return SK_ERR_CONFIG;
  if (g->E <= 0 || g->R <= 0 || g->N <= 0 || g->K <= 0 || g->E > (1 << 20) || g->R > MAX_INT || g->N > MAX_INT || g->K > MAX_INT) return SK_ERR_SHAPE;
  if (g->lda < (nn ? (g->K + 7) / 8 * 8 : g->K) || g->ldb < (nn ? g->N : g->K) || g->ldc < g->N || g->expert_b < 0) return SK_ERR_SHAPE;
  const int64_t step = mx ? 32 : (i8 ? 16 : 8);
  if ((!nn && (g->K % step)) || (g->lda % step) || (g->ldb % step) || (g->expert_b % step) || (nn && (g->N % 8))) return SK_ERR_ALIGN;
  *h = GroupedShape{mx ? GT_MX : i8 ? GT_I8 : (g->dtype == SK_BF16 ? GT_BF16 : GT_F16), nn, g->E, g->R, g->N, g->K, 0, (int)g->variant};
  // a tile's rows (NN: all K rows of an expert's weights) are addressed with 32-bit byte offsets
  const int64_t pairs = mx ? 4 : (i8 ? 2 : 1);   // values in 16 bits
  if (g->lda / pairs * 2 * 256 >= (int64_t)1 << 31 || g->ldb / pairs * 2 * (nn ? g->K + 64 : 256) >= (int64_t)1 << 31 || g->ldc * 2 * 256 >= (int64_t)1 << 31)
    return SK_ERR_SHAPE;
  if (mx && !g->scales_tiled && g->K / 32 * 256 >= (int64_t)1 << 31) return SK_ERR_SHAPE;
  if (mx && g->scales_tiled && !mx_tiled_fits(*h)) return SK_ERR_SHAPE;
  return SK_OK;
}

extern "C" size_t sk_grouped_workspace_bytes(const sk_grouped *g) {
  GroupedShape h;
  if (!g || check_shape(g, &h) != SK_OK || sk_device_info(&h.cus, nullptr, nullptr) != SK_OK) return 0;
  return h.type == GT_MX ? mx_workspace(h) : grouped_workspace(h);
}

extern "C" int sk_mx_scales_tiled(const sk_grouped *g) {
  GroupedShape h;
  if (!g || g->dtype != SK_MXFP4 || check_shape(g, &h) != SK_OK || sk_device_info(&h.cus, nullptr, nullptr) != SK_OK) return 0;
  return mx_needs_tiled(h);
}

extern "C" int sk_gemm_grouped(const sk_grouped *g, void *ws, size_t ws_bytes, void *stream) {
  if (!g || !g->A || !g->B || !g->C) return SK_ERR_NULL;
  const bool i8 = g->dtype == SK_I8, mx = g->dtype == SK_MXFP4, scaled = i8 || mx;
  if (!g->offsets && (!mx || g->E != 1)) return SK_ERR_NULL;
  if (scaled ? !g->scale_a || !g->scale_b : g->scale_a || g->scale_b) return scaled ? SK_ERR_NULL : SK_ERR_CONFIG;
  GroupedShape h;
  if (int rc = check_shape(g, &h)) return rc;
  if (misaligned(g->A, 15) || misaligned(g->B, 15) || misaligned(g->C, 1) || misaligned(g->bias, 1) || misaligned(g->offsets, 3) ||
      misaligned(g->scale_a, mx && g->scales_tiled ? 15 : 3) || misaligned(g->scale_b, mx && g->scales_tiled ? 15 : 3))
    return SK_ERR_ALIGN;
  if (reinterpret_cast<uintptr_t>(g->bias) >> EPI_ACT_SHIFT) return SK_ERR_CONFIG;   // not a device address
  if (sk_device_info(&h.cus, nullptr, nullptr) != SK_OK) return SK_ERR_DEVICE;
  h.variant = mx ? mx_variant(h) : grouped_variant(h);
  if (mx && !g->scales_tiled && mx_needs_tiled(h)) return SK_ERR_CONFIG;
  Workspace w;
  if (int rc = take_workspace(ws, ws_bytes, mx ? mx_workspace(h) : grouped_workspace(h), &w)) return rc;
  const int64_t pairs = mx ? 4 : (i8 ? 2 : 1);
  MxOperands a{};
  a.A = (const half_t *)g->A;
  a.B = (const half_t *)g->B;
  a.C = (half_t *)g->C;
  a.offsets = (const int *)g->offsets;
  a.bias = (const half_t *)g->bias;
  if (mx) {
    // (tiled: 16 bytes for 512 values of a row, all rows of these 512 together)
    const auto exponents = [&](const void *p, int64_t rows) {
      const int64_t blocks = g->K / 32, pairs = (g->K + 511) / 512;
      const uint8_t *at = (const uint8_t *)p;
      return g->scales_tiled ? MxExponents{at, at + rows * pairs * 16, 16, (int)(rows * 16)} : MxExponents{at, at + rows * blocks, (int)blocks, 16};
    };
    a.ea = exponents(g->scale_a, g->R);
    a.eb = exponents(g->scale_b, g->E * g->N);
  } else {
    a.s = Scales{(const float *)g->scale_a, (const float *)g->scale_b, g->out_dtype == SK_BF16};
  }
  a.lda = g->lda / pairs;
  a.ldb = g->ldb / pairs;
  a.ldc = g->ldc;
  a.expert_b = g->expert_b / pairs;
  a.E = (int)g->E;
  a.R = (int)g->R;
  a.N = (int)g->N;
  a.K = (int)(g->K / pairs);
  a.act = g->activation;
  a.spin_limit = g->spin_limit == 0 || g->spin_limit > MAX_INT ? 1 << 22 : (int)(g->spin_limit < 0 ? 0 : g->spin_limit);
  return status_of(mx ? launch_mx(a, h, g->out_dtype == SK_BF16, w, (hipStream_t)stream) : launch_grouped(a, h, w, (hipStream_t)stream));
}

extern "C" int sk_grouped_wgrad(const void *A, const void *B, const void *offsets, void *C, int dtype, int64_t E, int64_t R, int64_t M,
                                int64_t N, int64_t lda, int64_t ldb, int variant, void *stream) {
  if (variant < 0) return SK_ERR_CONFIG;
  if (dtype != SK_F16 && dtype != SK_BF16) return SK_ERR_CONFIG;
  if (!A || !B || !offsets || !C) return SK_ERR_NULL;
  if (E <= 0 || R <= 0 || M <= 0 || N <= 0 || E > (1 << 20) || R > MAX_INT || M > MAX_INT || N > MAX_INT) return SK_ERR_SHAPE;
  const int64_t width = (M + 7) / 8 * 8;
  if (lda < width || ldb < N) return SK_ERR_SHAPE;
  if ((lda % 8) || (ldb % 8) || (N % 8)) return SK_ERR_ALIGN;
  if (misaligned(A, 15) || misaligned(B, 15) || misaligned(C, 1) || misaligned(offsets, 3)) return SK_ERR_ALIGN;
  // the rows of an iteration are addressed with 32-bit byte offsets
  if (lda * 2 * 64 >= (int64_t)1 << 31 || ldb * 2 * 64 >= (int64_t)1 << 31) return SK_ERR_SHAPE;
  int cus = 0;
  if (sk_device_info(&cus, nullptr, nullptr) != SK_OK) return SK_ERR_DEVICE;
  WgradArgs a{};
  a.dC = (const half_t *)A;
  a.A = (const half_t *)B;
  a.dW = (half_t *)C;
  a.offsets = (const int *)offsets;
  a.lddc = lda;
  a.lda = ldb;
  a.E = (int)E;
  a.R = (int)R;
  a.N = (int)M;
  a.K = (int)N;
  a.width = (int)width;
  return status_of(launch_wgrad(a, dtype == SK_BF16, cus, variant, (hipStream_t)stream));
}
