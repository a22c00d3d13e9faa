// C ABI of the grouped products: argument checking and launch.
#include <hip/hip_runtime.h>

#include "grouped_launch.h"
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
  const bool i8 = g->dtype == SK_I8, nn = g->layout == SK_LAYOUT_NN;
  if (!i8 && g->dtype != SK_F16 && g->dtype != SK_BF16) return SK_ERR_CONFIG;
  if ((!nn && g->layout != SK_LAYOUT_NT) || (nn && i8)) return SK_ERR_CONFIG;
  if (i8 ? g->out_dtype != SK_F16 && g->out_dtype != SK_BF16 : g->out_dtype != g->dtype) return SK_ERR_CONFIG;
  if (g->activation < SK_ACT_NONE || g->activation > SK_ACT_SILU || g->variant < 0) return SK_ERR_CONFIG;
  if (g->E <= 0 || g->R <= 0 || g->N <= 0 || g->K <= 0 || g->E > (1 << 20) || g->R > MAX_INT || g->N > MAX_INT || g->K > MAX_INT) return SK_ERR_SHAPE;
  if (g->lda < (nn ? (g->K + 7) / 8 * 8 : g->K) || g->ldb < (nn ? g->N : g->K) || g->ldc < g->N || g->expert_b < 0) return SK_ERR_SHAPE;
  const int64_t step = i8 ? 16 : 8;
  if ((!nn && (g->K % step)) || (g->lda % step) || (g->ldb % step) || (g->expert_b % step) || (nn && (g->N % 8))) return SK_ERR_ALIGN;
  *h = GroupedShape{i8 ? GT_I8 : (g->dtype == SK_BF16 ? GT_BF16 : GT_F16), nn, g->E, g->R, g->N, g->K, 0, (int)g->variant};
  // a tile's rows (NN: all K rows of an expert's weights) are addressed with 32-bit byte offsets
  const int64_t bytes = i8 ? 1 : 2;
  if (g->lda * bytes * 256 >= (int64_t)1 << 31 || g->ldb * bytes * (nn ? g->K + 64 : 256) >= (int64_t)1 << 31 || g->ldc * 2 * 256 >= (int64_t)1 << 31)
    return SK_ERR_SHAPE;
  return SK_OK;
}

extern "C" size_t sk_grouped_workspace_bytes(const sk_grouped *g) {
  GroupedShape h;
  return g && check_shape(g, &h) == SK_OK && sk_device_info(&h.cus, nullptr, nullptr) == SK_OK ? grouped_workspace(h) : 0;
}

extern "C" int sk_gemm_grouped(const sk_grouped *g, void *ws, size_t ws_bytes, void *stream) {
  if (!g || !g->A || !g->B || !g->C || !g->offsets) return SK_ERR_NULL;
  const bool i8 = g->dtype == SK_I8;
  if (i8 ? !g->scale_a || !g->scale_b : g->scale_a || g->scale_b) return i8 ? SK_ERR_NULL : SK_ERR_CONFIG;
  GroupedShape h;
  if (int rc = check_shape(g, &h)) return rc;
  if (misaligned(g->A, 15) || misaligned(g->B, 15) || misaligned(g->C, 1) || misaligned(g->bias, 1) || misaligned(g->offsets, 3) ||
      misaligned(g->scale_a, 3) || misaligned(g->scale_b, 3))
    return SK_ERR_ALIGN;
  if (reinterpret_cast<uintptr_t>(g->bias) >> EPI_ACT_SHIFT) return SK_ERR_CONFIG;   // not a device address
  if (sk_device_info(&h.cus, nullptr, nullptr) != SK_OK) return SK_ERR_DEVICE;
  h.variant = grouped_variant(h);
  Workspace w;
  if (int rc = take_workspace(ws, ws_bytes, grouped_workspace(h), &w)) return rc;
  const int64_t pairs = i8 ? 2 : 1;
  GroupedArgs a{};
  a.A = (const half_t *)g->A;
  a.B = (const half_t *)g->B;
  a.C = (half_t *)g->C;
  a.offsets = (const int *)g->offsets;
  a.bias = (const half_t *)g->bias;
  a.s = Scales{(const float *)g->scale_a, (const float *)g->scale_b, g->out_dtype == SK_BF16};
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
  return status_of(launch_grouped(a, h, w, (hipStream_t)stream));
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
