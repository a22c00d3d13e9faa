// The operators of experts.py and the int8 quantiser in native code: the short way from the dispatcher to a launch, and their gradients.
//
// As in torch_ops.cpp: these check the operands, allocate the results and launch; a call that is not the ordinary case goes, with its
// arguments as they are, to the Python implementation (streamk::<name>_general), which answers it or raises.  The gradients are
// recorded here (the AutogradCUDA implementations), so that a training step of a small layer does not spend its time in the host's
// interpreter: product and both gradients of 500 rows, 8 experts of 2048 x 1024, took 132 us through Python's autograd functions.
#include <ATen/ATen.h>
#include <ATen/core/dispatch/Dispatcher.h>
#include <ATen/core/LegacyTypeDispatch.h>
#include <ATen/hip/EmptyTensor.h>
#include <c10/hip/HIPFunctions.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/library.h>

#include <initializer_list>
#include <mutex>
#include <optional>
#include <shared_mutex>
#include <string>
#include <tuple>
#include <vector>

#include "streamk.h"
#include "torch_ops.h"

namespace {

using at::Tensor;
typedef std::optional<Tensor> MaybeTensor;
typedef std::optional<at::ScalarType> MaybeType;

void *current_stream() { return (void *)c10::hip::getCurrentHIPStream().stream(); }
int dtype_of(at::ScalarType t) { return t == at::kHalf ? SK_F16 : (t == at::kBFloat16 ? SK_BF16 : (t == at::kFloat ? SK_F32 : (t == at::kChar ? SK_I8 : -1))); }
bool is16(const Tensor &t) { return t.scalar_type() == at::kHalf || t.scalar_type() == at::kBFloat16; }
bool aligned(const Tensor &t, uintptr_t bytes) { return reinterpret_cast<uintptr_t>(t.data_ptr()) % bytes == 0; }
// a matrix whose rows the kernels read in place
bool rows_in_place(const Tensor &t) {
  return t.dim() == 2 && t.is_cuda() && t.stride(1) == 1 && t.size(0) > 1 && t.stride(0) >= t.size(1) && t.stride(0) * (int64_t)t.element_size() % 16 == 0 && aligned(t, 16);
}
// the same of one row, whose stride says nothing
bool one_row_in_place(const Tensor &t) {
  return t.dim() == 2 && t.is_cuda() && t.stride(1) == 1 && t.size(0) == 1 && t.size(1) * (int64_t)t.element_size() % 16 == 0 && aligned(t, 16);
}
int64_t pitch(const Tensor &t) { return t.size(0) > 1 ? t.stride(0) : t.size(1); }
bool is_ints(const Tensor &t, const Tensor &like, int64_t dim) {
  return t.scalar_type() == at::kInt && t.dim() == dim && t.is_contiguous() && t.device() == like.device();
}
// a new tensor on the device of another one: the allocator's own entry, half a microsecond less than the dispatcher's
Tensor fresh(const Tensor &like, at::IntArrayRef shape, at::ScalarType type) {
  return Tensor(at::detail::empty_cuda(shape, type, like.device(), std::nullopt));
}
Tensor ints(const Tensor &like, at::IntArrayRef shape) { return fresh(like, shape, at::kInt); }

template <class F>
auto general(const char *name) {
  return c10::Dispatcher::singleton().findSchemaOrThrow((std::string("streamk::") + name + "_general").c_str(), "").typed<F>();
}
template <class F>
auto op(const char *name) {
  return c10::Dispatcher::singleton().findSchemaOrThrow((std::string("streamk::") + name).c_str(), "").typed<F>();
}
#define GENERAL(NAME, F, ...)                        \
  do {                                               \
    static const auto handle = general<F>(NAME);     \
    return handle.call(__VA_ARGS__);                 \
  } while (0)

// ---- the quantiser ----
std::tuple<Tensor, Tensor> quantize_i8(const Tensor &x) {
  at::AutoDispatchBelowADInplaceOrView guard;
  if (x.is_cuda() && is16(x) && x.dim() >= 1 && x.numel() > 0 && x.is_contiguous()) {
    const int64_t K = x.size(-1), M = x.numel() / K;
    Tensor q = fresh(x, x.sizes(), at::kChar), scale = fresh(x, x.sizes().slice(0, x.dim() - 1), at::kFloat);
    if (sk_quantize_i8(x.data_ptr(), dtype_of(x.scalar_type()), M, K, K, q.data_ptr(), K, scale.data_ptr(), current_stream()) == SK_OK) return {q, scale};
  }
  GENERAL("quantize_i8", decltype(quantize_i8), x);
}

// ---- the grouped product ----
bool grouped(const Tensor &rows, const Tensor &B, const Tensor &offsets, std::string_view layout, MaybeType out_dtype, const MaybeTensor &scale_a,
             const MaybeTensor &scale_b, const MaybeTensor &bias, std::string_view activation, int64_t variant, Tensor &C) {
  const at::ScalarType type = rows.scalar_type();
  const bool i8 = type == at::kChar, nn = layout == "nn";
  // ([K, N] weights multiply A's last piece of eight columns whole, those past K by zeros: they have to be finite, so they become zeros)
  const bool pad = nn && rows.is_cuda() && rows.dim() == 2 && rows.numel() > 0 && rows.size(1) % 8 != 0;
  const Tensor padded = pad ? at::constant_pad_nd(rows, {0, 8 - rows.size(1) % 8}) : Tensor(), &A = pad ? padded : rows;
  if ((!i8 && !is16(A)) || (!nn && layout != "nt") || (nn && i8) || B.scalar_type() != type || B.dim() != 3 || B.device() != A.device()) return false;
  if (!rows_in_place(A) && !one_row_in_place(A)) return false;
  const int64_t E = B.size(0), N = B.size(nn ? 2 : 1), K = B.size(nn ? 1 : 2), R = A.size(0);
  if (E == 0 || N == 0 || K == 0 || rows.size(1) != K || B.stride(2) != 1 || B.size(1) < 2 || !is_ints(offsets, A, 1) || offsets.size(0) != E + 1) return false;
  const at::ScalarType out = i8 ? out_dtype.value_or(at::kHalf) : type;
  if ((out != at::kHalf && out != at::kBFloat16) || (!i8 && out_dtype.has_value() && *out_dtype != type)) return false;
  sk_grouped g{};
  if (activation == "none") g.activation = SK_ACT_NONE;
  else if (activation == "relu") g.activation = SK_ACT_RELU;
  else if (activation == "gelu_tanh") g.activation = SK_ACT_GELU_TANH;
  else if (activation == "silu") g.activation = SK_ACT_SILU;
  else return false;
  const auto of = [&](const MaybeTensor &t, at::ScalarType want, int64_t d0, int64_t d1) {   // contiguous [d0, d1] (d1 0: [d0])
    return t->scalar_type() == want && t->dim() == (d1 ? 2 : 1) && t->size(0) == d0 && (!d1 || t->size(1) == d1) && t->is_contiguous() && t->device() == A.device();
  };
  if (scale_a.has_value() != i8 || scale_b.has_value() != i8) return false;
  if (i8 && (!of(scale_a, at::kFloat, R, 0) || !of(scale_b, at::kFloat, E, N))) return false;
  if (bias.has_value() && !of(bias, out, E, N)) return false;
  if (C.defined()) {
    if (!C.is_cuda() || C.scalar_type() != out || C.dim() != 2 || C.size(0) != R || C.size(1) != N || C.stride(1) != 1 || (R > 1 && C.stride(0) < N) || C.device() != A.device()) return false;
  } else {
    C = fresh(A, {R, N}, out);
  }
  g.dtype = dtype_of(type);
  g.layout = nn ? SK_LAYOUT_NN : SK_LAYOUT_NT;
  g.out_dtype = dtype_of(out);
  g.E = E, g.R = R, g.N = N, g.K = K;
  g.A = A.data_ptr(), g.B = B.data_ptr(), g.offsets = offsets.data_ptr(), g.C = C.data_ptr();
  g.lda = pitch(A), g.ldb = B.stride(1), g.ldc = R > 1 ? C.stride(0) : N, g.expert_b = E > 1 ? B.stride(0) : 0;
  g.bias = bias.has_value() ? bias->data_ptr() : nullptr;
  g.scale_a = i8 ? scale_a->data_ptr() : nullptr;
  g.scale_b = i8 ? scale_b->data_ptr() : nullptr;
  g.variant = variant;
  const size_t need = sk_grouped_workspace_bytes(&g);
  void *stream = current_stream();
  std::shared_lock<std::shared_mutex> lock(streamk_torch::g_mutex);
  streamk_torch::Buffer ws;
  if (need > 0 && !streamk_torch::find_workspace((int)c10::hip::current_device(), stream, need, &ws)) return false;
  return sk_gemm_grouped(&g, ws.ptr, ws.bytes, stream) == SK_OK;
}
Tensor gemm_grouped(const Tensor &A, const Tensor &B, const Tensor &offsets, c10::string_view layout, MaybeType out_dtype, const MaybeTensor &scale_a,
                    const MaybeTensor &scale_b, const MaybeTensor &bias, c10::string_view activation, int64_t variant) {
  at::AutoDispatchBelowADInplaceOrView guard;
  Tensor C;
  if (grouped(A, B, offsets, std::string_view(layout.data(), layout.size()), out_dtype, scale_a, scale_b, bias,
              std::string_view(activation.data(), activation.size()), variant, C))
    return C;
  GENERAL("gemm_grouped", decltype(gemm_grouped), A, B, offsets, layout, out_dtype, scale_a, scale_b, bias, activation, variant);
}
void gemm_grouped_out(const Tensor &A, const Tensor &B, const Tensor &offsets, const Tensor &out, c10::string_view layout, MaybeType out_dtype,
                      const MaybeTensor &scale_a, const MaybeTensor &scale_b, const MaybeTensor &bias, c10::string_view activation, int64_t variant) {
  at::AutoDispatchBelowADInplaceOrView guard;
  Tensor C = out;
  if (grouped(A, B, offsets, std::string_view(layout.data(), layout.size()), out_dtype.has_value() ? out_dtype : MaybeType(out.scalar_type()), scale_a,
              scale_b, bias, std::string_view(activation.data(), activation.size()), variant, C))
    return;
  GENERAL("gemm_grouped_out", decltype(gemm_grouped_out), A, B, offsets, out, layout, out_dtype, scale_a, scale_b, bias, activation, variant);
}

Tensor grouped_wgrad(const Tensor &A, const Tensor &B, const Tensor &offsets, int64_t variant) {
  at::AutoDispatchBelowADInplaceOrView guard;
  if (is16(A) && B.scalar_type() == A.scalar_type() && rows_in_place(A) && rows_in_place(B) && A.size(0) == B.size(0) && A.device() == B.device() &&
      A.size(1) % 8 == 0 && B.size(1) % 8 == 0 && A.size(1) > 0 && B.size(1) > 0 && is_ints(offsets, A, 1) && offsets.size(0) >= 2) {
    const int64_t E = offsets.size(0) - 1, M = A.size(1), N = B.size(1);
    Tensor C = fresh(A, {E, M, N}, A.scalar_type());
    if (sk_grouped_wgrad(A.data_ptr(), B.data_ptr(), offsets.data_ptr(), C.data_ptr(), dtype_of(A.scalar_type()), E, A.size(0), M, N, pitch(A), pitch(B),
                         (int)variant, current_stream()) == SK_OK)
      return C;
  }
  GENERAL("grouped_wgrad", decltype(grouped_wgrad), A, B, offsets, variant);
}

// ---- routing, dispatch, combination ----
typedef std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor> FiveTensors;
FiveTensors route_experts(const Tensor &logits, int64_t k) {
  at::AutoDispatchBelowADInplaceOrView guard;
  const int dtype = dtype_of(logits.scalar_type());
  if (logits.is_cuda() && dtype >= 0 && dtype != SK_I8 && logits.dim() == 2 && logits.size(0) > 0 && logits.is_contiguous() && k >= 1 && k <= logits.size(1)) {
    const int64_t T = logits.size(0), E = logits.size(1);
    Tensor weights = fresh(logits, {T, k}, at::kFloat), experts = ints(logits, {T, k}), offsets = ints(logits, {E + 1}),
           order = ints(logits, {T * k}), place = ints(logits, {T, k});
    const size_t bytes = sk_route_workspace_bytes(T, E, k);
    Tensor ws;
    if (bytes > 0) ws = fresh(logits, {(int64_t)bytes}, at::kByte);
    if (sk_route_experts(logits.data_ptr(), dtype, T, E, k, E, weights.data_ptr(), experts.data_ptr(), offsets.data_ptr(), order.data_ptr(), place.data_ptr(),
                         bytes > 0 ? ws.data_ptr() : nullptr, bytes, current_stream()) == SK_OK)
      return {weights, experts, offsets, order, place};
  }
  GENERAL("route_experts", decltype(route_experts), logits, k);
}
Tensor route_backward(const Tensor &weights, const Tensor &experts, const Tensor &dweights, int64_t E, at::ScalarType dtype) {
  at::AutoDispatchBelowADInplaceOrView guard;
  if (weights.is_cuda() && weights.scalar_type() == at::kFloat && weights.dim() == 2 && weights.size(0) > 0 && weights.is_contiguous() && is_ints(experts, weights, 2) &&
      experts.sizes() == weights.sizes() && dweights.scalar_type() == at::kFloat && dweights.sizes() == weights.sizes() && dweights.is_contiguous() &&
      dweights.device() == weights.device() && dtype_of(dtype) >= 0) {
    Tensor dlogits = fresh(weights, {weights.size(0), E}, dtype);
    if (sk_route_backward(weights.data_ptr(), experts.data_ptr(), dweights.data_ptr(), weights.size(0), E, weights.size(1), dtype_of(dtype), dlogits.data_ptr(),
                          current_stream()) == SK_OK)
      return dlogits;
  }
  GENERAL("route_backward", decltype(route_backward), weights, experts, dweights, E, dtype);
}
// (place undefined: none) an undefined tensor: not the ordinary case
Tensor dispatched(const Tensor &x, const Tensor &order, const Tensor &place, int64_t k) {
  if (!x.is_cuda() || (x.dim() != 1 && x.dim() != 2) || x.numel() == 0 || !x.is_contiguous() || k < 1 || !is_ints(order, x, 1) || order.size(0) != x.size(0) * k) return {};
  const int64_t T = x.size(0), width = x.dim() == 2 ? x.size(1) : 1, bytes = width * (int64_t)x.element_size();
  if (place.defined() && (!is_ints(place, x, 2) || place.size(0) != T || place.size(1) != k)) return {};
  Tensor rows = x.dim() == 2 ? fresh(x, {T * k, width}, x.scalar_type()) : fresh(x, {T * k}, x.scalar_type());
  const int rc = sk_dispatch_rows(x.data_ptr(), bytes, bytes, order.data_ptr(), place.defined() ? place.data_ptr() : nullptr, T, k, rows.data_ptr(), current_stream());
  return rc == SK_OK ? rows : Tensor();
}
Tensor dispatch_rows(const Tensor &x, const Tensor &order, int64_t k) {
  at::AutoDispatchBelowADInplaceOrView guard;
  const Tensor rows = dispatched(x, order, Tensor(), k);
  if (rows.defined()) return rows;
  GENERAL("dispatch_rows", decltype(dispatch_rows), x, order, k);
}
Tensor dispatch_routed(const Tensor &x, const Tensor &order, const Tensor &place) {
  at::AutoDispatchBelowADInplaceOrView guard;
  const Tensor rows = place.dim() == 2 ? dispatched(x, order, place, place.size(1)) : Tensor();
  if (rows.defined()) return rows;
  GENERAL("dispatch_routed", decltype(dispatch_routed), x, order, place);
}
Tensor combine_rows(const Tensor &y, const Tensor &place, const MaybeTensor &weights) {
  at::AutoDispatchBelowADInplaceOrView guard;
  if (y.is_cuda() && is16(y) && y.dim() == 2 && y.numel() > 0 && y.is_contiguous() && is_ints(place, y, 2) && y.size(0) == place.numel() &&
      (!weights.has_value() || (weights->scalar_type() == at::kFloat && weights->sizes() == place.sizes() && weights->is_contiguous() && weights->device() == y.device()))) {
    const int64_t T = place.size(0), k = place.size(1), H = y.size(1);
    Tensor out = fresh(y, {T, H}, y.scalar_type());
    if (sk_combine_rows(y.data_ptr(), dtype_of(y.scalar_type()), place.data_ptr(), weights.has_value() ? weights->data_ptr() : nullptr, T, k, H, out.data_ptr(),
                        current_stream()) == SK_OK)
      return out;
  }
  GENERAL("combine_rows", decltype(combine_rows), y, place, weights);
}
std::tuple<Tensor, Tensor> combine_backward(const Tensor &d_out, const Tensor &y, const Tensor &order, const Tensor &place, const Tensor &weights) {
  at::AutoDispatchBelowADInplaceOrView guard;
  if (y.is_cuda() && is16(y) && y.dim() == 2 && y.numel() > 0 && y.is_contiguous() && is_ints(place, y, 2) && is_ints(order, y, 1) && y.size(0) == place.numel() &&
      order.size(0) == y.size(0) && d_out.scalar_type() == y.scalar_type() && d_out.dim() == 2 && d_out.size(0) == place.size(0) && d_out.size(1) == y.size(1) &&
      d_out.is_contiguous() && d_out.device() == y.device() && weights.scalar_type() == at::kFloat && weights.sizes() == place.sizes() && weights.is_contiguous() &&
      weights.device() == y.device()) {
    Tensor dy = fresh(y, y.sizes(), y.scalar_type()), dw = fresh(weights, weights.sizes(), weights.scalar_type());
    if (sk_combine_backward(d_out.data_ptr(), y.data_ptr(), dtype_of(y.scalar_type()), order.data_ptr(), place.data_ptr(), weights.data_ptr(), place.size(0),
                            place.size(1), y.size(1), dy.data_ptr(), dw.data_ptr(), current_stream()) == SK_OK)
      return {dy, dw};
  }
  GENERAL("combine_backward", decltype(combine_backward), d_out, y, order, place, weights);
}

// ---- gradients ----
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
#define OP(NAME) op<decltype(NAME)>(#NAME)
// the operator's implementation behind autograd, by the dispatcher (tracing and fake tensors have theirs)
#define BELOW(NAME, ...)                             \
  do {                                               \
    static const auto handle = OP(NAME);             \
    at::AutoDispatchBelowADInplaceOrView guard;      \
    return handle.call(__VA_ARGS__);                 \
  } while (0)
bool wanted(const Tensor &t) { return at::GradMode::is_enabled() && t.requires_grad(); }
// (a dual tensor does not require a gradient: below autograd its tangent would be lost without a word)
void no_tangent(const char *what, std::initializer_list<const Tensor *> operands) {
  for (const Tensor *t : operands)
    TORCH_CHECK_NOT_IMPLEMENTED(!t || !t->defined() || !t->_fw_grad(0).defined(), "streamk: ", what, " has no forward-mode derivative");
}
const Tensor *get(const MaybeTensor &t) { return t.has_value() ? &*t : nullptr; }

// Passes a result on; who asks for its derivative by one of the operands that require one gets an error with the reason.
struct Refused : torch::autograd::Function<Refused> {
  static Tensor forward(AutogradContext *ctx, const Tensor &result, at::TensorList, const std::string &why) {
    ctx->saved_data["why"] = why;
    return result;
  }
  static variable_list backward(AutogradContext *ctx, variable_list) { TORCH_CHECK(false, "streamk: ", ctx->saved_data["why"].toStringRef()); }
};

// A gradient made of these tensors, which is not differentiable again (of interest with create_graph only).
Tensor once(const Tensor &gradient, std::initializer_list<Tensor> of) {
  if (!gradient.defined() || !at::GradMode::is_enabled()) return gradient;
  return Refused::apply(gradient, at::TensorList(of), "the gradients of the operators for experts are not differentiable again");
}

struct GroupedProduct : torch::autograd::Function<GroupedProduct> {
  static Tensor forward(AutogradContext *ctx, const Tensor &A, const Tensor &B, const Tensor &offsets, std::string layout, int64_t variant) {
    at::AutoDispatchBelowADInplaceOrView guard;
    static const auto product = OP(gemm_grouped);
    ctx->save_for_backward({A, B, offsets});
    ctx->saved_data["nn"] = layout == "nn";
    return product.call(A, B, offsets, layout, c10::nullopt, c10::nullopt, c10::nullopt, c10::nullopt, "none", variant);
  }
  static variable_list backward(AutogradContext *ctx, variable_list grads) {
    static const auto product = OP(gemm_grouped);
    static const auto wgrad = OP(grouped_wgrad);
    const auto saved = ctx->get_saved_variables();
    const Tensor &A = saved[0], &B = saved[1], &offsets = saved[2], &dC = grads[0];
    if (!dC.defined()) return {Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
    const bool nn = ctx->saved_data["nn"].toBool();
    Tensor dA, dB;
    {
      at::AutoDispatchBelowADInplaceOrView guard;
      // ('nt': dC [R, N] times B[e] [N, K], any N)
      if (ctx->needs_input_grad(0)) dA = product.call(dC, B, offsets, nn ? "nt" : "nn", c10::nullopt, c10::nullopt, c10::nullopt, c10::nullopt, "none", 0);
      if (ctx->needs_input_grad(1)) dB = nn ? wgrad.call(A, dC, offsets, 0) : wgrad.call(dC, A, offsets, 0);
    }
    return {once(dA, {dC, B}), once(dB, {dC, A}), Tensor(), Tensor(), Tensor()};
  }
};
Tensor gemm_grouped_autograd(const Tensor &A, const Tensor &B, const Tensor &offsets, c10::string_view layout, MaybeType out_dtype, const MaybeTensor &scale_a,
                             const MaybeTensor &scale_b, const MaybeTensor &bias, c10::string_view activation, int64_t variant) {
  no_tangent("the grouped product", {&A, &B, get(scale_a), get(scale_b), get(bias)});
  const bool plain = !scale_a.has_value() && !scale_b.has_value() && !bias.has_value() && activation == "none" &&
                     (!out_dtype.has_value() || *out_dtype == A.scalar_type()) && (layout == "nt" || layout == "nn");
  if (plain && (wanted(A) || wanted(B))) return GroupedProduct::apply(A, B, offsets, std::string(layout.data(), layout.size()), variant);
  const auto below = [&]() -> Tensor { BELOW(gemm_grouped, A, B, offsets, layout, out_dtype, scale_a, scale_b, bias, activation, variant); };
  if (!at::GradMode::is_enabled()) return below();
  std::vector<Tensor> recorded;
  for (const Tensor *t : {&A, &B, get(scale_a), get(scale_b), get(bias)})
    if (t && t->requires_grad()) recorded.push_back(*t);
  if (recorded.empty()) return below();
  return Refused::apply(below(), at::TensorList(recorded), "the grouped product has gradients only without bias, activation, scales and out");
}

struct RouteExperts : torch::autograd::Function<RouteExperts> {
  static variable_list forward(AutogradContext *ctx, const Tensor &logits, int64_t k) {
    at::AutoDispatchBelowADInplaceOrView guard;
    static const auto route = OP(route_experts);
    const FiveTensors r = route.call(logits, k);
    ctx->save_for_backward({std::get<0>(r), std::get<1>(r)});
    ctx->saved_data["E"] = logits.size(1);
    ctx->saved_data["dtype"] = (int64_t)logits.scalar_type();
    ctx->mark_non_differentiable({std::get<1>(r), std::get<2>(r), std::get<3>(r), std::get<4>(r)});
    return {std::get<0>(r), std::get<1>(r), std::get<2>(r), std::get<3>(r), std::get<4>(r)};
  }
  static variable_list backward(AutogradContext *ctx, variable_list grads) {
    static const auto back = OP(route_backward);
    const auto saved = ctx->get_saved_variables();
    if (!grads[0].defined()) return {Tensor(), Tensor()};
    Tensor dlogits;
    {
      at::AutoDispatchBelowADInplaceOrView guard;
      dlogits = back.call(saved[0], saved[1], grads[0], ctx->saved_data["E"].toInt(), (at::ScalarType)ctx->saved_data["dtype"].toInt());
    }
    return {once(dlogits, {saved[0], grads[0]}), Tensor()};
  }
};
FiveTensors route_experts_autograd(const Tensor &logits, int64_t k) {
  no_tangent("route_experts", {&logits});
  if (!wanted(logits)) BELOW(route_experts, logits, k);
  const variable_list r = RouteExperts::apply(logits, k);
  return {r[0], r[1], r[2], r[3], r[4]};
}

// (place: for the gradient of dispatch_rows, which is a combination without weights)
struct DispatchRows : torch::autograd::Function<DispatchRows> {
  static Tensor forward(AutogradContext *ctx, const Tensor &x, const Tensor &order, const Tensor &place) {
    at::AutoDispatchBelowADInplaceOrView guard;
    static const auto dispatch = OP(dispatch_routed);
    ctx->save_for_backward({place});
    return dispatch.call(x, order, place);
  }
  static variable_list backward(AutogradContext *ctx, variable_list grads) {
    static const auto combine = OP(combine_rows);
    if (!grads[0].defined()) return {Tensor(), Tensor(), Tensor()};
    Tensor dx;
    {
      at::AutoDispatchBelowADInplaceOrView guard;
      dx = combine.call(grads[0], ctx->get_saved_variables()[0], c10::nullopt);
    }
    return {once(dx, {grads[0]}), Tensor(), Tensor()};
  }
};
Tensor dispatch_routed_autograd(const Tensor &x, const Tensor &order, const Tensor &place) {
  no_tangent("dispatch_rows", {&x});
  if (wanted(x)) return DispatchRows::apply(x, order, place);
  BELOW(dispatch_routed, x, order, place);
}

struct CombineRows : torch::autograd::Function<CombineRows> {
  static Tensor forward(AutogradContext *ctx, const Tensor &y, const Tensor &weights, const Tensor &order, const Tensor &place) {
    at::AutoDispatchBelowADInplaceOrView guard;
    static const auto combine = OP(combine_rows);
    ctx->save_for_backward({y, weights, order, place});
    return combine.call(y, place, weights);
  }
  static variable_list backward(AutogradContext *ctx, variable_list grads) {
    static const auto back = OP(combine_backward);
    if (!grads[0].defined()) return {Tensor(), Tensor(), Tensor(), Tensor()};
    const auto saved = ctx->get_saved_variables();
    Tensor dy, dw;
    {
      at::AutoDispatchBelowADInplaceOrView guard;
      std::tie(dy, dw) = back.call(grads[0], saved[0], saved[2], saved[3], saved[1]);
    }
    return {once(dy, {grads[0], saved[1]}), once(dw, {grads[0], saved[0]}), Tensor(), Tensor()};
  }
};
Tensor combine_routed(const Tensor &y, const Tensor &weights, const Tensor &order, const Tensor &place) {
  return combine_rows(y, place, weights);
}
Tensor combine_routed_autograd(const Tensor &y, const Tensor &weights, const Tensor &order, const Tensor &place) {
  no_tangent("combine_rows", {&y, &weights});
  if (wanted(y) || wanted(weights)) return CombineRows::apply(y, weights, order, place);
  BELOW(combine_routed, y, weights, order, place);
}

}  // namespace

TORCH_LIBRARY_IMPL(streamk, CUDA, m) {
  m.impl("quantize_i8", &quantize_i8);
  m.impl("gemm_grouped", &gemm_grouped);
  m.impl("gemm_grouped_out", &gemm_grouped_out);
  m.impl("grouped_wgrad", &grouped_wgrad);
  m.impl("route_experts", &route_experts);
  m.impl("route_backward", &route_backward);
  m.impl("dispatch_rows", &dispatch_rows);
  m.impl("dispatch_routed", &dispatch_routed);
  m.impl("combine_rows", &combine_rows);
  m.impl("combine_routed", &combine_routed);
  m.impl("combine_backward", &combine_backward);
}
TORCH_LIBRARY_IMPL(streamk, AutogradCUDA, m) {
  m.impl("gemm_grouped", &gemm_grouped_autograd);
  m.impl("route_experts", &route_experts_autograd);
  m.impl("dispatch_routed", &dispatch_routed_autograd);
  m.impl("combine_routed", &combine_routed_autograd);
}
