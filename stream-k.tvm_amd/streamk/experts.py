"""The operators of a mixture of experts: products grouped by expert, their gradients, and the exchange of rows between tokens and experts.

    route = route_experts(logits, k)                     # the k experts of each token, their weights, the rows' order
    rows = dispatch_rows(x, route)                       # [T, H] -> [T k, H], sorted by expert
    h = streamk_grouped(rows, up, route.offsets, activation="silu")      # each expert's rows times its own weights
    out = combine_rows(streamk_grouped(h, down, route.offsets), route)   # the weighted sum of each token's rows

Every function is an operator of the `streamk` namespace and, under autograd, differentiable (backward) in its floating operands but for
`streamk_grouped_wgrad`, which is a gradient itself, and the grouped product with bias, activation or scales; forward-mode derivatives are
refused.  Sizes of groups stay on the device: no call waits for it.  Ordinary calls run, and record their
gradients, in native code (csrc/torch_ops_experts.cpp), which passes every other one on to the implementations here, registered as
`<name>_general`; without the native library those and the autograd functions here stand in.
"""
import ctypes
from typing import NamedTuple

import torch

from . import _lib, ops

_TYPES = {torch.float16: _lib.SK_F16, torch.bfloat16: _lib.SK_BF16}
MAX_EXPERTS, MAX_CHOSEN = 1024, 64
_ops = torch.ops.streamk
_NATIVE = _lib.torch_lib() is not None


def _operator(name, schema, run, fake):
    """Defines streamk::<name> and <name>_general; run is the implementation of the latter, and of both without the native library."""
    for suffix in ("", "_general"):
        ops._LIBRARY.define(f"{name}{suffix}{schema}")
        if suffix or not _NATIVE:
            ops._LIBRARY.impl(name + suffix, run, "CUDA")
    torch.library.register_fake(f"streamk::{name}", fake, lib=ops._LIBRARY)


def _no_tangent(what, *operands):
    """(without the native library, whose autograd implementations refuse by themselves)"""
    if any(isinstance(t, torch.Tensor) and torch.autograd.forward_ad.unpack_dual(t).tangent is not None for t in operands):
        raise NotImplementedError(f"streamk: {what} has no forward-mode derivative")


def _on_device(t, name, dtypes, dims):
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise TypeError(f"{name} must be a CUDA/HIP tensor")
    if t.dtype not in dtypes:
        raise TypeError(f"{name} must be {' or '.join(str(d) for d in dtypes)}, got {t.dtype}")
    if t.dim() != dims:
        raise ValueError(f"{name} must have {dims} dimension{'s' if dims > 1 else ''}, got {tuple(t.shape)}")


def _check_offsets(offsets, E, device):
    _on_device(offsets, "offsets", (torch.int32,), 1)
    if offsets.shape[0] != E + 1 or not offsets.is_contiguous() or offsets.device != device:
        raise ValueError(f"offsets must be a contiguous int32 vector of {E + 1} elements on {device}, got {tuple(offsets.shape)} on {offsets.device}")


def _pitch(t):
    """Row pitch of a matrix whose rows are taken as they stand (that of a single row says nothing, and need not be aligned)."""
    return t.stride(0) if t.shape[0] > 1 else (t.shape[1] + 15) // 16 * 16


# ---- the grouped product ----
def _rows(t):
    """t as the kernels can read it; a row that stands for many (a broadcast gradient) is written out."""
    t = ops._aligned_rows(t)
    return t.contiguous() if t.shape[0] > 1 and t.stride(0) < t.shape[1] else t


def _padded(t):
    """t with its columns filled up with zeros to a multiple of 8, its rows as the kernels read them."""
    if t.shape[1] % 8:
        return torch.nn.functional.pad(t, (0, 8 - t.shape[1] % 8))
    return _rows(t)


def _grouped(A, B, offsets, layout="nt", out_dtype=None, scale_a=None, scale_b=None, bias=None, activation="none", variant=0, out=None):
    if layout not in ("nt", "nn"):
        raise ValueError("layout must be 'nt' (B is [E, N, K]) or 'nn' (B is [E, K, N])")
    int8 = isinstance(A, torch.Tensor) and A.dtype == torch.int8
    _on_device(A, "A", (torch.int8,) if int8 else tuple(_TYPES), 2)
    _on_device(B, "B", (A.dtype,), 3)
    if A.device != B.device:
        raise ValueError(f"A is on {A.device}, B on {B.device}")
    E, N, K = B.shape if layout == "nt" else (B.shape[0], B.shape[2], B.shape[1])
    R = A.shape[0]
    if A.shape[1] != K:
        raise ValueError(f"K mismatch: A is {tuple(A.shape)}, B is {tuple(B.shape)} ({layout})")
    if E == 0 or N == 0 or K == 0:
        raise ValueError(f"B must not be empty, got {tuple(B.shape)}")
    if B.stride(2) != 1:
        raise ValueError("B must have unit stride along its last dimension")
    _check_offsets(offsets, E, A.device)
    if int8:
        if layout != "nt":
            raise ValueError("int8 weights are [E, N, K] ('nt')")
        if scale_a is None or scale_b is None:
            raise ValueError("int8 operands need scale_a and scale_b")
        for t, name, shape in ((scale_a, "scale_a", (R,)), (scale_b, "scale_b", (E, N))):
            if t.dtype != torch.float32 or tuple(t.shape) != shape or not t.is_contiguous() or t.device != A.device:
                raise ValueError(f"{name} must be contiguous float32 {shape} on {A.device}")
        out_dtype = torch.float16 if out_dtype is None else out_dtype
    else:
        if scale_a is not None or scale_b is not None:
            raise ValueError("scales belong to int8 operands")
        if out_dtype not in (None, A.dtype):
            raise ValueError(f"the result of {A.dtype} operands is {A.dtype}")
        out_dtype = A.dtype
    if out_dtype not in _TYPES:
        raise ValueError("out_dtype must be torch.float16 or torch.bfloat16")
    if activation not in _lib.ACTIVATIONS:
        raise ValueError(f"activation must be one of {sorted(k for k in _lib.ACTIVATIONS if k)} or None")
    if bias is not None and (bias.dtype != out_dtype or tuple(bias.shape) != (E, N) or not bias.is_contiguous() or bias.device != A.device):
        raise ValueError(f"bias must be contiguous {out_dtype} {(E, N)} on {A.device}")
    if out is not None:
        ops._check_out(out, R, N, out_dtype)
    C = torch.empty((R, N), dtype=out_dtype, device=A.device) if out is None else out
    if R == 0:
        return C
    # ([K, N] weights and a K that is no multiple of 8: the last piece of eight columns of A is multiplied whole, its columns past K by
    # zeros -- but zero times what lies beside a view may be NaN)
    A = _padded(A) if layout == "nn" and K % 8 else _rows(A)
    if layout == "nn" and 2 * B.stride(1) * (K + 64) >= 1 << 31:
        # the tiles address all rows of a [K, N] expert by 32-bit offsets, those of an [N, K] one a tile at a time
        turned = B.new_zeros((E, N, A.shape[1]))
        turned[:, :, :K].copy_(B.transpose(1, 2))
        B, K, layout = turned, A.shape[1], "nt"
    A = A[:, :K]
    ldb = B.stride(1) if B.shape[1] > 1 else (B.shape[2] + 15) // 16 * 16
    g = _lib.SkGrouped(dtype=_lib.SK_I8 if int8 else _TYPES[A.dtype], layout=ops._plan_mod._LAYOUTS[layout], out_dtype=_TYPES[out_dtype],
                       activation=_lib.ACTIVATIONS[activation], E=E, R=R, N=N, K=K, A=A.data_ptr(), B=B.data_ptr(),
                       offsets=offsets.data_ptr(), C=C.data_ptr(), lda=_pitch(A), ldb=ldb, ldc=max(C.stride(0), N),
                       expert_b=B.stride(0) if E > 1 else 0, bias=bias.data_ptr() if bias is not None else None,
                       scale_a=scale_a.data_ptr() if int8 else None, scale_b=scale_b.data_ptr() if int8 else None, variant=variant)
    ws = ops._workspace(_lib.lib().sk_grouped_workspace_bytes(ctypes.byref(g)), A.device)
    _lib.check(_lib.lib().sk_gemm_grouped(ctypes.byref(g), ws.data_ptr() if ws is not None else None, ws.numel() if ws is not None else 0,
                                          ops._stream_ptr()), "sk_gemm_grouped")
    return C


_GROUPED_TAIL = "str layout=\"nt\", ScalarType? out_dtype=None, Tensor? scale_a=None, Tensor? scale_b=None, Tensor? bias=None, str activation=\"none\", int variant=0"


def _grouped_fake(A, B, offsets, layout="nt", out_dtype=None, *rest):
    return A.new_empty((A.shape[0], B.shape[1 if layout == "nt" else 2]), dtype=out_dtype or (torch.float16 if A.dtype == torch.int8 else A.dtype))


def _grouped_out(A, B, offsets, out, layout="nt", out_dtype=None, scale_a=None, scale_b=None, bias=None, activation="none", variant=0):
    _grouped(A, B, offsets, layout, out.dtype if out_dtype is None else out_dtype, scale_a, scale_b, bias, activation, variant, out)


_operator("gemm_grouped", f"(Tensor A, Tensor B, Tensor offsets, {_GROUPED_TAIL}) -> Tensor", _grouped, _grouped_fake)
_operator("gemm_grouped_out", f"(Tensor A, Tensor B, Tensor offsets, Tensor(a!) out, {_GROUPED_TAIL}) -> ()", _grouped_out, lambda *args: None)


# ---- the gradient of its weights ----
def _wgrad(A, B, offsets, variant=0):
    _on_device(A, "A", tuple(_TYPES), 2)
    _on_device(B, "B", (A.dtype,), 2)
    if A.shape[0] != B.shape[0] or A.device != B.device:
        raise ValueError(f"A and B must have the same rows on one device, got {tuple(A.shape)} on {A.device} and {tuple(B.shape)} on {B.device}")
    _on_device(offsets, "offsets", (torch.int32,), 1)
    E, M, N = offsets.shape[0] - 1, A.shape[1], B.shape[1]
    if E < 1:
        raise ValueError("offsets must have two elements at least")
    _check_offsets(offsets, E, A.device)
    if N % 8:
        raise ValueError("B must have a multiple of 8 columns")
    C = torch.empty((E, M, N), dtype=A.dtype, device=A.device)
    if A.shape[0] == 0 or C.numel() == 0:
        return C.zero_()
    A, B = _padded(A), _rows(B)
    rc = _lib.lib().sk_grouped_wgrad(A.data_ptr(), B.data_ptr(), offsets.data_ptr(), C.data_ptr(), _TYPES[C.dtype], E, A.shape[0], M, N, _pitch(A),
                                     _pitch(B), variant, ops._stream_ptr())
    _lib.check(rc, "sk_grouped_wgrad")
    return C


_operator("grouped_wgrad", "(Tensor A, Tensor B, Tensor offsets, int variant=0) -> Tensor", _wgrad, lambda A, B, offsets, variant=0: A.new_empty((offsets.shape[0] - 1, A.shape[1], B.shape[1])))


class _GroupedProduct(torch.autograd.Function):
    @staticmethod
    def forward(ctx, A, B, offsets, layout, variant):
        ctx.save_for_backward(A, B, offsets)
        ctx.layout = layout
        return _ops.gemm_grouped(A, B, offsets, layout, variant=variant)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dC):
        A, B, offsets = ctx.saved_tensors
        dA = dB = None
        if ctx.needs_input_grad[0]:
            dA = _ops.gemm_grouped(dC, B, offsets, "nt" if ctx.layout == "nn" else "nn")
        if ctx.needs_input_grad[1]:
            dB = _ops.grouped_wgrad(dC, A, offsets) if ctx.layout == "nt" else _ops.grouped_wgrad(A, dC, offsets)
        return dA, dB, None, None, None


def streamk_grouped(A, B, offsets, *, layout="nt", scale_a=None, scale_b=None, out_dtype=None, out=None, bias=None, activation=None, variant=0):
    """Rows offsets[e] <= r < offsets[e + 1] of A [R, K] times the weights of expert e: C[r] = activation(A[r] @ B[e].T + bias[e]) for B
    [E, N, K] (layout 'nt'), A[r] @ B[e] for B [E, K, N] ('nn'); float16, bfloat16, or int8 ('nt') with scale_a [R] and scale_b
    [E, N] (float32), whose result is `out_dtype` (float16 by default).  offsets: int32 [E + 1] on the device, ascending from 0;
    groups of any size; rows behind the last group come out as zeros.  K is a multiple of 8 (int8: 16) for 'nt', N of 8 for 'nn', whose K
    may be any number (rows of a K that is no multiple of 8 are copied, and so are an expert's [K, N] weights from 2 GiB on).  bias: [E, N] in C's type.  Sums in fp32 (int8: exact), rounded
    once.  Differentiable in A and B without bias, activation, scales and out.  variant: which tiles run (sk_grouped in streamk.h); 0
    lets the sizes decide."""
    activation = activation or "none"
    if not _NATIVE:
        _no_tangent("the grouped product", A, B, bias, scale_a, scale_b)
    if torch.is_grad_enabled() and (A.requires_grad or B.requires_grad or (bias is not None and bias.requires_grad)):
        if bias is not None or activation != "none" or scale_a is not None or scale_b is not None or out is not None:
            raise ValueError("the grouped product has gradients only without bias, activation, scales and out")
        if out_dtype not in (None, A.dtype):
            raise ValueError(f"the result of {A.dtype} operands is {A.dtype}")
        if not _NATIVE:
            return _GroupedProduct.apply(A, B, offsets, layout, variant)
    if out is None:
        return _gemm_grouped(A, B, offsets, layout, out_dtype, scale_a, scale_b, bias, activation, variant)
    _ops.gemm_grouped_out(A, B, offsets, out, layout, out_dtype, scale_a, scale_b, bias, activation, variant)
    return out


def streamk_grouped_wgrad(dC, A, offsets, *, variant=0):
    """dB[e] = sum over the rows r of group e of dC[r]^T A[r]: [E, N, K] for dC [R, N] and A [R, K] (K a multiple of 8), the gradient of
    streamk_grouped's weights ('nt'); fp32 sums, a group without rows gives zeros.  variant: sk_grouped_wgrad in streamk.h."""
    return _ops.grouped_wgrad(dC, A, offsets, variant)


# ---- routing ----
class Route(NamedTuple):
    """Where tokens go.  Slot t k + j is token t's j-th expert."""
    weights: torch.Tensor   # float32 [T, k]: softmax of the chosen logits, 0 where there is no expert
    experts: torch.Tensor   # int32 [T, k]: the largest logit's first; -1 where fewer than k can be chosen
    offsets: torch.Tensor   # int32 [E + 1]: where each expert's rows begin
    order: torch.Tensor     # int32 [T k]: the slot of each sorted row, -1 from offsets[E] on
    place: torch.Tensor     # int32 [T, k]: the sorted row of each slot, -1 without an expert


_LOGITS = {torch.float16: _lib.SK_F16, torch.bfloat16: _lib.SK_BF16, torch.float32: _lib.SK_F32}


def _route(logits, k):
    _on_device(logits, "logits", tuple(_LOGITS), 2)
    T, E = logits.shape
    if not 1 <= E <= MAX_EXPERTS or not 1 <= k <= min(E, MAX_CHOSEN):
        raise ValueError(f"1 to {MAX_EXPERTS} experts, of which 1 to {MAX_CHOSEN} are chosen: got {E} and k = {k}")
    if logits.stride(1) != 1 and E > 1 or logits.stride(0) < E:
        logits = logits.contiguous()
    new = lambda *shape: torch.empty(shape, dtype=torch.int32, device=logits.device)  # noqa: E731
    weights, experts, offsets, order, place = torch.empty((T, k), dtype=torch.float32, device=logits.device), new(T, k), new(E + 1), new(T * k), new(T, k)
    if T == 0:
        offsets.zero_()
        return weights, experts, offsets, order, place
    L = _lib.lib()
    nbytes = L.sk_route_workspace_bytes(T, E, k)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=logits.device) if nbytes else None
    rc = L.sk_route_experts(logits.data_ptr(), _LOGITS[logits.dtype], T, E, k, max(logits.stride(0), E), weights.data_ptr(), experts.data_ptr(),
                            offsets.data_ptr(), order.data_ptr(), place.data_ptr(), ws.data_ptr() if nbytes else None, nbytes, ops._stream_ptr())
    _lib.check(rc, "sk_route_experts")
    return weights, experts, offsets, order, place


def _route_fake(logits, k):
    T, E = logits.shape
    new = lambda *shape: logits.new_empty(shape, dtype=torch.int32)  # noqa: E731
    return logits.new_empty((T, k), dtype=torch.float32), new(T, k), new(E + 1), new(T * k), new(T, k)


def _route_backward(weights, experts, dweights, E, dtype):
    T, k = weights.shape
    dlogits = torch.empty((T, E), dtype=dtype, device=weights.device)
    if T:
        rc = _lib.lib().sk_route_backward(weights.data_ptr(), experts.data_ptr(), dweights.contiguous().data_ptr(), T, E, k, _LOGITS[dtype],
                                          dlogits.data_ptr(), ops._stream_ptr())
        _lib.check(rc, "sk_route_backward")
    return dlogits


_operator("route_experts", "(Tensor logits, int k) -> (Tensor, Tensor, Tensor, Tensor, Tensor)", _route, _route_fake)
_operator("route_backward", "(Tensor weights, Tensor experts, Tensor dweights, int E, ScalarType dtype) -> Tensor", _route_backward,
          lambda weights, experts, dweights, E, dtype: weights.new_empty((weights.shape[0], E), dtype=dtype))


class _RouteExperts(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, k):
        out = _ops.route_experts(logits, k)
        ctx.save_for_backward(out[0], out[1])
        ctx.E, ctx.dtype = logits.shape[1], logits.dtype
        ctx.mark_non_differentiable(*out[1:])
        return tuple(out)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dweights, *_):
        weights, experts = ctx.saved_tensors
        return _ops.route_backward(weights, experts, dweights, ctx.E, ctx.dtype), None


def route_experts(logits, k):
    """Route of the tokens whose router logits are [T, E] (float32, float16 or bfloat16): the k largest of each, the largest first, equal
    ones by number.  -inf and NaN are never chosen: a token with fewer others has -1 and weight 0 in its last places, and one with none
    goes to no expert.  Differentiable: weights to logits."""
    if not _NATIVE:
        _no_tangent("route_experts", logits)
    if not _NATIVE and torch.is_grad_enabled() and isinstance(logits, torch.Tensor) and logits.requires_grad:
        return Route(*_RouteExperts.apply(logits, k))
    return Route(*_route_experts(logits, k))


def _dispatch(x, order, k, place=None):
    if not isinstance(x, torch.Tensor) or not x.is_cuda or x.dim() not in (1, 2):
        raise TypeError("x must be a CUDA/HIP tensor of one or two dimensions")
    _on_device(order, "order", (torch.int32,), 1)
    T = x.shape[0]
    if order.shape[0] != T * k or not order.is_contiguous() or order.device != x.device:
        raise ValueError(f"order must have T k = {T * k} elements on {x.device}, got {tuple(order.shape)} on {order.device}")
    out = torch.empty((T * k, *x.shape[1:]), dtype=x.dtype, device=x.device)
    if out.numel() == 0:
        return out
    if place is not None and (place.dtype != torch.int32 or tuple(place.shape) != (T, k) or not place.is_contiguous() or place.device != x.device):
        raise ValueError(f"place must be contiguous int32 {(T, k)} on {x.device}")
    if x.dim() == 2 and (x.stride(1) != 1 and x.shape[1] > 1 or x.stride(0) < x.shape[1]) or x.dim() == 1 and x.stride(0) < 1:
        x = x.contiguous()
    size = x.element_size()
    row_bytes = size * (x.shape[1] if x.dim() == 2 else 1)
    pitch = size * x.stride(0) if T > 1 else row_bytes
    rc = _lib.lib().sk_dispatch_rows(x.data_ptr(), row_bytes, pitch, order.data_ptr(), place.data_ptr() if place is not None else None, T, k, out.data_ptr(),
                                     ops._stream_ptr())
    _lib.check(rc, "sk_dispatch_rows")
    return out


def _combine(y, place, weights=None):
    _on_device(y, "y", tuple(_TYPES), 2)
    _on_device(place, "place", (torch.int32,), 2)
    T, k = place.shape
    if y.shape[0] != T * k or not place.is_contiguous() or place.device != y.device:
        raise ValueError(f"y must have T k = {T * k} rows on the device of place, got {tuple(y.shape)}")
    if weights is not None and (weights.dtype != torch.float32 or weights.shape != place.shape or not weights.is_contiguous() or weights.device != y.device):
        raise ValueError(f"weights must be contiguous float32 {tuple(place.shape)} on {y.device}")
    out = torch.empty((T, y.shape[1]), dtype=y.dtype, device=y.device)
    if out.numel() == 0:
        return out
    y = y.contiguous()
    rc = _lib.lib().sk_combine_rows(y.data_ptr(), _TYPES[y.dtype], place.data_ptr(), weights.data_ptr() if weights is not None else None, T, k, y.shape[1],
                                    out.data_ptr(), ops._stream_ptr())
    _lib.check(rc, "sk_combine_rows")
    return out


def _combine_backward(d_out, y, order, place, weights):
    T, k = place.shape
    d_out, y = d_out.contiguous(), y.contiguous()
    dy, dweights = torch.empty_like(y), torch.empty_like(weights)
    if y.numel() == 0:
        return dy, dweights.zero_()
    rc = _lib.lib().sk_combine_backward(d_out.data_ptr(), y.data_ptr(), _TYPES[y.dtype], order.data_ptr(), place.data_ptr(), weights.data_ptr(), T, k,
                                        y.shape[1], dy.data_ptr(), dweights.data_ptr(), ops._stream_ptr())
    _lib.check(rc, "sk_combine_backward")
    return dy, dweights


_dispatch_fake = lambda x, order, k: x.new_empty((order.shape[0], *x.shape[1:]))  # noqa: E731
_combine_fake = lambda y, place, weights=None: y.new_empty((place.shape[0], y.shape[1]))  # noqa: E731
_operator("dispatch_rows", "(Tensor x, Tensor order, int k) -> Tensor", _dispatch, _dispatch_fake)
_operator("combine_rows", "(Tensor y, Tensor place, Tensor? weights=None) -> Tensor", _combine, _combine_fake)
_operator("combine_backward", "(Tensor d_out, Tensor y, Tensor order, Tensor place, Tensor weights) -> (Tensor, Tensor)", _combine_backward,
          lambda d_out, y, order, place, weights: (y.new_empty(y.shape), weights.new_empty(weights.shape)))
# the same with all of a route that their gradients need
_operator("dispatch_routed", "(Tensor x, Tensor order, Tensor place) -> Tensor", lambda x, order, place: _dispatch(x, order, place.shape[1], place),
          lambda x, order, place: _dispatch_fake(x, order, place.shape[1]))
_operator("combine_routed", "(Tensor y, Tensor weights, Tensor order, Tensor place) -> Tensor",
          lambda y, weights, order, place: _combine(y, place, weights), lambda y, weights, order, place: _combine_fake(y, place))


class _DispatchRows(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, order, place):
        ctx.save_for_backward(place)
        return _ops.dispatch_rows(x, order, place.shape[1])

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, d_rows):
        place, = ctx.saved_tensors
        return _ops.combine_rows(d_rows, place), None, None


class _CombineRows(torch.autograd.Function):
    @staticmethod
    def forward(ctx, y, weights, order, place):
        ctx.save_for_backward(y, weights, order, place)
        return _ops.combine_rows(y, place, weights)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, d_out):
        y, weights, order, place = ctx.saved_tensors
        return (*_ops.combine_backward(d_out, y, order, place, weights), None, None)


def dispatch_rows(x, route):
    """The tokens' rows in the experts' order: [T k, H] for x [T, H] of any type (or [T k] for [T], such as the tokens' scales); zeros for
    the rows behind route.offsets[E].  Differentiable in x (float16 or bfloat16, two dimensions)."""
    if not _NATIVE:
        _no_tangent("dispatch_rows", x)
    if torch.is_grad_enabled() and isinstance(x, torch.Tensor) and x.requires_grad:
        _on_device(x, "x", tuple(_TYPES), 2)
        if not _NATIVE:
            return _DispatchRows.apply(x, route.order, route.place)
    return _dispatch_routed(x, route.order, route.place)


def combine_rows(y, route):
    """out[t] = sum over its experts of their weight times their row of y: [T, H] for y [T k, H] (float16 or bfloat16) in the experts' order;
    added in fp32, rounded once; a token without experts gets zeros.  Differentiable in y and route.weights."""
    if not _NATIVE:
        _no_tangent("combine_rows", y, route.weights)
    if not _NATIVE and torch.is_grad_enabled() and isinstance(y, torch.Tensor) and (y.requires_grad or route.weights.requires_grad):
        return _CombineRows.apply(y, route.weights, route.order, route.place)
    return _combine_routed(y, route.weights, route.order, route.place)


# (the overloads themselves: a call through the packet looks them up)
_gemm_grouped, _route_experts = _ops.gemm_grouped.default, _ops.route_experts.default
_dispatch_routed, _combine_routed = _ops.dispatch_routed.default, _ops.combine_routed.default
