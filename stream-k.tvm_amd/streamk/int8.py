"""int8 products with a scale for each token and output channel, and the quantiser of the tokens' rows.

`quantize_int8(x)` and `streamk_int8_scaled(q, Wq, scale, weight_scale)` are the two halves of a linear layer with int8 weights and
activations (`StreamKLinear(weight_format="int8")`); registered as `torch.ops.streamk.quantize_i8` and `gemm_i8_scaled`.  Inference
only, as the library's other products.
"""
import ctypes

import torch

from . import _lib, ops

_OUT_TYPES = {torch.float16: _lib.SK_F16, torch.bfloat16: _lib.SK_BF16}


def _check_scale(t, name, n, device):
    if not isinstance(t, torch.Tensor) or t.dtype != torch.float32 or tuple(t.shape) != (n,) or not t.is_contiguous() or t.device != device:
        raise ValueError(f"{name} must be a contiguous float32 vector of {n} elements on {device}")


def _check_out_dtype(dtype):
    if dtype not in _OUT_TYPES:
        raise ValueError("out_dtype must be torch.float16 or torch.bfloat16")


def plan_for(config, M, N, K, pitch_a=0, pitch_b=0):
    """The plan of an int8 product with scales: that of the int32 product, but for tuned entries of kernels that have no form with
    scales (a search of up to 64 rows may end with one), which do not count here."""
    plan = ops._plan_for(config, M, N, K, "int8", "nt", pitch_a, pitch_b)
    if config != "" or _lib.lib().sk_i8_scaled_takes(ctypes.byref(plan)):
        return plan
    plan = ops._plan_of(ops._UNTUNED, M, N, K, "int8", "nt")
    return plan if ops._takes_rows(plan, pitch_a, pitch_b) else ops._plan_of(ops._UNTUNED_LONG_ROWS, M, N, K, "int8", "nt")


def _run_i8_scaled(A, B, scale_a, scale_b, C, out_dtype, config="", bias=None, activation="none"):
    _check_out_dtype(out_dtype)
    A = ops._aligned_rows(A)
    ops._check_matrix(A, "A", torch.int8)
    ops._check_matrix(B, "B", torch.int8)
    M, K = A.shape
    N, Kb = B.shape
    if K != Kb:
        raise ValueError(f"K mismatch: A is {tuple(A.shape)}, B is {tuple(B.shape)}")
    _check_scale(scale_a, "scale_a", M, A.device)
    _check_scale(scale_b, "scale_b", N, A.device)
    ops._check_out(C, M, N, out_dtype)
    plan = plan_for(config, M, N, K, A.stride(0), B.stride(0))
    epi = ops._epilogue(bias, N, out_dtype, A.device, ops._act(activation))
    scales = _lib.SkScales(a=scale_a.data_ptr(), b=scale_b.data_ptr(), out_dtype=_OUT_TYPES[out_dtype])
    rc = _lib.lib().sk_gemm_i8_scaled(A.data_ptr(), B.data_ptr(), C.data_ptr(), M, N, K, A.stride(0), B.stride(0), C.stride(0),
                                      ctypes.byref(scales), *ops._ws_args(plan, A.device), ctypes.byref(epi) if epi is not None else None)
    _lib.check(rc, "sk_gemm_i8_scaled")


ops._register("gemm_i8_scaled", "Tensor A, Tensor B, Tensor scale_a, Tensor scale_b", f"ScalarType out_dtype, str config=\"\", {ops._EPI}",
              _run_i8_scaled, lambda A, B, sa, sb, out_dtype, *rest: ((A.shape[0], B.shape[0]), out_dtype))


def _check_quantised(x):
    if not isinstance(x, torch.Tensor) or x.dtype not in _OUT_TYPES:
        raise TypeError("x must be a float16 or bfloat16 tensor")
    if x.dim() < 1:
        raise ValueError("x must have at least one dimension")


def _quantize(x):
    _check_quantised(x)
    K = x.shape[-1]
    q = torch.empty(x.shape, dtype=torch.int8, device=x.device)
    scale = torch.empty(x.shape[:-1], dtype=torch.float32, device=x.device)
    if scale.numel() == 0:
        return q, scale
    if K == 0:
        return q, scale.zero_()
    rows = x.reshape(-1, K)
    if rows.stride(1) != 1 and K > 1:
        rows = rows.contiguous()
    pitch = rows.stride(0) if rows.shape[0] > 1 else K
    if pitch < K:   # (a row that stands for many)
        rows, pitch = rows.contiguous(), K
    rc = _lib.lib().sk_quantize_i8(rows.data_ptr(), _OUT_TYPES[x.dtype], rows.shape[0], K, pitch, q.data_ptr(), K, scale.data_ptr(), ops._stream_ptr())
    _lib.check(rc, "sk_quantize_i8")
    return q, scale


for _suffix in ("", "_general"):   # (the native implementation passes what is not ordinary on)
    ops._LIBRARY.define(f"quantize_i8{_suffix}(Tensor x) -> (Tensor, Tensor)")
    if _suffix or _lib.torch_lib() is None:
        ops._LIBRARY.impl("quantize_i8" + _suffix, _quantize, "CUDA")
torch.library.register_fake("streamk::quantize_i8", lambda x: (x.new_empty(x.shape, dtype=torch.int8), x.new_empty(x.shape[:-1], dtype=torch.float32)),
                            lib=ops._LIBRARY)


def quantize_int8(x):
    """(q int8, scale float32) of the rows of x [..., K] (float16 or bfloat16): scale = max |x| / 127 of each row, q = x / scale to the
    nearest integer (ties to even).  A row of zeros has scale 0; a row with an infinity or a NaN scale NaN and q = 0, so that its
    products are NaN."""
    return _quantize_i8(x)


def streamk_int8_scaled(A, B, scale_a, scale_b, *, out_dtype=torch.float16, out=None, plan=None, config=None, bias=None, activation=None, **kw):
    """C = activation(scale_a[:, None] * scale_b * (A @ B.T) + bias) for int8 A [M, K] and B [N, K]: exact int32 sums (whatever the
    values up to K = 131071), scales float32
    [M] and [N], C float16 or bfloat16 (`out_dtype`, which bias shares), rounded once.  Plans are those of streamk_int8; up to 64
    rows those that operator calls take."""
    cfg = ops._config_string(plan, config, kw)
    if out is None:
        return _gemm_i8_scaled(A, B, scale_a, scale_b, out_dtype, cfg, bias, activation or "none")
    torch.ops.streamk.gemm_i8_scaled_out(A, B, scale_a, scale_b, out, out.dtype, cfg, bias, activation or "none")
    return out


# (the overloads themselves: a call through the packet looks them up)
_quantize_i8, _gemm_i8_scaled = torch.ops.streamk.quantize_i8.default, torch.ops.streamk.gemm_i8_scaled.default
