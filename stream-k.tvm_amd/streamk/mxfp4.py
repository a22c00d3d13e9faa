"""Microscaled 4-bit floating point: a row is bytes of two e2m1 values (the first in the low half) and, for each 32 values, the biased exponent
of a power of two that they are multiplied by.

`quantize_mxfp4(x)` and `streamk_mxfp4(q, Wq, scale, weight_scale)` are the two halves of a linear layer on it
(`StreamKLinear(weight_format="mxfp4")`), `streamk_grouped` takes such operands for layers of experts; registered as
`torch.ops.streamk.quantize_mxfp4`, `dequantize_mxfp4` and `gemm_mxfp4`.  Inference only, as the library's other quantised products.
"""
import torch

from . import _lib, experts, ops

_FLOATS = {torch.float16: _lib.SK_F16, torch.bfloat16: _lib.SK_BF16, torch.float32: _lib.SK_F32}


@experts._where_it_is
def _quantize(x):
    if not isinstance(x, torch.Tensor) or x.dtype not in _FLOATS:
        raise TypeError("x must be a float16, bfloat16 or float32 tensor")
    if x.dim() < 1 or x.shape[-1] % 32:
        raise ValueError(f"the last dimension of x must be a multiple of 32, got {tuple(x.shape)}")
    K = x.shape[-1]
    q = torch.empty((*x.shape[:-1], K // 2), dtype=torch.uint8, device=x.device)
    scale = torch.empty((*x.shape[:-1], K // 32), dtype=torch.uint8, device=x.device)
    if scale.numel() == 0:
        return q, scale
    rows = x.reshape(-1, K)
    if rows.stride(1) != 1:
        rows = rows.contiguous()
    pitch = rows.stride(0) if rows.shape[0] > 1 else K
    if pitch < K:   # (a row that stands for many)
        rows, pitch = rows.contiguous(), K
    rc = _lib.lib().sk_quantize_mxfp4(rows.data_ptr(), _FLOATS[x.dtype], rows.shape[0], K, pitch, q.data_ptr(), scale.data_ptr(), ops._stream_ptr())
    _lib.check(rc, "sk_quantize_mxfp4")
    return q, scale


@experts._where_it_is
def _dequantize(q, scale, dtype):
    if not isinstance(q, torch.Tensor) or not q.is_cuda or q.dtype != torch.uint8:
        raise TypeError("q must be a CUDA/HIP tensor of bytes (uint8)")
    if dtype not in _FLOATS:
        raise ValueError("dtype must be torch.float16, torch.bfloat16 or torch.float32")
    if q.dim() < 1 or q.shape[-1] % 16:
        raise ValueError(f"the last dimension of q must be a multiple of 16 bytes, got {tuple(q.shape)}")
    K = 2 * q.shape[-1]
    if not isinstance(scale, torch.Tensor) or scale.dtype != torch.uint8 or tuple(scale.shape) != (*q.shape[:-1], K // 32) or scale.device != q.device:
        raise ValueError(f"scale must be uint8 {(*q.shape[:-1], K // 32)} on {q.device}")
    x = torch.empty((*q.shape[:-1], K), dtype=dtype, device=q.device)
    if x.numel() == 0:
        return x
    q, scale = q.contiguous(), scale.contiguous()
    if q.data_ptr() % 4:   # (a view that begins inside a word)
        q = q.clone()
    rc = _lib.lib().sk_dequantize_mxfp4(q.data_ptr(), scale.data_ptr(), x.numel() // K, K, _FLOATS[dtype], x.data_ptr(), ops._stream_ptr())
    _lib.check(rc, "sk_dequantize_mxfp4")
    return x


experts._operator("quantize_mxfp4", "(Tensor x) -> (Tensor, Tensor)", _quantize,
                  lambda x: (x.new_empty((*x.shape[:-1], x.shape[-1] // 2), dtype=torch.uint8), x.new_empty((*x.shape[:-1], x.shape[-1] // 32), dtype=torch.uint8)))
experts._operator("dequantize_mxfp4", "(Tensor q, Tensor scale, ScalarType dtype) -> Tensor", _dequantize,
                  lambda q, scale, dtype: q.new_empty((*q.shape[:-1], 2 * q.shape[-1]), dtype=dtype))

_TAIL = "str activation=\"none\", int variant=0"


def _product(A, B, scale_a, scale_b, out_dtype, bias=None, activation="none", variant=0):
    return experts._mx_product(A, B, None, scale_a, scale_b, out_dtype, bias, activation, variant, None)


def _product_out(A, B, scale_a, scale_b, out, bias=None, activation="none", variant=0):
    experts._mx_product(A, B, None, scale_a, scale_b, out.dtype, bias, activation, variant, out)


experts._operator("gemm_mxfp4", f"(Tensor A, Tensor B, Tensor scale_a, Tensor scale_b, ScalarType out_dtype, Tensor? bias=None, {_TAIL}) -> Tensor", _product,
                  lambda A, B, scale_a, scale_b, out_dtype, *rest: A.new_empty((A.shape[0], B.shape[0]), dtype=out_dtype))
experts._operator("gemm_mxfp4_out", f"(Tensor A, Tensor B, Tensor scale_a, Tensor scale_b, Tensor(a!) out, Tensor? bias=None, {_TAIL}) -> ()", _product_out,
                  lambda *args: None)


def quantize_mxfp4(x):
    """(q uint8 [..., K / 2], scale uint8 [..., K / 32]) of x [..., K] (float16, bfloat16 or float32, K a multiple of 32): of each 32
    neighbours scale = floor(log2 max |x|) + 125, at least 0, and each x / 2^(scale - 127) becomes the nearest of 0, .5, 1, 1.5, 2, 3, 4, 6 (ties to
    the even code) with its sign; what is above 6 becomes 6.  A block with an infinity or a NaN has scale 255 and codes 0: its values,
    and the products with them, are NaN."""
    return _quantize_mxfp4(x)


def dequantize_mxfp4(q, scale, dtype=torch.bfloat16):
    """The values [..., K] of q [..., K / 2] and scale [..., K / 32] in `dtype` (float16, bfloat16 or float32), rounded where it has no such
    number."""
    return _dequantize_mxfp4(experts._bytes(q), experts._bytes(scale), dtype)


def streamk_mxfp4(A, B, scale_a, scale_b, *, out_dtype=torch.float16, out=None, bias=None, activation=None, variant=0):
    """C = activation(A @ B.T + bias) for microscaled 4-bit A [M, K / 2] and B [N, K / 2] (uint8) with scale_a [M, K / 32] and scale_b
    [N, K / 32] (uint8), as quantize_mxfp4 makes them; K a multiple of 32.  C is float16 or bfloat16 (`out_dtype`, which bias shares),
    summed in fp32 and rounded once.  With more than some dozen rows and a K that is no multiple of 128, or hundreds of
    rows, scales are laid out anew on the way (sk_tile_mx_scales in streamk.h).  variant: which tiles run (sk_grouped in streamk.h); 0 lets the sizes decide."""
    A, B, scale_a, scale_b = (experts._bytes(t) for t in (A, B, scale_a, scale_b))
    if out is None:
        return _gemm_mxfp4(A, B, scale_a, scale_b, out_dtype, bias, activation or "none", variant)
    torch.ops.streamk.gemm_mxfp4_out(A, B, scale_a, scale_b, out, bias, activation or "none", variant)
    return out


# (the overloads themselves: a call through the packet looks them up)
_quantize_mxfp4, _dequantize_mxfp4 = torch.ops.streamk.quantize_mxfp4.default, torch.ops.streamk.dequantize_mxfp4.default
_gemm_mxfp4 = torch.ops.streamk.gemm_mxfp4.default
