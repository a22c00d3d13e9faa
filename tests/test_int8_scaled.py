"""int8 products with a scale for each token and output channel, and the row quantiser, against 64-bit arithmetic.

Tolerances: the int32 sums are exact; what is left is the conversion, two products and the bias in fp32 (relative 2^-22 of the value in
front of the activation, the fast exponential of silu and gelu included: 4e-6 of it and of one) and one rounding to C's type (2^-8 of
bfloat16, 2^-11 of fp16, 2^-24 absolute below fp16's normal numbers)."""
import ctypes
import math

import pytest
import torch

TYPES = {"float16": torch.float16, "bfloat16": torch.bfloat16}
ROUNDING = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


@pytest.fixture(scope="module")
def sk():
    import streamk
    streamk.lib()
    return streamk


def activate(x, name):
    return {None: lambda v: v, "relu": torch.relu, "silu": lambda v: v * torch.sigmoid(v),
            "gelu_tanh": lambda v: 0.5 * v * (1 + torch.tanh(math.sqrt(2 / math.pi) * (v + 0.044715 * v ** 3)))}[name](x)


def assert_scaled(C, pre, activation):
    want = activate(pre, activation)
    tol = ROUNDING[C.dtype] * want.abs() * 1.001 + 4e-6 * (pre.abs() + 1) + 2.0 ** -24
    off = (C.double() - want).abs()
    assert torch.isfinite(C).all()
    assert (off <= tol).all(), f"largest excess {(off - tol).max().item():.3g} at {int((off - tol).argmax())}"


def operands(M, N, K, seed):
    g = torch.Generator().manual_seed(seed)
    A = torch.randint(-127, 128, (M, K), generator=g, dtype=torch.int8).cuda()
    B = torch.randint(-127, 128, (N, K), generator=g, dtype=torch.int8).cuda()
    sa = (torch.rand(M, generator=g) + 0.5).cuda() * 0.01
    sb = (torch.rand(N, generator=g) + 0.5).cuda() / (73 * math.sqrt(K))
    return A, B, sa, sb


def product(A, B, sa, sb):
    return (A.double() @ B.double().T) * sa.double()[:, None] * sb.double()


# ---- on the CPU: refusals of the C ABI ----
def test_calls_are_refused_with_codes(sk):
    L, lib = sk.lib(), __import__("streamk._lib", fromlist=["x"])
    plan = sk.make_plan(64, 256, 256, "int8", "nt", cus=256, variant=12)
    sc = lib.SkScales(a=1 << 12, b=1 << 12, out_dtype=lib.SK_BF16)
    p = 1 << 12   # (an aligned address; every call below is refused before it is used)

    def call(A=p, B=p, C=p, K=256, lda=256, ldb=256, ldc=256, scales=sc, plan=plan):
        return L.sk_gemm_i8_scaled(A, B, C, 64, 256, K, lda, ldb, ldc, ctypes.byref(scales) if scales else None, ctypes.byref(plan), None, 0, None, None)
    assert call(A=None) == -1 and call(scales=None) == -1 and call(scales=lib.SkScales(a=None, b=p, out_dtype=0)) == -1
    assert call(scales=lib.SkScales(a=p, b=p, out_dtype=lib.SK_F32)) == -4
    assert call(scales=lib.SkScales(a=p, b=p, out_dtype=0, reserved=1)) == -4
    assert call(K=128) == -4                      # not the plan's
    assert call(lda=128) == -2 and call(ldc=255) == -2
    assert call(A=p + 8) == -3 and call(lda=264) == -3
    assert call(scales=lib.SkScales(a=p + 2, b=p, out_dtype=0)) == -3
    assert L.sk_quantize_i8(p, lib.SK_F32, 4, 64, 64, p, 64, p, None) == -4
    assert L.sk_quantize_i8(None, lib.SK_F16, 4, 64, 64, p, 64, p, None) == -1
    assert L.sk_quantize_i8(p, lib.SK_F16, 0, 64, 64, p, 64, p, None) == -2
    assert L.sk_quantize_i8(p, lib.SK_F16, 4, 64, 63, p, 64, p, None) == -2
    assert L.sk_quantize_i8(p + 1, lib.SK_F16, 4, 64, 64, p, 64, p, None) == -3


def test_fake_implementations(sk):
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        x = torch.empty(3, 5, 64, dtype=torch.bfloat16, device="cuda")
        q, s = torch.ops.streamk.quantize_i8(x)
        assert q.shape == x.shape and q.dtype == torch.int8 and s.shape == (3, 5) and s.dtype == torch.float32
        C = torch.ops.streamk.gemm_i8_scaled(q.view(15, 64), torch.empty(32, 64, dtype=torch.int8, device="cuda"), s.view(15),
                                             torch.empty(32, device="cuda"), torch.bfloat16)
        assert C.shape == (15, 32) and C.dtype == torch.bfloat16


# ---- the quantiser ----
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("M,K", [(1, 16), (3, 4096), (130, 1000), (7, 1), (5, 17), (2, 16392), (2, 40001), (300, 256)])
def test_quantiser(sk, dtype, M, K):
    g = torch.Generator().manual_seed(M + K)
    x = (torch.randn(M, K, generator=g) * torch.logspace(-6, 4, M)[:, None]).to(TYPES[dtype]).cuda()
    q, s = sk.quantize_int8(x)
    amax = x.double().abs().amax(1)
    assert torch.equal(s, (amax / 127).float())   # (in 64 bits: on the device torch divides by a number with its reciprocal)
    # nearest integer to x / s, ties to even, exactly
    want = torch.where(s[:, None] > 0, torch.round(x.double() / s.double()[:, None].clamp(min=1e-300)), 0).clamp(-127, 127)
    assert torch.equal(q.double(), want)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", sorted(TYPES))
def test_quantiser_rows_that_are_not_ordinary(sk, dtype):
    t = TYPES[dtype]
    x = torch.zeros(9, 64, dtype=t, device="cuda")
    x[1, 5] = math.inf
    x[2, 6] = math.nan
    x[3, 7] = -math.inf
    x[4] = torch.finfo(t).max
    x[5, :3] = torch.tensor([127, 0.5, -1.5])     # scale 1: ties to even
    x[6, 1] = torch.finfo(t).smallest_normal / 64   # a subnormal alone
    x[7] = -torch.finfo(t).max
    x[8, :2] = torch.tensor([-127, 2.5])
    q, s = sk.quantize_int8(x)
    assert s[0] == 0 and not q[0].any()
    for r in (1, 2, 3):
        assert torch.isnan(s[r]) and not q[r].any()
    assert (q[4] == 127).all() and (q[7] == -127).all()
    assert q[5, :3].tolist() == [127, 0, -2] and q[8, :2].tolist() == [-127, 2]
    assert torch.equal(s[6], (x[6].double().max() / 127).float())
    # strides, leading dimensions, nothing
    wide = torch.randn(6, 200, device="cuda").to(t)
    for v in (wide[:, 3:67], wide[::2], wide.t(), wide.view(2, 3, 200), wide[:, 8:136]):
        q, s = sk.quantize_int8(v)
        qc, sc = sk.quantize_int8(v.contiguous())
        assert torch.equal(q, qc) and torch.equal(s, sc) and q.shape == v.shape and s.shape == v.shape[:-1]
    q, s = sk.quantize_int8(wide[:0])
    assert q.shape == (0, 200) and s.shape == (0,)
    with pytest.raises(TypeError):
        sk.quantize_int8(wide.float())


# ---- the product ----
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("M,N,K", [(1, 16, 16), (1, 4096, 4096), (2, 1, 256), (7, 130, 272), (16, 513, 1040), (33, 300, 512), (64, 2048, 2048), (65, 1000, 528),
                                   (100, 1111, 4096), (128, 512, 8192), (257, 777, 1024), (1000, 1031, 2064), (2048, 2048, 1024), (2300, 4100, 512)])
def test_product(sk, dtype, M, N, K):
    A, B, sa, sb = operands(M, N, K, M * N + K)
    C = sk.streamk_int8_scaled(A, B, sa, sb, out_dtype=TYPES[dtype])
    assert_scaled(C, product(A, B, sa, sb), None)


@pytest.mark.gpu
@pytest.mark.parametrize("activation", [None, "relu", "gelu_tanh", "silu"])
@pytest.mark.parametrize("M", [1, 20, 100, 700])
def test_epilogue(sk, M, activation):
    N, K = 515, 512
    A, B, sa, sb = operands(M, N, K, M)
    bias = torch.randn(N, device="cuda").bfloat16()
    C = sk.streamk_int8_scaled(A, B, sa, sb, out_dtype=torch.bfloat16, bias=bias, activation=activation)
    assert_scaled(C, product(A, B, sa, sb) + bias.double(), activation)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("activation", [None, "relu", "gelu_tanh", "silu"])
@pytest.mark.parametrize("with_bias", [False, True])
def test_every_tile_rounds_alike(sk, dtype, activation, with_bias):
    M, N, K = 300, 520, 768
    A, B, sa, sb = operands(M, N, K, 9)
    bias = torch.randn(N, device="cuda").to(TYPES[dtype]) if with_bias else None
    run = lambda **config: sk.streamk_int8_scaled(A, B, sa, sb, out_dtype=TYPES[dtype], bias=bias, activation=activation, **config)  # noqa: E731
    want = run(bm=64, bn=64, variant=11)
    assert_scaled(want, product(A, B, sa, sb) + (bias.double() if with_bias else 0), activation)
    for config in (dict(bm=256, bn=256), dict(bm=128, bn=128, bk=64), dict(bm=128, bn=128, bk=128), dict(bm=64, bn=128, bk=64), dict(bm=128, bn=64, variant=11)):
        assert torch.equal(run(**config), want), config


@pytest.mark.gpu
@pytest.mark.parametrize("config", [dict(variant=9), dict(variant=12), dict(bm=128, bn=128), dict(bm=64, bn=128, bk=64), dict(bm=256, bn=256), dict(bm=256, bn=256, schedule="splitk", split=2),
                                    dict(bm=128, bn=128, schedule="splitk", split=4), dict(bm=64, bn=64, variant=11),
                                    dict(bm=128, bn=128, schedule="basic", grid=24, fixup="atomic")])
def test_every_kernel_and_fix_up_gives_the_same_bits(sk, config):
    M, N, K = 60, 520, 2048
    A, B, sa, sb = operands(M, N, K, 5)
    bias = torch.randn(N, device="cuda").half()
    want = sk.streamk_int8_scaled(A, B, sa, sb, bias=bias, activation="silu")
    assert_scaled(want, product(A, B, sa, sb) + bias.double(), "silu")
    assert torch.equal(sk.streamk_int8_scaled(A, B, sa, sb, bias=bias, activation="silu", **config), want)
    sk.workspace_status()


@pytest.mark.gpu
def test_views_and_out(sk):
    A, B, sa, sb = operands(40, 304, 512, 9)
    want = sk.streamk_int8_scaled(A, B, sa, sb)
    wide_a, wide_b = torch.zeros(40, 640, dtype=torch.int8, device="cuda"), torch.zeros(304, 544, dtype=torch.int8, device="cuda")
    wide_a[:, 64:576], wide_b[:, :512] = A, B
    assert torch.equal(sk.streamk_int8_scaled(wide_a[:, 64:576], wide_b[:, :512], sa, sb), want)
    shifted = torch.zeros(40, 513, dtype=torch.int8, device="cuda")
    shifted[:, 1:] = A
    assert torch.equal(sk.streamk_int8_scaled(shifted[:, 1:], B, sa, sb), want)   # (copied: its rows are not aligned)
    out = torch.full((40, 321), 7.0, dtype=torch.float16, device="cuda")
    assert sk.streamk_int8_scaled(A, B, sa, sb, out=out[:, 3:307]).data_ptr() == out[:, 3:307].data_ptr()
    assert torch.equal(out[:, 3:307], want) and (out[:, :3] == 7).all() and (out[:, 307:] == 7).all()
    assert sk.streamk_int8_scaled(A[:0], B, sa[:0], sb).shape == (0, 304)


@pytest.mark.gpu
def test_infinite_and_nan_scales_reach_their_rows_and_columns_only(sk):
    A, B, sa, sb = operands(5, 70, 256, 2)
    sa[1], sb[3] = math.nan, math.nan
    C = sk.streamk_int8_scaled(A, B, sa, sb)
    bad = torch.isnan(C)
    want = torch.zeros_like(bad)
    want[1], want[:, 3] = True, True
    assert torch.equal(bad, want)


@pytest.mark.gpu
def test_wrong_operands_are_refused(sk):
    A, B, sa, sb = operands(8, 32, 64, 1)
    f = sk.streamk_int8_scaled
    for args, kw, error in [((A.float(), B, sa, sb), {}, TypeError), ((A, B[:, :32], sa, sb), {}, ValueError), ((A, B, sa[:7], sb), {}, ValueError),
                            ((A, B, sa.half(), sb), {}, ValueError), ((A, B, sa, sb.cpu()), {}, ValueError), ((A, B, sa, sb), dict(out_dtype=torch.float32), ValueError),
                            ((A, B, sa, sb), dict(activation="tanh"), ValueError), ((A, B, sa, sb), dict(bias=torch.zeros(32, device="cuda")), ValueError),
                            ((A[:, :24], B[:, :24], sa, sb), {}, sk.StreamKError), ((A, B, sa, sb), dict(out=torch.empty(8, 31, device="cuda").half()), ValueError),
                            ((A, B, sa, sb), dict(variant=1), sk.StreamKError)]:
        with pytest.raises(error):
            f(*args, **kw)


@pytest.mark.gpu
def test_linear_layer_in_a_graph(sk):
    """Quantiser and product captured once and replayed on new inputs, with eager work between the replays."""
    torch.manual_seed(0)
    w = torch.randn(512, 1024, device="cuda").half()
    qw, sw = sk.quantize_int8(w)
    x = torch.randn(4, 1024, device="cuda").half()

    def layer():
        q, s = sk.quantize_int8(x)
        return sk.streamk_int8_scaled(q, qw, s, sw)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        layer()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        out = layer()
    for i in range(4):
        x.copy_(torch.randn(4, 1024, device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, layer())
