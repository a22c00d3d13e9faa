"""Microscaled 4-bit floating point against the definition in 64 bits: quantiser, values, products, products by expert.

Quantised codes and scales, and the values they stand for, are compared bit for bit.  Products: every term, two e2m1 numbers and two powers of
two, is exact; fp32 sums of n terms, in any order, are within 2 n 2^-24 of the sum of the terms' magnitudes (an MFMA may cut instead of
rounding: hence the 2), plus one rounding to the result's type (2^-8 of bfloat16, 2^-11 of fp16, 2^-24 absolute below fp16's normal
numbers); bias and activation as in the other tests of products: 4e-6 of the value in front of the activation and of one."""
import ctypes
import itertools
import math

import pytest
import torch

TYPES = {"float16": torch.float16, "bfloat16": torch.bfloat16, "float32": torch.float32}
ROUNDING = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
E2M1 = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)


@pytest.fixture(scope="module")
def sk():
    import streamk
    streamk.lib()
    return streamk


def plain_quantize(x):
    """(codes, scales) of x on the CPU, the nearest of all codes by its distance"""
    blocks = x.detach().double().cpu().reshape(*x.shape[:-1], -1, 32)
    most = blocks.abs().amax(-1)
    finite = torch.isfinite(blocks).all(-1)
    exponent = torch.where(finite & (most > 0), torch.frexp(torch.where(finite, most, 1.0)).exponent - 1 - 2, -127).clamp(min=-127)
    y = torch.where(finite[..., None], blocks, 0.0) / torch.pow(2.0, exponent.double())[..., None]
    distance = (y.abs().clamp(max=6.0)[..., None] - E2M1).abs()
    least = distance.amin(-1, keepdim=True)
    # (of two at the same distance the even code)
    code = torch.where(distance == least, torch.arange(8) + 8 * (torch.arange(8) % 2), 99).amin(-1) % 8
    code = torch.where(finite[..., None], code + 8 * torch.signbit(y), 0).flatten(-2)
    return (code[..., 0::2] + 16 * code[..., 1::2]).to(torch.uint8), torch.where(finite, exponent + 127, 255).to(torch.uint8)


def values(q, scale):
    """float64 values of codes and scales"""
    q, scale = q.cpu(), scale.cpu()
    table = torch.cat([E2M1, -E2M1])
    v = table[torch.stack([q & 15, q >> 4], -1).long()].flatten(-2).view(*scale.shape, 32)
    factor = torch.where(scale == 255, math.nan, torch.pow(2.0, scale.double() - 127))
    return (v * factor[..., None]).flatten(-2)


def assert_quantized(sk, x):
    q, scale = sk.quantize_mxfp4(x)
    want_q, want_scale = plain_quantize(x)
    assert q.shape == want_q.shape and scale.shape == want_scale.shape and q.dtype == scale.dtype == torch.uint8
    assert torch.equal(scale.cpu(), want_scale)
    # (the sign of a code of nothing says nothing)
    assert torch.equal(values(q, torch.full_like(scale, 127)), values(want_q, torch.full_like(want_scale, 127)))
    return q, scale


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("shape", [(1, 32), (3, 64), (7, 1056), (1000, 96), (2, 3, 4096), (32,), (33, 8224)])
def test_quantize(sk, dtype, shape):
    g = torch.Generator().manual_seed(1)
    x = torch.randn(shape, generator=g) * torch.exp(4 * torch.randn((*shape[:-1], 1), generator=g))
    x.view(-1)[::7] *= 0.01
    assert_quantized(sk, x.to(TYPES[dtype]).cuda())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
def test_quantize_every_number(sk, dtype):
    # every number of the type beside a block's maximum of every power of two that is not below it, and in blocks of its own
    bits = torch.arange(1 << 16, dtype=torch.int32).to(torch.uint16).view(TYPES[dtype])
    assert_quantized(sk, bits.view(-1, 32).cuda())
    finite = bits[torch.isfinite(bits)]
    finite = torch.cat([finite, finite.new_zeros(-len(finite) % 31)]).view(-1, 31)
    for e in range(-26, 16) if dtype == "float16" else range(-135, 128, 3):
        top = torch.full((len(finite), 1), 2.0 ** e, dtype=torch.float64).to(TYPES[dtype])
        small = torch.where(finite.double().abs() < 2.0 ** (e + 1), finite, torch.zeros_like(finite))
        assert_quantized(sk, torch.cat([small, top], 1).cuda())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", sorted(TYPES))
def test_quantize_special_blocks(sk, dtype):
    t = TYPES[dtype]
    x = torch.randn(12, 64, generator=torch.Generator().manual_seed(3)).to(t)
    x[0, 5], x[1, 40], x[2, 63], x[3, 0] = math.inf, -math.inf, math.nan, -math.nan
    x[4] = 0
    x[5, :32] = -0.0
    x[6] = torch.finfo(t).max
    x[7] = torch.finfo(t).smallest_normal
    x[8] = torch.finfo(t).smallest_normal * torch.finfo(t).eps
    x[9, 32:] = -torch.finfo(t).max
    q, scale = assert_quantized(sk, x.cuda())
    for out in TYPES.values():
        got, want = sk.dequantize_mxfp4(q, scale, out).double().cpu(), values(q, scale).to(out).double()
        assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.nan_to_num(7), want.nan_to_num(7))
        assert got[:2].isnan().sum() == 64


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", sorted(TYPES))
def test_dequantize_every_scale(sk, dtype):
    scale = torch.arange(256).to(torch.uint8).view(256, 1).repeat(1, 2).cuda()
    q = torch.randint(0, 256, (256, 32), generator=torch.Generator().manual_seed(5), dtype=torch.uint8).cuda()
    got, want = sk.dequantize_mxfp4(q, scale, TYPES[dtype]), values(q, scale).to(TYPES[dtype])
    assert got.dtype == TYPES[dtype] and torch.equal(got.cpu().isnan(), want.isnan())
    assert torch.equal(got.cpu().nan_to_num(nan=7), want.nan_to_num(nan=7))


@pytest.mark.gpu
def test_quantize_views(sk):
    g = torch.Generator().manual_seed(2)
    wide = torch.randn(40, 300, generator=g).half().cuda()
    for x in (wide[:, :64], wide[:, 3:99], wide[:, 8:40], wide[::2, 100:292], wide[:1, 1:33], wide[:1, :32].expand(5, 32), wide.t()[:, :32], wide[:, :256].view(40, 2, 4, 32)):
        assert_quantized(sk, x)
    q, s = sk.quantize_mxfp4(wide[:0, :64])
    assert q.shape == (0, 32) and s.shape == (0, 2) and sk.dequantize_mxfp4(q, s).shape == (0, 64)
    q, s = sk.quantize_mxfp4(wide[:, :96].contiguous())
    assert torch.equal(sk.dequantize_mxfp4(q[:, 16:32], s[:, 1:2]).double().cpu(), values(q[:, 16:32], s[:, 1:2]).to(torch.bfloat16).double())
    assert torch.equal(sk.dequantize_mxfp4(q[5:], s[5:]).double().cpu(), values(q[5:], s[5:]).to(torch.bfloat16).double())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", sorted(TYPES))
def test_arrays_larger_than_the_caches(sk, dtype):
    # 16384 and more blocks of rows, and the same in parts that stay below
    N, K = 8199, 8192
    x = torch.randn(N, K, device="cuda", generator=torch.Generator("cuda").manual_seed(2)).to(TYPES[dtype])
    x[8190:, 40] = math.inf
    q, scale = sk.quantize_mxfp4(x)
    back = sk.dequantize_mxfp4(q, scale, TYPES[dtype])
    for lo in range(0, N, 1000):
        part = slice(lo, lo + 1000)
        pq, ps = sk.quantize_mxfp4(x[part])
        assert torch.equal(q[part], pq) and torch.equal(scale[part], ps)
        assert torch.equal(back[part].view(torch.uint8), sk.dequantize_mxfp4(pq, ps, TYPES[dtype]).view(torch.uint8))


# ---- products ----
def activate(x, name):
    return {None: lambda v: v, "relu": torch.relu, "silu": lambda v: v * torch.sigmoid(v),
            "gelu_tanh": lambda v: 0.5 * v * (1 + torch.tanh(math.sqrt(2 / math.pi) * (v + 0.044715 * v ** 3)))}[name](x)


def operand(rows, K, seed, spread=6):
    """random codes and scales on the device: (q, scale, values in 64 bits)"""
    g = torch.Generator().manual_seed(seed)
    shape = rows if isinstance(rows, tuple) else (rows,)
    q = torch.randint(0, 256, (*shape, K // 2), generator=g, dtype=torch.uint8)
    scale = torch.randint(127 - spread, 128, (*shape, K // 32), generator=g, dtype=torch.uint8)
    return q.cuda(), scale.cuda(), values(q, scale).cuda()


def assert_near(C, want, terms, magnitudes, pre=None):
    tol = ROUNDING[C.dtype] * want.abs() * 1.001 + 1.2 * 2 * terms * 2.0 ** -24 * magnitudes + 2.0 ** -24
    if pre is not None:
        tol = tol + 4e-6 * (pre.abs() + 1)
    off = (C.double() - want).abs()
    assert torch.isfinite(C).all()
    assert (off <= tol).all(), f"largest excess {(off - tol).max().item():.3g} of {int((off > tol).sum())} values"


VARIANTS = (0, 1, 2, 3, 4, 5, 6, 7, 8, 9)


@pytest.mark.gpu
@pytest.mark.parametrize("variant", VARIANTS)
@pytest.mark.parametrize("M,N,K", [(1, 1, 32), (5, 1, 2080), (1, 2, 32), (1, 64, 256), (5, 77, 96), (16, 128, 1024), (17, 129, 1056), (33, 520, 2080), (64, 64, 4096), (100, 1000, 512),
                                   (1, 4096, 4096), (130, 257, 8224), (300, 515, 1312), (260, 300, 16448),
                                   (40, 200, 2944), (50, 72, 5024), (70, 130, 2560), (3, 300, 2848)])
def test_product(sk, variant, M, N, K):
    a, sa, va = operand(M, K, M + K)
    b, sb, vb = operand(N, K, N + K)
    want, magnitudes = va @ vb.T, va.abs() @ vb.abs().T
    for out in ROUNDING:
        assert_near(sk.streamk_mxfp4(a, b, sa, sb, out_dtype=out, variant=variant), want / 64 * 64, K, magnitudes)


@pytest.mark.gpu
def test_product_is_exact_where_sums_are(sk):
    # one scale for all, whole numbers: sums below 2^24 times a quarter, results of a few bits
    g = torch.Generator().manual_seed(9)
    for M, N, K in ((1, 64, 512), (40, 96, 1024), (256, 512, 512), (70, 300, 2048)):
        q = lambda rows: torch.where(torch.rand(rows, K // 2, generator=g) < 0.02, torch.randint(0, 256, (rows, K // 2), generator=g), 0).to(torch.uint8).cuda()  # noqa: E731
        a, b = q(M), q(N)
        sa, sb = torch.full((M, K // 32), 127, dtype=torch.uint8, device="cuda"), torch.full((N, K // 32), 127, dtype=torch.uint8, device="cuda")
        want = (values(a, sa) @ values(b, sb).T).cuda()
        assert torch.equal(sk.streamk_mxfp4(a, b, sa, sb).double(), want.half().double())


@pytest.mark.gpu
@pytest.mark.parametrize("M", [1, 20, 90, 300])
@pytest.mark.parametrize("activation", [None, "relu", "gelu_tanh", "silu"])
def test_epilogue(sk, M, activation):
    N, K = 300, 544
    a, sa, va = operand(M, K, 1, 3)
    b, sb, vb = operand(N, K, 2, 3)
    for out in ROUNDING:
        bias = torch.randn(N, generator=torch.Generator().manual_seed(3)).to(out).cuda()
        pre = va @ vb.T
        for extra in (None, bias):
            x = pre if extra is None else pre + extra.double()
            # (an activation's slope is at most 1.13: what the sum is off counts with it)
            assert_near(sk.streamk_mxfp4(a, b, sa, sb, out_dtype=out, bias=extra, activation=activation), activate(x, activation), K, 1.13 * (va.abs() @ vb.abs().T), x)


@pytest.mark.gpu
def test_scales_of_every_size_and_nan(sk):
    # one block far above or below the others, exponents from end to end; NaN blocks reach their row or column and no other
    M, N, K = 40, 70, 256
    a, sa, _ = operand(M, K, 1)
    b, sb, _ = operand(N, K, 2)
    sa[3], sb[:, 2] = 227, 30
    sa[4], sa[5, 1], sa[6] = 1, 250, 0
    va, vb = values(a, sa).cuda(), values(b, sb).cuda()
    want, magnitudes = va @ vb.T, va.abs() @ vb.abs().T
    C = sk.streamk_mxfp4(a, b, sa, sb, out_dtype=torch.bfloat16)
    tol = 2.0 ** -8 * want.abs() * 1.001 + 1.2 * 2 * K * 2.0 ** -24 * magnitudes + 2.0 ** -126
    # (row 5 has sums of magnitudes up to 5.75 2^128, beyond float32's largest number: a sum on the way may be infinite there)
    beyond = magnitudes >= 2.0 ** 128
    assert beyond.sum() == 32 and beyond[5].sum() == 32
    assert ((C.double() - want).abs() <= tol)[~beyond].all()
    sa[7, 0], sa[20, 7], sb[11, 3], sb[69, 7] = 255, 255, 255, 255
    for out in ROUNDING:
        C = sk.streamk_mxfp4(a[7:], b, sa[7:].contiguous(), sb, out_dtype=out).isnan()
        want = torch.zeros_like(C)
        want[0], want[13], want[:, 11], want[:, 69] = True, True, True, True
        assert torch.equal(C, want)


@pytest.mark.gpu
@pytest.mark.parametrize("K", [32, 96, 160, 288, 1056, 4128])
def test_what_lies_behind_a_row_does_not_count(sk, K):
    # rows of a wider matrix whose next values are infinite, and scales whose neighbours are NaN
    M, N = 37, 150
    a, sa, va = operand(M, K, 3)
    b, sb, vb = operand(N, K, 4)
    wide_a = torch.full((M, K // 2 + 64), 0x77, dtype=torch.uint8, device="cuda")
    wide_b = torch.full((N, K // 2 + 64), 0x77, dtype=torch.uint8, device="cuda")
    wide_a[:, :K // 2], wide_b[:, :K // 2] = a, b
    sa[1::2], sb[1::2] = 255, 255
    for variant in VARIANTS:
        C = sk.streamk_mxfp4(wide_a[:, :K // 2], wide_b[:, :K // 2], sa, sb, variant=variant)
        assert C[1::2].isnan().all() and C[:, 1::2].isnan().all()
        assert_near(C[::2, ::2], (va @ vb.T)[::2, ::2], K, (va.abs() @ vb.abs().T)[::2, ::2])


@pytest.mark.gpu
@pytest.mark.parametrize("rows_a,rows_b,blocks", [(1, 1, 1), (5, 64, 16), (65, 7, 17), (300, 130, 129), (64, 200, 256), (3, 70, 500)])
def test_tiled_scales(sk, rows_a, rows_b, blocks):
    g = torch.Generator().manual_seed(4)
    arrays = [torch.randint(0, 256, (rows, blocks), generator=g, dtype=torch.uint8).cuda() for rows in (rows_a, rows_b)]
    pairs = (blocks + 15) // 16
    tiled = [torch.full((pairs, rows, 16), 77, dtype=torch.uint8, device="cuda") for rows in (rows_a, rows_b)]
    stream = torch.cuda.current_stream().cuda_stream
    assert sk.lib().sk_tile_mx_scales(arrays[0].data_ptr(), rows_a, tiled[0].data_ptr(), arrays[1].data_ptr(), rows_b, tiled[1].data_ptr(), blocks, stream) == 0
    for t, a in zip(tiled, arrays):
        padded = torch.nn.functional.pad(a, (0, pairs * 16 - blocks))
        assert torch.equal(t, padded.view(-1, pairs, 16).transpose(0, 1))


SIZES = {"one": [5], "even": [16, 16, 16, 16], "skew": [1, 0, 70, 0, 200, 3], "empty": [0, 0, 0], "large": [300, 130], "many": [3] * 130}


def offsets_of(sizes):
    return torch.tensor([0, *itertools.accumulate(sizes)], dtype=torch.int32, device="cuda")


@pytest.mark.gpu
@pytest.mark.parametrize("variant", VARIANTS)
@pytest.mark.parametrize("sizes", sorted(SIZES))
@pytest.mark.parametrize("N,K", [(136, 96), (515, 1056), (64, 512)])
def test_by_expert(sk, variant, sizes, N, K):
    sizes = SIZES[sizes]
    R, E = sum(sizes) + 9, len(sizes)   # (nine rows behind the last group: zeros)
    a, sa, va = operand(R, K, 5)
    b, sb, vb = operand((E, N), K, 6)
    offsets = offsets_of(sizes)
    want, magnitudes, pre_bias = (torch.zeros(R, N, dtype=torch.float64, device="cuda") for _ in range(3))
    for out in ROUNDING:
        bias = torch.randn(E, N, generator=torch.Generator().manual_seed(1)).to(out).cuda()
        for e, (lo, hi) in enumerate(zip(offsets.tolist(), offsets.tolist()[1:])):
            want[lo:hi], magnitudes[lo:hi] = va[lo:hi] @ vb[e].T, va[lo:hi].abs() @ vb[e].abs().T
            pre_bias[lo:hi] = want[lo:hi] + bias[e].double()
        C = sk.streamk_grouped(a, b, offsets, scale_a=sa, scale_b=sb, out_dtype=out, variant=variant)
        assert_near(C, want, K, magnitudes)
        assert not C[-9:].any()
        C = sk.streamk_grouped(a, b, offsets, scale_a=sa, scale_b=sb, out_dtype=out, variant=variant, bias=bias, activation="silu")
        assert_near(C, activate(pre_bias, "silu"), K, 1.13 * magnitudes, pre_bias)


@pytest.mark.gpu
def test_offsets_of_any_content(sk):
    a, sa, va = operand(40, 128, 1)
    b, sb, vb = operand((3, 64), 128, 2)
    for offsets in ([5, 9, 20, 30], [0, 50, 60, 70], [-7, 10, 3, 90], [40, 30, 20, 10], [0, 0, 0, 0]):
        C = sk.streamk_grouped(a, b, torch.tensor(offsets, dtype=torch.int32, device="cuda"), scale_a=sa, scale_b=sb)
        at = [max(0, min(40, o)) for o in offsets]
        for i in range(1, 4):
            at[i] = max(at[i], at[i - 1])
        want, magnitudes = torch.zeros(40, 64, dtype=torch.float64, device="cuda"), torch.zeros(40, 64, dtype=torch.float64, device="cuda")
        for e in range(3):
            rows = slice(at[e], at[e + 1])
            want[rows], magnitudes[rows] = va[rows] @ vb[e].T, va[rows].abs() @ vb[e].abs().T
        assert_near(C, want, 128, magnitudes)


@pytest.mark.gpu
def test_views_and_out(sk):
    a, sa, va = operand(50, 512, 1)
    b, sb, vb = operand(200, 512, 2)
    want, magnitudes = va @ vb.T, va.abs() @ vb.abs().T
    wide = torch.full((50, 264), -1.0, dtype=torch.float16, device="cuda")
    out = wide[:, 3:203]
    assert sk.streamk_mxfp4(a, b, sa, sb, out=out) is out
    assert_near(out, want, 512, magnitudes)
    assert (wide[:, :3] == -1).all() and (wide[:, 203:] == -1).all()
    # rows that begin off 16 bytes, or a column slice, are copied; a single row of any pitch
    shifted = torch.zeros(50 * 256 + 8, dtype=torch.uint8, device="cuda")
    shifted[8:] = a.view(-1)
    assert_near(sk.streamk_mxfp4(shifted[8:].view(50, 256), b, sa, sb), want, 512, magnitudes)
    assert_near(sk.streamk_mxfp4(a[::7], b, sa[::7].contiguous(), sb), want[::7], 512, magnitudes[::7])
    assert_near(sk.streamk_mxfp4(a, b[::3], sa, sb[::3].contiguous()), want[:, ::3], 512, magnitudes[:, ::3])
    assert_near(sk.streamk_mxfp4(a[:1].expand(50, 256), b, sa[:1].repeat(50, 1), sb), want[:1].expand(50, 200), 512, magnitudes[:1].expand(50, 200))
    for name in ("float4_e2m1fn_x2", "float8_e8m0fnu"):
        assert hasattr(torch, name)
    C = sk.streamk_mxfp4(a.view(torch.float4_e2m1fn_x2), b.view(torch.float4_e2m1fn_x2), sa.view(torch.float8_e8m0fnu), sb.view(torch.float8_e8m0fnu))
    assert torch.equal(C, sk.streamk_mxfp4(a, b, sa, sb))
    assert sk.streamk_mxfp4(a[:0], b, sa[:0], sb).shape == (0, 200)
    assert sk.streamk_mxfp4(a, b[:1], sa, sb[:1]).shape == (50, 1)
    assert_near(sk.streamk_mxfp4(a, b[:1], sa, sb[:1]), want[:, :1], 512, magnitudes[:, :1])


@pytest.mark.gpu
@pytest.mark.parametrize("M,N,K", [(1, 512, 2080), (100, 600, 4096), (700, 520, 1024)])
def test_another_stream_and_a_graph(sk, M, N, K):
    x = torch.randn(M, K, generator=torch.Generator().manual_seed(1)).bfloat16().cuda()
    b, sb, vb = operand(N, K, 2)

    def step():
        q, s = sk.quantize_mxfp4(x)
        return sk.streamk_mxfp4(q, b, s, sb, out_dtype=torch.bfloat16, activation="relu")
    want = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        assert torch.equal(step(), want)
        side.synchronize()
        with torch.cuda.graph(graph, stream=side):
            C = step()
    for seed in (2, 3, 4):
        x.copy_(torch.randn(M, K, generator=torch.Generator().manual_seed(seed)).bfloat16())
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(C, step())
        # (the same on every launch, and on two streams at once)
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            one = step()
        two = step()
        torch.cuda.synchronize()
        assert torch.equal(one, C) and torch.equal(two, C)


@pytest.mark.gpu
@pytest.mark.parametrize("variant", VARIANTS)
def test_rows_of_a_wider_result(sk, variant):
    # columns 3 .. of rows of an odd pitch, in a product and by expert, with and without an end; what lies beside them stays
    M, N, K = 300, 267, 640
    a, sa, va = operand(M, K, 1)
    b, sb, vb = operand((2, N), K, 2)
    offsets = offsets_of([140, 160])
    want, magnitudes = torch.cat([va[:140] @ vb[0].T, va[140:] @ vb[1].T]), torch.cat([va[:140].abs() @ vb[0].abs().T, va[140:].abs() @ vb[1].abs().T])
    for out in ROUNDING:
        wide = torch.full((M, N + 10), 7.0, dtype=out, device="cuda")
        bias = torch.randn(2, N, generator=torch.Generator().manual_seed(3)).to(out).cuda()
        sk.streamk_mxfp4(a, b[0], sa, sb[0], out=wide[:, 3:3 + N], variant=variant)
        assert_near(wide[:140, 3:3 + N], want[:140], K, magnitudes[:140])
        sk.streamk_grouped(a, b, offsets, scale_a=sa, scale_b=sb, out=wide[:, 3:3 + N], variant=variant)
        assert_near(wide[:, 3:3 + N], want, K, magnitudes)
        sk.streamk_grouped(a, b, offsets, scale_a=sa, scale_b=sb, out=wide[:, 3:3 + N], bias=bias, activation="relu", variant=variant)
        pre = want + torch.cat([bias[0].double().expand(140, N), bias[1].double().expand(160, N)])
        assert_near(wide[:, 3:3 + N], pre.clamp(min=0), K, magnitudes, pre)
        assert (wide[:, :3] == 7).all() and (wide[:, 3 + N:] == 7).all()


@pytest.mark.gpu
def test_beyond_four_gigabytes(sk):
    # weights of 40 experts, 5.4e9 bytes, of which the first and the last have rows
    E, N, K, g = 40, 16384, 16384, torch.Generator("cuda").manual_seed(3)
    b = torch.empty(E, N, K // 2, dtype=torch.uint8, device="cuda").random_(generator=g)
    sb = torch.randint(120, 127, (E, N, K // 32), dtype=torch.uint8, device="cuda", generator=g)
    a, sa, va = operand(30, K, 9)
    offsets = offsets_of([14] + [0] * (E - 2) + [16])
    for variant in (0, 1, 2, 3, 5, 8):
        C = sk.streamk_grouped(a, b, offsets, scale_a=sa, scale_b=sb, out_dtype=torch.bfloat16, variant=variant)
        for e, r in ((0, slice(0, 14)), (E - 1, slice(14, 30))):
            n = slice(N - 100, N)
            vb = values(b[e, n], sb[e, n]).cuda()
            assert_near(C[r, n], va[r] @ vb.T, K, va[r].abs() @ vb.abs().T)
    del b, sb
    # rows: 4.9e9 bytes of A, 4.9e9 values and more of x
    M, K = 300000, 32768
    a = torch.empty(M, K // 2, dtype=torch.uint8, device="cuda").random_(generator=g)
    sa = torch.randint(120, 127, (M, K // 32), dtype=torch.uint8, device="cuda", generator=g)
    b, sb, vb = operand(70, K, 10)
    last = slice(M - 50, M)
    va = values(a[last], sa[last]).cuda()
    for variant in (0, 2, 5, 6):
        C = sk.streamk_mxfp4(a, b, sa, sb, out_dtype=torch.bfloat16, variant=variant)
        assert_near(C[last], va @ vb.T, K, va.abs() @ vb.abs().T)
    x = sk.dequantize_mxfp4(a, sa)
    assert torch.equal(x[last], sk.dequantize_mxfp4(a[last], sa[last]))
    q, scale = sk.quantize_mxfp4(x)
    want = sk.quantize_mxfp4(x[last])
    assert torch.equal(q[last], want[0]) and torch.equal(scale[last], want[1])


@pytest.mark.gpu
def test_the_tiles_that_the_sizes_ask_for_take_them(sk):
    """Exponents that would be beyond 2 GiB as some tiles want them: others run."""
    from streamk import _lib
    L, asked = _lib.lib(), 0
    for E, N, K, R in itertools.product((1, 8, 256), (64, 16384, 1 << 21), (32, 160, 4096, 4128, 16384, 16416), (1, 100, 3000, 100000, 1 << 24)):
        if E * N * K > 1 << 38 or R * K > 1 << 38 or R * N > 1 << 36:
            continue
        g = _lib.SkGrouped(dtype=_lib.SK_MXFP4, layout=_lib.LAYOUT_NT, out_dtype=_lib.SK_F16, activation=0, E=E, R=R, N=N, K=K, lda=K, ldb=K, ldc=N,
                           expert_b=N * K if E > 1 else 0)
        assert L.sk_grouped_workspace_bytes(ctypes.byref(g)) > 0, (E, N, K, R)
        g.scales_tiled = L.sk_mx_scales_tiled(ctypes.byref(g))
        asked += g.scales_tiled
        assert L.sk_grouped_workspace_bytes(ctypes.byref(g)) > 0, (E, N, K, R)
    assert asked > 10
    E, N, K, gen = 8, 15 << 17, 4128, torch.Generator("cuda").manual_seed(4)
    b = torch.empty(E, N, K // 2, dtype=torch.uint8, device="cuda").random_(generator=gen)
    sb = torch.randint(120, 127, (E, N, K // 32), dtype=torch.uint8, device="cuda", generator=gen)
    a, sa, va = operand(200 * E, K, 11)
    C = sk.streamk_grouped(a, b, offsets_of([200] * E), scale_a=sa, scale_b=sb, out_dtype=torch.bfloat16)
    for e, n in ((0, slice(0, 50)), (E - 1, slice(N - 50, N))):
        r, vb = slice(200 * e, 200 * e + 200), values(b[e, n], sb[e, n]).cuda()
        assert_near(C[r, n], va[r] @ vb.T, K, va[r].abs() @ vb.abs().T)


@pytest.mark.gpu
def test_the_choice_of_tiles_counts_on_the_cuts_that_are_made(sk):
    """256 x 256 tiles that whole rounds leave are cut along K from 8192 on: 6 x 14 tiles in two, which take less time than tiles of 128 x 256
    (68 and 71 to 76 us), where whole ones would take more.  With a K that is a multiple of 128 they alone want exponents tiled, which says
    that they are chosen."""
    from streamk import _lib
    if torch.cuda.get_device_properties(0).multi_processor_count != 256:
        pytest.skip("tiles of 256 CUs")
    R, N, K = 1431, 3492, 14080
    asks = []
    for variant in (0, 2, 7):
        g = _lib.SkGrouped(dtype=_lib.SK_MXFP4, layout=_lib.LAYOUT_NT, out_dtype=_lib.SK_F16, activation=0, E=1, R=R, N=N, K=K, lda=K, ldb=K, ldc=N, variant=variant)
        asks.append(_lib.lib().sk_mx_scales_tiled(ctypes.byref(g)))
    assert asks == [1, 1, 0]


@pytest.mark.gpu
def test_exponents_that_begin_inside_a_word(sk):
    for M, N, K in ((5, 40, 96), (300, 520, 4128), (600, 2000, 2048), ((1 << 27) + 3, 8, 32)):   # (the last: more rows than exponents are laid out anew for)
        gen = torch.Generator("cuda").manual_seed(M)
        a = torch.empty(M, K // 2, dtype=torch.uint8, device="cuda").random_(generator=gen)
        b, sb, vb = operand(N, K, 13)
        sa = torch.randint(120, 127, (M * (K // 32) + 1,), dtype=torch.uint8, device="cuda", generator=gen)[1:].view(M, K // 32)
        assert sa.data_ptr() % 4 == 1
        C = sk.streamk_mxfp4(a, b, sa, sb, out_dtype=torch.bfloat16)
        for r in (slice(0, 5), slice(M - 5, M)):
            va = values(a[r], sa[r]).cuda()
            assert_near(C[r], va @ vb.T, K, va.abs() @ vb.abs().T)


@pytest.mark.gpu
def test_wrong_operands_are_refused(sk):
    a, sa, _ = operand(6, 64, 1)
    b, sb, _ = operand((3, 40), 64, 2)
    offsets = offsets_of([1, 2, 3])
    for bad, kind in ((dict(A=a.half()), (TypeError, ValueError)), (dict(A=a[:, :16]), ValueError), (dict(B=b[0]), ValueError), (dict(B=b.to(torch.int8)), TypeError),
                      (dict(scale_a=None), ValueError), (dict(scale_b=None), ValueError), (dict(scale_a=sa.float()), TypeError), (dict(scale_a=sa[:5]), ValueError),
                      (dict(scale_b=sb[:, :39]), ValueError), (dict(scale_b=sb.transpose(0, 1).contiguous().transpose(0, 1)), ValueError),
                      (dict(offsets=offsets[:3]), ValueError), (dict(offsets=offsets.long()), TypeError), (dict(layout="nn"), ValueError),
                      (dict(out_dtype=torch.float32), ValueError), (dict(bias=torch.zeros(3, 40, device="cuda")), ValueError), (dict(activation="tanh"), ValueError),
                      (dict(scale_a=sa.cpu()), (TypeError, ValueError, RuntimeError))):
        with pytest.raises(kind):
            sk.streamk_grouped(**{**dict(A=a, B=b, offsets=offsets, scale_a=sa, scale_b=sb), **bad})
    for args in ((a, b[0], sa, None), (a, b[0, :, :16], sa, sb[0]), (a[:, :8], b[0, :, :8], sa[:, :1], sb[0, :, :1]), (a, b, sa, sb), (a, b[0].to(torch.int8), sa, sb[0])):
        with pytest.raises((TypeError, ValueError, RuntimeError)):
            sk.streamk_mxfp4(*args)
    for variant in (10, 11, -1):
        with pytest.raises(sk.StreamKError):
            sk.streamk_mxfp4(a, b[0], sa, sb[0], variant=variant)
    with pytest.raises(ValueError):
        sk.streamk_mxfp4(a, b[0], sa, sb[0], out_dtype=torch.float32)
    with pytest.raises(ValueError):
        sk.streamk_mxfp4(a, b[0], sa, sb[0], out=torch.empty(6, 39, dtype=torch.float16, device="cuda"))
    with pytest.raises(ValueError):
        sk.quantize_mxfp4(torch.zeros(4, 48, device="cuda"))
    with pytest.raises(TypeError):
        sk.quantize_mxfp4(torch.zeros(4, 64, device="cuda", dtype=torch.int32))
    with pytest.raises(ValueError):
        sk.dequantize_mxfp4(a, sa[:, :1])
    with pytest.raises(ValueError):
        sk.dequantize_mxfp4(a, sa, torch.float64)


def test_calls_are_refused_with_codes(sk):
    L, lib = sk.lib(), __import__("streamk._lib", fromlist=["x"])
    p = 1 << 12   # (an aligned address; every call below is refused before it is used)

    def product(**kw):
        d = dict(dtype=lib.SK_MXFP4, layout=0, out_dtype=lib.SK_F16, activation=0, E=2, R=10, N=64, K=64, A=p, B=p, offsets=p, C=p, lda=64, ldb=64, ldc=64, expert_b=4096,
                 scale_a=p, scale_b=p)
        return L.sk_gemm_grouped(ctypes.byref(lib.SkGrouped(**{**d, **kw})), None, 0, None)
    for bad in (dict(A=None), dict(scale_a=None), dict(scale_b=None), dict(offsets=None)):
        assert product(**bad) == -1, bad
    for bad in (dict(layout=1), dict(out_dtype=lib.SK_F32), dict(out_dtype=lib.SK_MXFP4), dict(activation=9), dict(variant=-1)):
        assert product(**bad) == -4, bad
    for bad in (dict(K=0), dict(lda=32), dict(ldb=32), dict(ldc=63), dict(lda=1 << 40), dict(R=1 << 31),
                dict(scales_tiled=1, N=1 << 27), dict(scales_tiled=1, R=1 << 26, K=2048, lda=2048, ldb=2048)):
        assert product(**bad) == -2, bad
    for bad in (dict(K=48), dict(lda=80), dict(ldb=80), dict(expert_b=4112), dict(A=p + 8), dict(B=p + 2), dict(C=p + 1), dict(scale_a=p + 1), dict(scale_b=p + 2),
                dict(scales_tiled=1, scale_a=p + 4), dict(offsets=p + 2)):
        assert product(**bad) == -3, bad
    quantize = lambda x=p, t=0, M=4, K=64, ld=64, q=p, s=p: L.sk_quantize_mxfp4(x, t, M, K, ld, q, s, None)  # noqa: E731
    assert quantize(x=None) == -1 and quantize(s=None) == -1 and quantize(t=6) == -4 and quantize(M=0) == -2 and quantize(ld=63) == -2 and quantize(K=40) == -3
    assert quantize(x=p + 1) == -3 and quantize(q=p + 2) == -3 and quantize(M=1 << 40, K=1 << 20, ld=1 << 20) == -2
    values_of = lambda q=p, s=p, M=4, K=64, t=0, x=p: L.sk_dequantize_mxfp4(q, s, M, K, t, x, None)  # noqa: E731
    assert values_of(q=None) == -1 and values_of(t=6) == -4 and values_of(K=40) == -3 and values_of(M=-1) == -2 and values_of(x=p + 1) == -3
    tile = lambda a=p, rows=4, ta=p, b=p, more=5, tb=p, blocks=3: L.sk_tile_mx_scales(a, rows, ta, b, more, tb, blocks, None)  # noqa: E731
    assert tile(a=None) == -1 and tile(tb=None) == -1 and tile(rows=0) == -2 and tile(more=1 << 31) == -2 and tile(blocks=0) == -2 and tile(ta=p + 8) == -3
    assert L.sk_mx_scales_tiled(None) == 0


def test_fake_implementations(sk):
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        x = torch.empty(5, 3, 128, dtype=torch.bfloat16, device="cuda")
        q, s = torch.ops.streamk.quantize_mxfp4(x)
        assert q.shape == (5, 3, 64) and s.shape == (5, 3, 4) and q.dtype == s.dtype == torch.uint8
        assert torch.ops.streamk.dequantize_mxfp4(q, s, torch.float32).shape == x.shape
        C = torch.ops.streamk.gemm_mxfp4(q[0], q[1], s[0], s[1], torch.bfloat16)
        assert C.shape == (3, 3) and C.dtype == torch.bfloat16
        off = torch.empty(6, dtype=torch.int32, device="cuda")
        assert torch.ops.streamk.gemm_grouped(q[0], q, off, scale_a=s[0], scale_b=s).dtype == torch.float16


def test_the_oracle_of_the_quantiser():
    """(plain_quantize itself, by a few blocks worked out by hand)"""
    x = torch.zeros(4, 32)
    x[0, :6] = torch.tensor([6.0, 0.25, 0.75, 2.5, 5.0, -7.9])     # scale 2^0: ties to the even code; 7.9 becomes 6
    x[1, 0] = 2.0 ** -140
    x[2, 3] = math.inf
    q, s = plain_quantize(x)
    assert s[:, 0].tolist() == [127, 0, 255, 0]
    assert values(q, s)[0, :6].tolist() == [6.0, 0.0, 1.0, 2.0, 4.0, -6.0]
    assert not q[1:].any()
