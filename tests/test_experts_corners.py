"""Operands, recordings and plans at the edge of what the operators for experts and int8 take.  Tolerances as in test_experts.py: fp32 sums
of n terms within 2 n 2^-24 of the sum of the terms' magnitudes, one rounding to the result's type."""
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


def assert_near(C, want, terms, magnitudes):
    tol = ROUNDING[C.dtype] * want.abs() * 1.001 + 1.2 * 2 * terms * 2.0 ** -24 * magnitudes + 2.0 ** -24
    off = (C.double() - want).abs()
    assert torch.isfinite(C).all()
    assert (off <= tol).all(), f"largest excess {(off - tol).max().item():.3g} of {int((off > tol).sum())} values"


def offsets_of(sizes):
    return torch.tensor([0] + torch.tensor(sizes).cumsum(0).tolist(), dtype=torch.int32, device="cuda")


def groups(sizes):
    start = 0
    for e, n in enumerate(sizes):
        yield e, slice(start, start + n)
        start += n


def rand(shape, dtype, seed, std=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * std).to(dtype).cuda()


def plain_kn(A, B, sizes):
    """A's rows times [K, N] weights in 64 bits, and the sums of magnitudes"""
    y = torch.zeros(A.shape[0], B.shape[2], dtype=torch.float64, device="cuda")
    m = torch.zeros_like(y)
    for e, at in groups(sizes):
        y[at], m[at] = A[at].double() @ B[e].double(), A[at].double().abs() @ B[e].double().abs()
    return y, m


# ---- [K, N] weights whose K is no multiple of 8 ----
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("variant", [0, 1, 5])
@pytest.mark.parametrize("sizes,K", [([10, 0, 150], 77), ([1], 77), ([3, 40], 1), ([0, 1], 1031), ([200, 7], 260)])
@pytest.mark.parametrize("beside", [math.nan, math.inf, 0.0])
def test_columns_beside_a_view_do_not_count(sk, dtype, variant, sizes, K, beside):
    R, N, t = sum(sizes), 64, TYPES[dtype]
    wide = torch.full((R, (K + 7) // 8 * 8 + 8), beside, dtype=t, device="cuda")
    A, B = wide[:, :K], rand((len(sizes), K, N), t, 2, 1 / math.sqrt(K))
    A.copy_(rand((R, K), t, 1))
    want, magnitudes = plain_kn(A, B, sizes)
    run = lambda a: sk.streamk_grouped(a, B, offsets_of(sizes), layout="nn", variant=variant)  # noqa: E731
    C = run(A)
    assert_near(C, want, K, magnitudes)
    # (rows that no 16-byte loads reach, and a row that stands for many)
    assert torch.equal(run(A.contiguous()), C)
    assert torch.equal(run(A[:1].expand(R, K)), run(A[:1].repeat(R, 1)))
    out = torch.empty_like(C)
    sk.streamk_grouped(A, B, offsets_of(sizes), layout="nn", variant=variant, out=out)
    assert torch.equal(out, C)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", sorted(TYPES))
def test_columns_beside_a_gradient_do_not_count(sk, dtype):
    sizes, N, K, t = [10, 0, 150], 77, 64, TYPES[dtype]
    R = sum(sizes)
    A, B = rand((R, K), t, 1), rand((3, N, K), t, 2, 0.125)
    wide = torch.full((R, 88), math.nan, dtype=t, device="cuda")
    d = wide[:, :N]
    d.copy_(rand((R, N), t, 3))
    x, w = A.clone().requires_grad_(), B.clone().requires_grad_()
    dx, dw = torch.autograd.grad(sk.streamk_grouped(x, w, offsets_of(sizes)), (x, w), d)
    for e, at in groups(sizes):
        assert_near(dx[at], d[at].double() @ B[e].double(), N, d[at].double().abs() @ B[e].double().abs())
        assert_near(dw[e], d[at].double().T @ A[at].double(), sizes[e], d[at].double().abs().T @ A[at].double().abs())
