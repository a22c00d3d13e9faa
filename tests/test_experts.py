"""The operators of a mixture of experts against 64-bit arithmetic: grouped products and their gradients, routing, dispatch, combination.

Tolerances of products: fp32 sums of n terms, in any order, are within 2 n 2^-24 of the sum of the terms' magnitudes (an MFMA may cut
instead of rounding: hence the 2), plus one rounding to the result's type (2^-8 of bfloat16, 2^-11 of fp16, 2^-24 absolute below
fp16's normal numbers); bias and activation as in the int8 tests: 4e-6 of the value in front of the activation and of one."""
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


def assert_near(C, want, terms, magnitudes, pre=None):
    tol = ROUNDING[C.dtype] * want.abs() * 1.001 + 1.2 * 2 * terms * 2.0 ** -24 * magnitudes + 2.0 ** -24
    if pre is not None:
        tol = tol + 4e-6 * (pre.abs() + 1)
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


def plain(A, B, sizes, layout="nt"):
    """(product, sums of magnitudes) in 64 bits; zeros for rows behind the last group"""
    a, b = A.double(), B.double() if layout == "nt" else B.double().transpose(1, 2)
    y = torch.zeros(A.shape[0], b.shape[1], dtype=torch.float64, device="cuda")
    m = torch.zeros_like(y)
    for e, at in groups(sizes):
        y[at], m[at] = a[at] @ b[e].T, a[at].abs() @ b[e].abs().T
    return y, m


SIZES = {"one": [1], "empty": [0, 0, 0], "single rows": [1, 0, 1, 1], "ragged": [3, 0, 17, 129, 1, 64], "one expert has all": [0, 300, 0, 0],
         "whole tiles": [128, 256, 128], "seventy experts": [(7 * i) % 11 for i in range(70)], "large": [700, 513, 1, 900]}


# ---- the grouped product ----
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("layout", ["nt", "nn"])
@pytest.mark.parametrize("sizes", sorted(SIZES))
@pytest.mark.parametrize("N,K", [(136, 72), (8, 8), (520, 256), (256, 512)])
def test_grouped_product(sk, dtype, layout, sizes, N, K):
    sizes = SIZES[sizes]
    R, E = sum(sizes) + 5, len(sizes)   # (five rows that no expert owns)
    A, B = rand((R, K), TYPES[dtype], R), rand((E, N, K) if layout == "nt" else (E, K, N), TYPES[dtype], N, 1 / math.sqrt(K))
    C = sk.streamk_grouped(A, B, offsets_of(sizes), layout=layout)
    want, magnitudes = plain(A, B, sizes, layout)
    assert_near(C, want, K, magnitudes)
    assert not C[R - 5:].any()


@pytest.mark.gpu
@pytest.mark.parametrize("N,K", [(1, 8), (77, 64), (131, 1032), (2049, 192)])
def test_grouped_product_of_odd_widths(sk, N, K):
    sizes = [5, 0, 40, 200]
    A, B = rand((245, K), torch.float16, 1), rand((4, N, K), torch.float16, 2, 1 / math.sqrt(K))
    want, magnitudes = plain(A, B, sizes)
    assert_near(sk.streamk_grouped(A, B, offsets_of(sizes)), want, K, magnitudes)


@pytest.mark.gpu
@pytest.mark.parametrize("activation", [None, "relu", "gelu_tanh", "silu"])
@pytest.mark.parametrize("rows", [6, 90, 2000])
def test_grouped_epilogue(sk, rows, activation):
    sizes = [rows // 2, 0, rows - rows // 2]
    A, B, bias = rand((rows, 128), torch.bfloat16, 3), rand((3, 200, 128), torch.bfloat16, 4, 0.1), rand((3, 200), torch.bfloat16, 5)
    C = sk.streamk_grouped(A, B, offsets_of(sizes), bias=bias, activation=activation)
    pre, magnitudes = plain(A, B, sizes)
    for e, at in groups(sizes):
        pre[at] += bias[e].double()
    assert_near(C, activate(pre, activation), 128, 1.2 * magnitudes, pre)


@pytest.mark.gpu
@pytest.mark.parametrize("out", sorted(TYPES))
@pytest.mark.parametrize("sizes", sorted(SIZES))
@pytest.mark.parametrize("N,K", [(136, 80), (515, 1040), (256, 256)])
def test_grouped_int8(sk, out, sizes, N, K):
    sizes = SIZES[sizes]
    R, E = sum(sizes) + 3, len(sizes)
    g = torch.Generator().manual_seed(R + N)
    A = torch.randint(-127, 128, (R, K), generator=g, dtype=torch.int8).cuda()
    B = torch.randint(-127, 128, (E, N, K), generator=g, dtype=torch.int8).cuda()
    sa, sb = (torch.rand(R, generator=g) + 0.5).cuda() * 0.01, (torch.rand(E, N, generator=g) + 0.5).cuda() / (73 * math.sqrt(K))
    bias = rand((E, N), TYPES[out], 7)
    C = sk.streamk_grouped(A, B, offsets_of(sizes), scale_a=sa, scale_b=sb, out_dtype=TYPES[out], bias=bias, activation="silu")
    pre, _ = plain(A, B, sizes)
    pre *= sa.double()[:, None]
    for e, at in groups(sizes):
        pre[at] = pre[at] * sb[e].double() + bias[e].double()
    assert_near(C, activate(pre, "silu"), 0, 0, pre)
    assert not C[R - 3:].any()


@pytest.mark.gpu
def test_grouped_views_and_out(sk):
    sizes = [30, 0, 41, 100]
    A, B = rand((171, 96), torch.float16, 1), rand((4, 72, 96), torch.float16, 2, 0.1)
    offsets = offsets_of(sizes)
    want = sk.streamk_grouped(A, B, offsets)
    wide_a = torch.zeros(171, 160, dtype=torch.float16, device="cuda")
    wide_a[:, 16:112] = A
    wide_b = torch.zeros(4, 80, 128, dtype=torch.float16, device="cuda")
    wide_b[:, :72, :96] = B
    assert torch.equal(sk.streamk_grouped(wide_a[:, 16:112], wide_b[:, :72, :96], offsets), want)
    shifted = torch.zeros(171, 97, dtype=torch.float16, device="cuda")
    shifted[:, 1:] = A
    assert torch.equal(sk.streamk_grouped(shifted[:, 1:], B, offsets), want)
    assert torch.equal(sk.streamk_grouped(A, B[:1].expand(4, 72, 96), offsets), sk.streamk_grouped(A, B[:1].repeat(4, 1, 1), offsets))
    out = torch.full((171, 79), 7.0, dtype=torch.float16, device="cuda")
    sk.streamk_grouped(A, B, offsets, out=out[:, 3:75])
    assert torch.equal(out[:, 3:75], want) and (out[:, :3] == 7).all() and (out[:, 75:] == 7).all()
    assert sk.streamk_grouped(A[:0], B, torch.zeros_like(offsets)).shape == (0, 72)
    one = sk.streamk_grouped(A[:1], B, offsets_of([0, 1, 0, 0]))
    assert_near(one, *[t for t in (plain(A[:1], B, [0, 1, 0, 0])[0], 96, plain(A[:1], B, [0, 1, 0, 0])[1])])


@pytest.mark.gpu
def test_values_of_other_experts_do_not_leak(sk):
    """NaN and infinities in the rows and weights around a group leave its results alone."""
    sizes = [20, 7, 40]
    A, B = rand((67, 64), torch.bfloat16, 1), rand((3, 48, 64), torch.bfloat16, 2)
    clean = sk.streamk_grouped(A, B, offsets_of(sizes))
    A[:20], A[27:] = math.nan, math.inf
    B[0], B[2] = math.inf, math.nan
    dirty = sk.streamk_grouped(A, B, offsets_of(sizes))
    assert torch.equal(dirty[20:27], clean[20:27]) and not torch.isfinite(dirty[:20]).any() and not torch.isfinite(dirty[27:]).any()


@pytest.mark.gpu
def test_grouped_on_another_stream_and_in_a_graph(sk):
    A, B = rand((300, 256), torch.float16, 1), rand((5, 256, 256), torch.float16, 2, 0.1)
    offsets = offsets_of([50, 0, 100, 150, 0])
    want = sk.streamk_grouped(A, B, offsets)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        assert torch.equal(sk.streamk_grouped(A, B, offsets), want)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        C = sk.streamk_grouped(A, B, offsets)
    for sizes in ([50, 0, 100, 150, 0], [0, 0, 0, 0, 300], [1, 2, 3, 4, 5], [60, 60, 60, 60, 60]):
        offsets.copy_(offsets_of(sizes))   # other groups in the same graph: the host does not know the sizes
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(C, sk.streamk_grouped(A, B, offsets))


# ---- its gradients ----
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("sizes", sorted(SIZES))
@pytest.mark.parametrize("M,N", [(136, 72), (77, 8), (520, 264), (256, 256)])
def test_weight_gradient(sk, dtype, sizes, M, N):
    sizes = SIZES[sizes]
    R, E = sum(sizes) + 4, len(sizes)
    dC, A = rand((R, M), TYPES[dtype], R), rand((R, N), TYPES[dtype], N)
    got = sk.streamk_grouped_wgrad(dC, A, offsets_of(sizes))
    assert got.shape == (E, M, N) and got.dtype == TYPES[dtype]
    for e, at in groups(sizes):
        want = dC[at].double().T @ A[at].double()
        assert_near(got[e], want, sizes[e], dC[at].double().abs().T @ A[at].double().abs())


@pytest.mark.gpu
def test_weight_gradient_ignores_other_groups_rows(sk):
    sizes = [20, 7, 40]
    dC, A = rand((67, 40), torch.float16, 1), rand((67, 64), torch.float16, 2)
    clean = sk.streamk_grouped_wgrad(dC, A, offsets_of(sizes))
    dC[:20], A[27:] = math.nan, math.inf
    assert torch.equal(sk.streamk_grouped_wgrad(dC, A, offsets_of(sizes))[1], clean[1])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("layout,N,K", [("nt", 72, 136), ("nt", 77, 64), ("nn", 72, 136), ("nt", 264, 520)])
def test_gradients_of_the_product(sk, dtype, layout, N, K):
    """Against the formulas, and against differences: the product is linear in each operand, so that f(A + V) - f(A - V) is exactly
    2 <dA, V> but for roundings (of f's values to 16 bits, of dA's)."""
    sizes = [33, 0, 130, 5]
    R, t = sum(sizes) + 2, TYPES[dtype]
    A, B = rand((R, K), t, 1), rand((4, N, K) if layout == "nt" else (4, K, N), t, 2, 0.1)
    dC = rand((R, N), t, 3)
    offsets = offsets_of(sizes)
    A.requires_grad_()
    B.requires_grad_()
    C = sk.streamk_grouped(A, B, offsets, layout=layout)
    dA, dB = torch.autograd.grad(C, (A, B), dC)
    A, B = A.detach(), B.detach()
    b = B.double() if layout == "nt" else B.double().transpose(1, 2)
    for e, at in groups(sizes):
        assert_near(dA[at], dC[at].double() @ b[e], N, dC[at].double().abs() @ b[e].abs())
        want, m = dC[at].double().T @ A[at].double(), dC[at].double().abs().T @ A[at].double().abs()
        if layout == "nn":
            want, m = want.T, m.T
        assert_near(dB[e], want, sizes[e], m)
    assert not dA[R - 2:].any()
    V, W = rand(A.shape, t, 4), rand(B.shape, t, 5, 0.1)
    value = lambda a, w: (sk.streamk_grouped(a, w, offsets, layout=layout).double() * dC.double()).sum()  # noqa: E731
    u = ROUNDING[t]
    for got, x, v, f in ((dA, A, V, lambda z: value(z, B)), (dB, B, W, lambda z: value(A, z))):
        up, down = (x + v), (x - v)   # (rounded: the step is what they differ by)
        step = up.double() - down.double()
        terms = (sk.streamk_grouped(up if x is A else A, up if x is B else B, offsets, layout=layout).double().abs() * dC.double().abs()).sum()
        # roundings are independent: 6 standard deviations of the sum, bounded by the root of the number of terms; u / sqrt 3 each
        bound = 6 * u * terms * 2 / math.sqrt(R * N) + 6 * u * (got.double().abs() * step.abs()).sum() / math.sqrt(got.numel())
        assert abs(f(up) - f(down) - (got.double() * step).sum()) <= bound


@pytest.mark.gpu
def test_only_the_gradient_that_is_asked_for(sk):
    A, B, offsets = rand((20, 64), torch.float16, 1), rand((2, 32, 64), torch.float16, 2), offsets_of([12, 8])
    B.requires_grad_()
    C = sk.streamk_grouped(A, B, offsets)
    C.sum().backward()
    assert A.grad is None and B.grad.shape == B.shape     # (an expanded gradient too: sum's)
    with pytest.raises(ValueError):
        sk.streamk_grouped(A, B, offsets, activation="silu")
    with torch.no_grad():
        sk.streamk_grouped(A, B, offsets, activation="silu")


# ---- routing ----
def plain_route(logits, k):
    """Token by token, in Python."""
    T, E = logits.shape
    weights, experts = torch.zeros(T, k, dtype=torch.float64), torch.full((T, k), -1, dtype=torch.int32)
    rows = [[] for _ in range(E)]
    for t, z in enumerate(logits.double().tolist()):
        best = sorted((e for e in range(E) if z[e] > -math.inf), key=lambda e: (-z[e], e))[:k]
        p = [math.exp(z[e] - z[best[0]]) for e in best]
        for j, e in enumerate(best):
            weights[t, j], experts[t, j] = p[j] / sum(p), e
            rows[e].append(t * k + j)
    order = [s for r in rows for s in r]
    offsets = [0]
    for r in rows:
        offsets.append(offsets[-1] + len(r))
    place = torch.full((T * k,), -1, dtype=torch.int32)
    for p, s in enumerate(order):
        place[s] = p
    return weights, experts, offsets, order + [-1] * (T * k - len(order)), place.view(T, k)


def assert_route(route, logits, k):
    weights, experts, offsets, order, place = plain_route(logits.cpu(), k)
    assert torch.equal(route.experts.cpu(), experts)
    assert route.offsets.tolist() == offsets and route.order.tolist() == order
    assert torch.equal(route.place.cpu(), place)
    # exp and the sum of at most 64 terms in fp32: 64 half units and the exponential's two
    assert ((route.weights.cpu().double() - weights).abs() <= 66 * 2.0 ** -24 * weights + 1e-38).all()


@pytest.mark.gpu
@pytest.mark.parametrize("T,E,k", [(1, 1, 1), (1, 8, 2), (5, 3, 3), (63, 64, 8), (64, 256, 8), (65, 65, 4), (64, 300, 2), (200, 1000, 64), (1000, 128, 6), (3001, 17, 5), (17, 1024, 10)])
def test_route(sk, T, E, k):
    g = torch.Generator().manual_seed(T * E + k)
    logits = (torch.randn(T, E, generator=g) * 2).bfloat16().float()   # (coarse: equal ones)
    assert_route(sk.route_experts(logits.cuda(), k), logits, k)
    closed = torch.rand(T, E, generator=g) < 0.6
    closed[::7] = True
    masked = logits.masked_fill(closed, -math.inf)
    assert_route(sk.route_experts(masked.cuda(), k), masked, k)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_route_of_special_values(sk, dtype):
    low = torch.finfo(dtype).min
    z = torch.tensor([[0.0, -0.0, 0.0, -0.0], [low, low, low, low], [low, 1, low, 1], [math.nan, 2, math.nan, 3], [math.nan] * 4, [-math.inf] * 4,
                      [-math.inf, low, -math.inf, 5], [7, 7, 7, 7], [-1e-30, 1e-30, 0, -1]], dtype=dtype)
    assert_route(sk.route_experts(z.cuda(), 3), z, 3)
    r = sk.route_experts(z.cuda(), 3)
    assert r.weights[1].tolist() == pytest.approx([1 / 3] * 3) and r.weights[4].tolist() == [0, 0, 0] and r.experts[0].tolist() == [0, 1, 2]
    wide = torch.zeros(9, 11, dtype=dtype, device="cuda")
    wide[:, 3:7] = z
    for v in (wide[:, 3:7], wide[:, 3:7].t().contiguous().t()):
        for a, b in zip(sk.route_experts(v, 3), r):
            assert torch.equal(a, b)
    empty = sk.route_experts(z[:0].cuda(), 2)
    assert empty.weights.shape == (0, 2) and empty.offsets.tolist() == [0] * 5 and empty.order.shape == (0,)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("T,E,k", [(5, 4, 2), (70, 300, 7), (1, 64, 64)])
def test_route_gradient(sk, dtype, T, E, k):
    g = torch.Generator().manual_seed(T)
    z = (torch.randn(T, E, generator=g) * 2).to(dtype)
    z[0, E // 2:] = -math.inf
    if T > 2:
        z[2] = -math.inf
    dw = torch.randn(T, k, generator=g)
    leaf = z.cuda().requires_grad_()
    r = sk.route_experts(leaf, k)
    got, = torch.autograd.grad(r.weights, leaf, dw.cuda())
    assert got.dtype == dtype and got.shape == z.shape
    # the formula in 64 bits on the same choice
    w, e = plain_route(z, k)[:2]
    dl = w * (dw.double() - (w * dw.double()).sum(1, keepdim=True))
    want = torch.zeros(T, E, dtype=torch.float64).scatter_add_(1, e.clamp(min=0).long(), dl)
    tol = (ROUNDING.get(dtype, 0.0) * want.abs() * 1.001 + 200 * 2.0 ** -24 * dw.abs().double().amax(1, keepdim=True) + (2.0 ** -24 if dtype == torch.float16 else 1e-37))
    assert ((got.cpu().double() - want).abs() <= tol).all()
    # differences of the weights in 64 bits, the choice held
    h, v = 1e-6, torch.randn(T, E, generator=g).double()

    def loss(x):
        c = torch.where(e >= 0, x.gather(1, e.clamp(min=0).long()), -math.inf)
        p = torch.where(e >= 0, torch.exp(c - c.max(1, keepdim=True).values.clamp(min=-1e300)), 0)
        return ((p / p.sum(1, keepdim=True).clamp(min=1e-300)) * dw.double()).sum()
    finite = torch.where(z.double() > -math.inf, z.double(), -1e4)
    slope = (loss(finite + h * v) - loss(finite - h * v)) / (2 * h)
    assert abs(slope - (want * v).sum()) <= 1e-6 * (1 + abs(slope))


# ---- dispatch and combination ----
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("T,E,k,H", [(1, 4, 2, 64), (33, 8, 2, 520), (7, 3, 3, 1), (50, 16, 5, 77), (300, 64, 8, 4096), (64, 8, 1, 1000),
                                     (2100, 16, 3, 300), (2048, 40, 9, 1032)])
def test_dispatch_and_combine(sk, dtype, T, E, k, H):
    t = TYPES[dtype]
    z = rand((T, E), torch.float32, T)
    z[rand((T, E), torch.float32, E) > 0.8] = -math.inf
    z[::5] = -math.inf
    route = sk.route_experts(z, k)
    x, y = rand((T, H), t, 1), rand((T * k, H), t, 2)
    rows = sk.dispatch_rows(x, route)
    order, place, weights = route.order.long(), route.place.long(), route.weights.double()
    assert torch.equal(rows, torch.where((order >= 0)[:, None], x[order.clamp(min=0) // k], 0))
    used = (place >= 0)[..., None]
    picked = torch.where(used, y.double()[place.clamp(min=0)], 0)
    out = sk.combine_rows(y, route)
    assert_near(out, (picked * weights[..., None]).sum(1), k, (picked * weights[..., None]).abs().sum(1))
    assert not out[::5].any()
    # gradients: formulas
    x.requires_grad_()
    y.requires_grad_()
    route.weights.requires_grad_()
    rows, out = sk.dispatch_rows(x, route), sk.combine_rows(y, route)
    d_rows, d_out = rand((T * k, H), t, 3), rand((T, H), t, 4)
    dx, dy, dw = torch.autograd.grad((rows, out), (x, y, route.weights), (d_rows, d_out))
    g = torch.where(used, d_rows.double()[place.clamp(min=0)], 0)
    assert_near(dx, g.sum(1), k, g.abs().sum(1))
    flat = weights.view(-1)[order.clamp(min=0)][:, None] * d_out.double()[order.clamp(min=0) // k]
    flat = torch.where((order >= 0)[:, None], flat, 0)
    assert_near(dy, flat, 1, flat.abs())
    terms = picked * d_out.double()[:, None, :]
    assert ((dw.double() - terms.sum(2)).abs() <= 2 * H * 2.0 ** -24 * terms.abs().sum(2) + 1e-37).all()
    # differences: the combination is linear in the weights
    wv = torch.rand(T, k, generator=torch.Generator().manual_seed(9)).cuda() * used[..., 0]
    moved = sk.combine_rows(y.detach(), route._replace(weights=route.weights.detach() + wv)).double() - out.detach().double()
    m = ((picked.abs() * (weights + wv.double())[..., None]).sum(1) * d_out.double().abs()).sum()
    assert abs((moved * d_out.double()).sum() - (dw.double() * wv.double()).sum()) <= 6 * ROUNDING[t] * 2 * m / math.sqrt(T * H) + 1e-6 * m


@pytest.mark.gpu
def test_dispatch_moves_any_type(sk):
    route = sk.route_experts(rand((20, 4), torch.float32, 1), 2)
    for x in (torch.randint(-128, 128, (20, 48), dtype=torch.int8, device="cuda"), torch.randn(20, device="cuda"), torch.randn(20, 3, device="cuda"),
              torch.randint(-128, 128, (20, 13), dtype=torch.int8, device="cuda"), torch.randn(20, 64, device="cuda").half()[:, 8:40], torch.randn(6, 20, device="cuda").t()):
        assert torch.equal(sk.dispatch_rows(x, route), x[route.order.long() // 2])
    assert sk.dispatch_rows(torch.empty(0, 8, device="cuda"), sk.route_experts(torch.empty(0, 4, device="cuda"), 2)).shape == (0, 8)


# ---- refusals ----
def test_calls_are_refused_with_codes(sk):
    L, lib = sk.lib(), __import__("streamk._lib", fromlist=["x"])
    p = 1 << 12   # (an aligned address; every call below is refused before it is used)

    def grouped(**kw):
        d = dict(dtype=lib.SK_F16, layout=0, out_dtype=lib.SK_F16, activation=0, E=2, R=10, N=64, K=64, A=p, B=p, offsets=p, C=p, lda=64, ldb=64, ldc=64, expert_b=4096)
        return L.sk_gemm_grouped(ctypes.byref(lib.SkGrouped(**{**d, **kw})), None, 0, None)
    assert L.sk_gemm_grouped(None, None, 0, None) == -1
    assert grouped(A=None) == -1 and grouped(offsets=None) == -1 and grouped(dtype=lib.SK_I8, out_dtype=0) == -1
    for bad in (dict(dtype=lib.SK_F32, out_dtype=lib.SK_F32), dict(out_dtype=lib.SK_BF16), dict(layout=2), dict(activation=4), dict(scale_a=p), dict(activation=-1),
                dict(dtype=lib.SK_I8, scale_a=p, scale_b=p, layout=1), dict(dtype=lib.SK_I8, scale_a=p, scale_b=p, out_dtype=lib.SK_F32)):
        assert grouped(**bad) == -4, bad
    for bad in (dict(E=0), dict(R=0), dict(N=0), dict(K=-8), dict(lda=56), dict(ldb=56), dict(ldc=63), dict(expert_b=-8), dict(R=1 << 31), dict(lda=1 << 40),
                dict(layout=1, K=65, lda=64)):
        assert grouped(**bad) == -2, bad
    for bad in (dict(K=60), dict(lda=68), dict(ldb=68), dict(expert_b=4100), dict(A=p + 8), dict(B=p + 2), dict(C=p + 1), dict(offsets=p + 2), dict(bias=p + 1),
                dict(layout=1, N=60), dict(dtype=lib.SK_I8, scale_a=p, scale_b=p, K=56)):
        assert grouped(**bad) == -3, bad
    wgrad = lambda A=p, dtype=0, E=2, R=5, M=64, N=64, lda=64, ldb=64: L.sk_grouped_wgrad(A, p, p, p, dtype, E, R, M, N, lda, ldb, 0, None)  # noqa: E731
    assert wgrad(A=None) == -1 and wgrad(dtype=lib.SK_I8) == -4 and wgrad(E=0) == -2 and wgrad(M=65, lda=64) == -2 and wgrad(N=60) == -3 and wgrad(A=p + 4) == -3
    route = lambda logits=p, dtype=1, T=100, E=8, k=2, ld=8, ws=p, n=1 << 20: L.sk_route_experts(logits, dtype, T, E, k, ld, p, p, p, p, p, ws, n, None)  # noqa: E731
    assert route(logits=None) == -1 and route(dtype=lib.SK_I8) == -4 and route(k=9) == -2 and route(E=1025, ld=1025) == -2 and route(ld=7) == -2 and route(T=0) == -2
    assert route(n=4) == -5 and route(ws=None) == -5 and route(ws=p + 2) == -3
    assert L.sk_route_workspace_bytes(16, 64, 8) == 0 and L.sk_route_workspace_bytes(100, 8, 2) > 0 and L.sk_route_workspace_bytes(100, 8, 9) == 0
    assert L.sk_route_backward(p, p, None, 4, 8, 2, 1, p, None) == -1 and L.sk_route_backward(p, p, p, 4, 8, 9, 1, p, None) == -2
    assert L.sk_dispatch_rows(p, 16, 8, p, p, 4, 2, p, None) == -2 and L.sk_dispatch_rows(None, 16, 16, p, None, 4, 2, p, None) == -1
    assert L.sk_combine_rows(p, lib.SK_F32, p, p, 4, 2, 8, p, None) == -4 and L.sk_combine_rows(p, 0, p, p, 4, 2, 0, p, None) == -2
    assert L.sk_combine_backward(p, p, 0, p, p, None, 4, 2, 8, p, p, None) == -1


def test_fake_implementations(sk):
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        new = lambda *s, dtype=torch.float16: torch.empty(*s, dtype=dtype, device="cuda")  # noqa: E731
        off = new(4, dtype=torch.int32)
        assert torch.ops.streamk.gemm_grouped(new(10, 64), new(3, 32, 64), off).shape == (10, 32)
        assert torch.ops.streamk.gemm_grouped(new(10, 64), new(3, 64, 32), off, "nn").shape == (10, 32)
        assert torch.ops.streamk.gemm_grouped(new(10, 64, dtype=torch.int8), new(3, 32, 64, dtype=torch.int8), off, "nt", torch.bfloat16).dtype == torch.bfloat16
        assert torch.ops.streamk.grouped_wgrad(new(10, 32), new(10, 64), off).shape == (3, 32, 64)
        w, e, o, order, place = torch.ops.streamk.route_experts(new(6, 3), 2)
        assert w.shape == e.shape == place.shape == (6, 2) and o.shape == (4,) and order.shape == (12,) and w.dtype == torch.float32 and e.dtype == torch.int32
        assert torch.ops.streamk.dispatch_rows(new(6, 64), order, 2).shape == (12, 64)
        assert torch.ops.streamk.combine_rows(new(12, 64), place, w).shape == (6, 64)


@pytest.mark.gpu
def test_wrong_operands_are_refused(sk):
    A, B, offsets = rand((20, 64), torch.float16, 1), rand((2, 32, 64), torch.float16, 2), offsets_of([12, 8])
    i8 = lambda t: (t * 10).to(torch.int8)  # noqa: E731
    for args, kw, error in [((A, B.bfloat16(), offsets), {}, TypeError), ((A.float(), B.float(), offsets), {}, TypeError), ((A, B[0], offsets), {}, ValueError),
                            ((A, B, offsets.long()), {}, TypeError), ((A, B, offsets[:2]), {}, ValueError), ((A, B, offsets.cpu()), {}, TypeError),
                            ((A[:, :32], B, offsets), {}, ValueError), ((A, B, offsets), dict(layout="tn"), ValueError), ((A, B, offsets), dict(activation="tanh"), ValueError),
                            ((A, B, offsets), dict(bias=torch.zeros(32, device="cuda").half()), ValueError), ((A, B, offsets), dict(out_dtype=torch.bfloat16), ValueError),
                            ((i8(A), i8(B), offsets), {}, ValueError), ((A, B, offsets), dict(scale_a=torch.ones(20, device="cuda")), ValueError),
                            ((A, B, offsets), dict(out=torch.empty(20, 31, device="cuda").half()), ValueError), ((A[:, :60], B[:, :, :60], offsets), {}, sk.StreamKError),
                            ((A, B.transpose(1, 2), offsets), dict(layout="nn"), ValueError)]:
        with pytest.raises(error):
            sk.streamk_grouped(*args, **kw)
    with pytest.raises(ValueError):
        sk.streamk_grouped_wgrad(A, A[:10], offsets)
    with pytest.raises(ValueError):
        sk.streamk_grouped_wgrad(A, A[:, :60], offsets)
    for z, k, error in [(torch.zeros(4, 8, device="cuda"), 9, ValueError), (torch.zeros(4, 8, device="cuda"), 0, ValueError), (torch.zeros(4, 1025, device="cuda"), 2, ValueError),
                        (torch.zeros(4, 8, device="cuda").double(), 2, TypeError), (torch.zeros(8, device="cuda"), 2, ValueError)]:
        with pytest.raises(error):
            sk.route_experts(z, k)
    route = sk.route_experts(torch.zeros(4, 8, device="cuda"), 2)
    with pytest.raises(ValueError):
        sk.dispatch_rows(torch.zeros(5, 8, device="cuda"), route)
    with pytest.raises(ValueError):
        sk.combine_rows(torch.zeros(7, 8, device="cuda").half(), route)


# ---- every kind of tile on every kind of groups ----
VARIANTS = [1, 2, 3, 4, 5, 6]


@pytest.mark.gpu
@pytest.mark.parametrize("variant", VARIANTS)
@pytest.mark.parametrize("kind", ["float16 nt", "bfloat16 nt", "float16 nn", "bfloat16 nn", "int8"])
@pytest.mark.parametrize("sizes", sorted(SIZES))
@pytest.mark.parametrize("N,K,padding", [(520, 256, 0), (264, 128, 24), (1032, 640, 0)])
def test_grouped_variants(sk, variant, kind, sizes, N, K, padding):
    sizes = SIZES[sizes]
    R, E = sum(sizes) + 2, len(sizes)
    offsets = offsets_of(sizes)
    out = torch.full((R, N + padding), 7.0, dtype=torch.bfloat16 if kind == "int8" else TYPES[kind.split()[0]], device="cuda")
    bias = rand((E, N), out.dtype, 5)
    if kind.endswith("nn") and variant > 2:
        return   # ([E, N, K] weights only)
    if kind == "int8":
        g = torch.Generator().manual_seed(R + N)
        A = torch.randint(-127, 128, (R, K), generator=g, dtype=torch.int8).cuda()
        B = torch.randint(-127, 128, (E, N, K), generator=g, dtype=torch.int8).cuda()
        sa, sb = (torch.rand(R, generator=g) + 0.5).cuda() * 0.01, (torch.rand(E, N, generator=g) + 0.5).cuda() / (73 * math.sqrt(K))
        run = lambda **kw: sk.streamk_grouped(A, B, offsets, scale_a=sa, scale_b=sb, variant=variant, **kw)  # noqa: E731
        pre, magnitudes = plain(A, B, sizes)
        pre, magnitudes = pre * sa.double()[:, None], 0
        for e, at in groups(sizes):
            pre[at] *= sb[e].double()
    else:
        layout = kind.split()[1]
        A, B = rand((R, K), out.dtype, R), rand((E, N, K) if layout == "nt" else (E, K, N), out.dtype, N, 1 / math.sqrt(K))
        run = lambda **kw: sk.streamk_grouped(A, B, offsets, layout=layout, variant=variant, **kw)  # noqa: E731
        pre, magnitudes = plain(A, B, sizes, layout)
    C = run(out_dtype=out.dtype)
    assert_near(C, pre, K, magnitudes, pre)
    assert not C[R - 2:].any()
    for e, at in groups(sizes):
        pre[at] += bias[e].double()
    run(out=out[:, :N], bias=bias, activation="gelu_tanh")
    want = activate(pre, "gelu_tanh")
    want[R - 2:] = 0
    assert_near(out[:, :N], want, K, 1.2 * magnitudes, pre)
    assert (out[:, N:] == 7).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("sizes", sorted(SIZES))
@pytest.mark.parametrize("N,K,padding", [(520, 256, 0), (264, 36, 24), (1032, 645, 0), (64, 1536, 0), (8, 1, 8)])
def test_grouped_kn_weights_on_tiles_that_stream_k(sk, dtype, sizes, N, K, padding):
    sizes = SIZES[sizes]
    R, E = sum(sizes) + 2, len(sizes)
    whole = torch.zeros(R, (K + 7) // 8 * 8, dtype=TYPES[dtype], device="cuda")
    A, B, bias = whole[:, :K], rand((E, K, N), TYPES[dtype], N, 1 / math.sqrt(K)), rand((E, N), TYPES[dtype], 5)
    A.copy_(rand((R, K), TYPES[dtype], R))
    out = torch.full((R, N + padding), 7.0, dtype=TYPES[dtype], device="cuda")
    pre, magnitudes = plain(A, B, sizes, "nn")
    for e, at in groups(sizes):
        pre[at] += bias[e].double()
    sk.streamk_grouped(A, B, offsets_of(sizes), layout="nn", variant=5, out=out[:, :N], bias=bias, activation="gelu_tanh")
    want = activate(pre, "gelu_tanh")
    want[R - 2:] = 0
    assert_near(out[:, :N], want, K, 1.2 * magnitudes, pre)
    assert (out[:, N:] == 7).all()
    again = torch.full_like(out, 7.0)
    sk.streamk_grouped(A, B, offsets_of(sizes), layout="nn", variant=5, out=again[:, :N], bias=bias, activation="gelu_tanh")
    assert torch.equal(out, again)


@pytest.mark.gpu
@pytest.mark.parametrize("N", [40, 37])
def test_rows_that_stand_for_many(sk, N):
    """Broadcast rows of A and broadcast gradients (those of a sum over the rows) have stride 0."""
    sizes, K = [5, 0, 25, 7], 64
    offsets, R = offsets_of(sizes), sum(sizes)
    B, row, d = rand((4, N, K), torch.float16, 1, 0.125), rand((1, K), torch.float16, 2), rand((1, N), torch.float16, 3)
    A = row.expand(R, K)
    assert torch.equal(sk.streamk_grouped(A, B, offsets), sk.streamk_grouped(A.contiguous(), B, offsets))
    for one, other in ((A, d.expand(R, N)), (A.contiguous(), d.expand(R, N)), (A, d.expand(R, N).contiguous())):
        x, w = one.detach().requires_grad_(), B.clone().requires_grad_()
        dx, dw = torch.autograd.grad(sk.streamk_grouped(x, w, offsets), (x, w), other)
        for e, at in groups(sizes):
            assert_near(dx[at], other[at].double() @ B[e].double(), N, other[at].double().abs() @ B[e].double().abs())
            assert_near(dw[e], other[at].double().T @ one[at].double(), sizes[e], other[at].double().abs().T @ one[at].double().abs())


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["float16", "bfloat16", "float16 nn", "bfloat16 nn", "int8"])
@pytest.mark.parametrize("sizes", [[1, 64, 65, 0, 128, 129, 192], [256, 257, 384, 385, 320], [127], [128, 128], [700, 60], [100] * 70])
@pytest.mark.parametrize("N,K", [(256, 128), (520, 640), (1024, 4096), (72, 256)])
def test_grouped_tiles_of_half_the_rows(sk, kind, sizes, N, K):
    """256 x 256 tiles of which at most 128 rows are used are another kind, also where they are cut along K."""
    R, E = sum(sizes) + 1, len(sizes)
    out = torch.full((R, N), 7.0, dtype=torch.float16 if kind == "int8" else TYPES[kind.split()[0]], device="cuda")
    bias, kw = rand((E, N), out.dtype, 5), {}
    if kind == "int8":
        g = torch.Generator().manual_seed(R + N)
        A = torch.randint(-127, 128, (R, K), generator=g, dtype=torch.int8).cuda()
        B = torch.randint(-127, 128, (E, N, K), generator=g, dtype=torch.int8).cuda()
        sa, sb = (torch.rand(R, generator=g) + 0.5).cuda() * 0.01, (torch.rand(E, N, generator=g) + 0.5).cuda() / (73 * math.sqrt(K))
        kw = dict(scale_a=sa, scale_b=sb)
        pre, magnitudes = plain(A, B, sizes)
        pre, magnitudes = pre * sa.double()[:, None], 0
        for e, at in groups(sizes):
            pre[at] *= sb[e].double()
    else:
        layout = "nn" if kind.endswith("nn") else "nt"
        A, B = rand((R, K), out.dtype, R), rand((E, N, K) if layout == "nt" else (E, K, N), out.dtype, N, 1 / math.sqrt(K))
        kw = dict(layout=layout)
        pre, magnitudes = plain(A, B, sizes, layout)
    C = sk.streamk_grouped(A, B, offsets_of(sizes), variant=2, out_dtype=out.dtype, **kw)
    assert_near(C, pre, K, magnitudes, pre)
    assert not C[R - 1:].any()
    for e, at in groups(sizes):
        pre[at] += bias[e].double()
    sk.streamk_grouped(A, B, offsets_of(sizes), variant=2, out=out, bias=bias, activation="silu", **kw)
    want = activate(pre, "silu")
    want[R - 1:] = 0
    assert_near(out, want, K, 1.2 * magnitudes, pre)
    assert torch.equal(C, sk.streamk_grouped(A, B, offsets_of(sizes), variant=2, out_dtype=out.dtype, **kw))


@pytest.mark.gpu
@pytest.mark.parametrize("variant", [1, 2])
@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("sizes", sorted(SIZES))
@pytest.mark.parametrize("M,N", [(513, 264), (256, 520), (64, 8)])
def test_weight_gradient_variants(sk, variant, dtype, sizes, M, N):
    sizes = SIZES[sizes]
    R = sum(sizes) + 3
    dC, A = rand((R, M), TYPES[dtype], R), rand((R, N), TYPES[dtype], N)
    got = sk.streamk_grouped_wgrad(dC, A, offsets_of(sizes), variant=variant)
    for e, at in groups(sizes):
        assert_near(got[e], dC[at].double().T @ A[at].double(), sizes[e], dC[at].double().abs().T @ A[at].double().abs())


@pytest.mark.gpu
def test_variants_that_do_not_take_a_problem_are_refused(sk):
    A, B, offsets = rand((20, 72), torch.float16, 1), rand((2, 32, 72), torch.float16, 2), offsets_of([12, 8])
    for variant in (2, 99, -1):
        with pytest.raises(sk.StreamKError) as e:
            sk.streamk_grouped(A, B, offsets, variant=variant)
        assert e.value.status == -4
    for variant in (99, -1):
        with pytest.raises(sk.StreamKError) as e:
            sk.streamk_grouped_wgrad(A, A, offsets, variant=variant)
        assert e.value.status == -4


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["float16 nt", "bfloat16 nn", "int8"])
@pytest.mark.parametrize("variant,sizes,N,K", [(2, [300, 0, 200], 512, 4096), (2, [300, 0, 200], 512, 4224), (2, [2000], 2304, 4096), (2, [40, 4000], 4352, 4096),
                                               (3, [3, 0, 9], 520, 4096), (4, [30, 100, 1], 264, 2176), (5, [70, 200], 1000, 2048), (6, [128, 64], 512, 8192)])
def test_tiles_that_are_cut_along_k(sk, kind, variant, sizes, N, K):
    """Tiles shared by several CTAs: right, and the same bits launch after launch, in whatever order the parts arrive."""
    if kind.endswith("nn") and variant > 2:
        return
    R, E = sum(sizes), len(sizes)
    offsets = offsets_of(sizes)
    if kind == "int8":
        g = torch.Generator().manual_seed(R)
        A = torch.randint(-127, 128, (R, K), generator=g, dtype=torch.int8).cuda()
        B = torch.randint(-127, 128, (E, N, K), generator=g, dtype=torch.int8).cuda()
        sa, sb = (torch.rand(R, generator=g) + 0.5).cuda() * 0.01, (torch.rand(E, N, generator=g) + 0.5).cuda() / (73 * math.sqrt(K))
        run = lambda: sk.streamk_grouped(A, B, offsets, scale_a=sa, scale_b=sb, variant=variant)  # noqa: E731
        pre, magnitudes = plain(A, B, sizes)
        pre, magnitudes = pre * sa.double()[:, None], 0
        for e, at in groups(sizes):
            pre[at] *= sb[e].double()
    else:
        dtype, layout = kind.split()
        A, B = rand((R, K), TYPES[dtype], R), rand((E, N, K) if layout == "nt" else (E, K, N), TYPES[dtype], N, 1 / math.sqrt(K))
        run = lambda: sk.streamk_grouped(A, B, offsets, layout=layout, variant=variant)  # noqa: E731
        pre, magnitudes = plain(A, B, sizes, layout)
    C = run()
    assert_near(C, pre, K, magnitudes, pre)
    for _ in range(5):
        assert torch.equal(run(), C)
    sk.workspace_status()


@pytest.mark.gpu
def test_operators_pass_opcheck(sk):
    o, check = torch.ops.streamk, torch.library.opcheck
    tests = ("test_schema", "test_faketensor", "test_aot_dispatch_dynamic")
    A, B, offsets = rand((20, 64), torch.float16, 1), rand((2, 32, 64), torch.float16, 2), offsets_of([12, 8])
    route = sk.route_experts(rand((10, 4), torch.float32, 3), 2)
    check(o.gemm_grouped, (A, B, offsets), test_utils=tests)
    check(o.gemm_grouped, (A.detach().requires_grad_(), B.detach().requires_grad_(), offsets), test_utils=tests)
    check(o.grouped_wgrad, (A[:, :32].contiguous(), A, offsets), test_utils=tests)
    check(o.route_experts, (rand((10, 4), torch.float32, 3), 2), test_utils=tests)
    check(o.dispatch_routed, (rand((10, 64), torch.float16, 4), route.order, route.place), test_utils=tests)
    check(o.combine_routed, (A, route.weights, route.order, route.place), test_utils=tests)
    check(o.quantize_i8, (A,), test_utils=tests)
    q, s = sk.quantize_int8(A)
    check(o.gemm_i8_scaled, (q, q, s, s, torch.float16), test_utils=tests)


@pytest.mark.gpu
def test_native_operators_answer_like_the_general_ones(sk):
    """The two implementations of every operator, on ordinary operands and on ones that the native one passes on."""
    o = torch.ops.streamk
    A, B, offsets = rand((20, 64), torch.float16, 1), rand((2, 32, 64), torch.float16, 2), offsets_of([12, 8])
    wide = torch.zeros(20, 80, dtype=torch.float16, device="cuda")
    wide[:, 1:65] = A
    logits, place = rand((10, 4), torch.float32, 3), None
    route = sk.route_experts(logits, 2)
    q, s = sk.quantize_int8(A)
    w, sw = sk.quantize_int8(B)
    calls = [("gemm_grouped", (A, B, offsets)), ("gemm_grouped", (wide[:, 1:65], B, offsets)), ("gemm_grouped", (A[:1], B, offsets_of([1, 0]))), ("gemm_grouped", (A[:0], B, offsets_of([0, 0]))),
             ("gemm_grouped", (A, B, offsets, "nt", None, None, None, rand((2, 32), torch.float16, 5), "silu")), ("gemm_grouped", (A, B[:, :1], offsets)),
             ("gemm_grouped", (q, w, offsets, "nt", torch.bfloat16, s, sw)), ("gemm_grouped", (q, w, offsets, "nt", None, s, sw)), ("gemm_grouped", (A, rand((2, 64, 32), torch.float16, 6), offsets, "nn")),
             ("grouped_wgrad", (A, A, offsets)), ("grouped_wgrad", (wide[:, :77], A, offsets)), ("route_experts", (logits, 2)), ("route_experts", (logits[:, 1:], 3)), ("route_experts", (logits.half(), 1)),
             ("route_backward", (route.weights, route.experts, route.weights, 4, torch.float32)), ("dispatch_rows", (A[:10], route.order, 2)), ("dispatch_rows", (wide[:10, 1:65], route.order, 2)),
             ("dispatch_rows", (s[:10].contiguous(), route.order, 2)), ("combine_rows", (A, route.place, route.weights)), ("combine_rows", (A, route.place)), ("combine_rows", (wide[:, 1:65], route.place)),
             ("combine_backward", (A[:10], A, route.order, route.place, route.weights)), ("combine_backward", (A[:1].expand(10, 64), A, route.order, route.place, route.weights)),
             ("quantize_i8", (A,)), ("quantize_i8", (wide[:, 1:65],)), ("quantize_i8", (B,))]
    for name, args in calls:
        got, want = getattr(o, name)(*args), getattr(o, name + "_general")(*args)
        for a, b in zip(got if isinstance(got, (tuple, list)) else [got], want if isinstance(want, (tuple, list)) else [want]):
            assert a.dtype == b.dtype and a.shape == b.shape and torch.equal(a, b), name
    out, ref = torch.empty(20, 40, dtype=torch.float16, device="cuda"), torch.empty(20, 40, dtype=torch.float16, device="cuda")
    o.gemm_grouped_out(A, B, offsets, out[:, :32])
    o.gemm_grouped_out_general(A, B, offsets, ref[:, :32])
    assert torch.equal(out[:, :32], ref[:, :32])


@pytest.mark.gpu
def test_gradients_of_gradients_are_refused(sk):
    A, B, offsets = rand((20, 64), torch.float16, 1).requires_grad_(), rand((2, 32, 64), torch.float16, 2), offsets_of([12, 8])
    C = sk.streamk_grouped(A, B, offsets)
    with pytest.raises(RuntimeError):
        g, = torch.autograd.grad(C.float().square().sum(), A, create_graph=True)
        g.sum().backward()


# ---- offsets that 32 bits do not hold ----
@pytest.mark.gpu
@pytest.mark.parametrize("variant", [0, 1, 2, 3, 6])
@pytest.mark.parametrize("kind", ["bfloat16", "int8"])
def test_weights_beyond_4_gib(sk, variant, kind):
    E, N, K, sizes = (5, 8192, 65536, [2, 0, 130, 1, 3]) if kind == "bfloat16" else (5, 16384, 65536, [2, 0, 130, 1, 3])
    R = sum(sizes)
    if kind == "int8":
        B = torch.empty((E, N, K), dtype=torch.int8, device="cuda").random_(-127, 128)
        A = torch.empty((R, K), dtype=torch.int8, device="cuda").random_(-127, 128)
        sa, sb = torch.rand(R, device="cuda") + 0.5, (torch.rand(E, N, device="cuda") + 0.5) / (73 ** 2 * 256)
        C = sk.streamk_grouped(A, B, offsets_of(sizes), scale_a=sa, scale_b=sb, variant=variant)
    else:
        B = torch.empty((E, N, K), dtype=torch.bfloat16, device="cuda").normal_(0, 1 / 256)
        A = rand((R, K), torch.bfloat16, 3)
        C = sk.streamk_grouped(A, B, offsets_of(sizes), variant=variant)
    for e, at in groups(sizes):
        for cols in (slice(0, 40), slice(N - 40, N)):
            pre = A[at].double() @ B[e, cols].double().T
            magnitudes = A[at].double().abs() @ B[e, cols].double().abs().T
            if kind == "int8":
                pre, magnitudes = pre * sa[at, None].double() * sb[e, cols].double(), 0
            assert_near(C[at, cols], pre, K, magnitudes, pre)


@pytest.mark.gpu
@pytest.mark.parametrize("layout,variant", [("nt", 0), ("nt", 1), ("nt", 2), ("nt", 6), ("nn", 1), ("nn", 2), ("nn", 5)])
def test_rows_beyond_4_gib(sk, layout, variant):
    R, N, K = 140_000, 16384, 64
    sizes = [R - 300, 300]
    A, B = rand((R, K), torch.bfloat16, 1), rand((2, N, K) if layout == "nt" else (2, K, N), torch.bfloat16, 2, 0.125)
    C = sk.streamk_grouped(A, B, offsets_of(sizes), layout=layout, variant=variant)
    assert C.numel() * 2 > 2 ** 32
    for rows in (slice(0, 5), slice(131_070, 131_075), slice(R - 305, R - 300), slice(R - 5, R)):
        e = int(rows.start >= sizes[0])
        W = B[e].double().T if layout == "nt" else B[e].double()
        assert_near(C[rows], A[rows].double() @ W, K, A[rows].double().abs() @ W.abs())


@pytest.mark.gpu
@pytest.mark.parametrize("variant", [0, 1, 2])
def test_weight_gradients_beyond_4_gib(sk, variant):
    sizes, N, K = [100, 0, 30, 0, 0, 0, 1, 0, 90], 16384, 16384
    dC, A = rand((sum(sizes), N), torch.bfloat16, 1), rand((sum(sizes), K), torch.bfloat16, 2)
    dW = sk.streamk_grouped_wgrad(dC, A, offsets_of(sizes), variant=variant)
    assert dW.numel() * 2 > 2 ** 32
    for e, at in groups(sizes):
        for rows in (slice(0, 8), slice(N - 8, N)):
            assert_near(dW[e, rows], dC[at, rows].double().T @ A[at].double(), sizes[e], dC[at, rows].double().abs().T @ A[at].double().abs())


@pytest.mark.gpu
def test_exchange_beyond_4_gib(sk):
    T, E, k, H = 70_000, 16, 4, 8192
    logits = torch.randn(T, E, device="cuda")
    route = sk.route_experts(logits, k)
    x = torch.randn(T, H, device="cuda", dtype=torch.bfloat16)
    rows = sk.dispatch_rows(x, route)
    assert rows.numel() * 2 > 2 ** 32
    for at in (slice(0, 10), slice(T * k - 10, T * k), slice(262_100, 262_200)):
        assert torch.equal(rows[at], x[route.order[at].long() // k])
    out = sk.combine_rows(rows, route)
    # (the same row k times, with weights that sum to one up to k fp32 roundings)
    assert ((out.float() - x.float()).abs() <= (2.0 ** -8 + 8 * 2.0 ** -24) * x.float().abs() + 1e-30).all()
    rows.requires_grad_()
    weights = route.weights.clone().requires_grad_()
    d_out = torch.randn(T, H, device="cuda", dtype=torch.bfloat16)
    d_rows, d_weights = torch.autograd.grad(sk.combine_rows(rows, route._replace(weights=weights)), (rows, weights), d_out)
    last = torch.arange(T * k - 10, T * k, device="cuda")
    slots = route.order[last].long()
    want = (weights.detach().flatten()[slots, None] * d_out[slots // k].float()).bfloat16()
    assert torch.equal(d_rows[last], want)
    y = rows.detach()[route.place[T - 1].long()].double()
    off = (d_weights[T - 1].double() - y @ d_out[T - 1].double()).abs()
    assert (off <= 2 * H * 2.0 ** -24 * (y.abs() @ d_out[T - 1].double().abs())).all()


# ---- NaN and infinities stay where they belong ----
@pytest.mark.gpu
@pytest.mark.parametrize("variant", VARIANTS)
@pytest.mark.parametrize("kind", ["float16 nt", "bfloat16 nn", "int8"])
def test_bad_rows_and_weights_of_other_experts(sk, variant, kind):
    """Experts 0, 2 and 5 own bad rows or weights; 1 and 6 have no rows, bad weights and no part in anything."""
    sizes, N, K = [3, 0, 130, 70, 257, 1, 0, 40], 264, 256
    if kind.endswith("nn") and variant not in (1, 2, 5):
        return   # ([E, N, K] weights only)
    R, offsets = sum(sizes) + 4, offsets_of(sizes)
    at = dict(groups(sizes))
    if kind == "int8":
        A, B = torch.empty((R, K), dtype=torch.int8, device="cuda").random_(-127, 128), torch.empty((len(sizes), N, K), dtype=torch.int8, device="cuda").random_(-127, 128)
        sa, sb = torch.rand(R, device="cuda") + 0.5, (torch.rand(len(sizes), N, device="cuda") + 0.5) / 73 ** 2
        clean = sk.streamk_grouped(A, B, offsets, scale_a=sa, scale_b=sb, variant=variant)
        sa[at[0].start] = float("nan")
        sa[at[2].stop - 1] = float("inf")
        sa[R - 4:] = float("nan")
        sb[1] = sb[6] = sb[5] = float("nan")
        C = sk.streamk_grouped(A, B, offsets, scale_a=sa, scale_b=sb, variant=variant)
    else:
        dtype, layout = TYPES[kind.split()[0]], kind.split()[1]
        A, B = rand((R, K), dtype, 1), rand((len(sizes), N, K) if layout == "nt" else (len(sizes), K, N), dtype, 2, 1 / 16)
        clean = sk.streamk_grouped(A, B, offsets, layout=layout, variant=variant)
        A[at[0].start, 5] = float("nan")
        A[at[2].stop - 1, K - 1] = float("inf")
        A[R - 4:] = float("nan")
        B[1] = B[6] = B[5] = float("nan")
        C = sk.streamk_grouped(A, B, offsets, layout=layout, variant=variant)
    bad = torch.zeros(R, dtype=torch.bool, device="cuda")
    bad[at[0].start] = bad[at[2].stop - 1] = bad[at[5]] = True
    assert torch.equal(C[~bad], clean[~bad])
    assert not torch.isfinite(C[bad]).any(1).any() if kind != "int8" else torch.isnan(C[at[0].start]).all() and torch.isnan(C[at[5]]).all()
    assert not C[R - 4:].any()


@pytest.mark.gpu
@pytest.mark.parametrize("variant", [1, 2])
@pytest.mark.parametrize("dtype", sorted(TYPES))
def test_bad_rows_in_weight_gradients(sk, variant, dtype):
    sizes, N, K = [3, 0, 130, 70, 257], 264, 256
    R, offsets, at = sum(sizes) + 4, offsets_of(sizes), dict(groups(sizes))
    dC, A = rand((R, N), TYPES[dtype], 1), rand((R, K), TYPES[dtype], 2)
    clean = sk.streamk_grouped_wgrad(dC, A, offsets, variant=variant)
    A[at[2].start] = float("nan")
    dC[at[2].stop - 1] = float("inf")
    A[R - 4:] = dC[R - 4:] = float("nan")
    dW = sk.streamk_grouped_wgrad(dC, A, offsets, variant=variant)
    for e in (0, 1, 3, 4):
        assert torch.equal(dW[e], clean[e])
    assert torch.isnan(dW[2]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("T", [5, 300])
def test_bad_rows_in_the_exchange(sk, T):
    """Tokens without experts, with fewer than k, and with bad rows: none of it reaches another token."""
    E, k, H = 6, 3, 72
    logits = torch.randn(T, E, device="cuda")
    logits[0] = float("-inf")
    logits[1, 1:] = float("-inf")
    logits[3, 2] = float("nan")
    route = sk.route_experts(logits, k)
    assert (route.experts[0] == -1).all() and (route.experts[1, 1:] == -1).all() and not (route.experts[3] == 2).any()
    x = torch.randn(T, H, device="cuda").bfloat16()
    x[2] = float("nan")
    rows = sk.dispatch_rows(x, route)
    of = route.order.long()
    assert torch.equal(torch.isnan(rows).all(1), (of >= 0) & (of // k == 2)) and not rows[of < 0].any()
    clean = torch.randn(T * k, H, device="cuda").bfloat16()
    # sorted row 0 and the rows of token 2 are bad; so are those that belong to no slot
    y = clean.clone()
    y[0] = float("nan")
    y[route.place[2].long()] = float("inf")
    y[of < 0] = float("nan")
    token = of[0] // k
    got, want = sk.combine_rows(y, route), sk.combine_rows(clean, route)
    good = torch.ones(T, dtype=torch.bool, device="cuda")
    good[token] = good[2] = False
    assert torch.equal(got[good], want[good]) and not torch.isfinite(got[~good]).any() and not got[0].any()
    y.requires_grad_()
    weights = route.weights.clone().requires_grad_()
    d_out = torch.randn(T, H, device="cuda").bfloat16()
    d_out[2] = float("nan")
    dy, dw = torch.autograd.grad(sk.combine_rows(y, route._replace(weights=weights)), (y, weights), d_out)
    mine = (of >= 0) & (of // k == 2)
    assert torch.isfinite(dy[~mine]).all() and torch.isfinite(dw[good]).all() and not dy[of < 0].any() and not dw[0].any()
    dx, = torch.autograd.grad(sk.dispatch_rows(x.requires_grad_(), route), x, torch.where(mine[:, None], float("nan"), torch.ones(T * k, H, device="cuda").bfloat16()))
    keep = torch.arange(T, device="cuda") != 2
    assert torch.equal(dx[keep], (route.experts >= 0).sum(1, keepdim=True).expand(T, H)[keep].bfloat16())
