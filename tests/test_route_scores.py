"""Routing by scores, with a bias for balance and in groups, against the definition worked out token by token in 64 bits.

Tolerances: the kernels compute in 64 bits and round once, so a weight is within half a unit of float32 of the definition's (2^-24 of it), and
a gradient within 2^-24 of it -- it is float32 before it is stored -- and half a unit of its own type; sums and quotients of up to 64
terms in 64 bits leave 1e-13 of the terms' magnitudes.  2^-149, 2^-25 and 2^-134 are (half) steps of the types' smallest numbers."""
import ctypes
import math

import pytest
import torch

TYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}
SMALLEST = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}


@pytest.fixture(scope="module")
def sk():
    import streamk
    streamk.lib()
    return streamk


def scores_of(z, kind):
    """of one token's logits (64 bits), with the limits of infinities; NaN and -inf count for nothing"""
    there = z > -math.inf
    if kind == "sigmoid":
        return torch.where(there, torch.sigmoid(z), 0)
    most = z[there].max() if there.any() else torch.tensor(0.0)
    e = torch.where(there, torch.where(z == most, torch.ones_like(z), torch.exp(z - most)), 0)
    return e / e.sum() if there.any() else e


def plain_route(logits, k, scores="softmax", bias=None, groups=1, chosen_groups=1, renormalize=True, scale=1.0):
    """(weights, experts, offsets, order, place) on the CPU"""
    z = logits.detach().double().cpu()
    T, E = z.shape
    b = bias.double().cpu() if bias is not None else torch.zeros(E, dtype=torch.float64)
    weights, experts = torch.zeros(T, k, dtype=torch.float64), torch.full((T, k), -1)
    for t in range(T):
        s = scores_of(z[t], scores)
        c = s + b
        can = [e for e in range(E) if z[t, e] > -math.inf and c[e] > -math.inf]
        if chosen_groups < groups:
            size = E // groups
            total = {}
            for g in range(groups):
                best = sorted((c[e].item() for e in can if e // size == g), reverse=True)[:2]
                if best:
                    total[g] = sum(best)
            open_groups = sorted(total, key=lambda g: (-total[g], g))[:chosen_groups]
            can = [e for e in can if e // size in open_groups]
        by = c if bias is not None else z[t]
        chosen = sorted(can, key=lambda e: (-by[e].item(), e))[:k]
        if not chosen:
            continue
        w = s[chosen]
        if renormalize:
            m = z[t, chosen].max()
            if scores == "sigmoid" and m < -500:   # (sigmoid is e^z there: the quotients of what underflows)
                w = torch.exp(z[t, chosen] - m)
            elif scores == "softmax":
                w = torch.where(z[t, chosen] == m, 1.0, torch.exp(z[t, chosen] - m))
            w = w / w.sum()
        weights[t, :len(chosen)] = w * scale
        experts[t, :len(chosen)] = torch.tensor(chosen)
    slots = sorted((e, i) for i, e in enumerate(experts.view(-1).tolist()) if e >= 0)
    order, place, offsets = torch.full((T * k,), -1), torch.full((T * k,), -1), torch.zeros(E + 1, dtype=torch.long)
    for p, (e, i) in enumerate(slots):
        order[p], place[i] = i, p
        offsets[e + 1:] += 1
    return weights, experts, offsets, order, place.view(T, k)


def assert_route(route, want):
    weights, *whole = want
    for got, w, name in zip(route[1:], whole, ("experts", "offsets", "order", "place")):
        assert torch.equal(got.cpu().long(), w), name
    off = (route.weights.detach().double().cpu() - weights).abs()
    assert (off <= 2.0 ** -24 * 1.001 * weights.abs() + 1e-13 + 2.0 ** -149).all()


def logits_of(T, E, seed, dtype=torch.float32, std=2.0, closed=0.0):
    g = torch.Generator().manual_seed(seed)
    z = (torch.randn(T, E, generator=g) * std).to(dtype)
    if closed:
        z[torch.rand(T, E, generator=g) < closed] = -math.inf
        z[torch.rand(T, generator=g) < closed / 2] = -math.inf
    return z.cuda()


def bias_of(E, seed):
    return (torch.randn(E, generator=torch.Generator().manual_seed(seed)) * 50).round().mul(0.001).cuda()


@pytest.mark.gpu
@pytest.mark.parametrize("scores", ["softmax", "sigmoid"])
@pytest.mark.parametrize("with_bias", [False, True])
@pytest.mark.parametrize("T,E,k,groups,chosen_groups", [(1, 1, 1, 1, 1), (1, 8, 2, 1, 1), (5, 8, 2, 4, 2), (64, 256, 8, 8, 4), (65, 64, 6, 8, 3), (3, 6, 3, 6, 3),
                                                         (130, 160, 6, 8, 1), (17, 1024, 64, 64, 32), (70, 300, 7, 3, 2), (9, 384, 8, 1, 1), (200, 36, 5, 4, 4),
                                                         (40, 250, 8, 10, 4), (40, 680, 12, 40, 9), (33, 60, 5, 20, 7), (300, 96, 5, 3, 2), (1500, 24, 3, 3, 2)])
def test_route_by_scores(sk, scores, with_bias, T, E, k, groups, chosen_groups):
    z, bias = logits_of(T, E, 7 * T + E, closed=0.3), bias_of(E, E) if with_bias else None
    for renormalize, scale in ((True, 2.5), (False, 1.0)):
        how = dict(scores=scores, bias=bias, groups=groups, chosen_groups=chosen_groups, renormalize=renormalize, scale=scale)
        assert_route(sk.route_experts(z, k, **how), plain_route(z, k, **how))


@pytest.mark.gpu
@pytest.mark.parametrize("scores", ["softmax", "sigmoid"])
@pytest.mark.parametrize("T", [1, 7, 16])
@pytest.mark.parametrize("E,groups", [(250, 10), (240, 40), (252, 12), (255, 3)])
def test_few_tokens_in_groups_that_leave_lanes_unused(sk, E, groups, T, scores):
    z, bias = logits_of(T, E, 7 * T + E, closed=0.3), bias_of(E, E)
    for how in (dict(bias=None, renormalize=False), dict(bias=bias, renormalize=True, scale=2.5)):
        how.update(scores=scores, groups=groups, chosen_groups=groups // 2)
        assert_route(sk.route_experts(z, 5, **how), plain_route(z, 5, **how))


@pytest.mark.gpu
def test_few_tokens_in_groups_of_any_size(sk):
    """Every pair of groups and experts that one workgroup routes with more experts to a lane than 256 without groups have."""
    pairs = [(groups * size, groups) for groups in range(2, 65) for size in range(1, 256 // groups + 1) if groups * -(-size // 4) > 64]
    assert len(pairs) == 69
    for E, groups in pairs:
        z, how = logits_of(2, E, E + groups), dict(scores="sigmoid", bias=bias_of(E, groups), groups=groups, chosen_groups=groups - 1, scale=2.5)
        assert_route(sk.route_experts(z, 6, **how), plain_route(z, 6, **how))


@pytest.mark.gpu
@pytest.mark.parametrize("scores", [None, "sigmoid"])
@pytest.mark.parametrize("E,k,sizes", [(1, 1, (64, 65, 300, 2051)), (3, 2, (33, 64, 65, 700, 2049)), (8, 2, (56, 65, 511, 2050, 4100)), (60, 3, (51, 52, 520, 1030, 2056)),
                                       (100, 5, (37, 513, 520)), (129, 6, (33, 257, 520)), (256, 8, (25, 26, 259, 600)), (300, 4, (1, 9, 520))])
def test_counts_of_every_number_of_blocks(sk, E, k, sizes, scores):
    for T in sizes:
        z = logits_of(T, E, T + E, closed=0.2)
        how = dict() if scores is None else dict(scores=scores, bias=bias_of(E, T))
        got, want = sk.route_experts(z, k, **how), plain_route(z, k, **how)
        for a, b in zip(got[1:], want[1:]):   # (the weights do not come from counts)
            assert torch.equal(a.cpu().long(), b)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("scores", ["softmax", "sigmoid"])
def test_equal_scores_go_by_number(sk, dtype, scores):
    z = torch.randint(-2, 3, (100, 64), generator=torch.Generator().manual_seed(1)).to(TYPES[dtype]).cuda()
    for bias in (None, torch.zeros(64, device="cuda"), torch.full((64,), -0.25, device="cuda")):
        for groups, chosen_groups in ((1, 1), (8, 3), (32, 5), (64, 20)):
            how = dict(scores=scores, bias=bias, groups=groups, chosen_groups=chosen_groups, renormalize=False)
            assert_route(sk.route_experts(z, 4, **how), plain_route(z, 4, **how))


@pytest.mark.gpu
def test_neighbours_beyond_32_bits(sk):
    # scores that are equal in float32 and not in 64 bits: 1 - e^-20 and 1 - e^-21, and sums with a bias
    z = torch.tensor([[20.0, 21.0, 19.5, 20.5]], device="cuda")
    bias = torch.full((4,), 0.5, device="cuda")
    assert (torch.sigmoid(z) + bias).unique().numel() == 1
    assert sk.route_experts(z, 4, scores="sigmoid", bias=bias).experts.tolist() == [[1, 3, 0, 2]]
    assert sk.route_experts(z, 2, scores="sigmoid", bias=bias, groups=2, chosen_groups=1).experts.tolist() == [[1, 0]]


@pytest.mark.gpu
@pytest.mark.parametrize("scores", ["softmax", "sigmoid"])
def test_special_values(sk, scores):
    inf, nan = math.inf, math.nan
    z = torch.tensor([[-inf, -inf, -inf, -inf], [nan, 1, nan, -inf], [inf, 0, inf, 1], [-800, -801, -900, -700], [800, 801, 900, 700],
                      [3e38, -3e38, 0, -inf], [-0.0, 0.0, -0.0, 0.0], [1e-45, 0, -1e-45, nan]], device="cuda")
    for bias in (None, torch.tensor([0.1, -0.1, 0.0, 0.2], device="cuda"), torch.tensor([-inf, 0.0, nan, 0.0], device="cuda")):
        for renormalize in (True, False):
            how = dict(scores=scores, bias=bias, renormalize=renormalize, scale=2.0)
            assert_route(sk.route_experts(z, 3, **how), plain_route(z, 3, **how))
            how.update(groups=2, chosen_groups=1)
            assert_route(sk.route_experts(z, 2, **how), plain_route(z, 2, **how))


@pytest.mark.gpu
def test_without_options_it_is_the_plain_route(sk):
    z = logits_of(300, 48, 3, closed=0.2)
    plain = sk.route_experts(z, 4)
    same = sk.route_experts(z, 4, scores="softmax", groups=4, chosen_groups=4)   # (all groups open, by the kernel with scores)
    for a, b in zip(plain[1:], same[1:]):
        assert torch.equal(a, b)
    # (the plain route's quotients of exponentials in 32 bits: a few units)
    assert torch.allclose(plain.weights, same.weights, rtol=1e-6, atol=0)


def plain_gradient(z, experts, dw, scores, renormalize, scale):
    """by the definition's derivative, through autograd in 64 bits"""
    z = z.detach().double().cpu().requires_grad_()
    experts = experts.cpu().long()
    there = experts >= 0
    total = torch.zeros((), dtype=torch.float64)
    for t in range(z.shape[0]):
        chosen = experts[t][there[t]]
        if len(chosen) == 0:
            continue
        s = torch.sigmoid(z[t]) if scores == "sigmoid" else torch.softmax(z[t][z[t] > -math.inf], 0)
        if scores == "softmax":   # (back to the experts' places)
            s = torch.zeros_like(z[t]).index_put((torch.nonzero(z[t] > -math.inf)[:, 0],), s)
        w = s[chosen]
        if renormalize:
            w = w / w.sum()
        total = total + (scale * w * dw[t][there[t]].double().cpu()).sum()
    if not total.requires_grad:
        return torch.zeros_like(z)
    return torch.nan_to_num(torch.autograd.grad(total, z)[0], nan=0.0)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("scores", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renormalize", [True, False])
@pytest.mark.parametrize("T,E,k,groups,chosen_groups", [(5, 4, 2, 1, 1), (70, 300, 7, 6, 2), (1, 64, 64, 1, 1), (100, 96, 8, 8, 4), (3, 1000, 5, 1, 1)])
def test_gradient(sk, dtype, scores, renormalize, T, E, k, groups, chosen_groups):
    z = logits_of(T, E, T + 3 * E, TYPES[dtype], closed=0.2).requires_grad_()
    bias = bias_of(E, 5)
    dw = torch.randn(T, k, generator=torch.Generator().manual_seed(2)).cuda()
    route = sk.route_experts(z, k, scores=scores, bias=bias, groups=groups, chosen_groups=chosen_groups, renormalize=renormalize, scale=2.5)
    got, = torch.autograd.grad(route.weights, z, dw)
    assert got.dtype == z.dtype and got.shape == z.shape
    want = plain_gradient(z, route.experts, dw, scores, renormalize, 2.5)
    tol = (torch.finfo(z.dtype).eps / 2 + 2.0 ** -23) * want.abs() + 1e-13 * (1 + 2.5 * dw.abs().sum(1, keepdim=True).double().cpu()) + SMALLEST[z.dtype]
    assert ((got.double().cpu() - want).abs() <= tol).all()


@pytest.mark.gpu
@pytest.mark.parametrize("scores,renormalize", [("softmax", False), ("sigmoid", True), ("sigmoid", False)])
def test_gradient_against_differences(sk, scores, renormalize):
    T, E, k = 4, 12, 3
    z = logits_of(T, E, 11)
    dw = torch.randn(T, k, generator=torch.Generator().manual_seed(4)).cuda()
    how = dict(scores=scores, renormalize=renormalize)
    leaf = z.clone().requires_grad_()
    route = sk.route_experts(leaf, k, **how)
    got, = torch.autograd.grad(route.weights, leaf, dw)
    h = 2.0 ** -7
    for t in range(T):
        for e in range(E):
            step = torch.zeros_like(z)
            step[t, e] = h
            up, down = sk.route_experts(z + step, k, **how), sk.route_experts(z - step, k, **how)
            if not (torch.equal(up.experts, route.experts) and torch.equal(down.experts, route.experts)):
                continue   # (a choice changes: no derivative)
            diff = ((up.weights - down.weights).double() * dw.double()).sum().item() / (2 * h)
            # weights of up to 1 in float32 (2^-24, k of them, by 2 h), z + h rounded (2^-22 for |z| < 8), third derivatives (at most 1) h^2 / 6
            tol = dw.abs().sum().item() * (2 * 2.0 ** -24 / (2 * h) + 2.0 ** -22 / h + h * h / 6)
            assert abs(got[t, e].item() - diff) <= tol


@pytest.mark.gpu
def test_strided_logits_and_another_stream(sk):
    wide = logits_of(33, 64, 9)
    z, bias = wide[:, 3:43], bias_of(40, 1)
    how = dict(scores="sigmoid", bias=bias, groups=4, chosen_groups=2)
    want = plain_route(z, 4, **how)
    assert_route(sk.route_experts(z, 4, **how), want)
    assert_route(sk.route_experts(z.t().contiguous().t(), 4, **how), want)
    assert_route(sk.route_experts(z[:1].expand(33, 40), 4, **how), plain_route(z[:1].expand(33, 40), 4, **how))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        route = sk.route_experts(z, 4, **how)
    side.synchronize()
    assert_route(route, want)
    empty = sk.route_experts(wide[:0], 4, scores="sigmoid", renormalize=False)
    assert empty.weights.shape == (0, 4) and empty.offsets.tolist() == [0] * 65
    leaf = wide[:0].clone().requires_grad_()
    grad, = torch.autograd.grad(sk.route_experts(leaf, 4, scores="sigmoid").weights.sum(), leaf)
    assert grad.shape == (0, 64)


@pytest.mark.gpu
@pytest.mark.parametrize("T", [16, 300])
def test_recorded_into_a_graph(sk, T):
    z, bias = logits_of(T, 64, 21).requires_grad_(), bias_of(64, 2)
    dw = torch.randn(T, 6, generator=torch.Generator().manual_seed(5)).cuda()
    how = dict(scores="sigmoid", bias=bias, groups=8, chosen_groups=4)

    def step():
        route = sk.route_experts(z, 6, **how)
        grad, = torch.autograd.grad(route.weights, z, dw)
        return type(route)(*(t.detach() for t in route)), grad   # (nothing keeps the graph of one step alive in the next)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        recorded, grad = step()
    for seed in (1, 2, 3):
        with torch.no_grad():
            z.copy_(logits_of(T, 64, seed))
            bias.copy_(bias_of(64, seed))
        graph.replay()
        torch.cuda.synchronize()
        route, d = step()
        for a, b in zip(recorded, route):
            assert torch.equal(a, b)
        assert torch.equal(grad, d)
        assert_route(route, plain_route(z, 6, **how))


@pytest.mark.gpu
def test_a_layer_step_with_balanced_experts(sk):
    """routing, dispatch, both products and the sum, forward and backward, against 64 bits on the same choice"""
    T, H, I, E, k = 50, 128, 64, 16, 4
    g = torch.Generator().manual_seed(0)
    x = torch.randn(T, H, generator=g).half().cuda().requires_grad_()
    router = (torch.randn(E, H, generator=g) / math.sqrt(H)).cuda().requires_grad_()
    up, down = ((torch.randn(s, generator=g) / 10).half().cuda().requires_grad_() for s in ((E, I, H), (E, H, I)))
    bias = bias_of(E, 3)
    route = sk.route_experts(x.float() @ router.t(), k, scores="sigmoid", bias=bias, groups=4, chosen_groups=2, scale=2.0)
    h = sk.streamk_grouped(sk.dispatch_rows(x, route), up, route.offsets)
    out = sk.combine_rows(sk.streamk_grouped(torch.relu(h), down, route.offsets), route)
    grads = torch.autograd.grad(out.float().square().sum(), (x, router, up, down))
    xd, rd, ud, dd = (t.detach().double().requires_grad_() for t in (x, router, up, down))
    experts = route.experts.long()
    s = torch.sigmoid(xd @ rd.t()).gather(1, experts)
    w = 2.0 * s / s.sum(1, keepdim=True)
    hidden = torch.relu(torch.matmul(ud[experts], xd[:, None, :, None]))
    want = (w[..., None] * torch.matmul(dd[experts], hidden)[..., 0]).sum(1)
    # six roundings to fp16 on the way forward, and as many back: 12 2^-11 of norms that the random signs do not let cancel, twice
    assert (out.double() - want).norm() <= 12 * 2.0 ** -11 * want.norm()
    for got, ref in zip(grads, torch.autograd.grad(want.square().sum(), (xd, rd, ud, dd))):
        assert (got.double() - ref).norm() <= 24 * 2.0 ** -11 * ref.norm()


@pytest.mark.gpu
def test_wrong_operands_are_refused(sk):
    z = logits_of(4, 12, 1)
    good = dict(scores="sigmoid")
    for bad, kind in ((dict(scores="tanh"), ValueError), (dict(groups=5), ValueError), (dict(groups=0), ValueError), (dict(groups=4, chosen_groups=5), ValueError),
                      (dict(groups=4, chosen_groups=0), ValueError), (dict(groups=12, chosen_groups=3), ValueError), (dict(scale=math.inf), ValueError),
                      (dict(scale=math.nan), ValueError), (dict(bias=torch.zeros(11, device="cuda")), ValueError), (dict(bias=torch.zeros(12)), TypeError),
                      (dict(bias=torch.zeros(12, device="cuda", dtype=torch.float16)), TypeError), (dict(bias=torch.zeros(24, device="cuda")[::2]), ValueError)):
        with pytest.raises(kind):
            sk.route_experts(z, 4, **{**good, **bad})
    for k in (0, 13):
        with pytest.raises(ValueError):
            sk.route_experts(z, k, **good)
    with pytest.raises((TypeError, NotImplementedError)):
        sk.route_experts(z.cpu(), 4, **good)
    with pytest.raises(TypeError):
        sk.route_experts(z.double(), 4, **good)
    with pytest.raises(NotImplementedError), torch.autograd.forward_ad.dual_level():
        sk.route_experts(torch.autograd.forward_ad.make_dual(z, z), 4, **good)
    leaf = z.clone().requires_grad_()
    grad, = torch.autograd.grad(sk.route_experts(leaf, 4, **good).weights.square().sum(), leaf, create_graph=True)
    with pytest.raises(RuntimeError):
        grad.sum().backward()


def test_calls_are_refused_with_codes(sk):
    from streamk import _lib
    L, one = sk.lib(), ctypes.c_void_p(4096)   # (never read: every call here is refused)

    def call(bias=None, scale=1.0, scores=1, groups=1, chosen=1, E=12, k=4, dtype=_lib.SK_F32, ld=None, logits=one, out=one, back=False, none=False):
        by = _lib.SkRouteScores(bias=bias, scale=scale, scores=scores, renormalize=1, groups=groups, chosen_groups=chosen)
        ref = None if none else ctypes.byref(by)
        if back:
            return L.sk_route_scored_backward(logits, dtype, 4, E, k, E if ld is None else ld, ref, one, one, out, None)
        return L.sk_route_scored(logits, dtype, 4, E, k, E if ld is None else ld, ref, one, one, one, one, out, one, 1 << 30, None)
    for back in (False, True):
        for bad in (dict(scores=2), dict(scale=math.inf), dict(scale=math.nan), dict(dtype=99), dict(groups=0), dict(groups=5), dict(groups=65, E=65), dict(groups=4, chosen=5),
                    dict(groups=4, chosen=0), dict(groups=4, chosen=1), dict(k=0), dict(k=13), dict(E=0), dict(E=2000, k=4), dict(ld=11), dict(logits=None), dict(out=None),
                    dict(bias=4098), dict(none=True)):
            assert call(back=back, **bad) < 0, bad


def test_fake_implementations(sk):
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        z = torch.empty(5, 16, device="cuda", dtype=torch.bfloat16)
        out = torch.ops.streamk.route_scored(z, 3, None, "sigmoid", True, 4, 2, 1.0)
        assert [tuple(t.shape) for t in out] == [(5, 3), (5, 3), (17,), (15,), (5, 3)] and out[0].dtype == torch.float32
        assert torch.ops.streamk.route_scored_backward(z, out[1], out[0], "sigmoid", True, 4, 2, 1.0).shape == z.shape
