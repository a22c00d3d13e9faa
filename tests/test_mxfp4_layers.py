"""Layers on microscaled 4-bit products and on routing by scores: StreamKLinear and StreamKMoE with weight_format="mxfp4", StreamKMoE's
scores, balance bias and groups, and a run of all of it together."""
import math

import pytest
import torch

TYPES = {"float16": torch.float16, "bfloat16": torch.bfloat16}
# unit roundoff: half the distance from 1 to the next number
ROUNDOFF = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
ROUTED = dict(scores="sigmoid", balance=True, groups=4, chosen_groups=2, scale=2.5)


@pytest.fixture(scope="module")
def sk():
    import streamk

    return streamk


def silu(x):
    return x * torch.sigmoid(x)


def assert_product(got, pre, bias_magnitude, magnitudes, K, activation):
    """Exact terms, summed in fp32 (2 K 2^-24 of their magnitudes: the matrix instructions may cut), 4e-6 of the value in front of the
    activation and of one for bias and activation, one rounding."""
    want = silu(pre) if activation else pre
    tol = ROUNDOFF[got.dtype] * want.abs() * 1.001 + 1.13 * 2.4 * K * 2.0 ** -24 * magnitudes + 4e-6 * (pre.abs() + 1) + 2.0 ** -24 + 2.0 ** -22 * bias_magnitude
    off = (got.double() - want).abs()
    assert (off <= tol).all(), f"largest excess {(off - tol).max().item():.3g}"


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["float16", "bfloat16", "float32"])
@pytest.mark.parametrize("rows,N,K", [((1,), 256, 512), ((3, 5), 100, 64), ((300,), 520, 1056), ((2, 0), 32, 32)])
def test_linear(sk, kind, rows, N, K):
    torch.manual_seed(N)
    linear = torch.nn.Linear(K, N, device="cuda", dtype=getattr(torch, kind))
    layer = sk.StreamKLinear.from_linear(linear, weight_format="mxfp4", activation="silu")
    assert layer.dtype == (torch.bfloat16 if kind == "bfloat16" else torch.float16)
    x = torch.randn(*rows, K, device="cuda").to(layer.dtype)
    got = layer(x)
    assert got.shape == (*rows, N) and got.dtype == x.dtype and not got.requires_grad
    if not got.numel():
        return
    w = sk.dequantize_mxfp4(layer.qweight, layer.weight_scale, torch.float32).double()
    assert torch.equal(w, sk.dequantize_mxfp4(*sk.quantize_mxfp4(linear.weight.detach()), torch.float32).double())
    a = sk.dequantize_mxfp4(*sk.quantize_mxfp4(x), torch.float32).double()
    bias = layer.bias.double()
    assert_product(got, a @ w.T + bias, bias.abs(), a.abs() @ w.abs().T, K, True)
    # state dict and back
    other = sk.StreamKLinear(K, N, bias=True, weight_format="mxfp4", activation="silu", dtype=layer.dtype, device="cuda")
    other.load_state_dict(layer.state_dict())
    assert torch.equal(other(x), got)


def plain_rows(sk, q, scale):
    return sk.dequantize_mxfp4(q, scale, torch.float32).double()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("size", [(1, 64, 96, 4, 2), (130, 288, 544, 8, 3), (33, 128, 256, 64, 6), (2100, 256, 128, 16, 2)])
@pytest.mark.parametrize("routed", [False, True])
def test_a_run_together(sk, dtype, size, routed):
    """The layer is the run of its operators, bit for bit, and each product of the run is that of the values it was given."""
    T, hidden, intermediate, experts, chosen = size
    torch.manual_seed(T + hidden)
    big = sk.StreamKMoE(hidden, intermediate, experts, chosen, weight_format=dtype, device="cuda", **(ROUTED if routed else {}))
    if routed:
        big.router_bias.copy_(0.1 * torch.randn(experts, device="cuda"))
    layer = sk.StreamKMoE.quantized(big, "mxfp4")
    x = torch.randn(T, hidden, device="cuda").to(TYPES[dtype])
    x[T // 2, 3] = math.nan if T > 1 else 0.0   # (that token goes to no expert)
    got = layer(x)
    everyone = torch.tensor([0, T], dtype=torch.int32, device="cuda")
    logits = sk.streamk_grouped(x, layer.router[None], everyone)
    route = sk.route_experts(logits, chosen, bias=layer.router_bias, **layer.routing)
    q, scale = sk.quantize_mxfp4(x)
    rows, row_scales = sk.dispatch_rows(q, route), sk.dispatch_rows(scale, route)
    h = sk.streamk_grouped(rows, layer.up, route.offsets, scale_a=row_scales, scale_b=layer.up_scale, out_dtype=x.dtype, activation="silu")
    hq, hs = sk.quantize_mxfp4(h)
    y = sk.streamk_grouped(hq, layer.down, route.offsets, scale_a=hs, scale_b=layer.down_scale, out_dtype=x.dtype)
    assert torch.equal(got, sk.combine_rows(y, route)) and torch.isfinite(got).all()
    if T > 1:
        assert not got[T // 2].any() and (route.experts[T // 2] == -1).all()
    ends = route.offsets.tolist()
    for e in range(experts):
        r = slice(ends[e], ends[e + 1])
        a, w = plain_rows(sk, rows[r], row_scales[r]), plain_rows(sk, layer.up[e], layer.up_scale[e])
        assert_product(h[r], a @ w.T, 0.0, a.abs() @ w.abs().T, hidden, True)
        a, w = plain_rows(sk, hq[r], hs[r]), plain_rows(sk, layer.down[e], layer.down_scale[e])
        assert_product(y[r], a @ w.T, 0.0, a.abs() @ w.abs().T, intermediate, False)
    assert not h[ends[-1]:].any() and not y[ends[-1]:].any()
    # the sums, in 64 bits: k fp32 steps and a rounding
    used = route.place >= 0
    terms = torch.where(used, route.weights, 0.0).double()[..., None] * y[route.place.clamp(min=0).long()].double() * used[..., None]
    assert ((got.double() - terms.sum(1)).abs() <= 1.001 * ROUNDOFF[x.dtype] * terms.sum(1).abs() + chosen * 2.0 ** -23 * terms.abs().sum(1) + 2.0 ** -24).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", sorted(TYPES))
def test_near_the_layer_in_16_bits(sk, dtype):
    """A code's step is half of the power of two below the value, so an even error in it a 0.14th of that power, 10 % of the value; values
    above six eighths of the block's largest power lose up to a quarter.  12 % for each of four operands, 24 % together; half as much again."""
    torch.manual_seed(1)
    layer = sk.StreamKMoE(512, 1024, 8, 2, weight_format=dtype, device="cuda")
    x = torch.randn(300, 512, device="cuda").to(TYPES[dtype])
    with torch.no_grad():
        got, want = sk.StreamKMoE.quantized(layer, "mxfp4")(x).double(), layer(x).double()
    assert ((got - want).norm() / want.norm()).item() <= 0.36


@pytest.mark.gpu
def test_in_a_graph(sk):
    torch.manual_seed(3)
    layer = sk.StreamKMoE.quantized(sk.StreamKMoE(128, 256, 8, 2, weight_format="bfloat16", device="cuda", **ROUTED), "mxfp4")
    linear = sk.StreamKLinear.from_linear(torch.nn.Linear(128, 128, device="cuda", dtype=torch.bfloat16), weight_format="mxfp4")
    x = torch.randn(40, 128, device="cuda").bfloat16()
    step = lambda: linear(layer(x))  # noqa: E731
    stream, graphs, outs = torch.cuda.Stream(), [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()], []
    with torch.no_grad(), torch.cuda.stream(stream):
        step()
        stream.synchronize()
        for g in graphs:
            with torch.cuda.graph(g, stream=stream):
                outs.append(step())
    for seed in range(4):   # (other tokens, other experts; two graphs, one after the other)
        torch.manual_seed(seed)
        x.copy_(torch.randn(x.shape, device="cuda"))
        layer.router_bias.copy_(torch.randn(8, device="cuda"))
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        with torch.no_grad():
            want = step()
        assert torch.equal(outs[0], want) and torch.equal(outs[1], want)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", sorted(TYPES))
def test_routing_by_scores_trains(sk, dtype):
    """The layer's gradients against those of its formula in 64 bits for the experts that were chosen: roundings as in the layer without
    scores, five of them on the way of each gradient; 8 and 16 unit roundoffs of the norms."""
    T, hidden, intermediate, experts, chosen = 60, 128, 96, 16, 3
    torch.manual_seed(5)
    layer = sk.StreamKMoE(hidden, intermediate, experts, chosen, weight_format=dtype, device="cuda", **ROUTED)
    layer.router_bias.copy_(0.3 * torch.randn(experts, device="cuda"))
    x = torch.randn(T, hidden, device="cuda").to(TYPES[dtype]).requires_grad_()
    g = torch.randn(T, hidden, device="cuda").to(TYPES[dtype])
    out = layer(x)
    out.backward(g)
    with torch.no_grad():
        route = layer.route(x)
    X, R, U, D = (t.detach().double().requires_grad_() for t in (x, layer.router, layer.up, layer.down))
    s = torch.sigmoid(X @ R.T).gather(1, route.experts.long())
    w = 2.5 * s / s.sum(1, keepdim=True)
    want = 0
    for j in range(chosen):
        e = route.experts[:, j].long()
        h = silu(torch.matmul(U[e], X[:, :, None])[..., 0])
        want = want + w[:, j:j + 1] * torch.matmul(D[e], h[:, :, None])[..., 0]
    want.backward(g.double())
    u = ROUNDOFF[TYPES[dtype]]
    assert ((out.double() - want).norm() / want.norm()).item() <= 8 * u
    for a, b in ((x, X), (layer.router, R), (layer.up, U), (layer.down, D)):
        assert ((a.grad.double() - b.grad).norm() / b.grad.norm()).item() <= 16 * u
    # a layer that is cast: the bias has been rounded, and is used
    with torch.no_grad():
        assert layer.to(TYPES[dtype]).route(x).experts.shape == (T, chosen) and layer.router_bias.dtype == TYPES[dtype]
    # a closed expert is not chosen
    layer.router_bias[3] = -math.inf
    with torch.no_grad():
        assert not (layer.route(x).experts == 3).any()


@pytest.mark.gpu
def test_without_tokens(sk):
    layer = sk.StreamKMoE(64, 64, 4, 2, weight_format="mxfp4", device="cuda")
    assert layer(torch.zeros(3, 0, 64, dtype=torch.float16, device="cuda")).shape == (3, 0, 64)
    assert not list(layer.parameters()) and layer.router_bias is None


def test_refusals(sk):
    for kw in (dict(in_features=48), dict(dtype=torch.float32)):
        with pytest.raises(ValueError):
            sk.StreamKLinear(**{**dict(in_features=64, out_features=8, weight_format="mxfp4"), **kw})
    layer = sk.StreamKLinear(64, 8, weight_format="mxfp4")
    for x in (torch.zeros(2, 64, dtype=torch.bfloat16), torch.zeros(2, 32, dtype=torch.float16)):
        with pytest.raises(ValueError):
            layer(x)
    with pytest.raises(ValueError):
        layer.plan_for(4)
    for args, kw in (((48, 64, 4, 2), dict(weight_format="mxfp4")), ((64, 48, 4, 2), dict(weight_format="mxfp4")), ((64, 64, 4, 2), dict(weight_format="mxfp4", dtype=torch.float32)),
                     ((64, 64, 4, 2), dict(scores="tanh")), ((64, 64, 8, 2), dict(groups=3)), ((64, 64, 8, 2), dict(groups=4, chosen_groups=5)),
                     ((64, 64, 8, 5), dict(groups=4, chosen_groups=2)), ((64, 64, 8, 2), dict(scale=math.inf)), ((64, 64, 8, 2), dict(groups=0))):
        with pytest.raises(ValueError):
            sk.StreamKMoE(*args, **kw)
    with pytest.raises(ValueError):
        sk.StreamKMoE.quantized(sk.StreamKMoE(64, 64, 4, 2), "q4")
    with pytest.raises(ValueError):
        sk.StreamKMoE.quantized(sk.StreamKMoE(64, 64, 4, 2, weight_format="int8"), "mxfp4")
    assert "scores=sigmoid" in repr(sk.StreamKMoE(64, 64, 4, 2, scores="sigmoid"))


@pytest.mark.parametrize("dtype", sorted(TYPES))
def test_the_balance_bias_of_a_layer_that_is_cast(sk, dtype):
    """A cast that rounds the bias says so; the rule in float32 arrives, to a unit roundoff, where steps added in 16 bits would not."""
    import warnings
    layer = sk.StreamKMoE(64, 64, 8, 2, weight_format=dtype, **ROUTED)
    bias = torch.linspace(-1, 1, 8)
    layer.router_bias.copy_(bias)
    with warnings.catch_warnings():
        warnings.simplefilter("error")
        layer.to("cpu")
        layer.float()
    assert torch.equal(layer.router_bias, bias)
    with pytest.warns(UserWarning, match="router_bias"):
        torch.nn.Sequential(layer).to(TYPES[dtype])
    with warnings.catch_warnings():
        warnings.simplefilter("error")
        layer.to(TYPES[dtype])
        sk.StreamKMoE(64, 64, 8, 2, weight_format=dtype).to(TYPES[dtype])   # (none to lose)
    alone = layer.router_bias.clone()
    for _ in range(1000):
        bias += 0.001
        alone += 0.001
        layer.router_bias.copy_(bias)
    want = torch.linspace(-1, 1, 8) + 1
    # (1000 float32 sums, and 0.001 in float32)
    assert ((layer.router_bias.double() - want.double()).abs() <= ROUNDOFF[TYPES[dtype]] * want.double() * 1.001 + 1000 * 2.0 ** -23).all()
    if dtype == "bfloat16":
        assert alone[-1] == 1   # 0.001 is less than half of the 2^-7 from 1 on
    layer.router_bias = layer.router_bias.float()
    assert layer.router_bias.dtype == torch.float32 and "router_bias" in layer.state_dict()
