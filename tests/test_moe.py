"""Layers that run the operators for experts and int8 together: StreamKMoE and StreamKLinear(weight_format="int8")."""
import math

import pytest
import torch

TYPES = {"float16": torch.float16, "bfloat16": torch.bfloat16}
# unit roundoff: half the distance from 1 to the next number
ROUNDOFF = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


@pytest.fixture(scope="module")
def sk():
    import streamk

    return streamk


def off(got, want):
    """Norm of the error relative to the norm of the result."""
    return ((got.double() - want.double()).norm() / want.double().norm()).item()


def plain(layer, x, route):
    """The layer's formula in float64 on the weights it holds, for the experts that were chosen; differentiable."""
    act = {"relu": torch.relu, "gelu_tanh": lambda z: torch.nn.functional.gelu(z, approximate="tanh"), "silu": torch.nn.functional.silu}[layer.activation]
    x, router, up, down = (t.detach().double().requires_grad_() for t in (x, layer.router, layer.up, layer.down))
    logits = x @ router.T
    weights = torch.softmax(logits.gather(1, route.experts.long()), 1)
    out = 0
    for j in range(layer.chosen):
        chosen = route.experts[:, j].long()
        y = torch.zeros_like(x)
        for e in range(layer.experts):
            rows = (chosen == e).nonzero()[:, 0]
            y = y.index_put((rows,), act(x[rows] @ up[e].T) @ down[e].T)
        out = out + weights[:, j:j + 1] * y
    return out, (x, router, up, down)


def make(sk, T, hidden, intermediate, experts, chosen, dtype, activation):
    torch.manual_seed(T + hidden)
    layer = sk.StreamKMoE(hidden, intermediate, experts, chosen, activation=activation, weight_format=dtype, device="cuda")
    return layer, torch.randn(T, hidden, device="cuda").to(TYPES[dtype])


SIZES = [(1, 64, 96, 4, 2), (7, 72, 40, 3, 3), (130, 264, 520, 8, 2), (33, 128, 256, 70, 6)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("activation", ["relu", "gelu_tanh", "silu"])
@pytest.mark.parametrize("size", SIZES)
def test_experts_layer(sk, dtype, activation, size):
    """Four roundings (hidden row, expert's row, sum; logits, whose rounding moves a weight by at most |z| u) of relative size u each, the
    first through the second product: together below 8 u of the result's norm."""
    layer, x = make(sk, *size, dtype, activation)
    with torch.no_grad():
        got = layer(x)
        want, _ = plain(layer, x, layer.route(x))
    assert got.dtype == x.dtype and got.shape == x.shape
    assert off(got, want) <= 8 * ROUNDOFF[x.dtype]
    assert torch.equal(layer(x.view(1, *x.shape))[0].detach(), layer(x).detach())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("size", SIZES)
def test_experts_layer_trains(sk, dtype, size):
    """The gradients of x, the router and both weights.  A gradient passes at most eight rounded tensors (the forward's four again, those
    of the activation, both products and the dispatch on the way back): 16 u.  The router's is a difference of sums over the
    experts' rows that nearly cancel: where it is small against them it is compared on their scale."""
    layer, x = make(sk, *size, dtype, "silu")
    x.requires_grad_()
    out = layer(x)
    with torch.no_grad():
        route = layer.route(x)
    want, leaves = plain(layer, x, route)
    d_out = torch.randn(out.shape, device="cuda").to(out.dtype)
    grads = torch.autograd.grad(out, (x, layer.router, layer.up, layer.down), d_out)
    wanted = torch.autograd.grad(want, leaves, d_out.double())
    u = ROUNDOFF[x.dtype]
    for name, g, w in zip(("x", "router", "up", "down"), grads, wanted):
        if name == "router":
            # of a token and an expert: |dweight| <= |d_out| |y|; y's and the logits' roundings move it by 8 u of that
            scale = (d_out.double().norm(dim=1) * want.detach().norm(dim=1) * x.detach().double().norm(dim=1)).norm().item() * math.sqrt(layer.chosen)
            assert (g.double() - w).norm().item() <= 16 * u * max(w.norm().item(), scale)
        else:
            assert off(g, w) <= 16 * u, name


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("size", [(1, 64, 96, 4, 2), (130, 272, 528, 8, 2), (33, 128, 256, 70, 6)])
def test_experts_layer_in_int8(sk, dtype, size):
    """Rounding to 127 steps of a row's largest value errs by max / (127 sqrt 12) a value: with max / rms of 3 to 4 for the inputs and
    weights and 6 for hidden rows 0.7 to 1.4 % of each operand's norm, below 2.5 % for the four together.  Twice that."""
    layer, x = make(sk, *size, dtype, "silu")
    small = sk.StreamKMoE.quantized(layer)
    with torch.no_grad():
        got, want = small(x), layer(x)
        assert torch.equal(small.route(x).experts, layer.route(x).experts)
    assert got.dtype == x.dtype and off(got, want) <= 0.05
    assert not list(small.parameters())
    assert not small(x.clone().requires_grad_()).requires_grad


@pytest.mark.gpu
@pytest.mark.parametrize("weight_format", ["float16", "int8"])
def test_experts_layer_in_a_graph(sk, weight_format):
    layer, x = make(sk, 24, 128, 256, 8, 2, "float16", "silu")
    if weight_format == "int8":
        layer = sk.StreamKMoE.quantized(layer)
    stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.no_grad(), torch.cuda.stream(stream):
        layer(x)
        stream.synchronize()
        with torch.cuda.graph(graph, stream=stream):
            out = layer(x)
    for seed in range(4):   # (other tokens, other experts)
        torch.manual_seed(seed)
        x.copy_(torch.randn(x.shape, device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        with torch.no_grad():
            assert torch.equal(out, layer(x))


@pytest.mark.gpu
def test_experts_layer_without_tokens(sk):
    for fmt in ("float16", "int8"):
        layer = sk.StreamKMoE(64, 64, 4, 2, weight_format=fmt, device="cuda")
        assert layer(torch.zeros(3, 0, 64, dtype=torch.float16, device="cuda")).shape == (3, 0, 64)


def test_experts_layer_refusals(sk):
    for args, kw in (((64, 64, 4, 5), {}), ((64, 64, 1025, 1), {}), ((64, 64, 100, 65), {}), ((64, 64, 4, 0), {}), ((60, 64, 4, 2), {}), ((72, 64, 4, 2), dict(weight_format="int8")), ((64, 64, 4, 2), dict(activation="tanh")),
                     ((64, 64, 4, 2), dict(weight_format="q4")), ((64, 64, 4, 2), dict(dtype=torch.float16)), ((64, 64, 4, 2), dict(weight_format="int8", dtype=torch.float32))):
        with pytest.raises(ValueError):
            sk.StreamKMoE(*args, **kw)
    layer = sk.StreamKMoE(64, 64, 4, 2)
    for x in (torch.zeros(2, 64), torch.zeros(2, 32, dtype=torch.bfloat16)):
        with pytest.raises(ValueError):
            layer(x)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("rows,N,K", [((1,), 256, 512), ((3, 5), 100, 64), ((300,), 520, 1040), ((2, 0), 32, 32)])
def test_linear_in_int8(sk, dtype, rows, N, K):
    """Against the formula on the values that were quantised, in float64: one rounding to the result's type, and three in fp32 (scales,
    product, sum).  Against the layer in 16 bits: see the experts' layer, two operands."""
    torch.manual_seed(N)
    linear = torch.nn.Linear(K, N, device="cuda", dtype=TYPES[dtype])
    layer = sk.StreamKLinear.from_linear(linear, weight_format="int8", activation="silu")
    assert layer.dtype == TYPES[dtype]
    x = torch.randn(*rows, K, device="cuda").to(TYPES[dtype])
    got = layer(x)
    assert got.shape == (*rows, N) and got.dtype == x.dtype
    if not got.numel():
        return
    q, scale = sk.quantize_int8(x)
    pre = (q.double() @ layer.qweight.double().T) * scale.double()[..., None] * layer.weight_scale.double() + layer.bias.double()
    want = torch.nn.functional.silu(pre)
    u = ROUNDOFF[x.dtype]
    magnitude = pre.abs() + 2 * layer.bias.double().abs()
    assert ((got.double() - want).abs() <= 1.01 * u * want.abs() + 8 * 2.0 ** -24 * magnitude + 2.0 ** -24).all()
    with torch.no_grad():
        assert off(got, torch.nn.functional.silu(linear(x).float())) <= 0.05


def test_linear_in_int8_refusals(sk):
    for args, kw in (((24, 8), {}), ((32, 8), dict(dtype=torch.float32))):
        with pytest.raises(ValueError):
            sk.StreamKLinear(*args, weight_format="int8", **kw)
    with pytest.raises(ValueError):
        sk.StreamKLinear(32, 8, dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        sk.StreamKLinear(32, 8, weight_format="int8")(torch.zeros(2, 32, dtype=torch.bfloat16))
