"""Microscaled 4-bit products and the routers of balanced experts, as cases to time: inputs, one pass, what it has to cost.

Three kinds of case:
  "route"    the experts of each token from softmax or sigmoid scores with a bias for balance, by groups of experts, the weights
             renormalised or not; in training the gradient of the logits too
  "product"  a linear layer on 4-bit floating point: rows of x in 16 bits are quantised (two e2m1 values to a byte, a power of two for
             each 32) and multiplied by weights that were quantised before; with several experts the rows are sorted by expert and each
             expert has its own weights
  "weights"  what becomes of weights: quantised, and the values that they then stand for
`own` false: plain torch in 32 bits (scores of a router in 64, which decide between neighbours), rounded once.  `own` true: the package's
entry points.
"""
import math
import os
import random
import sys

import torch

own = False

_TYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}


def _package():
    path = os.path.join(os.getcwd(), "stream-k.tvm_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import streamk
    return streamk


# ---- cases ----
def _route(name, T, E, k, **more):
    return dict(dict(name=name, kind="route", dtype="float32", T=T, E=E, k=k, scores="sigmoid", bias=True, groups=1, chosen_groups=1, renormalize=True,
                     scale=1.0, masked=False, backward=False), **more)


def _product(name, dtype, E, M, N, K, **more):
    return dict(dict(name=name, kind="product", dtype=dtype, E=E, M=M, N=N, K=K, skew=0.0, bias=False, activation="none"), **more)


def listed():
    return [
        # sixteen sequences decoding, eight of 256 experts out of four of eight groups: latency
        _route("route_16tokens", 16, 256, 8, groups=8, chosen_groups=4, scale=2.5),
        # the same router on a training batch with padding tokens and closed experts
        _route("route_8192tokens", 8192, 256, 8, groups=8, chosen_groups=4, scale=2.5, masked=True, backward=True),
        # softmax scores that stay as they are: every logit of a token has a gradient
        _route("route_4096tokens_softmax", 4096, 64, 6, dtype="bfloat16", scores="softmax", bias=False, renormalize=False, backward=True),
        # one token through a square layer: launches and host latency, then 9 MB of weights
        _product("product_1row", "bfloat16", 0, 1, 4096, 4096),
        # a short prompt through an MLP's first projection, bias and activation fused
        _product("product_100rows", "float16", 0, 100, 11008, 4096, bias=True, activation="silu"),
        # odd sizes: rows, columns and a K that is no power of two
        _product("product_777rows", "bfloat16", 0, 777, 2001, 4128, bias=True),
        # a batch of prompts: matrix-bound
        _product("product_4096rows", "bfloat16", 0, 4096, 8192, 8192),
        # one token, two of eight experts: the weights of two experts are all there is to read
        _product("experts_1token", "bfloat16", 8, 2, 11008, 4096),
        # 64 sequences decoding, two experts each: about sixteen rows an expert, all experts' weights
        _product("experts_64tokens", "float16", 8, 128, 11008, 4096, skew=0.5, activation="silu"),
        # a prompt of 4096 tokens, two of eight large experts: matrix-bound
        _product("experts_8192rows", "bfloat16", 8, 8192, 11008, 4096, skew=0.3),
        # a small layer's weights, odd
        dict(name="weights_1000rows", kind="weights", dtype="float16", N=1000, K=1056),
        # a large layer's weights: memory-bound
        dict(name="weights_28672rows", kind="weights", dtype="bfloat16", N=28672, K=8192),
    ]


def _log_int(rng, lo, hi, step=1):
    """An integer from lo to hi, spread evenly over its logarithm, a multiple of `step`."""
    v = math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))
    return max(step, min(hi // step * step, int(round(v / step)) * step))


_MOST = 8192 * 11008 * 4096        # multiply-adds of the largest listed product
_MOST_WEIGHTS = 8 * 11008 * 4096   # and its weights


def draw(rng):
    case = _draw(rng)
    case.pop("name", None)
    return case


def _draw(rng):
    kind = rng.choice(["route", "route", "product", "product", "experts", "experts", "weights"])
    if kind == "route":
        groups = rng.choice([1, 1, 2, 4, 8])
        E = groups * _log_int(rng, max(2, 8 // groups), 256 // groups)
        chosen_groups = rng.randint(1, groups)
        k = min(chosen_groups * (E // groups), _log_int(rng, 1, 16))
        bias = rng.random() < 0.6
        # (sums of two scores with different biases may tie in one rounding of 64 bits and not in another: logits of many digits do not)
        dtype = "float32" if bias and groups > 1 else rng.choice(["float32", "bfloat16", "float16"])
        return _route(None, _log_int(rng, 1, 8192), E, k, dtype=dtype, scores=rng.choice(["softmax", "sigmoid"]), bias=bias, groups=groups,
                      chosen_groups=chosen_groups, renormalize=rng.random() < 0.6, scale=rng.choice([1.0, 2.5]), masked=rng.random() < 0.4,
                      backward=rng.random() < 0.5)
    dtype = rng.choice(["float16", "bfloat16"])
    if kind == "weights":
        K = _log_int(rng, 32, 16384, 32)
        return dict(kind=kind, dtype=dtype, N=_log_int(rng, 1, min(65536, 28672 * 8192 // K)), K=K)
    K = _log_int(rng, 256, 16384, 32)
    E = 0 if kind == "product" else _log_int(rng, 1, 64)
    N = _log_int(rng, 256, max(256, min(28672, _MOST_WEIGHTS // (max(E, 1) * K))), 1 if rng.random() < 0.3 else 8)
    M = _log_int(rng, 1, min(16384, max(1, _MOST // (N * K))))
    return _product(None, dtype, E, M, N, K, skew=rng.choice([0.0, 0.3, 0.5, 1.0]) if E else 0.0, bias=rng.random() < 0.4,
                    activation=rng.choice(["none", "none", "relu", "gelu_tanh", "silu"]))


# ---- inputs ----
def _sizes(case, seed):
    """Rows of each expert: every row goes to an expert on its own, the experts' shares spread log-normally by `skew`."""
    rng = random.Random(seed * 1000003 + case["E"])
    shares = [math.exp(case["skew"] * rng.gauss(0, 1)) for _ in range(case["E"])]
    sizes = [0] * case["E"]
    for e in rng.choices(range(case["E"]), weights=shares, k=case["M"]):
        sizes[e] += 1
    return sizes


def _normal(gen, shape, std, dtype):
    return torch.randn(shape, generator=gen, device="cuda", dtype=dtype).mul_(std)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = _TYPES[case["dtype"]]
    if case["kind"] == "route":
        T, E = case["T"], case["E"]
        logits = torch.randn(T, E, generator=gen, device="cuda").mul_(2).to(dtype)
        if case["masked"]:
            closed = torch.rand(T, E, generator=gen, device="cuda") < 0.3
            closed |= torch.rand(T, 1, generator=gen, device="cuda") < 0.125
            logits.masked_fill_(closed, -math.inf)
        s = dict(case=case, logits=logits, bias=None)
        if case["bias"]:   # (steps of a thousandth, as a rule that counts tokens leaves them)
            s["bias"] = torch.randn(E, generator=gen, device="cuda").mul_(50).round_().mul_(0.001)
        if case["backward"]:
            s["d_weights"] = torch.randn(T, case["k"], generator=gen, device="cuda")
            logits.requires_grad_()
        return s
    N, K = case["N"], case["K"]
    if case["kind"] == "weights":   # rows of very different sizes
        x = _normal(gen, (N, K), 1 / math.sqrt(K), dtype)
        return dict(case=case, x=x.mul_(torch.exp(torch.randn(N, 1, generator=gen, device="cuda")).to(dtype)))
    E, M = case["E"], case["M"]
    s = dict(case=case, x=_normal(gen, (M, K), 1.0, dtype))
    # weights as a quantiser leaves them: codes of every kind, scales within a few powers of two of each other
    shape = (E, N) if E else (N,)
    codes = torch.randint(0, 256, (*shape, K // 2), generator=gen, device="cuda", dtype=torch.uint8)
    exponent = torch.randint(0, 3, (*shape, K // 32), generator=gen, device="cuda", dtype=torch.uint8)
    s["w"], s["scale"] = codes, exponent.add_(127 - 2 - int(math.log2(K) / 2))
    s["bias"] = _normal(gen, shape, 0.5, dtype) if case["bias"] else None
    if E:
        s["sizes"] = _sizes(case, seed)
        starts = [0]
        for n in s["sizes"]:
            starts.append(starts[-1] + n)
        s["offsets"] = torch.tensor(starts, dtype=torch.int32, device="cuda")
    return s


# ---- one pass ----
def run(state):
    kind = state["case"]["kind"]
    if own:
        return {"route": _own_route, "product": _own_product, "weights": _own_weights}[kind](state)
    with torch.no_grad():
        return {"route": _plain_route, "product": _plain_product, "weights": _plain_weights}[kind](state)


def _own_route(s):
    streamk = _package()
    c = s["case"]
    r = streamk.route_experts(s["logits"], c["k"], scores=c["scores"], bias=s["bias"], groups=c["groups"], chosen_groups=c["chosen_groups"],
                              renormalize=c["renormalize"], scale=c["scale"])
    got = dict(weights=r.weights.detach(), experts=r.experts, offsets=r.offsets, order=r.order, place=r.place)
    if c["backward"]:
        got["d_logits"], = torch.autograd.grad(r.weights, s["logits"], s["d_weights"])
    return got


def _own_product(s):
    streamk = _package()
    c = s["case"]
    q, scale = streamk.quantize_mxfp4(s["x"])
    options = dict(out_dtype=s["x"].dtype, bias=s["bias"], activation=None if c["activation"] == "none" else c["activation"])
    if c["E"]:
        return streamk.streamk_grouped(q, s["w"], s["offsets"], scale_a=scale, scale_b=s["scale"], **options)
    return streamk.streamk_mxfp4(q, s["w"], scale, s["scale"], **options)


def _own_weights(s):
    streamk = _package()
    q, scale = streamk.quantize_mxfp4(s["x"])
    return streamk.dequantize_mxfp4(q, scale, s["x"].dtype)


def _plain_route(s):
    c, E, G = s["case"], s["case"]["E"], s["case"]["groups"]
    T, k = c["T"], c["k"]
    z = s["logits"].detach().double()
    there = z > -math.inf
    if c["scores"] == "sigmoid":
        score = 1 / (1 + torch.exp(-z))
    else:
        most = z.amax(1, keepdim=True).clamp(min=-1e30)
        e = torch.exp(z - most)
        score = e / e.sum(1, keepdim=True).clamp(min=1e-300)
    # what the choice goes by: with neither bias nor groups the logits, in whose order the scores are
    key = torch.where(there, score + s["bias"].double() if c["bias"] else score, -math.inf)
    if G > 1:
        best = torch.sort(key.view(T, G, E // G), dim=2, descending=True).values[:, :, :2]
        of_group = torch.where(best > -math.inf, best, 0).sum(2)
        of_group = torch.where(best[:, :, 0] > -math.inf, of_group, -math.inf)
        first = torch.sort(of_group, dim=1, descending=True, stable=True).indices[:, :c["chosen_groups"]]
        open_group = torch.zeros(T, G, dtype=torch.bool, device="cuda").scatter_(1, first, True)
        key = torch.where(open_group.repeat_interleave(E // G, 1), key, -math.inf)
    if not c["bias"]:
        key = torch.where(key > -math.inf, z, -math.inf)
    best, experts = torch.sort(key, dim=1, descending=True, stable=True)
    best, experts = best[:, :k], experts[:, :k]
    chosen = best > -math.inf
    w = torch.where(chosen, score.gather(1, experts), 0)
    share = w / w.sum(1, keepdim=True).clamp(min=1e-300) if c["renormalize"] else w
    weights = share * c["scale"]
    experts = torch.where(chosen, experts, -1)
    flat = torch.where(chosen, experts, E).view(-1)
    order = torch.sort(flat, stable=True).indices
    counts = (flat[:, None] == torch.arange(E, device="cuda")).sum(0)
    offsets = torch.cat([counts.new_zeros(1), counts.cumsum(0)])
    place = torch.empty_like(order)
    place[order] = torch.arange(T * k, device="cuda")
    used = torch.arange(T * k, device="cuda") < offsets[E]
    got = dict(weights=weights.float(), experts=experts.int(), offsets=offsets.int(), order=torch.where(used, order, -1).int(),
               place=torch.where(chosen, place.view(T, k), -1).int())
    if c["backward"]:
        g = torch.where(chosen, s["d_weights"].double(), 0) * c["scale"]
        if c["renormalize"]:   # of the shares, then of the scores: a share's own score times its derivative by the logit
            g = share * (g - (share * g).sum(1, keepdim=True))
            d = torch.zeros_like(z).scatter_add_(1, experts.clamp(min=0), g * (1 - w) if c["scores"] == "sigmoid" else g)
        elif c["scores"] == "sigmoid":
            d = torch.zeros_like(z).scatter_add_(1, experts.clamp(min=0), g * w * (1 - w))
        else:
            d = torch.zeros_like(z).scatter_add_(1, experts.clamp(min=0), g * w) - score * (g * w).sum(1, keepdim=True)
        got["d_logits"] = d.to(s["logits"].dtype)
    return got


def _plain_quantize(x):
    """The values that x stands for in 4 bits, as e2m1 numbers and the power of two of each 32."""
    blocks = x.float().view(*x.shape[:-1], -1, 32)
    exponent = ((blocks.abs().amax(-1, keepdim=True).view(torch.int32) >> 23) - 127 - 2).clamp(min=-127)   # floor(log2 max) - 2
    y = torch.ldexp(blocks, -exponent)
    size = y.abs()
    step = torch.where(size < 2, 0.5, torch.where(size < 4, 1.0, 2.0))
    return torch.sign(y) * (torch.round(size / step) * step).clamp(max=6), exponent


def _plain_values(codes, scale):
    """float32 values of packed codes (low half first) and biased exponents."""
    both = torch.stack([codes & 15, codes >> 4], -1).flatten(-2)
    e, m = (both >> 1) & 3, (both & 1).float()
    size = torch.where(e == 0, 0.5 * m, (1 + 0.5 * m) * torch.exp2(e.float() - 1))
    value = torch.where(both >= 8, -size, size)
    return (value.view(*scale.shape, 32) * torch.exp2(scale.float() - 127)[..., None]).flatten(-2)


def _activate(x, name):
    if name == "relu":
        return x.clamp(min=0)
    if name == "silu":
        return x / (1 + torch.exp(-x))
    if name == "gelu_tanh":
        return x * 0.5 * (1 + torch.tanh(math.sqrt(2 / math.pi) * (x + 0.044715 * x * x * x)))
    return x


def _plain_product(s):
    c = s["case"]
    q, exponent = _plain_quantize(s["x"])
    x = torch.ldexp(q, exponent).flatten(-2)
    if not c["E"]:
        y = x @ _plain_values(s["w"], s["scale"]).t()
        if c["bias"]:
            y = y + s["bias"].float()
        return _activate(y, c["activation"]).to(s["x"].dtype)
    y = torch.empty(c["M"], c["N"], dtype=s["x"].dtype, device="cuda")
    at = 0
    for e, n in enumerate(s["sizes"]):
        if n == 0:
            continue
        part = x[at:at + n] @ _plain_values(s["w"][e], s["scale"][e]).t()
        if c["bias"]:
            part = part + s["bias"][e].float()
        y[at:at + n] = _activate(part, c["activation"]).to(y.dtype)
        at += n
    return y


def _plain_weights(s):
    q, exponent = _plain_quantize(s["x"])
    return torch.ldexp(q, exponent).flatten(-2).to(s["x"].dtype)


# ---- what a pass cannot do without ----
def work(case):
    if case["kind"] == "route":
        T, E, k = case["T"], case["E"], case["k"]
        size = 4 if case["dtype"] == "float32" else 2
        b = size * T * E + 16 * T * k + 4 * (E + 1) + (4 * E if case["bias"] else 0)   # logits; weights, experts, order, place; offsets; bias
        f = 10.0 * T * E
        if case["backward"]:
            b += 12 * T * k + size * T * E   # weights, experts and their gradient; the logits' gradient
            if case["scores"] == "softmax" and not case["renormalize"]:
                b += size * T * E            # and the logits again
            f += 10.0 * T * E
        return {"bytes": int(b), "flops": f}
    N, K = case["N"], case["K"]
    if case["kind"] == "weights":
        # 16 bits in and out, half a byte and a 32nd written and read between them
        return {"bytes": int(N * K * (4 + 2 * (0.5 + 1 / 32))), "flops": 4.0 * N * K}
    E, M = case["E"], case["M"]
    touched = sum(sum(n > 0 for n in _sizes(case, seed)) for seed in range(8)) / 8 if E else 1   # experts that have a row, on the average
    row = K / 2 + K / 32
    b = 2 * M * K + 2 * M * row + touched * N * row + 2 * M * N + (2 * touched * N if case["bias"] else 0) + 4 * (E + 1 if E else 0)
    return {"bytes": int(b), "flops": 2.0 * M * N * K}


# ---- the definitions in 64 bits ----
_E2M1 = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return {"route": _exact_route, "product": _exact_product, "weights": _exact_weights}[case["kind"]](s)


def _exact_route(s):
    c = s["case"]
    T, E, k, G = c["T"], c["E"], c["k"], c["groups"]
    z = s["logits"].detach().double().cpu()
    if c["scores"] == "sigmoid":
        score = torch.sigmoid(z)
    else:
        score = torch.nan_to_num(torch.softmax(z, 1), nan=0.0)
    by = score + s["bias"].double().cpu() if c["bias"] else score.clone()
    by[torch.isneginf(z)] = -math.inf
    if G > 1:
        pair = by.view(T, G, E // G).topk(min(2, E // G), dim=2).values
        total = torch.where(torch.isneginf(pair), torch.zeros_like(pair), pair).sum(2).masked_fill(torch.isneginf(pair[:, :, 0]), -math.inf)
        rank = torch.argsort(torch.argsort(-total, dim=1, stable=True), dim=1)
        by = by.view(T, G, E // G).masked_fill((rank >= c["chosen_groups"])[:, :, None], -math.inf).view(T, E)
    if not c["bias"]:
        by = torch.where(torch.isneginf(by), by, z)
    index = torch.argsort(-by, dim=1, stable=True)[:, :k]
    chosen = ~torch.isneginf(by.gather(1, index))
    logits = z.clone().requires_grad_()
    with torch.enable_grad():
        if c["scores"] == "sigmoid":
            picked = torch.sigmoid(logits.gather(1, index))
        else:   # (a token without an expert: any row of numbers will do)
            some = torch.where(torch.isneginf(z).all(1, keepdim=True), torch.zeros_like(z), logits)
            picked = torch.softmax(some, 1).gather(1, index)
        picked = torch.where(chosen, picked, torch.zeros_like(picked))
        if c["renormalize"]:
            total = picked.sum(1, keepdim=True)
            picked = picked / torch.where(total > 0, total, torch.ones_like(total))
        weights = picked * c["scale"]
    experts = torch.where(chosen, index, torch.full_like(index, -1))
    slots = sorted((int(e), i) for i, e in enumerate(experts.view(-1).tolist()) if e >= 0)
    order, place = [-1] * (T * k), [-1] * (T * k)
    for p, (_, i) in enumerate(slots):
        order[p], place[i] = i, p
    offsets = [0] * (E + 1)
    for e, _ in slots:
        offsets[e + 1] += 1
    for e in range(E):
        offsets[e + 1] += offsets[e]
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    got = dict(weights=weights.detach().cuda(), experts=experts.int().cuda(), offsets=ints(offsets), order=ints(order), place=ints(place).view(T, k))
    if c["backward"]:
        d, = torch.autograd.grad(weights, logits, torch.where(chosen, s["d_weights"].double().cpu(), torch.zeros_like(picked)))
        got["d_logits"] = torch.nan_to_num(d, nan=0.0).cuda()
    return got


def _exact_quantize(x):
    blocks = x.double().view(*x.shape[:-1], x.shape[-1] // 32, 32)
    most = blocks.abs().amax(-1, keepdim=True)
    power = torch.exp2(torch.where(most > 0, torch.frexp(most).exponent - 3.0, -127.0).clamp(min=-127.0))
    table = torch.tensor(_E2M1, dtype=torch.float64, device=x.device)
    size = (blocks / power).abs().clamp(max=6.0)
    above = torch.searchsorted(table, size).clamp(max=7)       # the first value of the table that is not below
    below = (above - 1).clamp(min=0)
    up, down = table[above] - size, size - table[below]
    nearest = torch.where((up < down) | ((up == down) & (above % 2 == 0)), above, below)
    return (torch.copysign(table[nearest], blocks) * power).flatten(-2)


def _exact_values(codes, scale):
    signed = torch.tensor(_E2M1 + [-v for v in _E2M1], dtype=torch.float64, device=codes.device)
    values = signed[torch.stack([codes % 16, codes // 16], -1).long()].view(*scale.shape, 32)
    return (values * torch.pow(torch.full((), 2.0, dtype=torch.float64, device=codes.device), scale.double() - 127).unsqueeze(-1)).flatten(-2)


def _exact_act(x, name):
    return {"none": lambda v: v, "relu": torch.relu, "silu": lambda v: v * torch.sigmoid(v),
            "gelu_tanh": lambda v: 0.5 * v * (1 + torch.tanh(math.sqrt(2 / math.pi) * (v + 0.044715 * v ** 3)))}[name](x)


def _exact_product(s):
    c = s["case"]
    x = _exact_quantize(s["x"])
    y = torch.empty(c["M"], c["N"], dtype=torch.float64, device="cuda")
    at = 0
    for e, n in enumerate(s["sizes"] if c["E"] else [c["M"]]):
        if n == 0:
            continue
        w, scale, bias = (s["w"], s["scale"], s["bias"]) if not c["E"] else (s["w"][e], s["scale"][e], s["bias"][e] if c["bias"] else None)
        part = torch.mm(x[at:at + n], _exact_values(w, scale).t())
        y[at:at + n] = _exact_act(part + bias.double() if c["bias"] else part, c["activation"])
        at += n
    return y


def _exact_weights(s):
    return _exact_quantize(s["x"])
