"""The operators around a mixture-of-experts layer and its 8-bit form, as cases to time: inputs, one pass, what it has to cost.

Four kinds of case:
  "int8"      a linear layer with int8 weights: rows of x in 16 bits are quantised with a scale for each row (token) and multiplied by
              int8 weights with a scale for each row of theirs (output channel)
  "grouped"   rows sorted by expert times each expert's own weights, groups of any size; 16-bit types, or int8 with both scales
  "gradient"  the same product in training: the product, the gradient of the rows and the gradient of the weights
  "exchange"  what stands before and behind the products: the k experts of each token from the router's logits, the tokens' rows in
              the experts' order, and the experts' rows added up for each token with the router's weights; in training all gradients
`own` false: plain torch in 32 bits, rounded once.  `own` true: the package's entry points.
"""
import math
import os
import random
import sys

import torch

own = False

_TYPES = {"float16": torch.float16, "bfloat16": torch.bfloat16}


def _package():
    path = os.path.join(os.getcwd(), "stream-k.tvm_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import streamk
    return streamk


# ---- cases ----
def listed():
    return [
        # one token through a square layer: launch and host latency, then 17 MB of weights
        dict(name="int8_1row", kind="int8", dtype="bfloat16", M=1, N=4096, K=4096, bias=False, activation="none"),
        # a short prompt through an MLP's first projection, bias and activation fused
        dict(name="int8_100rows", kind="int8", dtype="float16", M=100, N=11008, K=4096, bias=True, activation="silu"),
        # a batch of prompts: matrix-bound
        dict(name="int8_4096rows", kind="int8", dtype="bfloat16", M=4096, N=8192, K=8192, bias=False, activation="none"),
        # one token, two of eight experts: the weights of two experts are all there is to read
        dict(name="grouped_1token", kind="grouped", dtype="bfloat16", E=8, R=2, N=11008, K=4096, skew=0.0, bias=False, activation="none"),
        # 64 sequences decoding, two experts each: about sixteen rows an expert, all experts' weights
        dict(name="grouped_64tokens", kind="grouped", dtype="float16", E=8, R=128, N=11008, K=4096, skew=0.5, bias=False, activation="silu"),
        # 125 tokens times eight of sixteen small experts with int8 weights, ragged
        dict(name="grouped_int8_1000rows", kind="grouped", dtype="int8", E=16, R=1000, N=4096, K=2048, skew=0.5, bias=True, activation="none"),
        # a prompt of 2048 tokens times eight of 64 small experts, very unequal
        dict(name="grouped_64experts", kind="grouped", dtype="float16", E=64, R=16384, N=2048, K=4096, skew=1.0, bias=False, activation="none"),
        # a prompt of 4096 tokens, two of eight large experts: matrix-bound
        dict(name="grouped_8192rows", kind="grouped", dtype="bfloat16", E=8, R=8192, N=11008, K=4096, skew=0.3, bias=False, activation="none"),
        # a small training batch, ragged
        dict(name="gradient_500rows", kind="gradient", dtype="float16", E=8, R=500, N=2048, K=1024, skew=0.5),
        # a training step's share of a large layer
        dict(name="gradient_8192rows", kind="gradient", dtype="bfloat16", E=8, R=8192, N=11008, K=4096, skew=0.3),
        # sixteen sequences decoding, eight of 64 experts: latency
        dict(name="exchange_16tokens", kind="exchange", dtype="bfloat16", T=16, E=64, k=8, H=4096, masked=False, backward=False),
        # a training batch with padding tokens (no expert at all) and experts closed to some tokens, all gradients
        dict(name="exchange_8192tokens", kind="exchange", dtype="bfloat16", T=8192, E=64, k=8, H=2048, masked=True, backward=True),
    ]


def _log_int(rng, lo, hi, step=1):
    """An integer from lo to hi, spread evenly over its logarithm, a multiple of `step`."""
    v = math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))
    return max(step, min(hi // step * step, int(round(v / step)) * step))


_MOST = 8192 * 11008 * 4096        # multiply-adds of the largest listed product
_MOST_WEIGHTS = 8 * 11008 * 4096   # and its weights


def draw(rng):
    kind = rng.choice(["int8", "int8", "grouped", "grouped", "grouped", "gradient", "exchange"])
    if kind == "exchange":
        E = _log_int(rng, 4, 256)
        k = min(E, _log_int(rng, 1, 8))
        H = _log_int(rng, 256, 8192, 8)
        backward = rng.random() < 0.5
        T = _log_int(rng, 1, min(8192, 8192 * 8 * 2048 // (k * H)))
        return dict(kind=kind, dtype=rng.choice(["float16", "bfloat16"]), T=T, E=E, k=k, H=H, masked=rng.random() < 0.5, backward=backward)
    if kind == "int8":
        K = _log_int(rng, 512, 16384, 16)
        N = _log_int(rng, 512, 28672, 1 if rng.random() < 0.3 else 8)
        M = _log_int(rng, 1, min(8192, 4096 * 8192 * 8192 // (N * K)))
        return dict(kind=kind, dtype=rng.choice(["float16", "bfloat16"]), M=M, N=N, K=K, bias=rng.random() < 0.5,
                    activation=rng.choice(["none", "none", "relu", "gelu_tanh", "silu"]))
    dtype = rng.choice(["float16", "bfloat16", "int8"] if kind == "grouped" else ["float16", "bfloat16"])
    E = _log_int(rng, 1, 64)
    K = _log_int(rng, 256, 8192, 16 if dtype == "int8" else 8)
    N = _log_int(rng, 256, max(256, min(14336, _MOST_WEIGHTS // (E * K))), 1 if rng.random() < 0.3 else 8)
    R = _log_int(rng, 1, min(16384, max(1, _MOST // (N * K))))
    c = dict(kind=kind, dtype=dtype, E=E, R=R, N=N, K=K, skew=rng.choice([0.0, 0.3, 0.5, 1.0]))
    if kind == "grouped":
        c.update(bias=rng.random() < 0.3, activation=rng.choice(["none", "none", "relu", "gelu_tanh", "silu"]))
    return c


# ---- inputs ----
def _sizes(case, seed):
    """Rows of each expert: every row goes to an expert on its own, the experts' shares spread log-normally by `skew`."""
    rng = random.Random(seed * 1000003 + case["E"])
    shares = [math.exp(case["skew"] * rng.gauss(0, 1)) for _ in range(case["E"])]
    sizes = [0] * case["E"]
    for e in rng.choices(range(case["E"]), weights=shares, k=case["R"]):
        sizes[e] += 1
    return sizes


def _normal(gen, shape, std, dtype):
    return torch.randn(shape, generator=gen, device="cuda", dtype=dtype).mul_(std)


def _int8(gen, shape, K):
    """Weights as a row-wise quantiser leaves them (largest magnitude about 127, bell-shaped) and their scales."""
    q = torch.randn(shape, generator=gen, device="cuda").mul_(36).round_().clamp_(-127, 127).to(torch.int8)
    return q, torch.empty(shape[:-1], device="cuda").uniform_(0.5, 1.5, generator=gen).mul_(1 / (36 * math.sqrt(K)))


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    if case["kind"] == "exchange":
        T, E, k, H = case["T"], case["E"], case["k"], case["H"]
        dtype = _TYPES[case["dtype"]]
        logits = torch.randn(T, E, generator=gen, device="cuda").mul_(2).to(dtype).float()   # (rounded: equal ones occur)
        if case["masked"]:
            closed = torch.rand(T, E, generator=gen, device="cuda") < 0.3
            closed |= torch.rand(T, 1, generator=gen, device="cuda") < 0.125
            logits.masked_fill_(closed, -math.inf)
        s = dict(case=case, logits=logits, x=_normal(gen, (T, H), 1.0, dtype), y=_normal(gen, (T * k, H), 1.0, dtype))
        if case["backward"]:
            s.update(d_rows=_normal(gen, (T * k, H), 1.0, dtype), d_out=_normal(gen, (T, H), 1.0, dtype))
            for leaf in (logits, s["x"], s["y"]):
                leaf.requires_grad_()
        return s
    N, K = case["N"], case["K"]
    if case["kind"] == "int8":
        dtype = _TYPES[case["dtype"]]
        w, scale = _int8(gen, (N, K), K)
        x = _normal(gen, (case["M"], K), 1.0, dtype)
        return dict(case=case, x=x, w=w, scale=scale, bias=_normal(gen, (N,), 0.5, dtype) if case["bias"] else None)
    E, R = case["E"], case["R"]
    sizes = _sizes(case, seed)
    starts = [0]
    for n in sizes:
        starts.append(starts[-1] + n)
    s = dict(case=case, offsets=torch.tensor(starts, dtype=torch.int32, device="cuda"), sizes=sizes)
    if case["dtype"] == "int8":
        s["x"], s["scale_x"] = _int8(gen, (R, K), 1)
        s["w"], s["scale_w"] = _int8(gen, (E, N, K), K)
        dtype = torch.bfloat16
    else:
        dtype = _TYPES[case["dtype"]]
        s["x"], s["w"] = _normal(gen, (R, K), 1.0, dtype), _normal(gen, (E, N, K), 1 / math.sqrt(K), dtype)
    if case["kind"] == "gradient":
        s["dy"] = _normal(gen, (R, N), 1.0, dtype)
        s["x"].requires_grad_()
        s["w"].requires_grad_()
    else:
        s["bias"] = _normal(gen, (E, N), 0.5, dtype) if case["bias"] else None
    return s


# ---- one pass ----
def run(state):
    kind = state["case"]["kind"]
    if own:
        return {"int8": _own_int8, "grouped": _own_grouped, "gradient": _own_gradient, "exchange": _own_exchange}[kind](state)
    with torch.no_grad():
        return {"int8": _plain_int8, "grouped": _plain_grouped, "gradient": _plain_gradient, "exchange": _plain_exchange}[kind](state)


def _act(case):
    return None if case["activation"] == "none" else case["activation"]


def _own_int8(s):
    streamk = _package()
    q, scale = streamk.quantize_int8(s["x"])
    return streamk.streamk_int8_scaled(q, s["w"], scale, s["scale"], out_dtype=s["x"].dtype, bias=s["bias"], activation=_act(s["case"]))


def _own_grouped(s):
    streamk = _package()
    if s["case"]["dtype"] == "int8":
        return streamk.streamk_grouped(s["x"], s["w"], s["offsets"], scale_a=s["scale_x"], scale_b=s["scale_w"], out_dtype=torch.bfloat16,
                                       bias=s["bias"], activation=_act(s["case"]))
    return streamk.streamk_grouped(s["x"], s["w"], s["offsets"], bias=s["bias"], activation=_act(s["case"]))


def _own_gradient(s):
    streamk = _package()
    y = streamk.streamk_grouped(s["x"], s["w"], s["offsets"])
    dx, dw = torch.autograd.grad(y, (s["x"], s["w"]), s["dy"])
    return dict(y=y.detach(), dx=dx, dw=dw)


def _own_exchange(s):
    streamk = _package()
    r = streamk.route_experts(s["logits"], s["case"]["k"])
    rows = streamk.dispatch_rows(s["x"], r)
    out = streamk.combine_rows(s["y"], r)
    got = dict(weights=r.weights.detach(), experts=r.experts, offsets=r.offsets, order=r.order, rows=rows.detach(), out=out.detach())
    if s["case"]["backward"]:
        got["dx"], got["dy"], got["dlogits"] = torch.autograd.grad((rows, out), (s["x"], s["y"], s["logits"]), (s["d_rows"], s["d_out"]))
    return got


def _activate(x, name):
    if name == "relu":
        return x.clamp(min=0)
    if name == "silu":
        return x / (1 + torch.exp(-x))
    if name == "gelu_tanh":
        return x * 0.5 * (1 + torch.tanh(math.sqrt(2 / math.pi) * (x + 0.044715 * x * x * x)))
    return x


def _plain_int8(s):
    x = s["x"].float()
    scale = x.abs().amax(1, keepdim=True) / 127
    q = torch.round(x / scale.clamp(min=1e-30))
    y = (q @ s["w"].float().t()) * scale * s["scale"]
    if s["bias"] is not None:
        y = y + s["bias"].float()
    return _activate(y, s["case"]["activation"]).to(s["x"].dtype)


def _places(s):
    """Where each row stands in an [experts, rows of the largest expert] array."""
    rows = torch.arange(s["case"]["R"], device="cuda", dtype=torch.int32)
    expert = torch.searchsorted(s["offsets"][1:], rows, right=True)
    return expert, (rows - s["offsets"][expert]).long()


def _spread(s, x, expert, place):
    full = torch.zeros(s["case"]["E"], max(s["sizes"]), x.shape[1], device="cuda")
    full[expert, place] = x.float()
    return full


def _plain_grouped(s):
    expert, place = _places(s)
    y = torch.bmm(_spread(s, s["x"], expert, place), s["w"].float().transpose(1, 2))[expert, place]
    if s["case"]["dtype"] == "int8":
        y = y * s["scale_x"][:, None] * s["scale_w"][expert]
    if s["bias"] is not None:
        y = y + s["bias"].float()[expert]
    return _activate(y, s["case"]["activation"]).to(torch.bfloat16 if s["case"]["dtype"] == "int8" else s["x"].dtype)


def _plain_gradient(s):
    expert, place = _places(s)
    x, dy, w = _spread(s, s["x"], expert, place), _spread(s, s["dy"], expert, place), s["w"].float()
    y = torch.bmm(x, w.transpose(1, 2))[expert, place]
    dx = torch.bmm(dy, w)[expert, place]
    dw = torch.bmm(dy.transpose(1, 2), x)
    t = s["x"].dtype
    return dict(y=y.to(t), dx=dx.to(t), dw=dw.to(t))


def _plain_exchange(s):
    T, E, k = s["case"]["T"], s["case"]["E"], s["case"]["k"]
    dtype = s["x"].dtype
    best, experts = torch.sort(s["logits"], dim=1, descending=True, stable=True)
    best, experts = best[:, :k], experts[:, :k]
    chosen = best > -math.inf
    e = torch.where(chosen, torch.exp(best - best[:, :1]), 0)
    weights = torch.where(chosen, e / e.sum(1, keepdim=True), 0)
    experts = torch.where(chosen, experts, -1)
    flat = torch.where(chosen, experts, E).view(-1)
    order = torch.sort(flat, stable=True).indices
    counts = (flat[:, None] == torch.arange(E, device="cuda")).sum(0)
    offsets = torch.cat([counts.new_zeros(1), counts.cumsum(0)])
    place = torch.empty_like(order)
    place[order] = torch.arange(T * k, device="cuda")
    used = (torch.arange(T * k, device="cuda") < offsets[E])[:, None]
    rows = torch.where(used, s["x"][order // k], 0)
    place = place.view(T, k)
    y = torch.where(chosen[..., None], s["y"][place].float(), 0)
    out = (y * weights[..., None]).sum(1)
    got = dict(weights=weights, experts=experts.int(), offsets=offsets.int(), order=torch.where(used[:, 0], order, -1).int(), rows=rows, out=out.to(dtype))
    if s["case"]["backward"]:
        d_out = s["d_out"].float()
        got["dx"] = torch.where(chosen[..., None], s["d_rows"][place].float(), 0).sum(1).to(dtype)
        got["dy"] = torch.where(used, d_out[order // k] * weights.view(-1)[order][:, None], 0).to(dtype)
        dw = (y * d_out[:, None, :]).sum(2)
        dl = weights * (dw - (weights * dw).sum(1, keepdim=True))
        got["dlogits"] = torch.zeros(T, E, device="cuda").scatter_add_(1, experts.clamp(min=0), dl)
    return got


# ---- what a pass cannot do without ----
def work(case):
    if case["kind"] == "exchange":
        T, E, k, H = case["T"], case["E"], case["k"], case["H"]
        used = T * k * (0.875 if case["masked"] else 1.0)
        b = 4 * T * E + 12 * T * k + 4 * (E + 1)               # logits; weights, experts, order; offsets
        b += 2 * H * (T + T * k) + 2 * H * (used + T)          # x to rows, y to out
        f = 2.0 * used * H
        if case["backward"]:
            b += 2 * H * (used + T) + 2 * H * (T + used + T * k) + 4 * T * E   # rows' gradient to x's; out's gradient, y again, y's; logits'
            f += 5.0 * used * H
        return {"bytes": int(b), "flops": f}
    if case["kind"] == "int8":
        M, N, K = case["M"], case["N"], case["K"]
        return {"bytes": 2 * M * K + N * K + 4 * N + 2 * M * N + (2 * N if case["bias"] else 0), "flops": 2.0 * M * N * K}
    E, R, N, K = case["E"], case["R"], case["N"], case["K"]
    touched = sum(sum(n > 0 for n in _sizes(case, seed)) for seed in range(8)) / 8   # experts that have a row, on the average
    size = 1 if case["dtype"] == "int8" else 2
    if case["kind"] == "grouped":
        b = size * (touched * N * K + R * K) + 2 * R * N + 4 * (E + 1)
        if case["dtype"] == "int8":
            b += 4 * (touched * N + R)
        if case["bias"]:
            b += 2 * touched * N
        return {"bytes": int(b), "flops": 2.0 * R * N * K}
    # the weights and the rows once, the product, dy once, both gradients (an expert without rows has one too: zeros)
    return {"bytes": int(2 * (touched * N * K + R * K) + 2 * R * N + 2 * R * N + 2 * R * K + 2 * E * N * K) + 4 * (E + 1), "flops": 6.0 * R * N * K}


# ---- the definitions in 64 bits ----
def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return {"int8": _exact_int8, "grouped": _exact_grouped, "gradient": _exact_gradient, "exchange": _exact_exchange}[case["kind"]](s)


def _exact_act(x, name):
    return {"none": lambda v: v, "relu": torch.relu, "silu": lambda v: v * torch.sigmoid(v),
            "gelu_tanh": lambda v: 0.5 * v * (1 + torch.tanh(math.sqrt(2 / math.pi) * (v + 0.044715 * v ** 3)))}[name](x)


def _exact_int8(s):
    # q = round(x / scale) with the scale as the 32-bit number that it is kept as
    x = s["x"].double()
    scale = (x.abs().max(dim=1).values / 127).float().double()
    q = torch.round(x / torch.where(scale > 0, scale, 1)[:, None])
    y = torch.mm(q, s["w"].double().t()) * (scale[:, None] * s["scale"].double()[None, :])
    if s["bias"] is not None:
        y += s["bias"].double()
    return _exact_act(y, s["case"]["activation"])


def _groups(s):
    start = 0
    for e, n in enumerate(s["sizes"]):
        yield e, slice(start, start + n)
        start += n


def _exact_grouped(s):
    y = torch.empty(s["case"]["R"], s["case"]["N"], dtype=torch.float64, device="cuda")
    for e, at in _groups(s):
        y[at] = torch.mm(s["x"][at].double(), s["w"][e].double().t())
        if s["case"]["dtype"] == "int8":
            y[at] *= s["scale_x"][at].double()[:, None] * s["scale_w"][e].double()
        if s["bias"] is not None:
            y[at] += s["bias"][e].double()
    return _exact_act(y, s["case"]["activation"])


def _exact_gradient(s):
    R, N, K = s["case"]["R"], s["case"]["N"], s["case"]["K"]
    y = torch.empty(R, N, dtype=torch.float64, device="cuda")
    dx = torch.empty(R, K, dtype=torch.float64, device="cuda")
    dw = torch.empty(s["w"].shape, dtype=torch.float64, device="cuda")
    for e, at in _groups(s):
        x, dy, w = s["x"][at].double(), s["dy"][at].double(), s["w"][e].double()
        y[at], dx[at], dw[e] = torch.mm(x, w.t()), torch.mm(dy, w), torch.mm(dy.t(), x)
    return dict(y=y, dx=dx, dw=dw)


def _exact_exchange(s):
    T, E, k, H = s["case"]["T"], s["case"]["E"], s["case"]["k"], s["case"]["H"]
    z = s["logits"].double()
    # the place of an expert in its token's list: how many have a larger logit, or an equal one and a lower number
    number = torch.arange(E, device="cuda")
    rank = ((z[:, None, :] > z[:, :, None]) | ((z[:, None, :] == z[:, :, None]) & (number < number[:, None]))).sum(2)
    taken = (rank < k) & (z > -math.inf)
    p = torch.where(taken, torch.exp(z - z.max(dim=1, keepdim=True).values.clamp(min=-1e30)), 0.0)
    p = p / p.sum(1, keepdim=True).clamp(min=1e-300)
    token, expert = taken.nonzero(as_tuple=True)
    slot = rank[token, expert]
    weights = torch.zeros(T, k, dtype=torch.float64, device="cuda")
    experts = torch.full((T, k), -1, dtype=torch.int32, device="cuda")
    weights[token, slot], experts[token, slot] = p[token, expert], expert.int()
    # rows by expert, then token, then slot (a token has an expert once)
    by = torch.argsort(expert * T + token)
    token, expert, slot, n = token[by], expert[by], slot[by], token.numel()
    order = torch.full((T * k,), -1, dtype=torch.int32, device="cuda")
    order[:n] = (token * k + slot).int()
    offsets = torch.zeros(E + 1, dtype=torch.int32, device="cuda")
    offsets[1:] = taken.sum(0).cumsum(0).int()
    rows = torch.zeros(T * k, H, dtype=torch.float64, device="cuda")
    rows[:n] = s["x"].double()[token]
    w = p[token, expert][:, None]
    out = torch.zeros(T, H, dtype=torch.float64, device="cuda").index_add_(0, token, s["y"][:n].double() * w)
    got = dict(weights=weights, experts=experts, offsets=offsets, order=order, rows=rows, out=out)
    if s["case"]["backward"]:
        d_out = s["d_out"].double()[token]
        got["dx"] = torch.zeros(T, H, dtype=torch.float64, device="cuda").index_add_(0, token, s["d_rows"][:n].double())
        got["dy"] = torch.zeros(T * k, H, dtype=torch.float64, device="cuda")
        got["dy"][:n] = d_out * w
        dp = torch.zeros(T, E, dtype=torch.float64, device="cuda")
        dp[token, expert] = (d_out * s["y"][:n].double()).sum(1)
        got["dlogits"] = p * (dp - (p * dp).sum(1, keepdim=True))
    return got
