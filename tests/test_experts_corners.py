"""Operands, recordings and plans at the edge of what the operators for experts and int8 take.  Tolerances as in test_experts.py: fp32 sums
of n terms within 2 n 2^-24 of the sum of the terms' magnitudes, one rounding to the result's type."""
import ctypes
import math
import os
import random
import subprocess
import sys
import textwrap

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


def tiles_of(*kinds):
    """(kind, variant) of the tiles that there are: [K, N] weights have three of the six"""
    return [(kind, variant) for kind in kinds for variant in ((1, 2, 5) if kind.endswith("nn") else (1, 2, 3, 4, 5, 6))]


# ---- activations of what is not finite ----
ACTIVATIONS = ["relu", "gelu_tanh", "silu"]


def bad_row(A, B):
    """Row 1 of A makes NaN of every column, row 2 +infinity of the even columns of B [N, K] and -infinity of the odd ones, row 3 zeros."""
    A[1, 5] = math.nan
    A[2:4] = 0
    A[2, 0] = math.inf
    B[0::2, 0], B[1::2, 0] = 1, -1


def assert_bad_rows(C, clean, activation):
    assert torch.isnan(C[1]).all()
    assert torch.isposinf(C[2, 0::2]).all()
    # (gelu and silu of -infinity are the product -infinity * 0)
    assert (C[2, 1::2] == 0).all() if activation == "relu" else torch.isnan(C[2, 1::2]).all()
    assert not C[3].any()
    assert torch.equal(C[4:], clean[4:]) and torch.equal(C[0], clean[0])


@pytest.mark.gpu
@pytest.mark.parametrize("activation", ACTIVATIONS)
@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("M,kw", [(8, {}), (20, {}), (60, {}), (100, dict(bm=128, bn=128)), (300, dict(bm=256, bn=256)), (100, dict(variant=11)), (100, dict(layout="nn")), (300, dict(layout="nn"))])
def test_products_keep_nan_through_activations(sk, activation, dtype, M, kw):
    N, K, t = 264, 256, TYPES[dtype]
    run = sk.streamk_fp16 if dtype == "float16" else sk.streamk_bf16
    A, B = rand((M, K), t, 1), rand((N, K), t, 2, 1 / 16)
    good = A.clone()
    bad_row(A, B)
    W = B.T.contiguous() if kw.get("layout") == "nn" else B
    assert_bad_rows(run(A, W, activation=activation, **kw), run(good, W, activation=activation, **kw), activation)


@pytest.mark.gpu
@pytest.mark.parametrize("activation", ACTIVATIONS)
@pytest.mark.parametrize("kind,variant", tiles_of("float16 nt", "bfloat16 nt", "float16 nn", "bfloat16 nn"))
def test_grouped_products_keep_nan_through_activations(sk, activation, kind, variant):
    dtype, layout = kind.split()
    sizes, N, K, t = [70, 0, 130], 264, 256, TYPES[dtype]
    A, B, bias = rand((200, K), t, 1), rand((3, N, K), t, 2, 1 / 16), torch.zeros(3, N, dtype=t, device="cuda")
    good = A.clone()
    bad_row(A, B[0])
    W = B.transpose(1, 2).contiguous() if layout == "nn" else B
    run = lambda a, **kw: sk.streamk_grouped(a, W, offsets_of(sizes), layout=layout, variant=variant, activation=activation, **kw)  # noqa: E731
    assert_bad_rows(run(A), run(good), activation)
    assert_bad_rows(run(A, bias=bias), run(good, bias=bias), activation)


@pytest.mark.gpu
@pytest.mark.parametrize("activation", ACTIVATIONS)
@pytest.mark.parametrize("out", sorted(TYPES))
@pytest.mark.parametrize("variant", [1, 2, 3, 4, 5, 6])
def test_grouped_int8_products_keep_nan_through_activations(sk, activation, out, variant):
    sizes, N, K = [70, 0, 130], 264, 256
    g = torch.Generator().manual_seed(1)
    A, B = (torch.randint(-127, 128, s, generator=g, dtype=torch.int8).cuda() for s in ((200, K), (3, N, K)))
    sa, sb = torch.rand(200, device="cuda") * 0.01, torch.rand(3, N, device="cuda") * 0.01
    run = lambda: sk.streamk_grouped(A, B, offsets_of(sizes), scale_a=sa, scale_b=sb, out_dtype=TYPES[out], variant=variant, activation=activation)  # noqa: E731
    clean = run()
    sa[1], sb[2, 7] = math.nan, math.nan
    C, bad = run(), torch.zeros(200, N, dtype=torch.bool, device="cuda")
    bad[1], bad[70:, 7] = True, True
    assert torch.equal(torch.isnan(C), bad) and torch.equal(C[~bad], clean[~bad])


@pytest.mark.gpu
@pytest.mark.parametrize("activation", ACTIVATIONS)
@pytest.mark.parametrize("out", sorted(TYPES))
@pytest.mark.parametrize("M,config", [(1, {}), (20, {}), (60, dict(variant=9)), (60, dict(variant=12)), (100, {}), (300, dict(bm=64, bn=64, variant=11)), (300, dict(bm=128, bn=128)), (300, dict(bm=64, bn=128, bk=64)),
                                      (300, dict(bm=256, bn=256)), (300, dict(bm=256, bn=256, schedule="splitk", split=2)), (300, dict(bm=128, bn=128, schedule="splitk", split=4))])
def test_int8_products_keep_nan_through_activations(sk, activation, out, M, config):
    N, K = 264, 512
    g = torch.Generator().manual_seed(1)
    A, B = (torch.randint(-127, 128, s, generator=g, dtype=torch.int8).cuda() for s in ((M, K), (N, K)))
    sa, sb = torch.rand(M, device="cuda") * 0.01, torch.rand(N, device="cuda") * 0.01
    run = lambda: sk.streamk_int8_scaled(A, B, sa, sb, out_dtype=TYPES[out], activation=activation, **config)  # noqa: E731
    clean = run()
    sa[M // 2], sb[7] = math.nan, math.nan
    C, bad = run(), torch.zeros(M, N, dtype=torch.bool, device="cuda")
    bad[M // 2], bad[:, 7] = True, True
    assert torch.equal(torch.isnan(C), bad) and torch.equal(C[~bad], clean[~bad])


@pytest.mark.gpu
@pytest.mark.parametrize("M", [1, 7, 40, 200])
def test_other_products_keep_nan_through_relu(sk, M):
    N, K = 256, 512
    A = rand((M, K), torch.float16, 1)
    A[M // 2, 3] = math.nan
    q, s = sk.quantize_q4(rand((N, K), torch.float16, 2))
    f8 = A.to(torch.float8_e4m3fn)
    assert torch.isnan(f8[M // 2, 3].float())
    for C in (sk.streamk_q4(A, q, s, activation="relu"), sk.streamk_fp8(f8, rand((N, K), torch.float16, 3).to(torch.float8_e4m3fn), activation="relu")):
        bad = torch.isnan(C).all(1)
        assert bad[M // 2] and bad.sum() == 1 and torch.isnan(C).any(1).sum() == 1


@pytest.mark.gpu
@pytest.mark.parametrize("activation", ACTIVATIONS)
@pytest.mark.parametrize("weights", ["float16", "bfloat16", "int8"])
def test_a_bad_token_stays_bad_through_a_layer_of_experts(sk, activation, weights):
    torch.manual_seed(0)
    layer = sk.StreamKMoE(64, 96, 4, 2, activation=activation, weight_format="bfloat16" if weights == "int8" else weights, device="cuda")
    layer = sk.StreamKMoE.quantized(layer) if weights == "int8" else layer
    x = torch.randn(20, 64, device="cuda").to(layer.dtype)
    with torch.no_grad():
        # (the routes of the clean tokens: a NaN logit is never chosen, and such a token would go to no expert)
        route, clean = layer.route(x), layer(x)
        bad = x.clone()
        bad[3, 7] = math.nan
        layer.route = lambda rows: route
        runs = [layer(bad)]
    if weights != "int8":
        runs.append(layer(bad.requires_grad_()).detach())   # (recorded: the activation is an operation of its own)
    keep = torch.arange(20, device="cuda") != 3
    for out in runs:
        assert torch.isnan(out[3]).all() and torch.isfinite(out[keep]).all()
    assert torch.equal(runs[0][keep], clean[keep])


# ---- derivatives that do not exist are refused, in the native operators and in the ones that stand in for them ----
PACKAGE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "stream-k.tvm_amd", "streamk")


@pytest.fixture(params=["native", "without the native library"])
def run_with_fakes(request, tmp_path):
    """Runs code in a process of its own, under FakeTensorMode: operands A [10, 64], B [3, 32, 64], offsets, a route, and `new` for more."""
    package = tmp_path / "streamk"
    package.mkdir()
    for name in os.listdir(PACKAGE):
        if name != "__pycache__" and (request.param == "native" or name != "libstreamk_torch.so"):
            (package / name).symlink_to(os.path.join(PACKAGE, name))
    head = f"""
        import sys
        sys.path.insert(0, {str(tmp_path)!r})
        import torch, streamk as sk, streamk.experts as experts
        import torch.autograd.forward_ad as fw
        from torch._subclasses.fake_tensor import FakeTensorMode
        assert experts._NATIVE == {request.param == "native"}
        FakeTensorMode().__enter__()
        new = lambda *s, dtype=torch.float16: torch.empty(*s, dtype=dtype, device="cuda")
        A, B, offsets, logits = new(10, 64), new(3, 32, 64), new(4, dtype=torch.int32), new(5, 4, dtype=torch.float32)
        route = sk.route_experts(logits, 2)
        def refused(error, f):
            try:
                f()
            except error as e:
                return str(e)
            raise SystemExit("not refused")
        """
    env = {**os.environ, "PYTHONDONTWRITEBYTECODE": "1"}
    return lambda code: subprocess.run([sys.executable, "-c", textwrap.dedent(head) + textwrap.dedent(code)], check=True, timeout=100, env=env)


def test_forward_mode_is_refused(run_with_fakes):
    run_with_fakes("""
        with fw.dual_level():
            dual = lambda t: fw.make_dual(t, t.clone())
            for f in (lambda: sk.streamk_grouped(dual(A), B, offsets), lambda: sk.streamk_grouped(A, dual(B), offsets),
                      lambda: sk.streamk_grouped(A, B, offsets, bias=dual(new(3, 32)), activation="silu"),
                      lambda: sk.route_experts(dual(logits), 2), lambda: sk.dispatch_rows(dual(new(5, 64)), route),
                      lambda: sk.combine_rows(dual(A), route), lambda: sk.combine_rows(A, route._replace(weights=dual(route.weights)))):
                assert "forward-mode" in refused(NotImplementedError, f)
            sk.streamk_grouped(A, B, offsets)
        refused(NotImplementedError, lambda: torch.func.jvp(lambda a: sk.streamk_grouped(a, B, offsets), (A,), (A.clone(),)))
        """)


@pytest.mark.gpu
def test_a_product_without_gradients_says_so(sk):
    """Bias, activation and scales of a recorded call: the operator's result has a derivative that raises, not none."""
    o, offsets = torch.ops.streamk, offsets_of([12, 8])
    A, B, bias = rand((20, 64), torch.float16, 1), rand((2, 32, 64), torch.float16, 2), rand((2, 32), torch.float16, 3)
    q, s = sk.quantize_int8(A)
    w, sw = sk.quantize_int8(B)
    a, b, c, t = (x.clone().requires_grad_() for x in (A, B, bias, sw))
    calls = [((a, B, offsets, "nt", None, None, None, None, "silu"), (A, B, offsets, "nt", None, None, None, None, "silu")),
             ((A, b, offsets, "nt", None, None, None, bias, "none"), (A, B, offsets, "nt", None, None, None, bias, "none")),
             ((A, B, offsets, "nt", None, None, None, c, "relu"), (A, B, offsets, "nt", None, None, None, bias, "relu")),
             ((q, w, offsets, "nt", None, s, t), (q, w, offsets, "nt", None, s, sw))]
    for recorded, ordinary in calls:
        want, got = o.gemm_grouped(*ordinary), o.gemm_grouped(*recorded)
        assert got.requires_grad and not want.requires_grad and torch.equal(got, want)
        with pytest.raises(RuntimeError, match="has gradients only without bias"):
            got.sum().backward()
        with torch.no_grad():
            assert not o.gemm_grouped(*recorded).requires_grad
    # (what is not differentiated runs on: int8 scales that a recorded quantiser has made)
    q, s = sk.quantize_int8(a)
    assert torch.equal(sk.streamk_grouped(q, w, offsets, scale_a=s, scale_b=sw), o.gemm_grouped(q, w, offsets, "nt", None, s.detach(), sw))


@pytest.mark.gpu
def test_gradients_with_create_graph(sk):
    """create_graph gives the gradients; only differentiating them again is refused, by whatever they were made of."""
    offsets, logits = offsets_of([12, 8]), rand((10, 4), torch.float32, 4)
    A, B, x, y = rand((20, 64), torch.float16, 1), rand((2, 32, 64), torch.float16, 2), rand((10, 64), torch.float16, 3), rand((20, 64), torch.float16, 5)
    route = sk.route_experts(logits, 2)
    A, B, logits, x, y = (t.requires_grad_() for t in (A, B, logits, x, y))
    weights = route.weights.clone().requires_grad_()
    calls = [(lambda: sk.streamk_grouped(A, B, offsets), (A, B)), (lambda: sk.streamk_grouped(A, B.transpose(1, 2).contiguous(), offsets, layout="nn"), (A, B)),
             (lambda: sk.route_experts(logits, 2).weights, (logits,)), (lambda: sk.dispatch_rows(x, route), (x,)),
             (lambda: sk.combine_rows(y, route._replace(weights=weights)), (y, weights))]
    for call, leaves in calls:
        d = rand(call().shape, call().dtype, 7)
        want = torch.autograd.grad(call(), leaves, d)
        for g, w in zip(torch.autograd.grad(call(), leaves, d, create_graph=True), want):
            assert torch.equal(g, w)
        # the incoming gradient requires one
        d = d.requires_grad_()
        got = torch.autograd.grad(call(), leaves, d, create_graph=True)
        for i, (g, w) in enumerate(zip(got, want)):
            assert torch.equal(g, w) and g.requires_grad
            with pytest.raises(RuntimeError, match="not differentiable again"):
                torch.autograd.grad(g.float().sum(), d, retain_graph=True)
    # dB is made of A, dA of B
    dA, dB = torch.autograd.grad(sk.streamk_grouped(A, B, offsets), (A, B), d_of(A, B), create_graph=True)
    for g, leaf in ((dA, B), (dB, A)):
        with pytest.raises(RuntimeError, match="not differentiable again"):
            torch.autograd.grad(g.float().sum(), leaf, retain_graph=True)
    # a penalty on another layer's gradient
    z = rand((20, 64), torch.float32, 8).requires_grad_()
    loss = (sk.streamk_grouped(A, B, offsets).float().sum() + z.pow(3).sum())
    _, gz = torch.autograd.grad(loss, (A, z), create_graph=True)
    assert torch.allclose(torch.autograd.grad(gz.sum(), z)[0], 6 * z)


def d_of(A, B):
    return rand((A.shape[0], B.shape[1]), A.dtype, 9)


# ---- int8 products with scales and the tuned cache of the int32 ones ----
@pytest.fixture
def tuned(sk, monkeypatch):
    """entries(M, N, K, config) puts an int8 entry of the newest search into the tuned cache, for this test."""
    from streamk import ops
    from streamk import plan as plan_mod

    def enter(M, N, K, config):
        plan_mod.invalidate_tuned_cache()
        monkeypatch.setattr(plan_mod, "_tuned", {f"gfx950/int8/nt/{M}x{N}x{K}": {"config": config, "search": sys.modules["streamk.autotune"].SEARCH}})
        ops._plan_cache.clear()
    yield enter
    monkeypatch.undo()
    plan_mod.invalidate_tuned_cache()
    ops._plan_cache.clear()


def test_plans_without_scales_are_not_taken_from_the_tuned_cache(sk, tuned, monkeypatch):
    from streamk import int8, ops
    from streamk import plan as plan_mod
    monkeypatch.setattr(plan_mod, "num_cus", lambda: 256)
    takes = lambda p: sk.lib().sk_i8_scaled_takes(ctypes.byref(p))  # noqa: E731
    refused = 0
    for M, N, K in ((1, 4096, 4096), (16, 4096, 4096), (20, 520, 1040), (64, 2048, 8192), (100, 4096, 4096), (700, 1031, 2064)):
        for config in sk.candidate_configs(M, N, K, "int8", cus=256):
            try:
                plan = sk.make_plan(M, N, K, "int8", "nt", config)
            except sk.StreamKError:
                continue
            if takes(plan):
                continue
            refused += 1
            tuned(M, N, K, config)
            assert ops._plan_for("", M, N, K, "int8", "nt").kernel_id == plan.kernel_id   # (the int32 product's)
            for pitch in (0, 1 << 25):
                own = int8.plan_for("", M, N, K, pitch, pitch)
                assert takes(own) and (own.M, own.N, own.K) == (M, N, K) and own.kernel_id != plan.kernel_id
            assert int8.plan_for("variant=1", M, N, K).kernel_id == sk.make_plan(M, N, K, "int8", "nt", variant=1).kernel_id   # (what a caller names stays)
            assert takes(sk.StreamKLinear(K, N, weight_format="int8").plan_for(M))
    assert refused > 50


def test_untuned_plans_have_a_form_with_scales(sk, monkeypatch):
    from streamk import ops
    from streamk import plan as plan_mod
    monkeypatch.setattr(plan_mod, "num_cus", lambda: 256)
    rng = random.Random(5)
    for _ in range(400):
        M, N, K = (int(math.exp(rng.uniform(0, math.log(top)))) for top in (9000, 30000, 1200))
        for config in (ops._UNTUNED, ops._UNTUNED_LONG_ROWS):
            plan = ops._plan_of(config, M, N, 16 * K, "int8", "nt")
            assert sk.lib().sk_i8_scaled_takes(ctypes.byref(plan)), (M, N, 16 * K, sk.kernel_name(plan.kernel_id))


@pytest.mark.gpu
@pytest.mark.parametrize("M,N,K,config", [(16, 512, 1024, dict(bm=16, bn=16, bk=1024, schedule="dp")), (3, 260, 4096, dict(bm=16, bn=32, bk=1024, schedule="sk2", grid=256, fixup="reduce")),
                                          (60, 512, 1024, dict(bm=64, bn=64, bk=512, schedule="dp"))])
def test_int8_calls_after_a_search(sk, tuned, M, N, K, config):
    from streamk import ops
    assert not sk.lib().sk_i8_scaled_takes(ctypes.byref(sk.make_plan(M, N, K, "int8", "nt", config)))
    g = torch.Generator().manual_seed(1)
    A, B = (torch.randint(-127, 128, s, generator=g, dtype=torch.int8).cuda() for s in ((M, K), (N, K)))
    sa, sb = torch.rand(M, device="cuda") * 0.01, torch.rand(N, device="cuda") * 0.01
    run = lambda: sk.streamk_int8_scaled(A, B, sa, sb)  # noqa: E731
    want = run()
    layer = sk.StreamKLinear.from_linear(torch.nn.Linear(K, N, device="cuda", dtype=torch.float16), weight_format="int8")
    x = torch.randn(M, K, device="cuda").half()
    y = layer(x)
    tuned(M, N, K, config)
    for _ in range(2):   # (the second time the native operator knows the int32 product's plan)
        assert torch.equal(sk.streamk_int8(A, B).double(), A.double() @ B.double().T)
        assert torch.equal(run(), want) and torch.equal(layer(x), y)
    assert ops._plan_for("", M, N, K, "int8", "nt").kernel_id == sk.make_plan(M, N, K, "int8", "nt", config).kernel_id


@pytest.mark.gpu
@pytest.mark.parametrize("M,N,K", [(16, 512, 1024), (64, 512, 4096), (200, 512, 2048), (600, 1024, 1024)])
def test_every_plan_that_is_said_to_run_does(sk, M, N, K):
    g = torch.Generator().manual_seed(1)
    A, B = (torch.randint(-127, 128, s, generator=g, dtype=torch.int8).cuda() for s in ((M, K), (N, K)))
    sa, sb = torch.rand(M, device="cuda") * 0.01, torch.rand(N, device="cuda") * 0.01
    want, ran = sk.streamk_int8_scaled(A, B, sa, sb), 0
    for config in sk.candidate_configs(M, N, K, "int8"):
        try:
            plan = sk.make_plan(M, N, K, "int8", "nt", config)
        except sk.StreamKError:
            continue
        if sk.lib().sk_i8_scaled_takes(ctypes.byref(plan)):
            assert torch.equal(sk.streamk_int8_scaled(A, B, sa, sb, plan=plan), want), config
            ran += 1
        else:
            with pytest.raises(sk.StreamKError):
                sk.streamk_int8_scaled(A, B, sa, sb, plan=plan)
    sk.workspace_status()
    assert ran > 10


# ---- tiles that several CTAs share ----
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", sorted(TYPES))
def test_a_wait_that_gives_up_leaves_its_tile_alone(sk, dtype):
    """No polls at all: whoever comes last to a tile that is cut gives up.  Its part of C stays as it was, the workspace says so and is refused
    until it is a new one, and the flags of the late parts stand in nobody's way."""
    from streamk import _lib, ops
    E, R, N, K, t = 1, 256, 512, 4096, TYPES[dtype]   # (two tiles, each cut in four)
    A, B, offsets = rand((R, K), t, 1), rand((E, N, K), t, 2, 1 / 64), offsets_of([R])
    want = sk.streamk_grouped(A, B, offsets, variant=2)
    C = torch.full((R, N), 7.0, dtype=t, device="cuda")
    g = _lib.SkGrouped(dtype=_lib.SK_F16 if t == torch.float16 else _lib.SK_BF16, layout=0, out_dtype=_lib.SK_F16 if t == torch.float16 else _lib.SK_BF16, E=E, R=R, N=N, K=K,
                       A=A.data_ptr(), B=B.data_ptr(), offsets=offsets.data_ptr(), C=C.data_ptr(), lda=K, ldb=K, ldc=N, variant=2, spin_limit=-1)
    L = sk.lib()
    ws = ops._workspace(L.sk_grouped_workspace_bytes(ctypes.byref(g)), A.device)
    launch = lambda: L.sk_gemm_grouped(ctypes.byref(g), ws.data_ptr(), ws.numel(), ops._stream_ptr())  # noqa: E731
    try:
        assert launch() == 0
        torch.cuda.synchronize()
        assert (C == 7).all()
        flags = ws[256:256 + 4 * 1024].view(torch.int32)
        assert flags[:8].sum() == 6 and (flags[256:258] == 4).all()   # (three of four parts of each tile; the counters)
        with pytest.raises(sk.StreamKError) as e:
            sk.workspace_status()
        assert e.value.status == -8 and launch() == -8
        with pytest.raises(sk.StreamKError):
            sk.streamk_grouped(A, B, offsets, variant=2)
    finally:
        sk.reset_workspaces()
    assert torch.equal(sk.streamk_grouped(A, B, offsets, variant=2), want)
    sk.workspace_status()


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["float16 nt", "bfloat16 nt", "float16 nn", "bfloat16 nn", "int8"])
@pytest.mark.parametrize("variant,sizes,N,K", [(2, [300, 0, 200], 512, 4096), (2, [300, 0, 200], 512, 4224), (2, [100, 60, 0, 7], 1024, 8192), (2, [2000], 2304, 4096), (2, [40, 4000], 4352, 4096),
                                               (5, [70, 200], 1000, 2048), (5, [1, 3, 0, 500], 264, 8192), (5, [64] * 8, 2048, 1024)])
def test_shared_tiles_leave_the_workspace_as_it_was(sk, kind, variant, sizes, N, K):
    from streamk import ops
    R, E, offsets = sum(sizes), len(sizes), offsets_of(sizes)
    if kind == "int8":
        g = torch.Generator().manual_seed(R)
        A, B = (torch.randint(-127, 128, s, generator=g, dtype=torch.int8).cuda() for s in ((R, K), (E, N, K)))
        sa, sb = (torch.rand(R, generator=g) + 0.5).cuda() * 0.01, (torch.rand(E, N, generator=g) + 0.5).cuda() / (73 * math.sqrt(K))
        run = lambda: sk.streamk_grouped(A, B, offsets, scale_a=sa, scale_b=sb, variant=variant)  # noqa: E731
        want = torch.cat([(A[at].double() @ B[e].double().T) * sa[at].double()[:, None] * sb[e].double() for e, at in groups(sizes)])
        terms, magnitudes = 2, want.abs()
    else:
        dtype, layout = kind.split()
        A, W = rand((R, K), TYPES[dtype], R), rand((E, K, N), TYPES[dtype], N, 1 / math.sqrt(K))
        B = W if layout == "nn" else W.transpose(1, 2).contiguous()
        run = lambda: sk.streamk_grouped(A, B, offsets, layout=layout, variant=variant)  # noqa: E731
        want, magnitudes = plain_kn(A, W, sizes)
        terms = K
    C = run()
    assert_near(C, want, terms, magnitudes)
    for _ in range(5):
        assert torch.equal(run(), C)
    sk.workspace_status()
    words = ops._workspaces[(0, torch.cuda.current_stream().cuda_stream)][:256 + 4 * 1024].view(torch.int32)
    assert words[0] == 0 and not words[64:].any()   # (status; flags and counters)


# ---- experts whose weights span 2 GiB ----
@pytest.mark.gpu
@pytest.mark.parametrize("N,E,sizes", [(262144, 1, [20]), (262149, 2, [3, 130])])
def test_gradients_of_large_experts(sk, N, E, sizes):
    """The product takes them ([N, K] weights are addressed by tiles); so do the gradients, whose [K, N] form goes through a copy."""
    K, R, offsets = 4096, sum(sizes), offsets_of(sizes)
    A, d = rand((R, K), torch.bfloat16, 1), rand((R, N), torch.bfloat16, 2)
    B = torch.empty((E, N, K), dtype=torch.bfloat16, device="cuda").normal_(0, 1 / 64)
    assert B[0].numel() * 2 >= 2 ** 31
    x, w = A.clone().requires_grad_(), B.requires_grad_()
    dx, dw = torch.autograd.grad(sk.streamk_grouped(x, w, offsets), (x, w), d)
    B = B.detach()
    for e, at in groups(sizes):
        want, magnitudes = torch.zeros(sizes[e], K, dtype=torch.float64, device="cuda"), torch.zeros(sizes[e], K, dtype=torch.float64, device="cuda")
        for n in range(0, N, 32768):
            part, rows = B[e, n:n + 32768].double(), d[at, n:n + 32768].double()
            want += rows @ part
            magnitudes += rows.abs() @ part.abs()
        assert_near(dx[at], want, N, magnitudes)
        for cols in (slice(0, 9), slice(N - 9, N)):
            assert_near(dw[e, cols], d[at, cols].double().T @ A[at].double(), sizes[e], d[at, cols].double().abs().T @ A[at].double().abs())
    assert torch.equal(sk.streamk_grouped(d, B, offsets, layout="nn"), dx)


@pytest.mark.gpu
def test_large_experts_with_a_pitch_are_no_different(sk):
    """Few columns far apart: the span counts, not the size."""
    E, N, K, sizes = 2, 64, 1030, [5, 12]
    wide = torch.zeros((E, K, 1 << 20), dtype=torch.float16, device="cuda")
    B = wide[:, :, :N]
    B.copy_(rand((E, K, N), torch.float16, 2, 1 / 32))
    A = rand((17, K), torch.float16, 1)
    want, magnitudes = plain_kn(A, B, sizes)
    assert_near(sk.streamk_grouped(A, B, offsets_of(sizes), layout="nn"), want, K, magnitudes)


# ---- int8 layers of weights with more than 16 bits ----
def test_int8_layer_of_fp32_weights(sk):
    """On the CPU: quantised from what they are -- beyond fp16's largest number, below its smallest, next to a tie that fp16 would move."""
    linear = torch.nn.Linear(64, 9, bias=True)
    w = linear.weight.data
    w[1, 3] = 7e4
    w[2] = torch.arange(64) * 1e-12
    w[3] = 0
    w[4, 5] = math.inf
    w[5, 6] = math.nan
    w[6] = 0
    w[6, :3] = torch.tensor([127.0, 0.5 + 2.0 ** -20, 2.5])   # scale 1
    w[7, 0] = -3e38
    layer = sk.StreamKLinear.from_linear(linear, weight_format="int8", activation="relu")
    q, s = layer.qweight, layer.weight_scale
    assert layer.dtype == torch.float16 and layer.activation == "relu" and torch.equal(layer.bias, linear.bias.half())
    assert torch.isnan(s[4:6]).all() and not q[4:6].any() and s[3] == 0 and not q[3].any()
    assert q[6, :3].tolist() == [127, 1, 2] and q[7, 0] == -127 and torch.isfinite(s[[0, 1, 2, 6, 7, 8]]).all()
    for r in (0, 1, 2, 7, 8):
        want = w[r].double().abs().max() / 127
        assert s[r] == want.float() and torch.equal(q[r].double(), torch.round(w[r].double() / s[r].double()))


@pytest.mark.gpu
def test_int8_layer_of_fp32_weights_like_that_of_16_bits(sk):
    linear = torch.nn.Linear(512, 300, device="cuda", dtype=torch.float16)
    wide = torch.nn.Linear(512, 300, device="cuda")
    wide.load_state_dict({k: v.float() for k, v in linear.state_dict().items()})
    a, b = (sk.StreamKLinear.from_linear(m, weight_format="int8") for m in (linear, wide))
    for x, y in zip(a.state_dict().values(), b.state_dict().values()):
        assert x.dtype == y.dtype and torch.equal(x, y)
    wide.weight.data[7, 100] = 1e5
    c = sk.StreamKLinear.from_linear(wide, weight_format="int8")
    x = torch.randn(20, 512, device="cuda").half() * 1e-3
    assert torch.isfinite(c(x)).all()


# ---- more rows than a launch has threads for in one dimension ----
@pytest.mark.gpu
def test_quantiser_of_very_many_rows(sk):
    M = 2 ** 24 + 77
    x = torch.randn(M, 2, device="cuda").half()
    q, s = sk.quantize_int8(x)
    for at in (slice(0, 1000), slice(2 ** 21 - 500, 2 ** 21 + 500), slice(2 ** 24 - 500, M)):
        amax = x[at].double().abs().amax(1)
        assert torch.equal(s[at], (amax / 127).float())
        assert torch.equal(q[at].double(), torch.round(x[at].double() / s[at].double()[:, None]))


@pytest.mark.gpu
@pytest.mark.parametrize("T,k", [(2 ** 25 + 5, 2), (2 ** 26 + 3, 1)])
def test_exchange_of_very_many_rows(sk, T, k):
    logits = torch.randn(T, 3, device="cuda").requires_grad_()
    route = sk.route_experts(logits, k)
    x = torch.arange(T, device="cuda", dtype=torch.int32)
    rows = sk.dispatch_rows(x, route)
    assert torch.equal(rows, torch.div(route.order, k, rounding_mode="floor"))
    by_rows = torch.ops.streamk.dispatch_rows(x, route.order, k)   # (a wave a row, and not a wave a token)
    assert torch.equal(by_rows, rows)
    y = (rows % 1024)[:, None].half().requires_grad_()   # (exact in fp16, and so is the sum of a token's two)
    ones = torch.ones_like(route.weights).requires_grad_()
    out = sk.combine_rows(y, route._replace(weights=ones))
    assert torch.equal(out[:, 0], (k * (x % 1024)).half())
    dy, dw = torch.autograd.grad(out, (y, ones), (x % 512)[:, None].half())
    assert torch.equal(dy[:, 0], (rows % 512).half())
    assert torch.equal(dw, ((x % 1024).float() * (x % 512).float())[:, None].expand(T, k))
    dz, = torch.autograd.grad(route.weights, logits, torch.ones_like(route.weights))
    # (weights that sum to one: their sum has no gradient)
    assert dz[-1000:].abs().max() <= 8 * 2.0 ** -24


# ---- a single row, whose stride says nothing ----
@pytest.mark.gpu
@pytest.mark.parametrize("stride", [64, 97, 61, 1])
def test_a_single_row_of_any_stride(sk, stride):
    """Also where the native operator passes the call on: one column of weights, gradients of one row."""
    base = rand((200,), torch.float16, 1)
    row, offsets = base.as_strided((1, 64), (stride, 1)), offsets_of([1, 0])
    B = rand((2, 32, 64), torch.float16, 2)
    for weights in (B, B[:, :1]):
        assert_near(sk.streamk_grouped(row, weights, offsets), row.double() @ weights[0].double().T, 64, row.double().abs() @ weights[0].double().abs().T)
    W = rand((2, 64, 32), torch.float16, 3)
    assert torch.equal(sk.streamk_grouped(row, W, offsets, layout="nn"), sk.streamk_grouped(row.contiguous(), W, offsets, layout="nn"))
    d = base.as_strided((1, 32), (stride, 1), 80)
    for left in (d, base.as_strided((1, 29), (stride, 1), 80)):
        dw = sk.streamk_grouped_wgrad(left, row, offsets)
        assert torch.equal(dw[0], (left.double().T @ row.double()).half()) and not dw[1].any()
    q = torch.randint(-127, 128, (200,), dtype=torch.int8, device="cuda").as_strided((1, 64), (stride, 1))
    w, s, sw = torch.randint(-127, 128, (2, 1, 64), dtype=torch.int8, device="cuda"), torch.rand(1, device="cuda"), torch.rand(2, 1, device="cuda") * 1e-3
    want = (q.double() @ w[0].double().T) * s.double() * sw[0].double()
    assert_near(sk.streamk_grouped(q, w, offsets, scale_a=s, scale_b=sw), want, 2, want.abs())


# ---- a recorded call and a later one that needs a larger workspace ----
@pytest.mark.gpu
def test_a_recorded_call_keeps_its_workspace(sk):
    from streamk import ops
    sizes = [3, 0, 9]
    A, B, offsets = rand((12, 4096), torch.float16, 1), rand((3, 520, 4096), torch.float16, 2, 1 / 64), offsets_of(sizes)
    large_a, large_b, large_o = rand((700, 4096), torch.float16, 3), rand((2, 512, 4096), torch.float16, 4, 1 / 64), offsets_of([300, 400])
    small, large = (lambda: sk.streamk_grouped(A, B, offsets, variant=3)), (lambda: sk.streamk_grouped(large_a, large_b, large_o, variant=2))
    want, stream, graph = small(), torch.cuda.Stream(), torch.cuda.CUDAGraph()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        small()
        stream.synchronize()
        with torch.cuda.graph(graph, stream=stream):
            C = small()
        key = (0, stream.cuda_stream)
        old = ops._workspaces[key]
        size, address = old.numel(), old.data_ptr()
        del old
        large()
        assert ops._workspaces[key].numel() > size
        # whoever gets memory now must not get the recorded call's
        others = [torch.full((size,), 85, dtype=torch.uint8, device="cuda") for _ in range(8)]
        assert not any(t.data_ptr() <= address < t.data_ptr() + size for t in others)
        for _ in range(3):
            C.zero_()
            graph.replay()
            stream.synchronize()
            assert torch.equal(C, want) and all((t == 85).all() for t in others)
            large()


@pytest.mark.gpu
@pytest.mark.parametrize("variant", [3, 4, 6])
@pytest.mark.parametrize("dtype", sorted(TYPES))
def test_tiles_that_kn_weights_do_not_have(sk, variant, dtype):
    A, B = rand((20, 64), TYPES[dtype], 1), rand((2, 64, 32), TYPES[dtype], 2)
    with pytest.raises(sk.StreamKError) as e:
        sk.streamk_grouped(A, B, offsets_of([12, 8]), layout="nn", variant=variant)
    assert e.value.status == -4


# ---- offsets that are no offsets ----
@pytest.mark.gpu
@pytest.mark.parametrize("kind,variant", [(kind, 0) for kind in ("float16 nt", "bfloat16 nn", "int8")] + tiles_of("float16 nt", "bfloat16 nn", "int8"))
@pytest.mark.parametrize("offsets", [[0, 30, 10, 50], [-5, 20, 90, 40], [100, 0, 100, 0], [60, 50, 40, 30], [7, 7, 3, 100000], [0, 100] * 40 + [0], [(37 * i) % 101 for i in range(200)]])
def test_offsets_out_of_order(sk, kind, variant, offsets):
    """They are clamped to 0 .. R and to ascending order, one below another in front of it counting as that."""
    R, N, K, E = 100, 264, 256, len(offsets) - 1
    wild = torch.tensor(offsets, dtype=torch.int32, device="cuda")
    sane = wild.clamp(0, R).cummax(0).values
    if kind == "int8":
        g = torch.Generator().manual_seed(R)
        A, B = (torch.randint(-127, 128, s, generator=g, dtype=torch.int8).cuda() for s in ((R, K), (E, N, K)))
        sa, sb = torch.rand(R, generator=g).cuda(), (torch.rand(E, N, generator=g) / (73 * math.sqrt(K))).cuda()
        run = lambda o: sk.streamk_grouped(A, B, o, scale_a=sa, scale_b=sb, variant=variant)  # noqa: E731
    else:
        dtype, layout = kind.split()
        A, B = rand((R, K), TYPES[dtype], 1), rand((E, N, K) if layout == "nt" else (E, K, N), TYPES[dtype], 2, 1 / 16)
        run = lambda o: sk.streamk_grouped(A, B, o, layout=layout, variant=variant)  # noqa: E731
    C = run(sane.int())
    assert torch.equal(run(wild), C) and not C[:int(sane[0])].any() and not C[int(sane[-1]):].any()


@pytest.mark.gpu
def test_offsets_out_of_order_make_no_more_tiles(sk):
    """As they stand they would name 2^31 iterations and more."""
    R, N, K, E = 40960, 2048, 4096, 1024
    A, B = rand((R, K), torch.float16, 1), rand((1, N, K), torch.float16, 2, 1 / 64)
    wild = torch.tensor([0, R] * (E // 2) + [0], dtype=torch.int32, device="cuda")
    C = sk.streamk_grouped(A, B.expand(E, N, K), wild, variant=3)
    assert torch.equal(C, sk.streamk_grouped(A, B, offsets_of([R]), variant=3))
