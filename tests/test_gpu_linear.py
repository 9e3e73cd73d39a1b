"""GPU: fused_linear (futudiffu_amd/block_ops.py) against its 64-bit definition
(oracle/block_oracle.py), output and every gradient, in units of what is allowed: the bound
on 32-bit sums in any order and on the 16-bit dz, then one rounding."""

import pytest
import torch

from oracle import block_oracle as O

pytestmark = pytest.mark.gpu

BF, FP, F32 = torch.bfloat16, torch.float16, torch.float32


def _inputs(M, K, N, act, dtype=BF, bias=None, residual=False, seed=0, device="cpu"):
    g = torch.Generator().manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=g)

    rows = 2 * N if act == "swiglu" else N
    v = dict(x=normal(M, K).to(dtype), weight=(normal(rows, K) / K ** 0.5).to(dtype),
             bias=None if bias is None else (0.3 * normal(rows)).to(bias),
             residual=normal(M, N).to(dtype) if residual else None, dout=normal(M, N).to(dtype))
    return {k: None if t is None else t.to(device) for k, t in v.items()}


LEAVES = ("x", "weight", "bias", "residual")


def _run(v, act, grads=True, leaves=None):
    import futudiffu_amd as F
    v = dict(v)
    leaves = [k for k in (leaves or LEAVES) if v[k] is not None] if grads else []
    for k in leaves:
        v[k] = v[k].detach().requires_grad_()
    out = F.fused_linear(*(v[k] for k in LEAVES), activation=act)
    got = {"out": out.detach()}
    if grads:
        got.update(("d" + k, t) for k, t in zip(leaves, torch.autograd.grad(out, [v[k] for k in leaves], v["dout"])))
    return got


def _check(got, want, case=""):
    torch.cuda.synchronize()
    for name, g in got.items():
        exact, bound = want[name]
        w = O.worst(g, exact.to(g.device), bound.to(g.device))
        assert w <= 1.0, f"{case} {name}: {w:.3g} of what is allowed"


def _want(v, act):
    return O.linear(v["x"], v["weight"], v["bias"], v["residual"], act, v["dout"])


# sizes where a path changes or a tile is partly filled: single tokens, the few-row forms
# (16, 32, 64 rows on either side), one tile and its neighbours, odd widths, a contraction
# under one step, of one and of many, with a ragged last one
SHAPES = [(1, 1, 1), (1, 256, 40), (2, 256, 1536), (7, 33, 19), (16, 64, 16), (17, 200, 130), (33, 72, 48),
          (64, 3840, 24), (65, 8, 65), (70, 100, 9), (128, 64, 128), (129, 65, 257), (200, 136, 1000), (300, 16, 520),
          (256, 512, 256), (257, 520, 264), (1000, 24, 16), (513, 1001, 779), (1, 10240, 384), (100, 2048, 100)]


@pytest.mark.parametrize("M,K,N", SHAPES)
def test_outputs_and_gradients(cuda, M, K, N):
    for i, (act, dtype, bias, res) in enumerate((("none", BF, None, False), ("silu", FP, FP, True),
                                                 ("gelu", BF, F32, True), ("swiglu", BF, BF, True),
                                                 ("swiglu", FP, None, False))):
        print(M, K, N, act, dtype, bias, res, flush=True)
        v = _inputs(M, K, N, act, dtype, bias, res, seed=M + N + i, device=cuda)
        got = _run(v, act)
        _check(got, _want(v, act), f"{act} {dtype}")
        assert got["out"].dtype == dtype and (bias is None or got["dbias"].dtype == bias)
        plain = _run(v, act, grads=False)  # without gradients: the same bits
        assert torch.equal(plain["out"].view(torch.int16), got["out"].view(torch.int16))


@pytest.mark.parametrize("M,K,N,act", [(2300, 1536, 2048, "none"), (1280, 4096, 1536, "swiglu"),
                                       (4416, 1024, 3840, "gelu"), (300, 10240, 3840, "none"),
                                       (3071, 1000, 1004, "silu")])
def test_large_products(cuda, M, K, N, act):
    """Whole rounds of large tiles, and tiles cut along the contraction, in every layout."""
    v = _inputs(M, K, N, act, BF, BF, True, seed=M, device=cuda)
    _check(_run(v, act), _want(v, act), act)


def test_integer_products_are_exact(cuda):
    """Small integers: every sum is exact, so a wrong element or a lost or doubled product
    shows whatever the tolerance; through every form and layout."""
    g = torch.Generator().manual_seed(5)
    for M, K, N in ((5, 264, 136), (40, 1000, 1000), (200, 331, 140), (700, 520, 600), (2000, 72, 40), (1500, 2048, 1032)):
        print(M, K, N, flush=True)
        x, w, d = (torch.randint(-3, 4, s, generator=g).to(BF).to(cuda) for s in ((M, K), (N, K), (M, N)))
        v = dict(x=x, weight=w, bias=None, residual=None, dout=d)
        got = _run(v, "none")
        want = dict(out=x.double() @ w.double().T, dx=d.double() @ w.double(), dweight=d.double().T @ x.double())
        for k, t in want.items():
            assert torch.equal(got[k].double(), t.to(BF).double()), k


def test_strides_and_alignment(cuda):
    """Views: rows of a wider tensor, offsets of one element, transposed, expanded rows;
    batched inputs; the same values as the plain layout."""
    M, K, N = 150, 136, 72
    v = _inputs(M, K, N, "silu", BF, BF, True, seed=3, device=cuda)
    want = _want(v, "silu")

    def wide(t, off):
        w = torch.full((t.shape[0], t.shape[1] + 24), float("nan"), dtype=t.dtype, device=t.device)
        w[:, off:off + t.shape[1]] = t
        return w[:, off:off + t.shape[1]]

    for name, how in (("wide", lambda t: wide(t, 8)), ("offset", lambda t: wide(t, 1)),
                      ("transposed", lambda t: t.T.contiguous().T)):
        for keys in (("x",), ("weight",), ("residual",), ("dout",), ("x", "weight", "residual", "dout")):
            u = dict(v, **{k: how(v[k]) for k in keys})
            print(name, keys, flush=True)
            _check(_run(u, "silu"), want, f"{name} {keys}")
    u = dict(v, x=v["x"][:1].expand(M, K))
    _check(_run(u, "silu"), _want(u, "silu"), "expanded")
    batched = {k: t.reshape(3, 50, -1) if k in ("x", "residual", "dout") else t for k, t in v.items()}
    got = _run(batched, "silu")
    assert got["out"].shape == (3, 50, N) and got["dx"].shape == (3, 50, K)
    ref = _run(v, "silu")
    assert all(torch.equal(got[k].reshape(ref[k].shape), ref[k]) for k in ref)
    one = _run(dict(v, x=v["x"][0], residual=v["residual"][0], dout=v["dout"][0]), "silu")
    assert one["out"].shape == (N,)


def test_not_finite_values_stay_in_their_row(cuda):
    """Values that are not finite reach the outputs that depend on them alone, through tails
    of tiles and of the contraction too."""
    for M, K, N in ((20, 72, 40), (150, 331, 140), (600, 520, 300)):
        v = _inputs(M, K, N, "none", BF, None, False, seed=1, device=cuda)
        clean = _run(v, "none")
        u = dict(v, x=v["x"].clone(), weight=v["weight"].clone())
        u["x"][M - 1, K - 1] = float("nan")
        u["weight"][N - 1, 0] = float("inf")
        got = _run(u, "none", grads=False)["out"]
        assert torch.isnan(got[M - 1]).all() and not torch.isfinite(got[:, N - 1]).any()
        assert torch.equal(got[:M - 1, :N - 1], clean["out"][:M - 1, :N - 1])
        u = dict(v, dout=v["dout"].clone())
        u["dout"][0, N - 1] = float("nan")
        got = _run(u, "none")
        assert torch.isnan(got["dx"][0]).all() and torch.equal(got["dx"][1:], clean["dx"][1:])
        assert torch.isnan(got["dweight"][N - 1]).all() and torch.equal(got["dweight"][:N - 1], clean["dweight"][:N - 1])


def test_large_arguments_of_the_activations(cuda):
    """Far out an activation is 0 or the value itself, its gradient 0 or 1; no NaN."""
    z = torch.tensor([-3e4, -500.0, -90.0, -20.0, 20.0, 90.0, 500.0, 3e4])
    eye = torch.eye(8)
    for act in ("silu", "gelu"):
        for dtype in (BF, FP):
            v = dict(x=(z[:, None] * eye).to(dtype).to(cuda), weight=eye.to(dtype).to(cuda), bias=None, residual=None,
                     dout=torch.ones(8, 8, dtype=dtype, device=cuda))
            got = _run(v, act)
            o = got["out"].float().diagonal().cpu()
            assert torch.isfinite(got["out"]).all() and torch.isfinite(got["dx"]).all()
            assert torch.equal(o[4:], z[4:].to(dtype).float()) and (o[:3] == 0).all() and o[3].abs() < 1e-6
            d = got["dx"].float().diagonal().cpu()
            assert torch.equal(d[4:], torch.ones(4)) and d[:4].abs().max() < 1e-6


def test_empty_and_partial_gradients(cuda):
    v = _inputs(0, 40, 24, "swiglu", BF, BF, True, device=cuda)
    got = _run(v, "swiglu")
    assert got["out"].shape == (0, 24) and got["dx"].shape == (0, 40)
    assert not got["dweight"].any() and not got["dbias"].any()
    for act in ("none", "swiglu"):
        v = _inputs(130, 1000, 200, act, BF, F32, True, seed=7, device=cuda)
        ref = _run(v, act)
        for leaf in LEAVES:
            assert torch.equal(_run(v, act, leaves=(leaf,))["d" + leaf], ref["d" + leaf]), leaf
        for _ in range(2):
            again = _run(v, act)
            assert all(torch.equal(again[k], ref[k]) for k in ref)


def test_gradient_against_differences(cuda):
    """Central differences of the product itself along a random direction of the weight and
    the bias: fp16 outputs off by 2^-11 each, in quadrature, and the third-order term by
    halving the step."""
    for act in ("silu", "gelu", "swiglu"):
        v = _inputs(96, 64, 40, act, FP, F32, True, seed=2, device=cuda)
        got = _run(v, act)
        g = torch.Generator().manual_seed(1)
        for leaf, size in (("weight", 2.0 ** -5), ("bias", 2.0 ** -4)):
            # a step whose sums and halves are exact in the leaf's type
            step = (torch.randint(-2, 3, v[leaf].shape, generator=g) * size).to(v[leaf].dtype).to(cuda)
            base = (v[leaf] * 64).round() / 64
            u = dict(v, **{leaf: base})
            ana = (_run(u, act)["d" + leaf].double() * step.double()).sum()

            def diff(s):
                hi, lo = (_run(dict(u, **{leaf: base + t * step}), act, grads=False)["out"].double() for t in (s, -s))
                return ((hi - lo) * u["dout"].double()).sum() / (2 * s), hi

            (num, hi), (half, _) = diff(1.0), diff(0.5)
            noise = 4 * ((hi * 2.0 ** -11 * u["dout"].double()) ** 2).sum().sqrt()
            # dz and the gradient itself in fp16: 2^-11 each of terms added in quadrature
            own = 4 * 2.0 ** -11 * ((got["d" + leaf].double().abs() + 1) * step.double()).pow(2).sum().sqrt() * 8
            cubic = abs(float(num - half)) * 4 / 3 + 2 * float(noise)
            assert abs(float(num - ana)) <= float(noise + own) + cubic, (act, leaf, float(num), float(ana))


def test_other_stream_overlap_and_graph(cuda):
    a = _inputs(700, 1032, 640, "swiglu", BF, BF, True, seed=1, device=cuda)
    b = _inputs(40, 2048, 1000, "silu", FP, None, False, seed=2, device=cuda)
    ref_a, ref_b = _run(a, "swiglu"), _run(b, "silu")
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(4):
        with torch.cuda.stream(s1):
            x = _run(a, "swiglu")
        with torch.cuda.stream(s2):
            y = _run(b, "silu")
        torch.cuda.synchronize()
        assert all(torch.equal(x[k], ref_a[k]) for k in ref_a) and all(torch.equal(y[k], ref_b[k]) for k in ref_b)
    static = {k: t.clone() for k, t in a.items()}
    with torch.cuda.stream(s1):
        _run(static, "swiglu")
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s1):
        got = _run(static, "swiglu")
    for seed in (5, 6, 7):
        new = _inputs(700, 1032, 640, "swiglu", BF, BF, True, seed=seed, device=cuda)
        for k, t in new.items():
            static[k].copy_(t)
        graph.replay()
        torch.cuda.synchronize()
        want = _run(new, "swiglu")
        assert all(torch.equal(got[k], want[k]) for k in want)


def test_op_check_and_compile(cuda):
    for act in ("none", "swiglu"):
        v = _inputs(24, 40, 16, act, BF, F32, True, seed=4, device=cuda)
        args = [v[k].requires_grad_() for k in LEAVES]
        torch.library.opcheck(torch.ops.futudiffu_ii.fused_linear.default, (*args, act, True),
                              test_utils=("test_schema", "test_autograd_registration", "test_faketensor",
                                          "test_aot_dispatch_static"))
        import futudiffu_amd as F
        fn = torch.compile(lambda *a: F.fused_linear(*a, activation=act), backend="aot_eager", fullgraph=True)
        leaves = [v[k].detach().requires_grad_() for k in LEAVES]
        out = fn(*leaves)
        grads = torch.autograd.grad(out, leaves, v["dout"])
        want = _run(v, act)
        assert torch.equal(out, want["out"])
        assert all(torch.equal(t, want["d" + k]) for k, t in zip(LEAVES, grads))


def test_one_row_of_any_stride(cuda):
    """One row has no stride to speak of: a view whose row stride is beyond the limit."""
    g = torch.Generator().manual_seed(3)
    wide = torch.randn(1, (1 << 22) + 40, generator=g).to(BF).to(cuda)
    v = _inputs(1, 40, 24, "silu", BF, None, True, device=cuda)
    v["x"] = wide[:, 8:48]
    v["residual"] = wide[:, 64:88]
    v["dout"] = wide[:, 128:152]
    assert v["x"].stride(0) > 1 << 22
    _check(_run(v, "silu"), _want(v, "silu"))


def test_offsets_past_32_bits(cuda):
    """An x of more than 2^32 bytes, all zeros but a few rows: first, last and beyond 2^31 and
    2^32 bytes.  Small integers, so every sum is exact."""
    import futudiffu_amd as F
    K, M = 2048, (1 << 20) + 4100
    at = torch.tensor([0, 1, (1 << 19) - 1, 1 << 19, (1 << 20) - 1, 1 << 20, (1 << 20) + 5, M - 2, M - 1])
    g = torch.Generator().manual_seed(11)
    rows = torch.randint(-3, 4, (len(at), K), generator=g).to(BF)
    x = torch.zeros(M, K, dtype=BF, device=cuda)
    x[at.to(cuda)] = rows.to(cuda)
    for N in (24, 136):  # few columns, and tiles
        w = torch.randint(-2, 3, (N, K), generator=g).to(BF)
        d = torch.randint(-3, 4, (len(at), N), generator=g).to(BF)
        dout = torch.zeros(M, N, dtype=BF, device=cuda)
        dout[at.to(cuda)] = d.to(cuda)
        xg, wg = x.requires_grad_(), w.to(cuda).requires_grad_()
        out = F.fused_linear(xg, wg)
        want = torch.zeros(M, N, dtype=BF)
        want[at] = (rows.double() @ w.double().T).to(BF)
        assert torch.equal(out.detach().cpu(), want)
        dx, dw = torch.autograd.grad(out, (xg, wg), dout)
        assert torch.equal(dw.cpu(), (d.double().T @ rows.double()).to(BF))
        assert torch.equal(dx[at.to(cuda)].cpu(), (d.double() @ w.double()).to(BF))
        dx[at.to(cuda)] = 0
        assert dx.abs().amax().item() == 0
        del dx, out


@pytest.mark.parametrize("act", ["none", "swiglu"])
def test_gradients_are_not_differentiated(cuda, act):
    v = _inputs(5, 24, 16, act, BF, BF, True, device=cuda)
    import futudiffu_amd as F
    x = v["x"].requires_grad_()
    out = F.fused_linear(x, v["weight"], v["bias"], v["residual"], activation=act)
    with pytest.raises(RuntimeError, match="create_graph"):
        torch.autograd.grad(out, x, v["dout"], create_graph=True)


def test_residual_gradient_alone(cuda):
    v = _inputs(70, 24, 16, "gelu", BF, BF, True, device=cuda)
    got = _run(v, "gelu", leaves=("residual",))
    assert torch.equal(got["dresidual"], v["dout"])


@pytest.mark.parametrize("M,K,N", [(49, 72, 8200), (64, 136, 8184), (48, 1000, 9000), (33, 264, 40), (8300, 264, 50),
                                   (8100, 72, 64), (40, 4200, 17), (16, 5000, 300), (3, 328, 2000)])
def test_few_rows(cuda, M, K, N):
    """The few-row form's rings of stages (contractions that end in each of them, and one that
    every wave's first stage holds), its row counts and where tiles take over."""
    for i, (act, dtype, bias, res) in enumerate((("none", BF, BF, True), ("gelu", FP, F32, False),
                                                 ("swiglu", BF, BF, True))):
        print(M, K, N, act, flush=True)
        v = _inputs(M, K, N, act, dtype, bias, res, seed=M + K + i, device=cuda)
        got = _run(v, act, grads=False)
        _check(got, {"out": _want(v, act)["out"]}, act)


@pytest.mark.parametrize("act", ["silu", "gelu", "swiglu"])
def test_activations_over_the_whole_range(cuda, act):
    """To the largest finite value an activation is 0 or the value itself and its gradient 0 or 1,
    though squares and cubes on the way leave fp32's range."""
    z = torch.tensor([-3e38, -1e30, -1e20, -1e19, -1e13, 1e13, 1e19, 1e20, 1e30, 3e38])
    n = len(z)
    w = torch.eye(n)
    if act == "swiglu":  # z2 = 1 everywhere, from the bias
        w = torch.cat([w, torch.zeros(n, n)])
    bias = torch.cat([torch.zeros(n), torch.ones(n)]) if act == "swiglu" else None
    v = dict(x=torch.diag(z).to(BF).to(cuda), weight=w.to(BF).to(cuda), bias=None if bias is None else bias.to(cuda),
             residual=None, dout=torch.eye(n).to(BF).to(cuda))
    got = _run(v, act)
    o, d = got["out"].float().cpu(), got["dx"].float().cpu()
    assert torch.equal(o.diagonal(), z.clamp_min(0).to(BF).float())
    assert torch.isfinite(d).all() and torch.equal(d.diagonal(), (z > 0).float())


@pytest.mark.parametrize("M,K,N,act,dtype", [(333, 501, 389, "silu", FP), (331, 520, 777, "gelu", BF),
                                             (700, 264, 300, "swiglu", BF), (40, 72, 65, "swiglu", FP),
                                             (331, 520, 777, "none", BF)])
def test_gradients_have_one_rounding_more(cuda, M, K, N, act, dtype):
    """How far dx and dW are from the exact gradients, over all elements: their own rounding and
    that of dz = dout * act'(z) to the type, nothing else.  Both are computed in 64 bits.  32-bit
    sums add 2^-24 times the root of their terms (under 1600), under 2^-18 of a value, where a
    rounding is 2^-12 (fp16) or more, rms: under 2^-12 of it in quadrature.  A dz within that of a
    tie may round the other way, by as much.  1 % is allowed.  The bias's gradient adds dz
    unrounded: its own rounding alone."""
    v = _inputs(M, K, N, act, dtype, dtype, False, seed=M, device=cuda)
    got = _run(v, act)
    exact = {k: t[0] for k, t in _want(v, act).items()}
    x, w, d = (v[k].double() for k in ("x", "weight", "dout"))
    z = (x @ w.T + v["bias"].double()).requires_grad_()
    if act == "swiglu":
        y = torch.nn.functional.silu(z[:, :N]) * z[:, N:]
    else:
        y = {"none": lambda t: t, "silu": torch.nn.functional.silu,
             "gelu": lambda t: torch.nn.functional.gelu(t, approximate="tanh")}[act](z)
    dz, = torch.autograd.grad(y, z, d)
    rounded = dz.to(dtype).double()
    for k, t in (("dx", rounded @ w), ("dweight", rounded.T @ x), ("dbias", dz.sum(0))):
        want = float((t.to(dtype).double() - exact[k]).norm() / exact[k].norm())
        off = float((got[k].double() - exact[k]).norm() / exact[k].norm())
        print(act, dtype, k, f"{off:.4g} expected {want:.4g}", flush=True)
        assert off <= 1.01 * want, (k, off, want)
