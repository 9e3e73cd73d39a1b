"""GPU: MXFP4 (futudiffu_amd/mxfp4.py) against its 64-bit definition (oracle/mx_oracle.py).

Codes and scales bit for bit; the linear layer's output and gradients in units of what is
allowed: the bound on the matrix cores' sums and on the 16-bit dz, then one rounding."""

import pytest
import torch

from oracle import block_oracle as B
from oracle import mx_oracle as O

pytestmark = pytest.mark.gpu

BF, FP, F32 = torch.bfloat16, torch.float16, torch.float32
EPS = 1e-5


def _same(q, want, case=""):
    torch.cuda.synchronize()
    codes, scales = want
    assert q.codes.dtype == q.scales.dtype == torch.uint8
    assert torch.equal(q.scales, scales.to(q.scales.device)), f"{case}: scales"
    assert torch.equal(q.codes, codes.to(q.codes.device)), f"{case}: codes"


# ---------------------------------------------------------------- quantization

@pytest.mark.parametrize("M,K", [(1, 1), (1, 31), (1, 32), (3, 33), (5, 255), (7, 256), (16, 257), (17, 512), (33, 520),
                                 (2, 1001), (130, 3840), (4, 10240), (1000, 72), (15, 2056)])
def test_quantize(cuda, M, K):
    """Partly filled blocks, groups of 256 columns, shares of rows; padding is zeros; and back."""
    import futudiffu_amd as F
    g = torch.Generator().manual_seed(M + K)
    for dtype in (BF, FP):
        x = (torch.randn(M, K, generator=g) * torch.exp(2 * torch.randn(K, generator=g))).to(dtype)
        print(M, K, dtype, flush=True)
        want = O.quantize(x)
        q = F.mxfp4_quantize(x.to(cuda))
        _same(q, want, f"{M} {K} {dtype}")
        assert q.shape == x.shape
        for out in (BF, FP):
            back = F.mxfp4_dequantize(q, dtype=out)
            assert back.dtype == out and torch.equal(back.cpu(), O.dequantize(*want, K).to(out))


@pytest.mark.parametrize("dtype", [BF, FP])
def test_quantize_every_value(cuda, dtype):
    """Every finite 16-bit value as a block's largest, and beside larger ones: every tie, every scale,
    subnormals, the type's largest value."""
    import futudiffu_amd as F
    bits = torch.arange(1 << 16, dtype=torch.int32).to(torch.int16).view(dtype)
    v = bits[torch.isfinite(bits)]
    x = torch.zeros(v.numel(), 64, dtype=dtype)
    x[:, 7] = v
    x[:, 32 + 1] = v
    x[:, 32 + 30] = (v.double() * 1.75).clamp(-torch.finfo(dtype).max, torch.finfo(dtype).max).to(dtype)
    _same(F.mxfp4_quantize(x.to(cuda)), O.quantize(x))
    # against one large value: everything else lands on or between the small codes
    for top in (1.0, 1.5, 3.0, 5.0, 7.5):
        y = torch.full((v.numel() // 16 + 1, 32), top, dtype=dtype)
        small = v[v.abs() <= top]
        y.view(-1)[:small.numel()] = small
        _same(F.mxfp4_quantize(y.to(cuda)), O.quantize(y), top)


def test_quantize_what_is_not_finite(cuda):
    """NaN and infinities make their block NaN and no other; so they do in a product."""
    import futudiffu_amd as F
    g = torch.Generator().manual_seed(3)
    for dtype in (BF, FP):
        x = torch.randn(40, 300, generator=g).to(dtype)
        x[0, 0], x[3, 31], x[3, 32], x[7, 299], x[39, 64] = (float("nan"), float("inf"), -float("inf"), float("nan"),
                                                             -float("nan"))
        want = O.quantize(x)
        assert (want[1] == 255).sum() == 5
        q = F.mxfp4_quantize(x.to(cuda))
        _same(q, want)
        back = F.mxfp4_dequantize(q, dtype=dtype).double().cpu()
        assert torch.equal(back.isnan(), O.dequantize(*want, 300).isnan())
        assert torch.equal(back.nan_to_num(), O.dequantize(*want, 300).nan_to_num().to(dtype).double())


def test_quantize_shapes_and_strides(cuda):
    import futudiffu_amd as F
    g = torch.Generator().manual_seed(4)
    x = torch.randn(6, 50, 136, generator=g).to(BF).to(cuda)
    want = O.quantize(x.cpu())
    _same(F.mxfp4_quantize(x), want)
    wide = torch.full((6, 50, 160), float("nan"), dtype=BF, device=cuda)
    for off in (8, 1, 16):
        wide[..., off:off + 136] = x
        _same(F.mxfp4_quantize(wide[..., off:off + 136]), want, off)
    _same(F.mxfp4_quantize(x.transpose(0, 1).contiguous().transpose(0, 1)), want, "transposed")
    _same(F.mxfp4_quantize(x.transpose(1, 2).contiguous().transpose(1, 2)), want, "columns apart")
    _same(F.mxfp4_quantize(x[:, :1].expand(6, 50, 136)), O.quantize(x[:, :1].expand(6, 50, 136).cpu()), "expanded")
    one = F.mxfp4_quantize(x[0, 0])
    assert one.codes.shape == (128,) and F.mxfp4_dequantize(one).shape == (136,)
    for shape in ((0, 40), (3, 0, 40)):
        q = F.mxfp4_quantize(torch.empty(shape, dtype=BF, device=cuda))
        assert q.shape == shape and q.scales.shape == (1, 0, 8) and F.mxfp4_dequantize(q).shape == shape
    row = torch.randn(1, (1 << 22) + 40, generator=g).to(BF).to(cuda)[:, 8:48]  # one row has no stride to speak of
    _same(F.mxfp4_quantize(row), O.quantize(row.cpu()))
    # codes and scales of another alignment and order
    q = F.mxfp4_quantize(x[0])
    raw = torch.empty(q.codes.numel() + 1, dtype=torch.uint8, device=cuda)
    off = raw[1:].view(q.codes.shape)
    off.copy_(q.codes)
    sraw = torch.empty(q.scales.numel() + 1, dtype=torch.uint8, device=cuda)
    soff = sraw[1:].view(q.scales.shape)
    soff.copy_(q.scales)
    for codes, scales in ((off, soff), (q.codes.T.contiguous().T, q.scales.transpose(0, 1).contiguous().transpose(0, 1))):
        assert torch.equal(F.mxfp4_dequantize(F.MXFP4(codes, scales, 136)), F.mxfp4_dequantize(q))


# ---------------------------------------------------------------- linear

def _inputs(M, K, N, act, dtype=BF, bias=None, residual=False, seed=0, device="cpu"):
    import futudiffu_amd as F
    g = torch.Generator().manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=g)

    rows = 2 * N if act == "swiglu" else N
    v = dict(x=normal(M, K).to(dtype), bias=None if bias is None else (0.3 * normal(rows)).to(bias),
             residual=normal(M, N).to(dtype) if residual else None, dout=normal(M, N).to(dtype))
    v = {k: None if t is None else t.to(device) for k, t in v.items()}
    # channels of unlike size: scales that differ from block to block
    w = normal(rows, K) * torch.exp(normal(K)) / K ** 0.5
    codes, scales = O.quantize(w.to(BF))
    v["weight"] = F.MXFP4(codes.to(device), scales.to(device), K)
    v["values"] = O.dequantize(codes, scales, K).to(device)
    return v


LEAVES = ("x", "bias", "residual")


def _run(v, act, grads=True, leaves=None):
    import futudiffu_amd as F
    v = dict(v)
    leaves = [k for k in (leaves or LEAVES) if v[k] is not None] if grads else []
    for k in leaves:
        v[k] = v[k].detach().requires_grad_()
    out = F.mxfp4_linear(v["x"], v["weight"], v["bias"], v["residual"], activation=act)
    got = {"out": out.detach()}
    if grads:
        got.update(("d" + k, t) for k, t in zip(leaves, torch.autograd.grad(out, [v[k] for k in leaves], v["dout"])))
    return got


def _want(v, act, grads=True):
    return O.linear(v["x"], v["values"], v["bias"], v["residual"], act, v["dout"] if grads else None)


def _check(got, want, case=""):
    torch.cuda.synchronize()
    for name, g in got.items():
        exact, bound = want[name]
        w = B.worst(g, exact.to(g.device), bound.to(g.device))
        assert w <= 1.0, f"{case} {name}: {w:.3g} of what is allowed"


# single tokens, the few-row forms (16, 32, 48, 64 rows), tiles and their neighbours, odd widths,
# contractions under one stage of 256, of one and of many, with a ragged last one
SHAPES = [(1, 1, 1), (1, 256, 40), (2, 256, 1536), (7, 33, 19), (16, 64, 16), (17, 200, 130), (33, 264, 48), (48, 520, 40),
          (49, 1030, 24), (64, 3840, 24), (65, 8, 65), (70, 100, 9), (128, 256, 128), (129, 257, 257), (200, 136, 1000),
          (300, 16, 520), (256, 512, 256), (257, 1288, 264), (1000, 24, 16), (513, 1001, 779), (1, 10240, 384),
          (100, 2048, 100)]


@pytest.mark.parametrize("M,K,N", SHAPES)
def test_outputs_and_gradients(cuda, M, K, N):
    import futudiffu_amd as F
    for i, (act, dtype, bias, res) in enumerate((("none", BF, None, False), ("silu", FP, FP, True),
                                                 ("gelu", BF, F32, True), ("swiglu", BF, BF, True),
                                                 ("swiglu", FP, None, False))):
        print(M, K, N, act, dtype, bias, res, flush=True)
        v = _inputs(M, K, N, act, dtype, bias, res, seed=M + N + i, device=cuda)
        got = _run(v, act)
        _check(got, _want(v, act), f"{act} {dtype}")
        assert got["out"].dtype == got["dx"].dtype == dtype and (bias is None or got["dbias"].dtype == bias)
        plain = _run(v, act, grads=False)["out"]  # without gradients, and from codes: the same bits
        coded = F.mxfp4_linear(F.mxfp4_quantize(v["x"]), v["weight"], v["bias"], v["residual"], activation=act, dtype=dtype)
        for t in (plain, coded):
            assert torch.equal(t.view(torch.int16), got["out"].view(torch.int16))


@pytest.mark.parametrize("M,K,N,act", [(2300, 1536, 2048, "none"), (1280, 4096, 1536, "swiglu"),
                                       (4416, 1024, 3840, "gelu"), (300, 10240, 3840, "none"),
                                       (3071, 1000, 1004, "silu"), (700, 2600, 8200, "none")])
def test_large_products(cuda, M, K, N, act):
    """Whole rounds of tiles, and tiles cut along the contraction."""
    v = _inputs(M, K, N, act, BF, BF, True, seed=M, device=cuda)
    _check(_run(v, act), _want(v, act), act)


@pytest.mark.parametrize("M,K,N,acts", [
    # large tiles: with rows behind the last whole tile row, with the last round's tiles cut, with both
    (1110, 526, 7280, "swiglu"), (2229, 300, 7176, "none silu gelu"), (1536, 688, 12280, "none"),
    (6996, 578, 2352, "silu"), (4876, 300, 1728, "swiglu"),
    # in pieces of the contraction, and behind a whole round; several rounds
    (1609, 11030, 1216, "none gelu"), (700, 11030, 1400, "swiglu"), (9361, 3510, 1752, "none"),
    (1302, 300, 8960, "swiglu"), (1030, 300, 9576, "silu"),
    # tiles of half the size, one round and two
    (405, 524, 8520, "none silu gelu"), (137, 575, 8600, "swiglu"), (2319, 2091, 3208, "swiglu"),
    # small ones in pieces, rows of any alignment, two rounds
    (66, 4530, 6800, "none silu"), (65, 4937, 6667, "none gelu"), (97, 5792, 4371, "swiglu"),
    (102, 5196, 4416, "swiglu"), (813, 2875, 9571, "none"), (902, 300, 8387, "silu")])
def test_every_shape_of_tile(cuda, M, K, N, acts):
    for act in acts.split():
        for bias, residual in ((None, False), (F32, True)):
            print(M, K, N, act, bias, flush=True)
            v = _inputs(M, K, N, act, BF, bias, residual, seed=M + K, device=cuda)
            grads = act != "none" and residual  # z from every epilogue
            _check(_run(v, act, grads=grads, leaves=("bias",) if grads else None),
                   {k: t for k, t in _want(v, act, grads).items() if k in ("out", "dbias")}, act)
            del v


@pytest.mark.parametrize("M,K,N", [(5, 264, 136), (20, 1000, 1000), (40, 1000, 1000), (64, 600, 500), (200, 331, 140),
                                   (700, 520, 600), (2000, 72, 40), (1500, 2048, 1032), (300, 5000, 2000)])
def test_small_integers_are_exact(cuda, M, K, N):
    """Integers that the codes hold exactly, whatever the block's scale: every sum is exact, so a
    wrong element or scale or a lost or doubled product shows whatever the tolerance."""
    import futudiffu_amd as F
    g = torch.Generator().manual_seed(5 + M)
    held = torch.tensor([-6.0, -4, -3, -2, -1, 0, 0, 1, 2, 3, 4, 6])

    def ints(*shape, zoom=0):
        v = held[torch.randint(0, len(held), shape, generator=g)]
        v[:, :: 7] = v[:, :: 7].sign()
        v[:, 32:64] = v[:, 32:64].sign()  # a block of another scale
        return (v * 2.0 ** zoom).to(BF).to(cuda)

    x, w = ints(M, K), ints(N, K)
    assert torch.equal(O.rounded(x), x.double()) and torch.equal(O.rounded(w), w.double())
    d = torch.randint(-3, 4, (M, N), generator=g).to(BF).to(cuda)
    v = dict(x=x, weight=F.mxfp4_quantize(w), bias=None, residual=None, dout=d)
    got = _run(v, "none")
    assert torch.equal(got["out"].double(), (x.double() @ w.double().T).to(BF).double())
    assert torch.equal(got["dx"].double(), (d.double() @ w.double()).to(BF).double())
    got = _run(dict(v, x=ints(M, K, zoom=-60)), "none", grads=False)["out"]
    assert got.abs().max() < 2.0 ** -40


def test_strides_and_alignment(cuda):
    M, K, N = 150, 264, 72
    v = _inputs(M, K, N, "silu", BF, BF, True, seed=3, device=cuda)
    want = _want(v, "silu")

    def wide(t, off):
        w = torch.full((t.shape[0], t.shape[1] + 24), float("nan"), dtype=t.dtype, device=t.device)
        w[:, off:off + t.shape[1]] = t
        return w[:, off:off + t.shape[1]]

    for name, how in (("wide", lambda t: wide(t, 8)), ("offset", lambda t: wide(t, 1)),
                      ("transposed", lambda t: t.T.contiguous().T)):
        for keys in (("x",), ("residual",), ("dout",), ("x", "residual", "dout")):
            print(name, keys, flush=True)
            _check(_run(dict(v, **{k: how(v[k]) for k in keys}), "silu"), want, f"{name} {keys}")
    u = dict(v, x=v["x"][:1].expand(M, K))
    _check(_run(u, "silu"), _want(u, "silu"), "expanded")
    batched = {k: t.reshape(3, 50, -1) if k in ("x", "residual", "dout") else t for k, t in v.items()}
    got, ref = _run(batched, "silu"), _run(v, "silu")
    assert got["out"].shape == (3, 50, N) and got["dx"].shape == (3, 50, K)
    assert all(torch.equal(got[k].reshape(ref[k].shape), ref[k]) for k in ref)
    one = _run(dict(v, x=v["x"][0], residual=v["residual"][0], dout=v["dout"][0]), "silu")
    assert one["out"].shape == (N,)
    # some of a weight's rows: their codes in place, their scales a view
    w = v["weight"]
    part = w._replace(codes=w.codes[8:48], scales=w.scales[:, 8:48])
    u = dict(v, weight=part, values=v["values"][8:48], bias=v["bias"][8:48].contiguous(),
             residual=v["residual"][:, 8:48], dout=v["dout"][:, 8:48])
    _check(_run(u, "silu"), _want(u, "silu"), "rows")


@pytest.mark.parametrize("M,K,N", [(20, 264, 40), (150, 331, 140), (600, 520, 300)])
def test_not_finite_values_stay_in_their_row(cuda, M, K, N):
    """Through tails of tiles and of the contraction too; an x whose neighbouring rows end a tile."""
    v = _inputs(M, K, N, "none", BF, None, False, seed=1, device=cuda)
    clean = _run(v, "none")
    u = dict(v, x=v["x"].clone(), weight=v["weight"]._replace(scales=v["weight"].scales.clone()))
    u["x"][M - 1, K - 1] = float("nan")
    u["weight"].scales[0, N - 1, 0] = 255
    got = _run(u, "none", grads=False)["out"]
    assert torch.isnan(got[M - 1]).all() and torch.isnan(got[:, N - 1]).all()
    assert torch.equal(got[:M - 1, :N - 1], clean["out"][:M - 1, :N - 1])
    u = dict(v, dout=v["dout"].clone())
    u["dout"][0, N - 1] = float("nan")
    got = _run(u, "none")
    assert torch.isnan(got["dx"][0]).all() and torch.equal(got["dx"][1:], clean["dx"][1:])


@pytest.mark.parametrize("act", ["silu", "swiglu"])
def test_gradients_that_are_not_finite_stay_in_their_row(cuda, act):
    """NaN and infinities of dout through both parts of dz: an infinity is no NaN before it meets the weight."""
    v = _inputs(150, 264, 72, act, BF, F32, False, seed=1, device=cuda)
    v["weight"] = v["weight"]._replace(codes=v["weight"].codes & 0x77)  # no value is negative
    v["weight"].codes[0, 0] = 0x22
    u = dict(v, dout=v["dout"].abs())
    u["dout"][3, 7], u["dout"][5, 0] = float("nan"), float("inf")
    u["bias"] = v["bias"].abs() + 30.0  # act' and the gates are positive
    clean = _run(dict(u, dout=v["dout"].abs()), act)
    got = _run(u, act)
    assert torch.isnan(got["dx"][3]).all() and got["dx"][5, 0] == float("inf")
    keep = [i for i in range(150) if i not in (3, 5)]
    assert torch.equal(got["dx"][keep], clean["dx"][keep]) and torch.isfinite(clean["dx"]).all()
    assert torch.isnan(got["dbias"][7]) and got["dbias"][0] == float("inf")


def test_scales_of_the_whole_range(cuda):
    """The smallest and largest scales on both sides: their product, not the scales, has to fit."""
    import futudiffu_amd as F
    for M, N in ((4, 24), (100, 70)):
        x, w = torch.ones(M, 256, dtype=BF, device=cuda), torch.ones(N, 256, dtype=BF, device=cuda)
        for e in (-120, -60, 0, 60, 120):
            q = F.mxfp4_quantize(w * 2.0 ** -e)
            out = F.mxfp4_linear(x * 2.0 ** e, q)
            assert torch.equal(out, torch.full_like(out, 256.0)), e


def test_empty_and_partial_gradients(cuda):
    v = _inputs(0, 40, 24, "swiglu", BF, BF, True, device=cuda)
    got = _run(v, "swiglu")
    assert got["out"].shape == (0, 24) and got["dx"].shape == (0, 40) and not got["dbias"].any()
    for act in ("none", "swiglu"):
        v = _inputs(130, 1000, 200, act, BF, F32, True, seed=7, device=cuda)
        ref = _run(v, act)
        for leaf in LEAVES:
            assert torch.equal(_run(v, act, leaves=(leaf,))["d" + leaf], ref["d" + leaf]), leaf
        for _ in range(2):
            again = _run(v, act)
            assert all(torch.equal(again[k], ref[k]) for k in ref)


def test_gradient_against_differences(cuda):
    """Steps that the codes hold exactly: the output is the exact function of them, and central
    differences of it in 64 bits' sums give the gradient up to the outputs' and dz's roundings
    (2^-11 of each in fp16, independent) and the third-order term, told by halving the step."""
    g = torch.Generator().manual_seed(6)
    for act in ("none", "silu", "swiglu"):
        v = _inputs(40, 64, 24, act, FP, F32, True, seed=2, device=cuda)
        x = torch.randint(-1, 2, (40, 64), generator=g).double()
        x[:, ::32] = 4.0  # the scale stays 1
        step = torch.randint(-1, 2, (40, 64), generator=g).double() * 0.5
        step[:, ::32] = 0.0
        v["x"] = (x / 4).to(FP).to(cuda)
        s = (step / 4).to(FP).to(cuda)
        ana = (_run(v, act)["dx"].double() * s.double()).sum()

        def diff(t):
            hi, lo = (_run(dict(v, x=v["x"] + k * s), act, grads=False)["out"].double() for k in (t, -t))
            return ((hi - lo) * v["dout"].double()).sum() / (2 * t), hi

        num, hi = diff(1)
        noise = 4 * ((hi.abs() + 1) * 2.0 ** -11 * v["dout"].double()).pow(2).sum().sqrt()
        # the third derivative of an activation is at most 1.2 of its scale: half a step h changes z by dz = W h
        dz = (s.double() @ v["values"].T).abs()
        if act == "swiglu":
            d1, d2 = dz.chunk(2, -1)
            curve = (d1 ** 3 * 4 + 3 * d1 ** 2 * d2) / 6
        else:
            curve = dz ** 3 * (0.0 if act == "none" else 1.2) / 6
        cubic = (curve * v["dout"].double().abs()).sum()
        own = 8 * 2.0 ** -11 * (v["dout"].double().abs() @ v["values"][:24].abs() * s.double().abs()).pow(2).sum().sqrt()
        assert abs(float(num - ana)) <= float(noise + own + cubic), (act, float(num), float(ana))


@pytest.mark.parametrize("M,K,N,act,dtype", [(667, 1001, 779, "silu", FP), (331, 520, 777, "gelu", BF),
                                             (700, 264, 300, "swiglu", BF), (40, 72, 65, "swiglu", FP),
                                             (1300, 700, 5000, "silu", BF), (64, 1032, 4100, "swiglu", FP),
                                             # large tiles, whole and in pieces, with rows of any alignment too
                                             (4200, 4100, 320, "silu", FP), (2304, 4096, 600, "gelu", FP),
                                             (2304, 4095, 2000, "gelu", FP), (1, 520, 72, "swiglu", FP)])
def test_dx_has_its_own_rounding_alone(cuda, M, K, N, act, dtype):
    """How far dx is from the exact gradient, over all elements, against the exact values rounded
    to its type: what enters the product loses 2^-17 of a value or less, beside the 2^-12 (rms, of fp16)
    of the rounding under 2^-10 of it in quadrature; 32-bit sums of up to 10000 terms, and z's, under
    2^-16 of a value, 2^-8 of it in quadrature; 1 % is allowed.  A dz rounded to 16 bits would add 40 %."""
    v = _inputs(M, K, N, act, dtype, dtype, False, seed=M, device=cuda)
    got, exact = _run(v, act)["dx"].double(), _want(v, act)["dx"][0]
    want = float((exact.to(dtype).double() - exact).norm() / exact.norm())
    off = float((got - exact).norm() / exact.norm())
    print(act, dtype, f"{off:.4g} expected {want:.4g}", flush=True)
    assert off <= 1.01 * want, (off, want)


@pytest.mark.parametrize("dtype", [BF, FP])
def test_dz_past_the_types_range(cuda, dtype):
    """dout * act'(z) past fp16's largest value and under its smallest, beside a weight that brings dx back
    into the range: dx is the exact gradient's, rounded once."""
    # dz around 2^20 over a weight around 2^-16, and around 2^-23 over one around 2^8
    for zoom, up, thin, gate in ((-12, 2.0 ** 9, 1.0, 1000.0), (12, 2.0 ** -20, 2.0 ** -14, 0.0)):
        v = _inputs(150, 264, 72, "swiglu", dtype, F32, False, seed=3, device=cuda)
        w = v["weight"]
        scales = (w.scales.int() + zoom).clamp_min(0).to(torch.uint8)
        v.update(weight=w._replace(scales=scales), values=O.dequantize(w.codes, scales, w.columns),
                 x=v["x"] * thin, dout=v["dout"] * up)
        v["bias"][72:] = v["bias"][72:] * 2.0 ** -6 + gate
        _check(_run(v, "swiglu"), _want(v, "swiglu"), f"{dtype} {zoom}")


def _differences(act, call, grads, v, steps):
    """For the leaves of `steps`: the directional derivative from call's outputs by central differences of a
    whole and a half step, extrapolated ((4 d(1/2) - d(1)) / 3), that from grads, and how far they may
    be apart: the outputs' roundings (half a step of fp16, and MFMA of the product's size through the
    slopes) and the gradients' in quadrature, six times, and what the extrapolation leaves in 64 bits."""
    d, w, want = v["dout"].double(), v["values"], _want(v, act)

    def slope(value):
        one, half = (value(t) - value(-t) for t in (1, 0.5))
        return float((4 * half - one / 2) / 3)

    q = O.rounded(v["x"])
    more = 1.13 * O.MFMA * (q.abs() @ w.abs().T)
    if act == "swiglu":
        z1, z2 = (q @ w.T + v["bias"].double()).abs().chunk(2, -1)
        more = more.chunk(2, -1)[0] * z2 + more.chunk(2, -1)[1] * z1
    # a half step's pair of outputs enters 4 / 3 times each, a whole step's 1 / 6
    out = (((want["out"][0].abs() + 1) * 2.0 ** -11 + more) * d).norm() * (2 * (16 + 1 / 4) / 9) ** 0.5
    found = []
    for leaf, s in steps.items():
        moved = lambda t: {**v, leaf: v[leaf] + t * s}  # noqa: E731
        num = slope(lambda t: (call(moved(t)).double() * d).sum())
        ana = float((grads[leaf].double() * s.double()).sum())
        left = slope(lambda t: (_want(moved(t), act, False)["out"][0] * d).sum()) - float((want["d" + leaf][0] * s.double()).sum())
        own = (grads[leaf].double() * torch.finfo(grads[leaf].dtype).eps / 2 * s.double()).norm()
        found.append((leaf, num, ana, abs(left) + 6 * float(out + own)))
    return found


def _difference_inputs(act, device):
    """x and its steps, whole and halved, are multiples that the codes hold exactly; the steps go up the
    gradient in a few columns of each row, so that the derivative stands far above the roundings."""
    v = _inputs(40, 64, 24, act, FP, F32, False, seed=2, device=device)
    g = torch.Generator().manual_seed(6)
    x = torch.randint(-1, 2, (40, 64), generator=g).double()
    x[:, ::32] = 4.0  # the scale stays 1
    v["x"] = (x / 4).to(FP).to(device)
    want = _want(v, act)
    pick = torch.rand(40, 64, generator=g) < 0.15
    pick[:, ::32] = False
    steps = {"x": (want["dx"][0].sign() * pick.to(device) / 4).to(FP), "bias": (want["dbias"][0].sign() / 4).float()}
    for t in (1, -1, 0.5, -0.5):
        moved = v["x"] + t * steps["x"]
        assert torch.equal(O.rounded(moved), moved.double())
    return v, steps


@pytest.mark.parametrize("act", ["none", "silu", "gelu", "swiglu"])
def test_gradient_against_extrapolated_differences(cuda, act):
    """The gradients of x and the bias against differences of the outputs; what is allowed is a small
    part of the derivative, so a gradient that lacks a factor, a term or half of a swiglu fails."""
    v, steps = _difference_inputs(act, cuda)
    got = _run(v, act)
    call = lambda v: _run(v, act, grads=False)["out"]  # noqa: E731
    for leaf, num, ana, allowed in _differences(act, call, {"x": got["dx"], "bias": got["dbias"]}, v, steps):
        print(act, leaf, num, ana, allowed, flush=True)
        assert allowed < 0.02 * abs(ana) and abs(num - ana) <= allowed, (act, leaf, num, ana, allowed)


@pytest.mark.parametrize("act", ["none", "silu"])
def test_fp16_over_weights_past_its_range(cuda, act):
    """Blocks of a weight with scales from 2^-60 to 2^30 under an fp16 x, its columns sized so that the outputs
    fit: the forward takes every code as it is.  So does the gradient of an activation; without one
    dx takes the weight's values in fp16, infinite past 65504, in steps of 2^-24 under 2^-14, 0 where
    they are smaller."""
    M, K, N = 70, 352, 40
    v = _inputs(M, K, N, act, FP, F32, False, seed=8, device=cuda)
    w = v["weight"]
    zoom = torch.tensor([0, -60, 14, -14, -18, -22, -25, 20, 30, 2, 0], device=cuda)  # of each block of 32 columns
    scales = w.scales.transpose(0, 1).reshape(N, -1).int()
    scales[:, :11] = (scales[:, :11] + zoom).clamp(0, 254)
    scales = scales.to(torch.uint8).reshape(N, 2, 8).transpose(0, 1).contiguous()
    v.update(weight=w._replace(scales=scales), values=O.dequantize(w.codes, scales, K),
             x=(v["x"].float() * torch.exp2(-zoom.clamp_min(0).float()).repeat_interleave(32)).to(FP))
    if act != "none":
        v["dout"] = v["dout"] * 2.0 ** -20  # the largest block's dx fits
    got, want = _run(v, act), _want(v, act)
    in_fp16 = v["values"].to(FP).double()
    past = in_fp16.isinf().any(0)
    assert past.any() and ((in_fp16 != v["values"]) & ~in_fp16.isinf()).any() and torch.isfinite(got["out"]).all()
    if act == "none":
        assert not torch.isfinite(got["dx"][:, past]).any()
        d, used = v["dout"].double(), in_fp16[:, ~past]
        exact = d @ used
        exact = torch.where(exact.abs() >= 65520, exact.sign() * torch.inf, exact)  # what fp16 rounds to infinity
        want["dx"] = (exact, (N + 2) * 2.0 ** -24 * (d.abs() @ used.abs()))
        got["dx"] = got["dx"][:, ~past]
    _check(got, want, act)


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
    for M in (700, 20):
        static = _inputs(M, 1032, 640, "swiglu", BF, BF, True, seed=3, device=cuda)
        with torch.cuda.stream(s1):
            _run(static, "swiglu")
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s1):
            got = _run(static, "swiglu")
        for seed in (5, 6, 7):
            new = _inputs(M, 1032, 640, "swiglu", BF, BF, True, seed=seed, device=cuda)
            for k in ("x", "bias", "residual", "dout"):
                static[k].copy_(new[k])
            static["weight"].codes.copy_(new["weight"].codes)
            static["weight"].scales.copy_(new["weight"].scales)
            graph.replay()
            torch.cuda.synchronize()
            want = _run(new, "swiglu")
            assert all(torch.equal(got[k], want[k]) for k in want)


def test_graphs_of_one_pool_and_streams(cuda):
    """Products in pieces, of half tiles and of rows that they quantize themselves: two graphs whose workspaces lie in
    one pool replayed in turn on changing inputs, and eager calls on two streams at once."""
    import futudiffu_amd as F
    sizes = ((1609, 11030, 1216, "none"), (66, 4530, 6800, "silu"), (405, 524, 8520, "gelu"), (2, 264, 8208, "none"),
             (3, 1000, 48, "swiglu"), (200, 5000, 2000, "none"))

    def inputs(seed):
        return [_inputs(M, K, N, act, BF, F32, True, seed=seed + i, device=cuda)
                for i, (M, K, N, act) in enumerate(sizes)]

    def run(vs):
        return [F.mxfp4_linear(v["x"], v["weight"], v["bias"], v["residual"], activation=s[3]) for v, s in zip(vs, sizes)]

    statics, graphs, outs, pool = [inputs(0), inputs(10)], [], [], None
    for static in statics:
        run(static)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, pool=pool):
            outs.append(run(static))
        pool = graph.pool()
        graphs.append(graph)
    for turn in range(3):
        for i in (0, 1):
            new = inputs(100 * (turn + 1) + 10 * i)
            for old, v in zip(statics[i], new):
                for k in ("x", "bias", "residual"):
                    old[k].copy_(v[k])
                old["weight"].codes.copy_(v["weight"].codes)
                old["weight"].scales.copy_(v["weight"].scales)
            graphs[i].replay()
            torch.cuda.synchronize()
            assert _equal(outs[i], run(new)), (turn, i)
    want = [run(v) for v in statics]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(3):
        got = []
        for v, stream in zip(statics, streams):
            with torch.cuda.stream(stream):
                got.append(run(v))
        assert all(_equal(g, w) for g, w in zip(got, want))


def test_offsets_past_32_bits(cuda):
    """An x, and a dequantized tensor, of more than 2^32 bytes, all zeros but a few rows.  Small
    integers, so every sum is exact."""
    import futudiffu_amd as F
    K, M = 2048, (1 << 20) + 4100
    at = torch.tensor([0, 1, (1 << 19) - 1, 1 << 19, (1 << 20) - 1, 1 << 20, (1 << 20) + 5, M - 2, M - 1])
    g = torch.Generator().manual_seed(11)
    held = torch.tensor([-6.0, -4, -3, -2, -1, 0, 1, 2, 3, 4, 6])
    rows = held[torch.randint(0, 11, (len(at), K), generator=g)].to(BF)
    x = torch.zeros(M, K, dtype=BF, device=cuda)
    x[at.to(cuda)] = rows.to(cuda)
    q = F.mxfp4_quantize(x)
    back = F.mxfp4_dequantize(q)
    assert torch.equal(back[at.to(cuda)].cpu(), rows)
    back[at.to(cuda)] = 0
    assert back.abs().amax().item() == 0
    del back
    for N in (24, 136):
        w = held[torch.randint(0, 11, (N, K), generator=g)].to(BF)
        out = F.mxfp4_linear(x, F.mxfp4_quantize(w.to(cuda)))
        want = torch.zeros(M, N, dtype=BF)
        want[at] = (rows.double() @ w.double().T).to(BF)
        assert torch.equal(out.cpu(), want)
        assert torch.equal(F.mxfp4_linear(q, F.mxfp4_quantize(w.to(cuda))), out)


def test_gradients_past_32_bits(cuda):
    """An activation's dz of more than 2^32 bytes in each of its parts: few rows of dout are not zero."""
    import futudiffu_amd as F
    M, K, N = (1 << 20) + 37, 24, 2056
    v = _inputs(9, K, N, "silu", BF, None, False, seed=6, device=cuda)
    at = torch.tensor([0, 1, (1 << 19) - 1, 1 << 19, (1 << 20) - 1, 1 << 20, (1 << 20) + 5, M - 2, M - 1], device=cuda)
    x, d = torch.zeros(M, K, dtype=BF, device=cuda), torch.zeros(M, N, dtype=BF, device=cuda)
    x[at], d[at] = v["x"], v["dout"]
    x.requires_grad_()
    dx, = torch.autograd.grad(F.mxfp4_linear(x, v["weight"], activation="silu"), x, d)
    _check({"dx": dx[at]}, _want(v, "silu"))
    dx[at] = 0
    assert not dx.any()


@pytest.mark.parametrize("M,K,N", [(49, 264, 8200), (64, 520, 8184), (48, 1000, 9000), (33, 264, 40), (1, 5000, 15360),
                                   (16, 5000, 300), (3, 1300, 2000), (32, 10240, 100), (8, 2304, 4096)])
def test_few_rows(cuda, M, K, N):
    """The few-row form's rings of stages (contractions that end in each of them, and one that
    every wave's first stage holds), its row counts and where tiles take over."""
    for i, (act, dtype, bias, res) in enumerate((("none", BF, BF, True), ("gelu", FP, F32, False),
                                                 ("swiglu", BF, BF, True))):
        print(M, K, N, act, flush=True)
        v = _inputs(M, K, N, act, dtype, bias, res, seed=M + K + i, device=cuda)
        _check(_run(v, act, grads=False), {"out": _want(v, act, False)["out"]}, act)


@pytest.mark.parametrize("K,N", [(8, 5), (264, 40), (1000, 8192), (1000, 8208), (3840, 500), (4096, 48), (4104, 48),
                                 (333, 48)])
def test_few_rows_quantize_in_place(cuda, K, N):
    """Up to four rows are quantized by the product itself, where they are aligned and short: the
    bits of codes that were made before, whatever the rows hold and however they lie."""
    import futudiffu_amd as F
    for M in (1, 2, 3, 4, 5):
        for act, dtype in (("none", BF), ("swiglu", FP)):
            print(K, N, M, act, flush=True)
            v = _inputs(M, K, N, act, dtype, F32, True, seed=K + M, device=cuda)
            x = v["x"]
            x[M - 1, K - 1] = float("inf")
            x[M // 2, : K // 2] = 0.0
            if M > 1:
                x[0] *= 2.0 ** -14
            x[M - 1, : K // 3] *= 2.0 ** 9
            spread = torch.full((M, K + 16), float("nan"), dtype=dtype, device=cuda)
            spread[:, 8:K + 8] = x
            off = torch.cat([x.new_zeros(1), x.flatten()])[1:].view(M, K)  # two bytes off a boundary of 16
            for name, rows in (("rows", x), ("spread", spread[:, 8:K + 8]), ("columns", x.T.contiguous().T), ("off", off),
                               ("one", x[M - 1:].expand(M, K))):
                args = (v["weight"], v["bias"], v["residual"])
                got = F.mxfp4_linear(rows, *args, activation=act)
                want = F.mxfp4_linear(F.mxfp4_quantize(rows), *args, activation=act, dtype=dtype)
                assert torch.equal(got.view(torch.int16), want.view(torch.int16)), name
            _check({"out": F.mxfp4_linear(x, *args, activation=act)}, {"out": _want(v, act, False)["out"]}, act)


def test_rows_that_lie_backwards(cuda):
    """By the C entry: x's rows at a negative stride, the last one first in memory."""
    from futudiffu_amd import _lib
    import futudiffu_amd as F
    lib = _lib.load()
    M, K, N = 4, 264, 48
    v = _inputs(M, K, N, "none", BF, None, False, seed=4, device=cuda)
    back = v["x"].flip(0).contiguous()
    want = F.mxfp4_linear(v["x"], v["weight"])
    out = torch.empty(M, N, dtype=BF, device=cuda)
    size = lib.sage_mxfp4_linear_workspace_bytes(M, N, K, 0, 1, 0)
    ws = torch.empty(size, dtype=torch.uint8, device=cuda)
    status = lib.sage_mxfp4_linear(back[M - 1:].data_ptr(), -K, None, None, v["weight"].codes.data_ptr(),
                                   v["weight"].scales.data_ptr(), None, 0, None, 0, M, N, K, 0, 0, ws.data_ptr(), size, None,
                                   out.data_ptr(), torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    assert status == 0 and torch.equal(out, want)


@pytest.mark.parametrize("M,K,N", [(667, 1001, 779), (2000, 3840, 16), (7000, 264, 24), (192, 1536, 3840), (1025, 72, 8),
                                   (97, 776, 8300)])
def test_few_columns(cuda, M, K, N):
    """The few-row form in several groups of 64 rows (of 32 for a swiglu), the last one partly filled."""
    for i, (act, dtype, bias, res) in enumerate((("none", FP, F32, True), ("silu", BF, None, False),
                                                 ("swiglu", BF, BF, True))):
        print(M, K, N, act, flush=True)
        v = _inputs(M, K, N, act, dtype, bias, res, seed=M + K + i, device=cuda)
        _check(_run(v, act), _want(v, act), act)


# ---------------------------------------------------------------- norms

def _ids(lengths, n, batch):
    ids = torch.full((batch, n), -1, dtype=torch.int32)
    for b in range(batch):
        at = 0
        for i, x in enumerate(lengths):
            ids[b, at:at + x] = (i + b) % len(lengths)
            at += x
    return ids


def _norm_inputs(Bn, N, C, dtype, params, docs=None, seed=0):
    g = torch.Generator().manual_seed(seed)

    def normal(*shape, to=dtype, s=1.0, o=0.0):
        return (o + s * torch.randn(*shape, generator=g)).to(to)

    rows = (Bn, C) if docs is None else (Bn, docs[0], C)
    return dict(residual=normal(Bn, N, C, s=2.0), x=normal(Bn, N, C, s=1.5), weight=normal(C, to=params, s=0.3, o=1.0),
                cond=normal(*rows, to=params, s=0.5), next_weight=normal(C, to=params, s=0.3, o=1.0),
                next_scale=normal(*rows, to=params, s=0.5), doc_ids=None if docs is None else docs[1])


def _norm_check(v, eps=EPS, case=""):
    """Both norms of the inputs on their device: codes and scales bit for bit, hidden within one
    rounding."""
    import futudiffu_amd as F
    q = F.rms_norm_modulate_mxfp4(v["x"], v["weight"], v["cond"], doc_ids=v["doc_ids"], eps=eps)
    y = O.norm_values(v["x"], v["weight"], v["cond"], v["doc_ids"], eps)
    _same(q, O.quantize(y), f"{case} modulate")
    hidden, q = F.rms_norm_gate_residual_modulate_mxfp4(
        v["residual"], v["x"], v["weight"], v["cond"], v["next_weight"], v["next_scale"], doc_ids=v["doc_ids"], eps=eps)
    h, y = O.norm_values(v["x"], v["weight"], v["cond"], v["doc_ids"], eps, v["residual"], v["next_weight"], v["next_scale"])
    _same(q, O.quantize(y), f"{case} gate modulate")
    assert torch.equal(hidden, h.float().to(hidden.dtype)) or B.worst(hidden, h, 2.0 ** -40 * h.abs()) <= 1.0
    return hidden, q


@pytest.mark.parametrize("Bn,N,C", [(1, 1, 8), (1, 1, 1), (2, 3, 7), (1, 33, 64), (3, 17, 1000), (1, 65, 1001),
                                    (2, 130, 1024), (1, 9, 1032), (2, 40, 3840), (1, 31, 3841), (1, 5, 4104), (1, 19, 8192),
                                    (2, 3, 8191), (1, 700, 72)])
def test_norms(cuda, Bn, N, C):
    for dtype, params in ((BF, BF), (FP, F32)):
        print(Bn, N, C, dtype, params, flush=True)
        v = _norm_inputs(Bn, N, C, dtype, params, seed=N + C)
        _norm_check({k: None if t is None else t.to(cuda) for k, t in v.items()}, case=f"{Bn} {N} {C} {dtype}")


def test_norms_of_documents(cuda):
    """Rows of documents; tokens of none have scale 0, and behind a gate their x is not read: it may
    hold anything."""
    for C, dtype, params in ((72, BF, F32), (1001, FP, FP), (3840, BF, BF)):
        ids = _ids([30, 1, 0, 25], 64, 2)
        ids[1, 3] = 99
        v = _norm_inputs(2, 64, C, dtype, params, (4, ids), seed=C)
        v = {k: t.to(cuda) for k, t in v.items()}
        hidden, q = _norm_check(v, case=f"{C}")
        dead = (v["doc_ids"] < 0) | (v["doc_ids"] >= 4)
        u = dict(v, x=v["x"].masked_fill(dead[..., None], float("nan")))
        import futudiffu_amd as F
        h2, q2 = F.rms_norm_gate_residual_modulate_mxfp4(u["residual"], u["x"], u["weight"], u["cond"], u["next_weight"],
                                                         u["next_scale"], doc_ids=u["doc_ids"], eps=EPS)
        assert torch.equal(h2, hidden) and torch.equal(q2.codes, q.codes) and torch.equal(q2.scales, q.scales)


def test_norms_plain_and_strided(cuda):
    import futudiffu_amd as F
    v = {k: None if t is None else t.to(cuda) for k, t in _norm_inputs(2, 20, 264, BF, BF, seed=1).items()}
    for drop in ("weight", "cond", "next_weight", "next_scale"):
        _norm_check(dict(v, **{drop: None}), case=drop)
    _norm_check(dict(v, weight=None, cond=None, next_weight=None, next_scale=None), eps=0.0)
    want = _norm_check(v)
    wide = torch.full((2, 20, 300), float("nan"), dtype=BF, device=cuda)
    for off in (1, 8):
        wide[..., off:off + 264] = v["x"]
        got = _norm_check(dict(v, x=wide[..., off:off + 264]), case=off)
        assert torch.equal(got[1].codes, want[1].codes)
    _norm_check(dict(v, x=v["x"].transpose(0, 1).contiguous().transpose(0, 1),
                     residual=v["residual"].transpose(1, 2).contiguous().transpose(1, 2)), case="transposed")
    q = F.rms_norm_modulate_mxfp4(v["x"][0], v["weight"])
    _same(q, O.quantize(O.norm_values(v["x"][:1], v["weight"], None, None, EPS)[0]))
    assert F.rms_norm_modulate_mxfp4(torch.empty(2, 0, 40, dtype=BF, device=cuda)).shape == (2, 0, 40)
    h, q = F.rms_norm_gate_residual_modulate_mxfp4(*(torch.empty(0, 3, 40, dtype=BF, device=cuda),) * 2)
    assert h.shape == q.shape == (0, 3, 40)


def test_norms_of_rows_that_are_not_finite(cuda):
    """NaN and infinities stay in their token; rows of zeros and of one value."""
    import futudiffu_amd as F
    v = {k: None if t is None else t.to(cuda) for k, t in _norm_inputs(1, 12, 520, BF, BF, seed=2).items()}
    clean = F.rms_norm_modulate_mxfp4(v["x"], v["weight"], v["cond"])
    x = v["x"].clone()
    x[0, 2, 5], x[0, 4, 519], x[0, 6], x[0, 8] = float("nan"), float("inf"), 0.0, 2.0 ** 100
    q = F.rms_norm_modulate_mxfp4(x, v["weight"], v["cond"])
    keep = [i for i in range(12) if i not in (2, 4, 6, 8)]
    assert torch.equal(q.codes[:, keep], clean.codes[:, keep]) and torch.equal(q.scales[:, keep], clean.scales[:, keep])
    back = F.mxfp4_dequantize(q)
    assert back[0, 2].isnan().all() and back[0, 4, 512:].isnan().all() and not back[0, 6].any()
    assert torch.isfinite(back[0, 8]).all()
    _same(q._replace(codes=q.codes[:, [6, 8]], scales=q.scales[:, [6, 8]]),
          O.quantize(O.norm_values(x[:, [6, 8]], v["weight"], v["cond"], None, EPS)))
    r = v["residual"].clone()
    r[0, 3, 7] = float("inf")
    hidden, q = F.rms_norm_gate_residual_modulate_mxfp4(r, v["x"], v["weight"])
    assert hidden[0, 3, 7] == float("inf") and torch.isfinite(hidden).sum() == hidden.numel() - 1


def test_norms_of_extreme_sizes(cuda):
    """Parameters and rows where fp32 leaves its range or keeps few bits of a value: codes as ever."""
    v = {k: None if t is None else t.to(cuda) for k, t in _norm_inputs(2, 9, 520, BF, F32, seed=4).items()}
    big, small = 2.0 ** 100, 2.0 ** -100

    def like(t, value):
        return torch.full_like(t, value)

    some = torch.arange(520, device=cuda) % 3 == 0
    cases = dict(
        heavy=dict(weight=v["weight"] * big, next_weight=v["next_weight"] * big),
        light=dict(weight=v["weight"] * small, next_weight=v["next_weight"] * small),
        faint=dict(weight=v["weight"] * 2.0 ** -140, next_weight=v["next_weight"] * 2.0 ** -140),
        mixed=dict(weight=torch.where(some, v["weight"] * big, v["weight"] * small),
                   next_weight=torch.where(some, v["next_weight"] * big, v["next_weight"] * small)),
        none=dict(cond=like(v["cond"], -1.0), next_scale=like(v["next_scale"], -1.0)),
        hardly=dict(cond=like(v["cond"], -1.0 + 2.0 ** -20), next_scale=like(v["next_scale"], -1.0 + 2.0 ** -20)),
        opposed=dict(cond=v["cond"] * big, next_scale=v["next_scale"] * big, weight=v["weight"] * small,
                     next_weight=v["next_weight"] * small),
        vanishing=dict(cond=v["cond"] * 2.0 ** -140, weight=v["weight"] * 2.0 ** -40, residual=like(v["residual"], 0.0)),
        nothing=dict(cond=like(v["cond"], 0.0), residual=like(v["residual"], 0.0)))
    for name, change in cases.items():
        for eps in (EPS, 1e-30, 1e20):
            print(name, eps, flush=True)
            _norm_check(dict(v, **change), eps=eps, case=f"{name} {eps}")
    for scale in (2.0 ** 120, 2.0 ** 60, 2.0 ** -60, 2.0 ** -126, 2.0 ** -132):
        for eps in (EPS, 0.0):
            print(scale, eps, flush=True)
            _norm_check(dict(v, x=v["x"] * scale, residual=v["residual"] * scale), eps=eps, case=f"{scale} {eps}")
    for bad in (float("nan"), float("inf")):
        for key in ("weight", "next_weight", "cond", "next_scale"):
            t = v[key].clone()
            t[..., 77] = bad
            y = _norm_codes(dict(v, **{key: t}))
            for q, want in y:
                _same(q, O.quantize(want), f"{bad} {key}")


def test_norms_past_the_range_of_fp32(cuda):
    """Values of 2^128 and more, which a block's scale can hold up to 6 x 2^127 and which are the code of 6
    past that; beside blocks that fp32 holds, and beside an infinity."""
    import futudiffu_amd as F
    for C in (520, 1001, 3840):
        v = {k: None if t is None else t.to(cuda) for k, t in _norm_inputs(2, 9, C, BF, F32, seed=5).items()}
        few = torch.arange(C, device=cuda) // 32 % 3 == 0
        top = 0
        for zoom in (-4, -2, -1, 0, 1, 2, 3, 9, 30, 100):
            for part in (torch.ones_like(few), few):
                print(C, zoom, bool(part.all()), flush=True)
                w = torch.where(part, v["weight"] * 2.0 ** 126, v["weight"])
                w2 = torch.where(part, v["next_weight"] * 2.0 ** 126, v["next_weight"])
                u = dict(v, weight=w, next_weight=w2, cond=v["cond"] * 2.0 ** zoom, next_scale=v["next_scale"] * 2.0 ** zoom)
                got = F.rms_norm_modulate_mxfp4(u["x"], w, u["cond"], eps=EPS)
                _same(got, O.quantize(O.norm_values(u["x"], w, u["cond"], None, EPS)), zoom)
                h, y = O.norm_values(u["x"], v["weight"], v["cond"], None, EPS, u["residual"], w2, u["next_scale"])
                got2 = F.rms_norm_gate_residual_modulate_mxfp4(u["residual"], u["x"], v["weight"], v["cond"], w2,
                                                               u["next_scale"], eps=EPS)[1]
                _same(got2, O.quantize(y), zoom)
                top = max(top, int(got.scales[got.scales < 255].max()))
        assert top == 254
        bad = w.clone()
        bad[3] = float("inf")
        _same(F.rms_norm_modulate_mxfp4(v["x"], bad, v["cond"], eps=EPS),
              O.quantize(O.norm_values(v["x"], bad, v["cond"], None, EPS)), "inf")


def _norm_codes(v):
    import futudiffu_amd as F
    x, k = v["x"], v["doc_ids"]
    first = F.rms_norm_modulate_mxfp4(x, v["weight"], v["cond"], doc_ids=k, eps=EPS)
    _, second = F.rms_norm_gate_residual_modulate_mxfp4(v["residual"], x, v["weight"], v["cond"], v["next_weight"],
                                                        v["next_scale"], doc_ids=k, eps=EPS)
    return ((first, O.norm_values(x, v["weight"], v["cond"], k, EPS)),
            (second, O.norm_values(x, v["weight"], v["cond"], k, EPS, v["residual"], v["next_weight"], v["next_scale"])[1]))


def test_norms_decide_next_to_borders(cuda):
    """So many values that some lie within fp32's roundings of a border between two codes."""
    for dtype, params in ((BF, BF), (FP, F32)):
        v = _norm_inputs(1, 3000, 3840, dtype, params, seed=6)
        v = {k: None if t is None else t.to(cuda) for k, t in v.items()}
        for q, y in _norm_codes(v):
            _same(q, O.quantize(y), f"{dtype}")
            # y over its block's scale, against the borders
            e = torch.frexp(y.abs().reshape(-1, 32).amax(-1, keepdim=True))[1] - 3
            t = torch.ldexp(y.reshape(-1, 32).abs(), -e)
            near = sum(((t - b).abs() < 2.0 ** -22 * b).sum() for b in (0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0))
            assert near > 0


def test_norms_take_eps_in_64_bits(cuda):
    """An eps whose nearest fp32 value would put channels on the other side of a border between two codes:
    rows of ones, so that a channel is its weight over sqrt(1 + eps)."""
    import futudiffu_amd as F
    x = torch.ones(1, 3, 64, dtype=BF, device=cuda)
    told = 0
    for i in range(1, 3000):
        eps = 0.1 + i / 10007
        single = float(torch.tensor(eps, dtype=F32))
        borders = torch.tensor([5.0, 3.5, 2.5, 1.75, 1.25, 0.75, 0.25], dtype=torch.float64)
        w = (borders * (1 + eps) ** 0.5).float().double()
        apart = ((w / (1 + eps) ** 0.5 > borders) != (w / (1 + single) ** 0.5 > borders)).nonzero().flatten()
        if len(apart) == 0:
            continue
        told += 1
        weight = torch.ones(64)
        weight[0], weight[32] = 5.5, 5.5  # the scales are 1
        weight[40:40 + len(apart)] = w[apart].float()
        weight = weight.to(cuda)
        q = F.rms_norm_modulate_mxfp4(x, weight, eps=eps)
        _same(q, O.quantize(O.norm_values(x, weight, None, None, eps)), eps)
        q = F.rms_norm_gate_residual_modulate_mxfp4(x, torch.zeros_like(x), None, None, weight, eps=eps)[1]
        _same(q, O.quantize(O.norm_values(x, weight, None, None, eps)), eps)
    assert told >= 10, told


# ---------------------------------------------------------------- traced, refused

def _calls(device, seed=0):
    """(op, function of its tensors to a tuple of tensors, tensors)."""
    import futudiffu_amd as F
    g = torch.Generator().manual_seed(seed)

    def t(*shape, dtype=BF):
        return torch.randn(*shape, generator=g).to(dtype).to(device)

    C = 72
    ids = torch.tensor([[0, 0, 2, 1, -1, 1], [1, 5, 0, 0, 2, 2]], dtype=torch.int32, device=device)
    x, r, w, k, w2, k2 = t(2, 6, C), t(2, 6, C), t(C), t(2, 3, C), t(C), t(2, 3, C)
    qw = F.mxfp4_quantize(t(2 * C, C))
    flat = lambda q: (q.codes, q.scales)  # noqa: E731
    return [("mxfp4_quantize", lambda x: flat(F.mxfp4_quantize(x)), (x,)),
            ("rms_norm_modulate_mxfp4", lambda *a: flat(F.rms_norm_modulate_mxfp4(*a, doc_ids=ids)), (x, w, k)),
            ("rms_norm_gate_residual_modulate_mxfp4",
             lambda *a: (lambda h, q: (h, *flat(q)))(*F.rms_norm_gate_residual_modulate_mxfp4(*a, doc_ids=ids)),
             (r, x, w, k, w2, k2)),
            ("mxfp4_linear", lambda *a: (F.mxfp4_linear(a[0], qw, *a[1:], activation="swiglu"),),
             (x, t(2 * C, dtype=F32), r)),
            ("mxfp4_dequantize", lambda x: (F.mxfp4_dequantize(F.mxfp4_quantize(x), dtype=FP),), (x,)),
            ("mxfp4_linear_codes", lambda x, b: (F.mxfp4_linear(F.mxfp4_quantize(x), qw, b),), (x, t(2 * C)))]


def _equal(got, want):
    torch.cuda.synchronize()
    return len(got) == len(want) and all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("i", range(6))
def test_traced_graphs_compute(cuda, i):
    from torch.fx.experimental.proxy_tensor import make_fx
    name, fn, args = _calls(cuda)[i]
    new = _calls(cuda)[i][2]
    new = tuple(-2 * t for t in new)
    want = fn(*new)
    traced = make_fx(fn)(*args)
    assert any(name in str(n.target) for n in traced.graph.nodes)
    assert _equal(traced(*new), want)
    assert _equal(torch.jit.trace(fn, args, check_trace=False)(*new), want)
    assert _equal(torch.compile(fn, backend="aot_eager", fullgraph=True)(*new), want)
    xs = torch.stack([args[-1], 2 * args[-1], -args[-1]])  # vmap is a loop over samples
    got = torch.vmap(lambda t: fn(*args[:-1], t))(xs)
    for s in range(3):
        assert _equal([t[s] for t in got], fn(*args[:-1], xs[s]))
    for j, a in enumerate(args):
        for lazy, plain in ((torch._neg_view(a), -a),
                            (torch._efficientzerotensor(a.shape, dtype=a.dtype, device=cuda), torch.zeros_like(a))):
            put = lambda t: args[:j] + (t,) + args[j + 1:]  # noqa: E731
            assert _equal(fn(*put(lazy)), fn(*put(plain)))


@pytest.mark.parametrize("i", range(6))
def test_gradients_that_would_be_lost_raise(cuda, i):
    from torch.autograd import forward_ad
    name, fn, args = _calls(cuda)[i]
    for j, a in enumerate(args):
        put = lambda t: fn(*args[:j], t, *args[j + 1:])  # noqa: E731
        with forward_ad.dual_level(), pytest.raises(NotImplementedError, match="forward-mode"):
            put(forward_ad.make_dual(a, torch.ones_like(a)))
        if name == "mxfp4_linear":
            continue
        leaf = a.detach().requires_grad_()
        with pytest.raises(RuntimeError, match="carry no gradient"):
            put(leaf)
        with pytest.raises(Exception, match="carry no gradient"):
            torch.compile(put, backend="aot_eager", fullgraph=True)(leaf)
        with torch.no_grad():
            assert _equal(put(leaf), put(a))
    if name == "mxfp4_quantize":
        with pytest.raises(RuntimeError, match="carry no gradient"):
            torch.ops.futudiffu_ii.mxfp4_quantize(args[0].detach().requires_grad_())


def test_linear_op_check_and_compile(cuda):
    import futudiffu_amd as F
    for act in ("none", "swiglu"):
        v = _inputs(24, 40, 16, act, BF, F32, True, seed=4, device=cuda)
        w = v["weight"]
        x, b, r = (v[k].detach().requires_grad_() for k in LEAVES)
        tests = ("test_schema", "test_autograd_registration", "test_faketensor", "test_aot_dispatch_static")
        torch.library.opcheck(torch.ops.futudiffu_ii.mxfp4_linear.default, (x, *w, b, r, act, True), test_utils=tests)
        fn = torch.compile(lambda x, b, r: F.mxfp4_linear(x, w, b, r, activation=act), backend="aot_eager", fullgraph=True)
        out = fn(x, b, r)
        grads = torch.autograd.grad(out, (x, b, r), v["dout"])
        want = _run(v, act)
        assert torch.equal(out, want["out"]) and all(torch.equal(t, want["d" + k]) for k, t in zip(LEAVES, grads))
        ops = torch.ops.futudiffu_ii
        out = ops.mxfp4_linear(x, *w, b, r, act, True)[0]
        assert _equal(torch.autograd.grad(out, (x, b, r), v["dout"], retain_graph=True), [want["d" + k] for k in LEAVES])
        for y in (out, F.mxfp4_linear(x, w, b, r, activation=act)):
            with pytest.raises(RuntimeError, match="create_graph"):
                torch.autograd.grad(y, (x, b, r), v["dout"], create_graph=True)
        xs = torch.stack([v["x"], 2 * v["x"]]).requires_grad_()  # a gradient taken outside of vmap
        y = torch.vmap(lambda t: F.mxfp4_linear(t, w, b.detach(), r.detach(), activation=act))(xs)
        got, = torch.autograd.grad(y, xs, torch.stack([v["dout"]] * 2))
        for s in range(2):
            assert torch.equal(got[s], _run(dict(v, x=xs[s].detach()), act)["dx"])
    q = torch.ops.futudiffu_ii
    v = _norm_inputs(1, 5, 40, BF, BF, seed=1)
    x, r = v["x"].to(cuda), v["residual"].to(cuda)
    checks = ("test_schema", "test_faketensor")
    torch.library.opcheck(q.mxfp4_quantize.default, (x,), test_utils=checks)
    codes, scales = q.mxfp4_quantize(x)
    torch.library.opcheck(q.mxfp4_dequantize.default, (codes, scales, 40, FP), test_utils=checks)
    torch.library.opcheck(q.rms_norm_modulate_mxfp4.default, (x, None, None, None, EPS), test_utils=checks)
    torch.library.opcheck(q.rms_norm_gate_residual_modulate_mxfp4.default, (r, x, None, None, None, None, None, EPS),
                          test_utils=checks)


@pytest.mark.parametrize("act", ["none", "silu", "swiglu"])
def test_second_derivatives_raise(cuda, act):
    """The function and the op, with x the only leaf (a frozen bias or none), beside a bias, and by a
    transform; the residual's gradient alone is the incoming one."""
    import futudiffu_amd as F
    v = _inputs(24, 40, 16, act, BF, F32, True, seed=4, device=cuda)
    w, d = v["weight"], v["dout"]
    calls = (lambda x, b, r: F.mxfp4_linear(x, w, b, r, activation=act),
             lambda x, b, r: torch.ops.futudiffu_ii.mxfp4_linear(x, *w, b, r, act, True)[0])
    for call in calls:
        for b in (v["bias"], None):
            x = v["x"].detach().requires_grad_()
            want = torch.autograd.grad(call(x, b, v["residual"]), x, d)[0]
            assert torch.equal(want, _run(dict(v, bias=b), act)["dx"])
            with pytest.raises(RuntimeError, match="create_graph"):
                torch.autograd.grad(call(x, b, v["residual"]), x, d, create_graph=True)
            with pytest.raises(RuntimeError):  # torch's own: the ops have no formula for transforms
                torch.func.grad(lambda t: call(t, b, v["residual"]).float().sum())(v["x"])
        x, b = v["x"].detach().requires_grad_(), v["bias"].detach().requires_grad_()
        with pytest.raises(RuntimeError, match="create_graph"):
            torch.autograd.grad(call(x, b, None), b, d, create_graph=True)
        r = v["residual"].detach().requires_grad_()
        assert torch.equal(torch.autograd.grad(call(v["x"], v["bias"], r), r, d, create_graph=True)[0], d)


def test_training_over_a_weight_too_large_for_dx(cuda):
    """2^31 elements: the bias and the residual train; an x that wants a gradient is refused by the forward."""
    import futudiffu_amd as F
    n, k = 1 << 19, 4096
    w = F.MXFP4(torch.zeros(n, k // 2, dtype=torch.uint8, device=cuda),
                torch.full((k // 256, n, 8), 127, dtype=torch.uint8, device=cuda), k)
    w.codes[n - 1, k // 2 - 1] = 0x20  # 1 in the last column
    g = torch.Generator().manual_seed(1)
    x, d = torch.randn(3, k, generator=g).to(BF).to(cuda), torch.randn(3, n, generator=g).to(BF).to(cuda)
    b, r = torch.zeros(n, device=cuda, requires_grad=True), torch.randn(3, n, generator=g).to(BF).to(cuda).requires_grad_()
    out = F.mxfp4_linear(x, w, b, r)
    db, dr = torch.autograd.grad(out, (b, r), d)
    assert torch.equal(out[:, :-1], r[:, :-1]) and torch.equal(dr, d)
    q = O.rounded(x)[:, -1]
    assert torch.equal(out[:, -1], (q + r[:, -1].double()).to(BF))
    assert B.worst(db, d.double().sum(0), 4 * 2.0 ** -24 * d.double().abs().sum(0)) <= 1.0
    for call in (lambda t: F.mxfp4_linear(t, w, b, r), lambda t: torch.ops.futudiffu_ii.mxfp4_linear(t, *w, b, r, "none", True)):
        with pytest.raises(ValueError, match="2\\^31"):
            call(x.detach().requires_grad_())


# ---------------------------------------------------------------- together

H, D, C, F_ = 4, 64, 256, 640


def _block(p, q, x, t, freqs, ids, mask, mx=True):
    """A transformer block around the attention, its projections over MXFP4; with mx=False every
    operator's result from the 64-bit definitions, rounded as the operators round it."""
    import math
    import futudiffu_amd as F

    def linear(x, name, bias=None, act="none"):
        if mx:
            return F.mxfp4_linear(x, q[name], bias, activation=act, dtype=BF)
        values = O.dequantize(*q[name][:2], q[name].columns)
        return O.linear(x.to(BF) if x.dtype != BF else x, values, bias, None, act)["out"][0].to(BF)

    scale1, gate1, scale2, gate2 = linear(t, "w_ada", p["b_ada"]).chunk(4, dim=-1)
    if mx:
        y = F.rms_norm_modulate_mxfp4(x, p["norm1"], scale1, doc_ids=ids, eps=EPS)
    else:  # the codes' values are bf16 values, and their codes again
        y = O.rounded(O.norm_values(x, p["norm1"], scale1, ids, EPS)).to(BF)
    one = torch.ones(D, device=x.device)
    a = torch.ops.futudiffu_ii.sage_attn_qkv_masked(linear(y, "qkv"), one, one, freqs, mask, H, D, EPS, 1 / math.sqrt(D))[0]
    a = linear(a, "out")
    if mx:
        x, y = F.rms_norm_gate_residual_modulate_mxfp4(x, a, p["norm2"], gate1, p["ffn_norm1"], scale2, doc_ids=ids, eps=EPS)
    else:
        h, v = O.norm_values(a, p["norm2"], gate1, ids, EPS, x, p["ffn_norm1"], scale2)
        x, y = h.to(BF), O.rounded(v).to(BF)
    f = linear(linear(y, "w13", act="swiglu"), "w2")
    return F.rms_norm_gate_residual(x, f, p["ffn_norm2"], gate2, doc_ids=ids, eps=EPS)


def _block_state(device, lengths, pad, seed):
    import futudiffu_amd as F
    from futudiffu_amd import block_mask as BM
    g = torch.Generator().manual_seed(seed)

    def normal(*s, scale=1.0, offset=0.0):
        return (offset + scale * torch.randn(*s, generator=g)).to(BF).to(device)

    N = sum(lengths) + pad
    ids = torch.cat([torch.repeat_interleave(torch.arange(len(lengths)), torch.tensor(lengths)),
                     torch.full((pad,), -1)]).to(torch.int32)[None].to(device)
    p = {n: normal(C, scale=0.2, offset=1.0) for n in ("norm1", "norm2", "ffn_norm1", "ffn_norm2")}
    p["b_ada"] = normal(4 * C, scale=0.1)
    q = {n: F.mxfp4_quantize(normal(r, k, scale=k ** -0.5)) for n, r, k in (
        ("qkv", 3 * H * D, C), ("out", C, H * D), ("w13", 2 * F_, C), ("w2", C, F_), ("w_ada", 4 * C, 32))}
    ang = torch.rand(1, N, 1, D // 2, generator=g) * 6.283
    c, s = torch.cos(ang), torch.sin(ang)
    freqs = torch.stack([torch.stack([c, -s], -1), torch.stack([s, c], -1)], -2).to(device)
    x, t = normal(1, N, C, scale=1.5), normal(1, len(lengths), 32)
    return p, q, x, t, freqs, ids, BM.build_block_mask(list(lengths), N, device=device)


@pytest.mark.parametrize("lengths,pad", [((256, 128), 0), ((300, 77, 130), 5), ((40,), 0)])
def test_block(cuda, lengths, pad):
    """The operators one behind the other, as a block of a model in 4 bits uses them.  Every step is
    the definitions' on the step before's result, so only values that a 32-bit sum rounds to the other
    side of a bf16 tie differ, and the codes that this turns: of a block of 32 with one turned
    code 2^-3 of its norm.  Five products of bf16 outputs, where one in 2^7 rounds otherwise by 2^-8:
    2^-6 of the norm is allowed."""
    state = _block_state(cuda, lengths, pad, seed=sum(lengths))
    print("block", lengths, pad, flush=True)
    got, want = _block(*state), _block(*state, mx=False)
    err = float((got.double() - want.double()).norm() / want.double().norm())
    print("off by", err, flush=True)
    assert torch.isfinite(got).all() and err <= 2.0 ** -6, err


def test_block_captured(cuda):
    """The block in one graph: replays on new inputs equal eager calls bit for bit."""
    p, q, x, t, freqs, ids, mask = _block_state(cuda, (200, 120), 0, seed=9)
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        for _ in range(2):
            _block(p, q, x, t, freqs, ids, mask)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        got = _block(p, q, x, t, freqs, ids, mask)
    g = torch.Generator().manual_seed(10)
    for _ in range(3):
        x.copy_(torch.randn(x.shape, generator=g))
        t.copy_(torch.randn(t.shape, generator=g))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, _block(p, q, x, t, freqs, ids, mask))
