"""MXFP4 without a GPU: refusals of the Python functions and of the C entries, workspace sizes, and
the 64-bit oracle against the definition and differentiation."""

import pytest
import torch

import futudiffu_amd as F
from futudiffu_amd import _lib
from oracle import mx_oracle as O

fake_addresses = pytest.mark.skipif(torch.cuda.device_count() > 0,
                                    reason="argument-validation calls with fake device addresses run without a GPU")
BF = torch.bfloat16


def _weight(n, k):
    p = O.columns_held(k)
    return F.MXFP4(torch.zeros(n, p // 2, dtype=torch.uint8), torch.zeros(p // 256, n, 8, dtype=torch.uint8), k)


# ---- the oracle

def test_oracle_codes_are_the_nearest():
    """Every magnitude between the smallest and past the largest, ties among them: no value of the
    block's scale is nearer, and of two equally near the code is even."""
    x = torch.arange(-511, 512).double() / 64  # within 8 by 1/64: all ties
    rows = torch.zeros(x.numel(), 32, dtype=torch.float64)
    rows[:, 0] = 7.0  # the scale is 1
    rows[:, 5] = x
    codes, scales = O.quantize(rows)
    assert (scales[0, :, 0] == 127).all() and (scales[0, :, 1:] == 0).all() and (codes[:, 16:] == 0).all()
    got = codes[:, 2] >> 4
    table = torch.tensor(O.VALUES, dtype=torch.float64)
    off = (x.abs()[:, None] - table).abs()
    near = off.min(1).values
    mine = off.gather(1, (got & 7).long()[:, None])[:, 0]
    assert torch.equal(mine, near)
    tie = (off == near[:, None]).sum(1) == 2
    assert tie.sum() == 2 * 7 and (got[tie] % 2 == 0).all()
    assert torch.equal((got >= 8), torch.signbit(x))
    assert torch.equal(O.dequantize(codes, scales, 32)[:, 0], torch.full((x.numel(),), 6.0, dtype=torch.float64))


def test_oracle_scales():
    """amax / 2^e lies in [4, 8), down to the smallest scale; zeros, NaN and infinities."""
    top = torch.tensor([4.0, 7.99, 8.0, 2.0 ** -120, 2.0 ** -125, 2.0 ** -126, 2.0 ** -133, 3.0e38, 0.0], dtype=torch.float64)
    x = torch.zeros(top.numel(), 40, dtype=torch.float64)
    x[:, 3] = -top
    codes, scales = O.quantize(x)
    assert scales[0, :, 0].tolist() == [127, 127, 128, 5, 0, 0, 0, 252, 0]
    x[0, 9], x[1, 33] = float("nan"), float("inf")
    codes, scales = O.quantize(x)
    assert scales[0, 0, 0] == 255 and (codes[0, :16] == 0).all() and scales[0, 1, 1] == 255 and scales[0, 1, 0] == 127
    back = O.dequantize(codes, scales, 40)
    assert back[0, :32].isnan().all() and back[1, 32:].isnan().all() and not back[0, 32:].isnan().any()


def test_oracle_past_the_largest_scale():
    """The scale stops at 2^127 and the codes at 6."""
    x = torch.zeros(5, 32, dtype=torch.float64)
    x[:, 0] = torch.tensor([1.9 * 2.0 ** 128, 2.0 ** 129, 7.9 * 2.0 ** 127, 2.0 ** 130, 2.0 ** 200], dtype=torch.float64)
    codes, scales = O.quantize(x)
    assert scales[0, :, 0].tolist() == [253, 254, 254, 254, 254]
    assert O.dequantize(codes, scales, 32)[:, 0].tolist() == [1.5 * 2.0 ** 128, 2.0 ** 129] + [6 * 2.0 ** 127] * 3


def test_oracle_keeps_what_it_can_hold():
    """Values of a block's grid come back exactly; everything else within half a step of its place."""
    g = torch.Generator().manual_seed(1)
    x = torch.randn(50, 333, generator=g).double()
    q = O.rounded(x)
    assert torch.equal(O.rounded(q), q)
    b = torch.nn.functional.pad(x, (0, 19)).reshape(50, -1, 32)
    scale = torch.exp2(torch.floor(torch.log2(b.abs().amax(-1, keepdim=True))) - 2)
    r = b.abs() / scale
    half = torch.where(r < 2, 0.25, torch.where(r < 4, 0.5, 2.0)) * scale  # past 6: up to 2
    off = (torch.nn.functional.pad(q, (0, 19)).reshape(b.shape) - b).abs()
    assert (off <= half).all()


@pytest.mark.parametrize("act", ["none", "silu", "gelu", "swiglu"])
def test_oracle_gradients(act):
    """The oracle's gradients are those of its output in 64 bits with the rounding of x passed."""
    g = torch.Generator().manual_seed(2)
    n = 5
    x = torch.randn(4, 40, generator=g).to(BF)
    w = O.rounded(torch.randn(2 * n if act == "swiglu" else n, 40, generator=g))
    b, r, d = torch.randn(w.shape[0], generator=g), torch.randn(4, n, generator=g).to(BF), torch.randn(4, n, generator=g).to(BF)
    want = O.linear(x, w, b, r, act, d)
    leaf, bias = O.rounded(x).requires_grad_(), b.double().requires_grad_()
    z = leaf @ w.T + bias
    f = torch.nn.functional
    y = {"none": lambda t: t, "silu": f.silu, "gelu": lambda t: f.gelu(t, approximate="tanh"),
         "swiglu": lambda t: f.silu(t[:, :n]) * t[:, n:]}[act](z) + r.double()
    dx, db = torch.autograd.grad(y, (leaf, bias), d.double())
    for k, t in (("out", y.detach()), ("dx", dx), ("dbias", db)):
        torch.testing.assert_close(want[k][0], t, rtol=1e-12, atol=1e-12)


# ---- the Python functions

def test_cpu_tensors_are_refused():
    x, w = torch.zeros(2, 40, dtype=BF), _weight(6, 40)
    for call in (lambda: F.mxfp4_quantize(x), lambda: F.rms_norm_modulate_mxfp4(x),
                 lambda: F.rms_norm_gate_residual_modulate_mxfp4(x, x)):
        with pytest.raises(ValueError, match="must be a GPU tensor"):
            call()
    for call in (lambda: F.mxfp4_dequantize(w), lambda: F.mxfp4_linear(x, w), lambda: F.mxfp4_linear(w, w)):
        with pytest.raises(ValueError, match="must be on a GPU"):
            call()


def test_argument_checks():
    x, w = torch.zeros(2, 40, dtype=BF), _weight(6, 40)
    with pytest.raises(ValueError, match="at least one column"):
        F.mxfp4_quantize(x[:, :0])
    with pytest.raises(ValueError, match="at least one column"):
        F.mxfp4_quantize(x[0, 0])
    for bad in (x.float(), x.double(), x.int()):
        with pytest.raises(ValueError, match="bfloat16 or float16"):
            F.mxfp4_quantize(bad)
    for dtype in (torch.float32, torch.uint8):
        with pytest.raises(ValueError, match="dtype must be"):
            F.mxfp4_dequantize(w, dtype=dtype)
    for bad in (w._replace(columns=0), w._replace(columns=-3)):
        with pytest.raises(ValueError, match="columns must be"):
            F.mxfp4_dequantize(bad)
    for bad in (w._replace(columns=300), w._replace(codes=w.codes.int()), w._replace(codes=w.codes[:, :64])):
        with pytest.raises(ValueError, match="codes must be"):
            F.mxfp4_dequantize(bad)
    for bad in (w.scales[:, :5], w.scales[..., :4], w.scales[0], w.scales.int(), w.scales.repeat(2, 1, 1)):
        with pytest.raises(ValueError, match="scales must be"):
            F.mxfp4_dequantize(w._replace(scales=bad))
    for fn in (F.rms_norm_modulate_mxfp4, lambda t, k=None: F.rms_norm_gate_residual_modulate_mxfp4(t, t, None, None, k)):
        with pytest.raises(ValueError, match="weight must be"):
            fn(x, torch.zeros(7))
        with pytest.raises(ValueError, match="bfloat16 or float16"):
            fn(x.float())


def test_codes_carry_no_gradient():
    x = torch.zeros(2, 40, dtype=BF, requires_grad=True)
    b = torch.zeros(6, requires_grad=True)
    w = _weight(6, 40)
    q = _weight(2, 40)
    for call in (lambda: F.mxfp4_quantize(x), lambda: F.rms_norm_modulate_mxfp4(x),
                 lambda: F.rms_norm_modulate_mxfp4(x.detach(), torch.zeros(40, requires_grad=True)),
                 lambda: F.rms_norm_gate_residual_modulate_mxfp4(x.detach(), x), lambda: F.mxfp4_linear(q, w, b)):
        with pytest.raises(RuntimeError, match="carry no gradient"):
            call()
        with torch.no_grad(), pytest.raises(ValueError, match="GPU"):
            call()


def test_shape():
    assert _weight(6, 300).shape == (6, 300)
    assert F.MXFP4(torch.zeros(2, 3, 128, dtype=torch.uint8), None, 7).shape == (2, 3, 7)


def test_fakes_have_the_outputs_shapes():
    """Under a fake mode: what a compiler sees is what a call returns."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    ops = torch.ops.futudiffu_ii
    with FakeTensorMode():
        x = torch.empty(2, 5, 300, dtype=BF, device="cuda")
        codes, scales = ops.mxfp4_quantize(x)
        assert codes.shape == (2, 5, 256) and scales.shape == (2, 10, 8) and codes.dtype == scales.dtype == torch.uint8
        assert ops.mxfp4_dequantize(codes, scales, 300, torch.float16).shape == x.shape
        w = torch.empty(8, 256, dtype=torch.uint8, device="cuda"), torch.empty(2, 8, 8, dtype=torch.uint8, device="cuda"), 300
        for act, n in (("none", 8), ("swiglu", 4)):
            out, z = ops.mxfp4_linear(x, *w, None, None, act, True)
            assert out.shape == (2, 5, n) and z.shape == ((10, 8) if act == "swiglu" else (0,))
            q = ops.mxfp4_linear_codes(codes, scales, 300, *w, None, None, act, BF)
            assert q.shape == (2, 5, n) and q.dtype == BF
        dx, db = ops.mxfp4_linear_backward(out, *w, torch.empty(8, device="cuda"), z, "swiglu", [True, True])
        assert dx.shape == x.shape and db.shape == (8,) and db.dtype == torch.float32
        assert ops.rms_norm_modulate_mxfp4(x, None, None, None, 1e-5)[0].shape == codes.shape
        h, c, s = ops.rms_norm_gate_residual_modulate_mxfp4(x, x, None, None, None, None, None, 1e-5)
        assert h.shape == x.shape and c.shape == codes.shape and s.shape == scales.shape


@pytest.mark.parametrize("act", ["none", "silu", "swiglu"])
def test_gradients_of_the_op_are_not_differentiated(act):
    """As fused_linear's: whichever of x and the bias wants a gradient, alone or beside the other,
    create_graph=True raises.  A residual's gradient is the incoming one, which may be differentiated."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        x, r = torch.empty(5, 40, dtype=BF), torch.empty(5, 4, dtype=BF)
        n = 8 if act == "swiglu" else 4
        w = torch.empty(n, 128, dtype=torch.uint8), torch.empty(1, n, 8, dtype=torch.uint8), 40
        bias = torch.empty(n)
        for wants, of, twice in (("x", "x", False), ("b", "b", False), ("xb", "b", False), ("xb", "x", False),
                                 ("r", "r", True), ("xr", "r", False)):
            for b in (bias, None):
                t = dict(x=x.detach(), b=None if b is None else b.detach(), r=r.detach())
                if any(t[k] is None for k in wants):
                    continue
                for k in wants:
                    t[k].requires_grad_()

                def grad(**kw):
                    out = torch.ops.futudiffu_ii.mxfp4_linear(t["x"], *w, t["b"], t["r"], act, True)[0]
                    return torch.autograd.grad(out, t[of], torch.ones_like(out), **kw)[0]

                assert grad().shape == t[of].shape
                if twice:
                    assert grad(create_graph=True).shape == r.shape
                else:
                    with pytest.raises(RuntimeError, match="create_graph"):
                        grad(create_graph=True)


@pytest.mark.parametrize("wanted", [[], [True], [True, True, True]])
def test_gradient_op_takes_two_wanted(wanted):
    w = _weight(6, 40)
    with pytest.raises(ValueError, match="wanted must"):
        torch.ops.futudiffu_ii.mxfp4_linear_backward(torch.zeros(2, 6, dtype=BF), *w, None, None, "none", wanted)


def test_a_weight_too_large_for_dx():
    """Refused by the forward where x wants a gradient; a bias's gradient needs no rows of the weight."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        n, k = 1 << 19, 4096
        x, b = torch.empty(3, k, dtype=BF), torch.empty(n, requires_grad=True)
        w = torch.empty(n, k // 2, dtype=torch.uint8), torch.empty(k // 256, n, 8, dtype=torch.uint8), k

        def out(x):
            return torch.ops.futudiffu_ii.mxfp4_linear(x, *w, b, None, "none", True)[0]

        assert torch.autograd.grad(out(x), b, torch.empty(3, n, dtype=BF))[0].shape == (n,)
        with pytest.raises(ValueError, match="2\\^31"):
            out(x.requires_grad_())


# ---- the C entries

@fake_addresses
@pytest.mark.parametrize("over,status,msg", [
    (dict(m=0), 1, "positive"), (dict(k=0), 1, "positive"), (dict(m=1 << 24), 1, "exceeds"), (dict(k=1 << 22), 1, "exceeds"),
    (dict(dt=2), 1, "dtype"), (dict(codes=None), 1, "null"), (dict(scales=None), 1, "null"), (dict(t=None), 1, "null"),
    (dict(codes=72), 2, "16-byte"), (dict(scales=68), 2, "8-byte"), (dict(t=17), 2, "aligned to"),
])
def test_quantize_entries_refuse(over, status, msg):
    lib = _lib.load()
    a = dict(t=16, m=4, k=40, dt=0, codes=64, scales=64)
    a.update(over)
    assert lib.sage_mxfp4_quantize(a["t"], 40, a["m"], a["k"], a["dt"], a["codes"], a["scales"], None) == status
    assert msg in lib.sage_last_error().decode()
    assert lib.sage_mxfp4_dequantize(a["codes"], a["scales"], a["m"], a["k"], a["dt"], a["t"], None) == status
    assert msg in lib.sage_last_error().decode()


@fake_addresses
@pytest.mark.parametrize("over,status,msg", [
    (dict(m=0), 1, "positive"), (dict(n=0), 1, "positive"), (dict(k=0), 1, "positive"),
    (dict(m=1 << 24), 1, "exceeds"), (dict(n=1 << 22), 1, "exceeds"), (dict(k=1 << 22), 1, "exceeds"),
    (dict(act=4), 1, "activation"), (dict(act=-1), 1, "activation"), (dict(dt=2), 1, "dtype"),
    (dict(n=1 << 21, act=3), 1, "rows"), (dict(n=1 << 20, k=4096), 1, "2^31"),
    (dict(out=None), 1, "null"), (dict(w=None), 1, "null"), (dict(ws=None), 1, "null"), (dict(x=None), 1, "null"),
    (dict(x=None, xc=64), 1, "null"), (dict(r=64, rrs=15), 1, "apart"), (dict(r=64, rrs=1 << 22), 1, "apart"),
    (dict(x=17), 2, "aligned to"), (dict(out=65), 2, "aligned to"), (dict(bias=33), 2, "bias"),
    (dict(bias=34, bf32=1), 2, "bias"), (dict(z=34), 2, "z to 4"), (dict(w=72), 2, "16-byte"), (dict(ws=68), 2, "8-byte"),
    (dict(x=None, xc=72, xs=64), 2, "16-byte"), (dict(), 3, "workspace of"), (dict(wksp=72, bytes=1 << 30), 2, "workspace must"),
])
def test_linear_entry_refuses(over, status, msg):
    lib = _lib.load()
    a = dict(x=16, xrs=40, xc=None, xs=None, w=64, ws=64, bias=None, bf32=0, r=None, rrs=16, m=5, n=16, k=40, dt=0, act=0,
             wksp=None, bytes=0, z=None, out=64, st=None)
    a.update(over)
    assert lib.sage_mxfp4_linear(*a.values()) == status
    assert msg in lib.sage_last_error().decode()


@fake_addresses
def test_linear_entry_reads_rows_in_any_order():
    """Rows that lie backwards are quantized by the kernel that takes any stride: the few-row product's own
    offsets are 32-bit and not negative."""
    lib = _lib.load()
    args = (64, 64, None, 0, None, 0, 4, 16, 40, 0, 0, None, 0, None, 64, None)
    assert lib.sage_mxfp4_linear(1 << 20, -40, None, None, *args) == 3
    assert "workspace of" in lib.sage_last_error().decode()


@fake_addresses
@pytest.mark.parametrize("over,status,msg", [
    (dict(m=0), 1, "positive"), (dict(k=1 << 22), 1, "exceeds"), (dict(act=7), 1, "activation"),
    (dict(d=None), 1, "null"), (dict(w=None), 1, "null"), (dict(act=1), 1, "null"), (dict(drs=15), 1, "apart"),
    (dict(n=1 << 19, drs=1 << 19, k=4096), 1, "2^31"), (dict(d=17), 2, "aligned to"), (dict(dx=72), 2, "16-byte"),
    (dict(act=1, z=66), 2, "z must"), (dict(), 3, "workspace of"), (dict(wksp=72, bytes=1 << 30), 2, "workspace must"),
])
def test_linear_backward_entry_refuses(over, status, msg):
    lib = _lib.load()
    a = dict(d=16, drs=16, w=64, ws=64, z=None, m=4, n=16, k=40, dt=0, act=0, bf32=0, wksp=None, bytes=0, dx=64, db=64, st=None)
    a.update(over)
    assert lib.sage_mxfp4_linear_bwd(*a.values()) == status
    assert msg in lib.sage_last_error().decode()


@fake_addresses
def test_bias_gradient_over_a_large_weight():
    """The limit on the weight's 16-bit rows is dx's."""
    lib = _lib.load()
    n, k = 1 << 19, 4096
    size = lib.sage_mxfp4_linear_bwd_workspace_bytes
    assert size(64, n, 4, n, k, 0, 1) == size(64, n, 4, n, k, 0, 5) == 0 < size(64, n, 4, n, k, 0, 4)
    args = (64, n, 64, 64, None, 4, n, k, 0, 0, 0, None, 0)
    assert lib.sage_mxfp4_linear_bwd(*args, None, 64, None) == 3 and "workspace of" in lib.sage_last_error().decode()
    assert lib.sage_mxfp4_linear_bwd(*args, 64, 64, None) == 1 and "2^31" in lib.sage_last_error().decode()


@fake_addresses
def test_norm_entries_refuse():
    lib = _lib.load()

    def err():
        return lib.sage_last_error().decode()

    tail, bad = (1, None, 2, 8, 8, 0, 0, 1e-5), (1, None, 2, 8, 9000, 0, 0, 1e-5)
    x, k = (16, 64, 8), (32, 48, 8, 0)
    one, two = lib.sage_rms_norm_modulate_mxfp4, lib.sage_rms_norm_gate_residual_modulate_mxfp4
    rest = (80, 64, 8, *x, *k, 96, 112, 8, 0)
    assert one(*x, *k, *bad, 64, 64, None) == 1 and "exceeds" in err()
    assert one(None, 64, 8, *k, *tail, 64, 64, None) == 1 and "null" in err()
    assert one(*x, *k, *tail, None, 64, None) == 1 and "null" in err()
    assert one(*x, *k, *tail, 64, None, None) == 1 and "null" in err()
    assert one(*x, *k, *tail, 72, 64, None) == 2 and "16-byte" in err()
    assert one(17, 64, 8, *k, *tail, 64, 64, None) == 2 and "aligned" in err()
    assert two(*rest, *bad, 128, 64, 64, None) == 1 and "exceeds" in err()
    assert two(*rest, *tail, None, 64, 64, None) == 1 and "null" in err()
    assert two(*rest, *tail, 128, 64, None, None) == 1 and "null" in err()
    assert two(*rest, *tail, 129, 64, 64, None) == 2 and "aligned" in err()


@fake_addresses
def test_norm_entries_take_eps_in_64_bits():
    """No eps under 0, however small, and NaN neither."""
    lib = _lib.load()
    for eps in (-1e-300, -1.0, float("nan")):
        assert lib.sage_rms_norm_modulate_mxfp4(16, 64, 8, 32, 48, 8, 0, 1, None, 2, 8, 8, 0, 0, eps, 64, 64, None) == 1
        assert "eps" in lib.sage_last_error().decode()


def test_workspace_sizes():
    """x's codes and scales and the cut tiles' sums: none for sizes that the calls refuse, and with
    codes given never more than without."""
    lib = _lib.load()
    size = lib.sage_mxfp4_linear_workspace_bytes
    for m, n, k in ((1, 1, 1), (2, 15360, 256), (64, 11520, 3840), (65, 16, 1001), (1280, 3840, 10240), (4416, 20480, 3840),
                    (1 << 20, 136, 2048)):
        held = m * O.columns_held(k) // 2 + m * O.columns_held(k) // 32
        for act in range(4):
            with_x, without = size(m, n, k, act, 1, 1), size(m, n, k, act, 0, 1)
            assert held <= with_x - without <= held + 512
            # rows on 16-byte boundaries: the product quantizes few and short ones itself
            assert size(m, n, k, act, 2, 1) == (without if m <= 4 and k <= 4096 else with_x)
    for m, n, k, act in ((0, 1, 1, 0), (1, 0, 1, 0), (1, 1, 0, 0), (1 << 24, 1, 1, 0), (1, 1 << 22, 1, 0), (1, 1, 1 << 22, 0),
                         (1, 1, 1, 9), (4, 1 << 20, 4096, 0)):
        assert size(m, n, k, act, 1, 1) == 0
        assert lib.sage_mxfp4_linear_bwd_workspace_bytes(64, n, m, n, k, act, 5) == 0
    bwd = lib.sage_mxfp4_linear_bwd_workspace_bytes
    assert bwd(64, 16, 4, 16, 40, 0, 1) >= 16 * 40 * 2  # the weight's 16-bit rows
    assert bwd(64, 16, 4, 16, 40, 0, 4) < 16 * 40 * 2 + 4096
