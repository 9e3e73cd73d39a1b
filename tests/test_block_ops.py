"""The operators around the attention, without a GPU: refusals of the Python functions and
of the C entries, workspace sizes, and the 64-bit oracle against differentiation."""

import pytest
import torch

import futudiffu_amd as F
from futudiffu_amd import _lib
from oracle import block_oracle as O

fake_addresses = pytest.mark.skipif(torch.cuda.device_count() > 0,
                                    reason="argument-validation calls with fake device addresses run without a GPU")



@pytest.mark.parametrize("op", ["modulate", "gate", "gate_modulate"])
def test_norms_refuse_cpu_tensors(op):
    x = torch.zeros(1, 4, 8, dtype=torch.bfloat16)
    calls = {"modulate": lambda: F.rms_norm_modulate(x), "gate": lambda: F.rms_norm_gate_residual(x, x),
             "gate_modulate": lambda: F.rms_norm_gate_residual_modulate(x, x)}
    with pytest.raises(ValueError, match="must be a GPU tensor"):
        calls[op]()
    x.requires_grad_()
    with pytest.raises(ValueError, match="must be a GPU tensor"):
        calls[op]()


def test_norm_argument_checks():
    x = torch.zeros(2, 4, 8, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match=r"\[B, N, C\] or \[N, C\]"):
        F.rms_norm_modulate(x[0, 0])
    with pytest.raises(ValueError, match="bfloat16 or float16"):
        F.rms_norm_modulate(x.float())
    for w in (torch.zeros(7), torch.zeros(1, 8), torch.zeros(8, dtype=torch.float16), torch.zeros(8, dtype=torch.float64)):
        with pytest.raises(ValueError, match="weight must be"):
            F.rms_norm_modulate(x, w)
        with pytest.raises(ValueError, match="next_weight must be"):
            F.rms_norm_gate_residual_modulate(x, x, None, None, w)
    ids = torch.zeros(2, 4, dtype=torch.int32)
    for k, d in ((torch.zeros(8), False), (torch.zeros(1, 8), False), (torch.zeros(2, 3, 8), False),
                 (torch.zeros(2, 8), True), (torch.zeros(1, 3, 8), True), (torch.zeros(2, 0, 8), True),
                 (torch.zeros(2, 8, dtype=torch.float16), False)):
        with pytest.raises(ValueError, match="gate must be"):
            F.rms_norm_gate_residual(x, x, None, k, doc_ids=ids if d else None)
        with pytest.raises(ValueError, match="next_scale must be"):
            F.rms_norm_gate_residual_modulate(x, x, None, None, None, k, doc_ids=ids if d else None)
    with pytest.raises(ValueError, match="same documents"):
        F.rms_norm_gate_residual_modulate(x, x, None, torch.zeros(2, 3, 8), None, torch.zeros(2, 2, 8), doc_ids=ids)
    for bad in (torch.zeros(2, 3, dtype=torch.int32), torch.zeros(4, dtype=torch.int32)):
        with pytest.raises(ValueError, match="doc_ids must be"):
            F.rms_norm_modulate(x, doc_ids=bad)
    for t in (torch.zeros(2, 4), torch.zeros(2, 4, dtype=torch.bool)):
        with pytest.raises(ValueError, match="integers"):
            F.rms_norm_modulate(x, doc_ids=t)
    for r in (x[:1], x.half(), x[..., :4]):
        with pytest.raises(ValueError, match="residual must be"):
            F.rms_norm_gate_residual(r, x)
    for eps in (-1.0, float("nan")):
        with pytest.raises(ValueError, match="eps must be"):
            F.rms_norm_modulate(x, eps=eps)
    with pytest.raises(ValueError, match="at least one channel"):
        F.rms_norm_modulate(x[..., :0])


def test_linear_argument_checks():
    x, w = torch.zeros(3, 4, 8, dtype=torch.bfloat16), torch.zeros(6, 8, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="must be a GPU tensor"):
        F.fused_linear(x, w)
    with pytest.raises(ValueError, match="activation must be one of"):
        F.fused_linear(x, w, activation="relu")
    with pytest.raises(ValueError, match="bfloat16 or float16"):
        F.fused_linear(x.float(), w.float())
    for bad in (w[:, :7], w[0], w.half(), w[:0], w.float()):
        with pytest.raises(ValueError, match="weight must be"):
            F.fused_linear(x, bad)
    with pytest.raises(ValueError, match="even number of rows"):
        F.fused_linear(x, w[:5], activation="swiglu")
    for bad in (torch.zeros(5), torch.zeros(1, 6), torch.zeros(6, dtype=torch.float16)):
        with pytest.raises(ValueError, match="bias must be"):
            F.fused_linear(x, w, bad)
    for bad in (x, torch.zeros(3, 4, 6), torch.zeros(12, 6, dtype=torch.bfloat16)):
        with pytest.raises(ValueError, match="residual must be"):
            F.fused_linear(x, w, None, bad)
    out = torch.ops.futudiffu_ii.fused_linear_backward
    d = torch.zeros(3, 4, 6, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="must be a GPU tensor"):
        out(d, x, w, None, None, "silu", [True, True, False])


def _modulate(lib, **over):
    a = dict(x=16, xbs=64, xrs=8, w=32, s=48, sbs=8, sgs=0, g=1, doc=None, b=2, n=8, c=8, dt=0, f32=0, eps=1e-5,
             out=None, st=None)
    a.update(over)
    return lib.sage_rms_norm_modulate(*a.values())


@pytest.mark.parametrize("over,status,msg", [
    (dict(b=0), 1, "positive"),
    (dict(n=0), 1, "positive"),
    (dict(c=0), 1, "positive"),
    (dict(c=8193), 1, "exceeds 8192"),
    (dict(n=1 << 23), 1, "grid limit"),
    (dict(b=70000), 1, "grid limit"),
    (dict(b=1 << 12, n=1 << 11), 1, "grid limit"),
    (dict(g=2), 1, "needs doc_ids"),
    (dict(g=0, doc=64), 1, "groups"),
    (dict(g=20000, doc=64), 1, "32767"),
    (dict(dt=2), 1, "dtype"),
    (dict(f32=16), 1, "fp32_params"),
    (dict(eps=-1.0), 1, "eps"),
    (dict(eps=float("nan")), 1, "eps"),
    (dict(x=None, out=64), 1, "null"),
    (dict(), 1, "null"),
    (dict(x=17, out=64), 2, "aligned"),
    (dict(w=34, f32=1, out=64), 2, "parameter pointers"),
    (dict(s=50, f32=2, out=64), 2, "parameter pointers"),
])
@fake_addresses
def test_modulate_entry_refuses(over, status, msg):
    lib = _lib.load()
    assert _modulate(lib, **over) == status
    assert msg in lib.sage_last_error().decode()


@fake_addresses
def test_other_norm_entries_refuse():
    lib = _lib.load()

    def err():
        return lib.sage_last_error().decode()

    tail = (1, None, 2, 8, 8, 0, 0, 1e-5)
    bad = (1, None, 2, 8, 9000, 0, 0, 1e-5)
    x, k = (16, 64, 8), (32, 48, 8, 0)
    for t, out, msg in ((tail, None, "null"), (bad, 64, "exceeds")):
        assert lib.sage_rms_norm_gate_residual(80, 64, 8, *x, *k, *t, out, None) == 1 and msg in err()
        assert lib.sage_rms_norm_gate_residual_modulate(80, 64, 8, *x, *k, 96, 112, 8, 0, *t, 128, out, None) == 1
        assert msg in err()
    assert lib.sage_rms_norm_gate_residual(None, 64, 8, *x, *k, *tail, 64, None) == 1 and "null" in err()
    for fn in (lib.sage_rms_norm_modulate_bwd, lib.sage_rms_norm_gate_residual_bwd):
        assert fn(None, 64, 8, *x, *k, *tail, None, 0, 64, None, None, None) == 1 and "null" in err()
        assert fn(80, 64, 8, *x, *k, *bad, None, 0, 64, None, None, None) == 1 and "exceeds" in err()
        assert fn(80, 64, 8, *x, *k, *tail, None, 0, 64, 96, None, None) == 3 and "workspace of" in err()
        assert fn(80, 64, 8, *x, *k, *tail, 72, 1 << 20, 64, 96, None, None) == 2 and "workspace must be" in err()
    fn, y = lib.sage_rms_norm_gate_residual_modulate_bwd, (144, 64, 8, 80, 64, 8, 160, 64, 8)
    rest = (*x, *k, 96, 112, 8, 0)
    assert fn(*y, *rest, *tail, None, 0, None, 64, None, None, None, None, None) == 1 and "null" in err()
    assert fn(*y, *rest, *tail, None, 0, 176, 64, 192, None, None, None, None) == 3 and "workspace of" in err()


def test_norm_workspace_sizes():
    """fp32 sums of every chunk, document slot and norm, and an id per slot: at most a row a
    token (a slot a token of the chunk), none for sizes the calls refuse."""
    size = _lib.load().sage_rms_norm_bwd_workspace_bytes
    for b, n, c in ((1, 1, 1), (2, 1337, 1001), (1, 4416, 3840), (4, 4352, 3840), (1, 1 << 20, 64), (300, 7, 8192)):
        one = size(b, n, c, 1, 0, 0)
        cp = (c + 3) // 4 * 4
        chunks = one // (cp * 4 + 4)
        assert one == chunks * (cp * 4 + 4) and chunks >= b and chunks % b == 0 and chunks <= b * n
        assert n <= chunks // b * 512
        assert size(b, n, c, 1, 0, 1) == chunks * (2 * cp * 4 + 4)
        for g in (1, 3, 100):
            if b * g > 32767:
                continue
            slots = size(b, n, c, g, 1, 0) // (cp * 4 + 4)
            assert slots <= chunks * min(g + 1, -(-n // (chunks // b)))
    for bad in ((0, 1, 8, 1), (1, 0, 8, 1), (1, 1, 0, 1), (1, 1, 8193, 1), (1, 1 << 23, 8, 1), (2, 8, 8, 20000)):
        assert size(*bad, 1, 0) == 0


def _linear(lib, **over):
    a = dict(x=16, xs=72, w=32, ws=72, b=None, bf=0, r=None, rs=0, m=100, n=40, k=72, dt=0, act=0, ws_=None, wsb=0,
             z=None, out=None, st=None)
    a.update(over)
    return lib.sage_linear(*a.values())


@pytest.mark.parametrize("over,status,msg", [
    (dict(m=0), 1, "positive"),
    (dict(n=0), 1, "positive"),
    (dict(k=-1), 1, "positive"),
    (dict(act=4), 1, "activation"),
    (dict(dt=2), 1, "dtype"),
    (dict(m=1 << 24), 1, "exceeds"),
    (dict(k=1 << 22), 1, "exceeds"),
    (dict(n=1 << 20, k=1 << 11, ws=1 << 11), 1, "2^31 bytes"),
    (dict(n=1 << 19, k=1 << 11, ws=1 << 11, act=3), 1, "2^31 bytes"),
    (dict(n=1 << 12, ws=1 << 20), 1, "2^31 bytes"),
    (dict(), 1, "null"),
    (dict(xs=71, out=64), 1, "x rows are"),
    (dict(ws=71, out=64), 1, "weight rows are"),
    (dict(r=48, rs=39, out=64), 1, "residual rows are"),
    (dict(xs=1 << 22, out=64), 1, "2^22 or more"),
    (dict(x=17, out=64), 2, "aligned"),
    (dict(b=34, bf=1, out=64), 2, "bias must be aligned"),
    (dict(x=18, out=64), 3, "workspace of"),             # a copy of x
    (dict(m=1280, n=3840, k=10240, xs=10240, ws=10240, out=64), 3, "workspace of"),  # tiles in pieces
    (dict(x=18, out=64, ws_=72, wsb=1 << 30), 2, "workspace must be"),
])
@fake_addresses
def test_linear_entry_refuses(over, status, msg):
    lib = _lib.load()
    assert _linear(lib, **over) == status
    assert msg in lib.sage_last_error().decode()


@fake_addresses
def test_linear_backward_entry_refuses():
    lib = _lib.load()

    def call(**over):
        a = dict(d=16, ds=40, x=32, xs=72, w=48, ws=72, z=None, m=100, n=40, k=72, dt=0, act=0, bf=0, work=None, wsb=0,
                 dx=64, dw=None, db=None, st=None)
        a.update(over)
        return lib.sage_linear_bwd(*a.values()), lib.sage_last_error().decode()

    for over, status, msg in ((dict(d=None), 1, "null"), (dict(w=None), 1, "null"), (dict(dw=80, x=None), 1, "null"),
                              (dict(act=1), 1, "null"), (dict(ds=39), 1, "dout rows"), (dict(ws=71), 1, "weight rows"),
                              (dict(dw=80, xs=71), 1, "x rows"), (dict(d=17), 2, "aligned"),
                              (dict(db=82, bf=1), 2, "dbias"), (dict(dx=72), 2, "16-byte"),
                              (dict(d=18), 3, "workspace of"), (dict(act=1, z=96), 3, "workspace of"),
                              (dict(db=80), 3, "workspace of"),
                              (dict(d=18, work=72, wsb=1 << 30), 2, "workspace must be")):
        got = call(**over)
        assert got[0] == status and msg in got[1], (over, got)
    assert call(dx=None)[0] == 0  # nothing wanted


def test_linear_workspace_sizes():
    """Copies of operands that cannot be read in place, and the sums of cut tiles."""
    lib = _lib.load()
    size, bwd = lib.sage_linear_workspace_bytes, lib.sage_linear_bwd_workspace_bytes
    assert size(16, 72, 32, 72, 3, 40, 72, 0, 0) == 0
    up = lambda b: (b + 255) // 256 * 256  # noqa: E731
    assert size(18, 72, 32, 72, 3, 40, 72, 0, 0) == up(3 * 72 * 2)
    assert size(16, 73, 32, 73, 3, 40, 73, 0, 0) == up(3 * 80 * 2) + up(40 * 80 * 2)
    assert size(16, 72, 32, 72, 100, 65, 72, 0, 0) == size(16, 128, 32, 128, 100, 72, 128, 0, 1) == 0
    # 75 tiles of 256 x 256 in 3 pieces: their fp32 sums
    assert size(16, 10240, 32, 10240, 1280, 3840, 10240, 0, 0) == 75 * 3 * 256 * 256 * 4
    for bad in ((0, 8, 8), (8, 0, 8), (8, 8, 0), (1 << 24, 8, 8), (8, 1 << 22, 8)):
        assert size(16, 8, 32, 8, *bad, 0, 0) == bwd(16, 8, 32, 8, 48, 8, *bad, 0, 7) == 0
    assert bwd(16, 40, 32, 72, 48, 72, 100, 40, 72, 0, 0) == 0
    # the bias's column sums: chunks of 32 rows
    assert bwd(16, 40, 32, 72, 48, 72, 100, 40, 72, 0, 4) == up(4 * 40 * 4)


@pytest.mark.parametrize("act", ["none", "silu", "gelu", "swiglu"])
def test_linear_oracle_against_differentiation(act):
    """The oracle's gradients are the derivatives of its output (in 64 bits throughout: the
    roundings are in its bounds alone)."""
    g = torch.Generator().manual_seed(0)

    def normal(*s):
        return torch.randn(*s, generator=g, dtype=torch.float64)

    rows = 12 if act == "swiglu" else 6
    v = dict(x=normal(5, 7), weight=normal(rows, 7), bias=normal(rows), residual=normal(5, 6))
    d = normal(5, 6)
    want = O.linear(*v.values(), act, d)
    leaves = {k: t.clone().requires_grad_() for k, t in v.items()}
    out = O.linear(*leaves.values(), act)["out"][0]
    for k, t in zip(leaves, torch.autograd.grad(out, list(leaves.values()), d)):
        assert torch.allclose(want["d" + k][0], t, rtol=1e-10, atol=1e-12), k
    z = v["x"] @ v["weight"].T + v["bias"]
    plain = {"none": lambda: z, "silu": lambda: torch.nn.functional.silu(z),
             "gelu": lambda: torch.nn.functional.gelu(z, approximate="tanh"),
             "swiglu": lambda: torch.nn.functional.silu(z[:, :6]) * z[:, 6:]}[act]()
    assert torch.allclose(out.detach(), plain + v["residual"], rtol=1e-10)


@pytest.mark.parametrize("op", ["modulate", "gate", "gate_modulate"])
def test_norm_oracle_against_differentiation(op):
    """The oracle's gradients are the derivatives of its outputs."""
    g = torch.Generator().manual_seed(0)

    def normal(*s):
        return torch.randn(*s, generator=g, dtype=torch.float64)

    B, N, C, G = 2, 9, 10, 3
    ids = torch.tensor([[0, 0, 1, -1, 2, 2, 0, 1, 5], [2, 2, 2, 0, 0, 1, 1, -1, -1]])
    for docs in (None, ids):
        shape = (B, C) if docs is None else (B, G, C)
        v = dict(x=normal(B, N, C), weight=1 + 0.2 * normal(C), cond=normal(*shape))
        if op != "modulate":
            v["residual"] = normal(B, N, C)
        if op == "gate_modulate":
            v.update(next_weight=normal(C), next_scale=normal(*shape))
        d, dh = normal(B, N, C), normal(B, N, C)
        want = O.norms(op, doc_ids=docs, eps=1e-5, dout=d, dhidden=dh, **{"residual": None, **v}, ) if op != "modulate" \
            else O.norms(op, doc_ids=docs, eps=1e-5, dout=d, **v)
        leaves = {k: t.clone().requires_grad_() for k, t in v.items()}
        out = O.norms(op, doc_ids=docs, eps=1e-5, **leaves)
        pairs = [("out", d)] + ([("hidden", dh)] if op == "gate_modulate" else [])
        grads = torch.autograd.grad([out[k][0] for k, _ in pairs], list(leaves.values()), [t for _, t in pairs])
        for k, t in zip(leaves, grads):
            if op == "gate" and k == "residual":
                assert torch.equal(t, d)
            else:
                assert torch.allclose(want["d" + k][0], t, rtol=1e-10, atol=1e-12), (op, k)


def test_allowed_is_half_a_step():
    """The rounding of a value is within what is allowed, twice that is not."""
    g = torch.Generator().manual_seed(3)
    x = torch.randn(5000, generator=g, dtype=torch.float64) * torch.logspace(-6, 4, 5000, dtype=torch.float64)
    for dtype in (torch.bfloat16, torch.float16, torch.float32):
        y = x.to(dtype)
        assert O.worst(y, x, torch.zeros_like(x)) <= 1.0
        up = torch.nextafter(y.float(), torch.tensor(float("inf"))) if dtype == torch.float32 else \
            (y.view(torch.int16) + 1).view(dtype)
        assert O.worst(up, x, torch.zeros_like(x)) > 1.0
    assert O.worst(torch.tensor([float("nan")]), torch.tensor([1.0], dtype=torch.float64), torch.zeros(1)) == float("inf")


def _calls(params=torch.float32):
    """Every operator on CPU tensors, with all of its arguments: (op, function of its tensors,
    tensors)."""
    B, N, C, G = 2, 6, 16, 3
    ids = torch.zeros(B, N, dtype=torch.int32)

    def t(*shape, dtype=params):
        return torch.zeros(*shape, dtype=dtype)

    x, r = t(B, N, C, dtype=torch.bfloat16), t(B, N, C, dtype=torch.bfloat16)
    rows = t(2 * C, C, dtype=torch.bfloat16)
    return [("rms_norm_modulate", lambda *a: F.rms_norm_modulate(*a, doc_ids=ids), (x, t(C), t(B, G, C))),
            ("rms_norm_gate_residual", lambda *a: F.rms_norm_gate_residual(*a, doc_ids=ids),
             (r, x, t(C), t(B, G, C))),
            ("rms_norm_gate_residual_modulate", lambda *a: F.rms_norm_gate_residual_modulate(*a, doc_ids=ids),
             (r, x, t(C), t(B, G, C), t(C), t(B, G, C))),
            ("fused_linear", lambda *a: F.fused_linear(*a, activation="swiglu"), (x, rows, t(2 * C), r))]


@pytest.mark.parametrize("i", range(4))
def test_tangents_are_refused(i):
    """Forward-mode differentiation raises instead of returning a result without a tangent,
    whichever argument carries one; the registered ops too."""
    from torch.autograd import forward_ad
    name, fn, args = _calls()[i]
    for j, a in enumerate(args):
        with forward_ad.dual_level():
            dual = forward_ad.make_dual(a, torch.ones_like(a))
            call = args[:j] + (dual,) + args[j + 1:]
            with pytest.raises(NotImplementedError, match="forward-mode"):
                fn(*call)
            tail = ("swiglu", False) if name == "fused_linear" else (None, 1e-5)
            with pytest.raises(NotImplementedError, match="forward-mode"):
                getattr(torch.ops.futudiffu_ii, name)(*call, *tail)
            with pytest.raises((NotImplementedError, RuntimeError)):
                fn(*args[:j], dual.requires_grad_(), *args[j + 1:])
        with pytest.raises((NotImplementedError, RuntimeError)):
            torch.func.jvp(lambda t: fn(*args[:j], t, *args[j + 1:]), (a,), (torch.ones_like(a),))


def test_tangents_of_gradients_are_refused():
    from torch.autograd import forward_ad
    op = torch.ops.futudiffu_ii
    x, w = torch.zeros(2, 6, 16, dtype=torch.bfloat16), torch.zeros(16, 16, dtype=torch.bfloat16)
    with forward_ad.dual_level():
        d = forward_ad.make_dual(x, torch.ones_like(x))
        for call in (lambda: op.rms_norm_modulate_backward(d, x, None, None, None, 1e-5, [True] * 3),
                     lambda: op.rms_norm_gate_residual_backward(d, x, None, None, None, 1e-5, [True] * 3),
                     lambda: op.rms_norm_gate_residual_modulate_backward(x, d, x, x, None, None, None, None, None, 1e-5,
                                                                         [True] * 6),
                     lambda: op.fused_linear_backward(d, x, w, None, None, "none", [True] * 3)):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                call()


@pytest.mark.parametrize("grads", [False, True])
def test_a_trace_records_the_operators(grads):
    """Traced, a call is its op and a gradient the op's gradient, not the allocations of their
    results."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    from torch.fx.experimental.proxy_tensor import make_fx
    with FakeTensorMode(allow_non_fake_inputs=True):
        for name, fn, args in _calls(torch.bfloat16):
            if grads:
                args = tuple(a.requires_grad_() for a in args)

            def traced(*a):
                out = fn(*a)
                out = out if isinstance(out, tuple) else (out,)
                return torch.autograd.grad(out, a, [torch.ones_like(o) for o in out]) if grads else out

            got = {str(n.target) for n in make_fx(traced)(*args).graph.nodes if n.op == "call_function"}
            want = {f"futudiffu_ii.{name}.default"} | ({f"futudiffu_ii.{name}_backward.default"} if grads else set())
            assert want <= got and not any("aten.empty" in t for t in got), (name, got)


def test_dispatch_modes_see_the_operators():
    """A dispatch mode (counters, memory tools, checkpoint policies) sees each call and each
    gradient as its op."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    from torch.utils._python_dispatch import TorchDispatchMode

    class Seen(TorchDispatchMode):
        def __init__(self):
            super().__init__()
            self.ops = []

        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            self.ops.append(func.name())
            return func(*args, **(kwargs or {}))

    with FakeTensorMode():
        for name, fn, args in _calls():
            args = tuple(a.requires_grad_() for a in args)
            with Seen() as seen:
                out = fn(*args)
            assert f"futudiffu_ii::{name}" in seen.ops
            out = out if isinstance(out, tuple) else (out,)
            with Seen() as seen:
                grads = torch.autograd.grad(out, args, [torch.ones_like(o) for o in out])
            assert f"futudiffu_ii::{name}_backward" in seen.ops
            assert [g.shape for g in grads] == [a.shape for a in args] and [g.dtype for g in grads] == [a.dtype for a in args]


@pytest.mark.parametrize("i", range(4))
def test_gradients_of_the_ops_are_not_differentiated(i):
    """The registered ops refuse a second derivative as the functions do.  A residual's gradient
    is the incoming one, which may be differentiated."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        name, _, args = _calls(torch.bfloat16)[i]
        tail = (None, 1e-5)
        if name == "fused_linear":
            tail = ("swiglu", True)
        else:
            args = tuple(a[:, 0] if a.shape[1:2] == (3,) else a for a in args)
        residual = {"rms_norm_gate_residual": 0, "fused_linear": 3}.get(name)
        for j, a in enumerate(args):
            leaf = a.detach().requires_grad_()

            def grad(**kw):
                out = getattr(torch.ops.futudiffu_ii, name)(*args[:j], leaf, *args[j + 1:], *tail)
                out = out[0] if isinstance(out, (tuple, list)) else out
                return torch.autograd.grad(out, leaf, torch.ones_like(out), **kw)[0]

            assert grad().shape == a.shape
            if j == residual:
                assert grad(create_graph=True).shape == a.shape
            else:
                with pytest.raises(RuntimeError, match="create_graph"):
                    grad(create_graph=True)


def test_gradient_ops_are_not_differentiated():
    """Nor does a gradient op called by itself give a derivative without its own terms."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    op = torch.ops.futudiffu_ii
    with FakeTensorMode():
        x, w = torch.zeros(2, 6, 16, dtype=torch.bfloat16), torch.zeros(16, 16, dtype=torch.bfloat16)
        d = x.clone().requires_grad_()
        for out in (op.rms_norm_modulate_backward(d, x, None, None, None, 1e-5, [True] * 3),
                    op.rms_norm_gate_residual_backward(d, x, None, None, None, 1e-5, [True] * 3),
                    op.rms_norm_gate_residual_modulate_backward(x, d, x, x, None, None, None, None, None, 1e-5,
                                                                [True] * 6),
                    op.fused_linear_backward(d, x, w, None, None, "none", [True] * 3)):
            with pytest.raises(RuntimeError, match="cannot be differentiated"):
                torch.autograd.grad(out[0], d, torch.ones_like(out[0]))
