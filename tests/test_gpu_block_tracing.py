"""GPU: the block operators (futudiffu_amd/block_ops.py) under tracers, dispatch modes and
function transforms, and on lazy views: the results of the plain calls, or a refusal."""

import pytest
import torch

pytestmark = pytest.mark.gpu

B, N, C, G = 2, 6, 72, 3
BF, F32 = torch.bfloat16, torch.float32


def _calls(device, seed=0):
    """Every operator with all of its arguments: (op, function of its tensors, tensors)."""
    import futudiffu_amd as F
    g = torch.Generator().manual_seed(seed)

    def t(*shape, dtype=BF):
        return torch.randn(*shape, generator=g).to(dtype).to(device)

    ids = torch.tensor([[0, 0, 2, 1, -1, 1], [1, 5, 0, 0, 2, 2]], dtype=torch.int32, device=device)
    x, r, w, k, w2, k2 = t(B, N, C), t(B, N, C), t(C), t(B, G, C), t(C), t(B, G, C)
    return [("rms_norm_modulate", lambda *a: F.rms_norm_modulate(*a, doc_ids=ids), (x, w, k)),
            ("rms_norm_gate_residual", lambda *a: F.rms_norm_gate_residual(*a, doc_ids=ids), (r, x, w, k)),
            ("rms_norm_gate_residual_modulate",
             lambda *a: F.rms_norm_gate_residual_modulate(*a, doc_ids=ids), (r, x, w, k, w2, k2)),
            ("fused_linear", lambda *a: F.fused_linear(*a, activation="swiglu"),
             (x, t(2 * C, C), t(2 * C, dtype=F32), r))]


OPS = range(4)


def _outs(out):
    return out if isinstance(out, tuple) else (out,)


def _grads(fn, args, douts=None):
    args = tuple(a.detach().requires_grad_() for a in args)
    out = _outs(fn(*args))
    return torch.autograd.grad(out, args, [torch.ones_like(o) for o in out] if douts is None else douts)


def _equal(got, want):
    torch.cuda.synchronize()
    return len(got) == len(want) and all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("i", OPS)
def test_traced_graphs_compute(cuda, i):
    """A graph traced on one input gives another input's results: outputs and gradients."""
    from torch.fx.experimental.proxy_tensor import make_fx
    name, fn, args = _calls(cuda)[i]
    new = _calls(cuda, seed=1)[i][2]
    want = _outs(fn(*new))
    for traced in (make_fx(lambda *a: _outs(fn(*a)))(*args),
                   torch.jit.trace(lambda *a: _outs(fn(*a)), args, check_trace=False)):
        assert _equal(traced(*new), want)
    traced = make_fx(lambda *a: tuple(_grads(fn, a)))(*args)
    assert any(f"{name}_backward" in str(n.target) for n in traced.graph.nodes)
    assert _equal(traced(*new), _grads(fn, new))


@pytest.mark.parametrize("i", OPS)
def test_traced_gradients_of_an_eager_call(cuda, i):
    """The forward as it is, its gradients under a dispatch mode: the mode sees the op, and the
    gradients are the same."""
    from torch.utils._python_dispatch import TorchDispatchMode
    seen = []

    class Seen(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            seen.append(func.name())
            return func(*args, **(kwargs or {}))

    name, fn, args = _calls(cuda)[i]
    leaves = tuple(a.detach().requires_grad_() for a in args)
    out = _outs(fn(*leaves))
    d = [torch.ones_like(o) for o in out]
    with Seen():
        got = torch.autograd.grad(out, leaves, d)
    assert f"futudiffu_ii::{name}_backward" in seen
    assert _equal(got, _grads(fn, args))


@pytest.mark.parametrize("i", OPS)
def test_lazy_views(cuda, i):
    """A lazily negated view and zeros without storage are the values they stand for, in the
    arguments and in the gradients that come in."""
    name, fn, args = _calls(cuda)[i]
    for j, a in enumerate(args):
        for lazy, plain in ((torch._neg_view(a), -a),
                            (torch._efficientzerotensor(a.shape, dtype=a.dtype, device=cuda), torch.zeros_like(a))):
            print(name, j, lazy.is_neg(), lazy._is_zerotensor(), flush=True)
            put = lambda t: args[:j] + (t,) + args[j + 1:]  # noqa: E731
            assert _equal(_outs(fn(*put(lazy))), _outs(fn(*put(plain))))
    d = [torch.randn_like(o) for o in _outs(fn(*args))]
    assert _equal(_grads(fn, args, [torch._neg_view(t) for t in d]), _grads(fn, args, [-t for t in d]))


@pytest.mark.parametrize("i", OPS)
def test_vmap_is_a_loop_over_samples(cuda, i):
    name, fn, args = _calls(cuda)[i]
    at = {"rms_norm_modulate": 0, "rms_norm_gate_residual": 1, "rms_norm_gate_residual_modulate": 1, "fused_linear": 0}[name]
    xs = torch.stack([args[at], 2 * args[at], -args[at]])
    got = torch.vmap(lambda t: _outs(fn(*args[:at], t, *args[at + 1:])))(xs)
    for s in range(3):
        want = _outs(fn(*args[:at], xs[s], *args[at + 1:]))
        assert _equal([g[s] for g in got], want)


@pytest.mark.parametrize("i", OPS)
def test_transforms_without_a_formula_raise(cuda, i):
    """Forward mode, and reverse mode by a transform, raise: no zero tangent, no lost gradient."""
    from torch.autograd import forward_ad
    name, fn, args = _calls(cuda)[i]
    for j, a in enumerate(args):
        put = lambda t: _outs(fn(*args[:j], t, *args[j + 1:]))  # noqa: E731
        with pytest.raises(NotImplementedError, match="forward-mode"):
            torch.func.jvp(put, (a,), (torch.ones_like(a),))
        with pytest.raises(RuntimeError):
            torch.func.grad(lambda t: put(t)[0].float().sum())(a)
        with forward_ad.dual_level(), pytest.raises(NotImplementedError, match="forward-mode"):
            put(forward_ad.make_dual(a, torch.ones_like(a)))


@pytest.mark.parametrize("i", OPS)
def test_gradients_of_the_ops_are_not_differentiated(cuda, i):
    """The registered ops, called directly, refuse create_graph=True as the functions do; without
    it their gradients are the functions'."""
    name, fn, args = _calls(cuda)[i]
    ids = torch.tensor([[0, 0, 2, 1, -1, 1], [1, 5, 0, 0, 2, 2]], dtype=torch.int32, device=cuda)
    tail = ("swiglu", True) if name == "fused_linear" else (ids, 1e-5)
    leaves = tuple(a.detach().requires_grad_() for a in args)

    def outs():
        out = getattr(torch.ops.futudiffu_ii, name)(*leaves, *tail)
        return out[:1] if name == "fused_linear" else _outs(out)

    d = [torch.randn_like(o) for o in _outs(fn(*args))]
    assert _equal(torch.autograd.grad(outs(), leaves, d), _grads(fn, args, d))
    with pytest.raises(RuntimeError, match="create_graph"):
        torch.autograd.grad(outs(), leaves, d, create_graph=True)


@pytest.mark.parametrize("i", OPS)
def test_gradients_through_vmap(cuda, i):
    """A gradient that is taken outside of vmap: the samples' own."""
    name, fn, args = _calls(cuda)[i]
    for at in range(len(args)):
        put = lambda t: _outs(fn(*args[:at], t, *args[at + 1:]))  # noqa: E731
        xs = torch.stack([args[at], 2 * args[at], -args[at]]).requires_grad_()
        out = torch.vmap(put)(xs)
        got, = torch.autograd.grad(out, xs, [torch.ones_like(o) for o in out])
        for s in range(3):
            assert _equal([got[s]], _grads(put, (xs[s],))), (name, at)
