"""The operators around the attention, without a GPU: refusals of the Python functions and
of the C entries, workspace sizes, and the 64-bit oracle against differentiation."""

import pytest
import torch

import futudiffu_amd as F
from futudiffu_amd import _lib, block_ops
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
    check_w, check_c, docs = block_ops._check_weight, block_ops._check_cond, block_ops._check_docs
    for w in (torch.zeros(7), torch.zeros(1, 8), torch.zeros(8, dtype=torch.float16), torch.zeros(8, dtype=torch.float64)):
        with pytest.raises(ValueError, match="weight must be"):
            check_w("weight", w, x, 8)
    for k, d in ((torch.zeros(8), False), (torch.zeros(1, 8), False), (torch.zeros(2, 3, 8), False),
                 (torch.zeros(2, 8), True), (torch.zeros(1, 3, 8), True), (torch.zeros(2, 0, 8), True),
                 (torch.zeros(2, 8, dtype=torch.float16), False)):
        with pytest.raises(ValueError, match="gate must be"):
            check_c("gate", k, x, 2, 8, d)
    for ids in (torch.zeros(2, 3, dtype=torch.int32), torch.zeros(4, dtype=torch.int32)):
        with pytest.raises(ValueError, match="doc_ids must be"):
            docs(ids, x, 2, 4)
    for t in (torch.zeros(2, 4), torch.zeros(2, 4, dtype=torch.bool)):
        with pytest.raises(ValueError, match="integers"):
            docs(t, x, 2, 4)
    for r in (x[:1], x.half(), x[..., :4]):
        with pytest.raises(ValueError, match="residual must be"):
            block_ops._tokens("residual", r, x)


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
