"""GPU: the norms around the attention (futudiffu_amd/block_ops.py) against their 64-bit
definition (oracle/block_oracle.py), outputs and every gradient.

An error is measured in what is allowed: the bound on 32-bit arithmetic in any order, then
one rounding to the output's type.
"""

import pytest
import torch

from oracle import block_oracle as O

pytestmark = pytest.mark.gpu

EPS = 1e-5
BF, FP, F32 = torch.bfloat16, torch.float16, torch.float32


def _ids(lengths, n, batch):
    ids = torch.full((batch, n), -1, dtype=torch.int32)
    for b in range(batch):
        at = 0
        for i, x in enumerate(lengths):
            ids[b, at:at + x] = (i + b) % len(lengths)
            at += x
    return ids


def _inputs(op, B, N, C, dtype, params, docs, seed=0):
    """On the CPU; ``docs``: None, or (rows a batch item, ids [B, N])."""
    g = torch.Generator().manual_seed(seed)

    def normal(*shape, to=dtype, s=1.0, o=0.0):
        return (o + s * torch.randn(*shape, generator=g)).to(to)

    rows = (B, C) if docs is None else (B, docs[0], C)
    v = dict(x=normal(B, N, C, s=1.5), weight=normal(C, to=params, s=0.3, o=1.0), cond=normal(*rows, to=params, s=0.5),
             dout=normal(B, N, C))
    if op != "modulate":
        v["residual"] = normal(B, N, C, s=2.0)
    if op == "gate_modulate":
        v["next_weight"] = normal(C, to=params, s=0.3, o=1.0)
        v["next_scale"] = normal(*rows, to=params, s=0.5)
        v["dhidden"] = normal(B, N, C)
    v["doc_ids"] = None if docs is None else docs[1]
    return v


ORDER = {"modulate": ("x", "weight", "cond"), "gate": ("residual", "x", "weight", "cond"),
         "gate_modulate": ("residual", "x", "weight", "cond", "next_weight", "next_scale")}


def _call(op, v, eps=EPS):
    import futudiffu_amd as F
    fn = {"modulate": F.rms_norm_modulate, "gate": F.rms_norm_gate_residual,
          "gate_modulate": F.rms_norm_gate_residual_modulate}[op]
    got = fn(*(v[k] for k in ORDER[op]), doc_ids=v["doc_ids"], eps=eps)
    return {"hidden": got[0], "out": got[1]} if op == "gate_modulate" else {"out": got}


def _with_grads(op, v, eps=EPS, leaves=None):
    v = dict(v)
    leaves = [k for k in (leaves or ORDER[op]) if v[k] is not None]
    for k in leaves:
        v[k] = v[k].detach().requires_grad_()
    out = _call(op, v, eps)
    names = ["out", "hidden"] if op == "gate_modulate" else ["out"]
    grads = torch.autograd.grad([out[k] for k in names], [v[k] for k in leaves], [v["d" + k] for k in names])
    out = {k: t.detach() for k, t in out.items()}
    out.update({"d" + k: t for k, t in zip(leaves, grads)})
    return out


def _to(v, device):
    return {k: None if t is None else t.to(device) for k, t in v.items()}


def _want(op, v, eps=EPS):
    want = O.norms(op, v["x"], v["weight"], v["cond"], v["doc_ids"], eps, v.get("residual"), v.get("next_weight"),
                   v.get("next_scale"), v["dout"], v.get("dhidden"))
    if op == "gate":
        want["dresidual"] = (v["dout"].double(), torch.zeros_like(v["dout"], dtype=torch.float64))
    return want


def _check(got, want, case=""):
    torch.cuda.synchronize()
    for name, g in got.items():
        exact, bound = want[name]
        w = O.worst(g.cpu(), exact.cpu(), bound.cpu())
        assert w <= 1.0, f"{case} {name}: {w:.3g} of what is allowed"


SHAPES = [
    (1, 1, 8), (1, 1, 1), (2, 3, 7), (1, 33, 64), (3, 17, 1000), (1, 65, 1001), (2, 130, 1024), (1, 9, 1032),
    (2, 40, 3840), (1, 31, 3841), (1, 5, 4104), (1, 19, 8192), (2, 3, 8191), (1, 700, 72),
]


@pytest.mark.parametrize("B,N,C", SHAPES)
@pytest.mark.parametrize("op", ["modulate", "gate", "gate_modulate"])
def test_outputs_and_gradients(cuda, op, B, N, C):
    """Every width class (one wave, four and eight a token; runs of eight channels and odd
    widths), one conditioning row a batch item; both 16-bit types, fp32 parameters too."""
    for dtype, params in ((BF, BF), (FP, F32)):
        print(op, B, N, C, dtype, params, flush=True)
        v = _inputs(op, B, N, C, dtype, params, None, seed=N + C)
        got = _with_grads(op, _to(v, cuda))
        assert all(got[k].dtype == dtype for k in ("out", "dx"))
        assert got["dweight"].dtype == got["dcond"].dtype == params
        _check(got, _want(op, v))
        plain = _call(op, _to(v, cuda))  # without gradients: the same bits
        for k, t in plain.items():
            assert torch.equal(t.view(torch.int16), got[k].view(torch.int16))


DOCS = [
    (1, 300, 256, (100, 150), "contiguous"),      # 50 tokens of no document at the end
    (2, 1100, 72, (500, 333, 267), "contiguous"),  # rotated rows in the second batch item
    (1, 97, 3840, (40, 57), "contiguous"),
    (1, 600, 136, (600,), "interleaved"),          # 5 documents in turn: every chunk holds them all
    (1, 50, 1001, (1,) * 50, "contiguous"),        # a document a token
    (1, 64, 64, (), "contiguous"),                 # no token has a document
    (1, 64, 64, (64,), "outside"),                 # ids beyond the rows, and below 0
]


@pytest.mark.parametrize("B,N,C,lengths,kind", DOCS)
@pytest.mark.parametrize("op", ["modulate", "gate", "gate_modulate"])
def test_documents(cuda, op, B, N, C, lengths, kind):
    if kind == "interleaved":
        rows, ids = 5, (torch.arange(N, dtype=torch.int32) % 5).expand(B, N).contiguous()
    elif kind == "outside":
        rows, ids = 2, torch.tensor([0, 5, -7, 1, 2 ** 31 - 1, -2 ** 31], dtype=torch.int32).repeat(B, 11)[:, :N].contiguous()
    else:
        rows, ids = max(1, len(lengths)), _ids(lengths, N, B)
    for dtype, params in ((BF, F32), (FP, FP)):
        print(op, B, N, C, kind, dtype, flush=True)
        v = _inputs(op, B, N, C, dtype, params, (rows, ids), seed=C)
        _check(_with_grads(op, _to(v, cuda)), _want(op, v))


@pytest.mark.parametrize("op", ["modulate", "gate", "gate_modulate"])
def test_absent_parameters(cuda, op):
    """No weight (ones), no scale (0), no gate (1); gradients of the rest alone."""
    for keep in ((), ("weight",), ("cond",), ("next_weight",), ("next_scale",)):
        if op != "gate_modulate" and keep and keep[0].startswith("next"):
            continue
        v = _inputs(op, 2, 21, 520, BF, BF, None, seed=5)
        want = {k: None if k in ("weight", "cond", "next_weight", "next_scale") and k not in keep else t
                for k, t in v.items()}
        print(op, keep, flush=True)
        _check(_with_grads(op, _to(want, cuda)), _want(op, want))


@pytest.mark.parametrize("op", ["modulate", "gate", "gate_modulate"])
def test_strides_and_alignment(cuda, op):
    """Views: a channel slice of a wider tensor, an offset of one element, transposed
    channels, expanded conditioning rows, chunks of one projection; the rows around the
    outputs stay as they were (fresh tensors)."""
    B, N, C = 2, 37, 264
    v = _to(_inputs(op, B, N, C, BF, BF, None, seed=9), cuda)
    want = _want(op, {k: None if t is None else t.cpu() for k, t in v.items()})
    ref = _with_grads(op, v)
    _check(ref, want)

    def wide(t, off):
        w = torch.zeros(*t.shape[:-1], C + 40, dtype=t.dtype, device=t.device)
        w[..., off:off + C] = t
        return w[..., off:off + C]

    def swapped(t):
        return t.transpose(-1, -2).contiguous().transpose(-1, -2)

    tokens = [k for k in ("x", "residual", "dout", "dhidden") if k in v]
    for name, how in (("wide", lambda t: wide(t, 8)), ("offset", lambda t: wide(t, 1)), ("swapped", swapped),
                      ("batch-strided", lambda t: torch.stack([t, t], 1)[:, 0])):
        u = dict(v, **{k: how(v[k]) for k in tokens})
        got = _with_grads(op, u)
        print(op, name, flush=True)
        _check(got, want, name)
    conds = [k for k in ("cond", "next_scale") if k in v]
    proj = torch.cat([v[k] for k in conds] * 2, -1)
    u = dict(v, **dict(zip(conds, proj.chunk(2 * len(conds), -1))))
    _check(_with_grads(op, u), want, "chunks")
    u = dict(v, **{k: v[k][:1].expand(B, C) for k in conds})
    _check(_with_grads(op, u), _want(op, {k: None if t is None else t.cpu() for k, t in u.items()}), "expanded")


def test_two_dimensional_and_empty(cuda):
    import futudiffu_amd as F
    v = _to(_inputs("gate_modulate", 1, 11, 96, BF, BF, None, seed=2), cuda)
    three = _call("gate_modulate", v)
    flat = {k: t[0] if k in ("x", "residual") else t for k, t in v.items() if t is not None}
    two = _call("gate_modulate", dict(flat, doc_ids=None))
    assert all(torch.equal(two[k], three[k][0]) for k in two)
    ids = torch.zeros(11, dtype=torch.int64, device=cuda)
    got = F.rms_norm_modulate(flat["x"], flat["weight"], v["cond"][:, None], doc_ids=ids)
    assert torch.equal(got, F.rms_norm_modulate(v["x"], v["weight"], v["cond"])[0])
    for op in ORDER:
        for B, N in ((1, 0), (0, 4)):
            e = _to(_inputs(op, B, N, 96, BF, BF, None), cuda)
            got = _with_grads(op, e)
            assert got["out"].shape == (B, N, 96) and got["dx"].shape == (B, N, 96)
            assert not got["dweight"].any() and got["dcond"].shape == (B, 96) and not got["dcond"].any()


@pytest.mark.parametrize("op", ["modulate", "gate", "gate_modulate"])
def test_not_finite_and_zero_rows(cuda, op):
    """A token with an infinity or NaN spoils its own row alone; a row of zeros is fine."""
    v = _inputs(op, 1, 40, 256, BF, BF, None, seed=3)
    clean = _call(op, _to(v, cuda))
    bad = dict(v, x=v["x"].clone())
    bad["x"][0, 3, 7] = float("inf")
    bad["x"][0, 5, 9] = float("nan")
    bad["x"][0, 8] = 0
    got = _call(op, _to(bad, cuda))
    for k in got:
        g, c = got[k][0].float(), clean[k][0].float()
        assert torch.isnan(g[3]).any() and torch.isnan(g[5]).all()
        keep = [i for i in range(40) if i not in (3, 5, 8)]
        assert torch.equal(g[keep], c[keep]) and torch.isfinite(g[8]).all()
        if k != "out" or op == "gate":
            assert torch.equal(got[k][0, 8], v["residual"][0, 8].to(got[k].device))


@pytest.mark.parametrize("op", ["gate", "gate_modulate"])
def test_padding_behind_a_gate_is_not_read(cuda, op):
    """Whatever x holds in tokens of no document: the output is the residual's, and no
    gradient sees it."""
    ids = _ids((70, 50), 150, 1)
    v = _inputs(op, 1, 150, 1001, BF, F32, (2, ids), seed=12)
    v["x"][0, 120:130] = float("nan")
    v["x"][0, 130:140] = float("inf")
    for eps in (EPS, 0.0):
        got = _with_grads(op, _to(v, cuda), eps)
        _check(got, _want(op, v, eps))
        assert all(torch.isfinite(t).all() for t in got.values()) and not got["dx"][0, 120:].any()


def test_gradients_against_differences(cuda):
    """Central differences of the operator itself along random directions, in fp32 sums of
    fp16 outputs: the step is 2^-4 of the inputs' scale, so the difference's own error is the
    outputs' rounding (half a step of 2^-11 each, independent, over a sum of their squares)
    and the third-order term."""
    op = "gate_modulate"
    v = _inputs(op, 1, 64, 128, FP, F32, (2, _ids((30, 30), 64, 1)), seed=11)
    d = _to(v, cuda)
    got = _with_grads(op, d)
    g = torch.Generator().manual_seed(1)
    for leaf in ("weight", "cond", "next_weight", "next_scale"):
        step = torch.randn(v[leaf].shape, generator=g).to(cuda) * 2.0 ** -4
        hi, lo = (_call(op, dict(d, **{leaf: d[leaf] + s * step})) for s in (1, -1))
        num = sum(((hi[k].double() - lo[k].double()) * d["d" + k].double()).sum() for k in hi) / 2
        ana = (got["d" + leaf].double() * step.double()).sum()
        # each output is off by at most 2^-11 of itself (both sides), summed in quadrature x 4
        noise = 4 * sum(((hi[k].double() * 2.0 ** -11 * d["d" + k].double()) ** 2).sum() for k in hi).sqrt()
        cubic = 0.0
        if leaf in ("weight", "cond"):  # out depends on them through the second norm
            half = [_call(op, dict(d, **{leaf: d[leaf] + s * step / 2})) for s in (1, -1)]
            num2 = sum(((half[0][k].double() - half[1][k].double()) * d["d" + k].double()).sum() for k in hi)
            cubic = abs(float(num - num2)) * 4 / 3
        assert abs(float(num - ana)) <= float(noise) + cubic, (leaf, float(num), float(ana), float(noise), cubic)


@pytest.mark.parametrize("op", ["modulate", "gate", "gate_modulate"])
def test_repeatable_and_partial_gradients(cuda, op):
    """The same bits every time, and whichever gradients are asked for."""
    v = _to(_inputs(op, 2, 333, 1024, BF, F32, (3, _ids((100, 100, 133), 333, 2)), seed=4), cuda)
    ref = _with_grads(op, v)
    for _ in range(3):
        again = _with_grads(op, v)
        assert all(torch.equal(again[k], ref[k]) for k in ref)
    for leaf in ORDER[op]:
        one = _with_grads(op, v, leaves=(leaf,))
        assert torch.equal(one["d" + leaf], ref["d" + leaf]), leaf


def test_other_stream_and_overlapping_calls(cuda):
    v = _to(_inputs("gate_modulate", 1, 500, 2048, BF, BF, None, seed=6), cuda)
    u = _to(_inputs("gate_modulate", 1, 480, 1536, BF, BF, None, seed=7), cuda)
    ref, ref_u = _with_grads("gate_modulate", v), _with_grads("gate_modulate", u)
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(5):
        with torch.cuda.stream(s1):
            a = _with_grads("gate_modulate", v)
        with torch.cuda.stream(s2):
            b = _with_grads("gate_modulate", u)
        torch.cuda.synchronize()
        assert all(torch.equal(a[k], ref[k]) for k in ref) and all(torch.equal(b[k], ref_u[k]) for k in ref_u)


@pytest.mark.parametrize("op", ["modulate", "gate", "gate_modulate"])
def test_captured_step_replays(cuda, op):
    """Forward and backward in one graph, replayed on new inputs between eager work."""
    ids = _ids((100, 150), 300, 1)
    v = _to(_inputs(op, 1, 300, 512, BF, BF, (2, ids), seed=8), cuda)
    static = {k: None if t is None else t.clone() for k, t in v.items()}
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        _with_grads(op, static)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        got = _with_grads(op, static)
    for seed in (20, 21, 22):
        new = _to(_inputs(op, 1, 300, 512, BF, BF, (2, ids), seed=seed), cuda)
        for k, t in new.items():
            if t is not None:
                static[k].copy_(t)
        graph.replay()
        torch.cuda.synchronize()
        want = _with_grads(op, new)
        assert all(torch.equal(got[k], want[k]) for k in want), [k for k in want if not torch.equal(got[k], want[k])]


@pytest.mark.parametrize("op", ["modulate", "gate", "gate_modulate"])
def test_ops_check_and_compile(cuda, op):
    name = {"modulate": "rms_norm_modulate", "gate": "rms_norm_gate_residual",
            "gate_modulate": "rms_norm_gate_residual_modulate"}[op]
    v = _to(_inputs(op, 2, 20, 136, BF, F32, (2, _ids((8, 9), 20, 2)), seed=1), cuda)
    args = [v[k].requires_grad_() for k in ORDER[op]] + [v["doc_ids"], EPS]
    torch.library.opcheck(getattr(torch.ops.futudiffu_ii, name).default, tuple(args),
                          test_utils=("test_schema", "test_autograd_registration", "test_faketensor",
                                      "test_aot_dispatch_static"))
    want = _with_grads(op, v)
    compiled = torch.compile(lambda *a: tuple(_call(op, dict(v, **dict(zip(ORDER[op], a)))).values()),
                             backend="aot_eager", fullgraph=True)
    got = compiled(*(v[k].detach().requires_grad_() for k in ORDER[op]))
    assert all(torch.equal(a, b) for a, b in zip(got, (want[k] for k in (["hidden", "out"] if op == "gate_modulate" else ["out"]))))


@pytest.mark.parametrize("op", ["modulate", "gate", "gate_modulate"])
def test_ids_past_32_bits_are_of_no_document(cuda, op):
    v = _to(_inputs(op, 1, 40, 72, BF, F32, None, seed=2), cuda)
    ids = torch.arange(40, device=cuda).view(1, 40) % 3
    for k in ("cond", "next_scale"):
        if v.get(k) is not None:
            v[k] = torch.stack([v[k] * f for f in (1.0, -0.5)], 1)
    v["doc_ids"] = ids.int().masked_fill(ids == 2, -1)
    want = _with_grads(op, v)
    for far in ((1 << 32) + 1, -(1 << 32), 1 << 62):
        v["doc_ids"] = ids.masked_fill(ids == 2, far)
        got = _with_grads(op, v)
        assert all(torch.equal(got[k], want[k]) for k in want), far


@pytest.mark.parametrize("op", ["modulate", "gate", "gate_modulate"])
def test_gradients_are_not_differentiated(cuda, op):
    v = _to(_inputs(op, 1, 5, 64, BF, BF, None), cuda)
    v["x"] = v["x"].requires_grad_()
    out = _call(op, v)["out"]
    with pytest.raises(RuntimeError, match="create_graph"):
        torch.autograd.grad(out, v["x"], v["dout"], create_graph=True)


def test_offsets_past_32_bits(cuda):
    """Rows of an x and of a gradient beyond 2^32 bytes: all zeros but a few."""
    import futudiffu_amd as F
    C, N = 2048, (1 << 20) + 4100
    at = torch.tensor([0, (1 << 19) - 1, 1 << 19, (1 << 20) - 1, 1 << 20, N - 1])
    v = _inputs("modulate", 1, len(at), C, BF, F32, None, seed=4)
    x, dout = (torch.zeros(1, N, C, dtype=BF, device=cuda) for _ in range(2))
    x[:, at.to(cuda)], dout[:, at.to(cuda)] = v["x"].to(cuda), v["dout"].to(cuda)
    few = _with_grads("modulate", _to(v, cuda))
    v = _to(v, cuda)
    v["x"], v["dout"] = x, dout
    got = _with_grads("modulate", v)
    for k in ("out", "dx"):
        assert torch.equal(got[k][:, at.to(cuda)], few[k]), k
        got[k][:, at.to(cuda)] = 0
        assert got[k].abs().amax().item() == 0, k
    _check({k: got[k] for k in ("dweight", "dcond")}, {k: t for k, t in _want("modulate", _to(_inputs(
        "modulate", 1, len(at), C, BF, F32, None, seed=4), "cpu")).items()})


@pytest.mark.parametrize("B,N,C,lengths", [
    (1, 1500, 200, (3,) * 480),             # documents shorter than a chunk, a few partials each
    (2, 900, 1032, (500, 1, 399)),          # many partials a document, and one
    (1, 270000, 8, (140000, 7, 129000)),    # more chunks than one search takes
    (1, 270000, 8, (900,) * 290),
])
@pytest.mark.parametrize("op", ["modulate", "gate_modulate"])
def test_documents_and_chunks(cuda, op, B, N, C, lengths):
    """The sums of a document over its chunks: every form of the search for them."""
    print(op, B, N, C, len(lengths), flush=True)
    v = _inputs(op, B, N, C, BF, F32, (len(lengths), _ids(lengths, N, B)), seed=N)
    _check(_with_grads(op, _to(v, cuda)), _want(op, v))


@pytest.mark.parametrize("op", ["modulate", "gate", "gate_modulate"])
def test_ids_of_every_integer_type(cuda, op):
    """The same documents from ids of any integer type; one beyond 32 bits, with or without a
    sign, is of no document and does not wrap to one."""
    v = _to(_inputs(op, 2, 40, 72, BF, F32, None, seed=2), cuda)
    ids = torch.arange(80, device=cuda).view(2, 40) % 3  # 2: no document
    for k in ("cond", "next_scale"):
        if v.get(k) is not None:
            v[k] = torch.stack([v[k] * f for f in (1.0, -0.5)], 1)
    v["doc_ids"] = ids.int()
    want = _with_grads(op, v)
    far = {torch.uint8: (255,), torch.int8: (-128, 127), torch.int16: (-2 ** 15, 2 ** 15 - 1), torch.uint16: (2 ** 16 - 1,),
           torch.int32: (-2 ** 31, 2 ** 31 - 1), torch.uint32: (2 ** 31, 2 ** 31 + 1, 2 ** 32 - 1),
           torch.int64: (2 ** 32, 2 ** 32 + 1, -2 ** 32, -2 ** 63 + 1),
           torch.uint64: (2 ** 32, 2 ** 32 + 1, 2 ** 63, 2 ** 63 + 1, 2 ** 64 - 1)}
    for dtype, values in far.items():
        for value in (2, *values):
            print(op, dtype, value, flush=True)
            plain = [[value if i == 2 else i for i in row] for row in ids.tolist()]
            for device in ("cpu", cuda):
                v["doc_ids"] = torch.tensor(plain, dtype=dtype).to(device)
                got = _with_grads(op, v)
                assert all(torch.equal(got[k], want[k]) for k in want), (dtype, value, device)


@pytest.mark.parametrize("op", ["modulate", "gate", "gate_modulate"])
def test_compiled_gradients(cuda, op):
    """The gradients of the compiled function, whose formulas are the ops' own, are the eager
    ones bit for bit: all of them, with parameters absent, and where some leaves alone want one."""
    absent = {"modulate": ("weight", "cond"), "gate": ("weight", "cond"),
              "gate_modulate": ("weight", "cond", "next_weight", "next_scale")}[op]
    docs = (2, _ids((8, 9), 20, 2))
    cases = [((), ORDER[op])] + [((k,), ORDER[op]) for k in absent] + [((), (k,)) for k in ORDER[op]]
    for gone, leaves in cases:
        print(op, gone, leaves, flush=True)
        v = _to(_inputs(op, 2, 20, 136, BF, F32, docs, seed=1), cuda)
        v.update({k: None for k in gone})
        leaves = [k for k in leaves if v[k] is not None]
        want = _with_grads(op, v, leaves=leaves)
        names = [k for k in ORDER[op] if v[k] is not None]

        def fn(*a):
            got = _call(op, dict(v, **dict(zip(names, a))))
            return tuple(got[k] for k in outs)

        outs = ["out", "hidden"] if op == "gate_modulate" else ["out"]
        torch._dynamo.reset()
        args = [v[k].detach().requires_grad_(k in leaves) for k in names]
        out = torch.compile(fn, backend="aot_eager", fullgraph=True)(*args)
        grads = torch.autograd.grad(out, [args[names.index(k)] for k in leaves], [v["d" + k] for k in outs])
        assert all(torch.equal(o, want[k]) for o, k in zip(out, outs))
        for k, g in zip(leaves, grads):
            assert g.dtype == v[k].dtype and torch.equal(g, want["d" + k]), k
        for k in outs if len(outs) > 1 else ():  # one of two outputs alone
            one = [torch.autograd.grad(f(*args)[outs.index(k)], [args[names.index(j)] for j in leaves], v["d" + k],
                                       allow_unused=True)
                   for f in (fn, torch.compile(fn, backend="aot_eager", fullgraph=True))]
            for j, a, b in zip(leaves, *one):
                # behind hidden alone the second norm's parameters are not reached: zeros, or none
                assert torch.equal(torch.zeros_like(v[j]) if a is None else a, torch.zeros_like(v[j]) if b is None else b), (k, j)


@pytest.mark.parametrize("B,N,C,lengths", [
    (1, 270000, 8, None),                   # no documents: every chunk's partial
    (1, 270000, 8, (140000, 7, 129000)),    # more chunks than one search takes, and padding
    (1, 270000, 8, (900,) * 290),
    (2, 30011, 65, 5),                      # 5 documents in turn: every chunk holds them all
    (3, 700, 1032, (500, 1, 150)),
    (2, 333, 4104, (100, 200)),
])
@pytest.mark.parametrize("op", ["modulate", "gate", "gate_modulate"])
def test_parameter_sums_are_exact(cuda, op, B, N, C, lengths):
    """Sums that are exact whatever their order, so that a token lost or taken twice shows at any
    size: x of +-1 and eps 0 (xhat is x), small integers and halves elsewhere, every sum under
    2^24 of its unit.  gate + modulate: r = 0 and a gate of +-1 (hidden is +-1, its norm too), and
    dout in pairs of channels whose products with hidden cancel (its mean with hidden is 0)."""
    print(op, B, N, C, lengths, flush=True)
    g = torch.Generator().manual_seed(N)

    def pick(*shape, of):
        return torch.tensor(of, dtype=torch.float64)[torch.randint(len(of), shape, generator=g)]

    docs = None
    if isinstance(lengths, int):
        docs = (lengths, (torch.arange(N, dtype=torch.int32) % lengths).expand(B, N).contiguous())
    elif lengths:
        docs = (len(lengths), _ids(lengths, N, B))
    rows = (B, C) if docs is None else (B, docs[0], C)
    ids = torch.zeros(B, N, dtype=torch.int64) if docs is None else docs[1].long()
    G = 1 if docs is None else docs[0]
    live = (ids >= 0)[..., None]
    x = pick(B, N, C, of=(-1, 1))
    d, dh = pick(B, N, C, of=(-3, -2, -1, 1, 2, 3)), pick(B, N, C, of=(-2, -1, 0, 1, 2))
    cond = pick(*rows, of=(-1, 1) if op == "gate_modulate" else (-1, -0.5, 0, 1, 2))
    v = dict(x=x, weight=torch.ones(C), cond=cond)
    m = torch.zeros(B, N, C, dtype=torch.float64)  # of each token; 0 behind the last document
    at = ids.clamp_min(0)
    for b in range(B):
        m[b] = cond[b].view(G, C)[at[b]] * live[b]
    h_grad, xhat = d, x if op == "modulate" else x * live
    if op == "gate_modulate":
        r = x * ~live  # padding: hidden is the residual
        h = r + m * x
        scale2 = pick(*rows[:-1], (C + 1) // 2, of=(-2, -1, 0, 1)).repeat_interleave(2, -1)[..., :C]
        m2 = torch.stack([1 + scale2[b].view(G, C)[at[b]] * live[b] for b in range(B)])
        d[..., 1:C - C % 2:2] = -(d * h)[..., 0:C - C % 2:2] * h[..., 1:C - C % 2:2]
        if C % 2:
            d[..., -1] = 0
        v.update(residual=r, next_weight=torch.ones(C), next_scale=scale2, dhidden=dh)
        h_grad = dh + d * m2
        want2 = d * h
    elif op == "gate":
        v["residual"] = pick(B, N, C, of=(-1, 0, 1))
    v["dout"] = d
    params = ("weight", "cond", "next_weight", "next_scale")
    v = {k: t.to(F32 if k in params else BF).to(cuda) for k, t in v.items()}
    v["doc_ids"] = None if docs is None else docs[1].to(cuda)
    got = _with_grads(op, v, eps=0.0)

    def by_row(t):  # sums over the tokens of each conditioning row
        out = torch.zeros(B, G + 1, C, dtype=torch.float64)
        for b in range(B):
            out[b].index_add_(0, torch.where(ids[b] < 0, G, ids[b]), t[b])
        return out[:, :G].reshape(rows)

    one = 1 if op == "modulate" else 0
    want = {"dweight": (h_grad * xhat * (one + m)).sum((0, 1)), "dcond": by_row(h_grad * xhat)}
    if op == "gate_modulate":
        want.update(dnext_weight=(want2 * m2).sum((0, 1)), dnext_scale=by_row(want2))
    for k, t in want.items():
        bad = (got[k].cpu().double() != t).nonzero()
        assert not len(bad), (k, len(bad), bad[:3].tolist(), got[k].cpu()[tuple(bad[0])], t[tuple(bad[0])])
