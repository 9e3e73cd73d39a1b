"""GPU: the block operators together, as a transformer block uses them around the attention
from the QKV projection: norm + modulation, QKV projection, attention, out-projection, the
fused norms between the halves, gated feed-forward, and the gate onto the residual; forward
and every gradient, eager and captured.

The reference is the same block from torch's elementary operations in 64 bits, with the
attention op itself in its place (its output and gradient, in bf16): what is compared is
everything around it.  Values pass through up to seven roundings to bf16 one after the other
(each operator's output, or the gradient's way back through as many), half a step of 2^-8
each and independent, so a result may be off by 7^0.5 * 2^-9 of its norm, rms; 2^-6 is
allowed, three times that.
"""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

H, D, C, F_ = 4, 64, 256, 512
EPS = 1e-5


def _params(device, docs, seed=0):
    g = torch.Generator().manual_seed(seed)

    def normal(*s, scale=1.0, offset=0.0):
        return (offset + scale * torch.randn(*s, generator=g)).to(torch.bfloat16).to(device)

    p = {n: normal(C, scale=0.2, offset=1.0) for n in ("norm1", "norm2", "ffn_norm1", "ffn_norm2")}
    p.update(qkv=normal(3 * H * D, C, scale=C ** -0.5), out=normal(C, H * D, scale=(H * D) ** -0.5),
             w13=normal(2 * F_, C, scale=C ** -0.5), w2=normal(C, F_, scale=F_ ** -0.5),
             b_ada=normal(4 * C, scale=0.1), w_ada=normal(4 * C, 32, scale=32 ** -0.5))
    return p


def _inputs(device, N, docs, seed=0):
    g = torch.Generator().manual_seed(100 + seed)
    x = (1.5 * torch.randn(1, N, C, generator=g)).to(torch.bfloat16).to(device)
    t = torch.randn(1, docs, 32, generator=g).to(torch.bfloat16).to(device)
    ang = torch.rand(1, N, 1, D // 2, generator=g) * 6.283
    c, s = torch.cos(ang), torch.sin(ang)
    freqs = torch.stack([torch.stack([c, -s], -1), torch.stack([s, c], -1)], -2).to(device)
    dout = torch.randn(1, N, C, generator=g).to(torch.bfloat16).to(device)
    return x, t, freqs, dout


def _attention(qkv, freqs, mask):
    one = torch.ones(D, device=qkv.device)
    return torch.ops.futudiffu_ii.sage_attn_qkv_masked(qkv, one, one, freqs, mask, H, D, EPS, 1 / math.sqrt(D))[0]


def _block(p, x, t, freqs, ids, mask):
    import futudiffu_amd as F
    scale1, gate1, scale2, gate2 = F.fused_linear(t, p["w_ada"], p["b_ada"]).chunk(4, dim=-1)
    h = F.rms_norm_modulate(x, p["norm1"], scale1, doc_ids=ids, eps=EPS)
    a = F.fused_linear(_attention(F.fused_linear(h, p["qkv"]), freqs, mask), p["out"])
    x, h = F.rms_norm_gate_residual_modulate(x, a, p["norm2"], gate1, p["ffn_norm1"], scale2, doc_ids=ids, eps=EPS)
    f = F.fused_linear(F.fused_linear(h, p["w13"], activation="swiglu"), p["w2"])
    return F.rms_norm_gate_residual(x, f, p["ffn_norm2"], gate2, doc_ids=ids, eps=EPS)


class _Exactly(torch.autograd.Function):
    """The attention op in a 64-bit graph."""

    @staticmethod
    def forward(ctx, qkv, freqs, mask):
        with torch.enable_grad():
            leaf = qkv.to(torch.bfloat16).requires_grad_()
            out = _attention(leaf, freqs, mask)
        ctx.leaf, ctx.out = leaf, out
        return out.detach().double()

    @staticmethod
    def backward(ctx, d):
        g, = torch.autograd.grad(ctx.out, ctx.leaf, d.to(torch.bfloat16))
        return g.double(), None, None


def _plain(p, x, t, freqs, ids, mask):
    def unit(v):
        return v * torch.rsqrt(v.pow(2).mean(-1, keepdim=True) + EPS)

    def rows(v):
        live = (ids >= 0) & (ids < v.shape[1])
        picked = v[0][ids[0].long().clamp(0, v.shape[1] - 1)][None]
        return picked * live[..., None]

    scale1, gate1, scale2, gate2 = (t @ p["w_ada"].T + p["b_ada"]).chunk(4, dim=-1)
    h = unit(x) * p["norm1"] * (1 + rows(scale1))
    a = _Exactly.apply(h @ p["qkv"].T, freqs, mask) @ p["out"].T
    x = x + rows(gate1) * unit(a) * p["norm2"]
    h = unit(x) * p["ffn_norm1"] * (1 + rows(scale2))
    z1, z2 = (h @ p["w13"].T).chunk(2, -1)
    f = (z1 * torch.sigmoid(z1) * z2) @ p["w2"].T
    return x + rows(gate2) * unit(f) * p["ffn_norm2"]


def _run(fn, p, x, t, freqs, ids, mask, dout):
    leaves = {**{k: v.detach().requires_grad_() for k, v in p.items()}, "x": x.detach().requires_grad_(),
              "t": t.detach().requires_grad_()}
    out = fn(leaves, leaves["x"], leaves["t"], freqs, ids, mask)
    grads = torch.autograd.grad(out, list(leaves.values()), dout)
    return {"out": out.detach(), **{"d" + k: g for k, g in zip(leaves, grads)}}


def _layout(device, lengths, pad):
    from futudiffu_amd import block_mask as BM
    N = sum(lengths) + pad
    ids = torch.cat([torch.repeat_interleave(torch.arange(len(lengths)), torch.tensor(lengths)),
                     torch.full((pad,), -1)]).to(torch.int32)[None].to(device)
    return N, ids, BM.build_block_mask(lengths, N, device=device)


@pytest.mark.parametrize("lengths,pad", [((256, 128), 0), ((300, 77, 130), 5), ((64,), 0)])
def test_block_matches_the_plain_block(cuda, lengths, pad):
    N, ids, mask = _layout(cuda, list(lengths), pad)
    p = _params(cuda, len(lengths), seed=N)
    x, t, freqs, dout = _inputs(cuda, N, len(lengths), seed=N)
    print("block", lengths, pad, flush=True)
    got = _run(_block, p, x, t, freqs, ids, mask, dout)
    d64 = lambda v: v.double()  # noqa: E731
    want = _run(_plain, {k: d64(v) for k, v in p.items()}, d64(x), d64(t), freqs, ids, mask, d64(dout))
    for k, g in got.items():
        w = want[k]
        err = float((g.double() - w).norm() / w.norm())
        assert g.shape == w.shape and err <= 2.0 ** -6, (k, err)


def test_block_captured(cuda):
    """The whole training step of the block in one graph: replays on new inputs equal eager
    steps bit for bit."""
    N, ids, mask = _layout(cuda, [200, 120], 0)
    p = _params(cuda, 2)
    static = [v.clone() for v in _inputs(cuda, N, 2)]
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        for _ in range(2):
            _run(_block, p, *static[:3], ids, mask, static[3])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        got = _run(_block, p, *static[:3], ids, mask, static[3])
    for seed in (1, 2, 3):
        new = _inputs(cuda, N, 2, seed=seed)
        for a, b in zip(static, new):
            a.copy_(b)
        graph.replay()
        torch.cuda.synchronize()
        want = _run(_block, p, *new[:3], ids, mask, new[3])
        bad = [k for k in want if not torch.equal(got[k], want[k])]
        assert not bad, (seed, bad)
