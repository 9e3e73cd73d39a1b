"""64-bit restatement of the operators around the attention (futudiffu_amd/block_ops.py).

Each function returns the exact values of the given (already rounded) inputs, and bounds
on what 32-bit arithmetic in any order can add to them: ``terms * 2^-24`` times the same
formula over absolute values, where ``terms`` counts the roundings a value passes through.
A result rounded once more to a type is off by half a step of that type on top
(:func:`allowed`).
"""

from __future__ import annotations

import math

import torch
from torch import Tensor

U32 = 2.0 ** -24


def allowed(exact: Tensor, bound: Tensor, dtype: torch.dtype) -> Tensor:
    """How far a value of ``dtype`` may be from ``exact``: the 32-bit result's bound, then one
    rounding (half a step, absolute below the type's smallest normal value)."""
    eps, tiny = torch.finfo(dtype).eps, torch.finfo(dtype).tiny
    return bound + eps / 2 * (exact.abs() + bound).clamp_min(tiny)


def worst(got: Tensor, exact: Tensor, bound: Tensor) -> float:
    """The largest error in units of what is allowed; at most 1 passes.  Values that are not
    finite have to be the same."""
    g = got.detach().double().to(exact.device)
    fine = torch.isfinite(exact)
    same = torch.equal(fine, torch.isfinite(g)) and torch.equal(torch.isnan(exact), torch.isnan(g)) and bool(
        (g[~fine & ~torch.isnan(exact)] == exact[~fine & ~torch.isnan(exact)]).all())
    if not same:
        return math.inf
    if not fine.any():
        return 0.0
    a = allowed(exact, bound, got.dtype)[fine]
    return float(((g[fine] - exact[fine]).abs() / a.clamp_min(1e-300)).max())


def rows_of(cond: Tensor | None, doc_ids: Tensor | None, B: int, N: int, C: int, absent: float) -> Tensor:
    """The conditioning row of each token, ``[B, N, C]`` in 64 bits; 0 for a token of no document."""
    if cond is None:
        return torch.full((B, N, C), absent, dtype=torch.float64)
    out = torch.zeros(B, N, C, dtype=torch.float64, device=cond.device)
    for b in range(B):
        if doc_ids is None:
            out[b] = cond[b].double()
            continue
        for g in range(cond.shape[1]):
            out[b, doc_ids[b] == g] = cond[b, g].double()
    return out


def _row_sums(t: Tensor, cond: Tensor, doc_ids: Tensor | None) -> Tensor:
    if doc_ids is None:
        return t.sum(1)
    return torch.stack([torch.stack([t[b, doc_ids[b] == g].sum(0) for g in range(cond.shape[1])])
                        for b in range(cond.shape[0])])


def _unit(x: Tensor, eps: float):
    r = 1 / torch.sqrt((x * x).mean(-1, keepdim=True) + eps)
    return x * r, r


def _unit_back(g: Tensor, xhat: Tensor, r: Tensor) -> Tensor:
    return r * (g - xhat * (g * xhat).mean(-1, keepdim=True))


def _unit_back_abs(g: Tensor, xhat: Tensor, r: Tensor) -> Tensor:
    return r * (g.abs() + xhat.abs() * (g * xhat).abs().mean(-1, keepdim=True))


def norms(op: str, x: Tensor, weight, cond, doc_ids, eps: float, residual=None, next_weight=None, next_scale=None,
          dout=None, dhidden=None) -> dict[str, tuple[Tensor, Tensor]]:
    """``{name: (exact, bound)}`` of a norm operator's outputs, and with ``dout`` its gradients.

    Roundings of one value: a sum of C squares or products in chains of 16 and trees (under
    40 with the scaling around it, twice that where two norms follow each other); a channel
    sum over tokens in chains of at most 512 tokens of a chunk, a tree of 8, every 32nd chunk's
    partial and 32 of their sums (under 700 to 10^6 tokens).  Over many tokens that bound is
    wider than one token's part: sums that are exact in any order are what shows a token lost.
    """
    B, N, C = x.shape
    one = torch.ones(C, dtype=torch.float64, device=x.device)
    w = one if weight is None else weight.double()
    w2 = one if next_weight is None else next_weight.double()
    m = rows_of(cond, doc_ids, B, N, C, 0.0 if op == "modulate" else 1.0).to(x.device)
    if op == "modulate":
        m = 1 + m
    xd = x.double()
    xhat, r = _unit(xd, eps)
    if op != "modulate" and cond is not None and doc_ids is not None:  # tokens of no document: x is not read
        dead = ((doc_ids < 0) | (doc_ids >= cond.shape[1]))[..., None]
        xhat, r = xhat.masked_fill(dead, 0.0), r.masked_fill(dead, 0.0)
    p = xhat * w * m
    out = {}
    if op == "modulate":
        out["out"] = (p, 40 * U32 * p.abs())
    else:
        rd = residual.double()
        h = rd + p
        herr = 40 * U32 * p.abs() + U32 * h.abs()
        out["out" if op == "gate" else "hidden"] = (h, herr)
    if op == "gate_modulate":
        m2 = 1 + rows_of(next_scale, doc_ids, B, N, C, 0.0).to(x.device)
        hhat, r2 = _unit(h, eps)
        # h's own error, directly and through the norm
        lift = herr.norm(dim=-1, keepdim=True) / h.norm(dim=-1, keepdim=True).clamp_min(1e-300)
        hhat_err = r2 * herr + hhat.abs() * (lift + 40 * U32)
        y = hhat * w2 * m2
        out["out"] = (y, (w2 * m2).abs() * hhat_err + 4 * U32 * y.abs())
    if dout is None:
        return out
    d, derr = dout.double(), torch.zeros_like(xd)
    if op == "gate_modulate":
        d2 = d
        g2 = d2 * w2 * m2
        d = dhidden.double() + _unit_back(g2, hhat, r2)
        k2 = (g2 * hhat).abs().mean(-1, keepdim=True)
        derr = (40 * U32 * (_unit_back_abs(g2, hhat, r2) + dhidden.double().abs())
                + r2 * (hhat_err * k2 + hhat.abs() * (g2.abs() * hhat_err).mean(-1, keepdim=True))
                + (lift + 40 * U32) * _unit_back_abs(g2, hhat, r2))
        out["dresidual"] = (d, derr)
        out["dnext_weight"] = ((d2 * hhat * m2).sum((0, 1)),
                               ((d2 * m2).abs() * (hhat_err + 700 * U32 * hhat.abs())).sum((0, 1)))
        if next_scale is not None:
            out["dnext_scale"] = (_row_sums(d2 * hhat * w2, next_scale, doc_ids),
                                  _row_sums((d2 * w2).abs() * (hhat_err + 700 * U32 * hhat.abs()), next_scale,
                                            doc_ids))
    g, gerr = d * w * m, derr * (w * m).abs()
    out["dx"] = (_unit_back(g, xhat, r), 80 * U32 * _unit_back_abs(g, xhat, r) + _unit_back_abs(gerr, xhat, r))
    out["dweight"] = ((d * xhat * m).sum((0, 1)), ((700 * U32 * d.abs() + derr) * (xhat * m).abs()).sum((0, 1)))
    if cond is not None:
        out["dcond"] = (_row_sums(d * xhat * w, cond, doc_ids),
                        _row_sums((700 * U32 * d.abs() + derr) * (xhat * w).abs(), cond, doc_ids))
    return out


def _act(kind: str, z: Tensor):
    """The activation, its derivative, and bounds on both: how far 32-bit arithmetic is off."""
    if kind == "none":
        return z, torch.ones_like(z), torch.zeros_like(z), torch.zeros_like(z)
    if kind in ("silu", "swiglu"):
        u, up = z, torch.ones_like(z)
    else:
        a = math.sqrt(8 / math.pi)
        u, up = a * (z + 0.044715 * z ** 3), a * (1 + 3 * 0.044715 * z * z)
    s = torch.sigmoid(u)
    # exp(-u) by way of 2^: the exponent's rounding is |u| steps, the rest a few; s (1 - s) of
    # it reaches s; 1 - s cancels to half a step of 1
    serr = U32 * (s * (1 - s) * (2 * u.abs() + 4) + 4 * s)
    f, d = z * s, s + z * s * (1 - s) * up
    ferr = z.abs() * serr + 2 * U32 * f.abs()
    derr = serr + (z * up).abs() * (serr * (1 - 2 * s).abs() + U32 * s + 8 * U32 * s * (1 - s)) + 4 * U32 * d.abs()
    return f, d, ferr, derr


def linear(x: Tensor, weight: Tensor, bias, residual, activation: str, dout=None) -> dict[str, tuple[Tensor, Tensor]]:
    """``{name: (exact, bound)}`` of fused_linear's output, and with ``dout`` its gradients.

    A product of K terms is summed in any order: K roundings of at most the sum of the
    terms' sizes.  The gradient of z is rounded as the products' operand: half a step of the
    type.
    """
    eps = torch.finfo(x.dtype).eps
    xd, wd = x.double().reshape(-1, x.shape[-1]), weight.double()
    M, K = xd.shape
    z = xd @ wd.T
    zerr = (K + 2) * U32 * (xd.abs() @ wd.abs().T)
    if bias is not None:
        z = z + bias.double()
        zerr = zerr + U32 * (z.abs() + bias.double().abs())
    N = wd.shape[0]
    if activation == "swiglu":
        z1, z2 = z.chunk(2, -1)
        e1, e2 = zerr.chunk(2, -1)
        f, d, ferr, derr = _act(activation, z1)
        out, oerr = f * z2, (ferr + e1 * 1.1) * (z2.abs() + e2) + f.abs() * e2 + U32 * (f * z2).abs()
    else:
        f, d, ferr, derr = _act(activation, z)
        out, oerr = f, ferr + zerr * (1.0 if activation == "none" else 1.2)
    if residual is not None:
        out = out + residual.double().reshape(M, -1)
        oerr = oerr + U32 * out.abs()
    shape = (*x.shape[:-1], out.shape[-1])
    r = {"out": (out.reshape(shape), oerr.reshape(shape))}
    if dout is None:
        return r
    g = dout.double().reshape(M, -1)

    def kept(zz, ee):  # z as the backward has it: fp32
        return ee + U32 * zz.abs()

    if activation == "none":
        dz, unrounded, rounded = g, torch.zeros_like(g), torch.zeros_like(g)
    else:
        # |act''| is at most 0.5 (silu) and 1.13 (gelu)
        curve = 0.5 if activation in ("silu", "swiglu") else 1.13
        if activation == "swiglu":
            k1, k2 = kept(z1, e1), kept(z2, e2)
            a, b = g * z2 * d, g * f
            ae = g.abs() * (k2 * (d.abs() + derr) + z2.abs() * (curve * k1 + derr)) + g.abs() * k2 * curve * k1
            be = g.abs() * (1.1 * k1 + ferr)
            dz, unrounded = torch.cat([a, b], -1), torch.cat([ae, be], -1)
        else:
            dz, unrounded = g * d, g.abs() * (curve * kept(z, zerr) + derr)
        unrounded = unrounded + 4 * U32 * dz.abs()
        rounded = unrounded + eps / 2 * (dz.abs() + unrounded).clamp_min(torch.finfo(x.dtype).tiny)
    mag = dz.abs() + rounded
    r["dx"] = ((dz @ wd).reshape(x.shape), (rounded @ wd.abs() + (N + 2) * U32 * (mag @ wd.abs())).reshape(x.shape))
    r["dweight"] = (dz.T @ xd, rounded.T @ xd.abs() + (M + 2) * U32 * (mag.T @ xd.abs()))
    if bias is not None:
        r["dbias"] = (dz.sum(0), (unrounded + (M + 2) * U32 * (dz.abs() + unrounded)).sum(0))
    if residual is not None:
        r["dresidual"] = (dout.double(), torch.zeros_like(dout.double()))
    return r
