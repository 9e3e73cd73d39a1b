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
    sum over tokens in chains of at most 512 tokens, 64 chunks and 16 rows (under 700).
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
