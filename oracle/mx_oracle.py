"""64-bit restatement of MXFP4 and the operators over it (futudiffu_amd/mxfp4.py).

Quantization is exact but for the choice of the nearest code, so codes and scales are compared
bit for bit.  The products' bounds are block_oracle's; the matrix cores' sum of 64 scaled products is
not a chain of rounded fp32 additions, and is off by up to 2^-14 of the sum of the products' sizes
(2^-15.7 measured on 8-bit operands).
"""

from __future__ import annotations

import torch
from torch import Tensor

from oracle import block_oracle as B

VALUES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
MFMA = 2.0 ** -14
DZ = 2.0 ** -17  # what the two bf16 parts of an activation's dz leave of it: half a step of half a step


def columns_held(k: int) -> int:
    return -(-k // 256) * 256


def quantize(x: Tensor) -> tuple[Tensor, Tensor]:
    """Codes ``[..., P / 2]`` and scales ``[P / 256, rows, 8]`` of ``[..., K]`` values, as the
    package holds them."""
    k = x.shape[-1]
    p = columns_held(k)
    v = torch.zeros(x[..., :1].numel(), p, dtype=torch.float64, device=x.device)
    v[:, :k] = x.reshape(-1, k).double()
    b = v.reshape(v.shape[0], p // 32, 32)
    amax = b.abs().amax(-1)
    finite = torch.isfinite(b).all(-1)
    e = torch.frexp(torch.where(finite, amax, 1.0))[1].double() - 1  # amax = m 2^e, 1 <= m < 2
    e = torch.where(amax == 0, -127.0, (e - 2).clamp(-127.0, 127.0))
    r = (torch.where(finite[..., None], b, 0.0) / torch.exp2(e)[..., None]).clamp(-8.0, 8.0)
    # the nearest of the values; of two equally near the even code
    table = torch.tensor(VALUES, dtype=torch.float64, device=x.device)
    code = torch.zeros(r.shape, dtype=torch.uint8, device=x.device)
    best = r.abs()
    for i in range(1, 8):
        off = (r.abs() - table[i]).abs()
        nearer = (off < best) | ((off == best) & (i % 2 == 0))
        code = torch.where(nearer, i, code.int()).to(torch.uint8)
        best = torch.where(nearer, off, best)
    code = (code.int() + 8 * torch.signbit(r).int()).to(torch.uint8).reshape(*x.shape[:-1], p // 2, 2)
    scales = torch.where(finite, e + 127, 255.0).to(torch.uint8)
    scales = scales.reshape(-1, p // 256, 8).transpose(0, 1).contiguous()
    return code[..., 0] + 16 * code[..., 1], scales


def dequantize(codes: Tensor, scales: Tensor, k: int) -> Tensor:
    """The values in 64 bits."""
    table = torch.tensor(VALUES, dtype=torch.float64, device=codes.device)
    c = torch.stack([codes & 15, codes >> 4], -1).reshape(-1, codes.shape[-1] * 2).long()
    v = torch.where(c >= 8, -table[c & 7], table[c & 7])
    s = scales.transpose(0, 1).reshape(v.shape[0], -1)
    scale = torch.where(s == 255, torch.nan, torch.exp2(s.double() - 127))
    v = (v.reshape(v.shape[0], -1, 32) * scale[..., None]).reshape(v.shape)
    return v[:, :k].reshape(*codes.shape[:-1], k)


def rounded(x: Tensor) -> Tensor:
    """What MXFP4 makes of ``x``, in 64 bits."""
    return dequantize(*quantize(x), x.shape[-1])


def linear(x: Tensor, weight: Tensor, bias, residual, activation: str, dout=None) -> dict[str, tuple[Tensor, Tensor]]:
    """``{name: (exact, bound)}`` of mxfp4_linear over a weight of these exact values, and with
    ``dout`` its gradients: block_oracle's of the rounded ``x`` in 64 bits (whose dz it does not
    round), whose products are off by MFMA times the sum of their sizes on top, and that through
    the activation (its slope is at most 1.13, its curvature too); the dz of an activation by DZ of it."""
    k = x.shape[-1]
    q = rounded(x).reshape(-1, k)
    ref = B.linear(q, weight, bias, None if residual is None else residual.reshape(q.shape[0], -1),
                   activation, None if dout is None else dout.reshape(q.shape[0], -1))
    size = q.abs() @ weight.double().abs().T
    more = MFMA * size
    z = q @ weight.double().T
    if bias is not None:
        z = z + bias.double()
    r = {}
    if activation == "swiglu":
        z1, z2 = z.chunk(2, -1)
        m1, m2 = more.chunk(2, -1)
        f = (z1 * torch.sigmoid(z1)).abs()
        extra = 1.13 * m1 * (z2.abs() + m2) + f * m2
    else:
        extra = (1.0 if activation == "none" else 1.13) * more
    shape = (*x.shape[:-1], extra.shape[-1])
    r["out"] = (ref["out"][0].reshape(shape), (ref["out"][1] + extra).reshape(shape))
    if dout is None:
        return r
    g = dout.reshape(q.shape[0], -1).double().abs()
    if activation == "none":
        dz = size = torch.zeros_like(more)
    elif activation == "swiglu":
        dz = torch.cat([g * (1.13 * m1 * (z2.abs() + m2) + 1.13 * m2), g * 1.13 * m1], -1)
        size = torch.cat([g * 1.13 * (z2.abs() + m2), g * (f + 1.13 * m1)], -1)
    else:
        dz = g * 1.13 * more
        size = g * 1.13
    exact, bound = ref["dx"]
    off = dz + DZ * (size + dz)  # of the operand
    r["dx"] = (exact.reshape(x.shape), (bound + off @ weight.double().abs()).reshape(x.shape))
    if bias is not None:
        r["dbias"] = (ref["dbias"][0], ref["dbias"][1] + dz.sum(0))
    if residual is not None:
        r["dresidual"] = (dout.double(), torch.zeros_like(dout, dtype=torch.float64))
    return r


def norm_values(x: Tensor, weight, cond, doc_ids, eps: float, residual=None, next_weight=None, next_scale=None):
    """The modulated norm's values (and with a residual those of the hidden stream) in 64 bits."""
    op = "modulate" if residual is None else "gate_modulate"
    r = B.norms(op, x, weight, cond, doc_ids, eps, residual, next_weight, next_scale)
    return r["out"][0] if residual is None else (r["hidden"][0], r["out"][0])
