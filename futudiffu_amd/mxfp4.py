"""Microscaled 4-bit floating point (MXFP4) around the attention, on MI355X.

* :func:`mxfp4_quantize`, :func:`mxfp4_dequantize`  a tensor to :class:`MXFP4` and back
* :func:`mxfp4_linear`   a projection over a weight in MXFP4: ``act(q(x) weight^T + bias) + residual``
* :func:`rms_norm_modulate_mxfp4`, :func:`rms_norm_gate_residual_modulate_mxfp4`
  the norms before a projection, with their output in MXFP4

Columns in blocks of 32 share a scale ``2^e``; a column is a 4-bit code (e2m1), one of ``0, 0.5,
1, 1.5, 2, 3, 4, 6`` with a sign, times the scale.  Of a block whose largest magnitude is
``amax``, ``e = floor(log2 amax) - 2`` (the OCP microscaling specification's rule), from -127 to 127; codes are
the nearest, ties to the even one, and past 6 the code of 6.  A block that holds NaN or an
infinity is NaN as a whole.

A weight is quantized once::

    w = mxfp4_quantize(weight.detach())          # [N, K] bf16 or fp16
    y = mxfp4_linear(x, w, bias, activation="swiglu")

``mxfp4_linear`` of a tensor quantizes it in the call and differentiates in ``x`` (the rounding
passes the gradient on as it is), ``bias`` and ``residual``, once; the weight is frozen.  Everything
else here has codes as its result, which carry no gradient: a call that wants one raises.
Under ``torch.compile``, a tracer, a dispatch mode or ``vmap`` the functions go through the
custom ops ``futudiffu_ii::`` of their names.  Sums are added in a fixed order.
"""

from __future__ import annotations

from typing import NamedTuple

import torch
from torch import Tensor

from . import block_ops as _b


class MXFP4(NamedTuple):
    """Rows ``[..., columns]`` in MXFP4.

    ``codes``: uint8 ``[..., P / 2]``, ``P`` the columns rounded up to 256: the even column in the
    low half of its byte (sign, two bits of exponent, one of mantissa), zeros behind the last.
    ``scales``: uint8 ``[P / 256, rows, 8]``, ``rows`` the product of the leading sizes:
    ``scales[g, r, i]`` is ``e + 127`` of row ``r``'s columns ``256 g + 32 i`` to ``.. + 31``, 255 for
    NaN (of a block behind the last column any but 255: the products read it).
    """

    codes: Tensor
    scales: Tensor
    columns: int

    @property
    def shape(self) -> torch.Size:
        return torch.Size((*self.codes.shape[:-1], self.columns))


def _native():
    return _b._native or _b._load()


def _shapes(x: Tensor) -> tuple[Tensor, Tensor]:
    """Empty codes and scales of x's shape."""
    k = x.shape[-1]
    p = (k + 255) // 256 * 256
    return (x.new_empty((*x.shape[:-1], p // 2), dtype=torch.uint8),
            x.new_empty((p // 256, x.numel() // k, 8), dtype=torch.uint8))


_GRAD = ("MXFP4 codes carry no gradient: quantize under torch.no_grad() or detach the input (mxfp4_linear "
         "differentiates in an x that it quantizes itself)")


def _refuse_grad(ctx, inputs, output):
    # set-up of a gradient: an input wants one
    raise RuntimeError(_GRAD)


def _traced_without_grad(*tensors) -> bool:
    """Whether the call is being compiled; a gradient that it would lose is refused."""
    if not torch.compiler.is_compiling():
        return False
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise RuntimeError(_GRAD)
    return True


_b._define("mxfp4_quantize(Tensor x) -> (Tensor, Tensor)", lambda x: _native().mx_quantize(x), _shapes)
_b._define("mxfp4_dequantize(Tensor codes, Tensor scales, int columns, ScalarType dtype) -> Tensor",
           lambda *args: _native().mx_dequantize(*args),
           lambda codes, scales, columns, dtype: codes.new_empty((*codes.shape[:-1], columns), dtype=dtype))
_b._define("rms_norm_modulate_mxfp4(Tensor x, Tensor? weight, Tensor? scale, Tensor? doc_ids, float eps) "
           "-> (Tensor, Tensor)",
           lambda *args: _native().mx_modulate(*args), lambda x, weight, scale, doc_ids, eps: _shapes(x))
_b._define("rms_norm_gate_residual_modulate_mxfp4(Tensor residual, Tensor x, Tensor? weight, Tensor? gate, "
           "Tensor? next_weight, Tensor? next_scale, Tensor? doc_ids, float eps) -> (Tensor, Tensor, Tensor)",
           lambda *args: _native().mx_gate_modulate(*args),
           lambda residual, x, weight, gate, next_weight, next_scale, doc_ids, eps: (x.new_empty(x.shape),
                                                                                    *_shapes(x)))


def _columns_out(codes: Tensor, activation: str) -> int:
    return codes.shape[0] // (2 if activation == "swiglu" else 1)


_b._define("mxfp4_linear(Tensor x, Tensor codes, Tensor scales, int columns, Tensor? bias, Tensor? residual, "
           "str activation, bool keep_z) -> (Tensor, Tensor)",
           lambda x, *args: _b._present(_native().mx_linear_forward(x, *args), x),
           lambda x, codes, scales, columns, bias, residual, activation, keep_z: (
               x.new_empty(*x.shape[:-1], _columns_out(codes, activation)),
               x.new_empty(x.numel() // x.shape[-1], codes.shape[0], dtype=torch.float32)
               if keep_z and activation != "none" else x.new_empty(0)))
_b._define("mxfp4_linear_backward(Tensor dout, Tensor codes, Tensor scales, int columns, Tensor? bias, Tensor? z, "
           "str activation, bool[] wanted) -> (Tensor, Tensor)",
           lambda dout, *args: _b._present(_native().mx_linear_backward(dout, *args), dout),
           lambda dout, codes, scales, columns, bias, z, activation, wanted: (
               dout.new_empty(*dout.shape[:-1], columns) if wanted[0] else dout.new_empty(0),
               bias.new_empty(bias.shape) if wanted[1] and bias is not None else dout.new_empty(0)))
_b._define("mxfp4_linear_codes(Tensor x_codes, Tensor x_scales, int x_columns, Tensor codes, Tensor scales, "
           "int columns, Tensor? bias, Tensor? residual, str activation, ScalarType dtype) -> Tensor",
           lambda *args: _native().mx_linear_codes(*args),
           lambda x_codes, x_scales, x_columns, codes, scales, columns, bias, residual, activation, dtype:
           x_codes.new_empty(*x_codes.shape[:-1], _columns_out(codes, activation), dtype=dtype))


def _linear_setup(ctx, inputs, output):
    x, codes, scales, columns, bias, residual, activation, keep_z = inputs
    if x.requires_grad and codes.shape[0] * ((columns + 7) // 8 * 8) * 2 >= 1 << 31:
        raise ValueError(f"x wants a gradient: a weight of {codes.shape[0]} x {columns} has 2^31 bytes or more in 16 bits "
                         "(detach x, or split the weight)")
    ctx.mark_non_differentiable(output[1])
    ctx.save_for_backward(codes, scales, bias, output[1])
    ctx.columns, ctx.activation = columns, activation
    ctx.x_requires = x.requires_grad  # x is not saved, but its gradient and the bias's depend on it


def _linear_autograd(ctx, dout, dz):
    codes, scales, bias, z = ctx.saved_tensors
    _b._once(dout, bias)
    if ctx.x_requires and torch.is_grad_enabled():
        raise RuntimeError(_b._TWICE)
    wanted = [ctx.needs_input_grad[0], bias is not None and ctx.needs_input_grad[4]]
    dx = db = None
    if any(wanted):
        dx, db = torch.ops.futudiffu_ii.mxfp4_linear_backward(dout, codes, scales, ctx.columns, bias, z,
                                                              ctx.activation, wanted)
    return (dx if wanted[0] else None, None, None, None, db if wanted[1] else None,
            dout if ctx.needs_input_grad[5] else None, None, None)


torch.library.register_autograd("futudiffu_ii::mxfp4_linear", _linear_autograd, setup_context=_linear_setup,
                                lib=_b._ops)
torch.library.register_autograd("futudiffu_ii::mxfp4_linear_backward", _b._refuse_twice, lib=_b._ops)
for _name in ("mxfp4_quantize", "mxfp4_linear_codes", "rms_norm_modulate_mxfp4",
              "rms_norm_gate_residual_modulate_mxfp4"):
    torch.library.register_autograd(f"futudiffu_ii::{_name}", _b._refuse_twice, setup_context=_refuse_grad,
                                    lib=_b._ops)


# ---- the functions ---------------------------------------------------------------------

def mxfp4_quantize(x: Tensor) -> MXFP4:
    """``x`` ``[..., K]``, bfloat16 or float16, any strides, to MXFP4 along its last axis."""
    if _traced_without_grad(x):
        return MXFP4(*torch.ops.futudiffu_ii.mxfp4_quantize(x), x.shape[-1])
    return MXFP4(*_native().mxfp4_quantize(x), x.shape[-1])


def mxfp4_dequantize(q: MXFP4, *, dtype: torch.dtype = torch.bfloat16) -> Tensor:
    """What ``q`` stands for, as bfloat16 (exactly; infinite from ``2^128`` on, which only a norm's output
    reaches) or float16 (rounded where that is subnormal, infinite past 65504)."""
    if torch.compiler.is_compiling():
        return torch.ops.futudiffu_ii.mxfp4_dequantize(q.codes, q.scales, q.columns, dtype)
    return _native().mxfp4_dequantize(q.codes, q.scales, q.columns, dtype)


def mxfp4_linear(x: Tensor | MXFP4, weight: MXFP4, bias: Tensor | None = None, residual: Tensor | None = None, *,
                 activation: str = "none", dtype: torch.dtype = torch.bfloat16) -> Tensor:
    """``act(q(x) weight^T + bias) + residual``, both operands of the product in MXFP4.

    ``x`` is ``[..., K]``, bfloat16 or float16, quantized in the call and the output of its type;
    or MXFP4 already (of a norm, or shared by several projections) and the output of ``dtype``.
    ``weight`` holds rows ``[N, K]``, ``bias``, ``residual`` and ``activation`` are
    :func:`futudiffu_amd.fused_linear`'s.  Sums are fp32, the output is rounded once.

    The gradient of a tensor ``x`` is ``dz weight``, rounded once: for an activation the forward keeps
    ``z`` in fp32, and ``dz = dout * act'(z)`` enters the product as two bfloat16 parts.  Without
    one ``dz`` is ``dout``, and the weight's values are taken in ``x``'s type (exact in bfloat16; in
    float16 infinite past 65504, and rounded under 2^-23).  An ``x`` that wants a
    gradient needs a weight of under 2^31 bytes in 16 bits.
    """
    if isinstance(x, MXFP4):
        if _traced_without_grad(bias, residual):
            return torch.ops.futudiffu_ii.mxfp4_linear_codes(*x, *weight, bias, residual, activation, dtype)
        return _native().mxfp4_linear_codes(*x, *weight, bias, residual, activation, dtype)
    if torch.compiler.is_compiling():
        keep = activation != "none" and torch.is_grad_enabled() and any(
            t is not None and t.requires_grad for t in (x, bias))
        return torch.ops.futudiffu_ii.mxfp4_linear(x, *weight, bias, residual, activation, keep)[0]
    return _native().mxfp4_linear(x, *weight, bias, residual, activation)


def rms_norm_modulate_mxfp4(x: Tensor, weight: Tensor | None = None, scale: Tensor | None = None, *,
                            doc_ids: Tensor | None = None, eps: float = 1e-5) -> MXFP4:
    """:func:`futudiffu_amd.rms_norm_modulate` in MXFP4, quantized from the unrounded values
    (a value next to a border between two codes is decided in fp64 and falls on its own side)."""
    if _traced_without_grad(x, weight, scale):
        return MXFP4(*torch.ops.futudiffu_ii.rms_norm_modulate_mxfp4(x, weight, scale, doc_ids, eps), x.shape[-1])
    return MXFP4(*_native().rms_norm_modulate_mxfp4(x, weight, scale, doc_ids, eps), x.shape[-1])


def rms_norm_gate_residual_modulate_mxfp4(
        residual: Tensor, x: Tensor, weight: Tensor | None = None, gate: Tensor | None = None,
        next_weight: Tensor | None = None, next_scale: Tensor | None = None, *, doc_ids: Tensor | None = None,
        eps: float = 1e-5) -> tuple[Tensor, MXFP4]:
    """:func:`futudiffu_amd.rms_norm_gate_residual_modulate` with the second norm's output in MXFP4:
    ``(hidden, out)``, ``out`` quantized from the unrounded values as in
    :func:`rms_norm_modulate_mxfp4`."""
    if _traced_without_grad(residual, x, weight, gate, next_weight, next_scale):
        hidden, *out = torch.ops.futudiffu_ii.rms_norm_gate_residual_modulate_mxfp4(
            residual, x, weight, gate, next_weight, next_scale, doc_ids, eps)
    else:
        hidden, *out = _native().rms_norm_gate_residual_modulate_mxfp4(residual, x, weight, gate, next_weight,
                                                                       next_scale, doc_ids, eps)
    return hidden, MXFP4(*out, x.shape[-1])
