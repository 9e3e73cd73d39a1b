"""What surrounds the attention in a transformer block, on MI355X.

* :func:`rms_norm_modulate`      the norm before a block: ``xhat * weight * (1 + scale)``
* :func:`rms_norm_gate_residual` the norm after it: ``residual + gate * xhat * weight``
* :func:`rms_norm_gate_residual_modulate` the norm after one half of a block and the
  norm before the next, in one pass
* :func:`fused_linear`           a projection: ``act(x weight^T + bias) + residual``

``xhat = x / sqrt(mean(x^2) + eps)`` over the channels; arithmetic in fp32, one rounding
per output.  ``x`` is ``[B, N, C]`` (or ``[N, C]``), bfloat16 or float16, with any strides
(channels that are not contiguous are copied).  ``weight`` is ``[C]`` or None; ``scale``
and ``gate`` have a row per batch item, ``[B, C]``, or with ``doc_ids`` (integers ``[B, N]``,
as :func:`futudiffu_amd.build_doc_ids` makes them) a row per document of a packed
sequence, ``[B, G, C]``: a token whose id is not in ``0 .. G-1`` (padding) has scale 0 and
gate 0, and behind a gate its ``x`` is not read (no gate given: 1 for every token).
Parameters are of ``x``'s type or float32; chunks of one projection's output are read in
place.

The functions differentiate in reverse mode, once (not the gradients themselves); a
forward-mode tangent is refused.  Under ``torch.compile``, a tracer, a dispatch mode or
``vmap`` they go through the custom ops
``futudiffu_ii::rms_norm_modulate``, ``::rms_norm_gate_residual``,
``::rms_norm_gate_residual_modulate`` and ``::fused_linear``, which carry the same
gradients.  Sums are added in a fixed order, so results and gradients repeat bit for
bit.  An empty batch gives empty outputs and zero parameter gradients.
"""

from __future__ import annotations

import os

import torch
from torch import Tensor

from . import _lib

_native = None


def _load():
    """The host side of the operators (csrc/block_ops.cpp) over the package's library."""
    global _native
    if _native is None:
        path = os.path.join(os.path.dirname(os.path.abspath(__file__)), "_block_ops.so")
        if not os.path.exists(path):
            raise RuntimeError(f"{path} is not built; run `python futudiffu_amd/build.py` "
                               "(or __graft_entry__.build()) first")
        from . import _block_ops
        _block_ops.bind(_lib.load()._handle)
        _native = _block_ops
    return _native


_ops = torch.library.Library("futudiffu_ii", "FRAGMENT")


# ---- ops and their autograd formulas ---------------------------------------------------
#
# A gradient op returns an empty tensor in the place of a gradient that is not wanted
# (an op's outputs cannot be None).

def _define(schema: str, impl, fake) -> None:
    name = schema.split("(")[0]
    _ops.define(schema)
    _ops.impl(name, impl, "CompositeExplicitAutograd")
    torch.library.register_fake(f"futudiffu_ii::{name}", fake, lib=_ops)


def _present(grads, like: Tensor) -> tuple[Tensor, ...]:
    return tuple(like.new_empty(0) if g is None else g for g in grads)


def _fake_grads(like: Tensor, *pairs) -> tuple[Tensor, ...]:
    return tuple(like.new_empty(0) if t is None or not w else t.new_empty(t.shape) for t, w in pairs)


def _wanted(ctx, places, tensors) -> list[bool]:
    return [t is not None and ctx.needs_input_grad[i] for i, t in zip(places, tensors)]


def _only(grads, wanted):
    return [g if w else None for g, w in zip(grads, wanted)]


# The gradients are not themselves differentiable: a second derivative through these ops
# would lack every term that goes through them.

_TWICE = "the gradients of the block operators cannot be differentiated (create_graph=True)"


def _once(*tensors) -> None:
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise RuntimeError(_TWICE)


def _refuse_twice(ctx, *grads):
    raise RuntimeError(_TWICE)


_define("rms_norm_modulate(Tensor x, Tensor? weight, Tensor? scale, Tensor? doc_ids, float eps) -> Tensor",
        lambda *args: _load().modulate_forward(*args), lambda x, weight, scale, doc_ids, eps: x.new_empty(x.shape))
_define("rms_norm_modulate_backward(Tensor dout, Tensor x, Tensor? weight, Tensor? scale, Tensor? doc_ids, "
        "float eps, bool[] wanted) -> (Tensor, Tensor, Tensor)",
        lambda dout, x, weight, scale, doc_ids, eps, wanted: _present(
            _load().norm_backward(False, dout, x, weight, scale, doc_ids, eps, wanted), x),
        lambda dout, x, weight, scale, doc_ids, eps, wanted: _fake_grads(
            x, *zip((x, weight, scale), wanted)))
_define("rms_norm_gate_residual(Tensor residual, Tensor x, Tensor? weight, Tensor? gate, Tensor? doc_ids, "
        "float eps) -> Tensor",
        lambda *args: _load().gate_forward(*args), lambda residual, x, weight, gate, doc_ids, eps: x.new_empty(x.shape))
_define("rms_norm_gate_residual_backward(Tensor dout, Tensor x, Tensor? weight, Tensor? gate, Tensor? doc_ids, "
        "float eps, bool[] wanted) -> (Tensor, Tensor, Tensor)",
        lambda dout, x, weight, gate, doc_ids, eps, wanted: _present(
            _load().norm_backward(True, dout, x, weight, gate, doc_ids, eps, wanted), x),
        lambda dout, x, weight, gate, doc_ids, eps, wanted: _fake_grads(x, *zip((x, weight, gate), wanted)))
_define("rms_norm_gate_residual_modulate(Tensor residual, Tensor x, Tensor? weight, Tensor? gate, "
        "Tensor? next_weight, Tensor? next_scale, Tensor? doc_ids, float eps) -> (Tensor, Tensor)",
        lambda *args: _load().gate_modulate_forward(*args),
        lambda residual, x, weight, gate, next_weight, next_scale, doc_ids, eps: (x.new_empty(x.shape),
                                                                                 x.new_empty(x.shape)))
_define("rms_norm_gate_residual_modulate_backward(Tensor dhidden, Tensor dout, Tensor residual, Tensor x, "
        "Tensor? weight, Tensor? gate, Tensor? next_weight, Tensor? next_scale, Tensor? doc_ids, float eps, "
        "bool[] wanted) -> (Tensor, Tensor, Tensor, Tensor, Tensor, Tensor)",
        lambda dhidden, dout, residual, x, *rest: _present(
            _load().gate_modulate_backward(dhidden, dout, residual, x, *rest), x),
        lambda dhidden, dout, residual, x, weight, gate, next_weight, next_scale, doc_ids, eps, wanted: _fake_grads(
            x, (x, True), (x, wanted[1]), *zip((weight, gate, next_weight, next_scale), wanted[2:])))


def _modulate_setup(ctx, inputs, output):
    x, weight, scale, doc_ids, eps = inputs
    ctx.save_for_backward(x, weight, scale, doc_ids)
    ctx.eps = eps


def _modulate_autograd(ctx, dout):
    x, weight, scale, doc_ids = ctx.saved_tensors
    _once(dout, x, weight, scale)
    wanted = _wanted(ctx, (0, 1, 2), (x, weight, scale))
    grads = torch.ops.futudiffu_ii.rms_norm_modulate_backward(dout, x, weight, scale, doc_ids, ctx.eps, wanted)
    return *_only(grads, wanted), None, None


def _gate_setup(ctx, inputs, output):
    residual, x, weight, gate, doc_ids, eps = inputs
    ctx.save_for_backward(x, weight, gate, doc_ids)
    ctx.eps = eps


def _gate_autograd(ctx, dout):
    x, weight, gate, doc_ids = ctx.saved_tensors
    _once(dout, x, weight, gate)
    wanted = _wanted(ctx, (1, 2, 3), (x, weight, gate))
    grads = (None, None, None)
    if any(wanted):
        grads = torch.ops.futudiffu_ii.rms_norm_gate_residual_backward(dout, x, weight, gate, doc_ids, ctx.eps,
                                                                       wanted)
    return dout if ctx.needs_input_grad[0] else None, *_only(grads, wanted), None, None


def _gate_modulate_setup(ctx, inputs, output):
    residual, x, weight, gate, next_weight, next_scale, doc_ids, eps = inputs
    ctx.save_for_backward(residual, x, weight, gate, next_weight, next_scale, doc_ids)
    ctx.eps = eps


def _gate_modulate_autograd(ctx, dhidden, dout):
    residual, x, weight, gate, next_weight, next_scale, doc_ids = ctx.saved_tensors
    _once(dhidden, dout, residual, x, weight, gate, next_weight, next_scale)
    wanted = _wanted(ctx, range(6), (residual, x, weight, gate, next_weight, next_scale))
    grads = torch.ops.futudiffu_ii.rms_norm_gate_residual_modulate_backward(
        dhidden, dout, residual, x, weight, gate, next_weight, next_scale, doc_ids, ctx.eps, wanted)
    return *_only(grads, wanted), None, None


torch.library.register_autograd("futudiffu_ii::rms_norm_modulate", _modulate_autograd,
                                setup_context=_modulate_setup, lib=_ops)
torch.library.register_autograd("futudiffu_ii::rms_norm_gate_residual", _gate_autograd, setup_context=_gate_setup,
                                lib=_ops)
torch.library.register_autograd("futudiffu_ii::rms_norm_gate_residual_modulate", _gate_modulate_autograd,
                                setup_context=_gate_modulate_setup, lib=_ops)


_define("fused_linear(Tensor x, Tensor weight, Tensor? bias, Tensor? residual, str activation, bool keep_z) "
        "-> (Tensor, Tensor)",
        lambda x, weight, bias, residual, activation, keep_z: _present(
            _load().linear_forward(x, weight, bias, residual, activation, keep_z), x),
        lambda x, weight, bias, residual, activation, keep_z: (
            x.new_empty(*x.shape[:-1], weight.shape[0] // (2 if activation == "swiglu" else 1)),
            x.new_empty(x.numel() // x.shape[-1], weight.shape[0], dtype=torch.float32) if keep_z and activation != "none"
            else x.new_empty(0)))
_define("fused_linear_backward(Tensor dout, Tensor x, Tensor weight, Tensor? bias, Tensor? z, str activation, "
        "bool[] wanted) -> (Tensor, Tensor, Tensor)",
        lambda dout, x, weight, bias, z, activation, wanted: _present(
            _load().linear_backward(dout, x, weight, bias, z, activation, wanted), x),
        lambda dout, x, weight, bias, z, activation, wanted: _fake_grads(x, *zip((x, weight, bias), wanted)))


def _linear_setup(ctx, inputs, output):
    x, weight, bias, residual, activation, keep_z = inputs
    ctx.mark_non_differentiable(output[1])
    ctx.save_for_backward(x, weight, bias, output[1])
    ctx.activation = activation


def _linear_autograd(ctx, dout, dz):
    x, weight, bias, z = ctx.saved_tensors
    _once(dout, x, weight, bias)
    wanted = _wanted(ctx, range(3), (x, weight, bias))
    grads = (None, None, None)
    if any(wanted):
        grads = torch.ops.futudiffu_ii.fused_linear_backward(dout, x, weight, bias, z, ctx.activation, wanted)
    return *_only(grads, wanted), dout if ctx.needs_input_grad[3] else None, None, None


torch.library.register_autograd("futudiffu_ii::fused_linear", _linear_autograd, setup_context=_linear_setup, lib=_ops)
for _name in ("rms_norm_modulate", "rms_norm_gate_residual", "rms_norm_gate_residual_modulate", "fused_linear"):
    torch.library.register_autograd(f"futudiffu_ii::{_name}_backward", _refuse_twice, lib=_ops)


# ---- the functions ---------------------------------------------------------------------

def rms_norm_modulate(x: Tensor, weight: Tensor | None = None, scale: Tensor | None = None, *,
                      doc_ids: Tensor | None = None, eps: float = 1e-5) -> Tensor:
    """``xhat * weight * (1 + scale)``: the norm before a block with its modulation."""
    if torch.compiler.is_compiling():
        return torch.ops.futudiffu_ii.rms_norm_modulate(x, weight, scale, doc_ids, eps)
    return (_native or _load()).rms_norm_modulate(x, weight, scale, doc_ids, eps)


def rms_norm_gate_residual(residual: Tensor, x: Tensor, weight: Tensor | None = None, gate: Tensor | None = None, *,
                           doc_ids: Tensor | None = None, eps: float = 1e-5) -> Tensor:
    """``residual + gate * xhat * weight``: the norm after a block, gated, onto the residual."""
    if torch.compiler.is_compiling():
        return torch.ops.futudiffu_ii.rms_norm_gate_residual(residual, x, weight, gate, doc_ids, eps)
    return (_native or _load()).rms_norm_gate_residual(residual, x, weight, gate, doc_ids, eps)


def rms_norm_gate_residual_modulate(residual: Tensor, x: Tensor, weight: Tensor | None = None,
                                    gate: Tensor | None = None, next_weight: Tensor | None = None,
                                    next_scale: Tensor | None = None, *, doc_ids: Tensor | None = None,
                                    eps: float = 1e-5) -> tuple[Tensor, Tensor]:
    """``hidden = residual + gate * xhat * weight`` and the norm of ``hidden`` before the
    next block, ``(hidden, out)``.

    The second norm takes ``hidden`` unrounded: ``out`` is nearer the exact value than the
    two calls' one after the other, which normalize the rounded ``hidden``.
    """
    if torch.compiler.is_compiling():
        return torch.ops.futudiffu_ii.rms_norm_gate_residual_modulate(residual, x, weight, gate, next_weight,
                                                                      next_scale, doc_ids, eps)
    return (_native or _load()).rms_norm_gate_residual_modulate(residual, x, weight, gate, next_weight, next_scale,
                                                                doc_ids, eps)


def fused_linear(x: Tensor, weight: Tensor, bias: Tensor | None = None, residual: Tensor | None = None, *,
                 activation: str = "none") -> Tensor:
    """``act(x weight^T + bias) + residual`` in one product.

    ``x`` is ``[..., K]``, bfloat16 or float16; ``weight`` ``[N, K]`` of the same type;
    ``bias`` ``[N]`` of that type or float32; ``residual`` ``[..., N]``.  ``activation`` is
    "none", "silu", "gelu" (the tanh form) or "swiglu", whose weight and bias have the rows
    of the gate and then those it multiplies: ``silu(z[..., :N/2]) * z[..., N/2:]``, and the
    output ``N/2`` columns.  Sums are fp32, the output is rounded once.

    For the gradient of an activation the forward keeps ``z = x weight^T + bias`` in fp32 (in
    16 bits its rounding, beside that of ``dout * act'(z)``, would nearly double the error of a
    swiglu's gradients); ``dout * act'(z)`` is rounded to ``x``'s type as an operand of the
    products (in float16 it has to be at most 65504), and the bias's gradient adds it unrounded.
    """
    if torch.compiler.is_compiling():
        keep = activation != "none" and torch.is_grad_enabled() and any(
            t is not None and t.requires_grad for t in (x, weight, bias))
        return torch.ops.futudiffu_ii.fused_linear(x, weight, bias, residual, activation, keep)[0]
    return (_native or _load()).fused_linear(x, weight, bias, residual, activation)
