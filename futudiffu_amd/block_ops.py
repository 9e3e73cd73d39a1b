"""What surrounds the attention in a transformer block, on MI355X.

* :func:`rms_norm_modulate`      the norm before a block: ``xhat * weight * (1 + scale)``
* :func:`rms_norm_gate_residual` the norm after it: ``residual + gate * xhat * weight``
* :func:`rms_norm_gate_residual_modulate` the norm after one half of a block and the
  norm before the next, in one pass
* :func:`fused_linear`           a projection: ``act(x weight^T + bias) + residual``

``xhat = x / sqrt(mean(x^2) + eps)`` over the channels; arithmetic in fp32, one rounding
per output.  ``x`` is ``[B, N, C]`` (or ``[N, C]``), bfloat16 or float16, with any strides
(channels that are not contiguous are copied).  ``weight`` is ``[C]`` or None; ``scale``
and ``gate`` have a row per batch item, ``[B, C]``, or with ``doc_ids`` (int32 ``[B, N]``,
as :func:`futudiffu_amd.build_doc_ids` makes them) a row per document of a packed
sequence, ``[B, G, C]``: a token whose id is not in ``0 .. G-1`` (padding) has scale 0 and
gate 0, and behind a gate its ``x`` is not read.  Parameters are of ``x``'s type or float32; chunks of one projection's output are
read in place.

The functions differentiate.  Under ``torch.compile`` they go through the custom ops
``futudiffu_ii::rms_norm_modulate``, ``::rms_norm_gate_residual``,
``::rms_norm_gate_residual_modulate`` and ``::fused_linear``, which carry the same
gradients.  Sums are added in a fixed order, so results and gradients repeat bit for bit.  An empty batch gives empty outputs and zero parameter gradients.
"""

from __future__ import annotations

import functools

import torch
from torch import Tensor
from torch.autograd.function import once_differentiable

from . import _lib

_DTYPES = {torch.bfloat16: 0, torch.float16: 1}
_ops = torch.library.Library("futudiffu_ii", "FRAGMENT")


# The host's time is a large part of a small call, and all of a small training step, whose
# halves run on two threads: hence one pass over the arguments, sizes that depend on sizes
# alone kept, and no second look in the backward at what the forward checked.

def _launch(device: int, fn, *args) -> None:
    """``fn(*args, stream)`` on the current stream of ``device``, made the current device (the
    library launches there)."""
    if device == torch._C._cuda_getDevice():
        status = fn(*args, torch._C._cuda_getCurrentRawStream(device))
    else:
        with torch.cuda.device(device):
            status = fn(*args, torch._C._cuda_getCurrentRawStream(device))
    if status:
        _lib.check(status)


def _describe(t: Tensor) -> str:
    return f"{t.dtype} {list(t.shape)} on {t.device}"


def _tokens(name: str, t: Tensor, like: Tensor | None = None) -> Tensor:
    """A token tensor the kernels read in place: channels contiguous."""
    if like is not None and (t.shape != like.shape or t.dtype != like.dtype or t.get_device() != like.get_device()):
        raise ValueError(f"{name} must be a {_describe(like)} tensor, got {_describe(t)}")
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def _rows3(t: Tensor) -> tuple[int, int, int]:
    """Address and element strides per batch item and token."""
    s = t.stride()
    return (t.data_ptr(), s[0], s[1]) if len(s) == 3 else (t.data_ptr(), 0, s[0])


def _check_weight(name: str, w: Tensor, x: Tensor, C: int) -> Tensor:
    if w.shape != (C,) or w.get_device() != x.get_device() or (w.dtype != torch.float32 and w.dtype != x.dtype):
        raise ValueError(f"{name} must be a [{C}] tensor of {x.dtype} or float32 on {x.device}, got {_describe(w)}")
    return w.contiguous()


def _check_cond(name: str, k: Tensor, x: Tensor, B: int, C: int, docs: bool) -> tuple[Tensor, int, int, int]:
    """A conditioning tensor, its (batch, row) strides and its rows a batch item."""
    shape = k.shape
    ok = len(shape) == 3 and shape[0] == B and shape[1] >= 1 and shape[2] == C if docs else shape == (B, C)
    if not ok or k.get_device() != x.get_device() or (k.dtype != torch.float32 and k.dtype != x.dtype):
        want = f"[{B}, G, {C}] (with doc_ids)" if docs else f"[{B}, {C}]"
        raise ValueError(f"{name} must be a {want} tensor of {x.dtype} or float32 on {x.device}, got {_describe(k)}")
    if C != 1 and k.stride(-1) != 1:
        k = k.contiguous()
    return (k, k.stride(0), k.stride(1), shape[1]) if docs else (k, k.stride(0), 0, 1)


def _check_docs(doc_ids: Tensor, x: Tensor, B: int, N: int) -> Tensor:
    if doc_ids.shape != (B, N) and (x.ndim == 3 or doc_ids.shape != (N,)):
        raise ValueError(f"doc_ids must be [B, N] = [{B}, {N}], got {list(doc_ids.shape)}")
    if doc_ids.dtype.is_floating_point or doc_ids.dtype == torch.bool:
        raise ValueError(f"doc_ids must hold integers, got {doc_ids.dtype}")
    return doc_ids.to(device=x.device, dtype=torch.int32).contiguous()


def _wants_grad(*tensors: Tensor | None) -> bool:
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                return True
    return False


class _Norm:
    """The checked arguments of a norm call, as the library takes them."""

    __slots__ = ("x", "device", "dims", "doc", "weight", "cond", "next_weight", "next_scale", "head", "next", "tail",
                 "empty", "sizes")

    def __init__(self, x: Tensor, weight, cond_name: str, cond, doc_ids, eps: float, next_weight=None,
                 next_scale=None):
        shape = x.shape
        if len(shape) == 3:
            B, N, C = shape
        elif len(shape) == 2:
            B, (N, C) = 1, shape
        else:
            raise ValueError(f"x must be [B, N, C] or [N, C], got {list(shape)}")
        dtype = _DTYPES.get(x.dtype)
        if dtype is None:
            raise ValueError(f"x must be bfloat16 or float16, got {x.dtype}")
        if not x.is_cuda:
            raise ValueError(f"x must be a GPU tensor (device {x.device})")
        if not eps >= 0:
            raise ValueError(f"eps must be >= 0, got {eps}")
        if C < 1:
            raise ValueError(f"x needs at least one channel, got {list(shape)}")
        self.device = x.get_device()
        self.x = x = x if C == 1 or x.stride(-1) == 1 else x.contiguous()
        # tensors made for the call stay referenced until it is launched
        self.weight, self.cond, self.next_weight, self.next_scale, self.doc = weight, cond, next_weight, next_scale, None
        doc = 0
        if doc_ids is not None:
            self.doc = _check_docs(doc_ids, x, B, N)
            if cond is None and next_scale is None:
                self.doc = None  # nothing differs between documents
            else:
                doc = self.doc.data_ptr()
        f32 = wp = kp = kb = kg = 0
        groups = 0
        if weight is not None:
            self.weight = weight = _check_weight("weight", weight, x, C)
            wp, f32 = weight.data_ptr(), weight.dtype == torch.float32
        if cond is not None:
            self.cond, kb, kg, groups = _check_cond(cond_name, cond, x, B, C, self.doc is not None)
            kp = self.cond.data_ptr()
            f32 |= 2 * (cond.dtype == torch.float32)
        self.head = (wp, kp, kb, kg)
        w2 = sp = sb = sg = 0
        if next_weight is not None:
            self.next_weight = next_weight = _check_weight("next_weight", next_weight, x, C)
            w2 = next_weight.data_ptr()
            f32 |= 4 * (next_weight.dtype == torch.float32)
        if next_scale is not None:
            self.next_scale, sb, sg, rows = _check_cond("next_scale", next_scale, x, B, C, self.doc is not None)
            sp = self.next_scale.data_ptr()
            f32 |= 8 * (next_scale.dtype == torch.float32)
            if groups and groups != rows:
                raise ValueError(f"{cond_name} and next_scale must have a row for the same documents, got {groups} and "
                                 f"{rows}")
            groups = rows
        self.next = (w2, sp, sb, sg)
        groups = groups or 1
        self.sizes = (B, N, C, groups, doc != 0)
        self.tail = (groups, doc, B, N, C, dtype, int(f32), eps)
        self.empty = B == 0 or N == 0

    def workspace(self, fused: bool) -> Tensor:
        return torch.empty(_norm_workspace_bytes(*self.sizes, fused), dtype=torch.uint8, device=self.x.device)


@functools.lru_cache(maxsize=256)
def _norm_workspace_bytes(B: int, N: int, C: int, groups: int, docs: bool, fused: bool) -> int:
    return _lib.load().sage_rms_norm_bwd_workspace_bytes(B, N, C, groups, docs, fused)


def _grad(t: Tensor | None, wanted: bool) -> Tensor | None:
    return t.new_empty(t.shape) if wanted and t is not None else None


def _addr(t: Tensor | None) -> int:
    return 0 if t is None else t.data_ptr()


def _zero(*grads: Tensor | None) -> None:
    """The parameters' gradients of an empty batch."""
    for g in grads:
        if g is not None:
            g.zero_()


def _modulate_forward(x: Tensor, weight: Tensor | None, scale: Tensor | None, doc_ids: Tensor | None,
                      eps: float) -> Tensor:
    a = _Norm(x, weight, "scale", scale, doc_ids, eps)
    out = x.new_empty(x.shape)
    if not a.empty:
        _launch(a.device, _lib.load().sage_rms_norm_modulate, *_rows3(a.x), *a.head, *a.tail, out.data_ptr())
    return out


def _gate_forward(residual: Tensor, x: Tensor, weight: Tensor | None, gate: Tensor | None,
                  doc_ids: Tensor | None, eps: float) -> Tensor:
    a = _Norm(x, weight, "gate", gate, doc_ids, eps)
    r = _tokens("residual", residual, x)
    out = x.new_empty(x.shape)
    if not a.empty:
        _launch(a.device, _lib.load().sage_rms_norm_gate_residual, *_rows3(r), *_rows3(a.x), *a.head, *a.tail,
                out.data_ptr())
    return out


def _gate_modulate_forward(residual: Tensor, x: Tensor, weight: Tensor | None, gate: Tensor | None,
                           next_weight: Tensor | None, next_scale: Tensor | None, doc_ids: Tensor | None,
                           eps: float) -> tuple[Tensor, Tensor]:
    a = _Norm(x, weight, "gate", gate, doc_ids, eps, next_weight, next_scale)
    r = _tokens("residual", residual, x)
    hidden, out = x.new_empty(x.shape), x.new_empty(x.shape)
    if not a.empty:
        _launch(a.device, _lib.load().sage_rms_norm_gate_residual_modulate, *_rows3(r), *_rows3(a.x), *a.head,
                *a.next, *a.tail, hidden.data_ptr(), out.data_ptr())
    return hidden, out


def _norm_backward(name: str, cond_name: str, dout: Tensor, x: Tensor, weight: Tensor | None, cond: Tensor | None,
                   doc_ids: Tensor | None, eps: float, wanted) -> tuple[Tensor | None, ...]:
    """dx, dweight and the conditioning's gradient (None where not wanted)."""
    a = _Norm(x, weight, cond_name, cond, doc_ids, eps)
    d = _tokens("dout", dout, x)
    dx, dw, dc = _grad(x, wanted[0]), _grad(weight, wanted[1]), _grad(cond, wanted[2])
    if a.empty:
        _zero(dw, dc)
    elif dx is not None or dw is not None or dc is not None:
        ws = a.workspace(False) if dw is not None or dc is not None else None
        _launch(a.device, getattr(_lib.load(), name), *_rows3(d), *_rows3(a.x), *a.head, *a.tail, _addr(ws),
                0 if ws is None else ws.numel(), _addr(dx), _addr(dw), _addr(dc))
    return dx, dw, dc


def _gate_modulate_backward(dhidden: Tensor, dout: Tensor, residual: Tensor, x: Tensor, weight: Tensor | None,
                            gate: Tensor | None, next_weight: Tensor | None, next_scale: Tensor | None,
                            doc_ids: Tensor | None, eps: float, wanted) -> tuple[Tensor | None, ...]:
    """Gradients of residual, x, weight, gate, next_weight, next_scale (None where not
    wanted; the residual's, which the others come from, is always formed)."""
    a = _Norm(x, weight, "gate", gate, doc_ids, eps, next_weight, next_scale)
    r, d, dh = _tokens("residual", residual, x), _tokens("dout", dout, x), _tokens("dhidden", dhidden, x)
    dr, dx = x.new_empty(x.shape), _grad(x, wanted[1])
    dw, dg, dw2, ds = (_grad(p, w) for p, w in zip((weight, gate, next_weight, next_scale), wanted[2:]))
    if a.empty:
        _zero(dw, dg, dw2, ds)
    else:
        some = dw is not None or dg is not None or dw2 is not None or ds is not None
        ws = a.workspace(True) if some else None
        _launch(a.device, _lib.load().sage_rms_norm_gate_residual_modulate_bwd, *_rows3(dh), *_rows3(d), *_rows3(r),
                *_rows3(a.x), *a.head, *a.next, *a.tail, _addr(ws), 0 if ws is None else ws.numel(), dr.data_ptr(),
                _addr(dx), _addr(dw), _addr(dg), _addr(dw2), _addr(ds))
    return dr, dx, dw, dg, dw2, ds


_ACTIVATIONS = {"none": 0, "silu": 1, "gelu": 2, "swiglu": 3}


class _Linear:
    """The checked arguments of a linear call, as the library takes them."""

    __slots__ = ("x", "weight", "bias", "residual", "device", "shape", "M", "N", "K", "rows", "act", "dtype", "f32")

    def __init__(self, x: Tensor, weight: Tensor, bias: Tensor | None, residual: Tensor | None, activation: str):
        self.act = act = _ACTIVATIONS.get(activation)
        if act is None:
            raise ValueError(f"activation must be one of {sorted(_ACTIVATIONS)}, got {activation!r}")
        self.dtype = _DTYPES.get(x.dtype)
        if self.dtype is None or x.ndim < 1:
            raise ValueError(f"x must be a bfloat16 or float16 tensor [..., K], got {x.dtype} {list(x.shape)}")
        if not x.is_cuda:
            raise ValueError(f"x must be a GPU tensor (device {x.device})")
        self.device = device = x.get_device()
        lead = x.shape
        self.K = K = lead[-1]
        ws = weight.shape
        if len(ws) != 2 or ws[1] != K or K < 1 or ws[0] < 1 or weight.dtype != x.dtype or weight.get_device() != device:
            raise ValueError(f"weight must be a {x.dtype} [N, {K}] tensor on {x.device}, got {_describe(weight)}")
        self.rows = rows = ws[0]
        if act == 3 and rows % 2:
            raise ValueError(f"a swiglu weight has an even number of rows, got {rows}")
        self.N = N = rows // 2 if act == 3 else rows
        self.f32 = 0
        if bias is not None:
            self.f32 = int(bias.dtype == torch.float32)
            if bias.shape != (rows,) or bias.get_device() != device or not (self.f32 or bias.dtype == x.dtype):
                raise ValueError(f"bias must be a [{rows}] tensor of {x.dtype} or float32 on {x.device}, got "
                                 f"{_describe(bias)}")
            bias = bias.contiguous()
        self.shape = shape = (*lead[:-1], N)
        if residual is not None:
            if residual.shape != shape or residual.dtype != x.dtype or residual.get_device() != device:
                raise ValueError(f"residual must be a {x.dtype} {list(shape)} tensor on {x.device}, got "
                                 f"{_describe(residual)}")
            residual = _matrix(residual)
        self.x, self.weight, self.bias, self.residual = _matrix(x), _matrix(weight), bias, residual
        self.M = self.x.shape[0]


def _matrix(t: Tensor) -> Tensor:
    """``[..., C]`` as rows ``[M, C]`` the kernels read in place: columns contiguous, rows at
    least their width apart."""
    if t.ndim != 2:
        t = t.reshape(-1, t.shape[-1])
    M, C = t.shape
    rs, cs = t.stride()
    if (cs != 1 and C != 1) or (M > 1 and not C <= rs < 1 << 22):
        t = t.contiguous()
    return t


# the library takes addresses for their place within 16 bytes alone
@functools.lru_cache(maxsize=256)
def _linear_workspace_bytes(*args: int) -> int:
    return _lib.load().sage_linear_workspace_bytes(*args)


@functools.lru_cache(maxsize=256)
def _linear_bwd_workspace_bytes(*args: int) -> int:
    return _lib.load().sage_linear_bwd_workspace_bytes(*args)


def _linear_forward(x: Tensor, weight: Tensor, bias: Tensor | None, residual: Tensor | None, activation: str,
                    keep_z: bool) -> tuple[Tensor, Tensor | None]:
    a = _Linear(x, weight, bias, residual, activation)
    out = x.new_empty(a.shape)
    z = x.new_empty((a.M, a.rows)) if keep_z and a.act else None
    if a.M == 0:
        return out, z
    xp, xs, wp, ws = a.x.data_ptr(), a.x.stride(0), a.weight.data_ptr(), a.weight.stride(0)
    rp, rs = (0, 0) if a.residual is None else (a.residual.data_ptr(), a.residual.stride(0))
    bp = _addr(a.bias)
    size = _linear_workspace_bytes(xp & 15, xs, wp & 15, ws, a.M, a.N, a.K, a.act, (rp | bp) & 15 != 0 or rs & 7 != 0)
    work = torch.empty(size, dtype=torch.uint8, device=x.device) if size else None
    _launch(a.device, _lib.load().sage_linear, xp, xs, wp, ws, bp, a.f32, rp, rs, a.M, a.N, a.K, a.dtype, a.act,
            _addr(work), size, _addr(z), out.data_ptr())
    return out, z


def _linear_backward(dout: Tensor, x: Tensor, weight: Tensor, bias: Tensor | None, z: Tensor | None,
                     activation: str, wanted) -> tuple[Tensor | None, ...]:
    """dx, dweight, dbias (None where not wanted)."""
    a = _Linear(x, weight, bias, None, activation)
    if dout.shape != a.shape or dout.dtype != x.dtype or dout.get_device() != a.device:
        raise ValueError(f"dout must be a {x.dtype} {list(a.shape)} tensor on {x.device}, got {_describe(dout)}")
    if a.act and (z is None or z.shape != (a.M, a.rows) or z.dtype != x.dtype or not z.is_contiguous()):
        raise ValueError("the gradient of an activation needs the z that the forward kept (keep_z)")
    dx, dw, db = _grad(x, wanted[0]), _grad(weight, wanted[1]), _grad(bias, wanted[2])
    if a.M == 0:
        _zero(dw, db)
        return dx, dw, db
    want = (dx is not None) + 2 * (dw is not None) + 4 * (db is not None)
    if want:
        d = _matrix(dout)
        dp, ds, xp, xs, wp, ws = (d.data_ptr(), d.stride(0), a.x.data_ptr(), a.x.stride(0), a.weight.data_ptr(),
                                  a.weight.stride(0))
        size = _linear_bwd_workspace_bytes(dp & 15, ds, xp & 15, xs, wp & 15, ws, a.M, a.N, a.K, a.act, want)
        work = torch.empty(size, dtype=torch.uint8, device=x.device) if size else None
        _launch(a.device, _lib.load().sage_linear_bwd, dp, ds, xp, xs, wp, ws, _addr(z) if a.act else 0, a.M, a.N,
                a.K, a.dtype, a.act, a.f32, _addr(work), size, _addr(dx), _addr(dw), _addr(db))
    return dx, dw, db


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


_define("rms_norm_modulate(Tensor x, Tensor? weight, Tensor? scale, Tensor? doc_ids, float eps) -> Tensor",
        _modulate_forward, lambda x, weight, scale, doc_ids, eps: x.new_empty(x.shape))
_define("rms_norm_modulate_backward(Tensor dout, Tensor x, Tensor? weight, Tensor? scale, Tensor? doc_ids, "
        "float eps, bool[] wanted) -> (Tensor, Tensor, Tensor)",
        lambda dout, x, weight, scale, doc_ids, eps, wanted: _present(
            _norm_backward("sage_rms_norm_modulate_bwd", "scale", dout, x, weight, scale, doc_ids, eps, wanted), x),
        lambda dout, x, weight, scale, doc_ids, eps, wanted: _fake_grads(
            x, *zip((x, weight, scale), wanted)))
_define("rms_norm_gate_residual(Tensor residual, Tensor x, Tensor? weight, Tensor? gate, Tensor? doc_ids, "
        "float eps) -> Tensor",
        _gate_forward, lambda residual, x, weight, gate, doc_ids, eps: x.new_empty(x.shape))
_define("rms_norm_gate_residual_backward(Tensor dout, Tensor x, Tensor? weight, Tensor? gate, Tensor? doc_ids, "
        "float eps, bool[] wanted) -> (Tensor, Tensor, Tensor)",
        lambda dout, x, weight, gate, doc_ids, eps, wanted: _present(
            _norm_backward("sage_rms_norm_gate_residual_bwd", "gate", dout, x, weight, gate, doc_ids, eps, wanted),
            x),
        lambda dout, x, weight, gate, doc_ids, eps, wanted: _fake_grads(x, *zip((x, weight, gate), wanted)))
_define("rms_norm_gate_residual_modulate(Tensor residual, Tensor x, Tensor? weight, Tensor? gate, "
        "Tensor? next_weight, Tensor? next_scale, Tensor? doc_ids, float eps) -> (Tensor, Tensor)",
        _gate_modulate_forward,
        lambda residual, x, weight, gate, next_weight, next_scale, doc_ids, eps: (x.new_empty(x.shape),
                                                                                 x.new_empty(x.shape)))
_define("rms_norm_gate_residual_modulate_backward(Tensor dhidden, Tensor dout, Tensor residual, Tensor x, "
        "Tensor? weight, Tensor? gate, Tensor? next_weight, Tensor? next_scale, Tensor? doc_ids, float eps, "
        "bool[] wanted) -> (Tensor, Tensor, Tensor, Tensor, Tensor, Tensor)",
        lambda dhidden, dout, residual, x, *rest: _present(
            _gate_modulate_backward(dhidden, dout, residual, x, *rest), x),
        lambda dhidden, dout, residual, x, weight, gate, next_weight, next_scale, doc_ids, eps, wanted: _fake_grads(
            x, (x, True), (x, wanted[1]), *zip((weight, gate, next_weight, next_scale), wanted[2:])))


def _modulate_setup(ctx, inputs, output):
    x, weight, scale, doc_ids, eps = inputs
    ctx.save_for_backward(x, weight, scale, doc_ids)
    ctx.eps = eps


def _modulate_autograd(ctx, dout):
    x, weight, scale, doc_ids = ctx.saved_tensors
    wanted = _wanted(ctx, (0, 1, 2), (x, weight, scale))
    grads = torch.ops.futudiffu_ii.rms_norm_modulate_backward(dout, x, weight, scale, doc_ids, ctx.eps, wanted)
    return *_only(grads, wanted), None, None


def _gate_setup(ctx, inputs, output):
    residual, x, weight, gate, doc_ids, eps = inputs
    ctx.save_for_backward(x, weight, gate, doc_ids)
    ctx.eps = eps


def _gate_autograd(ctx, dout):
    x, weight, gate, doc_ids = ctx.saved_tensors
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


class _Modulate(torch.autograd.Function):
    """The op and its formula without the dispatch of a Python op, which takes the host longer
    than a step's kernels take the GPU."""

    @staticmethod
    def forward(ctx, *inputs):
        _modulate_setup(ctx, inputs, None)
        return _modulate_forward(*inputs)

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        x, weight, scale, doc_ids = ctx.saved_tensors
        return *_norm_backward("sage_rms_norm_modulate_bwd", "scale", dout, x, weight, scale, doc_ids, ctx.eps,
                               ctx.needs_input_grad[:3]), None, None


class _Gate(torch.autograd.Function):
    @staticmethod
    def forward(ctx, *inputs):
        _gate_setup(ctx, inputs, None)
        return _gate_forward(*inputs)

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        x, weight, gate, doc_ids = ctx.saved_tensors
        need = ctx.needs_input_grad
        return (dout if need[0] else None, *_norm_backward(
            "sage_rms_norm_gate_residual_bwd", "gate", dout, x, weight, gate, doc_ids, ctx.eps, need[1:4]), None, None)


class _GateModulate(torch.autograd.Function):
    @staticmethod
    def forward(ctx, *inputs):
        _gate_modulate_setup(ctx, inputs, None)
        return _gate_modulate_forward(*inputs)

    @staticmethod
    @once_differentiable
    def backward(ctx, dhidden, dout):
        residual, x, weight, gate, next_weight, next_scale, doc_ids = ctx.saved_tensors
        need = ctx.needs_input_grad
        grads = _gate_modulate_backward(dhidden, dout, residual, x, weight, gate, next_weight, next_scale, doc_ids,
                                        ctx.eps, need[:6])
        return *_only(grads, need), None, None


_define("fused_linear(Tensor x, Tensor weight, Tensor? bias, Tensor? residual, str activation, bool keep_z) "
        "-> (Tensor, Tensor)",
        lambda x, weight, bias, residual, activation, keep_z: _present(
            _linear_forward(x, weight, bias, residual, activation, keep_z), x),
        lambda x, weight, bias, residual, activation, keep_z: (
            x.new_empty(*x.shape[:-1], weight.shape[0] // (2 if activation == "swiglu" else 1)),
            x.new_empty(x.numel() // x.shape[-1], weight.shape[0]) if keep_z and activation != "none"
            else x.new_empty(0)))
_define("fused_linear_backward(Tensor dout, Tensor x, Tensor weight, Tensor? bias, Tensor? z, str activation, "
        "bool[] wanted) -> (Tensor, Tensor, Tensor)",
        lambda dout, x, weight, bias, z, activation, wanted: _present(
            _linear_backward(dout, x, weight, bias, z, activation, wanted), x),
        lambda dout, x, weight, bias, z, activation, wanted: _fake_grads(x, *zip((x, weight, bias), wanted)))


def _linear_setup(ctx, inputs, output):
    x, weight, bias, residual, activation, keep_z = inputs
    ctx.mark_non_differentiable(output[1])
    ctx.save_for_backward(x, weight, bias, output[1])
    ctx.activation = activation


def _linear_autograd(ctx, dout, dz):
    x, weight, bias, z = ctx.saved_tensors
    wanted = _wanted(ctx, range(3), (x, weight, bias))
    grads = (None, None, None)
    if any(wanted):
        grads = torch.ops.futudiffu_ii.fused_linear_backward(dout, x, weight, bias, z, ctx.activation, wanted)
    return *_only(grads, wanted), dout if ctx.needs_input_grad[3] else None, None, None


torch.library.register_autograd("futudiffu_ii::fused_linear", _linear_autograd, setup_context=_linear_setup, lib=_ops)


class _FusedLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, activation):
        out, z = _linear_forward(x, weight, bias, residual, activation, True)
        ctx.save_for_backward(x, weight, bias, z)
        ctx.activation = activation
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        x, weight, bias, z = ctx.saved_tensors
        need = ctx.needs_input_grad
        return (*_linear_backward(dout, x, weight, bias, z, ctx.activation, need[:3]), dout if need[3] else None, None)


# ---- the functions ---------------------------------------------------------------------

def rms_norm_modulate(x: Tensor, weight: Tensor | None = None, scale: Tensor | None = None, *,
                      doc_ids: Tensor | None = None, eps: float = 1e-5) -> Tensor:
    """``xhat * weight * (1 + scale)``: the norm before a block with its modulation."""
    if torch.compiler.is_compiling():
        return torch.ops.futudiffu_ii.rms_norm_modulate(x, weight, scale, doc_ids, eps)
    if _wants_grad(x, weight, scale):
        return _Modulate.apply(x, weight, scale, doc_ids, eps)
    return _modulate_forward(x, weight, scale, doc_ids, eps)


def rms_norm_gate_residual(residual: Tensor, x: Tensor, weight: Tensor | None = None, gate: Tensor | None = None, *,
                           doc_ids: Tensor | None = None, eps: float = 1e-5) -> Tensor:
    """``residual + gate * xhat * weight``: the norm after a block, gated, onto the residual."""
    if torch.compiler.is_compiling():
        return torch.ops.futudiffu_ii.rms_norm_gate_residual(residual, x, weight, gate, doc_ids, eps)
    if _wants_grad(residual, x, weight, gate):
        return _Gate.apply(residual, x, weight, gate, doc_ids, eps)
    return _gate_forward(residual, x, weight, gate, doc_ids, eps)


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
    if _wants_grad(residual, x, weight, gate, next_weight, next_scale):
        return _GateModulate.apply(residual, x, weight, gate, next_weight, next_scale, doc_ids, eps)
    return _gate_modulate_forward(residual, x, weight, gate, next_weight, next_scale, doc_ids, eps)


def fused_linear(x: Tensor, weight: Tensor, bias: Tensor | None = None, residual: Tensor | None = None, *,
                 activation: str = "none") -> Tensor:
    """``act(x weight^T + bias) + residual`` in one product.

    ``x`` is ``[..., K]``, bfloat16 or float16; ``weight`` ``[N, K]`` of the same type;
    ``bias`` ``[N]`` of that type or float32; ``residual`` ``[..., N]``.  ``activation`` is
    "none", "silu", "gelu" (the tanh form) or "swiglu", whose weight and bias have the rows
    of the gate and then those it multiplies: ``silu(z[..., :N/2]) * z[..., N/2:]``, and the
    output ``N/2`` columns.  Sums are fp32, the output is rounded once.

    For the gradient of an activation the forward keeps ``z = x weight^T + bias`` rounded to
    ``x``'s type, and ``dout * act'(z)`` is rounded to it as an operand of the products, each
    as a 16-bit framework does it; the bias's gradient adds it unrounded.
    """
    if torch.compiler.is_compiling():
        keep = activation != "none" and _wants_grad(x, weight, bias, residual)
        return torch.ops.futudiffu_ii.fused_linear(x, weight, bias, residual, activation, keep)[0]
    if _wants_grad(x, weight, bias, residual):
        return _FusedLinear.apply(x, weight, bias, residual, activation)
    return _linear_forward(x, weight, bias, residual, activation, False)[0]
