"""Activations kept in eight bits between the forward and the backward pass.

``Int8Linear`` already saves its input as int8; what stands between such layers would save
fp32 or bf16.  Here those activations are saved as int8 with one fp32 scale per 128
consecutive columns of a row (``scale = amax / 127``, ``q = rint(x * (127 / amax))``, each step
one fp32 rounding), and the backward kernels read the eight bits in place:

* ``checkpoint_i8`` / ``restore_i8``: put a tensor away and bring it back;
* ``saved_i8``: a context in which autograd saves its activations that way;
* ``rms_norm_i8`` / ``Int8RMSNorm`` and ``gated_act_i8`` / ``Int8GatedAct``: the norm and the gated
  activation of a feed-forward block, forward exact, saved inputs eight bits, both directions
  one pass over the data.

Tensors are fp32, bf16 or fp16 of any shape whose last dimension is the row.  A block whose
largest value is below 2^-119 comes back as zeros; one that holds an infinity or NaN comes
back as NaN.  Outputs whose rows are no multiple of eight columns have padded row strides.
"""

from __future__ import annotations

import contextlib
import ctypes
import math

import torch
import torch.nn as nn

from . import _native as nat

BLOCK = 128  # ECO_CKPT_BLOCK
_ACTS = {"silu": 0, "gelu": 1}
_FLOATS = (torch.float32, torch.bfloat16, torch.float16)


def _matrix(t: torch.Tensor, name: str) -> torch.Tensor:
    """``t`` as ``[rows, cols]`` with unit column stride (a view where its strides allow one)."""
    shape = t.shape
    if t.dtype not in _FLOATS or len(shape) < 1:
        raise AssertionError(f"{name} must be an fp32, bf16 or fp16 tensor of at least one dimension")
    if shape[-1] == 0:
        raise AssertionError(f"{name} has empty rows")
    m = t if len(shape) == 2 else t.reshape(-1, shape[-1])
    ld, unit = m.stride()
    return m if (unit == 1 or m.shape[1] == 1) and ld < 1 << 31 else m.contiguous()


def _empty_rows(like: torch.Tensor, rows: int, cols: int, dtype=None) -> torch.Tensor:
    """``[rows, cols]`` whose rows start on a multiple of eight elements."""
    if cols % 8 == 0:
        return like.new_empty((rows, cols), dtype=dtype)
    return like.new_empty((rows, (cols + 7) // 8 * 8), dtype=dtype)[:, :cols]


def _shaped(m: torch.Tensor, shape) -> torch.Tensor:
    return m if m.shape == shape else m.view(shape)


def _eight(like: torch.Tensor, rows: int, cols: int):
    """int8 rows and fp32 block scales of a ``[rows, cols]`` matrix."""
    return (like.new_empty((rows, (cols + 15) // 16 * 16), dtype=torch.int8),
            like.new_empty((rows, (cols + BLOCK - 1) // BLOCK), dtype=torch.float32))


def _spec(q, scale):
    return nat.SavedI8(q.data_ptr(), scale.data_ptr(), q.shape[1], scale.shape[1])


class Checkpoint8:
    """A tensor in eight bits: ``q`` int8 ``[rows, cols padded to 16]``, ``scale`` fp32 ``[rows,
    blocks]``, and the ``shape`` and ``dtype`` it had."""

    __slots__ = ("q", "scale", "shape", "dtype")

    def __init__(self, q, scale, shape, dtype):
        self.q, self.scale, self.shape, self.dtype = q, scale, shape, dtype

    def memory_bytes(self) -> int:
        return self.q.numel() + 4 * self.scale.numel()


def checkpoint_i8(x: torch.Tensor) -> Checkpoint8:
    """``x`` in eight bits (``restore_i8`` brings it back)."""
    dev = nat.require_cuda(x)
    m = _matrix(x, "x")
    rows, cols = m.shape
    with nat.on_device(dev):
        q, scale = _eight(m, rows, cols)
        nat.call("eco_ckpt_pack", m.data_ptr(), nat.TYPES[m.dtype], rows, cols, m.stride(0),
                 ctypes.byref(_spec(q, scale)), nat.stream())
    return Checkpoint8(q, scale, x.shape, x.dtype)


def restore_i8(c: Checkpoint8, dtype: torch.dtype | None = None) -> torch.Tensor:
    """The values the eight bits stand for, in the tensor's shape and its type (or ``dtype``)."""
    dtype = c.dtype if dtype is None else dtype
    if dtype not in _FLOATS:
        raise AssertionError("dtype must be fp32, bf16 or fp16")
    dev = nat.require_cuda(c.q, c.scale)
    rows, cols = c.q.shape[0], c.shape[-1]
    with nat.on_device(dev):
        x = _empty_rows(c.q, rows, cols, dtype)
        nat.call("eco_ckpt_restore", ctypes.byref(_spec(c.q, c.scale)), nat.TYPES[dtype], rows, cols, x.data_ptr(),
                 x.stride(0), nat.stream())
    return _shaped(x, c.shape)


def _is_weight(t: torch.Tensor) -> bool:
    base = t if t._base is None else t._base
    return isinstance(base, nn.Parameter) or (base.is_leaf and base.requires_grad)


@contextlib.contextmanager
def saved_i8(min_numel: int = 1 << 16):
    """Inside this context, autograd keeps the floating CUDA activations it saves in eight bits.

    Parameters and other leaves that ask for gradients (and views of them), tensors of other
    types or layouts and those of fewer than ``min_numel`` values are kept as they are.  A tensor that
    is not kept by its caller is freed; its backward formula reads what the eight bits stand for."""

    def pack(t):
        if not t.is_cuda or t.layout is not torch.strided or t.dtype not in _FLOATS or t.dim() < 1 or \
                t.numel() < max(1, min_numel) or _is_weight(t):
            return t
        return checkpoint_i8(t.detach())

    def unpack(s):
        return restore_i8(s) if isinstance(s, Checkpoint8) else s

    with torch.autograd.graph.saved_tensors_hooks(pack, unpack):
        yield


# ------------------------------------------------------------------ rms norm


class _RMSNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, eps):
        dev = nat.require_cuda(x, weight)
        m = _matrix(x, "x")
        rows, cols = m.shape
        if weight is not None:
            if weight.shape != (cols,) or weight.dtype not in (torch.float32, x.dtype):
                raise AssertionError(f"weight must be [{cols}], fp32 or of x's type")
            weight = weight.contiguous()
        eps = float(eps)
        if not (eps >= 0.0 and math.isfinite(eps)):
            raise ValueError("eps must not be negative")
        wants = ctx.needs_input_grad[0] or ctx.needs_input_grad[1]
        kind, w_kind = nat.TYPES[m.dtype], 0 if weight is None else nat.TYPES[weight.dtype]
        q = scale = rstd = saved = None
        with nat.on_device(dev):
            y = _empty_rows(m, rows, cols)
            if wants:
                q, scale = _eight(m, rows, cols)
                rstd = m.new_empty(rows, dtype=torch.float32)
                saved = ctypes.byref(_spec(q, scale))
            nat.call("eco_rms_norm", m.data_ptr(), m.stride(0), kind, rows, cols, nat.ptr(weight), w_kind, eps,
                     y.data_ptr(), y.stride(0), saved, nat.ptr(rstd), nat.stream())
        if wants:
            # q and the weight are open to saved-tensor hooks; scales and roots stay as they are
            ctx.save_for_backward(q, weight)
            ctx.own = (scale, rstd, x.shape, kind, w_kind)
        return _shaped(y, x.shape)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        q, weight = ctx.saved_tensors
        scale, rstd, shape, kind, w_kind = ctx.own
        m = _matrix(dy, "dy")
        rows, cols = m.shape
        with nat.on_device(m.device):
            dx = _empty_rows(m, rows, cols)
            dw = scratch = None
            room = 0
            if weight is not None and ctx.needs_input_grad[1]:
                dw = torch.empty_like(weight)
                room = nat.load().eco_rms_norm_bwd_scratch(rows, cols)
                scratch = m.new_empty(room, dtype=torch.float32)
            nat.call("eco_rms_norm_bwd", m.data_ptr(), m.stride(0), kind, rows, cols, nat.ptr(weight), w_kind,
                     ctypes.byref(_spec(q, scale)), rstd.data_ptr(), dx.data_ptr(), dx.stride(0), nat.ptr(dw),
                     nat.ptr(scratch), room, nat.stream())
        return _shaped(dx, shape), dw, None


def rms_norm_i8(x: torch.Tensor, weight: torch.Tensor | None = None, eps: float = 1e-6) -> torch.Tensor:
    """``x / sqrt(mean(x^2) + eps) * weight`` over the last dimension; ``x`` is saved in eight bits.

    ``weight``: ``[cols]``, fp32 or of ``x``'s type (None: ones).  Differentiable with respect to
    both; the reciprocal root is saved in fp32, and ``dweight`` sums its rows in a fixed order."""
    return _RMSNorm.apply(x, weight, eps)


class Int8RMSNorm(nn.Module):
    """``rms_norm_i8`` with its weight (ones at the start)."""

    def __init__(self, features: int, eps: float = 1e-6):
        super().__init__()
        self.weight = nn.Parameter(torch.ones(features))
        self.eps = eps

    def forward(self, x):
        return rms_norm_i8(x, self.weight, self.eps)

    def extra_repr(self):
        return f"{self.weight.shape[0]}, eps={self.eps}"


# ------------------------------------------------------------------ gated activation


class _GatedAct(torch.autograd.Function):
    @staticmethod
    def forward(ctx, gate, up, act):
        if act not in _ACTS:
            raise ValueError(f"act must be one of {sorted(_ACTS)}")
        dev = nat.require_cuda(gate, up)
        g = _matrix(gate, "gate")
        if up is None:
            if g.shape[1] % 2:
                raise AssertionError("without up, gate holds both halves: an even number of columns")
            cols = g.shape[1] // 2
            up_at, up_ld = g.data_ptr() + cols * g.element_size(), g.stride(0)
        else:
            if up.shape != gate.shape or up.dtype != gate.dtype:
                raise AssertionError("gate and up must have one shape and type")
            u, cols = _matrix(up, "up"), g.shape[1]
            up_at, up_ld = u.data_ptr(), u.stride(0)
        rows, kind = g.shape[0], nat.TYPES[g.dtype]
        wants = ctx.needs_input_grad[0] or ctx.needs_input_grad[1]
        with nat.on_device(dev):
            y = _empty_rows(g, rows, cols)
            eg = eu = (None, None)
            if wants:
                eg, eu = _eight(g, rows, cols), _eight(g, rows, cols)
            nat.call("eco_gated_act", g.data_ptr(), g.stride(0), up_at, up_ld, kind, _ACTS[act], rows, cols,
                     y.data_ptr(), y.stride(0), ctypes.byref(_spec(*eg)) if wants else None,
                     ctypes.byref(_spec(*eu)) if wants else None, nat.stream())
        if wants:
            ctx.save_for_backward(eg[0], eu[0])
            ctx.own = (eg[1], eu[1], act, up is None, gate.shape)
        return _shaped(y, (*gate.shape[:-1], cols))

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        gq, uq = ctx.saved_tensors
        gs, us, act, packed, shape = ctx.own
        m = _matrix(dy, "dy")
        rows, cols = m.shape
        with nat.on_device(m.device):
            if packed:
                dg, du = _empty_rows(m, rows, 2 * cols), None
                du_at, du_ld = dg.data_ptr() + cols * dg.element_size(), dg.stride(0)
            else:
                dg, du = _empty_rows(m, rows, cols), _empty_rows(m, rows, cols)
                du_at, du_ld = du.data_ptr(), du.stride(0)
            nat.call("eco_gated_act_bwd", m.data_ptr(), m.stride(0), nat.TYPES[m.dtype], _ACTS[act], rows, cols,
                     ctypes.byref(_spec(gq, gs)), ctypes.byref(_spec(uq, us)), dg.data_ptr(), dg.stride(0),
                     du_at, du_ld, nat.stream())
        return _shaped(dg, shape), None if packed else _shaped(du, shape), None


def gated_act_i8(gate: torch.Tensor, up: torch.Tensor | None = None, act: str = "silu") -> torch.Tensor:
    """``act(gate) * up``, both saved in eight bits; ``act``: ``"silu"`` or ``"gelu"`` (error function).

    With ``up`` None, ``gate`` holds both halves of one projection, ``[..., 2 F]``: gate, then up;
    the gradient comes as one tensor of that shape.  Differentiable."""
    return _GatedAct.apply(gate, up, act)


class Int8GatedAct(nn.Module):
    """``gated_act_i8`` of a projection that holds gate and up side by side."""

    def __init__(self, act: str = "silu"):
        super().__init__()
        if act not in _ACTS:
            raise ValueError(f"act must be one of {sorted(_ACTS)}")
        self.act = act

    def forward(self, x):
        return gated_act_i8(x, act=self.act)

    def extra_repr(self):
        return self.act
