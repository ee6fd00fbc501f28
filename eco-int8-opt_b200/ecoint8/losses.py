"""Post-training objectives on a model's logits, with their gradients.

The reference's one objective is cross entropy (``ecoint8.quant.cross_entropy_grad_i8``
here); these stand beside it, and need the log-probability of one given token per row:

* ``token_logprobs``: the log-probabilities (what old and reference policies are asked for);
* ``policy_loss``: clipped policy loss with a KL term against a reference;
* ``preference_loss``: a loss over pairs of log ratios (preferred against rejected sequences).

Each loss has two forms.  ``*_loss_grad`` returns the loss and the gradient with respect to
the logits in one call, as ``cross_entropy_grad_i8`` does: for loops that feed a gradient to
``backward_i8`` themselves (int8 logits with their scale ``s_out``; the gradient is fp32,
with respect to the dequantized logits, for ``quantize_tensor_dynamic``) and for CUDA-graph
capture.  ``*_loss`` is differentiable: its backward reads the logits again and computes the
probabilities anew, so nothing of the logits' size is kept.

Logits are ``[rows, vocab]`` or ``[batch, length, vocab]``, fp32, bf16, fp16 or int8, with any
row strides (``logits[:, :-1]`` is read in place) as long as the vocabulary is contiguous.
Rows with a false ``mask`` or a token outside ``[0, vocab)`` (such as -100) do not count: their
logits are not read and may hold anything, and their gradient is zero.  Sums over rows are
taken in fp64 and in a fixed order: the same call gives the same bits.  A row of infinities or
NaN that counts makes its results NaN.  A gradient row starts as far
behind a vector boundary as its logits row does, so gradients may come with padded strides.
"""

from __future__ import annotations

import ctypes
import math
from typing import NamedTuple

import torch

from . import _native as nat

_KINDS = {"sigmoid": 0, "hinge": 1, "ipo": 2}


class PolicyLoss(NamedTuple):
    """``loss``, ``kl`` (mean of the KL term) and ``clip_fraction``: 0-dim fp32 on the device;
    ``grad``: the logits' gradient (None from ``policy_loss``); ``logp``: fp32 per token, 0
    where a row does not count."""

    loss: torch.Tensor
    grad: torch.Tensor | None
    logp: torch.Tensor
    kl: torch.Tensor
    clip_fraction: torch.Tensor


class PreferenceLoss(NamedTuple):
    """``loss``: 0-dim fp32; ``grad``: the logits' gradient (None from ``preference_loss``);
    ``log_ratio`` fp32 ``[2 pairs]``: each sequence's sum (or mean) of ``logp - ref_logp``;
    ``margin`` fp32 ``[pairs]``: ``beta`` times the preferred less the rejected one's."""

    loss: torch.Tensor
    grad: torch.Tensor | None
    log_ratio: torch.Tensor
    margin: torch.Tensor


def _spec(x, mul):
    n0, n1, s0, s1 = (1, x.shape[0], 0, x.stride(0)) if x.dim() == 2 else (*x.shape[:2], x.stride(0), x.stride(1))
    return nat.Logits(x.data_ptr(), nat.TYPES[x.dtype], 0, n0, n1, s0, s1, x.shape[-1], mul)


class _Rows:
    """Logits as the kernels take them, with their tokens and mask."""

    __slots__ = ("x", "spec", "lead", "rows", "tokens", "mask", "gain", "dev")

    def __init__(self, logits, tokens, mask, temperature, s_out):
        self.dev = nat.require_cuda(logits, tokens, mask)
        dtype, shape = logits.dtype, logits.shape
        if dtype not in nat.TYPES or len(shape) not in (2, 3):
            raise AssertionError("logits must be fp32, bf16, fp16 or int8, [rows, vocab] or [batch, length, vocab]")
        self.lead = lead = shape[:-1]
        if tokens.dtype != torch.int64 or tokens.shape != lead:
            raise AssertionError(f"tokens must be int64 {list(lead)}, one per row of logits")
        if mask is not None and (mask.dtype not in (torch.bool, torch.uint8) or mask.shape != lead):
            raise AssertionError(f"mask must be bool {list(lead)}")
        if shape[-1] == 0:
            raise AssertionError("an empty vocabulary")
        temperature = float(temperature)
        if not 1e-15 <= temperature <= 1e15:
            raise ValueError("temperature must be positive (and within [1e-15, 1e15])")
        if (dtype is torch.int8) != (s_out is not None):
            raise ValueError("int8 logits need their scale s_out, and only they have one")
        scale = 1.0 if s_out is None else float(s_out)
        if not 1e-15 <= scale <= 1e15:
            raise ValueError("s_out must be positive (and within [1e-15, 1e15])")
        self.x = x = logits if logits.stride(-1) == 1 or shape[-1] == 1 else logits.contiguous()
        self.gain = 1.0 / temperature
        self.rows = tokens.numel()
        self.spec = _spec(x, scale / temperature)
        self.tokens = tokens.contiguous()
        self.mask = None if mask is None else mask.contiguous()

    def per_row(self, t, name):
        """A per-token fp32 tensor in the rows' order (broadcast to the tokens' shape)."""
        if t is None:
            return None
        if t.device != self.dev:
            nat.require_cuda(self.x, t)
        if t.dtype is not torch.float32:
            raise AssertionError(f"{name} must be fp32")
        if t.shape != self.lead:
            try:
                t = t.expand(self.lead)
            except RuntimeError:
                raise AssertionError(f"{name} must broadcast to {list(self.lead)}") from None
        return t.contiguous()

    def new_grad(self):
        """``(tensor, eco_grad_t)``: rows that start like the logits' rows, modulo a 16-byte vector of those."""
        x, cols = self.x, self.x.shape[-1]
        n0, n1 = self.spec.n0, self.spec.n1
        dtype = torch.float32 if x.dtype == torch.int8 else x.dtype
        es = x.element_size()
        per, skew, want0, want1 = 16 // es, x.data_ptr() % 16 // es, self.spec.s0, self.spec.s1
        s1 = cols + (want1 - cols) % per
        s0 = n1 * s1 + (want0 - n1 * s1) % per if n0 > 1 else n1 * s1
        if skew == 0 and s1 == cols and s0 == n1 * s1:
            g = x.new_empty(x.shape, dtype=dtype)
        else:
            shape, strides = ((n1, cols), (s1, 1)) if x.dim() == 2 else ((n0, n1, cols), (s0, s1, 1))
            g = x.new_empty(skew + n0 * s0, dtype=dtype).as_strided(shape, strides, skew)
        return g, nat.Grad(g.data_ptr(), s0, s1)

    def token_grad(self, stats: int, coef: int, scale=None):
        """The gradient from row statistics and coefficients (device addresses)."""
        with nat.on_device(self.dev):
            g, spec = self.new_grad()
            nat.call("eco_token_grad", ctypes.byref(self.spec), self.tokens.data_ptr(), stats, coef, nat.ptr(scale),
                     self.gain, ctypes.byref(spec), nat.stream())
        return g

    def workspace(self, pairs: int = 0):
        """``(buffer, fp64 log-probabilities and pairs, row statistics, coefficients)``: one allocation
        and the addresses of its three parts (statistics are two fp32 numbers per row)."""
        n = self.rows
        buf = self.tokens.new_empty(2 * n + pairs + (n + 1) // 2, dtype=torch.float64)
        at = buf.data_ptr()
        return buf, at, at + 8 * (n + pairs), at + 8 * (2 * n + pairs)

    def new(self, *shape, dtype=torch.float32):
        return self.tokens.new_empty(shape, dtype=dtype)


def _keep_rows(ctx, rows, buf, stats, coef=None):
    # The logits and tokens go through autograd's saved tensors (checked for changes in place,
    # and open to hooks that move or pack them); the row statistics and coefficients are the
    # kernels' own and stay where they are.
    ctx.save_for_backward(rows.x, rows.tokens)
    ctx.own = (rows.gain, rows.spec.mul, buf, stats, coef)


def _saved_rows(ctx):
    """``(rows, statistics, coefficients)``: the forward's rows over the tensors that autograd hands back."""
    x, tokens = ctx.saved_tensors
    gain, mul, _, stats, coef = ctx.own
    rows = _Rows.__new__(_Rows)
    rows.x = x if x.stride(-1) == 1 or x.shape[-1] == 1 else x.contiguous()
    rows.tokens, rows.mask, rows.gain, rows.dev = tokens.contiguous(), None, gain, x.device
    rows.lead, rows.rows = tokens.shape, tokens.numel()
    rows.spec = _spec(rows.x, mul)
    return rows, stats, coef


# ------------------------------------------------------------------ log-probabilities


class _TokenLogprobs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, tokens, mask, temperature, s_out):
        rows = _Rows(logits, tokens, mask, temperature, s_out)
        with nat.on_device(rows.dev):
            logp = rows.new(*rows.lead)
            stats = rows.new(rows.rows, 2) if ctx.needs_input_grad[0] else None
            nat.call("eco_token_logp", ctypes.byref(rows.spec), rows.tokens.data_ptr(), nat.ptr(rows.mask), None, 0,
                     logp.data_ptr(), None, nat.ptr(stats), None, nat.stream())
        if stats is not None:
            _keep_rows(ctx, rows, stats, stats.data_ptr())
        return logp

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dlogp):
        rows, stats, _ = _saved_rows(ctx)
        dlogp = dlogp.contiguous()
        return rows.token_grad(stats, dlogp.data_ptr()), None, None, None, None


def token_logprobs(logits: torch.Tensor, tokens: torch.Tensor, *, mask: torch.Tensor | None = None,
                   temperature: float = 1.0, s_out: float | None = None) -> torch.Tensor:
    """``log softmax(logits / temperature)`` at ``tokens``: fp32, the tokens' shape, 0 where a
    row does not count.  Differentiable with respect to floating logits."""
    return _TokenLogprobs.apply(logits, tokens, mask, temperature, s_out)


# ------------------------------------------------------------------ policy loss


def _policy_args(rows, old_logp, advantages, ref_logp, clip_low, clip_high, kl_coef, denom):
    old = rows.per_row(old_logp, "old_logp")
    adv = rows.per_row(advantages, "advantages")
    ref = rows.per_row(ref_logp, "ref_logp")
    clip_low, clip_high, kl_coef = float(clip_low), float(clip_high), float(kl_coef)
    if not (0.0 <= clip_low <= 1.0 and clip_high >= 0.0):
        raise ValueError("clip_low must lie in [0, 1] and clip_high must not be negative")
    if not math.isfinite(kl_coef):
        raise ValueError("kl_coef must be finite")
    if kl_coef != 0.0 and ref is None:
        raise ValueError("a KL term needs ref_logp")
    denom = 0.0 if denom is None else float(denom)
    if denom < 0.0 or not math.isfinite(denom):
        raise ValueError("denom must be positive")
    keep = (old, adv, ref)
    return keep, (old.data_ptr(), adv.data_ptr(), nat.ptr(ref), 1.0 - clip_low, 1.0 + clip_high, kl_coef, denom)


def policy_loss_grad(logits: torch.Tensor, tokens: torch.Tensor, old_logp: torch.Tensor, advantages: torch.Tensor, *,
                     ref_logp: torch.Tensor | None = None, mask: torch.Tensor | None = None, clip_low: float = 0.2,
                     clip_high: float = 0.2, kl_coef: float = 0.0, temperature: float = 1.0,
                     s_out: float | None = None, denom: float | None = None) -> PolicyLoss:
    """Clipped policy loss with a KL term, and its gradient with respect to the logits.

    Over the rows that count, with ``lp = token_logprobs(...)`` and ``r = exp(lp - old_logp)``::

        loss = sum(max(-A r, -A clip(r, 1 - clip_low, 1 + clip_high)) + kl_coef k) / denom
        k    = exp(ref_logp - lp) - (ref_logp - lp) - 1

    ``advantages`` (A), ``old_logp`` and ``ref_logp`` are fp32 and broadcast to the tokens' shape.
    ``denom``: default the number of rows that count (at least 1); a caller that splits a batch
    over steps or ranks gives the whole batch's.  No row that counts: loss and gradient 0.  One
    read of the logits and one write of the gradient; no host synchronisation."""
    rows = _Rows(logits, tokens, mask, temperature, s_out)
    keep, args = _policy_args(rows, old_logp, advantages, ref_logp, clip_low, clip_high, kl_coef, denom)
    with nat.on_device(rows.dev):
        g, spec = rows.new_grad()
        logp, terms, out = rows.new(*rows.lead), rows.new(3 * rows.rows + 64), rows.new(3)
        nat.call("eco_policy_grad", ctypes.byref(rows.spec), rows.tokens.data_ptr(), nat.ptr(rows.mask), *args,
                 rows.gain, logp.data_ptr(), terms.data_ptr(), out.data_ptr(), ctypes.byref(spec), nat.stream())
    loss, kl, clipped = out.unbind()
    return PolicyLoss(loss, g, logp, kl, clipped)


class _PolicyLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, tokens, mask, temperature, s_out, old_logp, advantages, ref_logp, *how):
        rows = _Rows(logits, tokens, mask, temperature, s_out)
        keep, args = _policy_args(rows, old_logp, advantages, ref_logp, *how)
        with nat.on_device(rows.dev):
            logp, out = rows.new(*rows.lead), rows.new(3)
            buf, lp64, stats, coef = rows.workspace()
            nat.call("eco_policy_forward", ctypes.byref(rows.spec), rows.tokens.data_ptr(), nat.ptr(rows.mask), *args,
                     logp.data_ptr(), lp64, stats, coef, out.data_ptr(), nat.stream())
        _keep_rows(ctx, rows, buf, stats, coef)
        loss, kl, clipped = out.unbind()
        ctx.mark_non_differentiable(logp, kl, clipped)
        ctx.set_materialize_grads(False)
        return loss, logp, kl, clipped

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dloss, *_):
        if dloss is None:
            return (None,) * 12
        rows, stats, coef = _saved_rows(ctx)
        return (rows.token_grad(stats, coef, dloss),) + (None,) * 11


def policy_loss(logits: torch.Tensor, tokens: torch.Tensor, old_logp: torch.Tensor, advantages: torch.Tensor, *,
                ref_logp: torch.Tensor | None = None, mask: torch.Tensor | None = None, clip_low: float = 0.2,
                clip_high: float = 0.2, kl_coef: float = 0.0, temperature: float = 1.0, s_out: float | None = None,
                denom: float | None = None) -> PolicyLoss:
    """``policy_loss_grad`` as a differentiable loss (``.grad`` is None; call ``.loss.backward()``).
    Gradients flow to the logits alone."""
    loss, logp, kl, clipped = _PolicyLoss.apply(logits, tokens, mask, temperature, s_out, old_logp, advantages,
                                                ref_logp, clip_low, clip_high, kl_coef, denom)
    return PolicyLoss(loss, None, logp, kl, clipped)


# ------------------------------------------------------------------ preference loss


def _preference(rows, with_grad, ref_logp, beta, kind, label_smoothing, average, cu_seqlens, denom):
    """``(workspace, its parts, loss, log ratios, margins, gradient or None)`` in one call."""
    ref = rows.per_row(ref_logp, "ref_logp")
    if ref is None:
        raise AssertionError("ref_logp must be given")
    if kind not in _KINDS:
        raise ValueError(f"kind must be one of {sorted(_KINDS)}")
    beta, label_smoothing = float(beta), float(label_smoothing)
    if not (beta > 0.0 and math.isfinite(beta)) or not 0.0 <= label_smoothing <= 1.0:
        raise ValueError("beta must be positive and label_smoothing lie in [0, 1]")
    if cu_seqlens is None:
        if len(rows.lead) != 2 or rows.lead[0] % 2 or rows.lead[0] == 0:
            raise AssertionError("logits must be [2 pairs, length, vocab], or packed rows with cu_seqlens")
        pairs, seq_len = rows.lead[0] // 2, rows.lead[1]
    else:
        nat.require_cuda(rows.x, cu_seqlens)
        if len(rows.lead) != 1:
            raise AssertionError("with cu_seqlens, logits must be packed: [rows, vocab]")
        if cu_seqlens.dtype != torch.int32 or cu_seqlens.dim() != 1 or cu_seqlens.numel() < 3 or \
                cu_seqlens.numel() % 2 == 0:
            raise AssertionError("cu_seqlens must be int32 [2 pairs + 1]")
        cu_seqlens = cu_seqlens.contiguous()
        pairs, seq_len = cu_seqlens.numel() // 2, 0
    denom = float(pairs) if denom is None else float(denom)
    if not (denom > 0.0 and math.isfinite(denom)):
        raise ValueError("denom must be positive")
    with nat.on_device(rows.dev):
        buf, wide, stats, coef = rows.workspace(pairs)
        g, spec = rows.new_grad() if with_grad else (None, None)
        out = rows.new(3 * pairs + 1)
        at = out.data_ptr()
        nat.call("eco_preference", ctypes.byref(rows.spec), rows.tokens.data_ptr(), nat.ptr(rows.mask), ref.data_ptr(),
                 nat.ptr(cu_seqlens), seq_len, pairs, _KINDS[kind], beta, label_smoothing, int(bool(average)), denom,
                 rows.gain, wide, stats, coef, at, at + 8 * pairs, at + 12 * pairs,
                 ctypes.byref(spec) if with_grad else None, nat.stream())
    log_ratio, margin, loss = out.split_with_sizes((2 * pairs, pairs, 1))
    return (buf, stats, coef), loss.view(()), log_ratio, margin, g


def preference_loss_grad(logits: torch.Tensor, tokens: torch.Tensor, ref_logp: torch.Tensor, *, beta: float = 0.1,
                         kind: str = "sigmoid", label_smoothing: float = 0.0, average: bool = False,
                         mask: torch.Tensor | None = None, cu_seqlens: torch.Tensor | None = None,
                         temperature: float = 1.0, s_out: float | None = None,
                         denom: float | None = None) -> PreferenceLoss:
    """Loss over pairs of sequences, and its gradient with respect to the logits.

    ``logits`` ``[2 pairs, length, vocab]``: the preferred sequences, then the rejected ones in
    the same order; or packed ``[rows, vocab]`` with ``cu_seqlens`` int32 ``[2 pairs + 1]`` on the
    device, not decreasing (rows outside ``[cu_seqlens[0], cu_seqlens[-1])`` do not count; offsets beyond the rows
    are cut there).  ``ref_logp``: the reference's log-probability of each token
    (``token_logprobs``).  With ``D`` a sequence's sum over its counting rows of ``logp - ref_logp``
    (``average``: over their number; 0 for a sequence without any) and ``h = beta (D_preferred -
    D_rejected)``::

        sigmoid: -(1 - e) log sigmoid(h) - e log sigmoid(-h)     e = label_smoothing
        hinge:   max(0, 1 - h)
        ipo:     (h / beta - 1 / (2 beta))^2

    (``label_smoothing`` belongs to ``sigmoid``; the others ignore it.)  ``loss``: the sum over the
    pairs by ``denom``, by default their number.  A sequence's gradient needs all its rows, so
    the logits are read twice."""
    rows = _Rows(logits, tokens, mask, temperature, s_out)
    _, loss, log_ratio, margin, g = _preference(rows, True, ref_logp, beta, kind, label_smoothing, average, cu_seqlens,
                                                denom)
    return PreferenceLoss(loss, g, log_ratio, margin)


class _PreferenceLoss(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, tokens, mask, temperature, s_out, *how):
        rows = _Rows(logits, tokens, mask, temperature, s_out)
        work, loss, log_ratio, margin, _ = _preference(rows, False, *how)
        _keep_rows(ctx, rows, *work)
        ctx.mark_non_differentiable(log_ratio, margin)
        ctx.set_materialize_grads(False)
        return loss, log_ratio, margin

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dloss, *_):
        if dloss is None:
            return (None,) * 12
        rows, stats, coef = _saved_rows(ctx)
        return (rows.token_grad(stats, coef, dloss),) + (None,) * 11


def preference_loss(logits: torch.Tensor, tokens: torch.Tensor, ref_logp: torch.Tensor, *, beta: float = 0.1,
                    kind: str = "sigmoid", label_smoothing: float = 0.0, average: bool = False,
                    mask: torch.Tensor | None = None, cu_seqlens: torch.Tensor | None = None,
                    temperature: float = 1.0, s_out: float | None = None,
                    denom: float | None = None) -> PreferenceLoss:
    """``preference_loss_grad`` as a differentiable loss (``.grad`` is None; call
    ``.loss.backward()``).  Gradients flow to the logits alone."""
    loss, log_ratio, margin = _PreferenceLoss.apply(logits, tokens, mask, temperature, s_out, ref_logp, beta, kind,
                                                    label_smoothing, average, cu_seqlens, denom)
    return PreferenceLoss(loss, None, log_ratio, margin)
