"""Objectives on token log-probabilities in 64 bits (oracle; test infrastructure only).

The formulas of ``ecoint8.losses``, one PyTorch expression each, on fp64 logits of any device;
gradients come from automatic differentiation.
"""

from __future__ import annotations

import torch


def counting(tokens, cols, mask=None, cu=None):
    """Which rows count."""
    keep = (tokens >= 0) & (tokens < cols)
    if mask is not None:
        keep = keep & mask.bool()
    if cu is not None:
        r = torch.arange(tokens.numel(), device=tokens.device).view(tokens.shape)
        keep = keep & (r >= cu[0]) & (r < cu[-1])
    return keep


def token_logprobs(x, tokens, keep):
    """``[...]`` fp64: log softmax at the token, 0 (and no gradient) where a row does not count."""
    flat, k = x.reshape(-1, x.shape[-1]), keep.reshape(-1)
    rows = flat[k]
    lp = torch.log_softmax(rows, -1).gather(-1, tokens.reshape(-1)[k][:, None])[:, 0]
    return torch.zeros(k.shape, dtype=x.dtype, device=x.device).masked_scatter(k, lp).view(tokens.shape)


def policy_loss(x, tokens, old, adv, ref=None, keep=None, low=0.8, high=1.2, kl_coef=0.0, denom=None):
    """``(loss, logp, kl, clip_fraction)``."""
    lp = token_logprobs(x, tokens, keep)
    n = max(1, int(keep.sum())) if denom is None else denom
    r = torch.exp(lp - old.double())
    free, held = -adv.double() * r, -adv.double() * r.clamp(low, high)
    kl = torch.zeros_like(lp)
    if ref is not None:
        d = ref.double() - lp
        kl = torch.expm1(d) - d
    zero = torch.zeros_like(lp)
    each = torch.where(free < held, held.detach(), free) + kl_coef * kl
    total = lambda t: torch.where(keep, t, zero).sum() / n  # noqa: E731
    return total(each), lp, total(kl), total((free < held).double())


def preference_loss(x, tokens, ref, keep, bounds, beta=0.1, kind="sigmoid", smooth=0.0, average=False, denom=None):
    """``(loss, log ratios, margins)``; ``bounds``: the sequences' ``(first, last + 1)`` rows, preferred first."""
    gap = torch.where(keep, token_logprobs(x, tokens, keep) - ref.double(), 0.0).reshape(-1)
    k = keep.reshape(-1)
    ratios = [gap[a:b].sum() / (max(1, int(k[a:b].sum())) if average else 1) for a, b in bounds]
    ratios = torch.stack(ratios)
    pairs = len(bounds) // 2
    h = beta * (ratios[:pairs] - ratios[pairs:])
    if kind == "sigmoid":
        ls = torch.nn.functional.logsigmoid
        each = -(1 - smooth) * ls(h) - smooth * ls(-h)
    elif kind == "hinge":
        each = (1 - h).clamp(min=0)
    else:
        each = (h / beta - 1 / (2 * beta)) ** 2
    return each.sum() / (pairs if denom is None else denom), ratios, h
