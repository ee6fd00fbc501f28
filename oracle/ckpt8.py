"""Activations in eight bits, in 64 bits (oracle; test infrastructure only).

The definition's fp32 roundings (the gain ``127 / amax``, ``x * gain`` and the scale ``amax / 127``)
are taken from fp64 results, which are exact or innocuously rounded twice; everything after
them is fp64.
"""

from __future__ import annotations

import math

import torch

BLOCK = 128
TINY = 2.0 ** -119


def stands_for(x):
    """fp64: the values that ``x`` (``[rows, cols]``, any type) stands for in eight bits."""
    out = []
    for part in x.double().split(BLOCK, 1):
        amax = part.abs().amax(1, keepdim=True)
        bad = ~torch.isfinite(part).all(1, keepdim=True)
        live = (amax >= TINY) & ~bad
        safe = torch.where(live, amax, 1.0)
        gain = (127.0 / safe).float().double()
        q = torch.round((torch.where(live, part, 0.0) * gain).float().double())
        v = torch.where(live, q * (safe / 127.0).float().double(), 0.0)
        out.append(torch.where(bad, math.nan, v))
    return torch.cat(out, 1)


def rms_norm(x, w, dy, eps):
    """``(y, dx, dw)`` with the backward on what the saved eight bits stand for."""
    x64, dy = x.double(), dy.double()
    w = torch.ones(x.shape[1], dtype=torch.float64, device=x.device) if w is None else w.double()
    rstd = 1 / torch.sqrt(x64.square().mean(1, keepdim=True) + eps)
    u = stands_for(x) * rstd
    dx = rstd * (w * dy - u * (w * dy * u).mean(1, keepdim=True))
    return x64 * rstd * w, dx, (dy * u).sum(0)


def gated(gate, up, dy, act):
    """``(y, dgate, dup)``."""
    fn = torch.nn.functional.silu if act == "silu" else torch.nn.functional.gelu
    y = fn(gate.double()) * up.double()
    with torch.enable_grad():
        g, u = stands_for(gate).requires_grad_(), stands_for(up).requires_grad_()
        dg, du = torch.autograd.grad(fn(g) * u, (g, u), dy.double())
    return y, dg, du
