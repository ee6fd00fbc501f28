"""Measured operators of ``ecoint8``: training objectives on a model's logits, and activations kept in eight bits.

Five operators, each with its gradient:

* ``policy``      clipped policy loss with a KL term, from logits (``ecoint8.losses.policy_loss_grad`` and
                  ``policy_loss``), and the token log-probabilities it starts from (``token_logprobs``);
* ``preference``  loss over pairs of log ratios, from logits (``preference_loss_grad``, ``preference_loss``);
* ``rms``         root-mean-square norm whose saved input is eight bits (``ecoint8.checkpoint.rms_norm_i8``);
* ``gated``       gated activation whose saved inputs are eight bits (``gated_act_i8``);
* ``pack``        a tensor put away in eight bits and brought back (``checkpoint_i8``, ``restore_i8``).

Eight bits means: blocks of 128 consecutive columns of a row share the fp32 scale ``amax / 127``;
``q = rint(fl32(x * fl32(127 / amax)))`` and the value it stands for is ``q * scale``.
"""

import math
import os
import sys

import torch

own = False

_TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16, "int8": torch.int8}
_BYTES = {"fp32": 4, "bf16": 2, "fp16": 2, "int8": 1}
_CLIP_LOW, _CLIP_HIGH = 0.2, 0.28
_S_OUT = 0.05  # the scale of int8 logits
_EPS = 1e-6
_BLOCK = 128


def _package():
    """This repository's package (reached only where ``own`` is true)."""
    root = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "eco-int8-opt_b200")
    if root not in sys.path:
        sys.path.insert(0, root)
    import ecoint8.checkpoint
    import ecoint8.losses

    return ecoint8


def listed():
    return [
        # a rollout's last few tokens on the 1000-way int8 head: the call's latency
        {"name": "policy_few_int8", "op": "policy", "form": "grad", "dtype": "int8", "b": 1, "s": 16, "v": 1000,
         "shifted": False, "kept": 1.0, "kl": 0.05, "temp": 1.0},
        # prompts and answers of one micro-batch, logits shifted by one against the tokens, odd vocabulary,
        # prompt tokens masked: no row starts on 16 bytes
        {"name": "policy_shifted_odd_fp16", "op": "policy", "form": "autograd", "dtype": "fp16", "b": 6, "s": 347,
         "v": 50257, "shifted": True, "kept": 0.6, "kl": 0.02, "temp": 0.9},
        # a full micro-batch of answers over a large vocabulary
        {"name": "policy_large_bf16", "op": "policy", "form": "grad", "dtype": "bf16", "b": 8, "s": 1024,
         "v": 131072, "shifted": False, "kept": 0.9, "kl": 0.05, "temp": 1.0},
        # log-probabilities of given tokens with their gradient (maximum likelihood on chosen tokens)
        {"name": "logprobs_fp32", "op": "policy", "form": "logprobs", "dtype": "fp32", "b": 4, "s": 512,
         "v": 32000, "shifted": False, "kept": 1.0, "kl": 0.0, "temp": 1.0},
        # two short pairs, one after the other in a padded batch
        {"name": "preference_few_fp32", "op": "preference", "form": "grad", "dtype": "fp32", "pairs": 2, "s": 48,
         "v": 1000, "packed": False, "kind": "sigmoid", "average": False, "smooth": 0.0},
        # pairs of ragged answers packed without padding, a few rows behind the last one
        {"name": "preference_packed_bf16", "op": "preference", "form": "grad", "dtype": "bf16", "pairs": 8, "s": 509,
         "v": 65536, "packed": True, "kind": "sigmoid", "average": False, "smooth": 0.1},
        # the norm of a handful of tokens
        {"name": "rms_few_bf16", "op": "rms", "dtype": "bf16", "t": 48, "c": 4096},
        # the batch and width of the wide configuration, fp32 as Int8Linear takes it
        {"name": "rms_large_fp32", "op": "rms", "dtype": "fp32", "t": 16384, "c": 8192},
        # a handful of tokens at an odd width
        {"name": "gated_few_odd_fp32", "op": "gated", "dtype": "fp32", "t": 37, "f": 1337, "act": "gelu"},
        # gate and up halves of one projection in a training batch
        {"name": "gated_large_bf16", "op": "gated", "dtype": "bf16", "t": 16384, "f": 8192, "act": "silu"},
        # the 784-wide input of a small network
        {"name": "pack_small_fp32", "op": "pack", "dtype": "fp32", "t": 128, "c": 784},
        # a layer's activations of one training batch
        {"name": "pack_large_bf16", "op": "pack", "dtype": "bf16", "t": 16384, "c": 8192},
    ]


def _spread(rng, low, high):
    """A whole number spread over the logarithm of [low, high]."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["policy", "policy", "preference", "rms", "gated", "pack"])
    floats = ["fp32", "bf16", "fp16"]
    if op == "policy":
        dtype, v = rng.choice(floats + ["int8"]), _spread(rng, 2, 131072)
        s = _spread(rng, 1, 1500)
        b = max(1, min(_spread(rng, 1, 64), (1 << 29) // (v * s)))
        form = rng.choice(["grad", "autograd", "logprobs"]) if dtype != "int8" else "grad"
        return {"op": op, "form": form, "dtype": dtype, "b": b, "s": max(1, min(s, (1 << 29) // v)), "v": v,
                "shifted": rng.random() < 0.4, "kept": rng.choice([0.1, 0.4, 0.8, 1.0]),
                "kl": rng.choice([0.0, 0.04]), "temp": rng.choice([1.0, 0.7])}
    if op == "preference":
        v, s = _spread(rng, 2, 131072), _spread(rng, 1, 1000)
        pairs = max(1, min(_spread(rng, 1, 16), (1 << 28) // (v * s)))
        return {"op": op, "form": rng.choice(["grad", "autograd"]), "dtype": rng.choice(floats), "pairs": pairs,
                "s": max(1, min(s, (1 << 28) // v)), "v": v, "packed": rng.random() < 0.5,
                "kind": rng.choice(["sigmoid", "hinge", "ipo"]), "average": rng.random() < 0.3,
                "smooth": rng.choice([0.0, 0.1])}
    width = _spread(rng, 1, 16384)
    t = max(1, min(_spread(rng, 1, 16384), (1 << 26) // width))
    if op == "gated":
        return {"op": op, "dtype": rng.choice(floats), "t": t, "f": width, "act": rng.choice(["silu", "gelu"])}
    return {"op": op, "dtype": rng.choice(floats), "t": t, "c": width}


def _randn(shape, gen, scale, dtype):
    return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32).mul_(scale).to(dtype)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = _TYPES[case["dtype"]]
    st = {"case": case}
    if case["op"] in ("policy", "preference"):
        v = case["v"]
        if case["op"] == "policy":
            lead = (case["b"], case["s"])
        elif case["packed"]:
            lens = torch.randint(0, case["s"] + 1, (2 * case["pairs"],), generator=gen, device="cuda")
            lens[0] = case["s"]
            st["cu"] = torch.cat([lens.new_zeros(1), lens.cumsum(0)]).to(torch.int32)
            lead = (2 * case["pairs"] * case["s"],)  # rows behind the last sequence belong to none
        else:
            lead = (2 * case["pairs"], case["s"])
        stored = (lead[0], lead[1] + 1) if case.get("shifted") else lead
        rows = math.prod(stored)
        flat = torch.empty((rows, v), device="cuda", dtype=dtype)
        tokens = torch.randint(0, v, (rows,), generator=gen, device="cuda")
        logp = torch.empty(rows, device="cuda", dtype=torch.float32)
        step = max(1, (1 << 28) // v)
        for i in range(0, rows, step):  # in parts: the largest logits fill gigabytes
            y = tokens[i:i + step, None]
            x = torch.randn((y.shape[0], v), generator=gen, device="cuda", dtype=torch.float32).mul_(2.0)
            # a sampled token is a likely one
            x.scatter_add_(1, y, torch.randn((y.shape[0], 1), generator=gen, device="cuda").add_(math.log(v) + 2.0))
            x = (x / _S_OUT).round().clamp(-127, 127) if dtype == torch.int8 else x
            flat[i:i + step] = x.to(dtype)
            x = (x * _S_OUT if dtype == torch.int8 else x) / case.get("temp", 1.0)
            logp[i:i + step] = x.gather(1, y)[:, 0] - torch.logsumexp(x, 1)
        cut = (slice(None), slice(0, lead[-1])) if case.get("shifted") else (slice(None),)
        st["logits"] = flat.view(*stored, v)[cut]
        st["tokens"] = tokens.view(stored)[cut].contiguous()
        logp = logp.view(stored)[cut].contiguous()
        st["ref"] = logp + torch.randn(lead, generator=gen, device="cuda") * 0.1
        kept = case.get("kept", 0.8)
        st["mask"] = torch.rand(lead, generator=gen, device="cuda") < kept
        st["mask"].view(-1)[0] = True
        if case["op"] == "policy":
            st["old"] = logp + torch.randn(lead, generator=gen, device="cuda") * 0.15
            st["adv"] = torch.randn((case["b"], 1), generator=gen, device="cuda").add_(0.5).expand(lead).contiguous()
            st["dlogp"] = torch.randn(lead, generator=gen, device="cuda") / max(1, math.prod(lead))
        return st
    t, c = case["t"], case.get("c", case.get("f", 0) * 2)
    x = torch.randn((t, c), generator=gen, device="cuda", dtype=torch.float32)
    # activations have columns far above the others
    x.mul_(torch.rand((c,), generator=gen, device="cuda").mul_(2.5).exp_().mul_(0.5))
    st["x"] = x.to(dtype)
    if case["op"] == "rms":
        st["w"] = torch.rand((c,), generator=gen, device="cuda").add_(0.5).to(dtype)
        st["dy"] = _randn((t, c), gen, 0.1, dtype)
    elif case["op"] == "gated":
        st["dy"] = _randn((t, case["f"]), gen, 0.1, dtype)
    return st


# ---------------------------------------------------------------- plain forms


def _in_logits(st):
    """Logits as fp32 numbers over the temperature, the tokens, and which rows count."""
    case = st["case"]
    x = st["logits"].to(torch.float32)
    x = x * _S_OUT if case["dtype"] == "int8" else x
    return x / case.get("temp", 1.0)


def _softmax_parts(x, tokens):
    """``(log-probability of each token in 64 bits, exp(x - max), its row sums)``."""
    m = x.amax(-1, keepdim=True)
    e = (x - m).exp()
    total = e.sum(-1, keepdim=True)
    at = x.gather(-1, tokens[..., None])
    return ((at - m).to(torch.float64) - total.to(torch.float64).log())[..., 0], e, total


def _row_gradient(e, total, tokens, coef, dtype):
    """``coef * (one at the token - probabilities)`` for each row, rounded to ``dtype``."""
    coef = coef.to(torch.float32)[..., None]
    g = e * (-coef / total)
    g.scatter_add_(-1, tokens[..., None], coef)
    return g.to(dtype)


def _plain_policy(st):
    case, tokens, mask = st["case"], st["tokens"], st["mask"]
    out = torch.float32 if case["dtype"] == "int8" else _TYPES[case["dtype"]]
    logp, e, total = _softmax_parts(_in_logits(st), tokens)
    if case["form"] == "logprobs":
        zero = torch.zeros_like(logp)
        coef = torch.where(mask, st["dlogp"].to(torch.float64), zero) / case["temp"]
        return {"logp": torch.where(mask, logp, zero).to(torch.float32),
                "grad": _row_gradient(e, total, tokens, coef, out)}
    n = mask.sum().clamp(min=1).to(torch.float64)
    adv = st["adv"].to(torch.float64)
    ratio = (logp - st["old"].to(torch.float64)).exp()
    free, held = -adv * ratio, -adv * ratio.clamp(1.0 - _CLIP_LOW, 1.0 + _CLIP_HIGH)
    behind = st["ref"].to(torch.float64) - logp
    kl = torch.expm1(behind) - behind
    zero = torch.zeros_like(logp)
    loss = torch.where(mask, torch.maximum(free, held) + case["kl"] * kl, zero).sum() / n
    coef = torch.where(free >= held, free, zero) - case["kl"] * torch.expm1(behind)
    coef = torch.where(mask, coef, zero) / (n * case["temp"])
    return {"loss": loss.to(torch.float32), "grad": _row_gradient(e, total, tokens, coef, out),
            "logp": torch.where(mask, logp, zero).to(torch.float32),
            "kl": (torch.where(mask, kl, zero).sum() / n).to(torch.float32),
            "clip_fraction": ((mask & (free < held)).sum() / n).to(torch.float32)}


def _plain_preference(st):
    case, tokens, mask, pairs = st["case"], st["tokens"], st["mask"], st["case"]["pairs"]
    logp, e, total = _softmax_parts(_in_logits(st), tokens)
    if case["packed"]:
        owner = torch.bucketize(torch.arange(tokens.numel(), device=tokens.device), st["cu"][1:], right=True)
    else:
        owner = torch.arange(2 * pairs, device=tokens.device).repeat_interleave(case["s"])
    owner, keep = owner.reshape(tokens.shape), mask
    keep = keep & (owner < 2 * pairs)
    owner = owner.clamp(max=2 * pairs - 1)
    zero = torch.zeros_like(logp)
    gap = torch.where(keep, logp - st["ref"].to(torch.float64), zero)
    ratios = gap.new_zeros(2 * pairs).index_add_(0, owner.reshape(-1), gap.reshape(-1))
    count = gap.new_zeros(2 * pairs).index_add_(0, owner.reshape(-1), keep.reshape(-1).to(torch.float64))
    per = count.clamp(min=1) if case["average"] else torch.ones_like(count)
    ratios = ratios / per
    beta, smooth = 0.1, case["smooth"]
    margin = beta * (ratios[:pairs] - ratios[pairs:])
    if case["kind"] == "sigmoid":
        far = (-margin.abs()).exp().log1p()
        loss = (1 - smooth) * (far + (-margin).clamp(min=0)) + smooth * (far + margin.clamp(min=0))
        slope = 1 / (1 + (-margin).exp()) - (1 - smooth)
    elif case["kind"] == "hinge":
        loss, slope = (1 - margin).clamp(min=0), -(margin < 1).to(torch.float64)
    else:
        off = margin / beta - 1 / (2 * beta)
        loss, slope = off * off, 2 * off / beta
    slope = slope * beta / pairs
    coef = torch.where(keep, (torch.cat([slope, -slope]) / per)[owner], zero)
    return {"loss": (loss.sum() / pairs).to(torch.float32),
            "grad": _row_gradient(e, total, tokens, coef, _TYPES[case["dtype"]]),
            "log_ratio": ratios.to(torch.float32), "margin": margin.to(torch.float32)}


def _plain_pack(x):
    """Eight-bit values and scales of ``x`` in blocks of 128 columns: ``(q, scale)`` as fp32 [t, blocks, 128], [t, blocks, 1]."""
    t, c = x.shape
    blocks = torch.zeros((t, -(-c // _BLOCK), _BLOCK), dtype=torch.float32, device=x.device)
    blocks.view(t, -1)[:, :c] = x
    amax = blocks.abs().amax(-1, keepdim=True)
    top = torch.full_like(amax, 127.0)  # tensors on both sides: a Python number would divide as its reciprocal
    q = (blocks * torch.where(amax > 0, top / amax, torch.zeros_like(amax))).round().clamp(-127, 127)
    return q, amax / top


def _plain_restore(q, scale, c):
    return (q * scale).view(q.shape[0], -1)[:, :c]


def _plain_rms(st):
    x, w, dy = st["x"].to(torch.float32), st["w"].to(torch.float32), st["dy"].to(torch.float32)
    c = x.shape[1]
    rstd = 1 / ((x * x).mean(1, keepdim=True) + _EPS).sqrt()
    y = x * rstd * w
    unit = _plain_restore(*_plain_pack(x), c) * rstd
    wdy = w * dy
    dx = rstd * (wdy - unit * (wdy * unit).mean(1, keepdim=True))
    dw = (dy * unit).sum(0, dtype=torch.float64)
    dtype = st["x"].dtype
    return {"y": y.to(dtype), "dx": dx.to(dtype), "dw": dw.to(dtype)}


def _plain_gated(st):
    f, silu = st["case"]["f"], st["case"]["act"] == "silu"
    x, dy = st["x"].to(torch.float32), st["dy"].to(torch.float32)
    gate, up = x[:, :f], x[:, f:]

    def slope(g):  # the activation's value over its input, and its derivative
        if silu:
            s = 1 / (1 + (-g).exp())
            return s, s * (1 + g * (1 - s))
        s = 0.5 * (1 + torch.erf(g * (1 / math.sqrt(2))))
        return s, s + g * (g * g * -0.5).exp() * (1 / math.sqrt(2 * math.pi))

    h = gate * slope(gate)[0] * up
    gate, up = _plain_restore(*_plain_pack(gate), f), _plain_restore(*_plain_pack(up), f)
    s, d = slope(gate)
    dx = torch.cat([dy * up * d, dy * gate * s], 1)
    dtype = st["x"].dtype
    return {"y": h.to(dtype), "dx": dx.to(dtype)}


def run(state):
    case, op = state["case"], state["case"]["op"]
    if own:
        return _own_run(state, case, op)
    if op == "policy":
        return _plain_policy(state)
    if op == "preference":
        return _plain_preference(state)
    if op == "rms":
        return _plain_rms(state)
    if op == "gated":
        return _plain_gated(state)
    x = state["x"]
    q, scale = _plain_pack(x.to(torch.float32))
    return {"x": _plain_restore(q, scale, x.shape[1]).to(x.dtype)}


def _own_run(st, case, op):
    """The same pass through the package's public calls."""
    eco = _package()
    if op == "policy":
        grad = case["form"] == "grad"
        logits = st["logits"] if grad else st["logits"].detach().requires_grad_()
        if case["form"] == "logprobs":
            logp = eco.losses.token_logprobs(logits, st["tokens"], mask=st["mask"], temperature=case["temp"])
            return {"logp": logp.detach(), "grad": torch.autograd.grad(logp, logits, st["dlogp"])[0]}
        f = eco.losses.policy_loss_grad if grad else eco.losses.policy_loss
        r = f(logits, st["tokens"], st["old"], st["adv"], ref_logp=st["ref"], mask=st["mask"], clip_low=_CLIP_LOW,
              clip_high=_CLIP_HIGH, kl_coef=case["kl"], temperature=case["temp"],
              s_out=_S_OUT if case["dtype"] == "int8" else None)
        g = r.grad if grad else torch.autograd.grad(r.loss, logits)[0]
        return {"loss": r.loss.detach(), "grad": g, "logp": r.logp, "kl": r.kl, "clip_fraction": r.clip_fraction}
    if op == "preference":
        grad = case["form"] == "grad"
        logits = st["logits"] if grad else st["logits"].detach().requires_grad_()
        f = eco.losses.preference_loss_grad if grad else eco.losses.preference_loss
        r = f(logits, st["tokens"], st["ref"], beta=0.1, kind=case["kind"], label_smoothing=case["smooth"],
              average=case["average"], mask=st["mask"], cu_seqlens=st.get("cu"))
        g = r.grad if grad else torch.autograd.grad(r.loss, logits)[0]
        return {"loss": r.loss.detach(), "grad": g, "log_ratio": r.log_ratio, "margin": r.margin}
    if op == "pack":
        return {"x": eco.checkpoint.restore_i8(eco.checkpoint.checkpoint_i8(st["x"]))}
    x = st["x"].detach().requires_grad_()
    if op == "rms":
        w = st["w"].detach().requires_grad_()
        y = eco.checkpoint.rms_norm_i8(x, w, eps=_EPS)
        dx, dw = torch.autograd.grad(y, (x, w), st["dy"])
        return {"y": y.detach(), "dx": dx, "dw": dw}
    y = eco.checkpoint.gated_act_i8(x, act=case["act"])
    return {"y": y.detach(), "dx": torch.autograd.grad(y, x, st["dy"])[0]}


def work(case):
    size = _BYTES[case["dtype"]]
    if case["op"] in ("policy", "preference"):
        lead = case["b"] * case["s"] if case["op"] == "policy" else 2 * case["pairs"] * case["s"]
        n = lead * case["v"]
        kept = case.get("kept", 0.8) * (0.5 if case.get("packed") else 1.0)
        # the logits of rows that count read once, every row of the gradient written once
        return {"bytes": n * (size * kept + (4 if case["dtype"] == "int8" else size)) + lead * 32, "flops": 5 * n * kept}
    if case["op"] == "gated":
        n = case["t"] * case["f"]
        saved = 2 * n + 8 * case["t"] * -(-case["f"] // _BLOCK)
        # gate and up read, the product and the eight bits written; dy and the eight bits read, both gradients written
        return {"bytes": size * 6 * n + 2 * saved, "flops": 30 * n}
    n = case["t"] * case["c"]
    saved = n + 4 * case["t"] * -(-case["c"] // _BLOCK)
    if case["op"] == "rms":
        return {"bytes": size * 4 * n + 2 * saved + size * 3 * case["c"], "flops": 16 * n}
    return {"bytes": size * 2 * n + 2 * saved, "flops": 6 * n}


# ---------------------------------------------------------------- 64 bits


def exact(case, seed):
    st = prepare(case, seed)
    f64 = torch.float64
    if case["op"] in ("policy", "preference"):
        lead, v = st["tokens"].shape, case["v"]
        tokens, mask = st["tokens"].reshape(-1), st["mask"].reshape(-1)
        rows = tokens.numel()
        temp, unit = case.get("temp", 1.0), _S_OUT if case["dtype"] == "int8" else 1.0
        part = max(1, (1 << 27) // v)
        logits = st["logits"].reshape(rows, v)
        lse = torch.empty(rows, dtype=f64, device="cuda")
        at = logits.gather(1, tokens[:, None])[:, 0].to(f64) * unit / temp
        for i in range(0, rows, part):
            lse[i:i + part] = torch.logsumexp(logits[i:i + part].to(f64) * unit / temp, 1)
        # the objective as a function of the log-probabilities alone; its slope by automatic differentiation
        logp = (at - lse).requires_grad_()
        out = {}
        if case["op"] == "policy" and case["form"] == "logprobs":
            total = (logp * st["dlogp"].reshape(-1).to(f64))[mask].sum()
            shown = torch.where(mask, logp.detach(), 0.0)
            out["logp"] = shown.reshape(lead)
        elif case["op"] == "policy":
            lp = logp[mask]
            old, ref, adv = (st[k].reshape(-1)[mask].to(f64) for k in ("old", "ref", "adv"))
            r = torch.exp(lp - old)
            surrogate = torch.minimum(adv * r, adv * torch.clip(r, 1 - _CLIP_LOW, 1 + _CLIP_HIGH))
            kl = torch.exp(ref - lp) - (ref - lp) - 1
            n = max(1, lp.numel())
            total = (case["kl"] * kl - surrogate).sum() / n
            out["logp"] = torch.where(mask, logp.detach(), 0.0).reshape(lead)
            out["kl"] = kl.detach().sum() / n
            out["clip_fraction"] = (surrogate < adv * r).sum().to(f64) / n
            out["loss"] = total.detach()
        else:
            pairs = case["pairs"]
            ends = st["cu"].tolist() if case["packed"] else [i * case["s"] for i in range(2 * pairs + 1)]
            gap = torch.where(mask, logp - st["ref"].reshape(-1).to(f64), 0.0)
            ratios = torch.stack([gap[a:z].sum() / (max(1, int(mask[a:z].sum())) if case["average"] else 1)
                                  for a, z in zip(ends, ends[1:])])
            margin = 0.1 * (ratios[:pairs] - ratios[pairs:])
            if case["kind"] == "sigmoid":
                e = case["smooth"]
                each = -(1 - e) * torch.nn.functional.logsigmoid(margin) - e * torch.nn.functional.logsigmoid(-margin)
            elif case["kind"] == "hinge":
                each = torch.relu(1 - margin)
            else:
                each = (margin / 0.1 - 5.0) ** 2
            total = each.mean()
            out["log_ratio"], out["margin"], out["loss"] = ratios.detach(), margin.detach(), total.detach()
        coef = torch.autograd.grad(total, logp)[0] / temp if mask.any() else torch.zeros_like(lse)
        grad = torch.empty((rows, v), dtype=torch.float32 if unit != 1.0 or rows * v > 1 << 28 else f64, device="cuda")
        for i in range(0, rows, part):
            g = torch.exp(logits[i:i + part].to(f64) * unit / temp - lse[i:i + part, None]) * -coef[i:i + part, None]
            g[torch.arange(g.shape[0], device="cuda"), tokens[i:i + part]] += coef[i:i + part]
            grad[i:i + part] = g
        out["grad"] = grad.reshape(*lead, v)
        return out
    x = st["x"]

    def stands_for(a):
        """What the eight bits of `a` stand for: the definition's two 32-bit roundings, all else in 64 bits."""
        got = []
        for part in a.to(f64).split(_BLOCK, 1):
            top = part.abs().max(1, keepdim=True).values
            gain = torch.where(top > 0, 127 / top, 0.0).float().to(f64)
            q = torch.round((part * gain).float().to(f64)).clamp(-127, 127)
            got.append(q * (top / 127).float().to(f64))
        return torch.cat(got, 1)

    if case["op"] == "pack":
        return {"x": stands_for(x)}
    dy = st["dy"].to(f64)
    if case["op"] == "rms":
        w, wide = st["w"].to(f64), x.to(f64)
        rstd = torch.rsqrt(wide.square().mean(1, keepdim=True) + _EPS)
        y = wide * rstd * w
        kept = stands_for(x) * rstd
        inner = torch.einsum("tc,tc,c->t", dy, kept, w)[:, None] / x.shape[1]
        return {"y": y, "dx": rstd * (dy * w - kept * inner), "dw": torch.einsum("tc,tc->c", dy, kept)}
    fn = torch.nn.functional.silu if case["act"] == "silu" else torch.nn.functional.gelu
    f = case["f"]
    y = fn(x[:, :f].to(f64)) * x[:, f:].to(f64)
    gate, up = stands_for(x[:, :f]).requires_grad_(), stands_for(x[:, f:]).requires_grad_()
    return {"y": y, "dx": torch.cat(torch.autograd.grad(fn(gate) * up, (gate, up), dy), 1)}
