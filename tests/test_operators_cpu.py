"""Objectives on log-probabilities and eight-bit activations: what needs no GPU.

The oracles of both against finite differences and against PyTorch's own formulas, and the
refusals of the C entry points (no call here launches anything).
"""

import ctypes
import math

import pytest
import torch

from oracle import ckpt8 as c8
from oracle import token_losses as tl


def _differences(f, x, g, directions=5):
    """Central differences along random directions: h^2 / 6 of the third derivative and eps |f| / h."""
    gen = torch.Generator().manual_seed(0)
    h = 1e-5
    for _ in range(directions):
        d = torch.randn(x.shape, generator=gen, dtype=torch.float64)
        d /= d.norm()
        diff = (f(x + h * d) - f(x - h * d)) / (2 * h)
        assert abs(float(diff - (g * d).sum())) <= 1e-7 * (1 + float(g.norm()))


def _logits(rows, cols, seed):
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, cols, dtype=torch.float64, generator=gen)
    tokens = torch.randint(0, cols, (rows,), generator=gen)
    tokens[1] = -100
    mask = torch.rand(rows, generator=gen) < 0.8
    return x, tokens, tl.counting(tokens, cols, mask), gen


def test_oracle_policy_loss_and_its_gradient():
    x, tokens, keep, gen = _logits(14, 23, 1)
    lp = tl.token_logprobs(x, tokens, keep)
    old, adv = lp + 0.2 * torch.randn(14, generator=gen), torch.randn(14, generator=gen)
    ref = lp + 0.2 * torch.randn(14, generator=gen)
    f = lambda v: tl.policy_loss(v, tokens, old, adv, ref, keep, 0.8, 1.2, 0.1)[0]  # noqa: E731
    leaf = x.clone().requires_grad_()
    (g,) = torch.autograd.grad(f(leaf), leaf)
    _differences(f, x, g)
    assert (g[~keep] == 0).all()
    # and written as a minimum of gains
    r = torch.exp(lp - old)
    gain = torch.minimum(adv * r, adv * r.clamp(0.8, 1.2))
    k = torch.exp(ref - lp) - (ref - lp) - 1
    want = (0.1 * k - gain)[keep].sum() / keep.sum()
    assert abs(float(f(x) - want)) <= 1e-12


@pytest.mark.parametrize("kind", ["sigmoid", "hinge", "ipo"])
@pytest.mark.parametrize("average", [False, True])
def test_oracle_preference_loss_and_its_gradient(kind, average):
    x, tokens, keep, gen = _logits(20, 9, 2)
    ref = torch.randn(20, generator=gen, dtype=torch.float64) - 2
    bounds = [(0, 6), (6, 6), (7, 13), (13, 20)]
    f = lambda v: tl.preference_loss(v, tokens, ref, keep, bounds, 0.3, kind, 0.1, average)[0]  # noqa: E731
    leaf = x.clone().requires_grad_()
    (g,) = torch.autograd.grad(f(leaf), leaf)
    _differences(f, x, g)
    assert (g[6] == 0).all()  # a row between two sequences


def test_oracle_eight_bits():
    x = torch.randn(3, 300)
    x[0] = 0
    x[1, 140] = math.nan
    v = c8.stands_for(x)
    assert (v[0] == 0).all() and torch.isnan(v[1, 128:256]).all() and torch.isfinite(v[1, :128]).all()
    amax = x[2, :128].abs().max()
    assert (v[2, :128] - x[2, :128].double()).abs().max() <= amax / 127 * 0.501
    assert (v[2, :128].abs().max() - amax).abs() <= amax * 2.0 ** -23
    # already on its grid, it stays there
    again = c8.stands_for(v[2:].float())
    assert (again - v[2:]).abs().max() <= 4 * 2.0 ** -24


def test_oracle_rms_norm_and_gated_gradients_at_exact_inputs():
    """Where the eight bits stand for the input itself, the backward is the true derivative."""
    gen = torch.Generator().manual_seed(3)
    q = torch.randint(-127, 128, (2, 128), generator=gen).double()
    q[:, 5] = 127.0
    x = q / 128  # amax 127 / 128: the scale is 2^-7, exactly
    assert torch.equal(c8.stands_for(x), x)
    w, dy = torch.rand(128, generator=gen).double(), torch.randn(2, 128, generator=gen).double()
    _, dx, dw = c8.rms_norm(x, w, dy, 1e-3)
    rms = lambda v, u: (v * torch.rsqrt(v.square().mean(1, keepdim=True) + 1e-3) * u * dy).sum()  # noqa: E731
    _differences(lambda v: rms(v, w), x, dx)
    _differences(lambda u: rms(x, u), w, dw)
    for act, fn in (("silu", torch.nn.functional.silu), ("gelu", torch.nn.functional.gelu)):
        _, dg, du = c8.gated(x, x.flip(1), dy, act)
        _differences(lambda v: (fn(v) * x.flip(1) * dy).sum(), x, dg)
        _differences(lambda v: (fn(x) * v * dy).sum(), x.flip(1), du)


# ------------------------------------------------------------------ refusals of the C entry points


def _lib():
    from ecoint8 import _native

    return _native, _native.load()


def _refused(rc, code, text):
    from ecoint8 import _native

    assert rc == code and text in _native.last_error(), (rc, _native.last_error())


def _logits_spec(**how):
    from ecoint8 import _native as nat

    v = dict(x=4096, type=nat.BF16, pad_=0, n0=1, n1=4, s0=0, s1=64, cols=64, mul=1.0)
    v.update(how)
    return ctypes.byref(nat.Logits(*v.values()))


def test_token_objectives_refuse_bad_arguments():
    nat, lib = _lib()
    bad = [(dict(cols=0), -1, "shape"), (dict(n1=-1), -1, "shape"), (dict(type=9), -1, "type"),
           (dict(mul=0.0), -1, "factor"), (dict(mul=1e31), -1, "factor"),
           (dict(mul=math.nan), -1, "factor"), (dict(x=4097), -2, "aligned"),
           (dict(x=None), -1, "null"), (dict(s1=-64), -1, "strides"), (dict(n0=1 << 20, n1=1 << 12), -1, "2^30 rows"),
           (dict(n1=(1 << 30) + 1), -1, "2^30 rows"),
           (dict(cols=(1 << 28) + 1), -1, "2^28")]
    for how, code, text in bad:
        _refused(lib.eco_token_logp(_logits_spec(**how), 8192, None, None, 0, 8192, None, None, None, None), code, text)
    _refused(lib.eco_token_logp(_logits_spec(), 8192, None, None, 0, None, None, None, None, None), -1, "output")
    _refused(lib.eco_token_logp(_logits_spec(), 8192, None, 8192, 0, 8192, None, None, None, None), -1, "sequences")
    grad = lambda *a: ctypes.byref(nat.Grad(*a))  # noqa: E731
    call = lambda g, **how: lib.eco_token_grad(_logits_spec(**how), 8192, 8192, 8192, None, 1.0, g, None)  # noqa: E731
    _refused(call(grad(None, 0, 64)), -1, "gradient layout")
    _refused(call(grad(8192, 0, 32)), -1, "gradient layout")
    _refused(call(grad(8194, 0, 64)), -2, "modulo 8 elements")
    _refused(call(grad(8192, 0, 65)), -2, "modulo 8 elements")
    _refused(call(grad(8196, 0, 64), type=nat.I8), -2, "modulo 16 elements")
    _refused(lib.eco_token_grad(_logits_spec(), 8192, None, 8192, None, 1.0, grad(8192, 0, 64), None), -1, "statistics")
    policy = lambda lo, hi, kl, old=8192, dn=0.0: lib.eco_policy_grad(  # noqa: E731
        _logits_spec(), 8192, None, old, 8192, None, lo, hi, kl, dn, 1.0, 8192, 8192, 8192, grad(8192, 0, 64), None)
    _refused(policy(1.2, 0.8, 0.0), -1, "clip range")
    _refused(policy(0.8, 1.2, math.inf), -1, "clip range")
    _refused(policy(0.8, 1.2, 0.0, old=None), -1, "null")
    _refused(lib.eco_policy_forward(_logits_spec(), 8192, None, 8192, 8192, None, 0.8, 1.2, 0.0, 0.0, None, None, 8192,
                                    8192, 8192, None), -1, "null")
    pairs = lambda **h: lib.eco_preference(  # noqa: E731
        _logits_spec(n1=8), 8192, None, h.get("ref", 8192), None, h.get("s", 4), h.get("pairs", 1), h.get("kind", 0),
        h.get("beta", 0.1), h.get("smooth", 0.0), 0, h.get("denom", 1.0), 1.0, 8192, 8192, 8192, 8192, 8192, 8192,
        h.get("grad"), None)
    _refused(pairs(s=5), -1, "more sequences")
    _refused(pairs(pairs=0), -1, "bad arguments")
    _refused(pairs(ref=None), -1, "bad arguments")
    _refused(pairs(kind=3), -1, "kind")
    _refused(pairs(grad=grad(8194, 0, 64)), -2, "modulo 8 elements")
    for h in (dict(beta=0.0), dict(beta=math.nan), dict(smooth=1.5), dict(denom=0.0)):
        _refused(pairs(**h), -1, "beta")


def test_eight_bit_activations_refuse_bad_arguments():
    nat, lib = _lib()
    ok = ctypes.byref(nat.SavedI8(8192, 8192, 64, 1))
    _refused(lib.eco_ckpt_pack(8192, 3, 4, 64, 64, ok, None), -1, "type")
    _refused(lib.eco_ckpt_pack(8192, 0, 4, 0, 64, ok, None), -1, "shape")
    _refused(lib.eco_ckpt_pack(8193, 0, 4, 64, 64, ok, None), -1, "input")
    for saved in ((None, 8192, 64, 1), (8192, 8192, 63, 1), (8192, 8192, 48, 1), (8200, 8192, 64, 1),
                  (8192, 8192, 64, 0), (8192, 8194, 64, 1)):
        _refused(lib.eco_ckpt_pack(8192, 0, 4, 64, 64, ctypes.byref(nat.SavedI8(*saved)), None), -1, "eight-bit")
    _refused(lib.eco_ckpt_restore(ok, 1, 4, 63, 8192, 63, None), -1, "too short")
    _refused(lib.eco_ckpt_restore(ok, 1, 4, 64, 8200, 64, None), -2, "eight elements")
    _refused(lib.eco_gated_act(8192, 64, 8192, 64, 0, 2, 4, 64, 8192, 64, ok, ok, None), -1, "activation")
    _refused(lib.eco_gated_act(8192, 64, 8192, 64, 0, 0, 4, 64, 8192, 64, ok, None, None), -1, "missing")
    _refused(lib.eco_gated_act_bwd(8192, 64, 0, 0, 4, 64, ok, ok, 8192, 32, 8192, 64, None), -1, "outputs")
    _refused(lib.eco_rms_norm(8192, 64, 1, 4, 64, 8192, 2, 1e-6, 8192, 64, ok, 8192, None), -1, "weight")
    _refused(lib.eco_rms_norm(8192, 64, 1, 4, 64, 8192, 1, -1.0, 8192, 64, ok, 8192, None), -1, "eps")
    _refused(lib.eco_rms_norm_bwd(8192, 64, 1, 4, 64, 8192, 1, ok, 8192, 8192, 64, 8192, 8192, 10, None), -1, "scratch")
    _refused(lib.eco_rms_norm_bwd(8192, 64, 1, 4, 64, None, 1, ok, 8192, 8192, 64, 8192, 8192, 1 << 20, None), -1,
             "needs the weight")
    assert lib.eco_rms_norm_bwd_scratch(0, 64) == 0 and lib.eco_rms_norm_bwd_scratch(4, 63) >= 64


def test_no_cpu_path():
    import ecoint8

    x, t = torch.zeros(4, 8), torch.zeros(4, dtype=torch.int64)
    z = torch.zeros(4)
    for f in (lambda: ecoint8.token_logprobs(x, t), lambda: ecoint8.policy_loss(x, t, z, z),
              lambda: ecoint8.preference_loss(x[None], t[None], z[None]), lambda: ecoint8.checkpoint_i8(x),
              lambda: ecoint8.rms_norm_i8(x), lambda: ecoint8.gated_act_i8(x)):
        with pytest.raises(RuntimeError, match="CUDA"):
            f()
