"""Objectives on token log-probabilities (``ecoint8.losses``) against the oracle in 64 bits.

Tolerances.  With S the spread of a row's logits (over the temperature) and K a bound of the
longest chain of additions in a row's sum (a thread's vectors, at most 16 up to 4096 of them and
one per 512 beyond; half a vector's terms, at most 8; at most 10 joins: below cols / 32 + 24 up to
1024 columns, cols / 128 + 24 up to 8192, cols / 512 + 24 beyond), the kernel's probabilities are
off by the relative error

    e = 2^-24 (6 S + K + 24):

the exponent (x - m) c has three roundings (the difference, the factor, the product), each at
most S 2^-24, in the term and again in the sum; each term's exponential and each addition adds
a few 2^-24 (2^-22 for the exponential).  A
log-probability is then off by e plus its own rounding |lp| 2^-24, a coefficient by its
derivative with respect to lp times that, and a stored gradient by half a step of its type.
"""

import math

import pytest
import torch

from oracle import token_losses as orc

pytestmark = pytest.mark.gpu

TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16, "int8": torch.int8}
S_OUT = 0.05


def _adds(cols):
    return (cols // 32 if cols <= 1024 else cols // 128 if cols <= 8192 else cols // 512) + 24


def _err(x):
    """The relative error of the kernel's probabilities for fp64 logits ``x``, per row."""
    x = torch.nan_to_num(x, nan=0.0, posinf=0.0, neginf=0.0)
    spread = x.amax(-1) - x.amin(-1)
    return (6 * spread + _adds(x.shape[-1])) * 2.0 ** -24


def _half_step(dtype):
    return torch.finfo(dtype).eps / 2


def _case(dtype, lead, cols, seed, keep=0.7, shifted=False, scale=2.0):
    gen = torch.Generator().manual_seed(seed)
    stored = (*lead[:-1], lead[-1] + 1) if shifted else lead
    x = torch.randn(*stored, cols, generator=gen) * scale
    if dtype == torch.int8:
        x = (x / S_OUT).round().clamp(-127, 127)
    x = x.to(dtype).cuda()
    x = x[:, :-1] if shifted else x
    tokens = torch.randint(0, cols, lead, generator=gen).cuda()
    mask = (torch.rand(lead, generator=gen) < keep).cuda()
    return x, tokens, mask, gen


def _fp64(x, temperature=1.0):
    x = x.double() * S_OUT if x.dtype == torch.int8 else x.double()
    return x, x / temperature


def _check_grad(got, want, x, coef, coef_err, unit, note=""):
    """|got - want| against the module's bound; ``coef`` fp64 per row, ``coef_err`` its absolute error."""
    p = torch.softmax(torch.nan_to_num(x), -1)
    # a 16-bit gradient's exponent takes in the coefficient: below 2^9 + 2^7 in size, rounded twice
    e = _err(x)[..., None] + (2.0 ** -14 if got.dtype != torch.float32 else 0.0)
    c, ce = coef.abs()[..., None], coef_err[..., None]
    tiny = torch.finfo(got.dtype).tiny * torch.finfo(got.dtype).eps  # half of the smallest subnormal step, and ftz
    tol = want.abs() * _half_step(got.dtype) + (c * e * unit + ce * unit) * (p + (want.abs() > c * 0.5 * unit)) + \
        c * unit * 2.0 ** -23 * (want.abs() > 0) + max(tiny, 2.0 ** -126) + ce * unit * p
    bad = (got.double() - want).abs() > tol
    assert not bad.any(), (note, int(bad.sum()), float(((got.double() - want).abs() / tol).max()))


# --------------------------------------------------------------------- log-probabilities

SHAPES = [((1,), 1), ((3,), 2), ((5,), 7), ((64,), 1000), ((33,), 1024), ((9,), 1025), ((7,), 4097), ((5,), 8192),
          ((4,), 8193), ((3,), 50257), ((2, 3), 777), ((2, 5), 12289), ((300,), 5)]


@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("lead,cols", SHAPES)
def test_token_logprobs_and_their_gradient(name, lead, cols):
    from ecoint8.losses import token_logprobs

    dtype, t = TYPES[name], 0.8
    x, tokens, mask, gen = _case(dtype, lead, cols, 11 * cols + len(lead))
    tokens.view(-1)[0] = -100 if tokens.numel() > 2 else tokens.view(-1)[0]
    raw, x64 = _fp64(x, t)
    raw.requires_grad_()
    keep = orc.counting(tokens, cols, mask)
    want = orc.token_logprobs(raw / t, tokens, keep)
    leaf = x.detach().requires_grad_() if dtype != torch.int8 else x
    got = token_logprobs(leaf, tokens, mask=mask, temperature=t, s_out=S_OUT if dtype == torch.int8 else None)
    tol = _err(x64) + want.abs() * 2.0 ** -24
    assert got.dtype == torch.float32 and got.shape == tokens.shape
    assert ((got.double() - want).abs() <= tol).all()
    assert (got[~keep] == 0).all()
    if dtype == torch.int8:
        return
    up = torch.randn(lead, generator=gen).cuda()
    (g,) = torch.autograd.grad(got, leaf, up)
    (gw,) = torch.autograd.grad(want, raw, up.double())
    assert g.dtype == dtype and g.shape == x.shape
    coef = torch.where(keep, up.double(), 0.0)
    _check_grad(g, gw, x64, coef, torch.zeros_like(coef), 1 / t)


@pytest.mark.parametrize("name", ["fp32", "bf16", "fp16"])
def test_strided_logits_are_read_in_place(name):
    """A vocabulary cut off a padded one, at an odd offset, and every other row."""
    from ecoint8.losses import token_logprobs

    dtype = TYPES[name]
    gen = torch.Generator().manual_seed(3)
    big = torch.randn(12, 1111, generator=gen).to(dtype).cuda()
    for x in (big[:, 3:1004], big[::2, 1:], big[::3, 5:6], big.t()[:700].t(), big[1:2].expand(6, -1)):
        tokens = torch.randint(0, x.shape[1], (x.shape[0],), generator=gen).cuda()
        keep = orc.counting(tokens, x.shape[1])
        leaf = x.detach().requires_grad_()
        raw = x.double().requires_grad_()
        got, want = token_logprobs(leaf, tokens), orc.token_logprobs(raw, tokens, keep)
        assert ((got.double() - want).abs() <= _err(x.double()) + want.abs() * 2.0 ** -24).all()
        (g,) = torch.autograd.grad(got.sum(), leaf)
        (gw,) = torch.autograd.grad(want.sum(), raw)
        one = torch.ones_like(want)
        _check_grad(g, gw, x.double(), one, one * 0, 1.0)


def test_far_and_minus_infinite_logits():
    from ecoint8.losses import token_logprobs

    x = torch.full((4, 1500), -math.inf)
    x[0, 7] = 3.0                              # one token possible
    x[1, ::2] = torch.linspace(-80, 80, 750)   # half the vocabulary banned, far apart
    x[2] = torch.finfo(torch.float32).min      # masked to the type's lowest value but for two
    x[2, [5, 900]] = torch.tensor([1.0, 2.0])
    x[3, 1] = 0.0                              # the token itself is banned
    low = torch.full((1, 1500), torch.finfo(torch.float32).min).cuda()  # nothing but the lowest value: uniform
    got = token_logprobs(low, torch.tensor([3]).cuda())
    assert abs(float(got) + math.log(1500)) <= _adds(1500) * 2.0 ** -24 + 8 * 2.0 ** -24
    tokens = torch.tensor([7, 1400, 900, 2])
    want = torch.log_softmax(x.double(), -1).gather(1, tokens[:, None])[:, 0]
    leaf = x.cuda().requires_grad_()
    got = token_logprobs(leaf, tokens.cuda())
    # the module's bound with the spread of what has weight: 0, 160 and 1
    tol = torch.tensor([_adds(1500), 6 * 160 + _adds(1500), 6 + _adds(1500), 0.0]) * 2.0 ** -24
    assert (got.cpu().double()[:3] - want[:3]).abs().le(tol[:3] + want[:3].abs() * 2.0 ** -24).all()
    assert got[3] == -math.inf
    (g,) = torch.autograd.grad(got[:3].sum(), leaf)
    p = torch.softmax(x.double(), -1)
    wg = torch.nn.functional.one_hot(tokens, 1500).double() - p
    wg[3] = 0
    assert (g.cpu().double() - wg).abs().max() <= (6 * 160 + _adds(1500)) * 2.0 ** -24


def test_rows_that_do_not_count_may_hold_anything():
    from ecoint8.losses import policy_loss_grad, token_logprobs

    x, tokens, _, gen = _case(torch.bfloat16, (40,), 3001, 5)
    mask = torch.zeros(40, dtype=torch.bool)
    mask[[0, 7, 39]] = True
    bad = x.clone()
    bad[~mask.cuda()] = float("nan")
    bad[3] = float("inf")
    tokens[~mask.cuda()] = -100
    tokens[5] = 3001
    clean = token_logprobs(x, tokens, mask=mask.cuda())
    assert torch.equal(token_logprobs(bad, tokens, mask=mask.cuda()), clean)
    assert torch.equal(token_logprobs(bad, tokens), clean)  # by the tokens alone
    old, adv = clean + 0.1, torch.randn(40, generator=gen).cuda()
    old[~mask.cuda()] = float("nan")
    adv[~mask.cuda()] = float("inf")
    a = policy_loss_grad(x, tokens, old, adv, ref_logp=old, kl_coef=0.1, mask=mask.cuda())
    b = policy_loss_grad(bad, tokens, old, adv, ref_logp=old, kl_coef=0.1)
    for u, v in zip(a, b):
        assert torch.equal(u, v) and torch.isfinite(u).all()
    assert (b.grad[~mask.cuda()] == 0).all() and (b.grad[mask.cuda()] != 0).any()


def test_a_row_of_nan_that_counts_gives_nan():
    from ecoint8.losses import policy_loss_grad, token_logprobs

    x, tokens, _, _ = _case(torch.float32, (6,), 2000, 6)
    x[2, 1999] = float("nan")
    x[4, 3] = float("inf")
    lp = token_logprobs(x, tokens)
    assert torch.isnan(lp[[2, 4]]).all() and torch.isfinite(lp[[0, 1, 3, 5]]).all()
    r = policy_loss_grad(x, tokens, torch.zeros(6).cuda(), torch.ones(6).cuda())
    assert torch.isnan(r.loss) and torch.isnan(r.grad[2]).all() and torch.isfinite(r.grad[0]).all()


# --------------------------------------------------------------------- policy loss


def _policy_inputs(x64, tokens, gen):
    lead = tokens.shape
    lp = torch.log_softmax(torch.nan_to_num(x64), -1).gather(-1, tokens.clamp(0, x64.shape[-1] - 1)[..., None])[..., 0]
    old = (lp + torch.randn(lead, generator=gen).cuda() * 0.3).float()
    ref = (lp + torch.randn(lead, generator=gen).cuda() * 0.2).float()
    adv = torch.randn(lead, generator=gen).cuda()
    return old, adv, ref


def _check_policy(r, grad, x, raw, x64, tokens, mask, old, adv, ref, t, kl, lo, hi, denom=None):
    cols = x.shape[-1]
    keep = orc.counting(tokens, cols, mask)
    raw = raw.detach().requires_grad_()
    loss, lp, klm, clip = orc.policy_loss(raw / t, tokens, old, adv, ref, keep, 1 - lo, 1 + hi, kl, denom)
    (gw,) = torch.autograd.grad(loss, raw) if keep.any() else (torch.zeros_like(raw),)
    lp = lp.detach()
    n = max(1, int(keep.sum())) if denom is None else denom
    # lp in the kernel's loss is fp64 of fp32 sums: off by e; r and exp(ref - lp) are fp32 exponentials
    e = _err(x64) + 2.0 ** -22
    ratio = torch.where(keep, torch.exp(lp - old.double()), 0.0)
    back = torch.exp(ref.double() - lp) if ref is not None else torch.zeros_like(lp)
    size = torch.where(keep, adv.double().abs() * ratio + abs(kl) * (back + 1), 0.0)
    # a ratio within its error of a clip border may fall on either side: none does in these inputs
    for edge in (1 - lo, 1 + hi):
        assert not (keep & ((ratio - edge).abs() <= 4 * e * ratio) & (adv != 0)).any()
    loss_tol = float((size * 4 * torch.where(keep, e, 0.0)).sum() / n + loss.abs() * 2.0 ** -23)
    assert abs(r.loss.double() - loss) <= loss_tol
    assert ((r.logp.double() - lp).abs() <= e + lp.abs() * 2.0 ** -24).all()
    d = torch.where(keep, back + 1 + (ref.double() - lp).abs(), 0.0) if ref is not None else torch.zeros_like(lp)
    assert abs(r.kl.double() - klm) <= float((d * 2 * torch.where(keep, e, 0.0)).sum() / n)
    assert abs(r.clip_fraction.double() - clip) <= clip * 2.0 ** -23
    coef = gw.gather(-1, tokens.clamp(0, cols - 1)[..., None])[..., 0]
    p_at = torch.exp(lp)
    free, held = -adv.double() * ratio, -adv.double() * ratio.clamp(1 - lo, 1 + hi)
    coef = torch.where(keep, torch.where(free < held, 0.0, free) - kl * (back - 1 if ref is not None else 0.0), 0.0) / n
    _check_grad(grad, gw, x64, coef, torch.where(keep, size / n * 4 * e, 0.0), 1 / t)
    del p_at


@pytest.mark.parametrize("form", ["grad", "autograd"])
@pytest.mark.parametrize("name", TYPES)
@pytest.mark.parametrize("lead,cols,shifted", [((1,), 3, False), ((37,), 1000, False), ((3, 11), 1001, True),
                                               ((2, 9), 5000, True), ((6,), 8200, False), ((2, 2), 50257, True)])
def test_policy_loss(form, name, lead, cols, shifted):
    from ecoint8.losses import policy_loss, policy_loss_grad

    dtype = TYPES[name]
    if form == "autograd" and dtype == torch.int8:
        pytest.skip("int8 logits carry no gradient")
    t, kl, lo, hi = 0.9, 0.05, 0.2, 0.28
    x, tokens, mask, gen = _case(dtype, lead, cols, cols + 5, shifted=shifted)
    mask.view(-1)[0] = True
    raw, x64 = _fp64(x, t)
    old, adv, ref = _policy_inputs(x64, tokens, gen)
    how = dict(ref_logp=ref, mask=mask, clip_low=lo, clip_high=hi, kl_coef=kl, temperature=t,
               s_out=S_OUT if dtype == torch.int8 else None)
    if form == "grad":
        r = policy_loss_grad(x, tokens, old, adv, **how)
        grad = r.grad
    else:
        leaf = x.detach().requires_grad_()
        r = policy_loss(leaf, tokens, old, adv, **how)
        (grad,) = torch.autograd.grad(r.loss, leaf)
    assert grad.shape == x.shape and grad.dtype == (torch.float32 if dtype == torch.int8 else dtype)
    _check_policy(r, grad, x, raw, x64, tokens, mask, old, adv, ref, t, kl, lo, hi)


# More rows than are in work at a time, several times over, for each width that is treated in
# its own way (by 16-byte vectors per row: up to 256, 512, 1024, 2048, and two sizes beyond).
MANY = [("fp32", (12007,), 37), ("bf16", (3, 4001), 1001), ("int8", (12007,), 503), ("fp16", (6007,), 3001),
        ("fp32", (2, 3001), 2000), ("int8", (6007,), 8001), ("bf16", (3001,), 8192), ("int8", (2501,), 12345),
        ("fp16", (2, 751), 12001), ("fp32", (1501,), 8001), ("int8", (1201,), 32000), ("bf16", (2, 451), 17003),
        ("fp32", (901,), 9001), ("int8", (901,), 40001), ("bf16", (501,), 150001), ("fp32", (2, 251), 75003)]


@pytest.mark.parametrize("name,lead,cols", MANY)
def test_rows_of_every_width_many_times_over(name, lead, cols):
    from ecoint8.losses import policy_loss_grad, token_logprobs

    t, kl, lo, hi = 0.9, 0.05, 0.2, 0.28
    x, tokens, mask, gen = _case(TYPES[name], lead, cols, cols, shifted=len(lead) == 2)
    tokens.view(-1)[::11] = -100
    tokens.view(-1)[5::101] = cols
    raw, x64 = _fp64(x, t)
    old, adv, ref = _policy_inputs(x64, tokens, gen)
    lp = orc.token_logprobs(x64, tokens, orc.counting(tokens, cols))
    for edge in (1 - lo, 1 + hi):  # ratios at a border of the clip may fall on either side: kept away from it
        old = torch.where((torch.exp(lp - old.double()) - edge).abs() < 1e-3, old + 0.01, old)
    s_out = S_OUT if name == "int8" else None
    got = token_logprobs(x, tokens, mask=mask, temperature=t, s_out=s_out)
    keep = orc.counting(tokens, cols, mask)
    want = torch.where(keep, lp, 0.0)
    assert ((got.double() - want).abs() <= _err(x64) + want.abs() * 2.0 ** -24).all()
    r = policy_loss_grad(x, tokens, old, adv, ref_logp=ref, mask=mask, clip_low=lo, clip_high=hi, kl_coef=kl,
                         temperature=t, s_out=s_out)
    _check_policy(r, r.grad, x, raw, x64, tokens, mask, old, adv, ref, t, kl, lo, hi)


def test_policy_without_reference_with_a_given_denominator_and_upstream_gradient():
    from ecoint8.losses import policy_loss, policy_loss_grad

    x, tokens, mask, gen = _case(torch.float32, (50,), 2049, 8)
    raw, x64 = _fp64(x)
    old, adv, _ = _policy_inputs(x64, tokens, gen)
    r = policy_loss_grad(x, tokens, old, adv, mask=mask, denom=123.0)
    _check_policy(r, r.grad, x, raw, x64, tokens, mask, old, adv, None, 1.0, 0.0, 0.2, 0.2, denom=123.0)
    assert r.kl == 0
    leaf = x.detach().requires_grad_()
    s = policy_loss(leaf, tokens, old, adv, mask=mask, denom=123.0)
    (s.loss * 4.0).backward()
    assert torch.equal(leaf.grad, r.grad * 4.0)  # a power of two scales every rounding alike


def test_no_row_counts_and_no_rows():
    from ecoint8.losses import policy_loss, policy_loss_grad, preference_loss_grad, token_logprobs

    x, tokens, _, _ = _case(torch.bfloat16, (5,), 1200, 9)
    z = torch.zeros(5, device="cuda")
    r = policy_loss_grad(x * float("nan"), tokens, z, z, mask=torch.zeros(5, dtype=torch.bool, device="cuda"))
    assert r.loss == 0 and r.kl == 0 and r.clip_fraction == 0 and (r.grad == 0).all() and (r.logp == 0).all()
    e, te, ze = x[:0], tokens[:0], z[:0]
    r = policy_loss_grad(e, te, ze, ze)
    assert r.loss == 0 and r.grad.shape == (0, 1200)
    leaf = e.detach().requires_grad_()
    policy_loss(leaf, te, ze, ze).loss.backward()
    assert leaf.grad.shape == (0, 1200)
    assert token_logprobs(e, te).shape == (0,)
    p = preference_loss_grad(x[None, :0].expand(2, 0, 1200), tokens[None, :0].expand(2, 0), z[:0].expand(2, 0))
    assert abs(float(p.loss) - math.log(2)) <= 2.0 ** -24 and (p.margin == 0).all()


def test_policy_gradient_against_differences():
    """Central differences of the kernel's own loss along random directions: with |d|_2 = 1 the
    third derivative of a row's term is below 8 (|A| r <= 8 here), so the truncation is at most
    8 h^2 / 6, and the losses' rounding 2^-23 |loss| / h."""
    from ecoint8.losses import policy_loss_grad

    x, tokens, _, gen = _case(torch.float32, (12,), 300, 21, scale=1.0)
    old, adv, ref = _policy_inputs(x.double(), tokens, gen)
    f = lambda v: policy_loss_grad(v, tokens, old, adv.clamp(-2, 2), ref_logp=ref, kl_coef=0.1, clip_low=1.0,  # noqa: E731
                                   clip_high=1e6)
    base = f(x)
    h = 2.0 ** -6
    for _ in range(4):
        d = torch.randn(x.shape, generator=gen).cuda()
        d /= d.norm()
        up, down = f(x + h * d).loss.double(), f(x - h * d).loss.double()
        diff, want = (up - down) / (2 * h), (base.grad.double() * d.double()).sum()
        tol = 8 * h * h / 6 + (base.loss.abs().double() + 1) * 2.0 ** -22 / h
        assert abs(diff - want) <= tol


# --------------------------------------------------------------------- preference loss


@pytest.mark.parametrize("form", ["grad", "autograd"])
@pytest.mark.parametrize("kind,average,smooth", [("sigmoid", False, 0.0), ("sigmoid", True, 0.2), ("hinge", False, 0.0),
                                                 ("ipo", True, 0.0)])
@pytest.mark.parametrize("name,cols,packed", [("fp32", 130, False), ("bf16", 1025, True), ("fp16", 9001, True),
                                              ("bf16", 777, False)])
def test_preference_loss(form, kind, average, smooth, name, cols, packed):
    from ecoint8.losses import preference_loss, preference_loss_grad

    dtype, pairs, s, beta = TYPES[name], 3, 13, 0.1
    if packed:
        lens = [13, 0, 1, 7, 5, 0]  # an empty preferred sequence, an empty rejected one
        ends = [2]  # two rows in front of the first, some behind the last
        for n in lens:
            ends.append(ends[-1] + n)
        lead, cu = (ends[-1] + 5,), torch.tensor(ends, dtype=torch.int32).cuda()
        bounds = list(zip(ends, ends[1:]))
    else:
        lead, cu, bounds = (2 * pairs, s), None, [(i * s, (i + 1) * s) for i in range(2 * pairs)]
    x, tokens, mask, gen = _case(dtype, lead, cols, cols, keep=0.8)
    tokens.view(-1)[3] = -100
    if not packed:
        mask[1] = False  # a sequence without any row that counts
    ref = (torch.log_softmax(x.double(), -1).gather(-1, tokens.clamp(min=0)[..., None])[..., 0]
           + torch.randn(lead, generator=gen).cuda() * 0.5).float()
    ref[~mask] = float("nan")
    raw = x.double().requires_grad_()
    keep = orc.counting(tokens, cols, mask, cu)
    loss, ratios, h = orc.preference_loss(raw, tokens, torch.nan_to_num(ref), keep, bounds, beta, kind, smooth,
                                          average)
    (gw,) = torch.autograd.grad(loss, raw)
    how = dict(beta=beta, kind=kind, label_smoothing=smooth, average=average, mask=mask, cu_seqlens=cu)
    if form == "grad":
        r = preference_loss_grad(x, tokens, ref, **how)
        grad = r.grad
    else:
        leaf = x.detach().requires_grad_()
        r = preference_loss(leaf, tokens, ref, **how)
        (grad,) = torch.autograd.grad(r.loss, leaf)
    e = _err(raw.detach())
    off = torch.stack([torch.where(keep, e, 0.0).reshape(-1)[a:b].sum() for a, b in bounds])  # of each sum
    assert ((r.log_ratio.double() - ratios).abs() <= off + ratios.abs() * 2.0 ** -24).all()
    dh = beta * (off[:pairs] + off[pairs:])
    assert ((r.margin.double() - h).abs() <= dh + h.abs() * 2.0 ** -24).all()
    # |d loss / d h| is at most 1 (sigmoid, hinge), 2 |off| / beta (ipo)
    slope = torch.ones_like(h) if kind != "ipo" else 2 * (h / beta - 0.5 / beta).abs() / beta + dh
    assert abs(r.loss.double() - loss) <= float((slope * dh).sum() / pairs + loss.abs() * 2.0 ** -23)
    coef = torch.zeros(keep.numel(), dtype=torch.float64, device="cuda")
    cerr = torch.zeros_like(coef)
    flat = keep.reshape(-1)
    with torch.enable_grad():
        hh = h.detach().requires_grad_()
        each, _ = _pair_terms(hh, kind, smooth, beta)
        (dl,) = torch.autograd.grad(each.sum() / pairs, hh)
    curve = 0.25 if kind == "sigmoid" else 2 / beta ** 2  # of the loss in h (hinge: constant slope)
    for q, (a, b) in enumerate(bounds):
        n = max(1, int(flat[a:b].sum())) if average else 1
        coef[a:b] = torch.where(flat[a:b], dl[q % pairs] * beta * (1 if q < pairs else -1) / n, 0.0)
        cerr[a:b] = torch.where(flat[a:b], curve * dh[q % pairs] * beta / pairs / n, 0.0)
    _check_grad(grad, gw, raw.detach(), coef.view(lead), cerr.view(lead), 1.0)


def _pair_terms(h, kind, smooth, beta):
    ls = torch.nn.functional.logsigmoid
    if kind == "sigmoid":
        return -(1 - smooth) * ls(h) - smooth * ls(-h), None
    if kind == "hinge":
        return (1 - h).clamp(min=0), None
    return (h / beta - 1 / (2 * beta)) ** 2, None


def test_offsets_outside_the_rows_are_cut():
    """cu_seqlens lives on the device, so its values cannot be refused; they are cut to the rows."""
    from ecoint8.losses import preference_loss_grad

    x, tokens, _, _ = _case(torch.float32, (10,), 40, 4)
    ref = torch.zeros(10, device="cuda")
    good = preference_loss_grad(x, tokens, ref, cu_seqlens=torch.tensor([0, 6, 10], dtype=torch.int32).cuda())
    cut = preference_loss_grad(x, tokens, ref, cu_seqlens=torch.tensor([-3, 6, 1 << 30], dtype=torch.int32).cuda())
    for a, b in zip(good, cut):
        assert torch.equal(a, b)
    back = preference_loss_grad(x, tokens, ref, cu_seqlens=torch.tensor([8, 6, 9], dtype=torch.int32).cuda())
    assert torch.isfinite(back.grad).all()


# --------------------------------------------------------------------- one call and another


def test_same_call_same_bits_on_another_stream_and_in_a_graph():
    from ecoint8.losses import policy_loss_grad, preference_loss_grad

    x, tokens, mask, gen = _case(torch.bfloat16, (4, 33), 4099, 13)
    old, adv, ref = _policy_inputs(x.double(), tokens, gen)

    def both():
        a = policy_loss_grad(x, tokens, old, adv, ref_logp=ref, kl_coef=0.1, mask=mask)
        return [*a, *preference_loss_grad(x, tokens, ref, mask=mask)]

    want = both()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = both()
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = both()
    second = torch.cuda.CUDAGraph()
    with torch.cuda.graph(second):
        again = both()
    new = torch.randn(x.shape, generator=gen).to(x.dtype).cuda()
    x.copy_(new)
    graph.replay()
    second.replay()
    want = both()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) and torch.equal(a, c) for a, b, c in zip(want, out, again))


def test_offsets_beyond_32_bits():
    """Logits of more than 2^31 values: the last rows are found."""
    from ecoint8.losses import policy_loss_grad, token_logprobs

    rows, cols = 16500, 131072
    x = torch.zeros(rows, cols, dtype=torch.bfloat16, device="cuda")
    tokens = torch.full((rows,), -100, device="cuda")
    tokens[-2:] = torch.tensor([cols - 1, 5])
    x[-2, cols - 1] = 7.0
    lp = token_logprobs(x, tokens)
    want = torch.log_softmax(x[-2:].double(), -1)[[0, 1], [cols - 1, 5]]
    assert ((lp[-2:].double() - want).abs() <= 2.0 ** -24 * (14 + _adds(cols) + 12)).all() and (lp[:-2] == 0).all()
    r = policy_loss_grad(x, tokens, lp, torch.ones(rows, device="cuda"))
    p = torch.softmax(x[-2:].double(), -1)
    wg = p / 2
    wg[[0, 1], [cols - 1, 5]] -= 0.5
    assert ((r.grad[-2:].double() - wg).abs() <= wg.abs() * (2.0 ** -8 + 2.0 ** -14) + 2.0 ** -126).all()
    assert not r.grad[:-2].any()


def test_refusals():
    from ecoint8.losses import policy_loss_grad, preference_loss_grad, token_logprobs

    x, tokens, mask, _ = _case(torch.float32, (6,), 50, 1)
    z = torch.zeros(6, device="cuda")
    for bad in (lambda: token_logprobs(x.double(), tokens), lambda: token_logprobs(x[0], tokens[0]),
                lambda: token_logprobs(x, tokens.int()), lambda: token_logprobs(x, tokens[:5]),
                lambda: token_logprobs(x, tokens, mask=z), lambda: token_logprobs(x[:, :0], tokens),
                lambda: policy_loss_grad(x, tokens, z.double(), z),
                lambda: policy_loss_grad(x, tokens, z, torch.zeros(4, device="cuda")),
                lambda: preference_loss_grad(x, tokens, z),
                lambda: preference_loss_grad(x[None].expand(3, -1, -1), tokens[None].expand(3, -1), z),
                lambda: preference_loss_grad(x, tokens, z, cu_seqlens=torch.tensor([0, 3, 6], device="cuda")),
                lambda: preference_loss_grad(x, tokens, z, cu_seqlens=torch.tensor([0, 6], dtype=torch.int32).cuda()),
                lambda: preference_loss_grad(x, tokens, z,
                                             cu_seqlens=torch.tensor([0, 2, 4, 6], dtype=torch.int32).cuda())):
        with pytest.raises(AssertionError):
            bad()
    for bad in (lambda: token_logprobs(x, tokens, temperature=0.0), lambda: token_logprobs(x, tokens, s_out=0.1),
                lambda: token_logprobs(x.to(torch.int8), tokens),
                lambda: token_logprobs(x.to(torch.int8), tokens, s_out=-1.0),
                lambda: policy_loss_grad(x, tokens, z, z, kl_coef=0.1),
                lambda: policy_loss_grad(x, tokens, z, z, clip_low=1.5),
                lambda: policy_loss_grad(x, tokens, z, z, denom=float("nan")),
                lambda: preference_loss_grad(x[None].expand(2, -1, -1), tokens[None].expand(2, -1), z, kind="other"),
                lambda: preference_loss_grad(x[None].expand(2, -1, -1), tokens[None].expand(2, -1), z, beta=0.0)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(RuntimeError, match="CUDA"):
        token_logprobs(x.cpu(), tokens.cpu())


def test_byte_masks_and_graphs_side_by_side():
    """A uint8 mask counts where it is not zero; two captured calls replay on two streams at once."""
    from ecoint8.losses import policy_loss_grad, preference_loss_grad

    x, tokens, mask, gen = _case(torch.bfloat16, (400,), 9000, 2)
    raw, x64 = _fp64(x)
    old, adv, ref = _policy_inputs(x64, tokens, gen)
    want = policy_loss_grad(x, tokens, old, adv, mask=mask)
    got = policy_loss_grad(x, tokens, old, adv, mask=mask.to(torch.uint8) * 7)
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    cu = torch.tensor([0, 90, 210, 333, 400], dtype=torch.int32).cuda()
    calls = (lambda: policy_loss_grad(x, tokens, old, adv, mask=mask), lambda: preference_loss_grad(
        x, tokens, ref, mask=mask, cu_seqlens=cu))
    wants = [c() for c in calls]
    streams = [torch.cuda.Stream() for _ in calls]
    graphs, outs = [], []
    torch.cuda.synchronize()
    for c, st in zip(calls, streams):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1], stream=st):
            outs.append(c())
    for _ in range(5):
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
    torch.cuda.synchronize()
    for w, o in zip(wants, outs):
        assert all(torch.equal(a, b) for a, b in zip(w, o))


def test_factors_that_would_leave_the_range_of_fp32_are_refused():
    from ecoint8.losses import token_logprobs

    x, tokens, _, _ = _case(torch.float32, (6,), 50, 1)
    for bad in (dict(temperature=1e-40), dict(temperature=1e40), dict(temperature=float("nan"))):
        with pytest.raises(ValueError):
            token_logprobs(x, tokens, **bad)
    with pytest.raises(ValueError):
        token_logprobs(x.to(torch.int8), tokens, s_out=1e30)
    # at the border every row is still its maximum and nothing else
    got = token_logprobs(x, x.argmax(1), temperature=1e-15)
    assert (got == 0).all()


# --------------------------------------------------------------------- as they are used


def test_strict_int8_training_step_on_the_policy_loss():
    """I8Sequential -> policy_loss_grad on its int8 logits -> int8 gradient -> backward_i8 -> I8ECO."""
    from ecoint8 import I8ECO, I8Linear, I8ReLU, I8Sequential
    from ecoint8.losses import policy_loss_grad, token_logprobs
    from ecoint8.quant import quantize_tensor_dynamic

    torch.manual_seed(0)
    net = I8Sequential(I8Linear(32, 64), I8ReLU(), I8Linear(64, 10)).cuda()
    X = torch.randn(128, 32)
    x0, sx0 = quantize_tensor_dynamic(X)
    net.calibrate(x0.cuda(), sx0)
    opt = I8ECO(net.int8_layers())
    x_i8 = net.quantize_input(X)[0].cuda()
    gen = torch.Generator().manual_seed(1)
    tokens = torch.randint(0, 10, (128,), generator=gen).cuda()
    adv = torch.randn(128, generator=gen).cuda()
    before = [l.w_i8.clone() for l in net.int8_layers()]
    logits, s_out = net.forward_i8(x_i8)
    old = token_logprobs(logits, tokens, s_out=s_out)
    r = policy_loss_grad(logits, tokens, old, adv, s_out=s_out)
    # every ratio is 1: the loss is -mean(A), the gradient the policy gradient's
    assert abs(float(r.loss) + float(adv.double().mean())) <= 2.0 ** -20 and r.clip_fraction == 0
    x64 = logits.double() * s_out
    want = -(adv.double()[:, None] / 128) * (torch.nn.functional.one_hot(tokens, 10) - torch.softmax(x64, -1))
    assert ((r.grad.double() - want).abs() <= want.abs() * 2.0 ** -18 + adv.abs().double()[:, None] * 2.0 ** -25).all()
    g_i8, s_g = quantize_tensor_dynamic(r.grad, stochastic=True)
    net.backward_i8(g_i8, s_g)
    opt.step()
    assert any(not torch.equal(a, l.w_i8) for a, l in zip(before, net.int8_layers()))


def test_int8_linear_head_trains_on_the_preference_loss():
    """Autograd through Int8Linear: the head's input gradient is the loss's gradient through
    the layer's own backward."""
    from ecoint8 import EcoSGDM, Int8Linear
    from ecoint8.losses import preference_loss, preference_loss_grad

    torch.manual_seed(0)
    head = Int8Linear(48, 301).cuda()
    h = torch.randn(4 * 11, 48).cuda().requires_grad_()
    tokens = torch.randint(0, 301, (4, 11)).cuda()
    ref = torch.full((4, 11), -5.0).cuda()
    logits = head(h).view(4, 11, 301)
    loss = preference_loss(logits, tokens, ref)
    loss.loss.backward()
    want = preference_loss_grad(logits.detach(), tokens, ref).grad
    again = head(h)
    (gh,) = torch.autograd.grad(again, h, want.reshape(44, 301))
    assert torch.equal(gh, h.grad) and torch.isfinite(gh).all() and gh.any()
    before = head.w_i8.clone()
    EcoSGDM([head], lr=1.0).step()
    assert not torch.equal(before, head.w_i8)
